// Rotary positions: (a, b) -> s (a cos t - b sin t, a sin t + b cos t) for every pair of a head,
// t = 2 pi * position * turns[slot].  One launch turns query and key together.
//
// Bound by memory: every element is read and written once, the positions and the frequencies are
// a few bytes a token.  A thread owns a fixed group of slots of a token (up to 8 pairs, two 16-byte
// vectors) and walks over heads, so the angles are evaluated once for many heads and no table of
// cosines exists.  Angles: position * turns is rounded in 64 bits and only its fraction of a turn
// is kept (exact to 2^-53 of the number of turns), so far positions lose nothing; sine and cosine
// of the fraction are evaluated in 32 bits (sincospif) and the turn itself is 32-bit arithmetic,
// rounded to the tensor's type once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "agb.h"
#include "packed.h"

namespace agb {
namespace {

constexpr int THREADS = 256;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(float x) { return x; }
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half narrow(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ float narrow(float x) { return x; }

// A unit is VEC pairs (2 * VEC elements of a head) or, behind the turned part, 2 * VEC copied
// elements.  Threads are numbered (token, head lane, unit), units fastest.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const RotaryArgs p, int units, int turned_units,
                                                         int head_lanes) {
  const int64_t index = int64_t(blockIdx.x) * THREADS + threadIdx.x;
  const int unit = int(index % units);
  const int64_t rest = index / units;
  const int lane = int(rest % head_lanes);
  const int64_t token = rest / head_lanes;
  if (token >= p.tokens) return;

  const bool copies = unit >= turned_units;
  float co[VEC], si[VEC];
  if (!copies) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int slot = unit * VEC + i;
      const int64_t at = token * p.axes + (p.axis ? p.axis[slot] : 0);
      const double position = p.position_type == 0   ? double(static_cast<const int*>(p.positions)[at])
                              : p.position_type == 1 ? double(static_cast<const int64_t*>(p.positions)[at])
                                                     : double(static_cast<const float*>(p.positions)[at]);
      const double turns = position * p.turns[slot];
      const float part = float(turns - rint(turns));
      sincospif(2.f * part, &si[i], &co[i]);
      co[i] *= p.amplitude;
      si[i] *= p.amplitude * p.direction;
    }
  }
  // first elements of the unit's two vectors
  int e0, e1;
  if (copies) {
    e0 = p.turned + (unit - turned_units) * 2 * VEC;
    e1 = e0 + VEC;
  } else if (INTERLEAVED) {
    e0 = unit * 2 * VEC;
    e1 = e0 + VEC;
  } else {
    e0 = unit * VEC;
    e1 = p.turned / 2 + e0;
  }
  const bool second = e1 < p.dim;  // the copied tail may end with a single vector

  using V = Vec<T, VEC>;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const RotaryPart part = p.part[which];
    const T* src = static_cast<const T*>(part.x) + token * part.row_stride;
    T* dst = static_cast<T*>(part.out) + token * part.heads * p.dim;
#pragma unroll 4
    for (int head = lane; head < part.heads; head += head_lanes) {
      const T* from = src + head * part.head_stride;
      T* to = dst + int64_t(head) * p.dim;
      V a = *reinterpret_cast<const V*>(from + e0);
      V b{};
      if (second) b = *reinterpret_cast<const V*>(from + e1);
      if (!copies) {
        if (INTERLEAVED && VEC > 1) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            const float x0 = widen(a.v[2 * i]), y0 = widen(a.v[2 * i + 1]);
            a.v[2 * i] = narrow<T>(x0 * co[i] - y0 * si[i]);
            a.v[2 * i + 1] = narrow<T>(x0 * si[i] + y0 * co[i]);
            const int j = VEC / 2 + i;
            const float x1 = widen(b.v[2 * i]), y1 = widen(b.v[2 * i + 1]);
            b.v[2 * i] = narrow<T>(x1 * co[j] - y1 * si[j]);
            b.v[2 * i + 1] = narrow<T>(x1 * si[j] + y1 * co[j]);
          }
        } else {  // also a single interleaved pair (VEC == 1): its two elements are a and b
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float x = widen(a.v[i]), y = widen(b.v[i]);
            a.v[i] = narrow<T>(x * co[i] - y * si[i]);
            b.v[i] = narrow<T>(x * si[i] + y * co[i]);
          }
        }
      }
      *reinterpret_cast<V*>(to + e0) = a;
      if (second) *reinterpret_cast<V*>(to + e1) = b;
    }
  }
}

template <typename T, int VEC>
cudaError_t launch(const RotaryArgs& p, cudaStream_t stream) {
  const int turned_units = p.turned / 2 / VEC;
  const int tail = p.dim - p.turned;
  const int units = turned_units + (tail + 2 * VEC - 1) / (2 * VEC);
  // One thread per (token, unit) and `head_lanes` heads side by side: with many tokens a thread
  // serves several heads with the angles it has evaluated, with few every head has its own threads.
  const int heads = p.part[0].heads > p.part[1].heads ? p.part[0].heads : p.part[1].heads;
  const int64_t wanted = int64_t(p.sm_count) * 2048;
  int lanes = 1;
  while (lanes < heads && (lanes * units < 32 || p.tokens * units * lanes < wanted)) lanes *= 2;
  if (lanes > heads) lanes = heads;
  const int64_t threads = p.tokens * units * lanes;
  const int64_t blocks = (threads + THREADS - 1) / THREADS;
  if (blocks > 2147483647ll) {
    set_error_detail("rotary_embed: too many tokens for one launch");
    return cudaErrorInvalidValue;
  }
  if (p.interleaved)
    rotary_kernel<T, VEC, true><<<unsigned(blocks), THREADS, 0, stream>>>(p, units, turned_units, lanes);
  else
    rotary_kernel<T, VEC, false><<<unsigned(blocks), THREADS, 0, stream>>>(p, units, turned_units, lanes);
  return cudaGetLastError();
}

// The widest vector that every address allows: row, head and pair strides, the turned part and the
// tail are multiples of it and the base addresses are aligned to it.
template <typename T>
cudaError_t dispatch(const RotaryArgs& p, cudaStream_t stream) {
  uint64_t bits = uint64_t(p.dim) | uint64_t(p.turned / 2) | uint64_t(p.dim - p.turned);
  for (const RotaryPart& part : p.part) {
    if (part.heads == 0) continue;
    bits |= uint64_t(part.row_stride) | uint64_t(part.head_stride);
    bits |= reinterpret_cast<uint64_t>(part.x) / sizeof(T) | reinterpret_cast<uint64_t>(part.out) / sizeof(T);
  }
  constexpr int WIDEST = 16 / int(sizeof(T));
  if (bits % WIDEST == 0) return launch<T, WIDEST>(p, stream);
  if (WIDEST > 4 && bits % 4 == 0) return launch<T, 4>(p, stream);
  if (bits % 2 == 0) return launch<T, 2>(p, stream);
  return launch<T, 1>(p, stream);
}

}  // namespace

cudaError_t rotary_embed(const RotaryArgs& p, cudaStream_t stream) {
  if (p.tokens == 0) return cudaSuccess;
  switch (p.type) {
    case 0: return dispatch<__nv_bfloat16>(p, stream);
    case 1: return dispatch<__half>(p, stream);
    default: return dispatch<float>(p, stream);
  }
}

}  // namespace agb
