// Rotary positions: (a, b) -> s (a cos t - b sin t, a sin t + b cos t) for every pair of a head,
// t = 2 pi * position * turns[slot].  One launch turns query and key together.
//
// Bound by memory: every element is read and written once, the positions and the frequencies are
// a few bytes a token.  A warp serves a token, or some of its heads where there are few tokens: its
// lanes evaluate the token's sines and cosines once, exchange them through shared memory, keep those of
// their slots in registers and walk over the heads in 16-byte vectors; no table of cosines exists.
// Angles: position * turns is rounded in 64 bits and only its fraction of a turn is kept (exact to
// 2^-53 of the number of turns), so far positions lose nothing; sine and cosine of the fraction are
// evaluated in 32 bits (sincospif) and the turn itself is 32-bit arithmetic, rounded to the
// tensor's type once.
//
// 65537 tokens of 32 and 8 heads of 128, bf16 (1342 MB): 221 us, 6.1 TB/s; 8190 tokens (168 MB) 27 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "agb.h"
#include "packed.h"

namespace agb {
namespace {

constexpr int THREADS = 256;
constexpr int BATCH = 2;  // units a lane has on their way: 32 bytes each, for 32 warps an SM

// Elements travel as 32-bit words: two of a 16-bit type, one of fp32.
template <typename T> struct Word;
template <> struct Word<__nv_bfloat16> {
  static constexpr int ELEMENTS = 2;
  static __device__ __forceinline__ float2 wide(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t narrow(float2 v) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Word<__half> {
  static constexpr int ELEMENTS = 2;
  static __device__ __forceinline__ float2 wide(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ uint32_t narrow(float2 v) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Word<float> {
  static constexpr int ELEMENTS = 1;
};

template <int W> struct alignas(W * 4) Words {
  uint32_t w[W];
};

// One unit of a head.  Half layout: W words of first elements and the W words of their partners;
// interleaved: W words of whole pairs.
template <typename T, int W, bool INTERLEAVED>
struct Pairs {
  static constexpr int ELEMENTS = W * Word<T>::ELEMENTS;                     // of one vector
  static constexpr int VECTORS = INTERLEAVED ? 1 : 2;
  static constexpr int SLOTS = INTERLEAVED ? ELEMENTS / 2 : ELEMENTS;
  static_assert(!INTERLEAVED || ELEMENTS >= 2, "a vector holds whole pairs");

  static __device__ __forceinline__ void turn(Words<W>& a, Words<W>& b, const float (&co)[SLOTS], const float (&si)[SLOTS]) {
    if constexpr (Word<T>::ELEMENTS == 1) {
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          const float x = __uint_as_float(a.w[2 * i]), y = __uint_as_float(a.w[2 * i + 1]);
          a.w[2 * i] = __float_as_uint(x * co[i] - y * si[i]);
          a.w[2 * i + 1] = __float_as_uint(x * si[i] + y * co[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float x = __uint_as_float(a.w[i]), y = __uint_as_float(b.w[i]);
          a.w[i] = __float_as_uint(x * co[i] - y * si[i]);
          b.w[i] = __float_as_uint(x * si[i] + y * co[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float2 x = Word<T>::wide(a.w[i]);
        if constexpr (INTERLEAVED) {
          a.w[i] = Word<T>::narrow(make_float2(x.x * co[i] - x.y * si[i], x.x * si[i] + x.y * co[i]));
        } else {
          const float2 y = Word<T>::wide(b.w[i]);
          a.w[i] = Word<T>::narrow(make_float2(x.x * co[2 * i] - y.x * si[2 * i], x.y * co[2 * i + 1] - y.y * si[2 * i + 1]));
          b.w[i] = Word<T>::narrow(make_float2(x.x * si[2 * i] + y.x * co[2 * i], x.y * si[2 * i + 1] + y.y * co[2 * i + 1]));
        }
      }
    }
  }
};

// The token's sines and cosines into this warp's part of shared memory.
__device__ __forceinline__ void evaluate(const RotaryArgs& p, int64_t token, int lane, float* cosines, float* sines) {
  for (int slot = lane; slot < p.turned / 2; slot += 32) {
    const int64_t at = token * p.axes + (p.axis ? p.axis[slot] : 0);
    const double position = p.position_type == 0   ? double(static_cast<const int*>(p.positions)[at])
                            : p.position_type == 1 ? double(static_cast<const int64_t*>(p.positions)[at])
                                                   : double(static_cast<const float*>(p.positions)[at]);
    const double turns = position * p.turns[slot];
    float s, c;
    sincospif(2.f * float(turns - rint(turns)), &s, &c);
    cosines[slot] = c * p.amplitude;
    sines[slot] = s * (p.amplitude * p.direction);
  }
  __syncwarp();
}

// One warp per (token, part of its heads: blockIdx.y).  Lanes are (head, unit), units fastest; with more
// units than lanes the warp goes over its heads once for every 32 units.
template <typename T, int W, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS, 4) rotary_kernel(const RotaryArgs p, int units, int turned_units, int parts) {
  using P = Pairs<T, W, INTERLEAVED>;
  extern __shared__ float4 shared[];
  const int lane = threadIdx.x & 31;
  const int pitch = (p.turned / 2 + 3) / 4 * 4;
  float* cosines = reinterpret_cast<float*>(shared) + (threadIdx.x >> 5) * 2 * pitch;
  float* sines = cosines + pitch;
  const int64_t token = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  evaluate(p, token, lane, cosines, sines);
  const int across = units < 32 ? 32 / units : 1;  // heads side by side
  const int step = across * parts;
  for (int base = 0; base < units; base += 32) {
    const int unit = base + (units < 32 ? lane % units : lane);
    if (unit >= units || (units < 32 && lane >= across * units)) continue;
    const bool copies = unit >= turned_units;
    int e0, e1;  // first elements of the unit's vectors
    if (copies) {
      e0 = p.turned + (unit - turned_units) * P::VECTORS * P::ELEMENTS;
      e1 = e0 + P::ELEMENTS;
    } else {
      e0 = unit * P::ELEMENTS;
      e1 = p.turned / 2 + e0;
    }
    const bool second = !INTERLEAVED && e1 < p.dim;  // the copied tail may end with a single vector
    float co[P::SLOTS], si[P::SLOTS];
    if (!copies)
#pragma unroll
      for (int i = 0; i < P::SLOTS; ++i) {
        co[i] = cosines[unit * P::SLOTS + i];
        si[i] = sines[unit * P::SLOTS + i];
      }
    const int head0 = int(blockIdx.y) * across + (units < 32 ? lane / units : 0);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int heads = p.part[which].heads;
      const int64_t stride = p.part[which].head_stride;
      const T* from = static_cast<const T*>(p.part[which].x) + token * p.part[which].row_stride + head0 * stride;
      T* to = static_cast<T*>(p.part[which].out) + (token * heads + head0) * p.dim;
#pragma unroll 1
      for (int head = head0; head < heads; head += BATCH * step) {
        Words<W> a[BATCH], b[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
          if (head + i * step < heads) {
            a[i] = *reinterpret_cast<const Words<W>*>(from + i * step * stride + e0);
            if (second) b[i] = *reinterpret_cast<const Words<W>*>(from + i * step * stride + e1);
          }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
          if (head + i * step < heads) {
            if (!copies) P::turn(a[i], b[i], co, si);
            *reinterpret_cast<Words<W>*>(to + int64_t(i * step) * p.dim + e0) = a[i];
            if (second) *reinterpret_cast<Words<W>*>(to + int64_t(i * step) * p.dim + e1) = b[i];
          }
        from += BATCH * step * stride;
        to += int64_t(BATCH * step) * p.dim;
      }
    }
  }
}

// Any alignment, element by element.
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(float x) { return x; }
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half narrow(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ float narrow(float x) { return x; }

template <typename T>
__global__ void __launch_bounds__(THREADS) rotary_any_kernel(const RotaryArgs p, int parts) {
  extern __shared__ float4 shared[];
  const int lane = threadIdx.x & 31;
  const int slots = p.turned / 2, pitch = (slots + 3) / 4 * 4;
  float* cosines = reinterpret_cast<float*>(shared) + (threadIdx.x >> 5) * 2 * pitch;
  float* sines = cosines + pitch;
  const int64_t token = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  evaluate(p, token, lane, cosines, sines);
  const int units = p.dim - slots;  // pairs, then copied elements
  for (const RotaryPart& part : p.part)
    for (int head = int(blockIdx.y); head < part.heads; head += parts) {
      const T* from = static_cast<const T*>(part.x) + token * part.row_stride + head * part.head_stride;
      T* to = static_cast<T*>(part.out) + (token * part.heads + head) * p.dim;
      for (int unit = lane; unit < units; unit += 32) {
        if (unit >= slots) {
          to[unit + slots] = from[unit + slots];
          continue;
        }
        const int e0 = p.interleaved ? 2 * unit : unit, e1 = p.interleaved ? e0 + 1 : e0 + slots;
        const float x = widen(from[e0]), y = widen(from[e1]);
        to[e0] = narrow<T>(x * cosines[unit] - y * sines[unit]);
        to[e1] = narrow<T>(x * sines[unit] + y * cosines[unit]);
      }
    }
}

// Few tokens: their heads are shared out over more warps, until there are about 32 warps for every SM.
struct Shape {
  dim3 grid;
  int warps, parts;
  size_t shared;
};
bool shape_of(const RotaryArgs& p, int across, Shape* s) {
  const int heads = p.part[0].heads > p.part[1].heads ? p.part[0].heads : p.part[1].heads;
  const int64_t most = (heads + across - 1) / across;
  int64_t parts = (int64_t(p.sm_count) * 32 + p.tokens - 1) / p.tokens;
  if (parts > most) parts = most;
  const size_t per_warp = size_t((p.turned / 2 + 3) / 4 * 4) * 2 * sizeof(float);
  s->warps = THREADS / 32;
  while (s->warps > 1 && s->warps * per_warp > 48 * 1024) s->warps /= 2;
  const int64_t blocks = (p.tokens + s->warps - 1) / s->warps;
  if (blocks > 2147483647ll || parts > 65535 || per_warp > 48 * 1024) {
    set_error_detail("rotary_embed: too many tokens for one launch or too large a head");
    return false;
  }
  s->grid = dim3(unsigned(blocks), unsigned(parts), 1);
  s->parts = int(parts);
  s->shared = s->warps * per_warp;
  return true;
}

template <typename T, int W, bool INTERLEAVED>
cudaError_t launch(const RotaryArgs& p, cudaStream_t stream) {
  using P = Pairs<T, W, INTERLEAVED>;
  constexpr int UNIT = P::VECTORS * P::ELEMENTS;
  const int turned_units = p.turned / UNIT;
  const int units = turned_units + (p.dim - p.turned + UNIT - 1) / UNIT;
  Shape s;
  if (!shape_of(p, units < 32 ? 32 / units : 1, &s)) return cudaErrorInvalidValue;
  rotary_kernel<T, W, INTERLEAVED><<<s.grid, s.warps * 32, s.shared, stream>>>(p, units, turned_units, s.parts);
  return cudaGetLastError();
}

// The widest vector that every address allows: row and head strides, the vectors' elements within a
// head and its tail are multiples of it and the base addresses are aligned to it.
template <typename T>
cudaError_t dispatch(const RotaryArgs& p, cudaStream_t stream) {
  uint64_t bits = uint64_t(p.dim) | uint64_t(p.turned);
  if (!p.interleaved) bits |= uint64_t(p.turned / 2);
  for (const RotaryPart& part : p.part) {
    if (part.heads == 0) continue;
    bits |= uint64_t(part.row_stride) | uint64_t(part.head_stride);
    bits |= reinterpret_cast<uint64_t>(part.x) / sizeof(T) | reinterpret_cast<uint64_t>(part.out) / sizeof(T);
  }
  bits *= sizeof(T);
  if (p.interleaved) {
    if (bits % 16 == 0) return launch<T, 4, true>(p, stream);
    if (bits % 8 == 0) return launch<T, 2, true>(p, stream);
  } else {
    if (bits % 16 == 0) return launch<T, 4, false>(p, stream);
    if (bits % 8 == 0) return launch<T, 2, false>(p, stream);
    if (bits % 4 == 0) return launch<T, 1, false>(p, stream);
  }
  Shape s;
  if (!shape_of(p, 1, &s)) return cudaErrorInvalidValue;
  rotary_any_kernel<T><<<s.grid, s.warps * 32, s.shared, stream>>>(p, s.parts);
  return cudaGetLastError();
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
