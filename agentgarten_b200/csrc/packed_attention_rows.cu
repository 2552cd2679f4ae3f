// Causal attention of few query rows per sequence (a single token against a long cache), forward.
//
// Bound by memory: every key and value is read once for all query heads of its group, which are the
// rows of one 16-row product (mma.sync: with 4 to 16 useful rows the 128-row products of the tile
// kernel would idle, and the tensor core is far from being the limit here).  A CTA of four warps
// works on a chunk of a sequence's keys for one key head; its warps take tiles of 16 keys in turn,
// each with its own ring of three stages (cp.async, no barrier between the warps), running maximum
// and FP32 accumulators.  The four are joined in shared memory, and a sequence of several chunks by
// a second launch, both in a fixed order.  Keys behind the last one are never read: their rows are
// filled with zeros.
#include "agb.h"
#include "packed.h"
#include "packed_common.cuh"

namespace agb {
namespace {

constexpr int WARPS = 4;
constexpr int KEYS = 16;     // keys of a tile
constexpr int STAGES = 3;
constexpr int QROWS = 16;    // rows of a product: (query row, head of the group)
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units

template <int DP>
constexpr int rows_smem() {
  return WARPS * STAGES * 2 * KEYS * DP * 2;
}

struct RowsParams {
  const void* q; const void* k; const void* v;
  void* out;
  float* lse;
  const int* q_offsets; const int* k_offsets; const int* k_lengths;
  int sequences;
  int64_t total_q, total_k;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int hq, hkv, group, dim, pieces, chunk;
  float scale_log2;
  float* part_out; float* part_lse;
  int* status;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool read) {
  const int bytes = read ? 16 : 0;  // the rest of the 16 bytes is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool FP16>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (FP16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte offset of the 16-byte word `word` of row `row` in a tile of rows of DP elements: words are
// permuted within 128 bytes so that the eight rows of a matrix fall into different banks.
template <int DP>
__device__ __forceinline__ uint32_t word_at(int row, int word) {
  return uint32_t(row * DP * 2 + ((word & ~7) | ((word ^ row) & 7)) * 16);
}

template <int DP, bool FP16>
__global__ void __launch_bounds__(WARPS * 32, 2) packed_rows_kernel(const RowsParams p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ PackedSpan span_smem;
  __shared__ float stat[WARPS][QROWS][2];  // maximum and sum of every warp's rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int piece = int(blockIdx.x % unsigned(p.pieces));
  const int kv_head = int((blockIdx.x / unsigned(p.pieces)) % unsigned(p.hkv));
  const int unit = int(blockIdx.x / (unsigned(p.pieces) * unsigned(p.hkv)));
  if (warp == 0) {
    const PackedSpan found = find_unit(unit, p.chunk, true, p.q_offsets, p.k_offsets, p.k_lengths, p.sequences,
                                       p.total_q, p.total_k, kv_head == 0 && piece == 0 ? p.status : nullptr);
    if (lane == 0) span_smem = found;
  }
  __syncthreads();
  const PackedSpan span = span_smem;
  const int head0 = kv_head * p.group + piece * QROWS;
  const int heads = min(QROWS, p.group - piece * QROWS);  // query heads side by side in the rows
  if (unit == 0) {  // rows behind the last sequence
    const int end = min(int64_t(max(p.q_offsets[p.sequences], 0)), p.total_q);
    const int words = heads * p.dim / 8;
    for (int64_t i = threadIdx.x; i < (p.total_q - end) * words; i += WARPS * 32) {
      const int64_t at = ((end + i / words) * p.hq + head0) * p.dim + (i % words) * 8;
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at) = make_uint4(0, 0, 0, 0);
    }
  }
  if (span.unit_in_sequence < 0 || span.rows == 0) return;
  const int flat = span.rows * heads;  // rows of the product, query row by query row
  const int chunks = (span.keys + p.chunk - 1) / p.chunk;
  // More rows than one product has are taken block by block over all keys by the first chunk's CTA.
  const bool split = chunks > 1 && flat <= QROWS;
  if (span.unit_in_sequence > 0 && (!split || span.unit_in_sequence >= chunks)) return;
  const int k_begin = split ? span.unit_in_sequence * p.chunk : 0;
  const int k_end = split ? min(span.keys, k_begin + p.chunk) : span.keys;
  const int tiles = (k_end - k_begin + KEYS - 1) / KEYS;

  const uint16_t* kp = static_cast<const uint16_t*>(p.k) + kv_head * p.k_head;
  const uint16_t* vp = static_cast<const uint16_t*>(p.v) + kv_head * p.v_head;
  const uint32_t mine = smem_u32(ring) + warp * STAGES * 2 * KEYS * DP * 2;
  constexpr int WORDS = DP / 8;  // 16-byte words of a row
  const int words = p.dim / 8;

  auto load = [&](int tile, int stage) {
    const uint32_t base = mine + stage * 2 * KEYS * DP * 2;
    const int first = k_begin + tile * KEYS;
#pragma unroll
    for (int i = 0; i < KEYS * WORDS / 32; ++i) {
      const int at = i * 32 + lane, row = at / WORDS, word = at % WORDS;
      const bool read = first + row < k_end && word < words;
      const int64_t key = int64_t(span.k0) + (read ? first + row : 0);
      const int element = read ? word * 8 : 0;
      copy16(base + word_at<DP>(row, word), kp + key * p.k_row + element, read);
      copy16(base + KEYS * DP * 2 + word_at<DP>(row, word), vp + key * p.v_row + element, read);
    }
  };

  for (int block = 0; block < flat; block += QROWS) {
    const int own = (tiles - warp + WARPS - 1) / WARPS;  // tiles warp, warp + 4, ...
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      if (s < own) load(warp + s * WARPS, s);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // queries as the A operand: rows lane / 4 and + 8, columns 2 (lane % 4) and + 8 of every 16
    uint32_t q[DP / 16][4];
    int seen[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int f = block + (lane >> 2) + 8 * r;
      const bool there = f < flat;
      const int row = there ? f / heads : 0, head = there ? f % heads : 0;
      seen[r] = there ? span.keys - span.rows + row + 1 - k_begin : 0;  // keys it sees, from k_begin on
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + (int64_t(span.q0) + row) * p.q_row + (head0 + head) * p.q_head;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e = kk * 16 + h * 8 + (lane & 3) * 2;
          q[kk][r + 2 * h] = there && e < p.dim ? *reinterpret_cast<const uint32_t*>(src + e) : 0u;
        }
    }
    const int visible = k_end - k_begin;
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

    for (int i = 0; i < own; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();
      {
        const int next = i + STAGES - 1;
        if (next < own) load(warp + next * WARPS, next % STAGES);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      const uint32_t base = mine + (i % STAGES) * 2 * KEYS * DP * 2;
      float s[2][4] = {};
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t b[4];  // keys 0-7 and 8-15 of the tile, elements 0-7 and 8-15 of the step
        ldmatrix4(b, base + word_at<DP>((lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
        mma16<FP16>(s[0], q[kk], b[0], b[1]);
        mma16<FP16>(s[1], q[kk], b[2], b[3]);
      }
      const int tile = warp + i * WARPS;
      float high[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int key = tile * KEYS + n * 8 + (lane & 3) * 2 + (c & 1);
          s[n][c] = key < visible && key < seen[c >> 1] ? s[n][c] * p.scale_log2 : -INFINITY;
          high[c >> 1] = fmaxf(high[c >> 1], s[n][c]);
        }
      bool grow = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        high[r] = fmaxf(high[r], __shfl_xor_sync(0xffffffffu, high[r], 1));
        high[r] = fmaxf(high[r], __shfl_xor_sync(0xffffffffu, high[r], 2));
        grow |= high[r] > top[r] + RESCALE_THRESHOLD;
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float now = fmaxf(top[r], high[r]);
          const float alpha = top[r] == -INFINITY ? 0.f : exp2f(top[r] - now);
          top[r] = now;
          sum[r] *= alpha;
#pragma unroll
          for (int d = 0; d < DP / 8; ++d) {
            o[d][2 * r] *= alpha;
            o[d][2 * r + 1] *= alpha;
          }
        }
      }
      // a row that has seen nothing yet has only -inf scores: any finite reference gives zeros
      const float ref[2] = {top[0] == -INFINITY ? 0.f : top[0], top[1] == -INFINITY ? 0.f : top[1]};
      uint32_t pr[4];  // the accumulator's layout is the A operand's: n gives the column half
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float e0 = exp2f(s[n][2 * r] - ref[r]), e1 = exp2f(s[n][2 * r + 1] - ref[r]);
          sum[r] += e0 + e1;
          pr[r + 2 * n] = pack16<FP16>(e0, e1);
        }
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        uint32_t b[4];  // keys 0-7 and 8-15, elements 0-7 and then 8-15 of the step
        ldmatrix4_t(b, base + KEYS * DP * 2 + word_at<DP>((lane & 7) + (((lane >> 3) & 1) << 3), d * 2 + (lane >> 4)));
        mma16<FP16>(o[2 * d], pr, b[0], b[1]);
        mma16<FP16>(o[2 * d + 1], pr, b[2], b[3]);
      }
      __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // Join the four warps in shared memory, in warp order.
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
    }
    __syncthreads();  // every warp is done with its ring
    float* acc = reinterpret_cast<float*>(ring);  // [WARPS][QROWS][DP]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = (lane >> 2) + 8 * r;
      if ((lane & 3) == 0) {
        stat[warp][row][0] = top[r];
        stat[warp][row][1] = sum[r];
      }
#pragma unroll
      for (int d = 0; d < DP / 8; ++d)
        *reinterpret_cast<float2*>(acc + (warp * QROWS + row) * DP + d * 8 + (lane & 3) * 2) =
            make_float2(o[d][2 * r], o[d][2 * r + 1]);
    }
    __syncthreads();
    const int quads = p.dim / 4;
    for (int at = threadIdx.x; at < min(QROWS, flat - block) * quads; at += WARPS * 32) {
      const int row = at / quads, e = (at % quads) * 4;
      float high = -INFINITY, total = 0.f;
      for (int w = 0; w < WARPS; ++w) high = fmaxf(high, stat[w][row][0]);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < WARPS; ++w) {
        const float share = stat[w][row][0] == -INFINITY ? 0.f : exp2f(stat[w][row][0] - high);
        const float4 y = *reinterpret_cast<const float4*>(acc + (w * QROWS + row) * DP + e);
        total += share * stat[w][row][1];
        x.x += share * y.x; x.y += share * y.y; x.z += share * y.z; x.w += share * y.w;
      }
      const float inv = total == 0.f ? 0.f : 1.f / total;
      x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
      const int f = block + row;
      if (split) {
        const int64_t slot = ((int64_t(unit) * p.hkv + kv_head) * p.pieces + piece) * QROWS + f;
        *reinterpret_cast<float4*>(p.part_out + slot * p.dim + e) = x;
        if (e == 0) p.part_lse[slot] = total == 0.f ? -INFINITY : high + log2f(total);
      } else {
        const int64_t q_row = int64_t(span.q0) + f / heads;
        const int head = head0 + f % heads;
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (q_row * p.hq + head) * p.dim + e) =
            make_uint2(pack16<FP16>(x.x, x.y), pack16<FP16>(x.z, x.w));
        if (e == 0 && p.lse)
          p.lse[int64_t(head) * p.total_q + q_row] = total == 0.f ? -INFINITY : (high + log2f(total)) * 0.6931471805599453f;
      }
    }
    __syncthreads();  // the ring is loaded again for the next block of rows
  }
}

// Joins the chunks of every row that had several: out = sum_c w_c o_c.  One CTA per (query row, head);
// its warps take chunks in turn and are added in warp order.
constexpr int JOIN_WARPS = 8;
template <bool FP16>
__global__ void __launch_bounds__(JOIN_WARPS * 32) packed_rows_join_kernel(const RowsParams p) {
  __shared__ float4 partial[JOIN_WARPS][32];
  __shared__ float weight[JOIN_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int row = int(blockIdx.x / unsigned(p.hq)), head = int(blockIdx.x % unsigned(p.hq));
  // the sequence of the row: 32-way search for the last s with q_offsets[s] <= row
  int low = 0, count = p.sequences;
  bool found = true;
  while (count > 0) {
    const int stride = (count + 31) / 32;
    const bool reached = lane * stride < count && p.q_offsets[low + lane * stride] <= row;
    const unsigned votes = __ballot_sync(0xffffffffu, reached);
    if (votes == 0) {
      found = false;
      break;
    }
    const int last = 31 - __clz(votes);
    const int behind = count - last * stride;
    low += last * stride;
    count = stride == 1 ? 0 : (behind < stride ? behind : stride);
  }
  const int q0 = p.q_offsets[low], q1 = p.q_offsets[low + 1];
  const int k0 = p.k_offsets[low], k1 = p.k_offsets[low + 1];
  const int keys = p.k_lengths ? p.k_lengths[low] : k1 - k0;
  found = found && row >= q0 && row < q1 && q1 <= p.total_q && k0 >= 0 && k1 >= k0 && k1 <= p.total_k && keys >= 0 &&
          keys <= k1 - k0;
  const int kv_head = head / p.group, in_group = head % p.group;
  const int piece = in_group / QROWS;
  const int heads = min(QROWS, p.group - piece * QROWS);
  const int chunks = (keys + p.chunk - 1) / p.chunk;
  after_previous_launch();
  if (!found || chunks <= 1 || (q1 - q0) * heads > QROWS) return;  // written by the first launch
  const int f = (row - q0) * heads + in_group % QROWS;
  const int64_t step = int64_t(p.hkv) * p.pieces * QROWS;
  const int64_t first = ((int64_t(k0) / p.chunk + low) * p.hkv * p.pieces + kv_head * p.pieces + piece) * QROWS + f;
  float high = -INFINITY;
  for (int c = lane; c < chunks; c += 32) high = fmaxf(high, p.part_lse[first + c * step]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f;
#pragma unroll 4
  for (int c = warp; c < chunks; c += warps) {
    const int64_t slot = first + c * step;
    const float l = p.part_lse[slot];
    const float share = l == -INFINITY ? 0.f : exp2f(l - high);
    total += share;
    if (lane * 4 < p.dim) {
      const float4 y = *reinterpret_cast<const float4*>(p.part_out + slot * p.dim + lane * 4);
      x.x += share * y.x; x.y += share * y.y; x.z += share * y.z; x.w += share * y.w;
    }
  }
  partial[warp][lane] = x;
  if (lane == 0) weight[warp] = total;
  __syncthreads();
  if (warp != 0) return;
  for (int w = 1; w < warps; ++w) {
    const float4 y = partial[w][lane];
    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    total += weight[w];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (lane * 4 < p.dim)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (int64_t(row) * p.hq + head) * p.dim + lane * 4) =
        make_uint2(pack16<FP16>(x.x * inv, x.y * inv), pack16<FP16>(x.z * inv, x.w * inv));
  if (lane == 0 && p.lse)
    p.lse[int64_t(head) * p.total_q + row] = total == 0.f ? -INFINITY : (high + log2f(total)) * 0.6931471805599453f;
}

template <int DP, bool FP16>
cudaError_t launch(const RowsParams& p, cudaStream_t stream) {
  const cudaError_t e = cudaFuncSetAttribute(packed_rows_kernel<DP, FP16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             rows_smem<DP>());
  if (e != cudaSuccess) return e;
  const int64_t grid = (p.total_k / p.chunk + p.sequences) * p.hkv * p.pieces;
  const int64_t joins = p.total_q * p.hq;
  if (grid > 2147483647ll || joins > 2147483647ll) {
    set_error_detail("packed_attention: too many chunks for one launch");
    return cudaErrorInvalidValue;
  }
  packed_rows_kernel<DP, FP16><<<unsigned(grid), WARPS * 32, rows_smem<DP>(), stream>>>(p);
  const cudaError_t launched = cudaGetLastError();
  if (launched != cudaSuccess || p.total_k <= p.chunk) return launched;
  const int64_t most = p.total_k / p.chunk + 1;  // chunks of a sequence
  const int warps = most < JOIN_WARPS ? int(most) : JOIN_WARPS;
  return launch_behind(packed_rows_join_kernel<FP16>, dim3(unsigned(joins)), warps * 32, 0, stream, p);
}

}  // namespace

cudaError_t packed_attention_rows(const PackedArgs& a, cudaStream_t stream) {
  RowsParams p{};
  p.q = a.q; p.k = a.k; p.v = a.v; p.out = a.out; p.lse = a.lse;
  p.q_offsets = a.q_offsets; p.k_offsets = a.k_offsets; p.k_lengths = a.k_lengths;
  p.sequences = a.sequences;
  p.total_q = a.total_q; p.total_k = a.total_k;
  p.q_row = a.q_row; p.q_head = a.q_head; p.k_row = a.k_row; p.k_head = a.k_head; p.v_row = a.v_row; p.v_head = a.v_head;
  p.hq = a.hq; p.hkv = a.hkv; p.group = a.hq / a.hkv; p.dim = a.dim;
  p.pieces = packed_rows_pieces(p.group);
  p.chunk = a.chunk;
  p.scale_log2 = a.scale * LOG2E;
  p.part_out = a.part_out; p.part_lse = a.part_lse;
  p.status = a.status;
  if (a.dim <= 64) return a.fp16 ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
  return a.fp16 ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
}

int packed_rows_pieces(int group) { return (group + QROWS - 1) / QROWS; }

}  // namespace agb
