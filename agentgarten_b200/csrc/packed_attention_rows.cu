// Causal attention of few query rows per sequence (a single token against a long cache), forward.
//
// Bound by memory: every key and value is read once for all query heads of its group, which are the
// rows of one 16-row product (mma.sync: with 4 to 16 useful rows the 128-row products of the tile
// kernel would idle, and the tensor core is far from being the limit here).  Every warp works by itself,
// with its own ring of three stages of 16 keys (cp.async), running maximum and FP32 accumulators, on
// jobs of (sequence, 16 rows, chunk of keys, key head); eight warps an SM keep 128 KB on their way, so
// the start and the end of one warp's job (2 to 3 us) hide behind the others.  (Four warps on one chunk,
// joined in shared memory, all stood still there: 129 us against 119 at the same chunks for 131071 keys.)  A
// sequence of several chunks is joined by a second launch, in a fixed order.  Keys behind the last
// one are never read: their rows are filled with zeros.
//
// Jobs are numbered over the keys that exist, sequence by sequence, and dealt out to as many warps as
// the GPU holds: a cache has room that nobody uses yet, and a block for every chunk of that room
// cost as much as half of the real ones.
//
// With 32 query and 8 key heads of 128: one token against 131071 keys (537 MB) 87 us, 6.1 TB/s, and 97 with
// the join; 24 tokens against caches of 60 to 8191 keys (184 MB) 38 us, 4.8 TB/s, and 45 with the join.
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
  int* part_jobs;
  int sm_count, most_jobs;
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

// The sequence of job number `at`.  A sequence has `blocks`
// blocks of 16 rows times `chunks` chunks of `length` keys: as many chunks as `p.chunk` asks for, or
// fewer where it has several blocks, so that the jobs of all stay within packed_rows_jobs().
// Converged warp; 32 sequences a step.  Sequences whose offsets do not fit have no jobs.  A warp's job
// numbers rise: the search goes on from where the last one ended (`base`, with `before` jobs behind it).
struct JobSpan {
  int sequence;  // -1: none
  int first, chunks, length;
  int q0, rows, k0, keys;
};
__device__ inline JobSpan find_job(int at, int heads, int& base, int& before, const RowsParams& p, int* status) {
  const int lane = threadIdx.x & 31;
  JobSpan span{-1, 0, 0, 0, 0, 0, 0, 0};
  for (; base < p.sequences; base += 32) {
    const int s = base + lane;
    const bool there = s < p.sequences;
    const int q0 = p.q_offsets[there ? s : 0], q1 = p.q_offsets[there ? s + 1 : 0];
    const int k0 = p.k_offsets[there ? s : 0], k1 = p.k_offsets[there ? s + 1 : 0];
    const int keys = there && p.k_lengths ? p.k_lengths[s] : k1 - k0;
    const bool fits = q0 >= 0 && q1 >= q0 && q1 <= p.total_q && k0 >= 0 && k1 >= k0 && k1 <= p.total_k && keys >= 0 &&
                      keys <= k1 - k0;
    if (there && status && (!fits || (s == 0 && (q0 != 0 || k0 != 0)))) atomicCAS(status, 0, kBadIndex);
    int chunks = 0, jobs = 0;
    if (there && fits && q1 > q0) {
      const int blocks = ((q1 - q0) * heads + QROWS - 1) / QROWS;
      const int asked = (keys + p.chunk - 1) / p.chunk;
      chunks = blocks == 1 ? max(1, asked) : max(1, asked / blocks);
      jobs = chunks * blocks;
    }
    int sum = jobs;  // inclusive over the lanes
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int other = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += other;
    }
    const bool here = jobs > 0 && at < before + sum;
    const unsigned votes = __ballot_sync(0xffffffffu, here);
    if (votes) {
      const int owner = __ffs(votes) - 1;
      auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, owner); };
      span.sequence = base + owner;
      span.chunks = of(chunks);
      span.first = before + of(sum - jobs);
      span.q0 = of(q0);
      span.rows = of(q1) - span.q0;
      span.k0 = of(k0);
      span.keys = of(keys);
      span.length = span.chunks == 1 ? span.keys : ((span.keys + span.chunks - 1) / span.chunks + KEYS - 1) / KEYS * KEYS;
      return span;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return span;
}

template <int DP, bool FP16>
__global__ void __launch_bounds__(WARPS * 32, 2) packed_rows_kernel(const RowsParams p) {
  extern __shared__ __align__(128) uint8_t ring[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int side = p.hkv * p.pieces;  // jobs side by side
  if (blockIdx.x < side) {            // rows behind the last sequence
    const int piece = int(blockIdx.x) % p.pieces, head0 = int(blockIdx.x) / p.pieces * p.group + piece * QROWS;
    const int heads = min(QROWS, p.group - piece * QROWS);
    const int end = int(min(int64_t(max(p.q_offsets[p.sequences], 0)), p.total_q));
    const int words = heads * p.dim / 8;
    for (int64_t i = threadIdx.x; i < (p.total_q - end) * words; i += WARPS * 32) {
      const int64_t at = ((end + i / words) * p.hq + head0) * p.dim + (i % words) * 8;
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at) = make_uint4(0, 0, 0, 0);
    }
  }
  allow_next_launch();  // the join's blocks take the places of the first to end
  // neighbouring warps take the same keys of neighbouring heads
  int base = 0, before = 0;
  for (int64_t job = int64_t(blockIdx.x) * WARPS + warp;; job += int64_t(gridDim.x) * WARPS) {
  const int unit = divide(int(job), side), rest = int(job) - unit * side;
  const int kv_head = divide(rest, p.pieces), piece = rest - kv_head * p.pieces;
  const int head0 = kv_head * p.group + piece * QROWS;
  const int heads = min(QROWS, p.group - piece * QROWS);  // query heads side by side in the rows
  // the pieces of a group have the same jobs: those of its first
  const JobSpan span = find_job(unit, min(QROWS, p.group), base, before, p, p.status);
  if (span.sequence < 0) return;
  if (unit == span.first && rest == 0 && lane == 0 && p.part_jobs) {  // for the join
    p.part_jobs[2 * span.sequence] = span.first;
    p.part_jobs[2 * span.sequence + 1] = span.chunks;
  }
  if (unit >= p.most_jobs) {  // offsets that fall make sequences overlap: more jobs than partial results
    if (lane == 0 && p.status) atomicCAS(p.status, 0, kBadIndex);
    return;
  }
  const int flat = span.rows * heads;  // rows of the products, query row by query row
  const int block = (unit - span.first) / span.chunks * QROWS, number = (unit - span.first) % span.chunks;
  const bool split = span.chunks > 1;
  const int k_begin = number * span.length;
  const int k_end = min(span.keys, k_begin + span.length);
  const int tiles = max(0, (k_end - k_begin + KEYS - 1) / KEYS);

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

  {
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      if (s < tiles) load(s, s);
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

    for (int i = 0; i < tiles; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();
      {
        const int next = i + STAGES - 1;
        if (next < tiles) load(next, next % STAGES);
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
      float high[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int key = i * KEYS + n * 8 + (lane & 3) * 2 + (c & 1);
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
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      const int f = block + (lane >> 2) + 8 * r;
      if (f >= flat) continue;
      const float inv = sum[r] == 0.f ? 0.f : 1.f / sum[r];
      const float log_sum = sum[r] == 0.f ? -INFINITY : top[r] + log2f(sum[r]);
      if (split) {
        const int64_t slot = ((int64_t(unit) * p.hkv + kv_head) * p.pieces + piece) * QROWS + f - block;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          const int e = d * 8 + (lane & 3) * 2;
          if (e < p.dim)
            *reinterpret_cast<float2*>(p.part_out + slot * p.dim + e) = make_float2(o[d][2 * r] * inv, o[d][2 * r + 1] * inv);
        }
        if ((lane & 3) == 0) p.part_lse[slot] = log_sum;
      } else {
        const int64_t q_row = int64_t(span.q0) + f / heads;
        const int head = head0 + f % heads;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + (q_row * p.hq + head) * p.dim;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          const int e = d * 8 + (lane & 3) * 2;
          if (e < p.dim) *reinterpret_cast<uint32_t*>(dst + e) = pack16<FP16>(o[d][2 * r] * inv, o[d][2 * r + 1] * inv);
        }
        if ((lane & 3) == 0 && p.lse) p.lse[int64_t(head) * p.total_q + q_row] = log_sum * 0.6931471805599453f;
      }
    }
    __syncwarp();  // the ring is loaded again for the next job
  }
  }
}

// Joins the chunks of every row that had several: out = sum_c w_c o_c.  One CTA per (query row, head);
// its warps take chunks in turn, relative to a maximum of their own, and are added in warp order.  The
// weights of 32 chunks are evaluated side by side, so that the results' loads wait for nothing.
constexpr int JOIN_WARPS = 16;
template <bool FP16>
__global__ void __launch_bounds__(JOIN_WARPS * 32) packed_rows_join_kernel(const RowsParams p) {
  __shared__ float4 partial[JOIN_WARPS][32];
  __shared__ float weight[JOIN_WARPS], tops[JOIN_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int row = int(blockIdx.x / unsigned(p.hq)), head = int(blockIdx.x % unsigned(p.hq));
  // the sequence of the row: 32-way search for the last s with q_offsets[s] <= row
  int low = 0;
  for (int count = p.sequences; count > 0;) {
    const int stride = (count + 31) / 32;
    const bool reached = lane * stride < count && p.q_offsets[low + lane * stride] <= row;
    const unsigned votes = __ballot_sync(0xffffffffu, reached);
    if (votes == 0) break;
    const int last = 31 - __clz(votes), behind = count - last * stride;
    low += last * stride;
    count = stride == 1 ? 0 : (behind < stride ? behind : stride);
  }
  const int q0 = p.q_offsets[low], q1 = p.q_offsets[low + 1], k0 = p.k_offsets[low], k1 = p.k_offsets[low + 1];
  const int keys = p.k_lengths ? p.k_lengths[low] : k1 - k0;
  const bool fits = q0 >= 0 && row >= q0 && row < q1 && q1 <= p.total_q && k0 >= 0 && k1 >= k0 && k1 <= p.total_k &&
                    keys >= 0 && keys <= k1 - k0;
  const int kv_head = head / p.group, in_group = head % p.group;
  const int piece = in_group / QROWS;
  const int heads = min(QROWS, p.group - piece * QROWS);
  after_previous_launch();
  if (!fits) return;
  const int first_job = p.part_jobs[2 * low], chunks = p.part_jobs[2 * low + 1];
  // written by the first launch, or never (offsets that fall)
  if (chunks <= 1 || first_job + chunks * (((q1 - q0) * heads + QROWS - 1) / QROWS) > p.most_jobs) return;
  const int f = (row - q0) * heads + in_group % QROWS;
  const int64_t step = int64_t(p.hkv) * p.pieces * QROWS;
  const int64_t first = ((int64_t(first_job) + f / QROWS * chunks) * p.hkv * p.pieces + kv_head * p.pieces + piece) * QROWS +
                        f % QROWS;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f, high = -INFINITY;
  for (int base = warp; base < chunks; base += 32 * warps) {
    const int mine = base + lane * warps;
    const float l = mine < chunks ? p.part_lse[first + mine * step] : -INFINITY;
    float now = l;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
    now = fmaxf(now, high);
    const float fade = high == -INFINITY ? 0.f : exp2f(high - now);
    high = now;
    x.x *= fade; x.y *= fade; x.z *= fade; x.w *= fade;
    total *= fade;
    const float share = l == -INFINITY ? 0.f : exp2f(l - high);
    const int count = min(32, (chunks - base + warps - 1) / warps);
    for (int i = 0; i < count; i += 8) {
      float4 y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i + k < count && lane * 4 < p.dim)
          y[k] = *reinterpret_cast<const float4*>(p.part_out + (first + int64_t(base + (i + k) * warps) * step) * p.dim + lane * 4);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = __shfl_sync(0xffffffffu, share, (i + k) & 31);
        if (i + k < count) {
          total += w;
          x.x += w * y[k].x; x.y += w * y[k].y; x.z += w * y[k].z; x.w += w * y[k].w;
        }
      }
    }
  }
  partial[warp][lane] = x;
  if (lane == 0) {
    weight[warp] = total;
    tops[warp] = high;
  }
  __syncthreads();
  if (warp != 0) return;
  for (int w = 0; w < warps; ++w) high = fmaxf(high, tops[w]);
  x = make_float4(0.f, 0.f, 0.f, 0.f);
  total = 0.f;
  for (int w = 0; w < warps; ++w) {
    const float share = tops[w] == -INFINITY ? 0.f : exp2f(tops[w] - high);
    const float4 y = partial[w][lane];
    x.x += share * y.x; x.y += share * y.y; x.z += share * y.z; x.w += share * y.w;
    total += share * weight[w];
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
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_shared_memory(packed_rows_kernel<DP, FP16>, rows_smem<DP>(), allowed);
  if (e != cudaSuccess) return e;
  const int64_t side = int64_t(p.hkv) * p.pieces, places = int64_t(p.sm_count) * 2;
  const int64_t jobs = int64_t(p.most_jobs) * side;
  int64_t grid = (jobs + WARPS - 1) / WARPS;
  if (grid > places) grid = places;
  if (grid < side) grid = side;  // each of the first `side` CTAs clears rows of one head
  const int64_t joins = p.total_q * p.hq;
  if (jobs + grid * WARPS > 2147483647ll || joins > 2147483647ll) {
    set_error_detail("packed_attention: too many chunks for one launch");
    return cudaErrorInvalidValue;
  }
  packed_rows_kernel<DP, FP16><<<unsigned(grid), WARPS * 32, rows_smem<DP>(), stream>>>(p);
  const cudaError_t launched = cudaGetLastError();
  if (launched != cudaSuccess || p.total_k <= p.chunk) return launched;
  const int64_t most = (p.total_k / p.chunk / p.sequences + 4) / 4;  // a quarter of a sequence's chunks
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
  p.part_out = a.part_out; p.part_lse = a.part_lse; p.part_jobs = a.part_jobs;
  p.status = a.status;
  p.sm_count = a.sm_count;
  p.most_jobs = int(packed_rows_jobs(a));
  if (a.dim <= 64) return a.fp16 ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
  return a.fp16 ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
}

int packed_rows_pieces(int group) { return (group + QROWS - 1) / QROWS; }

int64_t packed_rows_jobs(const PackedArgs& a) {
  const int group = a.hq / a.hkv, heads = group < QROWS ? group : QROWS;
  return a.total_k / a.chunk + a.total_q * heads / QROWS + 2 * int64_t(a.sequences);
}

}  // namespace agb
