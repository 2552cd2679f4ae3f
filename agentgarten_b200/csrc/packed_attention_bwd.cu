// Gradient of the causal attention over packed sequences, on tcgen05 (bf16 or fp16, heads of up to 128).
//
//   p = 2^(s - lse), delta = sum_d dO * O, ds = p (dO v^T - delta)
//   dq = scale ds k,  dk = scale ds^T q,  dv = p^T dO
//
// Two kernels, both without atomics, so a gradient is the same on every run:
//   packed_dq    one CTA per 128 (query row, head) pairs of up to 16 heads that share a key head walks the
//                key tiles up to its diagonal: S = Q K^T, dP = dO V^T, dQ += dS K.  It also writes delta for
//   packed_dkdv  one CTA per (128 key rows of a sequence, key head) walks the query tiles that see
//                them, 128 (query row, head) pairs at a time:
//                S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q.
// Shared heads are summed in the accumulators, in FP32.  P and dS are rounded to the tensors' type
// on their way into the tensor core (scale stays out of dS and is applied to the sums, which keeps
// small dS of fp16 above its underflow).  That rounding of dS takes the relative error of dq and dk in
// bf16 from the result's own 0.0017 to 0.0023; delta comes from the rounded O, which makes it 0.0027
// (200 rows).  Rows of a tile that belong to no one or to another sequence are cleared in shared memory
// before a product sums over them, so what they hold never spreads.
//
// Why two kernels of whole 128 x 128 blocks: dQ sums over keys and dK, dV over queries, and one kernel for
// both would add one of them up in memory with atomics.  The price is S and dP computed twice, seven
// products where five would do.  A block's score, dP and accumulator columns fill TMEM, so the overlap
// comes from the order of issue; one elected thread in a branch of its own issues (64 cycles for a product
// of 128 columns, where a lane elected for every instruction costs 91 to 105).
//
// What bounds it: at 8192 tokens, 32 query and 8 key heads of 128, the query side takes 630 us (three
// products, 1.31 PFLOP/s, tensor pipe active 66 % of the cycles) and the key side 804 us (four, 1.37
// PFLOP/s, 71 %): the elementwise work between a block's products.  Six prompts of 178 to 2045 rows take 92
// and 112 us, where the start and the end of every CTA and the longest key tile show as well.
#include "agb.h"
#include "packed.h"
#include "packed_common.cuh"
#include "tensormap.h"

#include <type_traits>

namespace agb {

bool make_packed_map(CUtensorMap* map, const void* base, int dim, int heads, int64_t rows, int64_t head_stride,
                     int64_t row_stride, int fold);

namespace {

constexpr int ROWS = 128;
constexpr int HALF_BYTES = 16384;  // 128 rows x 64 elements
constexpr int BWD_THREADS = 320;  // 8 elementwise warps, TMA producer, MMA issuer
constexpr int W_TMA = 8, W_MMA = 9;
constexpr float LOG2E = 1.4426950408889634f;

struct BwdParams {
  const int* q_offsets; const int* k_offsets; const int* k_lengths;
  int sequences;
  int64_t total_q, total_k;
  const void* out;      // dense [total_q, hq, dim]
  const void* grad;     // rows and heads at these strides
  int64_t grad_row, grad_head;
  const float* lse;     // [hq, total_q]
  float* delta;         // [hq, total_q]
  void* dq; void* dk; void* dv;  // dense
  int hq, hkv, group, dim;
  int shift;            // heads folded into a query tile's rows: 1 << shift
  int share;            // CTAs (a cluster) that share the query tiles of a key tile
  float scale, scale_log2;
  int* status;
};

template <int ATOMS>
__device__ __forceinline__ void load_tile(uint8_t* tile, const CUtensorMap* map, uint64_t* bar, int head, int row) {
  for (int a = 0; a < ATOMS; ++a) tma_load_3d(tile + a * HALF_BYTES, map, bar, a * 64, head, row);
}

// Writes 64 columns of a warp's 32 rows of an FP32 accumulator, scaled and rounded, through its 4 KB of
// stage.  Without `filled` (uniform over the warp) the accumulator holds nothing and zeros are
// written; so are the rows that are not `live`.
template <bool FP16>
__device__ __forceinline__ void store_columns(uint16_t* dst, int pitch, int head_pitch, int shift, uint32_t taddr, int left,
                                              float scale, int rows, bool filled, bool live, uint32_t stage, int lane) {
  uint32_t o[2][32];
  if (filled) {
    tmem_ld_32x32(taddr, o[0]);
    tmem_ld_32x32(taddr + 32, o[1]);
    tmem_ld_wait();
  }
  if (!filled || !live) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 32; ++i) o[h][i] = 0;
  }
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    const uint32_t* x = &o[g >> 2][(g & 3) * 8];
    uint4 v;
    v.x = pack16<FP16>(__uint_as_float(x[0]) * scale, __uint_as_float(x[1]) * scale);
    v.y = pack16<FP16>(__uint_as_float(x[2]) * scale, __uint_as_float(x[3]) * scale);
    v.z = pack16<FP16>(__uint_as_float(x[4]) * scale, __uint_as_float(x[5]) * scale);
    v.w = pack16<FP16>(__uint_as_float(x[6]) * scale, __uint_as_float(x[7]) * scale);
    put16(stage_word(stage, lane, g), v);
  }
  flush_rows(stage, reinterpret_cast<uint8_t*>(dst), pitch * 2, head_pitch * 2, shift, left * 2, rows, lane);
}

// Probabilities of a pair of scores, one pair in four on the FMA pipe (see exp2_fma).
template <bool FMA>
__device__ __forceinline__ float2 exp2_pair(float2 x) {
  return FMA ? exp2_fma(x) : make_float2(exp2f(x.x), exp2f(x.y));
}

// Seven tiles fill an SM (the ring of the operand that two products use has three stages, so that its
// next load is on its way while the later product runs; with two, every second tile waited for it).
// At least half of an SM's shared memory: two CTAs do not fit in its tensor memory.
constexpr int RING = 3;
template <int DP>
constexpr int bwd_smem() {
  const int bytes = 7 * (DP / 64) * HALF_BYTES + 4 * ROWS * 4 + 384;
  return bytes > 120 * 1024 ? bytes : 120 * 1024;
}
static_assert(bwd_smem<128>() <= 232448, "an SM's shared memory");

// ------------------------------------------------------------------------------- dQ
// Products are issued one tile staggered: S(j+1) = Q K^T | dQ += dS(j) K | dP(j+1) = dO V^T.  The
// exponentials of tile j+1 run under dQ(j) and dP(j+1), its dS under S(j+2).  Probabilities stay in
// registers; dS is packed over the first half of the dP columns it came from.
// TMEM: S[2] [0,256) dP [256,384) dQ [384,512).
template <int DP, bool FP16>
__global__ void __launch_bounds__(BWD_THREADS, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                 const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                 const BwdParams p) {
  constexpr int ATOMS = DP / 64;
  constexpr int TILE_BYTES = ATOMS * HALF_BYTES;
  extern __shared__ __align__(1024) uint8_t smem[];  // the swizzle counts addresses in blocks of 1024 bytes
  uint8_t* sQ = smem;
  uint8_t* sdO = smem + TILE_BYTES;
  uint8_t* sK = smem + 2 * TILE_BYTES;  // [RING]
  uint8_t* sV = smem + 5 * TILE_BYTES;  // [2]
  float* deltas = reinterpret_cast<float*>(smem + 7 * TILE_BYTES);  // [128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(deltas + 4 * ROWS);
  uint64_t* q_full = bars;        // Q and dO
  uint64_t* k_full = bars + 1;    // [RING]
  uint64_t* k_empty = bars + 4;   // [RING]
  uint64_t* v_full = bars + 7;    // [2]
  uint64_t* v_empty = bars + 9;   // [2]
  uint64_t* s_full = bars + 11;   // [2] S of a tile is in TMEM
  uint64_t* dp_full = bars + 13;  // dP of a tile is in TMEM
  uint64_t* ds_ready = bars + 14; // [2] dS of key chunk c of both halves written over dP (count 8)
  uint64_t* dq_done = bars + 16;  // every dQ product finished
  uint64_t* clean = bars + 17;    // rows of the last K and V tile behind the last key cleared
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* span_smem = reinterpret_cast<int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head_units = p.hq >> p.shift, unit = divide(int(blockIdx.x), head_units);
  const int head0 = (int(blockIdx.x) - unit * head_units) << p.shift;
  const int kv_head = head0 / p.group;
  const int step = ROWS >> p.shift;  // query rows of the tile
  const WaitGuard guard{abort_flag, p.status};

  if (warp == 0) {
    const PackedSpan span = find_piece(unit, step, false, p.q_offsets, p.k_offsets, p.k_lengths, p.sequences,
                                       p.total_q, p.total_k, head0 == 0 ? p.status : nullptr);
    if (lane == 0) *reinterpret_cast<PackedSpan*>(span_smem) = span;
  }
  if (warp == 1 && lane == 0) {
    *abort_flag = 0;
    mbar_init(q_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(&ds_ready[0], 8);
    mbar_init(&ds_ready[1], 8);
    mbar_init(dq_done, 1);
    mbar_init(clean, 1);
    for (int i = 0; i < RING; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
    }
    mbar_fence_init();
  }
  if (warp == W_MMA) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  allow_next_launch();
  const uint32_t tmem_base = *tmem_slot;
  const PackedSpan span = *reinterpret_cast<const PackedSpan*>(span_smem);
  constexpr uint32_t C_S = 0, C_DP = 256, C_DQ = 384;

  const bool covered = span.unit_in_sequence >= 0;
  const int first = covered ? span.unit_in_sequence * step : 0;
  const int rows = covered ? min(step, span.rows - first) : 0;
  const int q_row = span.q0 + first;
  const int reach = span.keys - span.rows + first;  // row i of the tile sees the keys up to reach + i
  const int seen_last = covered ? min(span.keys, reach + rows) : 0;
  const int n_tiles = seen_last > 0 ? (seen_last + ROWS - 1) / ROWS : 0;
  const int last_valid = span.keys - (n_tiles - 1) * ROWS;
  const bool ragged = n_tiles > 0 && last_valid < ROWS;

  if (warp == W_TMA) {
    if (n_tiles > 0) {
      bool ok = true;
      if (lane == 0) {
        mbar_expect_tx(q_full, 2 * TILE_BYTES);
        load_tile<ATOMS>(sQ, &tm_q, q_full, head0, q_row);
        load_tile<ATOMS>(sdO, &tm_do, q_full, head0, q_row);
        for (int j = 0; j < n_tiles && ok; ++j) {
          const int st = j % RING, sv = j & 1;
          if (!mbar_wait(&k_empty[st], ((j / RING) & 1) ^ 1, guard, kTimeoutProducer)) { ok = false; break; }
          mbar_expect_tx(&k_full[st], TILE_BYTES);
          load_tile<ATOMS>(sK + st * TILE_BYTES, &tm_k, &k_full[st], kv_head, span.k0 + j * ROWS);
          if (!mbar_wait(&v_empty[sv], ((j >> 1) & 1) ^ 1, guard, kTimeoutProducer)) { ok = false; break; }
          mbar_expect_tx(&v_full[sv], TILE_BYTES);
          load_tile<ATOMS>(sV + sv * TILE_BYTES, &tm_v, &v_full[sv], kv_head, span.k0 + j * ROWS);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (ragged && ok) {
        const int j = n_tiles - 1, st = j % RING, sv = j & 1;
        ok = mbar_wait_w(&k_full[st], (j / RING) & 1, guard, kTimeoutProducer) &&
             mbar_wait_w(&v_full[sv], (j >> 1) & 1, guard, kTimeoutProducer);
        if (ok) {
          clear_rows<ATOMS>(smem_u32(sK + st * TILE_BYTES), last_valid, lane);
          clear_rows<ATOMS>(smem_u32(sV + sv * TILE_BYTES), last_valid, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(clean);
        }
      }
      if (!ok || *abort_flag) {
        // give in-flight copies time to land before shared memory is released
        const uint64_t start = global_timer_ns();
        while (global_timer_ns() - start < 100000ull) {}
      }
    }
  } else if (warp == W_MMA) {
    if (n_tiles > 0 && elect_one()) {
      constexpr uint32_t idesc_kk = make_idesc_16(FP16, ROWS, ROWS, 0, 0);  // both K-major
      constexpr uint32_t idesc_mn = make_idesc_16(FP16, ROWS, DP, 0, 1);    // B MN-major
      const uint32_t q_addr = smem_u32(sQ), do_addr = smem_u32(sdO);
      bool ok = mbar_wait(q_full, 0, guard, kTimeoutMma);
      // S of tile j into buffer j & 1 (its last reader, the exponentials of tile j - 2, finished
      // before dS(j-2) was announced, which the dQ product of that tile waited for).
      auto score_s = [&](int j) -> bool {
        const int st = j % RING;
        if (!mbar_wait(&k_full[st], (j / RING) & 1, guard, kTimeoutMma)) return false;
        if (ragged && j == n_tiles - 1 && !mbar_wait(clean, 0, guard, kTimeoutMma)) return false;
        tc_fence_after_sync();
        const uint32_t k_addr = smem_u32(sK + st * TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (kk >> 2) * HALF_BYTES + (kk & 3) * 32;
          tc_mma_ss(tmem_base + C_S + (j & 1) * 128, make_smem_desc(q_addr + off, 16, 1024),
                      make_smem_desc(k_addr + off, 16, 1024), idesc_kk, kk != 0);
        }
        tc_commit(&s_full[j & 1]);
        return true;
      };
      // dP of tile j over dS(j-1), behind the dQ product that read it.
      auto score_p = [&](int j) -> bool {
        const int st = j & 1;
        if (!mbar_wait(&v_full[st], (j >> 1) & 1, guard, kTimeoutMma)) return false;
        tc_fence_after_sync();
        const uint32_t v_addr = smem_u32(sV + st * TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (kk >> 2) * HALF_BYTES + (kk & 3) * 32;
          tc_mma_ss(tmem_base + C_DP, make_smem_desc(do_addr + off, 16, 1024),
                      make_smem_desc(v_addr + off, 16, 1024), idesc_kk, kk != 0);
        }
        tc_commit(dp_full);
        tc_commit(&v_empty[st]);
        return true;
      };
      if (ok) ok = score_s(0);
      if (ok) ok = score_p(0);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int st = j % RING;
        if (j + 1 < n_tiles && !score_s(j + 1)) { ok = false; break; }
        const uint32_t k_addr = smem_u32(sK + st * TILE_BYTES);
        // 16 keys per step; the packed columns of the 32 keys [32 g, 32 g + 32) start at column
        // 32 g.  The warps announce dS in two parts (their first and their second 32 columns:
        // g = c and g = 2 + c), so half of the product is issued while they finish the rest.
#pragma unroll
        for (int c = 0; c < 2 && ok; ++c) {
          if (!mbar_wait(&ds_ready[c], j & 1, guard, kTimeoutMma)) { ok = false; break; }
          tc_fence_after_sync();
#pragma unroll
          for (int s4 = 0; s4 < 4; ++s4) {
            const int kk = (s4 >> 1) * 4 + c * 2 + (s4 & 1);
            tc_mma_ts(tmem_base + C_DQ, tmem_base + C_DP + (kk >> 1) * 32 + (kk & 1) * 8,
                        make_smem_desc(k_addr + kk * 2048, HALF_BYTES, 1024), idesc_mn, (j | c | s4) != 0);
          }
        }
        if (!ok) break;
        tc_commit(&k_empty[st]);
        if (j + 1 < n_tiles && !score_p(j + 1)) { ok = false; break; }
      }
      if (ok) tc_commit(dq_done);
    }
    __syncwarp();
  } else if (warp < 8) {
    // Warps q and q + 4 share the 32 rows of TMEM lane quarter q and take one half of the 128 key
    // columns each.
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lane_base = uint32_t(quarter * 32) << 16;
    const int my_row = quarter * 32 + lane;
    const int live = rows << p.shift, fold_mask = (1 << p.shift) - 1;
    const bool row_ok = my_row < live;
    const int64_t stat_index = int64_t(head0 + (my_row & fold_mask)) * p.total_q + q_row + (my_row >> p.shift);
    // delta of 16 rows a warp, four elements a lane, whole rows an instruction (one row a thread took 7000
    // cycles); all loads are on their way before the first sum
    {
      const int row0 = warp * 16, e = lane * 4;
      const uint16_t* o = static_cast<const uint16_t*>(p.out) + (int64_t(q_row) * p.hq + head0) * p.dim + e;
      const uint16_t* g = static_cast<const uint16_t*>(p.grad) + int64_t(q_row) * p.grad_row + head0 * p.grad_head + e;
      uint2 a[16], b[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        a[r] = b[r] = make_uint2(0, 0);
        const int down = row0 + r >> p.shift, across = row0 + r & fold_mask;
        if (row0 + r < live && e < p.dim) {
          a[r] = *reinterpret_cast<const uint2*>(o + (down * p.hq + across) * p.dim);
          b[r] = *reinterpret_cast<const uint2*>(g + down * p.grad_row + across * p.grad_head);
        }
      }
      float part[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float2 x0 = unpack16<FP16>(a[r].x), x1 = unpack16<FP16>(a[r].y);
        const float2 y0 = unpack16<FP16>(b[r].x), y1 = unpack16<FP16>(b[r].y);
        part[r] = fmaf(x0.x, y0.x, fmaf(x0.y, y0.y, fmaf(x1.x, y1.x, x1.y * y1.y)));
      }
      // sixteen sums over the lanes at once: every exchange halves the rows a lane still adds up
#pragma unroll
      for (int d = 16; d > 1; d /= 2) {
        const bool upper = lane & d;
#pragma unroll
        for (int r = 0; r < d / 2; ++r) {
          const float send = upper ? part[r] : part[r + d / 2], keep = upper ? part[r + d / 2] : part[r];
          part[r] = keep + __shfl_xor_sync(0xffffffffu, send, d);
        }
      }
      part[0] += __shfl_xor_sync(0xffffffffu, part[0], 1);
      if ((lane & 1) == 0) deltas[row0 + (lane >> 1)] = part[0];
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const float delta = deltas[my_row];
    if (row_ok && half == 0) p.delta[stat_index] = delta;
    const float lse2 = row_ok ? p.lse[stat_index] * LOG2E : 0.f;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    const float2 nl2 = make_float2(-lse2, -lse2);
    const float2 nd2 = make_float2(-delta, -delta);
    const int seen = row_ok ? min(span.keys, reach + (my_row >> p.shift) + 1) : 0;
    const int seen_first = rows == step ? min(span.keys, reach + 1) : 0;
    bool ok = n_tiles > 0;
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int buf = j & 1;
      if (!mbar_wait(&s_full[buf], (j >> 1) & 1, guard, kTimeoutSoftmax)) { ok = false; break; }
      tc_fence_after_sync();
      // only tiles with masked keys or rows pay for the masking; the test is uniform over the CTA
      const bool plain = seen_first >= (j + 1) * ROWS;
      const int valid = seen - j * ROWS;
      float2 prob[32];  // probabilities of this thread's 64 key columns, kept for dS
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t sv[32];
        tmem_ld_32x32(tmem_base + lane_base + C_S + buf * 128 + half * 64 + c * 32, sv);
        tmem_ld_wait();
        if (plain) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 x = ffma2(make_float2(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1])), sc2, nl2);
            prob[c * 16 + i] = i % 4 == 3 ? exp2_pair<true>(x) : exp2_pair<false>(x);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 x = ffma2(make_float2(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1])), sc2, nl2);
            const float2 e = exp2_pair<false>(x);
            const int col = half * 64 + c * 32 + 2 * i;
            prob[c * 16 + i] = make_float2(col >= valid ? 0.f : e.x, col + 1 >= valid ? 0.f : e.y);
          }
        }
      }
      if (!mbar_wait(dp_full, j & 1, guard, kTimeoutSoftmax)) { ok = false; break; }
      tc_fence_after_sync();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t dv[32], packed[16];
        tmem_ld_32x32(tmem_base + lane_base + C_DP + half * 64 + c * 32, dv);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 g = fadd2(make_float2(__uint_as_float(dv[2 * i]), __uint_as_float(dv[2 * i + 1])), nd2);
          const float2 ds = fmul2(prob[c * 16 + i], g);
          packed[i] = pack16<FP16>(ds.x, ds.y);
        }
        // the packed results land in columns this thread has already read
        tmem_st_32x16(tmem_base + lane_base + C_DP + half * 64 + c * 32, packed);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_ready[c]);
      }
    }
    if (ok) ok = mbar_wait(dq_done, 0, guard, kTimeoutEpilogue);
    if (n_tiles == 0 || ok) {
      tc_fence_after_sync();
      // every product is complete: the stages lie over the Q and dO tiles
      if (half < DP / 64) {
        const int64_t row = int64_t(q_row) + (quarter * 32 >> p.shift);
        store_columns<FP16>(static_cast<uint16_t*>(p.dq) + (row * p.hq + head0) * p.dim + half * 64, p.hq * p.dim, p.dim,
                            p.shift, tmem_base + lane_base + C_DQ + half * 64, p.dim - half * 64, p.scale,
                            live - quarter * 32, n_tiles > 0, true, smem_u32(smem + warp * 4096), lane);
      }
    }
    if (span.unit_in_sequence == -2) {  // rows behind the last sequence
      const int words = (p.dim << p.shift) / 8;
      for (int i = int(threadIdx.x); i < span.rows * words; i += 256)
        store16(static_cast<uint16_t*>(p.dq) + ((int64_t(span.q0) + i / words) * p.hq + head0) * p.dim + (i % words) * 8,
                make_uint4(0, 0, 0, 0));
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == W_MMA) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------- dK / dV
// With few key tiles, the two CTAs of a cluster take the items in turn and add their accumulators at
// the end through each other's shared memory, in the order of their ranks: the first key tile of a
// sequence is seen by all of its queries and would decide how long the launch takes.
// Items are blocks of 128 (query row, head) pairs that can see the tile, issued
// dV(i) | S^T(i+1) | dK(i) | dP^T(i+1): the exponentials of item i+1 run under dK(i) and dP^T(i+1), its
// dS^T under dV(i+1) and S^T(i+2).  Single score buffers: refilling one behind the product that
// reads its P^T / dS^T is safe, tcgen05.mma operations of one thread execute in issue order.
// TMEM: S^T [0,128) dP^T [128,256) dV [256,384) dK [384,512).  Warps k and k + 4 share the 32 key
// rows of lane quarter k and take 64 of the 128 query columns each, 32 at a time; the packed
// results overwrite the first 16 columns of the 32 they came from.
template <int DP, bool FP16>
__global__ void __launch_bounds__(BWD_THREADS, 1)
packed_dkdv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                   const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const BwdParams p) {
  constexpr int ATOMS = DP / 64;
  constexpr int TILE_BYTES = ATOMS * HALF_BYTES;
  extern __shared__ __align__(1024) uint8_t smem[];  // the swizzle counts addresses in blocks of 1024 bytes
  uint8_t* sK = smem;
  uint8_t* sV = smem + TILE_BYTES;
  uint8_t* sQ = smem + 2 * TILE_BYTES;      // [RING]
  uint8_t* sdO = smem + 5 * TILE_BYTES;     // [2]
  float* stats = reinterpret_cast<float*>(smem + 7 * TILE_BYTES);  // [2][-lse log2(e) [128], -delta [128]]
  uint64_t* bars = reinterpret_cast<uint64_t*>(stats + 4 * ROWS);
  uint64_t* kv_full = bars;
  uint64_t* q_full = bars + 1;      // [RING]
  uint64_t* q_empty = bars + 4;     // [RING]
  uint64_t* do_full = bars + 7;     // [2]
  uint64_t* do_empty = bars + 9;    // [2]
  uint64_t* st_full = bars + 11;    // S^T of an item complete
  uint64_t* dp_full = bars + 12;    // dP^T of an item complete
  uint64_t* pt_ready = bars + 13;   // [2] P^T of query chunk c of both halves written (count 8)
  uint64_t* ds_ready = bars + 15;   // dS^T written (count 8)
  uint64_t* grad_done = bars + 16;  // all gradient products finished
  uint64_t* stats_full = bars + 17; // [2] lse and delta of an item staged
  uint64_t* stats_empty = bars + 19;  // [2] and read (count 8)
  uint64_t* clean = bars + 21;      // [2] rows of a ragged query block behind the last query cleared
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* span_smem = reinterpret_cast<int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int member = int(blockIdx.x % unsigned(p.share));  // rank in the cluster
  const int kv_head = int((blockIdx.x / unsigned(p.share)) % unsigned(p.hkv));
  const int unit = int(blockIdx.x / (unsigned(p.share) * unsigned(p.hkv)));
  const int step = ROWS >> p.shift, fold_mask = (1 << p.shift) - 1;  // query rows of an item
  const WaitGuard guard{abort_flag, p.status};

  if (warp == 0) {
    const PackedSpan span = find_piece(unit, ROWS, true, p.q_offsets, p.k_offsets, p.k_lengths, p.sequences,
                                       p.total_q, p.total_k, kv_head == 0 && member == 0 ? p.status : nullptr);
    if (lane == 0) *reinterpret_cast<PackedSpan*>(span_smem) = span;
  }
  if (warp == 1 && lane == 0) {
    *abort_flag = 0;
    mbar_init(kv_full, 1);
    mbar_init(grad_done, 1);
    mbar_init(st_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(&pt_ready[0], 8);
    mbar_init(&pt_ready[1], 8);
    mbar_init(ds_ready, 8);
    for (int i = 0; i < RING; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&do_full[i], 1);
      mbar_init(&do_empty[i], 1);
      mbar_init(&clean[i], 1);
      mbar_init(&stats_full[i], 1);
      mbar_init(&stats_empty[i], 8);
    }
    mbar_fence_init();
  }
  if (warp == W_MMA) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const PackedSpan span = *reinterpret_cast<const PackedSpan*>(span_smem);
  constexpr uint32_t C_ST = 0, C_DPT = 128, C_DV = 256, C_DK = 384;

  const bool covered = span.unit_in_sequence >= 0;
  const int k_first = covered ? span.unit_in_sequence * ROWS : 0;
  const int k_rows = covered ? min(ROWS, span.room - k_first) : 0;       // rows this CTA writes
  const int k_valid = covered ? max(0, min(ROWS, span.keys - k_first)) : 0;
  const int shift = span.keys - span.rows;                                // query i sees the keys up to i + shift
  const int i0 = max(0, k_first - shift);                                 // the first query that sees the tile
  const int blocks = covered && k_valid > 0 && i0 < span.rows ? (span.rows - i0 + step - 1) / step : 0;
  const int all_items = blocks * (p.group >> p.shift);                    // of the cluster: heads, blocks fastest
  const int n_items = all_items > member ? (all_items - member + p.share - 1) / p.share : 0;
  const int tail_rows = span.rows - i0 - (blocks - 1) * step;             // queries of the last block
  const bool ragged = blocks > 0 && tail_rows < step;
  // block and first head of this member's first item, and how to go on to its next one
  int block = member, head0 = kv_head * p.group;
  auto settle = [&] {
    while (block >= blocks) {
      block -= blocks;
      head0 += 1 << p.shift;
    }
  };
  if (n_items > 0) settle();
  auto advance = [&] {
    block += p.share;
    settle();
  };

  if (warp == W_TMA) {
    if (n_items > 0) {
      if (lane == 0) {
        mbar_expect_tx(kv_full, 2 * TILE_BYTES);
        load_tile<ATOMS>(sK, &tm_k, kv_full, kv_head, span.k0 + k_first);
        load_tile<ATOMS>(sV, &tm_v, kv_full, kv_head, span.k0 + k_first);
      }
      bool ok = true, waited = false;
      for (int i = 0; i < n_items && ok; ++i) {
        const int st = i % RING, sd = i & 1;
        ok = mbar_wait_w(&q_empty[st], ((i / RING) & 1) ^ 1, guard, kTimeoutProducer);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(&q_full[st], TILE_BYTES);
          load_tile<ATOMS>(sQ + st * TILE_BYTES, &tm_q, &q_full[st], head0, span.q0 + i0 + block * step);
        }
        ok = mbar_wait_w(&do_empty[sd], ((i >> 1) & 1) ^ 1, guard, kTimeoutProducer);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(&do_full[sd], TILE_BYTES);
          load_tile<ATOMS>(sdO + sd * TILE_BYTES, &tm_do, &do_full[sd], head0, span.q0 + i0 + block * step);
        }
        // -lse * log2(e) (or -inf: probability 0) and -delta of the item's queries; delta is the other
        // kernel's, at whose end this one starts
        if (!waited) after_previous_launch();
        waited = true;
        {
          float nl[4], nd[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int q = i0 + block * step + (k * 32 + lane >> p.shift);
            const bool there = q < span.rows;
            const int64_t at = int64_t(head0 + (lane & fold_mask)) * p.total_q + span.q0 + q;
            nl[k] = there ? -p.lse[at] * LOG2E : -INFINITY;
            nd[k] = there ? -p.delta[at] : 0.f;
          }
          ok = mbar_wait_w(&stats_empty[sd], ((i >> 1) & 1) ^ 1, guard, kTimeoutProducer);
          if (!ok) break;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            stats[sd * 2 * ROWS + k * 32 + lane] = nl[k];
            stats[sd * 2 * ROWS + ROWS + k * 32 + lane] = nd[k];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&stats_full[sd]);
        }
        if (ragged && block == blocks - 1) {
          ok = mbar_wait_w(&q_full[st], (i / RING) & 1, guard, kTimeoutProducer) &&
               mbar_wait_w(&do_full[sd], (i >> 1) & 1, guard, kTimeoutProducer);
          if (!ok) break;
          clear_rows<ATOMS>(smem_u32(sQ + st * TILE_BYTES), tail_rows << p.shift, lane);
          clear_rows<ATOMS>(smem_u32(sdO + sd * TILE_BYTES), tail_rows << p.shift, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&clean[sd]);
        }
        if (i + 1 < n_items) advance();
      }
      if (!ok || *abort_flag) {
        const uint64_t start = global_timer_ns();
        while (global_timer_ns() - start < 100000ull) {}
      }
    }
  } else if (warp == W_MMA) {
    if (n_items > 0 && elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_16(FP16, ROWS, ROWS, 0, 0);  // 128 keys x 128 queries
      constexpr uint32_t idesc_g = make_idesc_16(FP16, ROWS, DP, 0, 1);    // 128 keys x d
      const uint32_t k_addr = smem_u32(sK), v_addr = smem_u32(sV);
      uint32_t cleaned = 0;  // bit sd: parity of the stage's next cleared block
      // S^T of item i (needs its Q in shared memory; the buffer's last reader, dV(i-1), was
      // issued before).
      auto score_s = [&](int i) -> bool {
        const int st = i % RING, sd = i & 1;
        if (!mbar_wait(&q_full[st], (i / RING) & 1, guard, kTimeoutMma)) return false;
        if (ragged && block == blocks - 1) {
          if (!mbar_wait(&clean[sd], (cleaned >> sd) & 1, guard, kTimeoutMma)) return false;
          cleaned ^= 1u << sd;
        }
        if (i + 1 < n_items) advance();
        tc_fence_after_sync();
        const uint32_t q_addr = smem_u32(sQ + st * TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (kk >> 2) * HALF_BYTES + (kk & 3) * 32;
          tc_mma_ss(tmem_base + C_ST, make_smem_desc(k_addr + off, 16, 1024),
                      make_smem_desc(q_addr + off, 16, 1024), idesc_s, kk != 0);
        }
        tc_commit(st_full);
        return true;
      };
      // dP^T of item i (the buffer's last reader, dK(i-1), was issued before).
      auto score_p = [&](int i) -> bool {
        if (!mbar_wait(&do_full[i & 1], (i >> 1) & 1, guard, kTimeoutMma)) return false;
        tc_fence_after_sync();
        const uint32_t do_addr = smem_u32(sdO + (i & 1) * TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (kk >> 2) * HALF_BYTES + (kk & 3) * 32;
          tc_mma_ss(tmem_base + C_DPT, make_smem_desc(v_addr + off, 16, 1024),
                      make_smem_desc(do_addr + off, 16, 1024), idesc_s, kk != 0);
        }
        tc_commit(dp_full);
        return true;
      };
      bool ok = mbar_wait(kv_full, 0, guard, kTimeoutMma);
      if (ok) ok = score_s(0);
      if (ok) ok = score_p(0);
      for (int i = 0; i < n_items && ok; ++i) {
        const int st = i % RING;
        const uint32_t q_addr = smem_u32(sQ + st * TILE_BYTES);
        const uint32_t do_addr = smem_u32(sdO + (i & 1) * TILE_BYTES);
        // 16 queries per step; the packed columns of the 32 queries [32 g, 32 g + 32) start at
        // column 32 g.  The warps announce P^T in two parts (their first and their second 32
        // columns: g = c and g = 2 + c).
#pragma unroll
        for (int c = 0; c < 2 && ok; ++c) {
          if (!mbar_wait(&pt_ready[c], i & 1, guard, kTimeoutMma)) { ok = false; break; }
          tc_fence_after_sync();
#pragma unroll
          for (int s4 = 0; s4 < 4; ++s4) {
            const int kk = (s4 >> 1) * 4 + c * 2 + (s4 & 1);
            tc_mma_ts(tmem_base + C_DV, tmem_base + C_ST + (kk >> 1) * 32 + (kk & 1) * 8,
                        make_smem_desc(do_addr + kk * 2048, HALF_BYTES, 1024), idesc_g, (i | c | s4) != 0);
          }
        }
        if (!ok) break;
        tc_commit(&do_empty[i & 1]);
        if (i + 1 < n_items && !score_s(i + 1)) { ok = false; break; }
        if (!mbar_wait(ds_ready, i & 1, guard, kTimeoutMma)) { ok = false; break; }
        tc_fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < ROWS / 16; ++kk)
          tc_mma_ts(tmem_base + C_DK, tmem_base + C_DPT + (kk >> 1) * 32 + (kk & 1) * 8,
                      make_smem_desc(q_addr + kk * 2048, HALF_BYTES, 1024), idesc_g, (i | kk) != 0);
        tc_commit(&q_empty[st]);
        if (i + 1 < n_items && !score_p(i + 1)) { ok = false; break; }
      }
      if (ok) tc_commit(grad_done);
    }
    __syncwarp();
  } else if (warp < 8) {
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lane_base = uint32_t(quarter * 32) << 16;
    const int tid = (warp << 5) + lane;      // 0..255
    const int key = quarter * 32 + lane;     // key row of this thread
    bool ok = n_items > 0;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    for (int i = 0; i < n_items && ok; ++i) {
      const int st = i & 1;
      const int q_first = i0 + block * step;
      const int q_rows = min(step, span.rows - q_first) << p.shift;  // (query row, head) pairs
      if (i + 1 < n_items) advance();
      const uint32_t my_stats = smem_u32(stats + st * 2 * ROWS + half * 64);
      // query column c sees this key where c >= from, of the block's q_rows; only blocks that mask
      // pay for it, and the test is uniform over the CTA
      const int from = key < k_valid ? max(0, k_first + key - shift - q_first) << p.shift : ROWS;
      const bool plain = k_valid == ROWS && q_rows == ROWS && k_first + ROWS - 1 - shift <= q_first;
      if (!mbar_wait(&stats_full[st], (i >> 1) & 1, guard, kTimeoutSoftmax)) { ok = false; break; }
      if (!mbar_wait(st_full, i & 1, guard, kTimeoutSoftmax)) { ok = false; break; }
      tc_fence_after_sync();
      float2 prob[32];  // the probabilities of this thread's 64 query columns, kept for dS^T
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t sv[32], pp[16];
        tmem_ld_32x32(tmem_base + lane_base + C_ST + half * 64 + c * 32, sv);
        tmem_ld_wait();
        auto four = [&](int k4, auto fma) {  // four query columns
          const uint4 nl = get16(my_stats + c * 128 + k4 * 16);
          const float2 x0 = ffma2(make_float2(__uint_as_float(sv[4 * k4]), __uint_as_float(sv[4 * k4 + 1])), sc2,
                                  make_float2(__uint_as_float(nl.x), __uint_as_float(nl.y)));
          const float2 x1 = ffma2(make_float2(__uint_as_float(sv[4 * k4 + 2]), __uint_as_float(sv[4 * k4 + 3])), sc2,
                                  make_float2(__uint_as_float(nl.z), __uint_as_float(nl.w)));
          prob[c * 16 + 2 * k4] = exp2_pair<false>(x0);
          prob[c * 16 + 2 * k4 + 1] = exp2_pair<decltype(fma)::value>(x1);
        };
        if (plain) {
#pragma unroll
          for (int k4 = 0; k4 < 8; ++k4) {
            if (k4 & 1) four(k4, std::true_type{});
            else four(k4, std::false_type{});
          }
        } else {
#pragma unroll
          for (int k4 = 0; k4 < 8; ++k4) {
            four(k4, std::false_type{});
            float2 &e0 = prob[c * 16 + 2 * k4], &e1 = prob[c * 16 + 2 * k4 + 1];
            const int col = half * 64 + c * 32 + 4 * k4;
            if (col < from || col >= q_rows) e0.x = 0.f;
            if (col + 1 < from || col + 1 >= q_rows) e0.y = 0.f;
            if (col + 2 < from || col + 2 >= q_rows) e1.x = 0.f;
            if (col + 3 < from || col + 3 >= q_rows) e1.y = 0.f;
          }
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) pp[k] = pack16<FP16>(prob[c * 16 + k].x, prob[c * 16 + k].y);
        // the packed results land in columns this thread has already read
        tmem_st_32x16(tmem_base + lane_base + C_ST + half * 64 + c * 32, pp);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pt_ready[c]);
      }
      if (!mbar_wait(dp_full, i & 1, guard, kTimeoutSoftmax)) { ok = false; break; }
      tc_fence_after_sync();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t dv[32], dd[16];
        tmem_ld_32x32(tmem_base + lane_base + C_DPT + half * 64 + c * 32, dv);
        tmem_ld_wait();
#pragma unroll
        for (int k4 = 0; k4 < 8; ++k4) {
          const uint4 nd = get16(my_stats + ROWS * 4 + c * 128 + k4 * 16);
          const float2 g0 = fadd2(make_float2(__uint_as_float(dv[4 * k4]), __uint_as_float(dv[4 * k4 + 1])),
                                  make_float2(__uint_as_float(nd.x), __uint_as_float(nd.y)));
          const float2 g1 = fadd2(make_float2(__uint_as_float(dv[4 * k4 + 2]), __uint_as_float(dv[4 * k4 + 3])),
                                  make_float2(__uint_as_float(nd.z), __uint_as_float(nd.w)));
          const float2 d0 = fmul2(prob[c * 16 + 2 * k4], g0), d1 = fmul2(prob[c * 16 + 2 * k4 + 1], g1);
          dd[2 * k4] = pack16<FP16>(d0.x, d0.y);
          dd[2 * k4 + 1] = pack16<FP16>(d1.x, d1.y);
        }
        tmem_st_32x16(tmem_base + lane_base + C_DPT + half * 64 + c * 32, dd);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(ds_ready);
        mbar_arrive(&stats_empty[st]);
      }
    }
    if (ok) ok = mbar_wait(grad_done, 0, guard, kTimeoutEpilogue);
    if ((all_items == 0 && member == 0) || (ok && p.share == 1)) {
      tc_fence_after_sync();
      // the two halves write one gradient each; every product is complete: the stages lie over the K
      // and V tiles.  Rows that are no keys (the room behind them) get zeros.
      const int64_t row = int64_t(span.k0) + k_first + quarter * 32;
      uint16_t* dst = static_cast<uint16_t*>(half == 0 ? p.dv : p.dk) + (row * p.hkv + kv_head) * p.dim;
#pragma unroll 1
      for (int c = 0; c < DP / 64; ++c)
        store_columns<FP16>(dst + c * 64, p.hkv * p.dim, 0, 0,
                            tmem_base + lane_base + (half == 0 ? C_DV : C_DK) + c * 64, p.dim - c * 64,
                            half == 0 ? 1.f : p.scale, k_rows - quarter * 32, n_items > 0, key < k_valid,
                            smem_u32(smem + warp * 4096), lane);
    }
    if (span.unit_in_sequence == -2 && member == 0) {  // rows behind the last sequence
      const int words = p.dim / 8;
      for (int i = tid; i < span.rows * words; i += 256) {
        const int64_t at = ((int64_t(span.k0) + i / words) * p.hkv + kv_head) * p.dim + (i % words) * 8;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dk) + at) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dv) + at) = make_uint4(0, 0, 0, 0);
      }
    }
  }
  after_previous_launch();
  if (p.share > 1 && all_items > 0) {
    // dV and dK side by side are 2 DP columns; each member adds up `width` of them.
    const int width = 2 * DP / p.share;
    const int quarter = warp & 3, half = (warp >> 2) & 1;
    const int key = quarter * 32 + lane;
    const uint32_t column0 = tmem_base + (uint32_t(quarter * 32) << 16) + C_DV;
    auto column = [&](int c) { return c < DP ? c : c - DP + int(C_DK - C_DV); };
    // 16-byte word w (of a row of `width` FP32 columns) of a sender's part
    auto place = [&](int sender, int row, int w) {
      return smem_u32(smem) + ((sender * ROWS + row) * width + (w & ~7) * 4) * 4 + ((w ^ row) & 7) * 16;
    };
    tc_fence_before_sync();
    cluster_sync();  // no member reads its tiles any more
    tc_fence_after_sync();
    if (warp < 8) {
      for (int to = 0; to < p.share; ++to) {
        if (to == member) continue;
        const int sender = member < to ? member : member - 1;
        for (int c = half * 32; c < width; c += 64) {
          uint32_t o[32] = {};  // a member without items adds nothing
          if (n_items > 0) {
            tmem_ld_32x32(column0 + column(to * width + c), o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int g = 0; g < 8; ++g)
            put16_member(place(sender, key, c / 4 + g), to, make_uint4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]));
        }
      }
    }
    cluster_sync();
    if (warp < 8) {
      for (int c = half * 32; c < width; c += 64) {
        const int at = member * width + c;
        uint32_t o[32] = {};
        if (n_items > 0) {
          tmem_ld_32x32(column0 + column(at), o);
          tmem_ld_wait();
        }
        float sum[32];
#pragma unroll 1
        for (int from = 0; from < p.share; ++from) {
          const int sender = from < member ? from : from - 1;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const uint4 v = from == member ? make_uint4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3])
                                           : get16(place(sender, key, c / 4 + g));
            sum[4 * g] = __uint_as_float(v.x) + (from == 0 ? 0.f : sum[4 * g]);
            sum[4 * g + 1] = __uint_as_float(v.y) + (from == 0 ? 0.f : sum[4 * g + 1]);
            sum[4 * g + 2] = __uint_as_float(v.z) + (from == 0 ? 0.f : sum[4 * g + 2]);
            sum[4 * g + 3] = __uint_as_float(v.w) + (from == 0 ? 0.f : sum[4 * g + 3]);
          }
        }
        if (key < k_rows) {  // rows that are no keys (the room behind them) get zeros
          const bool is_dv = at < DP;
          const int d0 = is_dv ? at : at - DP;
          const float scale = key < k_valid ? (is_dv ? 1.f : p.scale) : 0.f;
          uint16_t* dst = static_cast<uint16_t*>(is_dv ? p.dv : p.dk) +
                          ((int64_t(span.k0) + k_first + key) * p.hkv + kv_head) * p.dim + d0;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (key < k_valid) {
              v.x = pack16<FP16>(sum[8 * g] * scale, sum[8 * g + 1] * scale);
              v.y = pack16<FP16>(sum[8 * g + 2] * scale, sum[8 * g + 3] * scale);
              v.z = pack16<FP16>(sum[8 * g + 4] * scale, sum[8 * g + 5] * scale);
              v.w = pack16<FP16>(sum[8 * g + 6] * scale, sum[8 * g + 7] * scale);
            }
            if (d0 + g * 8 < p.dim) store16(dst + g * 8, v);
          }
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == W_MMA) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int DP, bool FP16>
cudaError_t launch(const BwdParams& p, const CUtensorMap& tq, const CUtensorMap& tdo, const CUtensorMap& tk,
                   const CUtensorMap& tv, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed_dq{0}, allowed_dkdv{0};
  cudaError_t e = allow_shared_memory(packed_dq_kernel<DP, FP16>, bwd_smem<DP>(), allowed_dq);
  if (e == cudaSuccess) e = allow_shared_memory(packed_dkdv_kernel<DP, FP16>, bwd_smem<DP>(), allowed_dkdv);
  if (e != cudaSuccess) return e;
  const int64_t q_grid = (p.total_q / (ROWS >> p.shift) + p.sequences + 1) * (p.hq >> p.shift);
  const int64_t k_units = (p.total_k / ROWS + p.sequences + 1) * p.hkv, k_grid = k_units * p.share;
  if (q_grid > 2147483647ll || k_grid > 2147483647ll) {
    set_error_detail("packed_attention: too many tiles for one launch");
    return cudaErrorInvalidValue;
  }
  packed_dq_kernel<DP, FP16><<<unsigned(q_grid), BWD_THREADS, bwd_smem<DP>(), stream>>>(tq, tdo, tk, tv, p);
  e = cudaGetLastError();
  if (e != cudaSuccess || !p.dk) return e;
  cudaLaunchAttribute attributes[2]{};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = unsigned(p.share);
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned(k_grid));
  config.blockDim = dim3(BWD_THREADS);
  config.dynamicSmemBytes = bwd_smem<DP>();
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, packed_dkdv_kernel<DP, FP16>, tq, tdo, tk, tv, p);
}

}  // namespace

cudaError_t packed_attention_bwd(const PackedArgs& a, const PackedGrads& g, cudaStream_t stream) {
  CUtensorMap tq, tdo, tk, tv;
  const int shift = fold_shift(a.hq / a.hkv);
  if (!make_packed_map(&tq, a.q, a.dim, a.hq, a.total_q, a.q_head, a.q_row, 1 << shift) ||
      !make_packed_map(&tdo, g.grad, a.dim, a.hq, a.total_q, g.grad_head, g.grad_row, 1 << shift) ||
      !make_packed_map(&tk, a.k, a.dim, a.hkv, a.total_k, a.k_head, a.k_row, 1) ||
      !make_packed_map(&tv, a.v, a.dim, a.hkv, a.total_k, a.v_head, a.v_row, 1))
    return cudaErrorInvalidValue;
  BwdParams p{};
  p.q_offsets = a.q_offsets; p.k_offsets = a.k_offsets; p.k_lengths = a.k_lengths;
  p.sequences = a.sequences;
  p.total_q = a.total_q; p.total_k = a.total_k;
  p.out = a.out; p.grad = g.grad; p.grad_row = g.grad_row; p.grad_head = g.grad_head;
  p.lse = a.lse; p.delta = g.delta;
  p.dq = g.dq; p.dk = g.dk; p.dv = g.dv;
  p.hq = a.hq; p.hkv = a.hkv; p.group = a.hq / a.hkv; p.dim = a.dim;
  p.scale = a.scale; p.scale_log2 = a.scale * LOG2E;
  p.status = a.status;
  p.shift = shift;
  // Two where one CTA a key tile leaves fewer than two for every SM.  (Four were slower everywhere: 198 us
  // against 116 for the key side of six prompts of 178 to 2045 rows, 43 against 24 for three of up to
  // 1000: clusters of four whole SMs wait for one another to start.)
  p.share = (a.total_k / ROWS + a.sequences) * a.hkv < int64_t(2) * a.sm_count ? 2 : 1;
  if (a.dim <= 64)
    return a.fp16 ? launch<64, true>(p, tq, tdo, tk, tv, stream) : launch<64, false>(p, tq, tdo, tk, tv, stream);
  return a.fp16 ? launch<128, true>(p, tq, tdo, tk, tv, stream) : launch<128, false>(p, tq, tdo, tk, tv, stream);
}

}  // namespace agb
