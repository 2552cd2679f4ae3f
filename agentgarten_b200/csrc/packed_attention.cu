// Causal attention over packed sequences, forward, on tcgen05 (bf16 or fp16, heads of up to 128).
//
//   s = scale q k^T over the visible keys (j <= i + keys - rows), p = softmax(s), out = p v
//
// One CTA per (piece of a sequence's queries, two score tiles, key range).  The two tiles of 128
// rows are two query heads that share a key head, or, when a key head has an odd number of query
// heads, two neighbouring tiles of one head; both read the same K and V tiles.
//   warps 0-3  softmax of tile 0: one query row per thread
//   warps 4-7  softmax of tile 1
//   warp 8     TMA producer (K and V through rings of two stages); clears the V rows behind the last
//              key, so that whatever lies there (another sequence, NaN) never meets a product
//   warp 9     MMA issuer: S_t = Q_t K^T, O_t += P_t V with P_t read from TMEM (one elected thread in a
//              branch of its own: a product then takes the pipe's 64 cycles, against 91 to 105 where
//              the whole warp runs the loop and elects a lane for every instruction)
//   warps 10-11 only complete the third warpgroup, which hands registers to the other two
// While one tile is in its softmax the tensor core works for the other.  The running maximum is
// only followed when it grows by more than 2^8: until then the scores are taken relative to the
// old one, which leaves the quotient unchanged.  Sums, maxima and O are FP32; P is rounded to the
// tensors' type, as an operand of the tensor core has to be.
//
// TMEM columns: S_0 [0,128) S_1 [128,256) O_0 [256,384) O_1 [384,512); P_t over the first half of S_t.
#include "agb.h"
#include "packed.h"
#include "packed_common.cuh"
#include "tensormap.h"

#include <type_traits>

namespace agb {
namespace {

constexpr int KV_STAGES = 2;
constexpr int ROWS = 128;          // rows of a score tile, keys of a key tile
constexpr int HALF_BYTES = 16384;  // 128 rows x 64 elements
constexpr int FWD_THREADS = 384;  // three warpgroups: softmax of tile 0, of tile 1, the rest
constexpr int SOFTMAX_REGS = 208, OTHER_REGS = 80;  // 2 x 208 + 80 fit the launch's 3 x 168
constexpr uint32_t COL_S = 0, COL_O = 256;
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units
// Of every eight pairs of unmasked scores, how many take the exponential of the FMA pipe: the
// special-function unit alone (16 a cycle) is as slow as the products of a tile.
constexpr int FMA_PAIRS = 2;
constexpr float LOG2E = 1.4426950408889634f;

template <int DP>
constexpr int fwd_smem() {
  // Q_0, Q_1, K ring, V ring.  Never less than half of an SM's shared memory: two CTAs do not fit
  // in its tensor memory, and the second would wait for the first in its allocation.
  const int bytes = (2 + 2 * KV_STAGES) * (DP / 64) * HALF_BYTES + 1024 + 512;
  return bytes > 120 * 1024 ? bytes : 120 * 1024;
}

struct FwdParams {
  const int* q_offsets; const int* k_offsets; const int* k_lengths;
  int sequences;
  int64_t total_q, total_k;
  void* out;
  float* lse;
  float* part_out; float* part_lse;
  int hq, dim, group, splits;
  int head_units;   // CTAs side by side for one piece: hq / 2 (pairs of heads) or hq
  int paired;       // 1: the tiles are two heads, 0: two neighbouring row tiles
  float scale_log2;
  int* status;
};

template <int DP, bool FP16>
__global__ void __launch_bounds__(FWD_THREADS, 1)
packed_tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const FwdParams p) {
  constexpr int ATOMS = DP / 64;
  constexpr int TILE_BYTES = ATOMS * HALF_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + 2 * TILE_BYTES;
  uint8_t* sV = sK + KV_STAGES * TILE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + KV_STAGES * TILE_BYTES);
  uint64_t* q_full = bars;         // 1
  uint64_t* k_full = bars + 1;     // [2]
  uint64_t* k_empty = bars + 3;    // [2]
  uint64_t* v_full = bars + 5;     // [2]
  uint64_t* v_empty = bars + 7;    // [2]
  uint64_t* s_full = bars + 9;     // [2 tiles] scores complete
  uint64_t* p_ready = bars + 11;   // [2 tiles][2 halves of the keys] probabilities in TMEM (count 4)
  uint64_t* o_done = bars + 15;    // [2 tiles] last product complete
  uint64_t* v_clean = bars + 17;   // rows behind the last key cleared
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* span_smem = reinterpret_cast<int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const WaitGuard guard{abort_flag, p.status};
  const int step = p.paired ? ROWS : 2 * ROWS;
  const int split = int(blockIdx.x % unsigned(p.splits));
  const int head_unit = int((blockIdx.x / unsigned(p.splits)) % unsigned(p.head_units));
  const int unit = int(blockIdx.x / (unsigned(p.splits) * unsigned(p.head_units)));

  if (warp == 0) {
    const PackedSpan span = find_piece(unit, step, false, p.q_offsets, p.k_offsets, p.k_lengths, p.sequences,
                                       p.total_q, p.total_k, head_unit == 0 && split == 0 ? p.status : nullptr);
    if (lane == 0) *reinterpret_cast<PackedSpan*>(span_smem) = span;
  }
  if (warp == 1 && lane == 0) {
    *abort_flag = 0;
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[2 * i], 4);
      mbar_init(&p_ready[2 * i + 1], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(v_clean, 1);
    mbar_fence_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const PackedSpan span = *reinterpret_cast<const PackedSpan*>(span_smem);

  // The tiles of this CTA.
  int head[2], first[2], rows[2], tiles[2];  // first: row within the sequence
  int kv_head = 0, lo = 0, hi = 0;           // range of key tiles
  if (p.paired) {
    head[0] = 2 * head_unit;
    head[1] = head[0] + 1;
  } else {
    head[0] = head[1] = head_unit;
  }
  kv_head = head[0] / p.group;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    first[t] = span.unit_in_sequence * step + (p.paired ? 0 : t * ROWS);
    rows[t] = span.unit_in_sequence < 0 ? 0 : max(0, min(ROWS, span.rows - first[t]));
    const int seen = min(span.keys, span.keys - span.rows + first[t] + rows[t]);  // keys of the last row
    tiles[t] = rows[t] == 0 || seen <= 0 ? 0 : (seen + ROWS - 1) / ROWS;
  }
  {
    const int most = max(tiles[0], tiles[1]);
    const int per = (most + p.splits - 1) / p.splits;
    lo = min(most, split * per);
    hi = min(most, lo + per);
#pragma unroll
    for (int t = 0; t < 2; ++t) tiles[t] = max(0, min(hi, tiles[t]) - lo);
  }
  const int n = hi - lo;
  // Keys of the last tile of the sequence that exist; its rows behind them are cleared.
  const int last_valid = span.keys - (hi - 1) * ROWS;
  const bool ragged = n > 0 && last_valid < ROWS;

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
  if (warp == 8) {
    // ------------------------------------------------------------------ TMA producer
    bool ok = true;
    if (n > 0) {
      if (lane == 0) {
        mbar_expect_tx(q_full, ((tiles[0] > 0) + (tiles[1] > 0)) * TILE_BYTES);
        for (int t = 0; t < 2; ++t)
          if (tiles[t] > 0)
            for (int a = 0; a < ATOMS; ++a)
              tma_load_3d(sQ + t * TILE_BYTES + a * HALF_BYTES, &tm_q, q_full, a * 64, head[t], span.q0 + first[t]);
        for (int j = 0; j < n && ok; ++j) {
          const int st = j % KV_STAGES;
          const uint32_t ph = ((j / KV_STAGES) & 1) ^ 1;
          const int row = span.k0 + (lo + j) * ROWS;
          if (!mbar_wait(&k_empty[st], ph, guard, kTimeoutProducer)) { ok = false; break; }
          mbar_expect_tx(&k_full[st], TILE_BYTES);
          for (int a = 0; a < ATOMS; ++a)
            tma_load_3d(sK + st * TILE_BYTES + a * HALF_BYTES, &tm_k, &k_full[st], a * 64, kv_head, row);
          if (!mbar_wait(&v_empty[st], ph, guard, kTimeoutProducer)) { ok = false; break; }
          mbar_expect_tx(&v_full[st], TILE_BYTES);
          for (int a = 0; a < ATOMS; ++a)
            tma_load_3d(sV + st * TILE_BYTES + a * HALF_BYTES, &tm_v, &v_full[st], a * 64, kv_head, row);
        }
        if (!ok || *abort_flag) {
          // give in-flight copies time to land before shared memory is released
          const uint64_t start = global_timer_ns();
          while (global_timer_ns() - start < 100000ull) {}
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (ragged && ok && mbar_wait_w(&v_full[(n - 1) % KV_STAGES], ((n - 1) / KV_STAGES) & 1, guard, kTimeoutProducer)) {
        // a row is 128 bytes of each atom whatever the swizzle, which permutes within the row
        uint8_t* tile = sV + ((n - 1) % KV_STAGES) * TILE_BYTES;
        for (int i = last_valid * 8 + lane; i < ROWS * 8; i += 32)
          for (int a = 0; a < ATOMS; ++a)
            *reinterpret_cast<uint4*>(tile + a * HALF_BYTES + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_clean);
      }
    }
  } else if (warp == 9) {
    // -------------------------------------------------------------------- MMA issuer
    if (n > 0 && elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_16(FP16, ROWS, ROWS, 0, 0);  // both K-major over d
      constexpr uint32_t idesc_o = make_idesc_16(FP16, ROWS, DP, 0, 1);    // P from TMEM, V MN-major
      auto scores = [&](int t, int j) {
        const uint32_t q_addr = smem_u32(sQ + t * TILE_BYTES);
        const uint32_t k_addr = smem_u32(sK + (j % KV_STAGES) * TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (kk >> 2) * HALF_BYTES + (kk & 3) * 32;
          tc_mma_ss(tmem_base + COL_S + t * 128, make_smem_desc(q_addr + off, 16, 1024),
                    make_smem_desc(k_addr + off, 16, 1024), idesc_s, kk != 0);
        }
        tc_commit(&s_full[t]);
      };
      bool ok = mbar_wait(q_full, 0, guard, kTimeoutMma) && mbar_wait(&k_full[0], 0, guard, kTimeoutMma);
      if (ok) {
        tc_fence_after_sync();
        for (int t = 0; t < 2; ++t)
          if (tiles[t] > 0) scores(t, 0);
        tc_commit(&k_empty[0]);
      }
      for (int j = 0; j < n && ok; ++j) {
        const int st = j % KV_STAGES;
        const bool more = j + 1 < n;
        if (!mbar_wait(&v_full[st], (j / KV_STAGES) & 1, guard, kTimeoutMma)) { ok = false; break; }
        if (!more && ragged && !mbar_wait(v_clean, 0, guard, kTimeoutMma)) { ok = false; break; }
        if (more && !mbar_wait(&k_full[(j + 1) % KV_STAGES], ((j + 1) / KV_STAGES) & 1, guard, kTimeoutMma)) { ok = false; break; }
        const uint32_t v_addr = smem_u32(sV + st * TILE_BYTES);
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= tiles[t]) continue;
#pragma unroll
          for (int c = 0; c < 2 && ok; ++c) {
            if (!mbar_wait(&p_ready[2 * t + c], j & 1, guard, kTimeoutMma)) { ok = false; break; }
            tc_fence_after_sync();
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
              const int kk = c * 4 + k4;  // 16 keys: P advances 8 packed columns, V 16 rows (2048 B)
              tc_mma_ts(tmem_base + COL_O + t * 128, tmem_base + COL_S + t * 128 + kk * 8,
                        make_smem_desc(v_addr + kk * 2048, HALF_BYTES, 1024), idesc_o, (j | kk) != 0);
            }
          }
          if (!ok) break;
          // behind the product above, which reads P from the buffer these scores refill: the
          // tensor core executes one thread's operations in issue order
          if (j + 1 < tiles[t]) scores(t, j + 1);
          else tc_commit(&o_done[t]);
        }
        if (!ok) break;
        tc_commit(&v_empty[st]);
        if (more) tc_commit(&k_empty[(j + 1) % KV_STAGES]);
      }
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    // ----------------------------------------------------------------------- softmax
    const int t = warp >> 2;
    const int quarter = warp & 3;                // TMEM lanes 32*quarter .. +31
    const uint32_t lane_base = uint32_t(quarter * 32) << 16;
    const int my_row = quarter * 32 + lane;
    const uint32_t col_s = tmem_base + lane_base + COL_S + t * 128;
    const uint32_t col_o = tmem_base + lane_base + COL_O + t * 128;
    const int my_tiles = t == 0 ? tiles[0] : tiles[1];
    const int my_first = t == 0 ? first[0] : first[1];
    const int my_rows = t == 0 ? rows[0] : rows[1];
    const int my_head = t == 0 ? head[0] : head[1];
    // keys that this row and the tile's first row see, from the first key of the range on
    const int before = span.keys - span.rows + my_first + 1 - lo * ROWS;
    const int seen = min(span.keys - lo * ROWS, before + my_row);
    const int seen_first = min(span.keys - lo * ROWS, before);
    float m_ref = -INFINITY;                     // reference maximum (log2 domain)
    float l_sum = 0.f;
    bool ok = true;
    for (int j = 0; j < my_tiles && ok; ++j) {
      if (!mbar_wait(&s_full[t], j & 1, guard, kTimeoutSoftmax)) { ok = false; break; }
      tc_fence_after_sync();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(col_s + c * 32, s[c]);
      tmem_ld_wait();
      const bool masked = seen_first < (j + 1) * ROWS;  // the diagonal and the ragged last tile
      if (masked) {
        const int valid = seen - j * ROWS;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i >= valid) s[c][i] = 0xff800000u;  // -inf
      }
      float m4[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        m4[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
        for (int i = 2; i < 32; i += 2)
          m4[c] = fmax3(m4[c], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
      }
      const float m_tile = fmax3(fmaxf(m4[0], m4[1]), m4[2], m4[3]) * p.scale_log2;
      // The previous product of this tile is complete: these scores were executed after it.
      const bool grow = m_tile > m_ref + RESCALE_THRESHOLD;
      if (__any_sync(0xffffffffu, grow)) {
        const float m_new = fmaxf(m_ref, m_tile);
        const float alpha = m_ref == -INFINITY ? 0.f : exp2f(m_ref - m_new);
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(col_o + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32(col_o + c * 32, o);
          }
          tmem_st_wait();
        }
        l_sum *= alpha;
        m_ref = m_new;
      }
      // A row that has seen nothing yet keeps m_ref = -inf: its scores are -inf and the shift is 0.
      const float shift = m_ref == -INFINITY ? 0.f : m_ref;
      const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
      const float2 shift2 = make_float2(-shift, -shift);
      float2 sum2 = make_float2(0.f, 0.f);
      auto probabilities = [&](auto all) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t packed[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const uint32_t* src = &s[2 * c + (i >> 4)][(2 * i) & 31];  // columns 2i, 2i+1 of half c
            const float2 x = ffma2(make_float2(__uint_as_float(src[0]), __uint_as_float(src[1])), scale2, shift2);
            const float2 e = decltype(all)::value && i % 8 < FMA_PAIRS ? exp2_fma(x) : make_float2(exp2f(x.x), exp2f(x.y));
            sum2 = fadd2(sum2, e);
            packed[i] = pack16<FP16>(e.x, e.y);
          }
          tmem_st_32x32(col_s + c * 32, packed);  // over the scores, which are in registers
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[2 * t + c]);
        }
      };
      if (masked) probabilities(std::false_type{});
      else probabilities(std::true_type{});
      l_sum += sum2.x + sum2.y;
    }
    // ---------------------------------------------------------------------- epilogue
    if (ok && my_tiles > 0) ok = mbar_wait(&o_done[t], 0, guard, kTimeoutEpilogue);
    if (ok) {
      tc_fence_after_sync();
      const float inv = l_sum == 0.f ? 0.f : 1.f / l_sum;
      const bool row_ok = my_row < my_rows;
      const int64_t row = int64_t(span.q0) + my_first + my_row;
      if (p.splits > 1) {
        const int64_t at = (int64_t(split) * p.total_q + row) * p.hq + my_head;
        if (my_tiles > 0) {
#pragma unroll 1
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(col_o + c * 32, o);
            tmem_ld_wait();
            if (row_ok) {
#pragma unroll
              for (int g = 0; g < 8; ++g)
                if (c * 32 + g * 4 < p.dim)
                  *reinterpret_cast<float4*>(p.part_out + at * p.dim + c * 32 + g * 4) =
                      make_float4(__uint_as_float(o[g * 4]) * inv, __uint_as_float(o[g * 4 + 1]) * inv,
                                  __uint_as_float(o[g * 4 + 2]) * inv, __uint_as_float(o[g * 4 + 3]) * inv);
            }
          }
        }
        if (row_ok) p.part_lse[at] = l_sum == 0.f ? -INFINITY : m_ref + log2f(l_sum);
      } else {
        // Through the tile's own Q rows in shared memory (every product that read them is complete), so
        // that a store writes whole rows: one row a thread would touch 32 lines an instruction.
        uint8_t* stage = sQ + t * TILE_BYTES + quarter * 32 * DP * 2;
        constexpr int WORDS = DP / 8;  // 16-byte words of a row, permuted against bank conflicts
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          if (my_tiles > 0) {
            tmem_ld_32x32(col_o + c * 32, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint4 v;
            v.x = pack16<FP16>(__uint_as_float(o[g * 8 + 0]) * inv, __uint_as_float(o[g * 8 + 1]) * inv);
            v.y = pack16<FP16>(__uint_as_float(o[g * 8 + 2]) * inv, __uint_as_float(o[g * 8 + 3]) * inv);
            v.z = pack16<FP16>(__uint_as_float(o[g * 8 + 4]) * inv, __uint_as_float(o[g * 8 + 5]) * inv);
            v.w = pack16<FP16>(__uint_as_float(o[g * 8 + 6]) * inv, __uint_as_float(o[g * 8 + 7]) * inv);
            *reinterpret_cast<uint4*>(stage + (lane * WORDS + ((c * 4 + g) ^ (lane & 7))) * 16) = v;
          }
        }
        __syncwarp();
        uint16_t* dst = static_cast<uint16_t*>(p.out) + ((row - lane) * p.hq + my_head) * p.dim;
        const int words = p.dim / 8, live = my_rows - quarter * 32;
#pragma unroll 4
        for (int i = lane; i < 32 * WORDS; i += 32) {
          const int r = i / WORDS, w = i % WORDS;
          if (r < live && w < words)
            *reinterpret_cast<uint4*>(dst + int64_t(r) * p.hq * p.dim + w * 8) =
                *reinterpret_cast<const uint4*>(stage + (r * WORDS + (w ^ (r & 7))) * 16);
        }
        if (row_ok && p.lse)
          p.lse[int64_t(my_head) * p.total_q + row] =
              l_sum == 0.f ? -INFINITY : (m_ref + log2f(l_sum)) * 0.6931471805599453f;
      }
    }
    // Rows behind the last sequence: zero (the merge does it for split launches).
    if (span.unit_in_sequence == -2 && p.splits == 1) {
      const int heads = p.paired ? 2 : 1;
      const int words = heads * p.dim / 8;  // 16-byte words of this CTA's heads in a row
      for (int i = int(threadIdx.x); i < span.rows * words; i += 256) {
        uint16_t* dst = static_cast<uint16_t*>(p.out) +
                        ((int64_t(span.q0) + i / words) * p.hq + head[0]) * p.dim + (i % words) * 8;
        *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins the key ranges of a split launch: out = sum_s w_s o_s, w_s = 2^(lse_s - max) / sum, in split
// order.  One warp per (row, head); lanes hold four elements each.
template <bool FP16>
__global__ void __launch_bounds__(256) packed_join_kernel(const float* __restrict__ part_out,
                                                          const float* __restrict__ part_lse, uint16_t* __restrict__ out,
                                                          float* __restrict__ lse, const int* __restrict__ q_offsets,
                                                          int sequences, int64_t total_q, int hq, int dim, int splits) {
  const int64_t unit = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (unit >= total_q * hq) return;
  const int lane = threadIdx.x & 31;
  const int64_t row = unit / hq;
  const int head = int(unit % hq);
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  float top = -INFINITY, weight = 0.f;
  if (row < q_offsets[sequences]) {
    for (int s = 0; s < splits; ++s) top = fmaxf(top, part_lse[(s * total_q + row) * hq + head]);
    for (int s = 0; s < splits; ++s) {
      const int64_t at = (s * total_q + row) * hq + head;
      const float l = part_lse[at];
      if (l == -INFINITY) continue;  // that range held no visible key
      const float w = exp2f(l - top);
      weight += w;
      if (lane * 4 < dim) {
        const float4 o = *reinterpret_cast<const float4*>(part_out + at * dim + lane * 4);
        sum.x += w * o.x; sum.y += w * o.y; sum.z += w * o.z; sum.w += w * o.w;
      }
    }
  }
  const float inv = weight == 0.f ? 0.f : 1.f / weight;
  if (lane * 4 < dim) {
    uint2 v;
    v.x = pack16<FP16>(sum.x * inv, sum.y * inv);
    v.y = pack16<FP16>(sum.z * inv, sum.w * inv);
    *reinterpret_cast<uint2*>(out + (row * hq + head) * dim + lane * 4) = v;
  }
  if (lse && lane == 0)
    lse[head * total_q + row] = weight == 0.f ? -INFINITY : (top + log2f(weight)) * 0.6931471805599453f;
}

template <int DP, bool FP16>
cudaError_t launch_tiles(const PackedArgs& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                         cudaStream_t stream) {
  const cudaError_t e = cudaFuncSetAttribute(packed_tiles_kernel<DP, FP16>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, fwd_smem<DP>());
  if (e != cudaSuccess) return e;
  FwdParams p{};
  p.q_offsets = a.q_offsets; p.k_offsets = a.k_offsets; p.k_lengths = a.k_lengths;
  p.sequences = a.sequences;
  p.total_q = a.total_q; p.total_k = a.total_k;
  p.out = a.out; p.lse = a.lse; p.part_out = a.part_out; p.part_lse = a.part_lse;
  p.hq = a.hq; p.dim = a.dim; p.group = a.hq / a.hkv; p.splits = a.splits;
  p.paired = p.group % 2 == 0;
  p.head_units = p.paired ? a.hq / 2 : a.hq;
  p.scale_log2 = a.scale * LOG2E;
  p.status = a.status;
  const int step = p.paired ? ROWS : 2 * ROWS;
  const int64_t grid = (a.total_q / step + a.sequences + 1) * p.head_units * p.splits;
  if (grid > 2147483647ll) {
    set_error_detail("packed_attention: too many tiles for one launch");
    return cudaErrorInvalidValue;
  }
  packed_tiles_kernel<DP, FP16><<<unsigned(grid), FWD_THREADS, fwd_smem<DP>(), stream>>>(tq, tk, tv, p);
  if (a.splits > 1) {
    const int64_t blocks = (a.total_q * a.hq + 7) / 8;
    packed_join_kernel<FP16><<<unsigned(blocks), 256, 0, stream>>>(
        a.part_out, a.part_lse, static_cast<uint16_t*>(a.out), a.lse, a.q_offsets, a.sequences, a.total_q, a.hq,
        a.dim, a.splits);
  }
  return cudaGetLastError();
}

}  // namespace

// A [rows, heads, dim] tensor in boxes of 64 elements x 1 head x 128 rows; elements behind dim read as zero.
bool make_packed_map(CUtensorMap* map, const void* base, int dim, int heads, int64_t rows, int64_t head_stride,
                     int64_t row_stride) {
  const uint64_t dims[3] = {uint64_t(dim), uint64_t(heads), uint64_t(rows)};
  const uint64_t strides[2] = {uint64_t(head_stride) * 2, uint64_t(row_stride) * 2};
  const uint32_t box[3] = {64, 1, 128};
  return encode_tensor_map_16bit(map, base, 3, dims, strides, box);
}

cudaError_t packed_attention_tiles(const PackedArgs& a, cudaStream_t stream) {
  CUtensorMap tq, tk, tv;
  if (!make_packed_map(&tq, a.q, a.dim, a.hq, a.total_q, a.q_head, a.q_row) ||
      !make_packed_map(&tk, a.k, a.dim, a.hkv, a.total_k, a.k_head, a.k_row) ||
      !make_packed_map(&tv, a.v, a.dim, a.hkv, a.total_k, a.v_head, a.v_row))
    return cudaErrorInvalidValue;
  if (a.dim <= 64)
    return a.fp16 ? launch_tiles<64, true>(a, tq, tk, tv, stream) : launch_tiles<64, false>(a, tq, tk, tv, stream);
  return a.fp16 ? launch_tiles<128, true>(a, tq, tk, tv, stream) : launch_tiles<128, false>(a, tq, tk, tv, stream);
}

}  // namespace agb
