// Causal attention over packed sequences, forward, on tcgen05 (bf16 or fp16, heads of up to 128).
//
//   s = scale q k^T over the visible keys (j <= i + keys - rows), p = softmax(s), out = p v
//
// A CTA works through items (piece of a sequence's queries, two score tiles, key range), which come in the
// order of falling length: it is launched for one and takes over further ones that have not started yet
// (one CTA fits an SM).  The rows of a tile are (query row, head) pairs of up to 16 heads that share a
// key head; the two tiles of an item are neighbours and read the same K and V tiles.  (With a tile of
// 128 rows of one head, sixteen prompts of 14 to 514 rows had a third more tiles.)
//   warps 0-3  softmax of tile 0: one query row per thread; then its output
//   warps 4-7  softmax of tile 1
//   warp 8     TMA producer (K and V through rings of two stages, which run on from item to item)
//   warp 9     MMA issuer: S_t = Q_t K^T, O_t += P_t V with P_t read from TMEM (one elected thread in a
//              branch of its own: a product then takes the pipe's 64 cycles, against 91 to 105 where
//              the whole warp runs the loop and elects a lane for every instruction)
//   warp 10    finds the items, up to two ahead
//   warp 11    clears the V rows behind the last key, so that whatever lies there (another sequence,
//              NaN) never meets a product
// The third warpgroup hands registers to the other two.  While one tile is in its softmax the tensor
// core works for the other, and while an item's outputs are written the next one's first scores are
// computed; with a CTA for every item its start (finding the piece, first loads) and end cost 7 us,
// as much as four key tiles.  The running maximum is only followed when it grows by more than 2^8:
// until then the scores are taken relative to the old one, which leaves the quotient unchanged.
// Sums, maxima and O are FP32; P is rounded to the tensors' type, as an operand of the tensor core has
// to be.
//
// What bounds it: 2048 cycles of products for a pair of 128 x 128 tiles against about 1600 of one
// tile's softmax, which has to lie between two of its products (2900 cycles measured).  With 32 query and 8
// key heads of 128: 435 us for a prompt of 8192 (1.26 PFLOP/s, tensor pipe active 63 % of the cycles), 1654 us
// for one of 16384 (1.33 PFLOP/s; 1880 to 1930 in calls without a pause, at the clocks that the power limit leaves).
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
constexpr float LOG2E = 1.4426950408889634f;
constexpr int STAGE_BYTES = 32 * 128;  // a warp's part of the output on its way: 32 rows x 128 bytes

template <int DP>
constexpr int fwd_smem() {
  // Q_0, Q_1, K ring, V ring, output stage.  Never less than half of an SM's shared memory: two CTAs do
  // not fit in its tensor memory, and the second would wait for the first in its allocation.
  const int bytes = (2 + 2 * KV_STAGES) * (DP / 64) * HALF_BYTES + 8 * STAGE_BYTES + 1024 + 1024;
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
  int shift;        // heads folded into a tile's rows: 1 << shift
  int head_units;   // items side by side for one piece: hq >> shift
  float scale_log2;
  int* status;
};

// What the roles need of an item.  Per tile: first query row within the sequence, query rows, key tiles
// (from the range's first on).
enum : int { ITEM_END = 0, ITEM_TILES = 1, ITEM_UNCOVERED = 2 };
struct Item {
  int kind, split;
  int first[2], rows[2], tiles[2];
  int head0, kv_head, q0, k0, query_rows, keys;
  int lo, n;        // range of key tiles
  int last_valid;   // keys that exist in the range's last tile (128 or more: all)
};
constexpr int ITEM_READERS = 11;  // eight softmax warps, producer, issuer, clearing warp

__device__ inline Item make_item(const PackedSpan& span, const FwdParams& p, int head_unit, int split) {
  Item item{};
  const int step = ROWS >> p.shift;  // query rows of a tile
  item.kind = span.unit_in_sequence == -2 ? ITEM_UNCOVERED : ITEM_TILES;
  item.split = split;
  item.q0 = span.q0;
  item.k0 = span.k0;
  item.query_rows = span.rows;
  item.keys = span.keys;
  item.head0 = head_unit << p.shift;
  item.kv_head = item.head0 / p.group;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    item.first[t] = (2 * span.unit_in_sequence + t) * step;
    item.rows[t] = item.kind == ITEM_TILES ? max(0, min(step, span.rows - item.first[t])) : 0;
    const int seen = min(span.keys, span.keys - span.rows + item.first[t] + item.rows[t]);  // keys of the last row
    item.tiles[t] = item.rows[t] == 0 || seen <= 0 ? 0 : (seen + ROWS - 1) / ROWS;
  }
  const int most = max(item.tiles[0], item.tiles[1]);
  const int per = (most + p.splits - 1) / p.splits;
  item.lo = min(most, split * per);
  const int hi = min(most, item.lo + per);
  item.n = hi - item.lo;
#pragma unroll
  for (int t = 0; t < 2; ++t) item.tiles[t] = max(0, min(hi, item.tiles[t]) - item.lo);
  item.last_valid = span.keys - (hi - 1) * ROWS;
  return item;
}

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
  uint8_t* sOut = sV + KV_STAGES * TILE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sOut + 8 * STAGE_BYTES);
  uint64_t* q_full = bars;         // 1
  uint64_t* q_empty = bars + 1;    // last scores of an item complete
  uint64_t* k_full = bars + 2;     // [2]
  uint64_t* k_empty = bars + 4;    // [2]
  uint64_t* v_full = bars + 6;     // [2]
  uint64_t* v_empty = bars + 8;    // [2]
  uint64_t* s_full = bars + 10;    // [2 tiles] scores complete
  uint64_t* p_ready = bars + 12;   // [2 tiles][2 halves of the keys] probabilities in TMEM (count 4)
  uint64_t* o_done = bars + 16;    // [2 tiles] last product complete
  uint64_t* v_ragged = bars + 18;  // an item's ragged last V tile is on its way
  uint64_t* v_clean = bars + 19;   // and its rows behind the last key are cleared
  uint64_t* item_full = bars + 20; // [2]
  uint64_t* item_empty = bars + 22;  // [2] (count ITEM_READERS)
  uint64_t* answer_full = bars + 24;
  uint64_t* item_loaded = bars + 25; // every load of an item is issued
  uint64_t* answer = bars + 26;      // 16 bytes: the next block taken over
  Item* items = reinterpret_cast<Item*>(bars + 28);  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const WaitGuard guard{abort_flag, p.status};

  if (warp == 1 && lane == 0) {
    *abort_flag = 0;
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[2 * i], 4);
      mbar_init(&p_ready[2 * i + 1], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], ITEM_READERS);
    }
    mbar_init(v_ragged, 1);
    mbar_init(v_clean, 1);
    mbar_init(answer_full, 1);
    mbar_init(item_loaded, 1);
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

  // The i-th item in its slot of the ring; a reader frees the slot once it has what it needs.
  auto item_wait = [&](int i, int code) { return mbar_wait(&item_full[i & 1], (i >> 1) & 1, guard, code); };
  auto item_free = [&](int i) { mbar_arrive(&item_empty[i & 1]); };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    if (warp == 8) {
      // ------------------------------------------------------------------ TMA producer
      if (lane == 0) {
        bool ok = true;
        int loads = 0;  // key tiles so far
        for (int i = 0, used = 0; ok; ++i) {
          if (!item_wait(i, kTimeoutProducer)) { ok = false; break; }
          const Item& it = items[i & 1];
          const int kind = it.kind, n = it.n, kv_head = it.kv_head, q0 = it.q0, row0 = it.k0 + it.lo * ROWS;
          const int head0 = it.head0, first[2] = {it.first[0], it.first[1]};
          const bool there[2] = {it.tiles[0] > 0, it.tiles[1] > 0}, ragged = it.last_valid < ROWS;
          item_free(i);
          if (kind == ITEM_END) break;
          if (n == 0) {
            mbar_arrive(item_loaded);
            continue;
          }
          if (!mbar_wait(q_empty, (used & 1) ^ 1, guard, kTimeoutProducer)) { ok = false; break; }
          ++used;
          mbar_expect_tx(q_full, (there[0] + there[1]) * TILE_BYTES);
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (there[t])
              for (int a = 0; a < ATOMS; ++a)
                tma_load_3d(sQ + t * TILE_BYTES + a * HALF_BYTES, &tm_q, q_full, a * 64, head0, q0 + first[t]);
          for (int j = 0; j < n && ok; ++j, ++loads) {
            const int st = loads % KV_STAGES;
            const uint32_t ph = ((loads / KV_STAGES) & 1) ^ 1;
            const int row = row0 + j * ROWS;
            if (!mbar_wait(&k_empty[st], ph, guard, kTimeoutProducer)) { ok = false; break; }
            mbar_expect_tx(&k_full[st], TILE_BYTES);
            for (int a = 0; a < ATOMS; ++a)
              tma_load_3d(sK + st * TILE_BYTES + a * HALF_BYTES, &tm_k, &k_full[st], a * 64, kv_head, row);
            if (!mbar_wait(&v_empty[st], ph, guard, kTimeoutProducer)) { ok = false; break; }
            mbar_expect_tx(&v_full[st], TILE_BYTES);
            for (int a = 0; a < ATOMS; ++a)
              tma_load_3d(sV + st * TILE_BYTES + a * HALF_BYTES, &tm_v, &v_full[st], a * 64, kv_head, row);
            if (ragged && j + 1 == n) mbar_arrive(v_ragged);
          }
          mbar_arrive(item_loaded);
        }
        if (!ok || *abort_flag) {
          // give in-flight copies time to land before shared memory is released
          const uint64_t start = global_timer_ns();
          while (global_timer_ns() - start < 100000ull) {}
        }
      }
    } else if (warp == 9) {
      // -------------------------------------------------------------------- MMA issuer
      if (elect_one()) {
        constexpr uint32_t idesc_s = make_idesc_16(FP16, ROWS, ROWS, 0, 0);  // both K-major over d
        constexpr uint32_t idesc_o = make_idesc_16(FP16, ROWS, DP, 0, 1);    // P from TMEM, V MN-major
        auto scores = [&](int t, int st) {
          const uint32_t q_addr = smem_u32(sQ + t * TILE_BYTES);
          const uint32_t k_addr = smem_u32(sK + st * TILE_BYTES);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            const uint32_t off = (kk >> 2) * HALF_BYTES + (kk & 3) * 32;
            tc_mma_ss(tmem_base + COL_S + t * 128, make_smem_desc(q_addr + off, 16, 1024),
                      make_smem_desc(k_addr + off, 16, 1024), idesc_s, kk != 0);
          }
          tc_commit(&s_full[t]);
        };
        bool ok = true;
        int loads = 0;             // key tiles of earlier items
        uint32_t done[2] = {0, 0}; // tiles' score blocks of earlier items
        for (int i = 0, used = 0, cleaned = 0; ok; ++i) {
          if (!item_wait(i, kTimeoutMma)) break;
          const Item& it = items[i & 1];
          const int kind = it.kind, n = it.n;
          const int tiles[2] = {it.tiles[0], it.tiles[1]};
          const bool ragged = it.last_valid < ROWS;
          item_free(i);
          if (kind == ITEM_END) break;
          if (n == 0) continue;
          ok = mbar_wait(q_full, used & 1, guard, kTimeoutMma) &&
               mbar_wait(&k_full[loads % KV_STAGES], (loads / KV_STAGES) & 1, guard, kTimeoutMma);
          if (!ok) break;
          ++used;
          tc_fence_after_sync();
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (tiles[t] > 0) scores(t, loads % KV_STAGES);
          tc_commit(&k_empty[loads % KV_STAGES]);
          if (n == 1) tc_commit(q_empty);
          for (int j = 0; j < n && ok; ++j) {
            const int st = (loads + j) % KV_STAGES, next = (loads + j + 1) % KV_STAGES;
            const bool more = j + 1 < n;
            if (!mbar_wait(&v_full[st], ((loads + j) / KV_STAGES) & 1, guard, kTimeoutMma)) { ok = false; break; }
            if (!more && ragged && !mbar_wait(v_clean, cleaned++ & 1, guard, kTimeoutMma)) { ok = false; break; }
            if (more && !mbar_wait(&k_full[next], ((loads + j + 1) / KV_STAGES) & 1, guard, kTimeoutMma)) { ok = false; break; }
            const uint32_t v_addr = smem_u32(sV + st * TILE_BYTES);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (!ok || j >= tiles[t]) continue;
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                if (!ok || !mbar_wait(&p_ready[2 * t + c], (done[t] + j) & 1, guard, kTimeoutMma)) { ok = false; break; }
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
              if (j + 1 < tiles[t]) scores(t, next);
              else tc_commit(&o_done[t]);
            }
            if (!ok) break;
            tc_commit(&v_empty[st]);
            if (more) tc_commit(&k_empty[next]);
            if (j + 2 == n) tc_commit(q_empty);
          }
          loads += n;
          done[0] += tiles[0];
          done[1] += tiles[1];
        }
      }
      __syncwarp();
    } else if (warp == 10) {
      // ------------------------------------------------------------------------ items
      // The next block is taken over once the last loads of the present item are issued, two key tiles
      // before its end: earlier, and CTAs with long items would take blocks from those that are free.
      uint32_t found = 0, asked = 0;
      for (int64_t unit = blockIdx.x;;) {
        const bool last = unit < 0;
        Item item{};
        bool work = last;
        if (!last) {
          const int side = p.head_units * p.splits;  // blocks of one piece, splits fastest
          const int piece = divide(int(unit), side), rest = int(unit) - piece * side;
          const int head_unit = divide(rest, p.splits), split = rest - head_unit * p.splits;
          const PackedSpan span = find_piece(piece, 2 * ROWS >> p.shift, false, p.q_offsets, p.k_offsets,
                                             p.k_lengths, p.sequences, p.total_q, p.total_k,
                                             head_unit == 0 && split == 0 ? p.status : nullptr);
          work = !(span.unit_in_sequence == -1 || (span.unit_in_sequence == -2 && span.rows == 0));
          if (work) item = make_item(span, p, head_unit, split);
        }
        if (work) {
          if (!mbar_wait_w(&item_empty[found & 1], ((found >> 1) & 1) ^ 1, guard, kTimeoutProducer)) break;
          if (lane == 0) {
            items[found & 1] = item;
            mbar_arrive(&item_full[found & 1]);
          }
          __syncwarp();
          if (last || !mbar_wait_w(item_loaded, found & 1, guard, kTimeoutProducer)) break;
          ++found;
        }
        if (lane == 0) steal(smem_u32(answer), answer_full);
        if (!mbar_wait_w(answer_full, asked++ & 1, guard, kTimeoutProducer)) break;
        unit = stolen(smem_u32(answer));
        __syncwarp();
      }
    } else {
      // ------------------------------------------------------------- rows behind the keys
      int loads = 0;
      for (int i = 0, cleaned = 0;; ++i) {
        if (!mbar_wait_w(&item_full[i & 1], (i >> 1) & 1, guard, kTimeoutProducer)) break;
        const int kind = items[i & 1].kind, n = items[i & 1].n, valid = items[i & 1].last_valid;
        __syncwarp();
        if (lane == 0) item_free(i);
        if (kind == ITEM_END) break;
        if (n == 0) continue;
        loads += n;
        if (valid >= ROWS) continue;
        // Once that load is issued its stage's barrier is in the phase of this tile, and stays there
        // until the rows are cleared: its parity then says whether the tile has arrived.
        const int st = (loads - 1) % KV_STAGES;
        if (!mbar_wait_w(v_ragged, cleaned++ & 1, guard, kTimeoutProducer) ||
            !mbar_wait_w(&v_full[st], ((loads - 1) / KV_STAGES) & 1, guard, kTimeoutProducer))
          break;
        clear_rows<ATOMS>(smem_u32(sV + st * TILE_BYTES), valid, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_clean);
      }
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
    const uint32_t stage = smem_u32(sOut + warp * STAGE_BYTES);
    bool ok = true;
    uint32_t done = 0, outs = 0;                 // score blocks and outputs of earlier items
    for (int i = 0; ok; ++i) {
      if (!item_wait(i, kTimeoutSoftmax)) break;
      const Item& it = items[i & 1];
      const int kind = it.kind, my_tiles = it.tiles[t], my_rows = it.rows[t], head0 = it.head0, split = it.split;
      const int q_row = it.q0 + it.first[t];     // first query row of the tile
      // keys that this row, and the warp's first and last row, see, from the first key of the range on
      const int it_keys = it.keys - it.lo * ROWS;
      const int before = it_keys - it.query_rows + it.first[t] + 1;
      const int seen = min(it_keys, before + (my_row >> p.shift));
      const int seen_warp = min(it_keys, before + (quarter * 32 >> p.shift));
      const int seen_most = min(it_keys, before + (quarter * 32 + 31 >> p.shift));
      const int uncovered0 = it.q0, uncovered = it.query_rows;
      __syncwarp();
      if (lane == 0) item_free(i);
      if (kind == ITEM_END) break;
      if (kind == ITEM_UNCOVERED) {  // zeros (the join writes them for split launches)
        const int words = (p.dim << p.shift) / 8;  // of the item's heads in a row
        if (p.splits == 1)
          for (int w = t * ROWS + my_row; w < uncovered * words; w += 2 * ROWS)
            store16(static_cast<uint16_t*>(p.out) + ((int64_t(uncovered0) + w / words) * p.hq + head0) * p.dim +
                        (w % words) * 8,
                    make_uint4(0, 0, 0, 0));
        continue;
      }
      float m_ref = -INFINITY;                   // reference maximum (log2 domain)
      float l_sum = 0.f;
      for (int j = 0; j < my_tiles && ok; ++j) {
        if (!mbar_wait(&s_full[t], (done + j) & 1, guard, kTimeoutSoftmax)) { ok = false; break; }
        tc_fence_after_sync();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(col_s + c * 32, s[c]);
        tmem_ld_wait();
        // Only the diagonal and the ragged last tile mask.  There, of the 32 keys of chunk c, every row of
        // the warp sees all (32 c + 32 <= sure), or none (32 c >= most), or the rows differ; all these
        // tests are uniform over the warp.
        const int sure = seen_warp - j * ROWS;
        const bool masked = sure < ROWS;
        if (masked) {
          const int valid = seen - j * ROWS;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c * 32 + 32 <= sure) continue;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (c * 32 + k >= valid) s[c][k] = 0xff800000u;  // -inf
          }
        }
        float m4[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          m4[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
          for (int k = 2; k < 32; k += 2) m4[c] = fmax3(m4[c], __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
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
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
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
        float2 sums[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[k] = make_float2(0.f, 0.f);
        // One pair of unmasked scores in four takes the exponential of the FMA pipe: a tile's share of
        // the special-function unit (16 a cycle) is as long as its products.  1661 us against 1690
        // without, 1708 for one in eight and 1747 for three in eight, at 16384 tokens.
        auto chunk = [&](const uint32_t (&x32)[32], uint32_t* to, auto all) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float2 x = ffma2(make_float2(__uint_as_float(x32[2 * k]), __uint_as_float(x32[2 * k + 1])), scale2, shift2);
            const float2 e = decltype(all)::value && k % 4 == 3 ? exp2_fma(x) : make_float2(exp2f(x.x), exp2f(x.y));
            sums[k & 3] = fadd2(sums[k & 3], e);
            to[k] = pack16<FP16>(e.x, e.y);
          }
        };
        auto hand_over = [&](const uint32_t (&packed)[32], int c) {
          tmem_st_32x32(col_s + c * 32, packed);  // over the scores, which are in registers
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[2 * t + c]);
        };
        if (!masked) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t packed[32];
            chunk(s[2 * c], packed, std::true_type{});
            chunk(s[2 * c + 1], packed + 16, std::true_type{});
            hand_over(packed, c);
          }
        } else {
          const int most = seen_most - j * ROWS;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t packed[32];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if ((2 * c + h) * 32 + 32 <= sure) chunk(s[2 * c + h], packed + 16 * h, std::true_type{});
              else if ((2 * c + h) * 32 < most) chunk(s[2 * c + h], packed + 16 * h, std::false_type{});
              else
#pragma unroll
                for (int k = 0; k < 16; ++k) packed[16 * h + k] = 0;
            }
            hand_over(packed, c);
          }
        }
        const float2 sum2 = fadd2(fadd2(sums[0], sums[1]), fadd2(sums[2], sums[3]));
        l_sum += sum2.x + sum2.y;
      }
      done += my_tiles;
      // ---------------------------------------------------------------------- output
      if (ok && my_tiles > 0) ok = mbar_wait(&o_done[t], outs++ & 1, guard, kTimeoutEpilogue);
      if (!ok) break;
      tc_fence_after_sync();
      const float inv = l_sum == 0.f ? 0.f : 1.f / l_sum;
      const bool partial = p.splits > 1;
      const int live = min(32, (my_rows << p.shift) - quarter * 32);    // rows of this warp
      const int64_t row = int64_t(q_row) + (quarter * 32 >> p.shift);   // the query row of its first
      const int head = head0 + (quarter * 32 & ((1 << p.shift) - 1));   // and the head (folds are at most 32)
      const int64_t at = ((partial ? int64_t(split) * p.total_q : 0) + row) * p.hq + head;
      if (live > 0 && !(partial && my_tiles == 0)) {
        // 128 bytes of every row at a time: 64 elements, or 32 of a partial result
#pragma unroll 1
        for (int c = 0; c < DP / 64; ++c) {
          uint32_t o[2][32];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (my_tiles > 0) tmem_ld_32x32(col_o + c * 64 + h * 32, o[h]);
            else
#pragma unroll
              for (int k = 0; k < 32; ++k) o[h][k] = 0;
          }
          tmem_ld_wait();
          if (partial) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int g = 0; g < 8; ++g)
                put16(stage_word(stage, lane, g),
                      make_uint4(__float_as_uint(__uint_as_float(o[h][g * 4 + 0]) * inv),
                                 __float_as_uint(__uint_as_float(o[h][g * 4 + 1]) * inv),
                                 __float_as_uint(__uint_as_float(o[h][g * 4 + 2]) * inv),
                                 __float_as_uint(__uint_as_float(o[h][g * 4 + 3]) * inv)));
              flush_rows(stage, reinterpret_cast<uint8_t*>(p.part_out + at * p.dim + c * 64 + h * 32),
                         p.hq * p.dim * 4, p.dim * 4, p.shift, (p.dim - c * 64 - h * 32) * 4, live, lane);
            }
          } else {
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              const uint32_t* x = &o[g >> 2][(g & 3) * 8];
              uint4 v;
              v.x = pack16<FP16>(__uint_as_float(x[0]) * inv, __uint_as_float(x[1]) * inv);
              v.y = pack16<FP16>(__uint_as_float(x[2]) * inv, __uint_as_float(x[3]) * inv);
              v.z = pack16<FP16>(__uint_as_float(x[4]) * inv, __uint_as_float(x[5]) * inv);
              v.w = pack16<FP16>(__uint_as_float(x[6]) * inv, __uint_as_float(x[7]) * inv);
              put16(stage_word(stage, lane, g), v);
            }
            flush_rows(stage, reinterpret_cast<uint8_t*>(static_cast<uint16_t*>(p.out) + at * p.dim + c * 64),
                       p.hq * p.dim * 2, p.dim * 2, p.shift, (p.dim - c * 64) * 2, live, lane);
          }
        }
      }
      if (lane < live) {
        const float log_sum = l_sum == 0.f ? -INFINITY : m_ref + log2f(l_sum);
        const int down = lane >> p.shift, across = lane & ((1 << p.shift) - 1);
        if (partial) p.part_lse[at + int64_t(down) * p.hq + across] = log_sum;
        else if (p.lse) p.lse[int64_t(head + across) * p.total_q + row + down] = log_sum * 0.6931471805599453f;
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
  const int head = int(unit - row * hq);
  const bool covered = row < q_offsets[sequences];
  after_previous_launch();
  const int64_t stride = total_q * hq;
  const float mine = covered && lane < splits ? part_lse[lane * stride + unit] : -INFINITY;  // splits <= 32
  float top = mine;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float share = mine == -INFINITY ? 0.f : exp2f(mine - top);  // 0: that range held no visible key
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  float weight = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float w = __shfl_sync(0xffffffffu, share, s);
    weight += w;
    if (w != 0.f && lane * 4 < dim) {
      const float4 o = *reinterpret_cast<const float4*>(part_out + (s * stride + unit) * dim + lane * 4);
      sum.x += w * o.x; sum.y += w * o.y; sum.z += w * o.z; sum.w += w * o.w;
    }
  }
  const float inv = weight == 0.f ? 0.f : 1.f / weight;
  if (lane * 4 < dim) {
    uint2 v;
    v.x = pack16<FP16>(sum.x * inv, sum.y * inv);
    v.y = pack16<FP16>(sum.z * inv, sum.w * inv);
    *reinterpret_cast<uint2*>(out + unit * dim + lane * 4) = v;
  }
  if (lse && lane == 0)
    lse[head * total_q + row] = weight == 0.f ? -INFINITY : (top + log2f(weight)) * 0.6931471805599453f;
}

template <int DP, bool FP16>
cudaError_t launch_tiles(const PackedArgs& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                         cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_shared_memory(packed_tiles_kernel<DP, FP16>, fwd_smem<DP>(), allowed);
  if (e != cudaSuccess) return e;
  FwdParams p{};
  p.q_offsets = a.q_offsets; p.k_offsets = a.k_offsets; p.k_lengths = a.k_lengths;
  p.sequences = a.sequences;
  p.total_q = a.total_q; p.total_k = a.total_k;
  p.out = a.out; p.lse = a.lse; p.part_out = a.part_out; p.part_lse = a.part_lse;
  p.hq = a.hq; p.dim = a.dim; p.group = a.hq / a.hkv; p.splits = a.splits;
  p.shift = fold_shift(p.group);
  p.head_units = a.hq >> p.shift;
  p.scale_log2 = a.scale * LOG2E;
  p.status = a.status;
  const int step = 2 * ROWS >> p.shift;
  const int64_t units = (a.total_q / step + a.sequences + 1) * p.head_units * p.splits;
  const int64_t blocks = (a.total_q * a.hq + 7) / 8;
  if (units > 2147483647ll || blocks > 2147483647ll) {
    set_error_detail("packed_attention: too many rows for one launch");
    return cudaErrorInvalidValue;
  }
  packed_tiles_kernel<DP, FP16><<<unsigned(units), FWD_THREADS, fwd_smem<DP>(), stream>>>(tq, tk, tv, p);
  const cudaError_t launched = cudaGetLastError();
  if (launched != cudaSuccess || a.splits == 1) return launched;
  return launch_behind(packed_join_kernel<FP16>, dim3(unsigned(blocks)), 256, 0, stream, a.part_out, a.part_lse,
                       static_cast<uint16_t*>(a.out), a.lse, a.q_offsets, a.sequences, a.total_q, a.hq, a.dim, a.splits);
}

}  // namespace

// A [rows, heads, dim] tensor in boxes of 64 elements x `fold` heads x 128 / fold rows; elements behind dim read
// as zero.
bool make_packed_map(CUtensorMap* map, const void* base, int dim, int heads, int64_t rows, int64_t head_stride,
                     int64_t row_stride, int fold) {
  const uint64_t dims[3] = {uint64_t(dim), uint64_t(heads), uint64_t(rows)};
  const uint64_t strides[2] = {uint64_t(head_stride) * 2, uint64_t(row_stride) * 2};
  const uint32_t box[3] = {64, uint32_t(fold), uint32_t(128 / fold)};
  return encode_tensor_map_16bit(map, base, 3, dims, strides, box);
}

cudaError_t packed_attention_tiles(const PackedArgs& a, cudaStream_t stream) {
  CUtensorMap tq, tk, tv;
  if (!make_packed_map(&tq, a.q, a.dim, a.hq, a.total_q, a.q_head, a.q_row, 1 << fold_shift(a.hq / a.hkv)) ||
      !make_packed_map(&tk, a.k, a.dim, a.hkv, a.total_k, a.k_head, a.k_row, 1) ||
      !make_packed_map(&tv, a.v, a.dim, a.hkv, a.total_k, a.v_head, a.v_row, 1))
    return cudaErrorInvalidValue;
  if (a.dim <= 64)
    return a.fp16 ? launch_tiles<64, true>(a, tq, tk, tv, stream) : launch_tiles<64, false>(a, tq, tk, tv, stream);
  return a.fp16 ? launch_tiles<128, true>(a, tq, tk, tv, stream) : launch_tiles<128, false>(a, tq, tk, tv, stream);
}

}  // namespace agb
