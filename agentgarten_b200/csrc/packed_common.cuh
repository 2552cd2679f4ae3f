// Shared pieces of the attention kernels over packed sequences.
//
// Work units.  Sequences of a packed tensor are cut into pieces of `step` rows.  Unit numbers are
// handed out without a prefix sum: the first unit of sequence s is offsets[s] / step + s, which
// leaves room for every sequence's ragged last piece, so a block finds its sequence by searching
// the offsets and units without a piece have nothing to do.  There are total / step + sequences + 1
// units; those behind the last sequence own the rows that no sequence covers.
#pragma once

#include "sm100.cuh"

#include <cuda_fp16.h>

#include <atomic>

namespace agb {

// 16-byte accesses of shared memory by its own addresses (through a pointer that was aligned by hand the
// compiler only sees generic memory: clearing a tile's rows took five times as long).
__device__ __forceinline__ void put16(uint32_t address, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 get16(uint32_t address) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ void store16(void* to, uint4 v) {
  asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};"
               ::"l"(__cvta_generic_to_global(to)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// The same address of another member of the cluster, and the barrier of all threads of a cluster.
__device__ __forceinline__ void put16_member(uint32_t address, int member, uint4 v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(address), "r"(member));
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};"
               ::"r"(remote), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Tiles of 128 rows are (query row, head) pairs: `fold` query heads that share a key head side by side,
// heads fastest, so that a short or ragged sequence fills them.  fold is a power of two, 1 << shift.
__host__ __device__ __forceinline__ int fold_shift(int group) {  // of the largest power of two in the group, up to 16
  int shift = 0;
  while (shift < 4 && (group >> shift) % 2 == 0) ++shift;
  return shift;
}

// 32 rows x 128 bytes of a warp from its stage in shared memory (4 KB; 16-byte word w of row r lies at word
// w ^ (r & 7)) to global memory: row r (of the first `live`) goes to dst + (r >> shift) * pitch + (r & (2^shift -
// 1)) * head_pitch bytes, of which `bytes` are left from there on.  Whole rows an instruction; stores of
// one row a thread would touch 32 lines each.
__device__ __forceinline__ uint32_t stage_word(uint32_t stage, int row, int word) {
  return stage + row * 128 + ((word ^ row) & 7) * 16;
}
__device__ __forceinline__ void flush_rows(uint32_t stage, uint8_t* dst, int pitch, int head_pitch, int shift, int bytes,
                                           int live, int lane) {
  __syncwarp();
  const int w = lane & 7, first = lane >> 3;
  uint4 v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = get16(stage_word(stage, k * 4 + first, w));
  if (w * 16 < bytes) {
    uint8_t* to = dst + w * 16;
    const int mask = (1 << shift) - 1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = k * 4 + first;
      if (r < live) store16(to + (r >> shift) * pitch + (r & mask) * head_pitch, v[k]);
    }
  }
  __syncwarp();
}

// Clears rows [from, 128) of a tile (ATOMS blocks of 128 rows x 128 bytes; a row is 128 bytes of each
// block whatever the swizzle, which permutes within the row); converged warp.
template <int ATOMS>
__device__ __forceinline__ void clear_rows(uint32_t tile, int from, int lane) {
#pragma unroll 4
  for (int i = from * 8 + lane; i < 128 * 8; i += 32)
#pragma unroll
    for (int a = 0; a < ATOMS; ++a) put16(tile + a * 16384 + i * 16, make_uint4(0, 0, 0, 0));
}

// Opts a kernel in to `bytes` of dynamic shared memory, once on every device (up to 64 of them are
// remembered; the call itself costs the host as much as half a launch).
template <typename Kernel>
cudaError_t allow_shared_memory(Kernel* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// A launch that may begin while the one before it still runs: its blocks take up what they can and wait
// (after_previous_launch) before they read what that launch writes.  Every thread waits, so the
// second launch never ends before the first.
// `allow_next_launch`: once every block of a launch has started, the next one's may fill the SMs that
// come free.
__device__ __forceinline__ void allow_next_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void after_previous_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_behind(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(unsigned(threads));
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

// Work of a block that has not started yet, taken over by a running one (cluster launch control): the
// hardware's own queue in place of a counter in memory.  `steal` asks, `stolen` reads the answer once
// `bar` has it (16 bytes): the number of the block taken over, or -1 when none is left (do not ask again).
__device__ __forceinline__ void steal(uint32_t answer, uint64_t* bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(answer), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ int64_t stolen(uint32_t answer) {
  uint32_t block = 0, taken = 0;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %1, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, _, _, _}, r;\n\t}"
      : "+r"(block), "=r"(taken) : "r"(answer) : "memory");
  // the answer is read before the next one may be written over it
  fence_proxy_async_smem();
  return taken ? int64_t(block) : -1;
}

// a / b of non-negative a and positive b: an estimate in 32-bit floating point, put right in integers (the
// compiler's own division takes a few hundred cycles before the first load of a block).
__device__ __forceinline__ int divide(int a, int b) {
  int q = int(__fdividef(float(a), float(b)));
  int r = a - q * b;
  while (r < 0) { --q; r += b; }
  while (r >= b) { ++q; r -= b; }
  return q;
}

struct PackedSpan {
  int unit_in_sequence;  // piece number within the sequence, or -1: none, or -2: rows behind the last sequence
  int sequence;
  int q0, rows;          // the sequence's query rows
  int k0, keys, room;    // its key rows, how many of them are keys, and how many belong to it
};

// Converged warp.  `by_keys`: units are pieces of the key rows, else of the query rows.  Every
// number that comes from the device lists is checked against the tensors before it is used.
__device__ inline PackedSpan find_unit(int unit, int step, bool by_keys, const int* __restrict__ q_offsets,
                                       const int* __restrict__ k_offsets, const int* __restrict__ k_lengths,
                                       int sequences, int64_t total_q, int64_t total_k, int* status) {
  const int lane = threadIdx.x & 31;
  const int* offsets = by_keys ? k_offsets : q_offsets;
  PackedSpan span{-1, 0, 0, 0, 0, 0, 0};
  // 32-way search for the last s in [0, sequences] whose first unit is <= unit
  int low = 0, count = sequences + 1;
  while (count > 0) {
    const int stride = (count + 31) / 32;
    const int s = low + lane * stride;
    const bool reached = lane * stride < count && offsets[s] / step + s <= unit;
    const unsigned votes = __ballot_sync(0xffffffffu, reached);
    if (votes == 0) break;
    const int last = 31 - __clz(votes);
    const int behind = count - last * stride;
    low += last * stride;
    count = stride == 1 ? 0 : (behind < stride ? behind : stride);
  }
  const int s = low;
  if (unit == 0 && lane == 0 && (q_offsets[0] != 0 || k_offsets[0] != 0) && status) atomicCAS(status, 0, kBadIndex);
  if (s >= sequences) {
    const int64_t end = offsets[sequences];
    const int64_t total = by_keys ? total_k : total_q;
    if (end < 0 || end > total) {
      if (lane == 0 && status) atomicCAS(status, 0, kBadIndex);
      return span;
    }
    span.unit_in_sequence = -2;
    span.sequence = sequences;
    const int64_t first = end + int64_t(unit - (end / step + sequences)) * step;
    span.q0 = span.k0 = int(first < total ? first : total);
    span.rows = span.keys = span.room = int(first < total ? (total - first < step ? total - first : step) : 0);
    return span;
  }
  const int q0 = q_offsets[s], q1 = q_offsets[s + 1], k0 = k_offsets[s], k1 = k_offsets[s + 1];
  const int keys = k_lengths ? k_lengths[s] : k1 - k0;
  if (q0 < 0 || q1 < q0 || q1 > total_q || k0 < 0 || k1 < k0 || k1 > total_k || keys < 0 || keys > k1 - k0) {
    if (lane == 0 && status) atomicCAS(status, 0, kBadIndex);
    return span;
  }
  const int piece = unit - (offsets[s] / step + s);
  const int extent = by_keys ? k1 - k0 : q1 - q0;
  // piece 0 exists for an empty sequence too
  if (piece < 0 || (piece > 0 && int64_t(piece) * step >= extent)) return span;
  span.unit_in_sequence = piece;
  span.sequence = s;
  span.q0 = q0;
  span.rows = q1 - q0;
  span.k0 = k0;
  span.keys = keys;
  span.room = k1 - k0;
  return span;
}

// The same for launches whose units differ in length: piece `rank` in the order of falling length, so
// that no long piece starts last.  Per sequence the pieces' lengths follow from three numbers: `count`
// pieces, the longest of `most`, each next one shorter by one, none counted longer than `cap`.  The
// rank is found by a binary search over the length, each step one sum over the sequences, which two
// registers a lane hold: up to MAX_RANKED sequences.  (With more there are enough pieces to even
// out by themselves.)  Ranks behind the last piece own the rows that no sequence covers.
constexpr int MAX_RANKED = 64;

__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

template <int R>  // sequences <= 32 R
__device__ inline PackedSpan find_ranked(int rank, int step, bool by_keys, const int* __restrict__ q_offsets,
                                         const int* __restrict__ k_offsets, const int* __restrict__ k_lengths,
                                         int sequences, int64_t total_q, int64_t total_k, int* status) {
  const int lane = threadIdx.x & 31;
  int q0[R], q1[R], k0[R], k1[R], keys[R], count[R], most[R], cap[R];
  bool bad = false;
  const int end = (by_keys ? k_offsets : q_offsets)[sequences];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int s = lane + 32 * i;
    const bool there = s < sequences;
    const int at = there ? s : 0;
    q0[i] = q_offsets[at];
    q1[i] = q_offsets[at + (there ? 1 : 0)];
    k0[i] = k_offsets[at];
    k1[i] = k_offsets[at + (there ? 1 : 0)];
    keys[i] = there && k_lengths ? k_lengths[at] : k1[i] - k0[i];
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int rows = q1[i] - q0[i];
    const bool fits = q0[i] >= 0 && rows >= 0 && q1[i] <= total_q && k0[i] >= 0 && k1[i] >= k0[i] &&
                      k1[i] <= total_k && keys[i] >= 0 && keys[i] <= k1[i] - k0[i];
    const bool there = lane + 32 * i < sequences;
    bad = bad || !fits || (there && lane + i == 0 && (q0[0] != 0 || k0[0] != 0));
    if (by_keys) {  // piece p is seen by the rows behind it: all of them while it lies before the first one
      count[i] = there && fits ? (k1[i] - k0[i] + step - 1) / step : 0;
      most[i] = ((keys[i] > rows ? keys[i] : rows) + step - 1) / step;
      cap[i] = (rows + step - 1) / step;
    } else {        // the last piece sees all keys, each earlier one a tile less
      count[i] = there && fits ? (rows + step - 1) / step : 0;
      most[i] = cap[i] = (keys[i] + step - 1) / step;
    }
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0 && status) atomicCAS(status, 0, kBadIndex);
  PackedSpan span{-1, 0, 0, 0, 0, 0, 0};
  auto sum_of = [&](auto of_register) {
    int sum = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) sum += of_register(i);
    return warp_sum(sum);
  };
  const int all = sum_of([&](int i) { return count[i]; });
  if (rank >= all) {
    const int64_t total = by_keys ? total_k : total_q;
    if (end < 0 || end > total) return span;
    const int64_t first = end + int64_t(rank - all) * step;
    span.unit_in_sequence = -2;
    span.sequence = sequences;
    span.q0 = span.k0 = int(first < total ? first : total);
    span.rows = span.keys = span.room = int(first < total ? (total - first < step ? total - first : step) : 0);
    return span;
  }
  // pieces of a lane's sequences that are at least `length` long
  auto longer = [&](int i, int length) {
    const int n = most[i] - length + 1;
    return length > cap[i] || n < 0 ? 0 : (n < count[i] ? n : count[i]);
  };
  if (sequences == 1) {
    const int piece = by_keys ? rank : count[0] - 1 - rank;
    span.unit_in_sequence = __shfl_sync(0xffffffffu, piece, 0);
    span.q0 = __shfl_sync(0xffffffffu, q0[0], 0);
    span.rows = __shfl_sync(0xffffffffu, q1[0], 0) - span.q0;
    span.k0 = __shfl_sync(0xffffffffu, k0[0], 0);
    span.room = __shfl_sync(0xffffffffu, k1[0], 0) - span.k0;
    span.keys = __shfl_sync(0xffffffffu, keys[0], 0);
    return span;
  }
  int low = 0x7fffffff, high = 0;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (count[i] > 0) {
      low = min(low, min(cap[i], most[i] - count[i] + 1));
      high = max(high, cap[i]);
    }
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high) + 1;  // nothing is this long
  while (high - low > 1) {  // the greatest length that more than `rank` pieces reach
    const int middle = low + (high - low) / 2;
    if (sum_of([&](int i) { return longer(i, middle); }) > rank) low = middle;
    else high = middle;
  }
  // the pieces of exactly this length, sequence by sequence
  int behind[R], here[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    behind[i] = longer(i, low + 1);
    here[i] = longer(i, low) - behind[i];
  }
  int index = rank - sum_of([&](int i) { return behind[i]; });
#pragma unroll
  for (int i = 0; i < R; ++i) {
    int before = here[i];  // inclusive sum over the lanes
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int other = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before += other;
    }
    const int sum = __shfl_sync(0xffffffffu, before, 31);
    if (index < sum) {
      const int owner = __ffs(__ballot_sync(0xffffffffu, index < before)) - 1;
      const int nth = behind[i] + index - (before - here[i]);  // in the order of falling length
      auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, owner); };
      const int piece = by_keys ? nth : count[i] - 1 - nth;
      span.unit_in_sequence = of(piece);
      span.sequence = owner + 32 * i;
      span.q0 = of(q0[i]);
      span.rows = of(q1[i]) - span.q0;
      span.k0 = of(k0[i]);
      span.room = of(k1[i]) - span.k0;
      span.keys = of(keys[i]);
      return span;
    }
    index -= sum;
  }
  return span;
}

// Piece of a tile launch: ranked by length where that is possible.
__device__ __forceinline__ PackedSpan find_piece(int unit, int step, bool by_keys, const int* __restrict__ q_offsets,
                                                 const int* __restrict__ k_offsets, const int* __restrict__ k_lengths,
                                                 int sequences, int64_t total_q, int64_t total_k, int* status) {
  if (sequences <= 32)
    return find_ranked<1>(unit, step, by_keys, q_offsets, k_offsets, k_lengths, sequences, total_q, total_k, status);
  if (sequences <= MAX_RANKED)
    return find_ranked<2>(unit, step, by_keys, q_offsets, k_offsets, k_lengths, sequences, total_q, total_k, status);
  PackedSpan span = find_unit(unit, step, by_keys, q_offsets, k_offsets, k_lengths, sequences, total_q, total_k, status);
  if (!by_keys && span.unit_in_sequence >= 0) {  // late pieces of a sequence see the most keys and come first
    const int pieces = (span.rows + step - 1) / step;
    span.unit_in_sequence = pieces == 0 ? -1 : pieces - 1 - span.unit_in_sequence;
  }
  return span;
}

// Instruction descriptor for fp16 or bf16 operands (format 0 / 1), fp32 accumulation.
__host__ __device__ constexpr uint32_t make_idesc_16(bool fp16, int m, int n, int a_mn_major, int b_mn_major) {
  return make_idesc_bf16(m, n, a_mn_major, b_mn_major) & (fp16 ? ~((1u << 7) | (1u << 10)) : ~0u);
}

template <bool FP16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (FP16) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  return pack_bf16(lo, hi);
}
template <bool FP16>
__device__ __forceinline__ float2 unpack16(uint32_t v) {
  if (FP16) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  return make_float2(bf16_lo(v), bf16_hi(v));
}

// 2^x for two finite or NaN x, on the FMA pipe instead of the special-function unit: x = n + f with n the
// nearest integer (Cody and Waite), a polynomial of degree 4 for 2^f that is off by at most 2.6e-6 of
// it on [-1/2, 1/2] (fitted for the smallest largest relative error), and n added to the exponent.
// x is taken as at least -126; NaN stays without a finite value of use.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  asm("max.NaN.f32 %0, %1, 0fC2FC0000;" : "=f"(x.x) : "f"(x.x));
  asm("max.NaN.f32 %0, %1, 0fC2FC0000;" : "=f"(x.y) : "f"(x.y));
  const float2 magic = make_float2(12582912.f, 12582912.f);  // 1.5 * 2^23: the sum's last bits are n
  const float2 t = fadd2(x, magic);
  const float2 n = fadd2(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = ffma2(n, make_float2(-1.f, -1.f), x);
  float2 p = ffma2(f, make_float2(0.00957010196f, 0.00957010196f), make_float2(0.0559178607f, 0.0559178607f));
  p = ffma2(p, f, make_float2(0.240247448f, 0.240247448f));
  p = ffma2(p, f, make_float2(0.693121815f, 0.693121815f));
  p = ffma2(p, f, make_float2(0.999999261f, 0.999999261f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}

}  // namespace agb
