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

namespace agb {

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

}  // namespace agb
