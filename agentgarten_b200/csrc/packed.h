// Host-callable launchers of the rotary positions and of the attention over packed sequences.
// Every launcher enqueues on the given stream and returns a cudaError_t; none allocates.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace agb {

// ------------------------------------------------------------------------ rotary positions
// Turns the first `turned` elements of every head of x by position * turns * 2 pi and copies the
// rest: pair j is (x[j], x[turned / 2 + j]), or (x[2 j], x[2 j + 1]) when interleaved.  Up to two
// tensors (query and key) share the tokens; a part with heads == 0 is absent.  direction -1 turns
// back (the gradient).  `out` is dense [tokens, heads, dim]; strides are in elements.
struct RotaryPart {
  const void* x;
  void* out;
  int64_t row_stride, head_stride;
  int heads;
};
struct RotaryArgs {
  RotaryPart part[2];
  const void* positions;   // [tokens, axes]: int32 (0), int64 (1) or fp32 (2)
  int position_type;
  const double* turns;     // [turned / 2] turns per position
  const int* axis;         // [turned / 2] column of positions that turns the slot, or null (column 0)
  int axes;
  float amplitude, direction;
  int64_t tokens;
  int dim, turned, interleaved;
  int type;                // 0 bf16, 1 fp16, 2 fp32
  int sm_count;
};
cudaError_t rotary_embed(const RotaryArgs& args, cudaStream_t stream);

// ---------------------------------------------------------------- packed causal attention
// q [total_q, hq, dim], k / v [total_k, hkv, dim] in bf16 or fp16 with unit inner stride, 16-byte
// aligned rows and heads (strides in elements); dim is a multiple of 8, at most 128.  Sequence s
// owns query rows [q_offsets[s], q_offsets[s + 1]) and the first k_lengths[s] (null: all) of the
// key rows [k_offsets[s], k_offsets[s + 1]); its queries are the last rows of its keys.  out is
// dense [total_q, hq, dim], lse fp32 [hq, total_q] (may be null).  Rows without a visible key and
// rows behind the last sequence become zero.  Offsets that do not fit the tensors are reported
// through the status word and their sequence is skipped.
struct PackedArgs {
  const void* q; const void* k; const void* v;
  void* out;
  float* lse;
  const int* q_offsets; const int* k_offsets; const int* k_lengths;
  int sequences;
  int64_t total_q, total_k;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int hq, hkv, dim, fp16;
  float scale;
  int* status;
  // FP32 partial results of the keys' ranges: with splits > 1 the tile kernel's [splits, total_q, hq, dim]
  // and [splits, total_q, hq]; for the few-row kernel, whose ranges are chunks of `chunk` keys,
  // [units, hkv, pieces, 16, dim] and [units, hkv, pieces, 16] with units = packed_rows_jobs()
  // and pieces = packed_rows_pieces(hq / hkv), with the first job and the chunks of every sequence in
  // part_jobs [sequences, 2] (unused when total_k <= chunk).
  int splits, chunk;
  int sm_count;
  float* part_out;
  float* part_lse;
  int* part_jobs;
};
cudaError_t packed_attention_tiles(const PackedArgs& args, cudaStream_t stream);
// The same function for few query rows; right for any.
cudaError_t packed_attention_rows(const PackedArgs& args, cudaStream_t stream);
int packed_rows_pieces(int group);
int64_t packed_rows_jobs(const PackedArgs& args);  // at most, of one key head and piece

// Gradient: args carries the forward's tensors (out and lse filled in); grad [total_q, hq, dim] with
// the strides given, dq / dk / dv dense like q / k / v, delta fp32 scratch [hq, total_q].  Rows of no
// sequence and key rows behind k_lengths receive zeros.
struct PackedGrads {
  const void* grad;
  int64_t grad_row, grad_head;
  void* dq; void* dk; void* dv;  // dk and dv may both be null: not wanted
  float* delta;
};
cudaError_t packed_attention_bwd(const PackedArgs& args, const PackedGrads& grads, cudaStream_t stream);

}  // namespace agb
