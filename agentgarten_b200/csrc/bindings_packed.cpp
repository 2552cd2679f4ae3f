// Python bindings of the rotary positions and of the attention over packed sequences.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>

#include "agb.h"
#include "bindings.h"
#include "packed.h"

namespace agb_python {
namespace {

using torch::Tensor;

cudaStream_t stream_of(const Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

void check(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e), " (", agb::error_detail(), ")");
}

int sm_count(const Tensor& t) { return at::cuda::getDeviceProperties(t.device().index())->multiProcessorCount; }

// [..., heads, dim] as (tokens, heads, dim) with one stride between tokens, copied when it has none.
Tensor token_rows(const Tensor& t) {
  int64_t expected = 0;
  bool uniform = t.stride(-1) == 1 || t.size(-1) == 1;
  for (int64_t i = t.dim() - 3; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (expected && t.stride(i) != expected) uniform = false;
    expected = t.stride(i) * t.size(i);
  }
  return uniform ? t : t.contiguous();
}

int64_t row_stride_of(const Tensor& t) {
  for (int64_t i = t.dim() - 3; i >= 0; --i)
    if (t.size(i) > 1) return t.stride(i);
  return t.size(-2) * t.size(-1);
}

std::vector<Tensor> rotary_embed(const Tensor& query, const c10::optional<Tensor>& key, const Tensor& positions,
                                 const Tensor& turns, const c10::optional<Tensor>& axis, double amplitude,
                                 bool interleaved, bool backwards) {
  c10::cuda::CUDAGuard guard(query.device());
  agb::RotaryArgs a{};
  const int64_t tokens = positions.numel() / (axis.has_value() ? positions.size(-1) : 1);
  const Tensor where = positions.contiguous();
  std::vector<Tensor> held, out;
  for (int i = 0; i < (key.has_value() ? 2 : 1); ++i) {
    held.push_back(token_rows(i == 0 ? query : *key));
    const Tensor& x = held.back();
    out.push_back(torch::empty(x.sizes(), x.options()));
    a.part[i].x = x.data_ptr();
    a.part[i].out = out.back().data_ptr();
    a.part[i].heads = int(x.size(-2));
    a.part[i].row_stride = row_stride_of(x);
    a.part[i].head_stride = x.size(-2) == 1 ? x.size(-1) : x.stride(-2);
  }
  a.positions = where.data_ptr();
  a.position_type = where.scalar_type() == torch::kInt32 ? 0 : where.scalar_type() == torch::kInt64 ? 1 : 2;
  a.turns = turns.data_ptr<double>();
  a.axis = axis.has_value() ? axis->data_ptr<int>() : nullptr;
  a.axes = axis.has_value() ? int(where.size(-1)) : 1;
  a.amplitude = float(amplitude);
  a.direction = backwards ? -1.f : 1.f;
  a.tokens = tokens;
  a.dim = int(query.size(-1));
  a.turned = 2 * int(turns.numel());
  a.interleaved = interleaved;
  a.type = query.scalar_type() == torch::kBFloat16 ? 0 : query.scalar_type() == torch::kHalf ? 1 : 2;
  a.sm_count = sm_count(query);
  check(agb::rotary_embed(a, stream_of(query)), "rotary_embed");
  return out;
}

// Strides that the tensor maps take: unit inner stride, everything else 16-byte aligned and not zero.
Tensor mappable(const Tensor& t) {
  const bool fits = (t.size(2) == 1 || t.stride(2) == 1) && (t.size(1) == 1 || (t.stride(1) % 8 == 0 && t.stride(1) > 0)) &&
                    (t.size(0) == 1 || (t.stride(0) % 8 == 0 && t.stride(0) > 0)) &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
int64_t head_stride(const Tensor& t) { return t.size(1) == 1 ? t.size(2) : t.stride(1); }
int64_t row_stride(const Tensor& t) { return t.size(0) == 1 ? t.size(1) * t.size(2) : t.stride(0); }

agb::PackedArgs packed_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_offsets,
                            const Tensor& k_offsets, const c10::optional<Tensor>& k_lengths, double scale) {
  agb::PackedArgs a{};
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
  a.q_offsets = q_offsets.data_ptr<int>();
  a.k_offsets = k_offsets.data_ptr<int>();
  a.k_lengths = k_lengths.has_value() ? k_lengths->data_ptr<int>() : nullptr;
  a.sequences = int(q_offsets.size(0) - 1);
  a.total_q = q.size(0); a.total_k = k.size(0);
  a.q_row = row_stride(q); a.q_head = head_stride(q);
  a.k_row = row_stride(k); a.k_head = head_stride(k);
  a.v_row = row_stride(v); a.v_head = head_stride(v);
  a.hq = int(q.size(1)); a.hkv = int(k.size(1)); a.dim = int(q.size(2));
  a.fp16 = q.scalar_type() == torch::kHalf;
  a.scale = float(scale);
  a.status = status_word(q.device().index()).data_ptr<int>();
  a.splits = 1;
  return a;
}

// The kernels are chosen by the totals alone: the lengths are on the device.
//
// The few-row kernel where the sequences have on average no more rows than one of its products.
bool few_rows(const agb::PackedArgs& a) {
  const int heads = std::min(a.hq / a.hkv, 16);
  return a.total_q * heads <= int64_t(16) * a.sequences;
}

// Keys of a chunk: about three CTAs for every place (two on an SM), and never so few that joining them shows.
int rows_chunk(const agb::PackedArgs& a, int sms) {
  const int64_t work = a.total_k * a.hkv * agb::packed_rows_pieces(a.hq / a.hkv);
  const int64_t chunk = (work / (int64_t(sms) * 2 * 3) + 63) / 64 * 64;
  return int(std::min<int64_t>(std::max<int64_t>(chunk, 256), 8192));
}

// Key ranges of a tile: the count that makes the estimated launch shortest.  In units of one key
// tile's work (about 0.9 us): the longest CTA, twice the mean's, or all of the work over the SMs;
// then the join, about 4 us and the partial results' way to memory and back.
int tile_splits(const agb::PackedArgs& a, int sms) {
  const bool paired = (a.hq / a.hkv) % 2 == 0;
  const double step = paired ? 128 : 256;
  const double rows = double(a.total_q) / a.sequences, keys = double(a.total_k) / a.sequences;
  const double pieces = std::ceil(rows / step);
  const double seen = std::max(keys - rows / 2, rows / 2);  // of a row, on average
  const double tiles = std::ceil(seen / 128);
  const double all = a.sequences * pieces * (paired ? a.hq / 2 : a.hq) * tiles / sms;
  const double partial = double(a.total_q) * a.hq * a.dim * 8 / 6.5e6 / 0.9;
  int best = 1;
  double best_cost = std::max(2 * tiles, all);
  for (int s = 2; s <= 16 && 2 * tiles / s >= 4; ++s) {
    const double cost = std::max(std::ceil(2 * tiles / s), all) + 4 / 0.9 + s * partial;
    if (cost < 0.9 * best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}

// (out, lse [hq, total_q] or an empty tensor)
std::tuple<Tensor, Tensor> packed_attention_fwd(const Tensor& query, const Tensor& key, const Tensor& value,
                                                const Tensor& q_offsets, const Tensor& k_offsets,
                                                const c10::optional<Tensor>& k_lengths, double scale, bool want_lse) {
  c10::cuda::CUDAGuard guard(query.device());
  Tensor out = torch::empty(query.sizes(), query.options());
  const auto fp32 = query.options().dtype(torch::kFloat32);
  Tensor lse = torch::empty({want_lse ? query.size(1) : 0, query.size(0)}, fp32);
  if (query.numel() == 0) return {out, lse};
  if (key.size(0) == 0 || q_offsets.size(0) == 1) {
    out.zero_();
    lse.fill_(-INFINITY);
    return {out, lse};
  }
  const Tensor q = mappable(query), k = mappable(key), v = mappable(value);
  agb::PackedArgs a = packed_args(q, k, v, q_offsets, k_offsets, k_lengths, scale);
  a.out = out.data_ptr();
  a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  Tensor part_out, part_lse;
  const int sms = sm_count(q), group = a.hq / a.hkv;
  if (few_rows(a)) {
    const int64_t pieces = agb::packed_rows_pieces(group);
    a.chunk = rows_chunk(a, sms);
    if (a.total_k > a.chunk) {
      const int64_t slots = (a.total_k / a.chunk + a.sequences) * a.hkv * pieces * 16;
      part_out = torch::empty({slots, a.dim}, fp32);
      part_lse = torch::empty({slots}, fp32);
      a.part_out = part_out.data_ptr<float>();
      a.part_lse = part_lse.data_ptr<float>();
    }
    check(agb::packed_attention_rows(a, stream_of(q)), "packed_attention");
    return {out, lse};
  }
  a.splits = tile_splits(a, sms);
  if (a.splits > 1) {
    part_out = torch::empty({a.splits, a.total_q, a.hq, a.dim}, fp32);
    part_lse = torch::empty({a.splits, a.total_q, a.hq}, fp32);
    a.part_out = part_out.data_ptr<float>();
    a.part_lse = part_lse.data_ptr<float>();
  }
  check(agb::packed_attention_tiles(a, stream_of(q)), "packed_attention");
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> packed_attention_bwd(
    const Tensor& grad_out, const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& out,
    const Tensor& lse, const Tensor& q_offsets, const Tensor& k_offsets, const c10::optional<Tensor>& k_lengths,
    double scale) {
  c10::cuda::CUDAGuard guard(query.device());
  Tensor dq = torch::empty(query.sizes(), query.options());
  Tensor dk = torch::empty(key.sizes(), key.options());
  Tensor dv = torch::empty(value.sizes(), value.options());
  if (query.numel() == 0 || key.size(0) == 0 || q_offsets.size(0) == 1) {
    dq.zero_();
    dk.zero_();
    dv.zero_();
    return {dq, dk, dv};
  }
  const Tensor q = mappable(query), k = mappable(key), v = mappable(value), grad = mappable(grad_out);
  Tensor delta = torch::empty(lse.sizes(), lse.options());
  agb::PackedArgs a = packed_args(q, k, v, q_offsets, k_offsets, k_lengths, scale);
  a.out = out.data_ptr();
  a.lse = lse.data_ptr<float>();
  agb::PackedGrads g{};
  g.grad = grad.data_ptr();
  g.grad_row = row_stride(grad); g.grad_head = head_stride(grad);
  g.dq = dq.data_ptr(); g.dk = dk.data_ptr(); g.dv = dv.data_ptr();
  g.delta = delta.data_ptr<float>();
  check(agb::packed_attention_bwd(a, g, stream_of(q)), "packed_attention_bwd");
  return {dq, dk, dv};
}

}  // namespace

void bind_packed(pybind11::module& m) {
  m.def("rotary_embed", &rotary_embed);
  m.def("packed_attention_fwd", &packed_attention_fwd);
  m.def("packed_attention_bwd", &packed_attention_bwd);
}

}  // namespace agb_python
