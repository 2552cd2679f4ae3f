// Python bindings of the rotary positions and of the attention over packed sequences.
//
// A call checks its arguments, launches and (where a gradient is wanted) records its node here, in
// one step from Python: with the checks and the autograd function in Python a call cost 20 us of the
// host and a training step of two calls 140 us, more than the kernels of a short prompt.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
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
  int64_t expected = -1;  // the stride that goes on where the inner dimensions end
  bool uniform = t.stride(-1) == 1 || t.size(-1) == 1;
  for (int64_t i = t.dim() - 3; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (expected >= 0 && t.stride(i) != expected) uniform = false;
    expected = t.stride(i) * t.size(i);
  }
  return uniform ? t : t.contiguous();
}

int64_t row_stride_of(const Tensor& t) {
  for (int64_t i = t.dim() - 3; i >= 0; --i)
    if (t.size(i) > 1) return t.stride(i);
  return t.size(-2) * t.size(-1);
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptionalTensor = c10::optional<Tensor>;

std::atomic<int64_t> launches{0};

[[noreturn]] void refuse_value(const char* op, const std::string& why) {
  throw pybind11::value_error(std::string(op) + ": " + why);
}
[[noreturn]] void refuse_type(const char* op, const std::string& why) {
  throw pybind11::type_error(std::string(op) + ": " + why);
}

Tensor empty(at::IntArrayRef sizes, const Tensor& like) {
  return at::detail::empty_cuda(sizes, like.scalar_type(), like.device(), c10::nullopt);
}
Tensor empty_fp32(at::IntArrayRef sizes, const Tensor& like) {
  return at::detail::empty_cuda(sizes, at::kFloat, like.device(), c10::nullopt);
}

bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
bool wants_grad(const Tensor& t) { return t.requires_grad(); }

// A gradient of these kernels has no gradient of its own: asking for one raises, as Python's
// once_differentiable does.
variable_list once(variable_list grads, const char* op) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list present;
  for (const Tensor& g : grads)
    if (g.defined()) present.push_back(g.detach().requires_grad_(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(op) + " is differentiable once: its gradient has no gradient", int(present.size()));
  variable_list guarded = (*error)(std::move(present));
  size_t at = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = guarded[at++];
  return grads;
}

// ------------------------------------------------------------------------------- rotary positions
struct Turn {
  Tensor positions, turns;
  OptionalTensor axis;
  double amplitude;
  bool interleaved;
};

// query and key (either may be undefined) turned by their positions
std::pair<Tensor, Tensor> turn(const Tensor& query, const Tensor& key, const Turn& by, bool backwards) {
  const Tensor& some = query.defined() ? query : key;
  c10::cuda::CUDAGuard guard(some.device());
  agb::RotaryArgs a{};
  const Tensor where = by.positions.contiguous();
  Tensor held[2], out[2];
  for (int i = 0; i < 2; ++i) {
    const Tensor& given = i == 0 ? query : key;
    if (!given.defined()) continue;
    held[i] = token_rows(given);
    const Tensor& x = held[i];
    out[i] = empty(x.sizes(), x);
    a.part[i].x = x.data_ptr();
    a.part[i].out = out[i].data_ptr();
    a.part[i].heads = int(x.size(-2));
    a.part[i].row_stride = row_stride_of(x);
    a.part[i].head_stride = x.size(-2) == 1 ? x.size(-1) : x.stride(-2);
  }
  a.positions = where.data_ptr();
  a.position_type = where.scalar_type() == torch::kInt32 ? 0 : where.scalar_type() == torch::kInt64 ? 1 : 2;
  a.turns = by.turns.data_ptr<double>();
  a.axis = by.axis.has_value() ? by.axis->data_ptr<int>() : nullptr;
  a.axes = by.axis.has_value() ? 3 : 1;
  a.amplitude = float(by.amplitude);
  a.direction = backwards ? -1.f : 1.f;
  a.tokens = where.numel() / a.axes;
  a.dim = int(some.size(-1));
  a.turned = 2 * int(by.turns.numel());
  a.interleaved = by.interleaved;
  a.type = some.scalar_type() == torch::kBFloat16 ? 0 : some.scalar_type() == torch::kHalf ? 1 : 2;
  a.sm_count = sm_count(some);
  check(agb::rotary_embed(a, stream_of(some)), "rotary_embed");
  ++launches;
  return {out[0], out[1]};
}

// The gradient of a turn is the turn back: nothing of the values is kept.
struct RotaryEmbed : public torch::autograd::Function<RotaryEmbed> {
  static variable_list forward(AutogradContext* ctx, const Tensor& query, const OptionalTensor& key,
                               const Tensor& positions, const Tensor& turns, const OptionalTensor& axis,
                               double amplitude, bool interleaved) {
    const Turn by{positions, turns, axis, amplitude, interleaved};
    ctx->save_for_backward({positions, turns, axis.value_or(Tensor())});
    ctx->saved_data["amplitude"] = amplitude;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    auto out = turn(query, key.value_or(Tensor()), by, false);
    return key.has_value() ? variable_list{out.first, out.second} : variable_list{out.first};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Turn by{saved[0], saved[1], saved[2].defined() ? OptionalTensor(saved[2]) : c10::nullopt,
                  ctx->saved_data["amplitude"].toDouble(), ctx->saved_data["interleaved"].toBool()};
    const Tensor dq = grads[0], dk = grads.size() > 1 ? grads[1] : Tensor();
    std::pair<Tensor, Tensor> back;
    if (dq.defined() || dk.defined()) back = turn(dq, dk, by, true);
    return once({back.first, back.second, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, "rotary_embed");
  }
};

// Query and key turned, or None where the kernel does not cover the call.
c10::optional<variable_list> rotary_embed(const Tensor& query, const OptionalTensor& key, const Tensor& positions,
                                          const Tensor& turns, const OptionalTensor& axis, double amplitude,
                                          bool interleaved) {
  static const char* op = "rotary_embed";
  const int64_t dims = query.dim();
  auto fits = [&](const Tensor& t) {
    if (t.dim() != dims || dims < 3 || t.size(-1) != query.size(-1) || t.size(-2) == 0) return false;
    for (int64_t i = 0; i + 2 < dims; ++i)
      if (t.size(i) != query.size(i)) return false;
    return true;
  };
  if (!fits(query)) refuse_value(op, "query is not [..., heads, dim]");
  if (key.has_value() && !fits(*key)) refuse_value(op, "key is not [..., heads, dim] over the query's leading dimensions");
  const auto type = query.scalar_type();
  if ((key.has_value() && key->scalar_type() != type) ||
      (type != torch::kBFloat16 && type != torch::kHalf && type != torch::kFloat32 && type != torch::kFloat64))
    refuse_type(op, "query and key are both bf16, fp16, fp32 or fp64");
  if (2 * turns.numel() > query.size(-1)) refuse_value(op, "more elements to turn than a head has");
  const bool axes = axis.has_value();
  bool matches = positions.dim() == dims - 2 + (axes ? 1 : 0) && (!axes || positions.size(-1) == 3);
  for (int64_t i = 0; matches && i + 2 < dims; ++i) matches = positions.size(i) == query.size(i);
  if (!matches) refuse_value(op, "positions have the query's leading dimensions, and three axes where the frequencies have");
  if (positions.scalar_type() != torch::kInt32 && positions.scalar_type() != torch::kInt64 &&
      positions.scalar_type() != torch::kFloat32)
    refuse_type(op, "positions are int32, int64 or fp32");
  if (positions.device() != query.device() || turns.device() != query.device() ||
      (key.has_value() && key->device() != query.device()) || (axes && axis->device() != query.device()))
    refuse_value(op, "query, key, positions and frequencies are on one device");
  if (turns.scalar_type() != torch::kFloat64 || !turns.is_contiguous() || turns.dim() != 1 || turns.numel() == 0 ||
      (axes && (axis->scalar_type() != torch::kInt32 || !axis->is_contiguous() || axis->numel() != turns.numel())))
    refuse_value(op, "frequencies are what rotary_frequencies gives");
  if (type == torch::kFloat64 || has_tangent(query) || (key.has_value() && has_tangent(*key))) return c10::nullopt;
  if (at::GradMode::is_enabled() && (wants_grad(query) || (key.has_value() && wants_grad(*key))))
    return RotaryEmbed::apply(query, key, positions, turns, axis, amplitude, interleaved);
  auto out = turn(query, key.value_or(Tensor()), {positions, turns, axis, amplitude, interleaved}, false);
  return variable_list{out.first, out.second};
}

// ---------------------------------------------------------------------------- packed attention
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
  a.sm_count = sm_count(q);
  return a;
}

// The kernels are chosen by the totals alone: the lengths are on the device.
//
// The few-row kernel where a sequence has on average at most two of its blocks of 16 (query row, head)
// pairs.  Per call, few-row against tile kernel, with 32 query and 8 key heads of 128: eight prompts of
// 8 / 17 rows 5.6 : 8.7, 9.5 : 8.9 us; 64 of 8 / 17 rows 17 : 29, 36 : 29.  (It is also the faster one for a
// single prompt of up to 64 rows, 7.2 : 8.8 us; but there a prompt would come out a rounding different
// alone than among others.)
bool few_rows(const agb::PackedArgs& a) {
  return a.total_q * std::min(a.hq / a.hkv, 16) <= int64_t(32) * a.sequences;
}

// Keys of a chunk.  Eight warps an SM take one job each at a time.  Where chunks of at most 512 keys give no
// more jobs than that, just such chunks: a job is a chain of loads, and there is no second one to hide
// its end.  Longer ones would leave uneven caches with a long tail, so there about three jobs for every
// warp.  Per call, this rule against three jobs of at least 128 keys, 32 query and 8 key heads of 128: one
// token against 500 / 4000 / 32000 / 38000 keys 11.3 : 14.8, 13.8 : 15.4, 35.1 : 37.4, 37.9 : 45.1 us; 16 tokens
// against 1200 each 23 : 28, 32 against 1000 each 34.2 : 35.8; eight prompts of 8 rows on 1000, the one that
// lost, 25.6 : 25.1.
int rows_chunk(const agb::PackedArgs& a, int sms) {
  const int64_t side = int64_t(a.hkv) * agb::packed_rows_pieces(a.hq / a.hkv), warps = int64_t(sms) * 8;
  if (a.total_k <= int64_t(128) * a.sequences) return 128;
  const int64_t spare = warps - a.sequences * side;  // a sequence's last chunk is a short one
  if (2 * spare >= warps) {
    const int64_t once = (a.total_k * side + spare - 1) / spare;
    if (once <= 512) return int((std::max<int64_t>(once, 32) + 31) / 32 * 32);
  }
  const int64_t chunk = (a.total_k * side / (3 * warps) + 63) / 64 * 64;
  return int(std::min<int64_t>(std::max<int64_t>(chunk, 128), 8192));
}

// Key ranges of a tile: the count that makes the estimated launch shortest.  In units of one key
// tile's work (about 0.9 us): the longest CTA, twice the mean's, or all of the work over the SMs;
// then the join, about 4 us and the partial results' way to memory and back.  With the rule and in one
// range, 32 query and 8 key heads of 128, cold caches: 40 rows against 5000 keys 25 : 72 us, 512 against
// 4000 64 : 66, 512 against 20000 164 : 264, four prompts of 64 against 4000 46 : 66; eight of 200 against
// 2000 and a prompt of 1024 stay in one range.
int tile_splits(const agb::PackedArgs& a, int sms) {
  int fold = 1;
  while (fold < 16 && (a.hq / a.hkv) % (2 * fold) == 0) fold *= 2;
  const double step = 256 / fold;
  const double rows = double(a.total_q) / a.sequences, keys = double(a.total_k) / a.sequences;
  const double pieces = std::ceil(rows / step);
  const double seen = std::max(keys - rows / 2, rows / 2);  // of a row, on average
  const double tiles = std::ceil(seen / 128);
  const double all = a.sequences * pieces * (a.hq / fold) * tiles / sms;
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
std::pair<Tensor, Tensor> attend(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& q_offsets,
                                 const Tensor& k_offsets, const OptionalTensor& k_lengths, double scale, bool want_lse) {
  c10::cuda::CUDAGuard guard(query.device());
  Tensor out = empty(query.sizes(), query), lse;
  if (want_lse) lse = empty_fp32({query.size(1), query.size(0)}, query);
  if (query.numel() == 0) return {out, lse};
  if (key.size(0) == 0 || q_offsets.size(0) == 1) {
    out.zero_();
    return {out, lse};
  }
  const Tensor q = mappable(query), k = mappable(key), v = mappable(value);
  agb::PackedArgs a = packed_args(q, k, v, q_offsets, k_offsets, k_lengths, scale);
  a.out = out.data_ptr();
  a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  Tensor part_out, part_lse, part_jobs;
  const int sms = sm_count(q), group = a.hq / a.hkv;
  if (few_rows(a)) {
    const int64_t pieces = agb::packed_rows_pieces(group);
    a.chunk = rows_chunk(a, sms);
    if (a.total_k > a.chunk) {
      const int64_t slots = agb::packed_rows_jobs(a) * a.hkv * pieces * 16;
      part_out = empty_fp32({slots, a.dim}, q);
      part_lse = empty_fp32({slots}, q);
      part_jobs = empty({a.sequences, 2}, q_offsets);
      a.part_jobs = part_jobs.data_ptr<int>();
      a.part_out = part_out.data_ptr<float>();
      a.part_lse = part_lse.data_ptr<float>();
    }
    check(agb::packed_attention_rows(a, stream_of(q)), "packed_attention");
    launches += a.total_k > a.chunk ? 2 : 1;
    return {out, lse};
  }
  a.splits = tile_splits(a, sms);
  if (a.splits > 1) {
    part_out = empty_fp32({a.splits, a.total_q, a.hq, a.dim}, q);
    part_lse = empty_fp32({a.splits, a.total_q, a.hq}, q);
    a.part_out = part_out.data_ptr<float>();
    a.part_lse = part_lse.data_ptr<float>();
  }
  check(agb::packed_attention_tiles(a, stream_of(q)), "packed_attention");
  launches += a.splits > 1 ? 2 : 1;
  return {out, lse};
}

struct PackedAttention : public torch::autograd::Function<PackedAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& query, const Tensor& key, const Tensor& value,
                        const Tensor& q_offsets, const Tensor& k_offsets, const OptionalTensor& k_lengths, double scale) {
    auto [out, lse] = attend(query, key, value, q_offsets, k_offsets, k_lengths, scale, true);
    ctx->save_for_backward({query, key, value, out, lse, q_offsets, k_offsets, k_lengths.value_or(Tensor())});
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &query = saved[0], &key = saved[1], &value = saved[2], &out = saved[3], &lse = saved[4];
    const OptionalTensor k_lengths = saved[7].defined() ? OptionalTensor(saved[7]) : c10::nullopt;
    c10::cuda::CUDAGuard guard(query.device());
    const bool key_side = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    Tensor dq = empty(query.sizes(), query), dk, dv;
    if (key_side) {
      dk = empty(key.sizes(), key);
      dv = empty(value.sizes(), value);
    }
    if (query.numel() == 0 || key.size(0) == 0 || saved[5].size(0) == 1) {
      dq.zero_();
      if (key_side) {
        dk.zero_();
        dv.zero_();
      }
    } else {
      const Tensor q = mappable(query), k = mappable(key), v = mappable(value), grad = mappable(grads[0]);
      Tensor delta = empty_fp32(lse.sizes(), lse);
      agb::PackedArgs a = packed_args(q, k, v, saved[5], saved[6], k_lengths, ctx->saved_data["scale"].toDouble());
      a.out = out.data_ptr();
      a.lse = lse.data_ptr<float>();
      agb::PackedGrads g{};
      g.grad = grad.data_ptr();
      g.grad_row = row_stride(grad);
      g.grad_head = head_stride(grad);
      g.dq = dq.data_ptr();
      if (key_side) {
        g.dk = dk.data_ptr();
        g.dv = dv.data_ptr();
      }
      g.delta = delta.data_ptr<float>();
      check(agb::packed_attention_bwd(a, g, stream_of(q)), "packed_attention");
      launches += key_side ? 2 : 1;
    }
    return once({dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()}, "packed_attention");
  }
};

// The attention, or None where the kernels do not cover the call.
c10::optional<Tensor> packed_attention(const Tensor& query, const Tensor& key, const Tensor& value,
                                       const Tensor& q_offsets, const OptionalTensor& k_offsets,
                                       const OptionalTensor& k_lengths, c10::optional<double> scale_given) {
  static const char* op = "packed_attention";
  if (query.dim() != 3 || key.dim() != 3 || value.sizes() != key.sizes() || query.size(2) != key.size(2))
    refuse_value(op, "query, key and value are not [total, heads, dim] with one dim");
  const int64_t heads = query.size(1), dim = query.size(2);
  if (heads == 0 || dim == 0 || key.size(1) == 0 || heads % key.size(1))
    refuse_value(op, "the query heads are not a multiple of the key heads");
  const auto type = query.scalar_type();
  if (key.scalar_type() != type || value.scalar_type() != type || !c10::isFloatingType(type))
    refuse_type(op, "query, key and value have one floating type");
  if (!k_offsets.has_value() && query.size(0) != key.size(0))
    refuse_value(op, "k_offsets are needed where keys and queries are not the same rows");
  const Tensor& keys_at = k_offsets.has_value() ? *k_offsets : q_offsets;
  const auto device = query.device();
  bool together = key.device() == device && value.device() == device;
  for (const Tensor* t : {&q_offsets, &keys_at, k_lengths.has_value() ? &*k_lengths : &q_offsets}) {
    if (t->scalar_type() != torch::kInt32 || t->dim() != 1 || !t->is_contiguous())
      refuse_type(op, "offsets and lengths are contiguous int32 vectors");
    together = together && t->device() == device;
  }
  if (q_offsets.size(0) < 1 || keys_at.size(0) != q_offsets.size(0) ||
      (k_lengths.has_value() && k_lengths->size(0) != q_offsets.size(0) - 1))
    refuse_value(op, "sequences + 1 offsets of queries and of keys, and one length a sequence");
  if (!together) refuse_value(op, "all tensors are on one device");
  if (std::max(query.size(0), key.size(0)) >= (int64_t(1) << 31) - 256) refuse_value(op, "rows are counted in 32 bits");
  const double scale = scale_given.has_value() ? *scale_given : 1.0 / std::sqrt(double(dim));
  if (!(scale > 0) || std::isinf(scale)) refuse_value(op, "scale is positive");
  if ((type != torch::kBFloat16 && type != torch::kHalf) || dim % 8 || dim > 128 || heads * dim >= (1 << 24) || has_tangent(query) ||
      has_tangent(key) || has_tangent(value))
    return c10::nullopt;
  if (at::GradMode::is_enabled() && (wants_grad(query) || wants_grad(key) || wants_grad(value)))
    return PackedAttention::apply(query, key, value, q_offsets, keys_at, k_lengths, scale);
  return attend(query, key, value, q_offsets, keys_at, k_lengths, scale, false).first;
}

}  // namespace

void bind_packed(pybind11::module& m) {
  m.def("rotary_embed", &rotary_embed);
  m.def("packed_attention", &packed_attention);
  m.def("packed_launches", [] { return launches.load(); });
}

}  // namespace agb_python
