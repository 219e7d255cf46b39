// The host side of attention and of its position bias: arguments, copies where a layout needs one, results, launches, and the autograd nodes.
#include "torch_common.h"

#include <ATen/SavedTensorHooks.h>

#include <array>

namespace {

const char* const kAttention = "attention";
const char* const kBias = "the position bias";

// [batch, heads, rows, width] as the kernels load it; `width` is the tensor's rounded up to whole 16-byte pieces
struct Heads {
  at::Tensor held;
  gact_rows rows{};
};
gact_rows rows_of(const at::Tensor& t, bool transposed) {     // transposed: [batch, rows, heads, width]
  return {out(t), t.stride(0), t.stride(transposed ? 2 : 1), t.stride(transposed ? 1 : 2)};
}
Heads heads_of(const at::Tensor& given, int64_t width, const Place& at) {
  Heads h;
  const at::Tensor t = given.is_neg() ? given.resolve_neg() : given;
  const int64_t e = (int64_t)t.element_size();
  bool fits = t.size(3) == width && (t.numel() == 0 || (aligned(in(t)) && (width == 1 || t.stride(3) == 1)));
  for (int d = 0; d < 3 && fits; d++) fits = t.size(d) <= 1 || t.stride(d) * e % 16 == 0;
  if (fits && t.size(2) > 1) fits = t.stride(2) >= width && t.stride(2) * e <= GACT_ATTENTION_MAX_STRIDE;
  if (fits) {
    h.held = t;
    h.rows = {in(t), t.stride(0), t.stride(1), t.stride(2)};
    return h;
  }
  const std::array<int64_t, 4> shape{t.size(0), t.size(2), t.size(1), width};
  h.held = t.size(3) == width ? at.empty(shape, t.scalar_type()) : at.zeros(shape, t.scalar_type());
  h.held.narrow(3, 0, t.size(3)).copy_(t.transpose(1, 2));
  h.rows = rows_of(h.held, true);
  return h;
}
// a result of the kernels, [batch, rows, heads, padded width], as [batch, heads, rows, width]: the heads of a row lie side by side
at::Tensor result_of(const at::Tensor& t, int64_t width) {
  return (t.size(3) == width ? t : t.narrow(3, 0, width).contiguous()).transpose(1, 2);
}

struct Call {
  int64_t batch, heads, kv_heads, queries, keys, width, padded;
  bool causal;
  float scale;
  int64_t distances() const { return std::max<int64_t>(queries + keys - 1, 0); }
};
Call call_of(const at::Tensor& q, const at::Tensor& k, bool causal, double scale) {
  const int64_t piece = 16 / (int64_t)q.element_size();
  return {q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3), round_up(q.size(3), piece), causal, (float)scale};
}
// the operands, laid out, and what the library takes of them
struct Operands {
  Heads q, k, v;
  at::Tensor bias, mask;
  gact_attention a{};
};
Operands operands_of(const Call& c, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& bias, const at::Tensor& mask,
                     const Place& at) {
  Operands o{heads_of(q, c.padded, at), heads_of(k, c.padded, at), heads_of(v, c.padded, at), bias, mask, {}};
  if (bias.defined()) o.bias = dense_of(bias);
  if (mask.defined() && c.keys > 1 && mask.stride(1) != 1) o.mask = mask.contiguous();
  o.a.dtype = dtype_code(q.scalar_type());
  o.a.causal = c.causal;
  o.a.batch = c.batch;
  o.a.heads = c.heads;
  o.a.kv_heads = c.kv_heads;
  o.a.queries = c.queries;
  o.a.keys = c.keys;
  o.a.width = c.padded;
  o.a.scale = c.scale;
  o.a.bias = (const float*)in(o.bias);
  o.a.mask = (const uint8_t*)in(o.mask);
  o.a.mask_stride = o.mask.defined() ? o.mask.stride(0) : 0;
  o.a.q = o.q.rows;
  o.a.k = o.k.rows;
  o.a.v = o.v.rows;
  return o;
}
// -> [batch, queries, heads, padded width]
at::Tensor forward(const Operands& o, const Call& c, at::ScalarType dtype, const at::Tensor& lse, const at::Tensor& rest, const Place& at) {
  const at::Tensor y = at.empty({c.batch, c.queries, c.heads, c.padded}, dtype);
  const at::Tensor ws = at.bytes(gact_attention_workspace_bytes(&o.a));
  const gact_rows rows = rows_of(y, true);
  check_status(gact_attention_forward(&o.a, &rows, (float*)out(lse), (int8_t*)out(rest), out(ws), at.stream));
  return y;
}

struct AttentionBackward : public Node {
  SavedVariable query, key, value, bias, mask, result, lse, rest;
  Call c{};
  at::ScalarType dtype = at::kFloat;
  bool has_bias = false, has_mask = false;
  // hooks for saved tensors may give back other values: probabilities from these and sums from those that were given would be no probabilities
  bool again_forward = false;
  // The bias of a call under hooks, which do not get it: in codes of few bits the values that hide a key would leave nothing of the others.
  at::Tensor held_bias;
  int64_t bias_version = 0;
  bool released = false;
  std::string name() const override { return "OpAttentionBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&query, &key, &value, &bias, &mask, &result, &lse, &rest}) give_up(*v);
    held_bias.reset();
    released = true;
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    variable_list results(4);
    const at::Tensor& dy = grads[0];
    if (!dy.defined()) return results;
    TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
    check_grad(dy);
    const at::Tensor q = again(query, dtype, {c.batch, c.heads, c.queries, c.width}, dy, false);
    const at::Tensor k = again(key, dtype, {c.batch, c.kv_heads, c.keys, c.width}, dy, false);
    const at::Tensor v = again(value, dtype, {c.batch, c.kv_heads, c.keys, c.width}, dy, false);
    at::Tensor b, m, y, l, r;
    if (held_bias.defined()) {
      TORCH_CHECK(held_bias._version() == bias_version, "the bias has been modified by an inplace operation since op_attention was given it");
      b = held_bias;
    } else if (has_bias) b = again(bias, at::kFloat, {c.heads, c.distances()}, dy, false);
    if (has_mask) m = again(mask, at::kBool, {c.batch, c.keys}, dy, false);
    if (!again_forward) {
      y = result.unpack(shared_from_this());
      l = again(lse, at::kFloat, {c.batch, c.heads, c.queries}, dy);
      if (dtype != at::kFloat) r = again(rest, at::kChar, {c.batch, c.queries, c.heads, c.padded}, dy);
    }
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const Place at(dy);
      const Operands o = operands_of(c, q, k, v, b, m, at);
      Heads kept;
      if (again_forward) {
        l = at.empty({c.batch, c.heads, c.queries}, at::kFloat);
        if (dtype != at::kFloat) r = at.empty({c.batch, c.queries, c.heads, c.padded}, at::kChar);
        kept.held = forward(o, c, dtype, l, r, at);
        kept.rows = rows_of(kept.held, true);
      } else {
        kept = heads_of(y, c.padded, at);
      }
      const Heads grad = heads_of(dy, c.padded, at);
      const bool need[3] = {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)};
      at::Tensor made[3];
      gact_rows rows[3];
      for (int i = 0; i < 3; i++) {
        if (!need[i]) continue;
        made[i] = at.empty({c.batch, i ? c.keys : c.queries, i ? c.kv_heads : c.heads, c.padded}, dtype);
        rows[i] = rows_of(made[i], true);
      }
      const bool need_bias = has_bias && task_should_compute_output(3);
      if (need_bias) results[3] = at.empty({c.heads, c.distances()}, at::kFloat);
      const at::Tensor ws = at.bytes(gact_attention_backward_workspace_bytes(&o.a, need_bias));
      check_status(gact_attention_backward(&o.a, &kept.rows, (const float*)in(l), (const int8_t*)in(r), &grad.rows, need[0] ? &rows[0] : nullptr, need[1] ? &rows[1] : nullptr,
                                           need[2] ? &rows[2] : nullptr, (float*)out(results[3]), out(ws), at.stream));
      for (int i = 0; i < 3; i++)
        if (need[i]) results[i] = result_of(made[i], c.width);
    }
    return once(std::move(results), "op_attention");
  }
};

at::Tensor attention(const at::Tensor& q_given, const at::Tensor& k_given, const at::Tensor& v_given, const std::optional<at::Tensor>& b_given,
                     const std::optional<at::Tensor>& mask, bool causal, const std::optional<double>& scale_given, const Autocast& autocast, bool hooked) {
  check_like(k_given, q_given, "key", autocast);
  check_like(v_given, q_given, "value", autocast);
  TORCH_CHECK(q_given.dim() == 4 && k_given.dim() == 4 && v_given.dim() == 4, "query, key and value must be [batch, heads, rows, width]");
  TORCH_CHECK(v_given.sizes() == k_given.sizes(), "value must have key's shape ", k_given.sizes(), ", got ", v_given.sizes());
  const int64_t heads = q_given.size(1), kv_heads = k_given.size(1), width = q_given.size(3);
  TORCH_CHECK(k_given.size(0) == q_given.size(0) && k_given.size(3) == width, "key must have query's batch and width, got ", k_given.sizes(), " for ",
              q_given.sizes());
  TORCH_CHECK(width >= 1 && width <= GACT_ATTENTION_MAX_WIDTH, "attention takes heads of 1 to ", GACT_ATTENTION_MAX_WIDTH, " values");
  TORCH_CHECK(heads >= 1 && heads <= 65535 && kv_heads >= 1 && heads % kv_heads == 0, "the number of query's heads must be a multiple of that of key's");
  TORCH_CHECK(q_given.size(2) <= GACT_ATTENTION_MAX_LENGTH && k_given.size(2) <= GACT_ATTENTION_MAX_LENGTH, "attention takes up to ",
              GACT_ATTENTION_MAX_LENGTH, " queries and keys");
  const double scale = scale_given ? *scale_given : 1.0 / std::sqrt((double)width);
  TORCH_CHECK((float)scale > 0.0f && std::isfinite((float)scale * 1.44269504f), "scale must be a positive number below 2.3e38");
  const int64_t distances = std::max<int64_t>(q_given.size(2) + k_given.size(2) - 1, 0);
  if (b_given) {
    TORCH_CHECK(autocast || b_given->scalar_type() == at::kFloat, "The type of bias is not correct!");
    TORCH_CHECK(b_given->device() == q_given.device(), "bias is on another device");
    TORCH_CHECK(b_given->dim() == 2 && b_given->size(0) == heads && b_given->size(1) == distances, "bias must be [heads, queries + keys - 1] = [", heads, ", ",
                distances, "], got ", b_given->sizes());
  }
  if (mask) {
    TORCH_CHECK(mask->device() == q_given.device(), "mask is on another device");
    TORCH_CHECK(mask->dim() == 2 && mask->size(0) == q_given.size(0) && mask->size(1) == k_given.size(2), "mask must be [batch, keys] = [", q_given.size(0), ", ",
                k_given.size(2), "], got ", mask->sizes());
  }
  for (const auto& t : {std::optional<at::Tensor>(q_given), std::optional<at::Tensor>(k_given), std::optional<at::Tensor>(v_given), b_given})
    no_tangent(t, "op_attention");
  const bool keep = torch::autograd::compute_requires_grad(q_given, k_given, v_given, b_given);
  if (keep) refuse_stale_leaves({&q_given, &k_given, &v_given, held(b_given)}, q_given);
  const at::Tensor q = cast(q_given, autocast), k = cast(k_given, autocast), v = cast(v_given, autocast);
  const std::optional<at::Tensor> bias = b_given ? std::optional<at::Tensor>(b_given->to(at::kFloat)) : b_given;
  const Call c = call_of(q, k, causal, scale);
  at::Tensor y, lse, rest;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Place at(q);
    const Operands o = operands_of(c, q, k, v, bias ? *bias : at::Tensor(), mask ? *mask : at::Tensor(), at);
    if (keep && !hooked) {
      lse = at.empty({c.batch, c.heads, c.queries}, at::kFloat);
      if (q.scalar_type() != at::kFloat) rest = at.empty({c.batch, c.queries, c.heads, c.padded}, at::kChar);
    }
    y = result_of(forward(o, c, q.scalar_type(), lse, rest, at), c.width);
  }
  if (keep) {
    const std::shared_ptr<AttentionBackward> node(new AttentionBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, k, v, bias));
    node->c = c;
    node->dtype = q.scalar_type();
    node->has_bias = bias.has_value();
    node->has_mask = mask.has_value();
    node->again_forward = hooked;
    node->query = SavedVariable(q, false);
    node->key = SavedVariable(k, false);
    node->value = SavedVariable(v, false);
    if (bias && hooked) {
      TORCH_CHECK(!bias->is_inference(), "Inference tensors cannot be saved for backward. To work around you can make a clone to get a normal tensor and use it in autograd.");
      node->held_bias = bias->detach();
      node->bias_version = bias->_version();
    } else if (bias) {
      node->bias = SavedVariable(*bias, false);
    }
    if (mask) node->mask = SavedVariable(*mask, false);
    torch::autograd::set_history(y, node);
    if (!hooked) {
      node->result = SavedVariable(y, true);
      node->lse = SavedVariable(lse, false);
      if (rest.defined()) node->rest = SavedVariable(rest, false);
    }
  }
  return y;
}

// ---- the position bias ----
struct Distances {
  int64_t buckets, heads, queries, keys, most;
  bool both;
};
struct PositionBiasBackward : public Node {
  Distances d{};
  at::ScalarType dtype = at::kFloat;
  std::string name() const override { return "OpPositionBiasBackward"; }
  variable_list apply(variable_list&& grads) override {
    variable_list results(1);
    if (!grads[0].defined() || !task_should_compute_output(0)) return results;
    check_grad(grads[0]);
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const Place at(grads[0]);
      const at::Tensor grad = dense_of(grads[0]);
      results[0] = at.empty({d.buckets, d.heads}, dtype);
      check_status(gact_position_bias_backward((const float*)in(grad), dtype_code(dtype), d.buckets, d.heads, d.queries, d.keys, d.both, d.most,
                                               out(results[0]), at.stream));
    }
    return once(std::move(results), "op_position_bias");
  }
};
at::Tensor position_bias(const at::Tensor& table, Distances d) {
  TORCH_CHECK(table.dim() == 2, "table must be [buckets, heads]");
  d.buckets = table.size(0);
  d.heads = table.size(1);
  TORCH_CHECK(d.queries >= 1 && d.queries <= GACT_ATTENTION_MAX_LENGTH && d.keys >= 1 && d.keys <= GACT_ATTENTION_MAX_LENGTH, "the position bias takes 1 to ",
              GACT_ATTENTION_MAX_LENGTH, " queries and keys");
  TORCH_CHECK(d.heads >= 1 && d.heads <= 65535 && d.buckets <= GACT_MAX_BUCKETS && d.buckets >= (d.both ? 4 : 2) && (!d.both || d.buckets % 2 == 0),
              "the position bias takes 1 to 65535 heads and 2 to ", GACT_MAX_BUCKETS, " buckets, an even number and 4 at least where it is bidirectional");
  TORCH_CHECK(d.most > (d.both ? d.buckets / 4 : d.buckets / 2) && d.most <= GACT_ATTENTION_MAX_LENGTH, "max_distance must be above ",
              d.both ? d.buckets / 4 : d.buckets / 2, " for ", d.buckets, " buckets, and at most ", GACT_ATTENTION_MAX_LENGTH);
  no_tangent(table, "op_position_bias");
  const bool keep = torch::autograd::compute_requires_grad(table);
  if (keep) refuse_stale_leaves({&table}, table);
  at::Tensor bias;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Place at(table);
    const at::Tensor t = dense_of(table);
    bias = at.empty({d.heads, d.queries + d.keys - 1}, at::kFloat);
    check_status(gact_position_bias(in(t), dtype_code(t.scalar_type()), d.buckets, d.heads, d.queries, d.keys, d.both, d.most, (float*)out(bias), at.stream));
  }
  if (keep) {
    const std::shared_ptr<PositionBiasBackward> node(new PositionBiasBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(table));
    node->d = d;
    node->dtype = table.scalar_type();
    torch::autograd::set_history(bias, node);
  }
  return bias;
}

// ---- what Python calls ----
// attention(query, key, value, bias or None, mask or None, causal, scale or None, autocast's type or None) -> result
PyObject* py_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 8, kAttention);
  const at::Tensor &q = tensor_of(args[0], "query"), &k = tensor_of(args[1], "key"), &v = tensor_of(args[2], "value");
  const std::optional<at::Tensor> bias = tensor_or_none(args[3], "bias");
  std::optional<at::Tensor> mask;
  if (args[4] != Py_None) {
    TORCH_CHECK_TYPE(THPVariable_Check(args[4]), "mask must be a tensor");
    mask = THPVariable_Unpack(args[4]);
    TORCH_CHECK(mask->defined() && mask->is_cuda(), "mask must be a CUDA tensor!");
    TORCH_CHECK(plain(*mask), "mask must be a plain dense tensor");
    TORCH_CHECK(mask->scalar_type() == at::kBool, "The type of mask is not correct!");
  }
  const int causal = PyObject_IsTrue(args[5]);
  if (causal < 0) throw python_error();
  std::optional<double> scale;
  if (args[6] != Py_None) scale = number_of(args[6]);
  const Autocast autocast = autocast_of(args[7]);
  const bool hooked = at::SavedTensorDefaultHooks::get_hooks().has_value();
  return THPVariable_Wrap(without_gil([&] { return attention(q, k, v, bias, mask, causal != 0, scale, autocast, hooked); }));
  END_HANDLE_TH_ERRORS
}

// position_bias(table, queries, keys, bidirectional, max_distance) -> bias
PyObject* py_position_bias(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 5, kBias);
  const at::Tensor& table = tensor_of(args[0], "table");
  const int both = PyObject_IsTrue(args[3]);
  if (both < 0) throw python_error();
  const Distances d{0, 0, integer_of(args[1]), integer_of(args[2]), integer_of(args[4]), both != 0};
  return THPVariable_Wrap(without_gil([&] { return position_bias(table, d); }));
  END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef gact_attention_methods[] = {FASTCALL("attention", py_attention), FASTCALL("position_bias", py_position_bias), {nullptr, nullptr, 0, nullptr}};
