// The host side of the layers that train on 8-bit checkpoints: arguments, copies where a layout needs one, results, launches, and the
// autograd nodes, whose backward passes run without Python.  A call that cannot be taken is refused here, with the reason.
#include <torch/csrc/python_headers.h>

#include <ATen/EmptyTensor.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <cstdint>
#include <memory>
#include <mutex>
#include <string>

#include "gact_hip.h"
#include "torch_layers.h"

namespace {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

constexpr int64_t kGroup = 256;
constexpr int64_t kLargeWeights = (int64_t)16 << 20;      // bytes

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return GACT_F32;
    case at::kHalf: return GACT_F16;
    case at::kBFloat16: return GACT_BF16;
    default: return -1;
  }
}

void check_status(int rc) { TORCH_CHECK(rc == GACT_OK, "gact: ", gact_strerror(rc)); }

c10::DispatchKeySet wrapped_keys() {
  return c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::ZeroTensor,
                              c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper});
}
bool plain(const at::Tensor& t) { return t.layout() == at::kStrided && t.has_storage() && !t.key_set().has_any(wrapped_keys()); }
// a tensor (or parameter) itself, no subclass and no wrapper, dense on the GPU
const at::Tensor& tensor_of(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  TORCH_CHECK(t.defined() && t.is_cuda(), name, " must be a CUDA tensor!");
  TORCH_CHECK(plain(t), name, " must be a plain dense tensor");
  TORCH_CHECK(dtype_code(t.scalar_type()) >= 0, "The type of ", name, " is not correct!");
  return t;
}
std::optional<at::Tensor> tensor_or_none(PyObject* o, const char* name) {
  if (o == Py_None) return std::nullopt;
  return tensor_of(o, name);
}
// The type that autocast runs an operator in; its arguments may then be of others
using Autocast = std::optional<at::ScalarType>;
void check_like(const at::Tensor& t, const at::Tensor& like, const char* name, const Autocast& autocast) {
  TORCH_CHECK(autocast || t.scalar_type() == like.scalar_type(), "The type of ", name, " is not correct!");
  TORCH_CHECK(t.device() == like.device(), name, " is on another device");
}
void check_vector(const std::optional<at::Tensor>& t, const char* name, int64_t size, const at::Tensor& like, const Autocast& autocast) {
  if (!t) return;
  check_like(*t, like, name, autocast);
  TORCH_CHECK(t->dim() == 1 && t->size(0) == size, "The dimension of ", name, " is not correct!");
}
// the argument as autocast's operators take it, differentiably
at::Tensor cast(const at::Tensor& t, const Autocast& autocast) { return autocast ? t.to(*autocast) : t; }
std::optional<at::Tensor> cast(const std::optional<at::Tensor>& t, const Autocast& autocast) {
  return t && autocast ? std::optional<at::Tensor>(t->to(*autocast)) : t;
}

// Everything a call needs to know about where it runs
struct Place {
  c10::Device device;
  c10::DeviceGuard guard;
  void* stream;
  bool ordinary;
  explicit Place(const at::Tensor& t)
      : device(t.device()), guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()), ordinary(gact_torch_ordinary()) {}
  at::Tensor empty(c10::IntArrayRef shape, at::ScalarType dtype) const {
    if (ordinary) return gact_torch_empty(shape, dtype, device);
    return at::empty(shape, at::TensorOptions().dtype(dtype).device(device));
  }
  at::Tensor bytes(int64_t size) const { return size ? empty({size}, at::kByte) : at::Tensor(); }
  at::Tensor zeros(c10::IntArrayRef shape, at::ScalarType dtype) const {
    return at::zeros(shape, at::TensorOptions().dtype(dtype).device(device));
  }
};
const void* in(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// A tensor as rows of its last dimension whose columns lie side by side, `ld` elements from one row to the next
struct Rows {
  at::Tensor held;
  int64_t rows = 0, cols = 0, ld = 0;
  const void* data() const { return in(held); }
};
Rows rows_of(const at::Tensor& tensor, const char* name, int64_t most = GACT_LAYER_MAX_COLS) {
  TORCH_CHECK(tensor.dim() >= 1, "The dimension of ", name, " is not correct!");
  Rows r;
  r.cols = tensor.size(-1);
  TORCH_CHECK(r.cols > 0 && r.cols <= most, name, " has ", r.cols, " columns: 1 to ", most, " are taken");
  r.rows = tensor.numel() / r.cols;
  TORCH_CHECK(r.rows <= GACT_LAYER_MAX_ROWS, name, " has more than ", GACT_LAYER_MAX_ROWS, " rows");
  r.held = tensor.is_neg() ? tensor.resolve_neg() : tensor;
  r.ld = r.cols;
  if (r.rows == 0 || r.held.is_contiguous()) return r;
  if (r.held.dim() != 2) r.held = r.held.reshape({r.rows, r.cols});       // a view where the strides allow it
  const bool beside = r.held.stride(1) == 1 || r.cols == 1;
  if (beside && r.rows == 1) return r;
  if (beside && r.held.stride(0) >= r.cols && r.held.stride(0) <= 4 * GACT_LAYER_MAX_COLS)
    r.ld = r.held.stride(0);
  else
    r.held = r.held.contiguous();
  return r;
}
int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// rows as the products load them: 16-byte aligned and whole 16-byte pieces
Rows product_rows(const Rows& r, const Place& at) {
  const int64_t piece = 16 / (int64_t)r.held.element_size();
  if (r.cols % piece == 0 && r.ld % piece == 0 && aligned(r.data())) return r;
  Rows padded = r;
  padded.ld = round_up(r.cols, 8);
  padded.held = at.empty({r.rows, padded.ld}, r.held.scalar_type());
  check_status(gact_pad_rows(r.data(), dtype_code(r.held.scalar_type()), r.rows, r.cols, r.ld, out(padded.held), padded.ld, at.stream));
  return padded;
}

struct Kept {     // a checkpoint's tensors
  at::Tensor codes, scale, mn;
};
Kept room_for(int64_t rows, int64_t cols, const Place& at) {
  const int64_t groups = (cols + kGroup - 1) / kGroup;
  return {at.empty({rows, round_up(cols, 16)}, at::kChar), at.empty({rows, groups}, at::kFloat), at.empty({rows, groups}, at::kFloat)};
}
Kept compress(const Rows& x, const Place& at) {
  Kept k = room_for(x.rows, x.cols, at);
  check_status(gact_checkpoint(x.data(), dtype_code(x.held.scalar_type()), x.rows, x.cols, x.ld, out(k.codes), k.codes.size(1),
                               (float*)out(k.scale), (float*)out(k.mn), at.stream));
  return k;
}
at::Tensor weight_product(const Rows& grad, const Kept& k, int64_t cols, at::ScalarType dtype, const Place& at) {
  if (grad.rows == 0) return at.zeros({grad.cols, cols}, dtype);
  const int code = dtype_code(dtype);
  const at::Tensor result = at.empty({grad.cols, cols}, dtype);
  const at::Tensor ws = at.bytes(gact_product_workspace_bytes(code, grad.cols, cols, grad.rows));
  check_status(gact_checkpoint_product(grad.data(), grad.ld, in(k.codes), k.codes.size(1), (const float*)in(k.scale), (const float*)in(k.mn),
                                       code, grad.rows, grad.cols, cols, out(result), out(ws), at.stream));
  return result;
}

at::Tensor dense(const std::optional<at::Tensor>& t) {
  if (!t) return at::Tensor();
  return t->is_contiguous() && !t->is_neg() ? *t : t->resolve_neg().contiguous();
}
void no_tangent(const std::optional<at::Tensor>& t, const char* operation) {
  TORCH_CHECK(!t.has_value() || !torch::autograd::isFwGradDefined(*t), operation, " has no forward-mode derivative");
}

// A leaf whose gradient's accumulator was made on the default stream - an eager graph of it is still alive - cannot be differentiated in a
// pass that is being captured: autograd would make the default stream wait for the capture, which the runtime answers by ending it, and
// torch by ending the process.
void refuse_stale_leaves(std::initializer_list<const at::Tensor*> tensors, const at::Tensor& like) {
  const c10::hip::HIPStream current = c10::hip::getCurrentHIPStream(like.device().index());
  hipStreamCaptureStatus status;
  if (current.stream() == nullptr || hipStreamIsCapturing(current.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  for (const at::Tensor* t : tensors) {
    if (!t || !t->requires_grad() || !t->is_leaf()) continue;
    const std::shared_ptr<Node> accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!accumulator) continue;
    const std::optional<c10::Stream> stream = accumulator->stream();
    TORCH_CHECK(!stream || stream->id() != 0,
                "a training pass is captured while an eager graph of one of its leaves, made on the default stream, is alive: drop it first");
  }
}
const at::Tensor* held(const std::optional<at::Tensor>& t) { return t ? &*t : nullptr; }

// results of a backward pass that is itself being differentiated: an error once somebody goes through them
variable_list once(variable_list grads, const char* name) {
  if (!c10::GradMode::is_enabled()) return grads;
  const auto stop = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice a function that was marked with @once_differentiable: ") + name, (int64_t)grads.size());
  for (at::Tensor& g : grads)      // the error's node hangs on tensors that need a gradient, which the result does through what was saved
    if (g.defined()) g = g.detach().set_requires_grad(true);
  return (*stop)(std::move(grads));
}
void give_up(SavedVariable& v) { v.reset_data(); }
// What was saved, as it was saved: hooks for saved tensors may give back anything, and the kernels would read it as if it were the same
at::Tensor again(SavedVariable& v, at::ScalarType dtype, c10::IntArrayRef shape, const at::Tensor& grad, bool dense = true) {
  const at::Tensor t = v.unpack();
  TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.scalar_type() == dtype && t.device() == grad.device() && t.sizes() == shape &&
                  (!dense || (t.is_contiguous() && !t.is_neg())),
              "the hooks for saved tensors gave back another tensor than they were given");
  return dense && !aligned(in(t)) ? t.clone() : t;      // a place in a larger buffer, say
}
Kept again(SavedVariable& codes, SavedVariable& scale, SavedVariable& mn, int64_t rows, int64_t cols, const at::Tensor& grad) {
  const int64_t groups = (cols + kGroup - 1) / kGroup;
  return {again(codes, at::kChar, {rows, round_up(cols, 16)}, grad), again(scale, at::kFloat, {rows, groups}, grad),
          again(mn, at::kFloat, {rows, groups}, grad)};
}
// a gradient that the kernels can read: no batch of them, no subclass
void check_grad(const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda() && plain(t), "the gradient must be a plain dense tensor");
}

// ---- layer norm ----
struct LayerNormBackward : public Node {
  SavedVariable weight, stats, codes, scale, mn;
  bool has_weight = false;
  bool released = false;
  std::string name() const override { return "OpLayerNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&weight, &stats, &codes, &scale, &mn}) give_up(*v);
    released = true;
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);      // what is saved is not released beside a pass that reads it
    variable_list result(3);
    if (!grads[0].defined()) return result;
    TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
    check_grad(grads[0]);
    const int64_t cols = grads[0].size(-1), rows = grads[0].numel() / cols;
    const at::Tensor w = has_weight ? again(weight, grads[0].scalar_type(), {cols}, grads[0], false) : at::Tensor();
    const at::Tensor st = again(stats, at::kFloat, {rows, 2}, grads[0]);
    const Kept k = again(codes, scale, mn, rows, cols, grads[0]);
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const Place at(grads[0]);
      const at::ScalarType dtype = grads[0].scalar_type();
      const Rows dy = rows_of(grads[0], "grad", GACT_NORM_MAX_COLS);
      const bool need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
      const at::Tensor dx = at.empty(grads[0].sizes(), dtype);
      at::Tensor dw, db;
      if (dy.rows == 0) {
        if (need_w) dw = at.zeros({dy.cols}, dtype);
        if (need_b) db = at.zeros({dy.cols}, dtype);
      } else {
        if (need_w) dw = at.empty({dy.cols}, dtype);
        if (need_b) db = at.empty({dy.cols}, dtype);
        const at::Tensor ws = need_w || need_b ? at.bytes(gact_norm_workspace_bytes(dy.rows, dy.cols)) : at::Tensor();
        const at::Tensor dense = w.defined() ? (w.is_neg() ? w.resolve_neg() : w).contiguous() : w;
        check_status(gact_norm_backward(dy.data(), dy.ld, in(dense), in(k.codes), k.codes.size(1), (const float*)in(k.scale), (const float*)in(k.mn),
                                        (const float*)in(st), dtype_code(dtype), dy.rows, dy.cols, out(dx), out(dw), out(db),
                                        (float*)out(ws), at.stream));
      }
      if (task_should_compute_output(0)) result[0] = dx;
      result[1] = dw;
      result[2] = db;
    }
    return once(std::move(result), "op_layer_norm");
  }
};

at::Tensor layer_norm(const at::Tensor& x_given, const std::optional<at::Tensor>& w_given, const std::optional<at::Tensor>& b_given, double eps,
                      const Autocast& autocast) {
  TORCH_CHECK(x_given.dim() >= 1 && x_given.size(-1) > 0 && x_given.size(-1) <= GACT_NORM_MAX_COLS, "layer norm takes 1 to ", GACT_NORM_MAX_COLS,
              " columns");
  const int64_t cols = x_given.size(-1);
  check_vector(w_given, "weight", cols, x_given, autocast);
  check_vector(b_given, "bias", cols, x_given, autocast);
  for (const auto& t : {std::optional<at::Tensor>(x_given), w_given, b_given}) no_tangent(t, "op_layer_norm");
  const bool keep = torch::autograd::compute_requires_grad(x_given, w_given, b_given);
  if (keep) refuse_stale_leaves({&x_given, held(w_given), held(b_given)}, x_given);
  const at::Tensor input = cast(x_given, autocast);
  const std::optional<at::Tensor> weight = cast(w_given, autocast), bias = cast(b_given, autocast);
  at::Tensor y;
  Kept k;
  at::Tensor stats;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Place at(input);
    const at::Tensor w = dense(weight), b = dense(bias);
    const Rows x = rows_of(input, "data", GACT_NORM_MAX_COLS);
    y = at.empty(input.sizes(), input.scalar_type());
    if (keep) {
      k = room_for(x.rows, cols, at);
      stats = at.empty({x.rows, 2}, at::kFloat);
    }
    check_status(gact_norm_forward(x.data(), x.ld, in(w), in(b), dtype_code(input.scalar_type()), x.rows, cols, (float)eps, out(y), out(k.codes),
                                   keep ? k.codes.size(1) : 0, (float*)out(k.scale), (float*)out(k.mn), (float*)out(stats), at.stream));
  }
  if (keep) {
    const std::shared_ptr<LayerNormBackward> node(new LayerNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(input, weight, bias));
    node->has_weight = weight.has_value();
    if (weight) node->weight = SavedVariable(*weight, false);
    node->stats = SavedVariable(stats, false);
    node->codes = SavedVariable(k.codes, false);
    node->scale = SavedVariable(k.scale, false);
    node->mn = SavedVariable(k.mn, false);
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- linear layers ----
struct LinearBackward : public Node {
  SavedVariable weight, codes, scale, mn, z_codes, z_scale, z_mn;
  int activation = GACT_ACT_NONE;
  int64_t inner = 0, outer = 0;
  at::ScalarType weight_dtype = at::kFloat;      // under autocast not the layer's type
  bool released = false;
  std::string name() const override { return "OpLinearBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&weight, &codes, &scale, &mn, &z_codes, &z_scale, &z_mn}) give_up(*v);
    released = true;
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    variable_list result(4);
    const at::Tensor& dy = grads[0];
    if (!dy.defined()) return result;
    TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
    const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
    if (task_should_compute_output(3)) result[3] = dy;
    check_grad(dy);
    const int64_t rows = dy.numel() / outer;
    at::Tensor w;
    Kept k, z;
    if (need_x) w = again(weight, weight_dtype, {outer, inner}, dy, false);
    if (need_w) k = again(codes, scale, mn, rows, inner, dy);
    if (activation != GACT_ACT_NONE && (need_x || need_w || need_b)) z = again(z_codes, z_scale, z_mn, rows, outer, dy);
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const Place at(dy);
      const at::ScalarType dtype = dy.scalar_type();
      const int code = dtype_code(dtype);
      const Rows g = rows_of(dy, "grad");
      c10::SmallVector<int64_t, 5> shape(dy.sizes().begin(), dy.sizes().end());
      shape.back() = inner;
      if (g.rows == 0) {
        if (need_x) result[0] = at.zeros(shape, dtype);
        if (need_w) result[1] = at.zeros({outer, inner}, weight_dtype);
        if (need_b) result[2] = at.zeros({outer}, dtype);
      } else {
        // dz: the gradient itself where there is no activation and the products can load it
        Rows dz = g;
        const int64_t piece = 16 / (int64_t)g.held.element_size();
        const bool fits = outer % piece == 0 && g.ld % piece == 0 && aligned(g.data());
        const bool own = (need_x || need_w) && (activation != GACT_ACT_NONE || !fits);
        if (own) {
          dz.ld = round_up(outer, 8);
          dz.held = at.empty({g.rows, dz.ld}, dtype);
        }
        if (need_b) result[2] = at.empty({outer}, dtype);
        if (own || need_b) {
          const at::Tensor ws = need_b ? at.bytes(gact_activation_workspace_bytes(g.rows, outer)) : at::Tensor();
          check_status(gact_activation_backward(g.data(), g.ld, in(z.codes), z.codes.defined() ? z.codes.size(1) : 0,
                                                (const float*)in(z.scale), (const float*)in(z.mn), activation, code, g.rows, outer,
                                                own ? out(dz.held) : nullptr, dz.ld, out(result[2]), (float*)out(ws), at.stream));
        }
        if (need_x) {
          const Rows held = product_rows(rows_of(w.to(dtype), "weight"), at);
          result[0] = at.empty(shape, dtype);
          const at::Tensor ws = at.bytes(gact_product_workspace_bytes(code, g.rows, inner, outer));
          check_status(gact_product(dz.data(), dz.ld, held.data(), held.ld, code, g.rows, outer, inner, out(result[0]), out(ws), at.stream));
        }
        if (need_w) result[1] = weight_product(dz, k, inner, dtype, at).to(weight_dtype);
      }
    }
    return once(std::move(result), "op_linear");
  }
};

// Under autocast the node saves the weight as it was given and rounds it again: a rounded copy would be memory of its own until the backward
// pass, and hooks for saved tensors that leave a model's parameters as they are would not know it
at::Tensor linear(const at::Tensor& x_given, const at::Tensor& weight, const std::optional<at::Tensor>& b_given, int activation,
                  const std::optional<at::Tensor>& r_given, const Autocast& autocast) {
  check_like(weight, x_given, "weight", autocast);
  TORCH_CHECK(x_given.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x_given.size(-1), "weight must be [outer, ",
              x_given.dim() ? std::to_string(x_given.size(-1)) : std::string("-"), "], got ", weight.sizes());
  const int64_t outer = weight.size(0), inner = weight.size(1);
  TORCH_CHECK(inner > 0 && inner <= GACT_LAYER_MAX_COLS && outer > 0 && outer <= GACT_LAYER_MAX_COLS, "a linear layer takes 1 to ",
              GACT_LAYER_MAX_COLS, " columns on either side");
  check_vector(b_given, "bias", outer, x_given, autocast);
  c10::SmallVector<int64_t, 5> shape(x_given.sizes().begin(), x_given.sizes().end());
  shape.back() = outer;
  if (r_given) {
    check_like(*r_given, x_given, "residual", autocast);
    TORCH_CHECK(r_given->sizes() == c10::IntArrayRef(shape), "residual must have the result's shape ", c10::IntArrayRef(shape));
  }
  for (const auto& t : {std::optional<at::Tensor>(x_given), std::optional<at::Tensor>(weight), b_given, r_given}) no_tangent(t, "op_linear");
  const bool needs = torch::autograd::compute_requires_grad(x_given, weight, b_given, r_given);
  if (needs) refuse_stale_leaves({&x_given, &weight, held(b_given), held(r_given)}, x_given);
  const at::Tensor input = cast(x_given, autocast);
  const std::optional<at::Tensor> bias = cast(b_given, autocast), residual = cast(r_given, autocast);
  const bool keep_x = needs && weight.requires_grad();
  const bool keep_z = needs && activation != GACT_ACT_NONE && torch::autograd::compute_requires_grad(input, weight, bias);
  at::Tensor y;
  Kept k, z;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Place at(input);
    const at::ScalarType dtype = input.scalar_type();
    const at::Tensor b = dense(bias);
    const Rows x = rows_of(input, "data");
    y = at.empty(shape, dtype);
    if (keep_z) z = room_for(x.rows, outer, at);
    if (keep_x) k = x.rows ? compress(x, at) : room_for(0, inner, at);
    if (x.rows) {
      Rows a = x, w = rows_of(weight.to(dtype), "weight"), r;
      int64_t depth = inner;
      // unaligned rows: few of them go to the kernel as they are where that costs less than copies of both operands (64 rows, 8191 to 8192: halves
      // 246 us as they are, 94 copied, floats 205 and 190; 37 rows, 4095 to 4096: 46 and 30, 44 and 51; 17 rows, 771 to 1285: 6 as they are, and a
      // copy is a launch of 4).  Up to 16 rows never: 8191 to 8192 98 and 74 us, no more than the copies for 64 rows
      if (x.rows > GACT_LINEAR_FEW_ROWS || (x.rows > 16 && inner * outer * (int64_t)input.element_size() >= kLargeWeights)) {
        a = product_rows(a, at);
        w = product_rows(w, at);
        depth = round_up(inner, 16 / (int64_t)a.held.element_size());      // behind the last column both are padded copies with zeros
      }
      if (residual) r = rows_of(*residual, "residual");
      const at::Tensor ws = at.bytes(gact_linear_workspace_bytes(dtype_code(dtype), x.rows, depth, outer, keep_z));
      check_status(gact_linear(a.data(), a.ld, w.data(), w.ld, in(b), residual ? r.data() : nullptr, r.ld, activation, dtype_code(dtype),
                               x.rows, depth, outer, out(y), out(z.codes), keep_z ? z.codes.size(1) : 0, (float*)out(z.scale),
                               (float*)out(z.mn), out(ws), at.stream));
    }
  }
  if (needs) {
    const std::shared_ptr<LinearBackward> node(new LinearBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(input, weight, bias, residual));
    node->activation = activation;
    node->inner = inner;
    node->outer = outer;
    node->weight_dtype = weight.scalar_type();
    if (input.requires_grad()) node->weight = SavedVariable(weight, false);
    if (keep_x) {
      node->codes = SavedVariable(k.codes, false);
      node->scale = SavedVariable(k.scale, false);
      node->mn = SavedVariable(k.mn, false);
    }
    if (keep_z) {
      node->z_codes = SavedVariable(z.codes, false);
      node->z_scale = SavedVariable(z.scale, false);
      node->z_mn = SavedVariable(z.mn, false);
    }
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- what Python calls ----
// the operator itself: its allocations and launches may wait for the GPU, and other threads of Python's go on meanwhile
template <typename F>
auto without_gil(const F& call) {
  const WithoutGil released;
  return call();
}
double number_of(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int64_t integer_of(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
// How many there are, and that no trace is being recorded: of these operators it would hold the results' allocations and nothing that fills them
void arguments(Py_ssize_t n, Py_ssize_t wanted) {
  TORCH_CHECK_TYPE(n == wanted, "expected ", wanted, " arguments, got ", n);
  TORCH_CHECK(!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer), "the layers on 8-bit checkpoints cannot be traced");
}

Autocast autocast_of(PyObject* o) {
  if (o == Py_None) return std::nullopt;
  TORCH_CHECK_TYPE(THPDtype_Check(o), "a type is expected");
  const at::ScalarType t = ((THPDtype*)o)->scalar_type;
  TORCH_CHECK(dtype_code(t) >= 0, "autocast's type is not correct");
  return t;
}

// layer_norm(x, weight or None, bias or None, eps, autocast's type or None) -> y
PyObject* py_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 5);
  const double eps = number_of(args[3]);
  const at::Tensor& x = tensor_of(args[0], "data");
  const std::optional<at::Tensor> weight = tensor_or_none(args[1], "weight"), bias = tensor_or_none(args[2], "bias");
  const Autocast autocast = autocast_of(args[4]);
  return THPVariable_Wrap(without_gil([&] { return layer_norm(x, weight, bias, eps, autocast); }));
  END_HANDLE_TH_ERRORS
}

// linear(x, weight, bias or None, activation's number, residual or None, autocast's type or None) -> y
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 6);
  const int64_t act = integer_of(args[3]);
  TORCH_CHECK(act >= GACT_ACT_NONE && act <= GACT_ACT_SILU, "unknown activation");
  const at::Tensor& x = tensor_of(args[0], "data");
  const at::Tensor& weight = tensor_of(args[1], "weight");
  const std::optional<at::Tensor> bias = tensor_or_none(args[2], "bias"), residual = tensor_or_none(args[4], "residual");
  const Autocast autocast = autocast_of(args[5]);
  return THPVariable_Wrap(without_gil([&] { return linear(x, weight, bias, (int)act, residual, autocast); }));
  END_HANDLE_TH_ERRORS
}

// takes(x, weight or None, bias or None, whether it is a linear layer and no layer norm, whether autocast is on) -> whether the operator runs
// these arguments: what it would refuse, and what a trace or a mode of torch's would not see, is for torch's own
PyObject* py_takes(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "expected 5 arguments, got ", n);
  const bool linear = args[3] == Py_True, autocast = args[4] == Py_True;
  if (gact_torch_dispatched()) Py_RETURN_FALSE;
  const at::Tensor* given[3] = {};
  for (int i = 0; i < 3; i++) {
    if (i && args[i] == Py_None) continue;
    if (!THPVariable_Check(args[i])) Py_RETURN_FALSE;
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    if (!t.defined() || !t.is_cuda() || !plain(t) || dtype_code(t.scalar_type()) < 0 || torch::autograd::isFwGradDefined(t)) Py_RETURN_FALSE;
    given[i] = &t;
    if (t.device() != given[0]->device() || (t.scalar_type() != given[0]->scalar_type() && !autocast)) Py_RETURN_FALSE;
  }
  const at::Tensor &x = *given[0], *const weight = given[1], *const bias = given[2];
  const int64_t most = linear ? GACT_LAYER_MAX_COLS : GACT_NORM_MAX_COLS;
  if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > most || x.numel() / x.size(-1) > GACT_LAYER_MAX_ROWS) Py_RETURN_FALSE;
  int64_t across = x.size(-1);
  if (linear) {
    if (!weight || weight->dim() != 2 || weight->size(1) != across || weight->size(0) < 1 || weight->size(0) > most) Py_RETURN_FALSE;
    across = weight->size(0);
  } else if (weight && (weight->dim() != 1 || weight->size(0) != across)) {
    Py_RETURN_FALSE;
  }
  if (bias && (bias->dim() != 1 || bias->size(0) != across)) Py_RETURN_FALSE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyObject* tuple_of(const Kept& k) {
  PyObject* const t = PyTuple_New(3);
  if (!t) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor* e : {&k.codes, &k.scale, &k.mn}) {
    PyObject* const w = THPVariable_Wrap(*e);
    if (!w) {
      Py_DECREF(t);
      return nullptr;
    }
    PyTuple_SET_ITEM(t, i++, w);
  }
  return t;
}

// checkpoint(x) -> (codes, scale, min)
PyObject* py_checkpoint(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 1);
  const at::Tensor& input = tensor_of(args[0], "data");
  return tuple_of(without_gil([&] {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Place at(input);
    const Rows x = rows_of(input, "data");
    return x.rows ? compress(x, at) : room_for(0, x.cols, at);
  }));
  END_HANDLE_TH_ERRORS
}

// a checkpoint's (codes, scale, min, shape, dtype) as Python holds it, its parts made sure to belong together
struct Given {
  Kept kept;
  c10::SmallVector<int64_t, 5> shape;
  int64_t rows = 1, cols = 0;
  at::ScalarType dtype;
};
Given given(PyObject* const* args) {
  Given g;
  TORCH_CHECK_TYPE(PyTuple_Check(args[3]) && THPDtype_Check(args[4]), "a Checkpoint is expected");
  g.dtype = ((THPDtype*)args[4])->scalar_type;
  for (Py_ssize_t d = 0; d < PyTuple_GET_SIZE(args[3]); d++) g.shape.push_back(integer_of(PyTuple_GET_ITEM(args[3], d)));
  TORCH_CHECK(!g.shape.empty() && g.shape.back() > 0 && g.shape.back() <= GACT_LAYER_MAX_COLS && dtype_code(g.dtype) >= 0,
              "the checkpoint's shape or type is not correct");
  g.cols = g.shape.back();
  for (size_t d = 0; d + 1 < g.shape.size(); d++)
    TORCH_CHECK(g.shape[d] >= 0 && !__builtin_mul_overflow(g.rows, g.shape[d], &g.rows), "the checkpoint's shape or type is not correct");
  const int64_t widths[3] = {round_up(g.cols, 16), (g.cols + kGroup - 1) / kGroup, (g.cols + kGroup - 1) / kGroup};
  const at::Tensor* first = nullptr;
  at::Tensor* const kept[3] = {&g.kept.codes, &g.kept.scale, &g.kept.mn};
  for (int i = 0; i < 3; i++) {
    TORCH_CHECK_TYPE(THPVariable_Check(args[i]), "a Checkpoint is expected");
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    if (!first) first = &t;
    TORCH_CHECK(t.defined() && t.is_cuda() && t.device() == first->device() && t.scalar_type() == (i ? at::kFloat : at::kChar) && t.dim() == 2 &&
                    t.size(0) == g.rows && t.size(1) == widths[i] && t.is_contiguous() && !t.is_neg() && (g.rows == 0 || aligned(in(t))),
                "the checkpoint's codes, scale or min do not belong to shape ", c10::IntArrayRef(g.shape));
    *kept[i] = t;
  }
  return g;
}

// restore(codes, scale, min, shape, dtype) -> tensor
PyObject* py_restore(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 5);
  const Given g = given(args);
  return THPVariable_Wrap(without_gil([&] {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Place at(g.kept.codes);
    const at::Tensor result = at.empty(g.shape, g.dtype);
    if (g.rows)
      check_status(gact_restore(in(g.kept.codes), g.kept.codes.size(1), (const float*)in(g.kept.scale), (const float*)in(g.kept.mn),
                                dtype_code(g.dtype), g.rows, g.cols, out(result), at.stream));
    return result;
  }));
  END_HANDLE_TH_ERRORS
}

// checkpoint_product(codes, scale, min, shape, dtype, grad) -> [outer, cols]
PyObject* py_checkpoint_product(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 6);
  const Given g = given(args);
  const at::Tensor& grad = tensor_of(args[5], "grad");
  TORCH_CHECK(grad.scalar_type() == g.dtype, "The type of grad is not correct!");
  TORCH_CHECK(grad.device() == g.kept.codes.device(), "grad is on another device");
  no_tangent(grad, "op_checkpoint_product");
  return THPVariable_Wrap(without_gil([&] {
    at::Tensor result;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const Place at(grad);
      Rows r = rows_of(grad, "grad");
      TORCH_CHECK(r.rows == g.rows, "grad has ", r.rows, " rows, the checkpoint ", g.rows);
      if (r.rows) r = product_rows(r, at);
      result = weight_product(r, g.kept, g.cols, g.dtype, at);
    }
    // no backward pass: the result of a gradient that has a history says so to who goes through it
    return torch::autograd::compute_requires_grad(grad) ? once({result}, "op_checkpoint_product")[0] : result;
  }));
  END_HANDLE_TH_ERRORS
}

#define FASTCALL(name, f) {name, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}

}  // namespace

PyMethodDef gact_layer_methods[] = {FASTCALL("layer_norm", py_layer_norm), FASTCALL("linear", py_linear), FASTCALL("takes", py_takes), FASTCALL("checkpoint", py_checkpoint),
                                    FASTCALL("restore", py_restore), FASTCALL("checkpoint_product", py_checkpoint_product),
                                    {nullptr, nullptr, 0, nullptr}};
