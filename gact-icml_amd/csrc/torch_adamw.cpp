// The host side of AdamW's step over many tensors: arguments, gradients in their parameter's order of memory, launches.
#include "torch_common.h"

#include <ATen/ops/empty_strided.h>

#include <map>
#include <tuple>
#include <vector>

namespace {

const char* const kAdamw = "AdamW's step";

// the items of a list or tuple
struct Items {
  PyObject* held;
  explicit Items(PyObject* o, const char* name) : held(o) {
    TORCH_CHECK_TYPE(PyList_Check(o) || PyTuple_Check(o), name, " must be a list or tuple");
  }
  Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(held); }
  PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(held, i); }
};
const at::Tensor& state_tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  TORCH_CHECK(t.defined() && t.is_cuda(), name, " must be a CUDA tensor!");
  TORCH_CHECK(plain(t) && !t.is_neg(), name, " must be a plain dense tensor");
  return t;
}
bool same_places(const at::Tensor& a, const at::Tensor& b) {     // whether equal indices are equal places in memory
  if (a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); d++)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

struct State {
  at::Tensor m, v, scale;
  bool codes() const { return scale.defined(); }
};
// a state's (exp_avg, exp_avg_sq, scale or None), its parts made sure to belong together
State state_of(PyObject* o) {
  TORCH_CHECK_TYPE((PyTuple_Check(o) || PyList_Check(o)) && PySequence_Fast_GET_SIZE(o) == 3, "a state must be an AdamWState");
  const Items items(o, "a state");
  State s;
  s.m = state_tensor(items[0], "exp_avg");
  s.v = state_tensor(items[1], "exp_avg_sq");
  if (items[2] != Py_None) s.scale = state_tensor(items[2], "scale");
  const bool codes = s.codes();
  TORCH_CHECK(s.m.scalar_type() == (codes ? at::kChar : at::kFloat), "The type of exp_avg is not correct!");
  TORCH_CHECK(s.v.scalar_type() == (codes ? at::kByte : at::kFloat), "The type of exp_avg_sq is not correct!");
  TORCH_CHECK(s.m.is_non_overlapping_and_dense() && same_places(s.m, s.v), "exp_avg and exp_avg_sq must be dense and of one layout");
  TORCH_CHECK(s.m.device() == s.v.device() && (!codes || s.m.device() == s.scale.device()), "a state's tensors are on different devices");
  if (codes) {
    TORCH_CHECK(s.scale.scalar_type() == at::kFloat, "The type of scale is not correct!");
    const int64_t groups = (s.m.numel() + 255) / 256;
    TORCH_CHECK(s.scale.dim() == 2 && s.scale.size(0) == groups && s.scale.size(1) == 2 && s.scale.is_contiguous(), "scale must be a contiguous [", groups, ", 2]");
  }
  TORCH_CHECK(s.m.numel() == 0 || (aligned(in(s.m)) && aligned(in(s.v)) && (!codes || (uintptr_t)in(s.scale) % 8 == 0)),
              "a state's tensors must begin at multiples of 16 bytes");
  return s;
}

// Memory that a launch touches: what is written must be nobody else's
struct Range {
  uintptr_t begin, end;
  bool written;
};
void add_range(std::vector<Range>& ranges, const at::Tensor& t, bool written) {
  if (!t.defined() || t.numel() == 0) return;
  const uintptr_t begin = (uintptr_t)in(t);
  ranges.push_back({begin, begin + (uintptr_t)(t.numel() * (int64_t)t.element_size()), written});
}
void refuse_overlaps(std::vector<Range>& ranges) {
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;
  for (const Range& r : ranges) {
    TORCH_CHECK(r.begin >= written && !(r.written && r.begin < any), "parameters, gradients and states must not share memory");
    any = std::max(any, r.end);
    if (r.written) written = std::max(written, r.end);
  }
}
void changed(const at::Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// a number, or where on the GPU it is
template <typename N>
struct NumberAt {
  N value{};
  at::Tensor at;
};
template <typename N>
NumberAt<N> number_at(PyObject* o, const char* name, at::ScalarType type) {
  NumberAt<N> n;
  if (THPVariable_Check(o)) {
    n.at = state_tensor(o, name);
    TORCH_CHECK(n.at.numel() == 1 && n.at.scalar_type() == type, name, " must be one ", type, " where it is a tensor");
  } else if constexpr (std::is_same<N, double>::value) {
    n.value = number_of(o);
  } else {
    n.value = integer_of(o);
  }
  return n;
}

struct One {
  at::Tensor p, g;
  State state;
};

void step_all(std::vector<One>& all, const NumberAt<int64_t>& step, const NumberAt<double>& lr, gact_adamw_options options) {
  const at::AutoDispatchBelowADInplaceOrView below;
  // per device, type and kind of state, in the order of the list
  std::map<std::tuple<c10::DeviceIndex, int, int>, std::vector<One*>> kinds;
  std::vector<Range> ranges;
  for (One& o : all) {
    if (o.p.numel() == 0) continue;
    for (const at::Tensor* t : {&step.at, &lr.at})
      TORCH_CHECK(!t->defined() || t->device() == o.p.device(), "step and lr, where they are tensors, must be on the parameters' device");
    kinds[{o.p.device().index(), dtype_code(o.p.scalar_type()), o.state.codes() ? 8 : 32}].push_back(&o);
    add_range(ranges, o.p, true);
    add_range(ranges, o.state.m, true);
    add_range(ranges, o.state.v, true);
    add_range(ranges, o.state.scale, true);
    if (!o.g.is_neg() && same_places(o.g, o.p)) add_range(ranges, o.g, false);
  }
  refuse_overlaps(ranges);
  for (const auto& kind : kinds) {
    const Place at(kind.second[0]->p);
    options.step = step.value;
    options.lr = lr.value;
    options.step_at = (const int64_t*)in(step.at);
    options.lr_at = (const float*)in(lr.at);
    std::vector<gact_adamw_tensor> tensors;
    tensors.reserve(kind.second.size());
    for (One* o : kind.second) {
      if (o->g.is_neg() || !same_places(o->g, o->p)) {
        const at::Tensor like = at::empty_strided(o->p.sizes(), o->p.strides(), o->p.options());
        like.copy_(o->g);
        o->g = like;
      }
      tensors.push_back({out(o->p), in(o->g), out(o->state.m), out(o->state.v), (float*)out(o->state.scale), o->p.numel()});
    }
    check_status(gact_adamw(tensors.data(), (int64_t)tensors.size(), std::get<1>(kind.first), std::get<2>(kind.first), &options, at.stream));
  }
  for (const One& o : all)
    for (const at::Tensor* t : {&o.p, &o.state.m, &o.state.v, &o.state.scale}) changed(*t);
}

// ---- what Python calls ----
// adamw(params, grads, states, step, lr, beta1, beta2, eps, weight_decay)
PyObject* py_adamw(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 9, kAdamw);
  const Items params(args[0], "params"), grads(args[1], "grads"), states(args[2], "states");
  TORCH_CHECK(grads.size() == params.size() && states.size() == params.size(), "as many grads and states as params are expected");
  const NumberAt<int64_t> step = number_at<int64_t>(args[3], "step", at::kLong);
  const NumberAt<double> lr = number_at<double>(args[4], "lr", at::kFloat);
  gact_adamw_options options{};
  options.beta1 = number_of(args[5]);
  options.beta2 = number_of(args[6]);
  options.eps = number_of(args[7]);
  options.decay = number_of(args[8]);
  TORCH_CHECK(step.at.defined() || step.value >= 1, "step counts from 1 on");
  TORCH_CHECK((lr.at.defined() || (lr.value >= 0.0 && std::isfinite(lr.value))) && options.eps >= 0.0 && std::isfinite(options.eps) && options.decay >= 0.0 &&
                  std::isfinite(options.decay) && options.beta1 >= 0.0 && options.beta1 < 1.0 && options.beta2 >= 0.0 && options.beta2 < 1.0,
              "lr, eps and weight_decay must be 0 or more, and the betas from 0 to below 1");
  std::vector<One> all((size_t)params.size());
  for (Py_ssize_t i = 0; i < params.size(); i++) {
    One& o = all[(size_t)i];
    o.p = tensor_of(params[i], "a parameter");
    o.g = tensor_of(grads[i], "a gradient");
    TORCH_CHECK(!o.p.is_neg() && o.p.is_non_overlapping_and_dense(), "a parameter must be dense in memory");
    TORCH_CHECK(o.p.is_leaf(), "a parameter must be a leaf");
    TORCH_CHECK(o.g.sizes() == o.p.sizes() && o.g.scalar_type() == o.p.scalar_type() && o.g.device() == o.p.device(),
                "a gradient must have its parameter's shape, type and device");
    o.state = state_of(states[i]);
    TORCH_CHECK(same_places(o.state.m, o.p) && o.state.m.device() == o.p.device(), "a state must have its parameter's shape, layout and device");
  }
  without_gil([&] {
    step_all(all, step, lr, options);
    return 0;
  });
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// adamw_values(states in 8 bits) -> (exp_avg, exp_avg_sq)
PyObject* py_adamw_values(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 1, kAdamw);
  const Items states(args[0], "states");
  TORCH_CHECK(states.size() > 0, "a state at least is expected");
  std::vector<State> all;
  std::vector<gact_adamw_tensor> tensors;
  int64_t total = 0;
  for (Py_ssize_t i = 0; i < states.size(); i++) {
    all.push_back(state_of(states[i]));
    const State& s = all.back();
    TORCH_CHECK(s.codes(), "states in 8 bits are expected");
    TORCH_CHECK(s.m.device() == all[0].m.device(), "the states are on different devices");
    tensors.push_back({nullptr, nullptr, const_cast<void*>(in(s.m)), const_cast<void*>(in(s.v)), (float*)const_cast<void*>(in(s.scale)), s.m.numel()});
    total += s.m.numel();
  }
  at::Tensor made[2];
  without_gil([&] {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Place at(all[0].m);
    for (at::Tensor& t : made) t = at.empty({total}, at::kFloat);
    check_status(gact_adamw_values(tensors.data(), (int64_t)tensors.size(), (float*)out(made[0]), (float*)out(made[1]), at.stream));
    return 0;
  });
  PyObject* const pair = PyTuple_New(2);
  if (!pair) return nullptr;
  for (Py_ssize_t i = 0; i < 2; i++) {
    PyObject* const w = THPVariable_Wrap(made[i]);
    if (!w) {
      Py_DECREF(pair);
      return nullptr;
    }
    PyTuple_SET_ITEM(pair, i, w);
  }
  return pair;
  END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef gact_adamw_methods[] = {FASTCALL("adamw", py_adamw), FASTCALL("adamw_values", py_adamw_values), {nullptr, nullptr, 0, nullptr}};
