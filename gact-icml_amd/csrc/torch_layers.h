// What the two files of gact_torch.so share.
#pragma once
#include <torch/csrc/python_headers.h>

#include <ATen/core/Tensor.h>

// a mode, transform or trace of torch's around the call that acts on the dispatcher's operators
bool gact_torch_dispatched();
// neither that nor a mode that acts on torch's functions
bool gact_torch_ordinary();
// torch.empty on the GPU without the dispatcher's way there; for ordinary calls
at::Tensor gact_torch_empty(c10::IntArrayRef shape, at::ScalarType dtype, c10::Device device);
// The GIL is released as long as this lives, and is back before an exception that leaves its scope becomes one of Python's
struct WithoutGil {
  PyThreadState* const state = PyEval_SaveThread();
  WithoutGil() = default;
  WithoutGil(const WithoutGil&) = delete;
  ~WithoutGil() { PyEval_RestoreThread(state); }
};
// the layers' functions, which the module takes beside its own
extern PyMethodDef gact_layer_methods[];
