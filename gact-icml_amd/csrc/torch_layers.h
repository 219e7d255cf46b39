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
// the layers' functions, which the module takes beside its own
extern PyMethodDef gact_layer_methods[];
