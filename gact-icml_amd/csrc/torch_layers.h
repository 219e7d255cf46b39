// What the two files of gact_torch.so share.
#pragma once
#include <torch/csrc/python_headers.h>

#include <ATen/core/Tensor.h>

// no mode, transform or trace of torch's around the call
bool gact_torch_ordinary();
// torch.empty on the GPU without the dispatcher's way there; for ordinary calls
at::Tensor gact_torch_empty(c10::IntArrayRef shape, at::ScalarType dtype, c10::Device device);
// the layers' functions, which the module takes beside its own
extern PyMethodDef gact_layer_methods[];
