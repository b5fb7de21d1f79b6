// What the operator files (torch_*.cpp) share.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include <initializer_list>

#include "../../include/trifast_b200.h"

namespace trifast_torch {

int32_t dtype_code(at::ScalarType t);
// A failed call of the C ABI as an exception.
void check_rc(int rc, const char* what);
// First thing in every call: if an earlier kernel on this device gave up on one of its
// bounded waits, its outputs (and those of every launch since) were never written.  Costs one
// read of host memory when nothing is wrong.
void raise_if_device_gave_up(c10::DeviceIndex dev, cudaStream_t stream);
// In the autograd kernels: an input with a tangent is refused, since no operator has a forward-mode derivative and all of
// them run below autograd, where it would be lost without a word.
void refuse_tangents(const char* op, std::initializer_list<const at::Tensor*> inputs);

}  // namespace trifast_torch
