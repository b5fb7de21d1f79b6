// What the operator files (torch_*.cpp) share.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include "../../include/trifast_b200.h"

namespace trifast_torch {

int32_t dtype_code(at::ScalarType t);
// A failed call of the C ABI as an exception.
void check_rc(int rc, const char* what);
// First thing in every call: if an earlier kernel on this device gave up on one of its
// bounded waits, its outputs (and those of every launch since) were never written.  Costs one
// read of host memory when nothing is wrong.
void raise_if_device_gave_up(c10::DeviceIndex dev, cudaStream_t stream);

}  // namespace trifast_torch
