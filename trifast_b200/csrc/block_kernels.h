// Host interface of the memory-bound operators of a pair stack's blocks: layer_norm.cu and dropout_add.cu.
#pragma once

#include "common.cuh"

namespace trifast {

struct LayerNormArgs {
  const void *x, *dy, *weight, *bias;   // weight, bias: null for 1 and 0
  void *y, *dx, *dweight, *dbias;       // any of the gradients may be null
  int64_t rows, ld_x, ld_dy;            // rows of x and dy may be further apart than their width
  int width, dtype, affine_dtype;
  int classes;                          // set by the launcher
  float eps;
  float* partials;                      // layer_norm_workspace_floats()
};
// Whether rows `ld` elements apart begin at the same places of 16-byte pieces as dense ones: what the kernels take.
bool layer_norm_rows_fit(int64_t ld, int width, int dtype);
// Whether rows are too long for a block's registers.
bool layer_norm_in_passes(int width, int dtype);
// fp32 words of workspace that the gradients of weight and bias need.
int64_t layer_norm_workspace_floats(int64_t rows, int width, int dtype);
cudaError_t layer_norm_forward(const LayerNormArgs& a, cudaStream_t s);
cudaError_t layer_norm_backward(const LayerNormArgs& a, cudaStream_t s);

struct DropoutArgs {
  const void *x, *residual;     // residual: null for 0
  void* y;
  int64_t outer, mid, inner;    // the mask has outer x inner entries, shared along mid
  int dtype;
  uint64_t threshold;           // of 2^32: a word below it drops
  float scale;
  uint64_t seed, offset;
  const int64_t* seed_ptr;      // added to seed, or null
};
cudaError_t dropout_add(const DropoutArgs& a, cudaStream_t s);

}  // namespace trifast
