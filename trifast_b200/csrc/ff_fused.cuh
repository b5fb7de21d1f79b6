// Host interface of the feed-forward block's fused kernels (ff_fused.cu).
#pragma once

#include "ff_gemm.cuh"

namespace trifast {
namespace ff {

enum FusedWhat { kForward, kDx, kDw };

// Widths (of x and of y) that the fused kernels take: X, a chunk of the weights and the results have to lie in one
// multiprocessor's memories.
constexpr int kFusedWidth = 128;

struct FusedArgs {
  int what;
  bool bf16;
  Matrix x, dy, wg, wu, wd;
  Matrix out;          // kForward: y.  kDx: dx
  bool y_tma;          // TMA can write it
  // kDw: fp32 sums (splits, dWg | dWu | dWd)
  float* partials;
  int64_t partial_stride;
  int splits;
  bool add;            // to what is there
  unsigned int* status;
};
cudaError_t fused(const FusedArgs& g, cudaStream_t s);
// Shares of the rows in a kDw launch: chunks of hidden units times shares fill the multiprocessors.
int fused_weight_splits(int64_t rows, int64_t hidden, int sms);

}  // namespace ff
}  // namespace trifast
