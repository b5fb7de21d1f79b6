// Host interface of the feed-forward block's matrix products (ff_gemm.cu) and of the kernels around
// them (ff_support.cu).
#pragma once

#include "common.cuh"

namespace trifast {
namespace ff {

// A matrix as the products read or write it: `rows` x `cols` 16-bit elements, rows `pitch` elements
// apart (a multiple of 8), in `planes` planes (1; or 3, the parts of fp32 values, see ff_support.cu),
// `plane` elements apart.
struct Matrix {
  void* p;
  int64_t rows, cols, pitch;
  int planes;
  int64_t plane;
};

// What is made of the accumulators of a tile.
enum Mode {
  kGate,    // h = silu(X Wg^T) * (X Wu^T)
  kLinear,  // Y = A B^T (+ A1 B1^T)
  kHidden,  // da, db, h from X Wg^T, X Wu^T and dY Wd
  kWeight,  // fp32 sums of A^T B over rows, three products in one launch
};

struct GemmArgs {
  int mode;
  bool bf16;         // type of the 16-bit elements
  bool b_mn;         // kLinear: B is (K, N), N contiguous (else (N, K), K contiguous)
  int products;      // kLinear: 1 or 2 (their sum)
  Matrix a[3], b[3]; // kGate: a0 = X, b = Wg, Wu.  kHidden: a0 = dY, a1 = X, b = Wg, Wu, Wd
  Matrix out[3];     // kGate: h.  kHidden: da, db, h.  kLinear: y, in the call's own type
  bool y_tma;        // TMA can write y
  // kWeight: partial sums, fp32, by split, product and row (of partial_pitch(n)); added to what is there if `add`
  float* partials;
  int64_t partial_stride;
  int splits;
  bool add;
  unsigned int* status;
};
// Row tiles (of 128) that a weight gradient's sum in TMEM takes at most; its runs are added in fp32 rounded to nearest.  The
// accumulators of TMEM round towards zero and lose 1.0e-7 of a sum of positive terms with every MMA of 16 of them (4.1e-4 of
// a sum over 512 tiles, 1.4e-3 over 1800): 1024 MMAs stay within a quarter of fp16's rounding.
constexpr int kRunTiles = 128;
// Row pitch of partial sums: whole 16-byte pieces.
__host__ __device__ inline int64_t partial_pitch(int64_t n) { return (n + 3) / 4 * 4; }
cudaError_t gemm(const GemmArgs& g, cudaStream_t s);
// Row splits of a kWeight launch over `rows` rows whose products have m[i] x n[i] results.
int weight_splits(const int64_t* m, const int64_t* n, int64_t rows, bool f32, int sms);

// The forward pass of at most kFewRows rows (ff_few.cu).  h: rows x pitch fp32, pitch a multiple of 8 that holds `hidden`.
constexpr int kFewRows = 8;
struct FewArgs {
  const void *x, *wg, *wu, *wd;
  void* y;
  float* h;        // not used by a cluster
  int64_t ld;
  int rows, width, hidden, width_out, pitch, dtype;
};
cudaError_t few_rows(const FewArgs& a, cudaStream_t s);
bool few_rows_in_cluster(int64_t rows, int64_t width, int64_t hidden, int64_t width_out, int elem);   // (needs no h)

// dst (dst.planes planes, columns padded with zeros to dst.pitch) from src (rows x dst.cols of the call's type, `ld` apart).
// Rows behind the last are left as they are: the tensor maps end before them.
struct StageJob {
  const void* src;
  int64_t ld, rows;
  Matrix dst;
};
constexpr int kStageJobs = 5;
cudaError_t stage(const StageJob* jobs, int count, int dtype, cudaStream_t s);
// The sums over `splits` of three products' partial sums (rows[j] x cols[j] each), in `dtype`, to dst[0], dst[1] and dst[2].
cudaError_t sum_partials(const float* partials, int splits, int64_t stride, void* const (&dst)[3], const int64_t (&rows)[3],
                         const int64_t (&cols)[3], int dtype, cudaStream_t s);

}  // namespace ff
}  // namespace trifast
