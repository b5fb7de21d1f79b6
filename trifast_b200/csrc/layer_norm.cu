// Layer norm over the last dimension, and its gradients:
//     mu = mean(x),  r = (mean((x - mu)^2) + eps)^-1/2,  xh = (x - mu) r,  y = xh w + b
//     g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum of dy
//
// A row lies in the registers of TPR threads (8, 16 or 32 lanes of a warp, or a whole block), E elements
// each, so that x is read once, its variance is that of the deviations from the mean, and the backward
// makes both again from x instead of reading them (8 bytes a row less, for two more reductions, which the
// memory hides).  A thread has the same columns in all of its rows: w and b stay in registers, and so do
// its sums for dw and db, which meet in shared memory, then as one partial row a block, and are summed in a
// fixed order by a second kernel.  All arithmetic is in fp32; every result is rounded once.
//
// What bounds it: memory.  Rows whose bytes are no multiple of 16 are read element by element; rows beyond
// 8192 elements (kMaxRow) are walked in passes instead.

#include <type_traits>

#include "block_kernels.h"

namespace trifast {
namespace {

constexpr int kMaxRow = 8192;

template <typename T, int VEC> struct Raw;
template <typename T> struct Raw<T, 1> { T v; };
template <> struct Raw<float, 4> { uint4 v; };
template <> struct Raw<__nv_bfloat16, 8> { uint4 v; };
template <> struct Raw<__half, 8> { uint4 v; };

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Raw<T, VEC>& r, float* f) {
  T t[VEC];
  memcpy(t, &r, sizeof(t));
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] = to_f32<T>(t[e]);
}
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> pack(const float* f) {
  T t[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) t[e] = from_f32<T>(f[e]);
  Raw<T, VEC> r;
  memcpy(&r, t, sizeof(t));
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> zero_raw() {
  Raw<T, VEC> r;
  memset(&r, 0, sizeof(r));
  return r;
}

__device__ __forceinline__ float affine_at(const void* p, int dtype, int i) {
  switch (dtype) {
    case TRIFAST_F32: return reinterpret_cast<const float*>(p)[i];
    case TRIFAST_BF16: return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
    default: return __half2float(reinterpret_cast<const __half*>(p)[i]);
  }
}

// Sums over the TPR threads of a row, N at a time.  `buf`: shared memory of each call site's own, two
// call sites at least in a loop (a thread that is a call behind still reads the other's).
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float* v, float (*buf)[32]) {
#pragma unroll
  for (int m = (TPR < 32 ? TPR : 32) / 2; m > 0; m >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) buf[i][warp] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 32; ++w) s += buf[i][w];
      v[i] = s;
    }
  }
}

template <int TPR> constexpr int kBlock = TPR > 32 ? TPR : 256;

// Where a thread's elements lie: piece k at column (k * TPR + lane) * VEC.
template <int TPR, int VEC>
__device__ __forceinline__ int col_of(int lane, int k) { return (k * TPR + lane) * VEC; }

template <typename T, int VEC, int K>
__device__ __forceinline__ void load_row(Raw<T, VEC>* r, const T* p, bool valid, int width, int lane, int tpr) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * tpr + lane) * VEC;
    r[k] = valid && c < width ? *reinterpret_cast<const Raw<T, VEC>*>(p + c) : zero_raw<T, VEC>();
  }
}

// Mean and 1 / standard deviation of R rows.
template <typename T, int VEC, int TPR, int K, int R>
__device__ __forceinline__ void statistics(const Raw<T, VEC> (*x)[K], int width, int lane, float inv_width, float eps, float* mean,
                                           float* rstd, float (*buf)[8][32]) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mean[r] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float f[VEC];
      unpack<T, VEC>(x[r][k], f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) mean[r] += f[e];
    }
  }
  row_sums<TPR, R>(mean, buf[0]);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mean[r] *= inv_width;
    rstd[r] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (col_of<TPR, VEC>(lane, k) < width) {
        float f[VEC];
        unpack<T, VEC>(x[r][k], f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) rstd[r] = fmaf(f[e] - mean[r], f[e] - mean[r], rstd[r]);
      }
    }
  }
  row_sums<TPR, R>(rstd, buf[1]);
#pragma unroll
  for (int r = 0; r < R; ++r) rstd[r] = rsqrtf(fmaf(rstd[r], inv_width, eps));
}

template <typename T, int VEC, int TPR, int K, int R>
__global__ void __launch_bounds__(kBlock<TPR>) layer_norm_fwd_kernel(LayerNormArgs a) {
  constexpr int kGroups = kBlock<TPR> / TPR;
  __shared__ float buf[2][8][32];
  const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const float inv_width = 1.f / (float)a.width;
  after_previous();
  float w[K * VEC], b[K * VEC];
#pragma unroll
  for (int i = 0; i < K * VEC; ++i) {
    const int c = col_of<TPR, VEC>(lane, i / VEC) + i % VEC;
    w[i] = a.weight && c < a.width ? affine_at(a.weight, a.affine_dtype, c) : 1.f;
    b[i] = a.bias && c < a.width ? affine_at(a.bias, a.affine_dtype, c) : 0.f;
  }
  for (int64_t base = (int64_t)blockIdx.x * kGroups * R; base < a.rows; base += (int64_t)gridDim.x * kGroups * R) {
    Raw<T, VEC> x[R][K];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kGroups + grp;
      load_row<T, VEC, K>(x[r], reinterpret_cast<const T*>(a.x) + row * a.ld_x, row < a.rows, a.width, lane, TPR);
    }
    float mean[R], rstd[R];
    statistics<T, VEC, TPR, K, R>(x, a.width, lane, inv_width, a.eps, mean, rstd, buf);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kGroups + grp;
      T* y = reinterpret_cast<T*>(a.y) + row * a.width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float f[VEC];
        unpack<T, VEC>(x[r][k], f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = fmaf((f[e] - mean[r]) * rstd[r], w[k * VEC + e], b[k * VEC + e]);
        const int c = col_of<TPR, VEC>(lane, k);
        if (row < a.rows && c < a.width) *reinterpret_cast<Raw<T, VEC>*>(y + c) = pack<T, VEC>(f);
      }
    }
  }
}

template <typename T, int VEC, int TPR, int K, int R>
__global__ void __launch_bounds__(kBlock<TPR>) layer_norm_bwd_kernel(LayerNormArgs a) {
  constexpr int kGroups = kBlock<TPR> / TPR, E = K * VEC;
  __shared__ float buf[3][8][32];
  const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const float inv_width = 1.f / (float)a.width;
  after_previous();
  float w[E], dw[E], db[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = col_of<TPR, VEC>(lane, i / VEC) + i % VEC;
    w[i] = a.weight && c < a.width ? affine_at(a.weight, a.affine_dtype, c) : 1.f;
    dw[i] = db[i] = 0.f;
  }
  for (int64_t base = (int64_t)blockIdx.x * kGroups * R; base < a.rows; base += (int64_t)gridDim.x * kGroups * R) {
    Raw<T, VEC> x[R][K], dy[R][K];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kGroups + grp;
      load_row<T, VEC, K>(x[r], reinterpret_cast<const T*>(a.x) + row * a.ld_x, row < a.rows, a.width, lane, TPR);
      load_row<T, VEC, K>(dy[r], reinterpret_cast<const T*>(a.dy) + row * a.ld_dy, row < a.rows, a.width, lane, TPR);
    }
    float mean[R], rstd[R], s[2 * R];
    statistics<T, VEC, TPR, K, R>(x, a.width, lane, inv_width, a.eps, mean, rstd, buf);
    // (elements behind the row, and rows behind the last, have dy = 0)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float f[VEC], d[VEC];
        unpack<T, VEC>(x[r][k], f);
        unpack<T, VEC>(dy[r][k], d);
        if (base + r * kGroups + grp < a.rows && col_of<TPR, VEC>(lane, k) < a.width) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float xh = (f[e] - mean[r]) * rstd[r], g = d[e] * w[k * VEC + e];
            s[2 * r] += g;
            s[2 * r + 1] = fmaf(g, xh, s[2 * r + 1]);
            dw[k * VEC + e] = fmaf(d[e], xh, dw[k * VEC + e]);
            db[k * VEC + e] += d[e];
          }
        }
      }
    }
    if (a.dx == nullptr) continue;
    row_sums<TPR, 2 * R>(s, buf[2]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kGroups + grp;
      const float m1 = s[2 * r] * inv_width, m2 = s[2 * r + 1] * inv_width;
      T* dx = reinterpret_cast<T*>(a.dx) + row * a.width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float f[VEC], d[VEC];
        unpack<T, VEC>(x[r][k], f);
        unpack<T, VEC>(dy[r][k], d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = (f[e] - mean[r]) * rstd[r];
          f[e] = rstd[r] * (fmaf(d[e], w[k * VEC + e], -m1) - xh * m2);
        }
        const int c = col_of<TPR, VEC>(lane, k);
        if (row < a.rows && c < a.width) *reinterpret_cast<Raw<T, VEC>*>(dx + c) = pack<T, VEC>(f);
      }
    }
  }
  if (a.partials == nullptr) return;
  float* out = a.partials + (int64_t)blockIdx.x * 2 * a.width;
  if constexpr (TPR > 32) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = col_of<TPR, VEC>(lane, i / VEC) + i % VEC;
      if (c < a.width) {
        out[c] = dw[i];
        out[a.width + c] = db[i];
      }
    }
  } else {
    // rows of one warp, then the eight warps
    __shared__ float sum[8][2][TPR * E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
#pragma unroll
      for (int m = TPR; m < 32; m <<= 1) {
        dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], m);
        db[i] += __shfl_xor_sync(0xffffffffu, db[i], m);
      }
      const int c = col_of<TPR, VEC>(lane, i / VEC) + i % VEC;
      if ((threadIdx.x & 31) < TPR) {
        sum[threadIdx.x >> 5][0][c] = dw[i];
        sum[threadIdx.x >> 5][1][c] = db[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.width; i += kBlock<TPR>) {
      const int which = i >= a.width, c = i - which * a.width;
      float v = 0.f;
#pragma unroll
      for (int g = 0; g < 8; ++g) v += sum[g][which][c];
      out[i] = v;
    }
  }
}

// ------------------------------------------------------------------ rows beyond kMaxRow
constexpr int kLongThreads = 512, kLongRows = 64;   // rows of one partial sum of the columns

template <typename T>
__device__ __forceinline__ void long_statistics(const T* x, int width, float eps, float* mean, float* rstd, float (*buf)[1][32]) {
  float m = 0.f, v = 0.f;
  for (int c = threadIdx.x; c < width; c += kLongThreads) m += to_f32<T>(x[c]);
  row_sums<kLongThreads, 1>(&m, buf[0]);
  m /= (float)width;
  for (int c = threadIdx.x; c < width; c += kLongThreads) {
    const float d = to_f32<T>(x[c]) - m;
    v = fmaf(d, d, v);
  }
  row_sums<kLongThreads, 1>(&v, buf[1]);
  *mean = m;
  *rstd = rsqrtf(v / (float)width + eps);
}

template <typename T, bool BWD>
__global__ void __launch_bounds__(kLongThreads) layer_norm_long_kernel(LayerNormArgs a, float* row_stats) {
  __shared__ float buf[4][1][32];
  after_previous();
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld_x;
    float mean, rstd;
    long_statistics<T>(x, a.width, a.eps, &mean, &rstd, buf);
    if constexpr (!BWD) {
      T* y = reinterpret_cast<T*>(a.y) + row * a.width;
      for (int c = threadIdx.x; c < a.width; c += kLongThreads) {
        const float w = a.weight ? affine_at(a.weight, a.affine_dtype, c) : 1.f, b = a.bias ? affine_at(a.bias, a.affine_dtype, c) : 0.f;
        y[c] = from_f32<T>(fmaf((to_f32<T>(x[c]) - mean) * rstd, w, b));
      }
    } else {
      if (row_stats && threadIdx.x == 0) {
        row_stats[2 * row] = mean;
        row_stats[2 * row + 1] = rstd;
      }
      if (!a.dx) continue;
      const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.ld_dy;
      T* dx = reinterpret_cast<T*>(a.dx) + row * a.width;
      float s1 = 0.f, s2 = 0.f;
      for (int c = threadIdx.x; c < a.width; c += kLongThreads) {
        const float g = to_f32<T>(dy[c]) * (a.weight ? affine_at(a.weight, a.affine_dtype, c) : 1.f);
        s1 += g;
        s2 = fmaf(g, (to_f32<T>(x[c]) - mean) * rstd, s2);
      }
      row_sums<kLongThreads, 1>(&s1, buf[2]);
      row_sums<kLongThreads, 1>(&s2, buf[3]);
      s1 /= (float)a.width;
      s2 /= (float)a.width;
      for (int c = threadIdx.x; c < a.width; c += kLongThreads) {
        const float g = to_f32<T>(dy[c]) * (a.weight ? affine_at(a.weight, a.affine_dtype, c) : 1.f);
        dx[c] = from_f32<T>(rstd * (g - s1 - (to_f32<T>(x[c]) - mean) * rstd * s2));
      }
    }
  }
}

// Partial sums of dy xh and dy over kLongRows rows: a thread has one column.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(LayerNormArgs a, const float* __restrict__ row_stats) {
  after_previous();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.width) return;
  const int64_t lo = (int64_t)blockIdx.y * kLongRows, hi = lo + kLongRows < a.rows ? lo + kLongRows : a.rows;
  float dw = 0.f, db = 0.f;
  for (int64_t r = lo; r < hi; ++r) {
    const float d = to_f32<T>(reinterpret_cast<const T*>(a.dy)[r * a.ld_dy + c]);
    const float xh = (to_f32<T>(reinterpret_cast<const T*>(a.x)[r * a.ld_x + c]) - row_stats[2 * r]) * row_stats[2 * r + 1];
    dw = fmaf(d, xh, dw);
    db += d;
  }
  float* out = a.partials + (int64_t)blockIdx.y * 2 * a.width;
  out[c] = dw;
  out[a.width + c] = db;
}

// ------------------------------------------------------------------ the blocks' partial sums
template <typename W>
__global__ void __launch_bounds__(1024) layer_norm_sum_kernel(const float* __restrict__ partials, int blocks, int width, W* dweight, W* dbias) {
  __shared__ float sum[32][33];
  after_previous();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  float v = 0.f;
  if (c < 2 * width)
#pragma unroll 4
    for (int b = y; b < blocks; b += 32) v += partials[(int64_t)b * 2 * width + c];
  sum[y][x] = v;
  __syncthreads();
  v = sum[x][y];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  const int col = blockIdx.x * 32 + y;
  if (x == 0 && col < 2 * width) {
    if (col < width) {
      if (dweight) dweight[col] = from_f32<W>(v);
    } else if (dbias) {
      dbias[col - width] = from_f32<W>(v);
    }
  }
}

cudaError_t sum_blocks(const LayerNormArgs& a, int blocks, cudaStream_t s) {
  const dim3 g((unsigned)((2 * a.width + 31) / 32));
  switch (a.affine_dtype) {
    case TRIFAST_F32: return launch_early(layer_norm_sum_kernel<float>, g, 1024, 0, s, a.partials, blocks, a.width, (float*)a.dweight, (float*)a.dbias);
    case TRIFAST_BF16:
      return launch_early(layer_norm_sum_kernel<__nv_bfloat16>, g, 1024, 0, s, a.partials, blocks, a.width, (__nv_bfloat16*)a.dweight, (__nv_bfloat16*)a.dbias);
    default: return launch_early(layer_norm_sum_kernel<__half>, g, 1024, 0, s, a.partials, blocks, a.width, (__half*)a.dweight, (__half*)a.dbias);
  }
}

// ------------------------------------------------------------------ dispatch
// Threads a row and elements a thread, by width.
struct RowShape {
  int tpr, e;
};
constexpr RowShape row_shape(int width) {
  return width <= 64 ? RowShape{8, 8}
         : width <= 128 ? RowShape{16, 8}
         : width <= 256 ? RowShape{32, 8}
         : width <= 512 ? RowShape{32, 16}
         : width <= 1024 ? RowShape{128, 8}
         : width <= 2048 ? RowShape{128, 16}
         : width <= 4096 ? RowShape{256, 16}
                         : RowShape{512, 16};
}
// Blocks of the backward at most: eight a multiprocessor (three of whole rows, whose partial sums are wide).
constexpr int most_blocks(int tpr) { return 148 * (tpr > 32 ? 3 : 8); }
constexpr int kFwdRows = 4, kBwdRows = 2;   // rows a group of threads has in flight

int64_t bwd_blocks(int64_t rows, int width) {
  const int tpr = row_shape(width).tpr;
  const int64_t per = (int64_t)(tpr > 32 ? 1 : 256 / tpr) * kBwdRows, b = (rows + per - 1) / per;
  return b < most_blocks(tpr) ? b : most_blocks(tpr);
}

template <auto Kernel>
int blocks_per_sm(int threads) {
  static std::atomic<int> known{0};
  int b = known.load(std::memory_order_relaxed);
  if (b == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&b, Kernel, threads, 0) != cudaSuccess || b < 1) b = 1;
    known.store(b, std::memory_order_relaxed);
  }
  return b;
}

template <typename T, int VEC, int TPR, int E, bool BWD>
cudaError_t launch_row(const LayerNormArgs& a, cudaStream_t s, int* blocks) {
  constexpr int kThreads = kBlock<TPR>, R = BWD ? kBwdRows : (E > 8 ? kFwdRows / 2 : kFwdRows);
  constexpr auto kern = [] {
    if constexpr (BWD) return &layer_norm_bwd_kernel<T, VEC, TPR, E / VEC, R>;
    else return &layer_norm_fwd_kernel<T, VEC, TPR, E / VEC, R>;
  }();
  const int64_t per = (int64_t)(kThreads / TPR) * R, need = (a.rows + per - 1) / per;
  int64_t most = (int64_t)sm_count() * blocks_per_sm<kern>(kThreads);
  if (BWD && most > most_blocks(TPR)) most = most_blocks(TPR);
  *blocks = (int)(need < most ? need : most);
  return launch_early(kern, dim3((unsigned)*blocks), kThreads, 0, s, a);
}

template <typename T, int VEC, bool BWD>
cudaError_t launch_width(const LayerNormArgs& a, cudaStream_t s, int* blocks) {
  const RowShape r = row_shape(a.width);
  switch (r.tpr) {
    case 8: return launch_row<T, VEC, 8, 8, BWD>(a, s, blocks);
    case 16: return launch_row<T, VEC, 16, 8, BWD>(a, s, blocks);
    case 32: return r.e == 8 ? launch_row<T, VEC, 32, 8, BWD>(a, s, blocks) : launch_row<T, VEC, 32, 16, BWD>(a, s, blocks);
    case 128: return r.e == 8 ? launch_row<T, VEC, 128, 8, BWD>(a, s, blocks) : launch_row<T, VEC, 128, 16, BWD>(a, s, blocks);
    case 256: return launch_row<T, VEC, 256, 16, BWD>(a, s, blocks);
    default: return launch_row<T, VEC, 512, 16, BWD>(a, s, blocks);
  }
}

template <typename T, bool BWD>
cudaError_t launch_type(const LayerNormArgs& a, cudaStream_t s, int* blocks) {
  if (a.width > kMaxRow) {
    const unsigned grid = (unsigned)(a.rows < 4 * sm_count() ? a.rows : 4 * sm_count());
    float* stats = nullptr;
    *blocks = (int)((a.rows + kLongRows - 1) / kLongRows);
    if (BWD && a.partials) stats = a.partials + (int64_t)*blocks * 2 * a.width;
    cudaError_t e = launch_early(layer_norm_long_kernel<T, BWD>, dim3(grid), kLongThreads, 0, s, a, stats);
    if (e != cudaSuccess || !stats) return e;
    return launch_early(layer_norm_columns_kernel<T>, dim3((unsigned)((a.width + 255) / 256), (unsigned)*blocks), 256, 0, s, a, (const float*)stats);
  }
  constexpr int kVec = 16 / sizeof(T);
  auto whole = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = a.width % kVec == 0 && whole(a.x) && whole(a.y) && whole(a.dx) && whole(a.dy) &&
                   (a.rows == 1 || (a.ld_x % kVec == 0 && (!BWD || a.ld_dy % kVec == 0)));
  return vec ? launch_width<T, kVec, BWD>(a, s, blocks) : launch_width<T, 1, BWD>(a, s, blocks);
}

template <bool BWD>
cudaError_t launch_any(const LayerNormArgs& a, cudaStream_t s, int* blocks) {
  switch (a.dtype) {
    case TRIFAST_F32: return launch_type<float, BWD>(a, s, blocks);
    case TRIFAST_BF16: return launch_type<__nv_bfloat16, BWD>(a, s, blocks);
    default: return launch_type<__half, BWD>(a, s, blocks);
  }
}

}  // namespace

int64_t layer_norm_workspace_floats(int64_t rows, int width, int) {
  if (width > kMaxRow) return (rows + kLongRows - 1) / kLongRows * 2 * width + 2 * rows;
  return bwd_blocks(rows, width) * 2 * width;
}

cudaError_t layer_norm_forward(const LayerNormArgs& a, cudaStream_t s) {
  int blocks;
  return launch_any<false>(a, s, &blocks);
}

cudaError_t layer_norm_backward(const LayerNormArgs& a, cudaStream_t s) {
  int blocks;
  const cudaError_t e = launch_any<true>(a, s, &blocks);
  return e != cudaSuccess || !a.partials ? e : sum_blocks(a, blocks, s);
}

}  // namespace trifast
