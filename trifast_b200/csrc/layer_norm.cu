// Layer norm over the last dimension, and its gradients:
//     mu = mean(x),  r = (mean((x - mu)^2) + eps)^-1/2,  xh = (x - mu) r,  y = xh w + b
//     g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum of dy
//
// A row lies in the registers of TPR threads (4 to 32 lanes of a warp, or a whole block), up to 16 elements each, so
// that x is read once, its variance is that of the deviations from the mean, and the backward makes both again
// from x instead of reading them (8 bytes a row less).  Two sums at a time go around: mean(x) with mean(g), which does
// not need it; then the variance with sum(g (x - mu)).  A thread has the same columns in all of its rows: w and
// b stay in registers, and so do its sums for dw and db, which meet in shared memory, then as one partial row a
// block, and are summed in a fixed order by a second kernel.  All arithmetic is in fp32; every result is rounded once.
//
// Rows whose bytes are no multiple of 16 (SHIFT) are read in the 16-byte pieces that they lie in all the same: rows of
// one class modulo 8 (fp32: 4) begin at the same place of a piece, and a block takes rows of one class, so that its
// threads keep their columns.  What a piece holds of other rows is set to zero.
//
// What bounds it: memory (1,048,576 x 128 bf16: 87 us forward, 135 backward, 6.2 and 6.0 TB/s).  Rows beyond 8192 elements
// (kMaxRow) are walked in passes instead.

#include <type_traits>

#include "block_kernels.h"
#include "tc_common.cuh"

namespace trifast {
namespace {

constexpr int kMaxRow = 8192;   // elements, with those of its first piece that are not its own

using tc::fadd2;
using tc::ffma2;
using tc::fmul2;

// A 16-byte piece of a row.
template <typename T> constexpr int kVec = 16 / sizeof(T);
template <typename T>
__device__ __forceinline__ void unpack(const uint4& r, float* f) {
  if constexpr (std::is_same<T, float>::value) {
    f[0] = __uint_as_float(r.x);
    f[1] = __uint_as_float(r.y);
    f[2] = __uint_as_float(r.z);
    f[3] = __uint_as_float(r.w);
  } else {
    tc::unpack2<T>(r.x, f[0], f[1]);
    tc::unpack2<T>(r.y, f[2], f[3]);
    tc::unpack2<T>(r.z, f[4], f[5]);
    tc::unpack2<T>(r.w, f[6], f[7]);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float* f) {
  if constexpr (std::is_same<T, float>::value)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(tc::pack2<T>(f[0], f[1]), tc::pack2<T>(f[2], f[3]), tc::pack2<T>(f[4], f[5]), tc::pack2<T>(f[6], f[7]));
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

// The pieces of a row that a thread has: piece k begins at column (k * TPR + lane) * VEC - shift.
template <typename T, int TPR, int K, bool SHIFT>
struct RowPieces {
  static constexpr int VEC = kVec<T>, E = K * VEC;
  int lane, width, shift;
  int64_t rows;

  __device__ __forceinline__ int col(int k) const { return (k * TPR + lane) * VEC - (SHIFT ? shift : 0); }
  __device__ __forceinline__ bool any(int k) const { return col(k) < width; }
  __device__ __forceinline__ bool has(int k, int e) const {
    return SHIFT ? (unsigned)(col(k) + e) < (unsigned)width : any(k);
  }
  // Whether some of the piece is not the row's: the first one's and the last one's lanes.
  __device__ __forceinline__ bool edge(int k) const { return SHIFT && (col(k) < 0 || col(k) + VEC > width); }
  // Row `row` of `tensor`, zeros behind the last one.  (Nothing is read behind the tensor's end; before its beginning lies
  // nothing of a piece: the first row's shift is 0.)
  __device__ __forceinline__ void load(uint4* r, const void* tensor, int64_t ld, int64_t row) const {
    const T* t = reinterpret_cast<const T*>(tensor);
    const T *p = t + row * ld, *end = t + (rows - 1) * ld + width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      r[k] = make_uint4(0, 0, 0, 0);
      if (row >= rows || !any(k)) continue;
      if (SHIFT && p + col(k) + VEC > end) {
        T t[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) t[e] = has(k, e) ? p[col(k) + e] : from_f32<T>(0.f);
        memcpy(&r[k], t, 16);
      } else {
        r[k] = *reinterpret_cast<const uint4*>(p + col(k));
      }
    }
  }
  // The values, 0 where they are not the row's.
  __device__ __forceinline__ void values(const uint4* r, float* f) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      unpack<T>(r[k], f + k * VEC);
      if (edge(k)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[k * VEC + e] = has(k, e) ? f[k * VEC + e] : 0.f;
      }
    }
  }
  // f - mean, 0 where the value is not the row's.
  __device__ __forceinline__ void center(float* f, float mean) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float m = any(k) ? mean : 0.f;
#pragma unroll
      for (int e = 0; e < VEC; e += 2) fadd2(f[k * VEC + e], f[k * VEC + e + 1], f[k * VEC + e], f[k * VEC + e + 1], -m, -m);
      if (edge(k)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[k * VEC + e] = has(k, e) ? f[k * VEC + e] : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(T* p, const float* f) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!any(k)) continue;
      if (edge(k)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (has(k, e)) p[col(k) + e] = from_f32<T>(f[k * VEC + e]);
      } else {
        *reinterpret_cast<uint4*>(p + col(k)) = pack<T>(f + k * VEC);
      }
    }
  }
  __device__ __forceinline__ void affine(const void* a, int dtype, float otherwise, float* w) const {
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = a && has(i / VEC, i % VEC) ? affine_at(a, dtype, col(i / VEC) + i % VEC) : otherwise;
  }
};

// The rows of a block: of class `first` modulo `step`, from the block's place among those of its class.
struct BlockRows {
  int64_t first, step, stride;   // stride: rows of the class between two turns of the block
  int shift;
};
template <bool SHIFT>
__device__ __forceinline__ BlockRows block_rows(const LayerNormArgs& a, int vec, int per_turn) {
  if (!SHIFT) return {(int64_t)blockIdx.x * per_turn, 1, (int64_t)gridDim.x * per_turn, 0};
  // (the grid is a multiple of the classes)
  const int cls = blockIdx.x % a.classes, place = blockIdx.x / a.classes;
  return {cls + (int64_t)place * per_turn * a.classes, a.classes, (int64_t)(gridDim.x / a.classes) * per_turn * a.classes,
          (int)((int64_t)cls * a.width % vec)};
}

template <int E>
__device__ __forceinline__ float sum_of(const float* f) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int e = 0; e < E; e += 2) fadd2(s0, s1, s0, s1, f[e], f[e + 1]);
  return s0 + s1;
}
template <int E>
__device__ __forceinline__ float dot_of(const float* f, const float* g) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int e = 0; e < E; e += 2) ffma2(s0, s1, f[e], f[e + 1], g[e], g[e + 1], s0, s1);
  return s0 + s1;
}

template <typename T, int TPR, int K, int R, bool SHIFT>
__global__ void __launch_bounds__(kBlock<TPR>) layer_norm_fwd_kernel(LayerNormArgs a) {
  constexpr int kGroups = kBlock<TPR> / TPR;
  using P = RowPieces<T, TPR, K, SHIFT>;
  constexpr int E = P::E;
  __shared__ float buf[2][R][32];
  const int grp = threadIdx.x / TPR;
  const BlockRows rows = block_rows<SHIFT>(a, kVec<T>, kGroups * R);
  const P p{(int)(threadIdx.x % TPR), a.width, rows.shift, a.rows};
  const float inv_width = 1.f / (float)a.width;
  after_previous();
  float w[E], b[E];
  p.affine(a.weight, a.affine_dtype, 1.f, w);
  p.affine(a.bias, a.affine_dtype, 0.f, b);
  uint4 raw[R][K];
  auto load = [&](int64_t base) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + (r * kGroups + grp) * rows.step;
      p.load(raw[r], a.x, a.ld_x, row);
    }
  };
  if (rows.first < a.rows) load(rows.first);
  for (int64_t base = rows.first; base < a.rows; base += rows.stride) {
    float f[R][E], mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      p.values(raw[r], f[r]);
      mean[r] = sum_of<E>(f[r]);
    }
    if (base + rows.stride < a.rows) load(base + rows.stride);   // on their way meanwhile
    row_sums<TPR, R>(mean, buf[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      p.center(f[r], mean[r] * inv_width);
      rstd[r] = dot_of<E>(f[r], f[r]);
    }
    row_sums<TPR, R>(rstd, buf[1]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + (r * kGroups + grp) * rows.step;
      const float s = rsqrtf(fmaf(rstd[r], inv_width, a.eps));
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        fmul2(f[r][e], f[r][e + 1], f[r][e], f[r][e + 1], s, s);
        ffma2(f[r][e], f[r][e + 1], f[r][e], f[r][e + 1], w[e], w[e + 1], b[e], b[e + 1]);
      }
      if (row < a.rows) p.store(reinterpret_cast<T*>(a.y) + row * a.width, f[r]);
    }
  }
}

template <typename T, int TPR, int K, int R, bool SHIFT>
__global__ void __launch_bounds__(kBlock<TPR>) layer_norm_bwd_kernel(LayerNormArgs a) {
  constexpr int kGroups = kBlock<TPR> / TPR;
  using P = RowPieces<T, TPR, K, SHIFT>;
  constexpr int E = P::E, VEC = P::VEC;
  __shared__ float buf[2][2 * R][32];
  const int grp = threadIdx.x / TPR;
  const BlockRows rows = block_rows<SHIFT>(a, VEC, kGroups * R);
  const P p{(int)(threadIdx.x % TPR), a.width, rows.shift, a.rows};
  const float inv_width = 1.f / (float)a.width;
  after_previous();
  float w[E], dw[E], db[E];
  p.affine(a.weight, a.affine_dtype, 1.f, w);
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = db[i] = 0.f;
  uint4 raw_x[R][K], raw_dy[R][K];
  auto load = [&](int64_t base) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + (r * kGroups + grp) * rows.step;
      p.load(raw_x[r], a.x, a.ld_x, row);
      p.load(raw_dy[r], a.dy, a.ld_dy, row);
    }
  };
  if (rows.first < a.rows) load(rows.first);
  for (int64_t base = rows.first; base < a.rows; base += rows.stride) {
    float f[R][E], d[R][E], s[2 * R], t[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      p.values(raw_x[r], f[r]);
      p.values(raw_dy[r], d[r]);     // (0 behind the last row)
      s[2 * r] = sum_of<E>(f[r]);
      s[2 * r + 1] = dot_of<E>(d[r], w);
    }
    if (base + rows.stride < a.rows) load(base + rows.stride);   // on their way meanwhile
    row_sums<TPR, 2 * R>(s, buf[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      p.center(f[r], s[2 * r] * inv_width);
      float t0 = 0.f, t1 = 0.f;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float g0, g1;
        fmul2(g0, g1, d[r][e], d[r][e + 1], w[e], w[e + 1]);
        ffma2(t0, t1, g0, g1, f[r][e], f[r][e + 1], t0, t1);
      }
      t[2 * r] = dot_of<E>(f[r], f[r]);
      t[2 * r + 1] = t0 + t1;
    }
    row_sums<TPR, 2 * R>(t, buf[1]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + (r * kGroups + grp) * rows.step;
      const float rstd = rsqrtf(fmaf(t[2 * r], inv_width, a.eps)), m1 = s[2 * r + 1] * inv_width, m2 = t[2 * r + 1] * rstd * inv_width;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float &x0 = f[r][e], &x1 = f[r][e + 1], &d0 = d[r][e], &d1 = d[r][e + 1];
        fmul2(x0, x1, x0, x1, rstd, rstd);
        ffma2(dw[e], dw[e + 1], d0, d1, x0, x1, dw[e], dw[e + 1]);
        fadd2(db[e], db[e + 1], db[e], db[e + 1], d0, d1);
        ffma2(d0, d1, d0, d1, w[e], w[e + 1], -m1, -m1);
        ffma2(d0, d1, x0, x1, -m2, -m2, d0, d1);
        fmul2(d0, d1, d0, d1, rstd, rstd);
      }
      if (a.dx && row < a.rows) p.store(reinterpret_cast<T*>(a.dx) + row * a.width, d[r]);
    }
  }
  if (a.partials == nullptr) return;
  float* out = a.partials + (int64_t)blockIdx.x * 2 * a.width;
  if constexpr (TPR > 32) {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (p.has(i / VEC, i % VEC)) {
        const int c = p.col(i / VEC) + i % VEC;
        out[c] = dw[i];
        out[a.width + c] = db[i];
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
      if ((threadIdx.x & 31) < TPR && p.has(i / VEC, i % VEC)) {
        const int c = p.col(i / VEC) + i % VEC;
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
// Threads a row and elements a thread, by the elements of its pieces.
struct RowShape {
  int tpr, e;
};
constexpr RowShape row_shape(int width) {
  return width <= 64 ? RowShape{4, 16}
         : width <= 128 ? RowShape{8, 16}
         : width <= 256 ? RowShape{16, 16}
         : width <= 512 ? RowShape{32, 16}
         : width <= 1024 ? RowShape{128, 8}
         : width <= 2048 ? RowShape{128, 16}
         : width <= 4096 ? RowShape{256, 16}
                         : RowShape{512, 16};
}
// Classes of rows that begin at the same place of a 16-byte piece, and the elements of a row's pieces.
int row_classes(int width, int vec) {
  int c = vec;
  while (c > 1 && width % 2 == 0) {
    width /= 2;
    c /= 2;
  }
  return c;
}
int pieces_width(int width, int vec) { return row_classes(width, vec) > 1 ? width + vec - 1 : width; }
// Blocks of the backward at most: eight a multiprocessor (three of whole rows, whose partial sums are wide).
constexpr int most_blocks(int tpr) { return 148 * (tpr > 32 ? 3 : 8); }

int64_t bwd_blocks(int64_t rows, int width, int vec) {
  const int tpr = row_shape(pieces_width(width, vec)).tpr, classes = row_classes(width, vec);
  const int64_t per = tpr > 32 ? 1 : 256 / tpr, b = (rows + per - 1) / per;
  const int64_t most = b < most_blocks(tpr) ? b : most_blocks(tpr);
  return (most + classes - 1) / classes * classes;
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

template <typename T, int TPR, int E, bool SHIFT, bool BWD>
cudaError_t launch_row(const LayerNormArgs& a, cudaStream_t s, int* blocks) {
  // rows that a group of threads works on at a time; in the backward two where it is a block of 128, which waits
  // for all of its threads twice a turn (more threads leave no registers for it)
  constexpr int kThreads = kBlock<TPR>, R = BWD && TPR != 128 ? 1 : 2, K = E / kVec<T>;
  constexpr auto kern = [] {
    if constexpr (BWD) return &layer_norm_bwd_kernel<T, TPR, K, R, SHIFT>;
    else return &layer_norm_fwd_kernel<T, TPR, K, R, SHIFT>;
  }();
  const int64_t per = (int64_t)(kThreads / TPR) * R, need = (a.rows + per - 1) / per;
  int64_t most = (int64_t)sm_count() * blocks_per_sm<kern>(kThreads);
  if (BWD && most > most_blocks(TPR)) most = most_blocks(TPR);
  if (need < most) most = need;
  *blocks = (int)(SHIFT ? (most + a.classes - 1) / a.classes * a.classes : most);
  return launch_early(kern, dim3((unsigned)*blocks), kThreads, 0, s, a);
}

template <typename T, bool SHIFT, bool BWD>
cudaError_t launch_width(const LayerNormArgs& a, cudaStream_t s, int* blocks) {
  const RowShape r = row_shape(pieces_width(a.width, kVec<T>));
  switch (r.tpr) {
    case 4: return launch_row<T, 4, 16, SHIFT, BWD>(a, s, blocks);
    case 8: return launch_row<T, 8, 16, SHIFT, BWD>(a, s, blocks);
    case 16: return launch_row<T, 16, 16, SHIFT, BWD>(a, s, blocks);
    case 32: return launch_row<T, 32, 16, SHIFT, BWD>(a, s, blocks);
    case 128: return r.e == 8 ? launch_row<T, 128, 8, SHIFT, BWD>(a, s, blocks) : launch_row<T, 128, 16, SHIFT, BWD>(a, s, blocks);
    case 256: return launch_row<T, 256, 16, SHIFT, BWD>(a, s, blocks);
    default: return launch_row<T, 512, 16, SHIFT, BWD>(a, s, blocks);
  }
}

template <typename T, bool BWD>
cudaError_t launch_type(LayerNormArgs a, cudaStream_t s, int* blocks) {
  a.classes = row_classes(a.width, kVec<T>);
  if (pieces_width(a.width, kVec<T>) > kMaxRow) {
    const unsigned grid = (unsigned)(a.rows < 4 * sm_count() ? a.rows : 4 * sm_count());
    float* stats = nullptr;
    *blocks = (int)((a.rows + kLongRows - 1) / kLongRows);
    if (BWD && a.partials) stats = a.partials + (int64_t)*blocks * 2 * a.width;
    cudaError_t e = launch_early(layer_norm_long_kernel<T, BWD>, dim3(grid), kLongThreads, 0, s, a, stats);
    if (e != cudaSuccess || !stats) return e;
    return launch_early(layer_norm_columns_kernel<T>, dim3((unsigned)((a.width + 255) / 256), (unsigned)*blocks), 256, 0, s, a, (const float*)stats);
  }
  if (a.classes == 1) return launch_width<T, false, BWD>(a, s, blocks);
  return launch_width<T, true, BWD>(a, s, blocks);
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

bool layer_norm_rows_fit(int64_t ld, int width, int dtype) {
  const int vec = dtype == TRIFAST_F32 ? 4 : 8;
  return (ld - width) % vec == 0;
}

int64_t layer_norm_workspace_floats(int64_t rows, int width, int dtype) {
  const int vec = dtype == TRIFAST_F32 ? 4 : 8;
  if (pieces_width(width, vec) > kMaxRow) return (rows + kLongRows - 1) / kLongRows * 2 * width + 2 * rows;
  return bwd_blocks(rows, width, vec) * 2 * width;
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
