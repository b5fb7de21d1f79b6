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
// threads keep their columns.  What a piece holds of other rows is replaced.
//
// What bounds it: memory (1,048,576 x 128 bf16: 87 us forward, 135 backward, 6.2 and 6.0 TB/s); with SHIFT the instructions
// of its edges and the registers of their masks (65,536 x 1999 bf16: 110 and 222 us, 2000: 94 and 161).  Rows beyond 8192
// elements (kMaxRow) are walked in passes instead.

#include <type_traits>

#include "block_kernels.h"
#include "pieces.cuh"
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
// call sites at least in a loop (a thread that is a call behind still reads the other's); no_sums() before the first.
template <int TPR, int N>
__device__ __forceinline__ void no_sums(float (*buf)[N][32]) {   // of the warps that the block has not
  if constexpr (TPR > 32)
    for (int i = threadIdx.x; i < 2 * N * 32; i += blockDim.x) {
      const int w = i % 32;
      if (w * 32 >= (int)blockDim.x) buf[i / 32 / N][i / 32 % N][w] = 0.f;
    }
}
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

// Threads of a block, of one of whole rows at most: it has as many warps as its row needs.
template <int TPR> constexpr int kBlock = TPR > 32 ? TPR : 256;
// Blocks a multiprocessor that the registers are held down for (0: as they come).
template <int TPR, int E, bool SHIFT, bool BWD>
constexpr int kResident = !SHIFT ? 0 : TPR <= 32 || TPR == 256 || TPR == 320 ? 2 : !BWD && TPR == 160 && E == 16 ? 3 : 0;
template <int TPR> __device__ __forceinline__ int row_threads() { return TPR > 32 ? (int)blockDim.x : TPR; }

// The pieces of a row that a thread has: piece k begins at column (k * threads + lane) * VEC - shift.
//
// With SHIFT the first piece and the last one have places that are not the row's.  In x they get a value of the row's from
// the same piece, which then counts n times too often: the sum takes n of them back, the sum of squares n of their
// deviations' (which are no larger than what stays: nothing cancels).  In dy they are zero.
template <typename T, int TPR, int K, bool SHIFT>
struct RowPieces {
  static constexpr int VEC = kVec<T>, E = K * VEC;
  int lane, threads, width, shift;
  int64_t rows;
  float before, behind[K];   // places of the first piece, and of each other, that are not the row's
  uint32_t own0[4], own1[4];  // the bits that are the row's: of piece 0, and of the last piece if that is another

  __device__ __forceinline__ RowPieces(int lane, int threads, int width, int shift, int64_t rows)
      : lane(lane), threads(threads), width(width), shift(shift), rows(rows) {
    before = SHIFT && lane == 0 && shift > 0 ? (float)(shift + max(0, VEC - shift - width)) : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) behind[k] = SHIFT && any(k) && !first(k) ? (float)max(0, col(k) + VEC - width) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      own0[i] = SHIFT ? own(0, i) : 0;
      own1[i] = 0;
#pragma unroll
      for (int k = 1; k < K; ++k)
        if (SHIFT && any(k)) own1[i] = own(k, i);
    }
  }
  __device__ __forceinline__ int col(int k) const { return (k * threads + lane) * VEC - (SHIFT ? shift : 0); }
  __device__ __forceinline__ bool any(int k) const { return col(k) < width; }
  __device__ __forceinline__ bool has(int k, int e) const {
    return SHIFT ? (unsigned)(col(k) + e) < (unsigned)width : any(k);
  }
  // Whether some places of the piece are not the row's: before its first element, or behind its last one.
  __device__ __forceinline__ bool first(int k) const { return SHIFT && k == 0 && col(0) < 0; }
  __device__ __forceinline__ bool last(int k) const { return SHIFT && col(k) + VEC > width; }
  __device__ __forceinline__ bool edge(int k) const { return any(k) && (first(k) || last(k)); }

  // Row `row` of `tensor`, zeros behind the last one.  (Nothing is read behind the tensor's end; before its beginning lies
  // nothing of a piece: the first row's shift is 0.)
  __device__ __forceinline__ void load(uint4* r, const void* tensor, int64_t ld, int64_t row) const {
    const T* p = reinterpret_cast<const T*>(tensor) + row * ld;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      r[k] = make_uint4(0, 0, 0, 0);
      if (row >= rows || !any(k)) continue;
      if (last(k) && row + VEC >= rows) {   // (VEC rows more are VEC elements at least)
        T t[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) t[e] = has(k, e) ? p[col(k) + e] : from_f32<T>(0.f);
        memcpy(&r[k], t, 16);
      } else {
        r[k] = *reinterpret_cast<const uint4*>(p + col(k));
      }
    }
  }
  // The bits of word i of piece k that are the row's.
  __device__ __forceinline__ uint32_t own(int k, int i) const {
    if constexpr (VEC == 4) return has(k, i) ? ~0u : 0u;
    return (has(k, 2 * i) ? 0xffffu : 0u) | (has(k, 2 * i + 1) ? 0xffff0000u : 0u);
  }
  // The values; in the other places a value of the row's (FILL) or 0.
  template <bool FILL>
  __device__ __forceinline__ void values(const uint4* r, float* f) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      uint4 v = r[k];
      if (edge(k)) {
        uint32_t fill = 0;
        if constexpr (FILL) {   // the piece's last value or its first one
          fill = first(k) ? v.w : v.x;
          if constexpr (VEC == 8) fill = __byte_perm(fill, 0, first(k) ? 0x3232 : 0x1010);
          if (first(k) && last(k)) {
            const int word = VEC == 4 ? shift : shift >> 1;
            fill = word & 2 ? (word & 1 ? v.w : v.z) : (word & 1 ? v.y : v.x);
            if constexpr (VEC == 8) fill = __byte_perm(fill, 0, shift & 1 ? 0x3232 : 0x1010);
          }
        }
        const uint32_t* m = k == 0 ? own0 : own1;
        v = make_uint4((v.x & m[0]) | (fill & ~m[0]), (v.y & m[1]) | (fill & ~m[1]), (v.z & m[2]) | (fill & ~m[2]), (v.w & m[3]) | (fill & ~m[3]));
      }
      unpack<T>(v, f + k * VEC);
    }
  }
  // What the places that are not the row's have added to a sum of f, or of its squares.
  __device__ __forceinline__ float sum(const float* f) const {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int e = 0; e < E; e += 2) fadd2(s0, s1, s0, s1, f[e], f[e + 1]);
    if constexpr (SHIFT) {
      s0 = fmaf(-before, f[0], s0);
#pragma unroll
      for (int k = 0; k < K; ++k) s1 = fmaf(-behind[k], f[k * VEC + VEC - 1], s1);
    }
    return s0 + s1;
  }
  __device__ __forceinline__ float squares(const float* f) const {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int e = 0; e < E; e += 2) ffma2(s0, s1, f[e], f[e + 1], f[e], f[e + 1], s0, s1);
    if constexpr (SHIFT) {
      s0 = fmaf(-before * f[0], f[0], s0);
#pragma unroll
      for (int k = 0; k < K; ++k) s1 = fmaf(-behind[k] * f[k * VEC + VEC - 1], f[k * VEC + VEC - 1], s1);
    }
    return s0 + s1;
  }
  // f - mean; pieces behind the row stay 0.
  __device__ __forceinline__ void center(float* f, float mean) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float m = any(k) ? mean : 0.f;
#pragma unroll
      for (int e = 0; e < VEC; e += 2) fadd2(f[k * VEC + e], f[k * VEC + e + 1], f[k * VEC + e], f[k * VEC + e + 1], -m, -m);
    }
  }
  __device__ __forceinline__ void store(T* p, const float* f) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!any(k)) continue;
      T* to = p + col(k);
      const uint4 v = pack<T>(f + k * VEC);
      if (!edge(k)) {
        *reinterpret_cast<uint4*>(to) = v;
      } else if (first(k) && last(k)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (has(k, e)) to[e] = from_f32<T>(f[k * VEC + e]);
      } else {
        store_part(to, v, first(k), first(k) ? VEC - shift : width - col(k));
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
__device__ __forceinline__ float dot_of(const float* f, const float* g) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int e = 0; e < E; e += 2) ffma2(s0, s1, f[e], f[e + 1], g[e], g[e + 1], s0, s1);
  return s0 + s1;
}

template <typename T, int TPR, int K, int R, bool SHIFT>
__global__ void __launch_bounds__(kBlock<TPR>, (kResident<TPR, K * kVec<T>, SHIFT, false>)) layer_norm_fwd_kernel(LayerNormArgs a) {
  constexpr int kGroups = kBlock<TPR> / TPR;
  using P = RowPieces<T, TPR, K, SHIFT>;
  constexpr int E = P::E;
  __shared__ float buf[2][R][32];
  const int grp = TPR > 32 ? 0 : threadIdx.x / TPR;
  const BlockRows rows = block_rows<SHIFT>(a, kVec<T>, kGroups * R);
  const P p((int)(threadIdx.x - grp * TPR), row_threads<TPR>(), a.width, rows.shift, a.rows);
  const float inv_width = 1.f / (float)a.width;
  no_sums<TPR, R>(buf);
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
      p.template values<true>(raw[r], f[r]);
      mean[r] = p.sum(f[r]);
    }
    if (base + rows.stride < a.rows) load(base + rows.stride);   // on their way meanwhile
    row_sums<TPR, R>(mean, buf[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      p.center(f[r], mean[r] * inv_width);
      rstd[r] = p.squares(f[r]);
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
__global__ void __launch_bounds__(kBlock<TPR>, (kResident<TPR, K * kVec<T>, SHIFT, true>)) layer_norm_bwd_kernel(LayerNormArgs a) {
  constexpr int kGroups = kBlock<TPR> / TPR;
  using P = RowPieces<T, TPR, K, SHIFT>;
  constexpr int E = P::E, VEC = P::VEC;
  __shared__ float buf[2][2 * R][32];
  const int grp = TPR > 32 ? 0 : threadIdx.x / TPR;
  const BlockRows rows = block_rows<SHIFT>(a, VEC, kGroups * R);
  const P p((int)(threadIdx.x - grp * TPR), row_threads<TPR>(), a.width, rows.shift, a.rows);
  const float inv_width = 1.f / (float)a.width;
  no_sums<TPR, 2 * R>(buf);
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
      p.template values<true>(raw_x[r], f[r]);
      p.template values<false>(raw_dy[r], d[r]);     // (0 behind the last row)
      s[2 * r] = p.sum(f[r]);
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
      t[2 * r] = p.squares(f[r]);
      t[2 * r + 1] = t0 + t1;
    }
    row_sums<TPR, 2 * R>(t, buf[1]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + (r * kGroups + grp) * rows.step;
      // (0 behind the last row: its zeros have no variance, and without an eps the inverse of that would reach dw)
      const float rstd = row < a.rows ? rsqrtf(fmaf(t[2 * r], inv_width, a.eps)) : 0.f;
      const float m1 = s[2 * r + 1] * inv_width, m2 = t[2 * r + 1] * rstd * inv_width;
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
// Threads a row (of a whole block: at most) and elements a thread, by the elements of its pieces.
struct RowShape {
  int tpr, e;
};
// Sixteen elements a thread where the registers allow it: fewer sums between threads.  The masks of SHIFT cost up to 25
// registers, so its rows of fp32 (four pieces of sixteen elements) take eight up to 256, and its wide rows more threads of
// eight, or one row at a time of two blocks a multiprocessor: a block alone waits at its sums with nothing beside it
// (32,768 rows of 4095: bf16 forward 484 us with 512 threads for their 288, 203 with eight elements, 137 so).
template <typename T, bool SHIFT, bool BWD>
constexpr RowShape row_shape(int width) {
  constexpr bool f32 = std::is_same<T, float>::value;
  if (SHIFT && f32 && width <= 256)
    return width <= 32 ? RowShape{4, 8} : width <= 64 ? RowShape{8, 8} : width <= 128 ? RowShape{16, 8} : RowShape{32, 8};
  if (SHIFT && width > 2560 && width <= 5120) {
    if (!f32 && !BWD) return {320, 16};
    if (f32 || width > 4096) return {640, 8};
  }
  if (!SHIFT && f32 && BWD && width > 4096 && width <= 5120) return {640, 8};
  return width <= 64 ? RowShape{4, 16}
         : width <= 128 ? RowShape{8, 16}
         : width <= 256 ? RowShape{16, 16}
         : width <= 512 ? RowShape{32, 16}
         : width <= 1280 ? RowShape{160, 8}
         : width <= 2560 ? RowShape{160, 16}
         : width <= 4096 ? RowShape{256, 16}
                         : RowShape{512, 16};
}
// (all of its bounds are multiples of 32)
template <typename T, bool SHIFT, bool BWD>
constexpr bool shape_used(int tpr, int e) {
  for (int w = 32; w <= kMaxRow; w += 32) {
    const RowShape r = row_shape<T, SHIFT, BWD>(w);
    if (r.tpr == tpr && r.e == e) return true;
  }
  return false;
}
// The elements of a row's pieces.
int pieces_width(int width, int vec) { return row_classes(width, vec) > 1 ? width + vec - 1 : width; }
// Blocks of the backward at most: eight a multiprocessor (three of wide rows, whose partial sums are wide too).
constexpr int most_blocks(int tpr) { return 148 * (tpr > 160 ? 3 : 8); }

int64_t bwd_blocks(int64_t rows, int width, int vec) {
  const int classes = row_classes(width, vec), w = pieces_width(width, vec);
  const RowShape r = vec == 4 ? (classes > 1 ? row_shape<float, true, true>(w) : row_shape<float, false, true>(w))
                              : (classes > 1 ? row_shape<__half, true, true>(w) : row_shape<__half, false, true>(w));
  const int tpr = r.tpr;
  const int64_t per = tpr > 32 ? 1 : 256 / tpr, b = (rows + per - 1) / per;
  const int64_t most = b < most_blocks(tpr) ? b : most_blocks(tpr);
  return (most + classes - 1) / classes * classes;
}

template <auto Kernel>
int blocks_per_sm(int threads) {
  static std::atomic<int> known[32];   // by the block's warps
  int b = known[threads / 32].load(std::memory_order_relaxed);
  if (b == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&b, Kernel, threads, 0) != cudaSuccess || b < 1) b = 1;
    known[threads / 32].store(b, std::memory_order_relaxed);
  }
  return b;
}

template <typename T, int TPR, int E, bool SHIFT, bool BWD>
cudaError_t launch_row(const LayerNormArgs& a, cudaStream_t s, int* blocks) {
  // rows that a group of threads works on at a time; in the backward two where it is a block of up to 160, which waits
  // for all of its threads twice a turn (more threads leave no registers for it)
  constexpr int R = (BWD && TPR != 160) || TPR == 320 ? 1 : 2, K = E / kVec<T>;
  const int pieces = (pieces_width(a.width, kVec<T>) + kVec<T> - 1) / kVec<T>;
  const int threads = TPR > 32 ? (pieces + 32 * K - 1) / (32 * K) * 32 : kBlock<TPR>;
  constexpr auto kern = [] {
    if constexpr (BWD) return &layer_norm_bwd_kernel<T, TPR, K, R, SHIFT>;
    else return &layer_norm_fwd_kernel<T, TPR, K, R, SHIFT>;
  }();
  const int64_t per = (TPR > 32 ? 1 : threads / TPR) * R, need = (a.rows + per - 1) / per;
  int64_t most = (int64_t)sm_count() * blocks_per_sm<kern>(threads);
  if (BWD && most > most_blocks(TPR)) most = most_blocks(TPR);
  // whole classes of blocks, and no more than run at a time: a few that came after the others would double the time
  const int64_t classes = SHIFT ? a.classes : 1, all = (need + classes - 1) / classes * classes;
  most = most < classes ? classes : most / classes * classes;
  *blocks = (int)(all < most ? all : most);
  return launch_early(kern, dim3((unsigned)*blocks), threads, 0, s, a);
}

template <typename T, bool SHIFT, bool BWD>
cudaError_t launch_width(const LayerNormArgs& a, cudaStream_t s, int* blocks) {
  const RowShape r = row_shape<T, SHIFT, BWD>(pieces_width(a.width, kVec<T>));
  cudaError_t error = cudaErrorInvalidValue;
  auto with = [&](auto tpr, auto e) {
    constexpr int TPR = decltype(tpr)::value, E = decltype(e)::value;
    if constexpr (shape_used<T, SHIFT, BWD>(TPR, E))
      if (r.tpr == TPR && r.e == E) error = launch_row<T, TPR, E, SHIFT, BWD>(a, s, blocks);
  };
  using std::integral_constant;
  auto both = [&](auto tpr) {
    with(tpr, integral_constant<int, 8>{});
    with(tpr, integral_constant<int, 16>{});
  };
  both(integral_constant<int, 4>{});
  both(integral_constant<int, 8>{});
  both(integral_constant<int, 16>{});
  both(integral_constant<int, 32>{});
  both(integral_constant<int, 160>{});
  both(integral_constant<int, 256>{});
  both(integral_constant<int, 320>{});
  both(integral_constant<int, 512>{});
  both(integral_constant<int, 640>{});
  return error;
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

bool layer_norm_in_passes(int width, int dtype) { return pieces_width(width, dtype == TRIFAST_F32 ? 4 : 8) > kMaxRow; }

int64_t layer_norm_workspace_floats(int64_t rows, int width, int dtype) {
  const int vec = dtype == TRIFAST_F32 ? 4 : 8;
  if (layer_norm_in_passes(width, dtype)) return (rows + kLongRows - 1) / kLongRows * 2 * width + 2 * rows;
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
