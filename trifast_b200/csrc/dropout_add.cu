// Dropout with the residual sum, and its gradient (the same without a residual):
//     y = residual + keep x / (1 - p)
// keep is never stored.  Its entry i is word i % 4 of Philox-4x32 with ten rounds (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter (i / 4, offset) under the key
// `seed`, and keeps where the word, of 2^32, is not below p.  x is (outer, mid, inner) and the mask (outer,
// inner), shared along mid: a thread makes the words of its eight columns once and walks along mid with
// them.
//
// A dropped value is cleared bit by bit before the arithmetic, so that nothing of it enters.
//
// What bounds it: memory where the mask is shared (1,048,576 x 128 bf16: 128 us with a residual, 89 without, 6.3 and 6.0
// TB/s); the generator where every element has a word of its own (38.8 million bf16 elements about 50 us, 155 MB: 17 cycles a
// round and scheduler for two chains of two products).

#include "block_kernels.h"
#include "pieces.cuh"
#include "tc_common.cuh"

namespace trifast {
namespace {

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t block, uint64_t offset, uint64_t key) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint32_t ph = __umulhi(c0, 0xD2511F53u), qh = __umulhi(c2, 0xCD9E8D57u);
    uint32_t pl, ql;
    asm("mul.lo.u32 %0, %1, %2;" : "=r"(pl) : "r"(c0), "r"(0xD2511F53u));
    asm("mul.lo.u32 %0, %1, %2;" : "=r"(ql) : "r"(c2), "r"(0xCD9E8D57u));
    c0 = qh ^ c1 ^ k0;
    c1 = ql;
    c2 = ph ^ c3 ^ k1;
    c3 = pl;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// Eight words from mask entry `entry`, a multiple of eight, on.
__device__ __forceinline__ void words8(uint64_t entry, uint64_t offset, uint64_t key, uint32_t* w) {
  const Words lo = philox(entry / 4, offset, key), hi = philox(entry / 4 + 1, offset, key);
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = e < 4 ? lo.w[e] : hi.w[e - 4];
}

// Eight elements in 16-byte pieces (one of 16-bit types, two of fp32), and the bits that stay of them.
template <typename T> constexpr int kPieces = sizeof(T) / 2;
template <typename T> struct Eight { uint4 v[kPieces<T>]; };

template <typename T>
__device__ __forceinline__ Eight<T> keep_mask(const uint32_t* w, uint64_t threshold) {
  uint32_t k[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) k[e] = (uint64_t)w[e] >= threshold ? 0xffffffffu : 0u;
  Eight<T> m;
  if constexpr (sizeof(T) == 4) {
    m.v[0] = make_uint4(k[0], k[1], k[2], k[3]);
    m.v[1] = make_uint4(k[4], k[5], k[6], k[7]);
  } else {
    m.v[0] = make_uint4(__byte_perm(k[0], k[1], 0x5410), __byte_perm(k[2], k[3], 0x5410), __byte_perm(k[4], k[5], 0x5410),
                        __byte_perm(k[6], k[7], 0x5410));
  }
  return m;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float* f) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
  } else {
    tc::unpack2<T>(u.x, f[0], f[1]);
    tc::unpack2<T>(u.y, f[2], f[3]);
    tc::unpack2<T>(u.z, f[4], f[5]);
    tc::unpack2<T>(u.w, f[6], f[7]);
  }
}

// res + (x & mask) scale
template <typename T, bool RES>
__device__ __forceinline__ uint4 apply(uint4 x, const uint4& res, const uint4& m, float scale) {
  constexpr int N = 16 / sizeof(T);
  x.x &= m.x;
  x.y &= m.y;
  x.z &= m.z;
  x.w &= m.w;
  float f[N], r[N];
  unpack<T>(x, f);
  if (RES) unpack<T>(res, r);
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    if (RES)
      tc::ffma2(f[e], f[e + 1], f[e], f[e + 1], scale, scale, r[e], r[e + 1]);
    else
      tc::fmul2(f[e], f[e + 1], f[e], f[e + 1], scale, scale);
  }
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(tc::pack2<T>(f[0], f[1]), tc::pack2<T>(f[2], f[3]), tc::pack2<T>(f[4], f[5]), tc::pack2<T>(f[6], f[7]));
}

__device__ __forceinline__ uint64_t key_of(const DropoutArgs& a) { return a.seed + (a.seed_ptr ? (uint64_t)*a.seed_ptr : 0); }

// Eight words from any entry on (of which those before 0 mean nothing).
__device__ __forceinline__ void words8_at(int64_t entry, uint64_t offset, uint64_t key, uint32_t* w) {
  uint32_t all[12];
#pragma unroll
  for (int b = 0; b < 3; ++b) {
    const Words q = philox((uint64_t)((entry >> 2) + b), offset, key);
#pragma unroll
    for (int e = 0; e < 4; ++e) all[4 * b + e] = q.w[e];
  }
  const int skip = (int)(entry & 3);
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = skip & 2 ? (skip & 1 ? all[e + 3] : all[e + 2]) : (skip & 1 ? all[e + 1] : all[e]);
}

// Shared masks whose inner extent is a multiple of eight: a thread has eight columns and `walk` steps of mid, `mids`
// apart.  Columns run fastest over the threads, then the first `mids` steps of mid, then outer.
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_shared_kernel(DropoutArgs a, int64_t cols, int64_t mids, int walk) {
  constexpr int U = 4, N = kPieces<T>;   // steps in flight
  after_previous();
  const uint64_t key = key_of(a);
  const int64_t total = a.outer * mids * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t col = i % cols, om = i / cols, m0 = om % mids, o = om / mids;
    uint32_t w[8];
    words8((uint64_t)(o * a.inner + col * 8), a.offset, key, w);
    const Eight<T> mask = keep_mask<T>(w, a.threshold);
    const int64_t first = (o * a.mid + m0) * a.inner + col * 8, step = mids * a.inner;   // elements
    const int steps = (int)min((int64_t)walk, (a.mid - m0 + mids - 1) / mids);
    const T* x = reinterpret_cast<const T*>(a.x) + first;
    const T* r = reinterpret_cast<const T*>(a.residual) + first;
    T* y = reinterpret_cast<T*>(a.y) + first;
    int s = 0;
    for (; s + U <= steps; s += U, x += U * step, r += U * step, y += U * step) {
      uint4 vx[U][N], vr[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < N; ++k) {
          vx[u][k] = reinterpret_cast<const uint4*>(x + u * step)[k];
          if (RES) vr[u][k] = reinterpret_cast<const uint4*>(r + u * step)[k];
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < N; ++k) reinterpret_cast<uint4*>(y + u * step)[k] = apply<T, RES>(vx[u][k], vr[u][k], mask.v[k], a.scale);
    }
    for (; s < steps; ++s, x += step, r += step, y += step) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const uint4 vr = RES ? reinterpret_cast<const uint4*>(r)[k] : make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(y)[k] = apply<T, RES>(reinterpret_cast<const uint4*>(x)[k], vr, mask.v[k], a.scale);
      }
    }
  }
}

// Every element its own word: the tensor as one row of pieces of eight, two of them a thread at a time; the last
// elements one by one.
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_own_kernel(DropoutArgs a) {
  constexpr int N = kPieces<T>;
  after_previous();
  const uint64_t key = key_of(a);
  const int64_t pieces = a.inner / 8, stride = (int64_t)gridDim.x * 256;
  const uint4* x = reinterpret_cast<const uint4*>(a.x);
  const uint4* r = reinterpret_cast<const uint4*>(a.residual);
  uint4* y = reinterpret_cast<uint4*>(a.y);
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t i = i0; i < pieces; i += 2 * stride) {
    uint4 vx[2][N], vr[2][N];
    Eight<T> mask[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (i + u * stride < pieces)
#pragma unroll
        for (int k = 0; k < N; ++k) {
          vx[u][k] = x[(i + u * stride) * N + k];
          if (RES) vr[u][k] = r[(i + u * stride) * N + k];
        }
    // (four blocks of words side by side: a round is one chain of products)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t w[8];
      words8((uint64_t)(i + u * stride) * 8, a.offset, key, w);
      mask[u] = keep_mask<T>(w, a.threshold);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (i + u * stride < pieces)
#pragma unroll
        for (int k = 0; k < N; ++k) y[(i + u * stride) * N + k] = apply<T, RES>(vx[u][k], vr[u][k], mask[u].v[k], a.scale);
  }
  if (i0 < a.inner % 8) {
    const int64_t e = pieces * 8 + i0;
    const Words b = philox((uint64_t)e / 4, a.offset, key);
    const int at = (int)(e % 4);
    const uint32_t w = at == 0 ? b.w[0] : at == 1 ? b.w[1] : at == 2 ? b.w[2] : b.w[3];
    const float v = (uint64_t)w >= a.threshold ? to_f32<T>(reinterpret_cast<const T*>(a.x)[e]) : 0.f;
    reinterpret_cast<T*>(a.y)[e] =
        from_f32<T>(RES ? fmaf(v, a.scale, to_f32<T>(reinterpret_cast<const T*>(a.residual)[e])) : v * a.scale);
  }
}

// (1000 x 1000 maps with one mask for all columns, bf16, a column a thread and in pieces: 9 places 20 and 23 us, 33 84 and 49)
constexpr int kShiftInner = 16;

// Shared masks of other inner extents: the rows (o, m) begin inside 16-byte pieces, at the same place for every
// `classes`-th m.  A thread has eight places that begin with a piece and the steps m0, m0 + mids, ... of mid, `mids` a
// multiple of the classes: it reads whole pieces and writes what the row has of them.  (1024 x 1024 x 127 bf16 with one mask
// for all columns and a residual: 137 us; one column a thread 279; 128 columns 132.)
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_shift_kernel(DropoutArgs a, int64_t cols, int64_t mids) {
  constexpr int U = 2, N = kPieces<T>, V = 16 / sizeof(T);   // steps in flight, pieces and elements of one
  after_previous();
  const uint64_t key = key_of(a);
  const int64_t total = a.outer * mids * cols, step = mids * a.inner;
  const T *xs = reinterpret_cast<const T*>(a.x), *rs = reinterpret_cast<const T*>(a.residual);
  const int64_t end = a.outer * a.mid * a.inner;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t p = i % cols, om = i / cols, m0 = om % mids, o = om / mids;
    if (m0 >= a.mid) continue;
    const int64_t row = (o * a.mid + m0) * a.inner;
    const int shift = (int)(row % V);
    const int64_t col = p * 8 - shift;
    if (col >= a.inner) continue;
    uint32_t w[8];
    words8_at(o * a.inner + col, a.offset, key, w);
    const Eight<T> mask = keep_mask<T>(w, a.threshold);
    int lo[N], hi[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      lo[k] = (int)max((int64_t)0, -col - k * V);
      hi[k] = (int)min((int64_t)V, a.inner - col - k * V);
    }
    auto load = [&](const T* t, int64_t e) {   // nothing behind the tensor's end
      if (e + V <= end) return *reinterpret_cast<const uint4*>(t + e);
      T v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = e + j < end ? t[e + j] : from_f32<T>(0.f);
      uint4 u;
      memcpy(&u, v, 16);
      return u;
    };
    int64_t e = row + col;
    for (int64_t m = m0; m < a.mid; m += U * mids, e += U * step) {
      uint4 vx[U][N], vr[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (m + u * mids < a.mid)
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (hi[k] > 0) {
              vx[u][k] = load(xs, e + u * step + k * V);
              if (RES) vr[u][k] = load(rs, e + u * step + k * V);
            }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (m + u * mids < a.mid)
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (hi[k] > 0) {   // (a row of kShiftInner places ends in another piece than it begins in)
              T* to = reinterpret_cast<T*>(a.y) + e + u * step + k * V;
              const uint4 v = apply<T, RES>(vx[u][k], vr[u][k], mask.v[k], a.scale);
              if (lo[k] == 0 && hi[k] == V)
                *reinterpret_cast<uint4*>(to) = v;
              else
                store_part(to, v, lo[k] > 0, lo[k] > 0 ? V - lo[k] : hi[k]);
            }
    }
  }
}

// Shared masks of few places, of which the pieces would be edges for the most part: a thread has one column.
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_column_kernel(DropoutArgs a, int64_t mids) {
  after_previous();
  const uint64_t key = key_of(a);
  const int64_t total = a.outer * mids * a.inner;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t col = i % a.inner, om = i / a.inner, m0 = om % mids, o = om / mids;
    const uint64_t entry = (uint64_t)(o * a.inner + col);
    const Words b = philox(entry / 4, a.offset, key);
    const int at = (int)(entry % 4);
    const uint32_t w = at == 0 ? b.w[0] : at == 1 ? b.w[1] : at == 2 ? b.w[2] : b.w[3];
    const bool keep = (uint64_t)w >= a.threshold;
    int64_t e = (o * a.mid + m0) * a.inner + col;
#pragma unroll 4
    for (int64_t m = m0; m < a.mid; m += mids, e += mids * a.inner) {
      const float v = keep ? to_f32<T>(reinterpret_cast<const T*>(a.x)[e]) : 0.f;
      reinterpret_cast<T*>(a.y)[e] =
          from_f32<T>(RES ? fmaf(v, a.scale, to_f32<T>(reinterpret_cast<const T*>(a.residual)[e])) : v * a.scale);
    }
  }
}

unsigned blocks_for(int64_t threads, int64_t most) {
  const int64_t b = (threads + 255) / 256;
  return (unsigned)(b < most ? b : most);
}

template <typename T, bool RES>
cudaError_t launch_type(DropoutArgs a, cudaStream_t s) {
  const int64_t sms = sm_count();
  if (a.mid == 1) {   // (no entry has two elements)
    a.inner *= a.outer;
    a.outer = 1;
    const int64_t threads = a.inner / 16 > a.inner % 8 ? a.inner / 16 : a.inner % 8;
    return launch_early(dropout_own_kernel<T, RES>, dim3(blocks_for(threads < 1 ? 1 : threads, sms * 8)), 256, 0, s, a);
  }
  const bool whole = a.inner % 8 == 0, few = a.inner < kShiftInner;
  const int vec = 16 / (int)sizeof(T), classes = row_classes(a.inner, vec);
  const int64_t cols = whole ? a.inner / 8 : few ? a.inner : (a.inner + vec - 1 + 7) / 8, lanes = a.outer * cols;
  // Steps of mid that a thread walks with one mask: as many as leave eight blocks of 256 threads a multiprocessor.
  int64_t walk = lanes * a.mid / (sms * 8 * 256);
  walk = walk < 1 ? 1 : walk > 64 ? 64 : walk;
  if (walk > a.mid) walk = a.mid;
  int64_t mids = (a.mid + walk - 1) / walk;
  if (!whole && !few) mids = (mids + classes - 1) / classes * classes;
  const unsigned blocks = blocks_for(lanes * mids, 1 << 30);
  if (whole) return launch_early(dropout_shared_kernel<T, RES>, dim3(blocks), 256, 0, s, a, cols, mids, (int)walk);
  if (few) return launch_early(dropout_column_kernel<T, RES>, dim3(blocks), 256, 0, s, a, mids);
  return launch_early(dropout_shift_kernel<T, RES>, dim3(blocks), 256, 0, s, a, cols, mids);
}

}  // namespace

cudaError_t dropout_add(const DropoutArgs& a, cudaStream_t s) {
  const bool r = a.residual != nullptr;
  switch (a.dtype) {
    case TRIFAST_F32: return r ? launch_type<float, true>(a, s) : launch_type<float, false>(a, s);
    case TRIFAST_BF16: return r ? launch_type<__nv_bfloat16, true>(a, s) : launch_type<__nv_bfloat16, false>(a, s);
    default: return r ? launch_type<__half, true>(a, s) : launch_type<__half, false>(a, s);
  }
}

}  // namespace trifast
