// Dropout with the residual sum, and its gradient (the same without a residual):
//     y = residual + keep x / (1 - p)
// keep is never stored.  Its entry i is word i % 4 of Philox-4x32 with ten rounds (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter (i / 4, offset) under the key
// `seed`, and keeps where the word, of 2^32, is not below p.  x is (outer, mid, inner) and the mask (outer,
// inner), shared along mid: a thread makes the words of its eight columns once and walks along mid with
// them.
//
// What bounds it: memory where the mask is shared.

#include "block_kernels.h"

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
    const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)q;
    c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Piece { T v[VEC]; };

// A thread: VEC columns of inner (8 elements, or one where they cannot be read whole), `walk` steps of mid.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) dropout_add_kernel(DropoutArgs a, int64_t cols, int64_t mids, int walk) {
  constexpr int U = 4;   // loads in flight
  using P = Piece<T, VEC>;
  after_previous();
  const uint64_t key = a.seed + (a.seed_ptr ? (uint64_t)*a.seed_ptr : 0);
  const int64_t total = a.outer * mids * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    // columns run fastest, then the first `mids` steps of mid, then outer
    const int64_t col = i % cols, om = i / cols, m0 = om % mids, o = om / mids;
    const uint64_t entry = (uint64_t)(o * a.inner + col * VEC);
    uint32_t word[VEC];
    if constexpr (VEC == 8) {
      if (entry % 4 == 0) {
        const Words lo = philox(entry / 4, a.offset, key), hi = philox(entry / 4 + 1, a.offset, key);
#pragma unroll
        for (int e = 0; e < 8; ++e) word[e] = e < 4 ? lo.w[e] : hi.w[e - 4];
      } else {
        const Words b[3] = {philox(entry / 4, a.offset, key), philox(entry / 4 + 1, a.offset, key), philox(entry / 4 + 2, a.offset, key)};
        const int skip = (int)(entry % 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          word[e] = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k == skip) word[e] = b[(e + k) / 4].w[(e + k) % 4];
        }
      }
    } else {
      const Words b = philox(entry / 4, a.offset, key);
      const int at = (int)(entry % 4);
      word[0] = at == 0 ? b.w[0] : at == 1 ? b.w[1] : at == 2 ? b.w[2] : b.w[3];
    }
    uint32_t keep = 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) keep |= (uint32_t)((uint64_t)word[e] >= a.threshold) << e;
    for (int w0 = 0; w0 < walk; w0 += U) {
      P x[U], r[U];
      int64_t at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t m = m0 + (int64_t)(w0 + u) * mids;
        const bool in = w0 + u < walk && m < a.mid;
        at[u] = in ? (o * a.mid + m) * a.inner + col * VEC : -1;
        if (in) {
          x[u] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(a.x) + at[u]);
          if (a.residual) r[u] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(a.residual) + at[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (at[u] < 0) continue;
        P y;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          // (a dropped value does not enter: not an infinity or NaN either)
          float v = (keep >> e) & 1 ? to_f32<T>(x[u].v[e]) * a.scale : 0.f;
          if (a.residual) v += to_f32<T>(r[u].v[e]);
          y.v[e] = from_f32<T>(v);
        }
        *reinterpret_cast<P*>(reinterpret_cast<T*>(a.y) + at[u]) = y;
      }
    }
  }
}

template <typename T, int VEC>
cudaError_t launch_vec(const DropoutArgs& a, cudaStream_t s) {
  const int64_t cols = a.inner / VEC, lanes = a.outer * cols;
  // Steps of mid that a thread walks with one mask: as many as leave eight blocks of 256 threads a multiprocessor.
  const int64_t want = (int64_t)sm_count() * 8 * 256;
  int64_t walk = lanes * a.mid / want;
  if (walk < 1) walk = 1;
  if (walk > a.mid) walk = a.mid;
  if (walk > 64) walk = 64;
  const int64_t mids = (a.mid + walk - 1) / walk, total = lanes * mids;
  const int64_t blocks = (total + 255) / 256;
  return launch_early(dropout_add_kernel<T, VEC>, dim3((unsigned)(blocks < 1 << 30 ? blocks : 1 << 30)), 256, 0, s, a, cols, mids, (int)walk);
}

template <typename T>
cudaError_t launch_type(const DropoutArgs& a, cudaStream_t s) {
  constexpr uintptr_t kBytes = 8 * sizeof(T);
  auto whole = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & (kBytes - 1)) == 0; };
  if (a.inner % 8 == 0 && whole(a.x) && whole(a.residual) && whole(a.y)) return launch_vec<T, 8>(a, s);
  return launch_vec<T, 1>(a, s);
}

}  // namespace

cudaError_t dropout_add(const DropoutArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case TRIFAST_F32: return launch_type<float>(a, s);
    case TRIFAST_BF16: return launch_type<__nv_bfloat16>(a, s);
    default: return launch_type<__half>(a, s);
  }
}

}  // namespace trifast
