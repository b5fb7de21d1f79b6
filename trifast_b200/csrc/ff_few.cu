// The feed-forward block's forward pass for a few rows (a token or so at a time): both products on the CUDA cores, a
// warp to a hidden unit and then to a result, which read every weight once.  Hidden values are fp32.
//
// What bounds it: the launches, and the latency of one read of the weights (width 128, hidden 512, one row: 11.0 us a
// call on the tensor-core kernels, whose tiles are 128 rows and whose 2 x 4 tiles walk the contraction alone).

#include <type_traits>

#include "ff_gemm.cuh"
#include "tc_common.cuh"

namespace trifast {
namespace ff {
namespace {

constexpr int kWarps = 8;

// N neighbours as fp32: 16-byte reads, or one element.
template <typename T, int N>
__device__ __forceinline__ void read(const T* p, float* f) {
  if constexpr (N == 1) {
    f[0] = to_f32<T>(*p);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + e);
      f[e] = v.x;
      f[e + 1] = v.y;
      f[e + 2] = v.z;
      f[e + 3] = v.w;
    }
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    tc::unpack2<T>(v.x, f[0], f[1]);
    tc::unpack2<T>(v.y, f[2], f[3]);
    tc::unpack2<T>(v.z, f[4], f[5]);
    tc::unpack2<T>(v.w, f[6], f[7]);
  }
}

template <int R>
__device__ __forceinline__ void warp_sum(float* v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] += __shfl_xor_sync(0xffffffffu, v[r], m);
}

template <typename T, int R, int N>
__global__ void __launch_bounds__(32 * kWarps) few_hidden_kernel(const T* __restrict__ x, int64_t ld, int rows, const T* __restrict__ wg,
                                                                 const T* __restrict__ wu, float* __restrict__ h, int width, int hidden,
                                                                 int pitch) {
  after_previous();
  const int unit = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (unit >= hidden) return;
  float a[R] = {}, b[R] = {};
#pragma unroll 2
  for (int c = lane * N; c < width; c += 32 * N) {
    float g[N], u[N];
    read<T, N>(wg + (int64_t)unit * width + c, g);
    read<T, N>(wu + (int64_t)unit * width + c, u);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v[N];
      read<T, N>(x + min(r, rows - 1) * ld + c, v);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        a[r] = fmaf(v[e], g[e], a[r]);
        b[r] = fmaf(v[e], u[e], b[r]);
      }
    }
  }
  warp_sum<R>(a);
  warp_sum<R>(b);
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane == r && r < rows) h[r * pitch + unit] = a[r] / (1.f + expf(-a[r])) * b[r];
}

template <typename T, int R, int N>
__global__ void __launch_bounds__(32 * kWarps) few_result_kernel(const float* __restrict__ h, int rows, const T* __restrict__ wd, T* __restrict__ y,
                                                                 int hidden, int pitch, int width_out) {
  after_previous();
  const int o = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (o >= width_out) return;
  float s[R] = {};
#pragma unroll 2
  for (int c = lane * N; c < hidden; c += 32 * N) {
    float w[N];
    read<T, N>(wd + (int64_t)o * hidden + c, w);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v[N];
      read<float, N>(h + min(r, rows - 1) * pitch + c, v);
#pragma unroll
      for (int e = 0; e < N; ++e) s[r] = fmaf(v[e], w[e], s[r]);
    }
  }
  warp_sum<R>(s);
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane == r && r < rows) y[(int64_t)r * width_out + o] = from_f32<T>(s[r]);
}

template <typename T, int R>
cudaError_t launch(const FewArgs& a, cudaStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const int blocks = (a.hidden + kWarps - 1) / kWarps, outs = (a.width_out + kWarps - 1) / kWarps;
  const T *x = (const T*)a.x, *wg = (const T*)a.wg, *wu = (const T*)a.wu, *wd = (const T*)a.wd;
  const bool whole = a.width % N == 0 && (a.rows == 1 || a.ld % N == 0);
  cudaError_t e = launch_early(whole ? few_hidden_kernel<T, R, N> : few_hidden_kernel<T, R, 1>, dim3(blocks), 32 * kWarps, 0, s, x, a.ld, a.rows,
                               wg, wu, a.h, a.width, a.hidden, a.pitch);
  if (e != cudaSuccess) return e;
  return launch_early(a.hidden % N == 0 ? few_result_kernel<T, R, N> : few_result_kernel<T, R, 1>, dim3(outs), 32 * kWarps, 0, s,
                      (const float*)a.h, a.rows, wd, (T*)a.y, a.hidden, a.pitch, a.width_out);
}

template <typename T>
cudaError_t launch_rows(const FewArgs& a, cudaStream_t s) {
  return a.rows == 1 ? launch<T, 1>(a, s) : a.rows <= 4 ? launch<T, 4>(a, s) : launch<T, kFewRows>(a, s);
}

}  // namespace

cudaError_t few_rows(const FewArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case TRIFAST_F32: return launch_rows<float>(a, s);
    case TRIFAST_BF16: return launch_rows<__nv_bfloat16>(a, s);
    default: return launch_rows<__half>(a, s);
  }
}

}  // namespace ff
}  // namespace trifast
