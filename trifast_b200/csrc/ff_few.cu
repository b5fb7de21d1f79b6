// The feed-forward block's forward pass for a few rows (a token or so at a time): both products on the CUDA cores, a
// warp to a hidden unit and then a warp or a block to a result, which read every weight once.  Hidden values are fp32.
//
// What bounds it: the launches, and the latency of one read of the weights.  Small blocks (a megabyte of weights) are
// one kernel, a cluster of eight CTAs whose warps write their hidden values into the shared memory of all eight; larger
// ones two kernels over all multiprocessors.  (Width 128, hidden 512, one row: 11.0 us a call on the tensor-core
// kernels, whose tiles are 128 rows, 9.5 as two kernels.)

#include <type_traits>

#include "ff_device.cuh"

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

// The sums of a block's eight warps, in all of them.
template <int R>
__device__ __forceinline__ void block_sum(float* v) {
  __shared__ float sum[kWarps][R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane == r) sum[warp][r] = v[r];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    v[r] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v[r] += sum[w][r];
  }
}

// silu(x wg^T) * (x wu^T) of one hidden unit: in lane r that of row r
template <typename T, int R, int N>
__device__ __forceinline__ float unit_value(const T* __restrict__ x, int64_t ld, int rows, const T* __restrict__ wg, const T* __restrict__ wu,
                                            int width, int lane) {
  float a[R] = {}, b[R] = {};
#pragma unroll 2
  for (int c = lane * N; c < width; c += 32 * N) {
    float g[N], u[N];
    read<T, N>(wg + c, g);
    read<T, N>(wu + c, u);
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
  float h = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane == r) h = a[r] / (1.f + expf(-a[r])) * b[r];
  return h;
}

// One result: in lane r that of row r (h: rows `pitch` apart).  BLOCK: by the eight warps of a block together.
template <typename T, int R, int N, bool BLOCK>
__device__ __forceinline__ float result_value(const float* h, int rows, const T* __restrict__ wd, int hidden, int pitch, int lane) {
  constexpr int kLanes = BLOCK ? 32 * kWarps : 32;
  float s[R] = {};
#pragma unroll 2
  for (int c = (BLOCK ? (int)threadIdx.x : lane) * N; c < hidden; c += kLanes * N) {
    float w[N];
    read<T, N>(wd + c, w);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v[N];
      read<float, N>(h + min(r, rows - 1) * pitch + c, v);
#pragma unroll
      for (int e = 0; e < N; ++e) s[r] = fmaf(v[e], w[e], s[r]);
    }
  }
  warp_sum<R>(s);
  if constexpr (BLOCK) block_sum<R>(s);
  float y = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane == r) y = s[r];
  return y;
}

template <typename T, int R, int N>
__global__ void __launch_bounds__(32 * kWarps) few_hidden_kernel(FewArgs p) {
  after_previous();
  const int unit = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (unit >= p.hidden) return;
  const float h = unit_value<T, R, N>((const T*)p.x, p.ld, p.rows, (const T*)p.wg + (int64_t)unit * p.width, (const T*)p.wu + (int64_t)unit * p.width,
                                      p.width, lane);
  if (lane < p.rows) p.h[lane * p.pitch + unit] = h;
}

template <typename T, int R, int N, bool BLOCK>
__global__ void __launch_bounds__(32 * kWarps) few_result_kernel(FewArgs p) {
  after_previous();
  const int o = BLOCK ? blockIdx.x : blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (o >= p.width_out) return;
  const float y = result_value<T, R, N, BLOCK>(p.h, p.rows, (const T*)p.wd + (int64_t)o * p.hidden, p.hidden, p.pitch, lane);
  if ((BLOCK ? (int)threadIdx.x : lane) < p.rows) ((T*)p.y)[(int64_t)lane * p.width_out + o] = from_f32<T>(y);
}

// Both, by a cluster.  N, M: neighbours read at a time along the width and along the hidden units.
constexpr int kClusterCtas = 8, kClusterThreads = 1024, kClusterWarps = kClusterCtas * kClusterThreads / 32;
template <typename T, int R, int N, int M>
__global__ void __launch_bounds__(kClusterThreads) few_cluster_kernel(FewArgs p) {
  extern __shared__ __align__(16) float few_h[];   // (rows, pitch)
  after_previous();
  const int rank = (int)cluster_rank(), warp = rank * (kClusterThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t own = tc::smem_u32(few_h);
  cluster_sync();   // (all CTAs are there to be written to)
  for (int unit = warp; unit < p.hidden; unit += kClusterWarps) {
    const float h = unit_value<T, R, N>((const T*)p.x, p.ld, p.rows, (const T*)p.wg + (int64_t)unit * p.width,
                                        (const T*)p.wu + (int64_t)unit * p.width, p.width, lane);
    if (lane < p.rows) {
#pragma unroll
      for (int c = 0; c < kClusterCtas; ++c)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(in_cta(own + 4u * (lane * p.pitch + unit), c)), "f"(h) : "memory");
    }
  }
  cluster_sync();
  for (int o = warp; o < p.width_out; o += kClusterWarps) {
    const float y = result_value<T, R, M, false>(few_h, p.rows, (const T*)p.wd + (int64_t)o * p.hidden, p.hidden, p.pitch, lane);
    if (lane < p.rows) ((T*)p.y)[(int64_t)lane * p.width_out + o] = from_f32<T>(y);
  }
}

template <typename T, int R>
cudaError_t launch(const FewArgs& a, cudaStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const bool in = a.width % N == 0 && (a.rows == 1 || a.ld % N == 0), out = a.hidden % N == 0;
  if (few_rows_in_cluster(a.rows, a.width, a.hidden, a.width_out, sizeof(T))) {
    const auto kern = in && out ? few_cluster_kernel<T, R, N, N> : in ? few_cluster_kernel<T, R, N, 1> : out ? few_cluster_kernel<T, R, 1, N>
                                                                                                        : few_cluster_kernel<T, R, 1, 1>;
    return launch_clusters(kern, dim3(kClusterCtas), kClusterThreads, (size_t)a.rows * a.pitch * sizeof(float), s, kClusterCtas, a);
  }
  const cudaError_t e =
      launch_early(in ? few_hidden_kernel<T, R, N> : few_hidden_kernel<T, R, 1>, dim3((a.hidden + kWarps - 1) / kWarps), 32 * kWarps, 0, s, a);
  if (e != cudaSuccess) return e;
  // A block to a result where a warp to each would be too few for the device and read for long (bf16, 8 rows, width 1024,
  // hidden 4096: 14 us, a warp 21; 6 rows, 801 and 3001: 13 and 86.  The hidden units are more and their rows shorter: a block
  // to each took 11.7 us for 6.3, 5 rows, 289 and 909.)
  const bool block = a.width_out <= 148 * kWarps && a.hidden > 64 * (out ? N : 1);
  const auto result = block ? (out ? few_result_kernel<T, R, N, true> : few_result_kernel<T, R, 1, true>)
                            : (out ? few_result_kernel<T, R, N, false> : few_result_kernel<T, R, 1, false>);
  return launch_early(result, dim3(block ? a.width_out : (a.width_out + kWarps - 1) / kWarps), 32 * kWarps, 0, s, a);
}

template <typename T>
cudaError_t launch_rows(const FewArgs& a, cudaStream_t s) {
  return a.rows == 1 ? launch<T, 1>(a, s) : a.rows <= 4 ? launch<T, 4>(a, s) : launch<T, kFewRows>(a, s);
}

}  // namespace

// One cluster reads at most a megabyte of weights (eight multiprocessors would take longer over more), and its hidden
// values fit the shared memory that needs no opt-in.
bool few_rows_in_cluster(int64_t rows, int64_t width, int64_t hidden, int64_t width_out, int elem) {
  return hidden * (2 * width + width_out) * elem <= 1 << 20 && rows * ((hidden + 7) / 8 * 8) * (int64_t)sizeof(float) <= 40 << 10;
}

cudaError_t few_rows(const FewArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case TRIFAST_F32: return launch_rows<float>(a, s);
    case TRIFAST_BF16: return launch_rows<__nv_bfloat16>(a, s);
    default: return launch_rows<__half>(a, s);
  }
}

}  // namespace ff
}  // namespace trifast
