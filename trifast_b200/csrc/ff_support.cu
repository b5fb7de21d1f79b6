// Kernels around the products of the feed-forward block: operands laid out for them, and the sum of the
// weight gradients' partial sums.

#include <type_traits>

#include "ff_gemm.cuh"
#include "tc_common.cuh"

namespace trifast {
namespace ff {
namespace {

// Matrices with rows of 16-byte pitch, and fp32 as three bf16 planes.  A value is cut, not rounded, to its upper 8
// significant bits, and what is left again: the three parts hold its 24 bits exactly and have one sign.  A thread makes
// eight columns of a row; rows behind the last are zero.
struct StageJobs {
  StageJob job[kStageJobs];
  int64_t end[kStageJobs];   // threads up to and with each
  int count;
};
template <typename T>
__global__ void __launch_bounds__(256) stage_kernel(const __grid_constant__ StageJobs jobs) {
  after_previous();
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < jobs.end[jobs.count - 1]; i += (int64_t)gridDim.x * blockDim.x) {
    int j = 0;
    while (i >= jobs.end[j]) ++j;
    const StageJob& job = jobs.job[j];
    const Matrix& dst = job.dst;
    const int64_t at = i - (j ? jobs.end[j - 1] : 0), per_row = dst.pitch / 8;
    const int64_t r = at / per_row, c = (at % per_row) * 8;
    const T* src = reinterpret_cast<const T*>(job.src) + r * job.ld + c;
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = r < job.rows && c + e < dst.cols ? src[e] : from_f32<T>(0.f);
    uint16_t* out = reinterpret_cast<uint16_t*>(dst.p) + r * dst.pitch + c;
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t a = __float_as_uint(v[2 * e]), b = __float_as_uint(v[2 * e + 1]);
          u[e] = __byte_perm(a, b, 0x7632);
          v[2 * e] -= __uint_as_float(a & 0xffff0000u);
          v[2 * e + 1] -= __uint_as_float(b & 0xffff0000u);
        }
        *reinterpret_cast<uint4*>(out + q * dst.plane) = make_uint4(u[0], u[1], u[2], u[3]);
      }
    } else {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint16_t lo, hi;
        memcpy(&lo, &v[2 * e], 2);
        memcpy(&hi, &v[2 * e + 1], 2);
        u[e] = lo | (uint32_t)hi << 16;
      }
      *reinterpret_cast<uint4*>(out) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
}

// Eight warps of a block take an eighth of the splits each, in order, and their sums are added in order, all in fp32.  A
// thread makes N neighbours: four where all counts are multiples of four.
struct Results {
  void* dst[3];
  int64_t end[3];
};
template <typename T, int N>
__global__ void __launch_bounds__(256) sum_partials_kernel(const float* __restrict__ partials, int splits, int64_t stride, Results r) {
  __shared__ float sum[8][32 * N];
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = ((int64_t)blockIdx.x * 32 + lane) * N;
  const int lo = splits * warp / 8, hi = splits * (warp + 1) / 8;
  float s[N];
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] = 0.f;
  if (i < r.end[2]) {
#pragma unroll 4
    for (int k = lo; k < hi; ++k) {
      if constexpr (N == 4) {
        const float4 v = *reinterpret_cast<const float4*>(partials + k * stride + i);
        s[0] += v.x;
        s[1] += v.y;
        s[2] += v.z;
        s[3] += v.w;
      } else {
        s[0] += partials[k * stride + i];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) sum[warp][lane * N + e] = s[e];
  __syncthreads();
  if (warp != 0 || i >= r.end[2]) return;
#pragma unroll
  for (int w = 1; w < 8; ++w)
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] += sum[w][lane * N + e];
  const int at = i < r.end[0] ? 0 : i < r.end[1] ? 1 : 2;
  T* dst = reinterpret_cast<T*>(at == 0 ? r.dst[0] : at == 1 ? r.dst[1] : r.dst[2]) + (i - (at == 0 ? 0 : at == 1 ? r.end[0] : r.end[1]));
  if constexpr (N == 4 && std::is_same<T, float>::value) {
    *reinterpret_cast<float4*>(dst) = make_float4(s[0], s[1], s[2], s[3]);
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(tc::pack2<T>(s[0], s[1]), tc::pack2<T>(s[2], s[3]));
  } else {
    *dst = from_f32<T>(s[0]);
  }
}

dim3 grid_for(int64_t threads) {
  const int64_t b = (threads + 255) / 256, most = (int64_t)sm_count() * 16;
  return dim3((unsigned)(b < most ? b : most));
}

}  // namespace

cudaError_t stage(const StageJob* jobs, int count, int dtype, cudaStream_t s) {
  StageJobs a = {};
  for (int j = 0; j < count; ++j) {
    a.job[a.count] = jobs[j];
    a.end[a.count] = (a.count ? a.end[a.count - 1] : 0) + jobs[j].dst.rows * (jobs[j].dst.pitch / 8);
    ++a.count;
  }
  if (count == 0) return cudaSuccess;
  const dim3 g = grid_for(a.end[count - 1]);
  return dtype == TRIFAST_F32 ? launch_early(stage_kernel<float>, g, 256, 0, s, a) : launch_early(stage_kernel<__half>, g, 256, 0, s, a);
}

template <typename T>
cudaError_t sum_type(const float* partials, int splits, int64_t stride, const Results& r, bool four, cudaStream_t s) {
  return four ? launch_early(sum_partials_kernel<T, 4>, dim3((unsigned)((r.end[2] + 127) / 128)), 256, 0, s, partials, splits, stride, r)
              : launch_early(sum_partials_kernel<T, 1>, dim3((unsigned)((r.end[2] + 31) / 32)), 256, 0, s, partials, splits, stride, r);
}

cudaError_t sum_partials(const float* partials, int splits, int64_t stride, void* const (&dst)[3], const int64_t (&count)[3], int dtype,
                         cudaStream_t s) {
  Results r = {};
  bool four = true;
  for (int j = 0; j < 3; ++j) {
    r.dst[j] = dst[j];
    r.end[j] = (j ? r.end[j - 1] : 0) + count[j];
    four = four && count[j] % 4 == 0;
  }
  switch (dtype) {
    case TRIFAST_F32: return sum_type<float>(partials, splits, stride, r, four, s);
    case TRIFAST_BF16: return sum_type<__nv_bfloat16>(partials, splits, stride, r, four, s);
    default: return sum_type<__half>(partials, splits, stride, r, four, s);
  }
}

}  // namespace ff
}  // namespace trifast
