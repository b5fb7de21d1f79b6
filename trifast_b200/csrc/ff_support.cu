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
// eight columns of a row, kUnits times, all read before the first is written: it reads the aligned 16-byte pieces that they lie
// in and shifts them into place (element by element, the loads of 6280 x 913 bf16 and its weights took 12.6 us).  Columns
// behind the last are zero.  The pieces of all rows run over the lanes (262,144 x 65 bf16: 17.4 us; 55 with 16 lanes for
// the nine pieces of a row, one at a time).
template <typename T> constexpr int kUnits = sizeof(T) == 2 ? 4 : 2;
struct StageJobs {
  StageJob job[kStageJobs];
  int64_t end[kStageJobs];    // warps' turns up to and with each
  int count;
};
template <typename T>
__global__ void __launch_bounds__(256) stage_kernel(const __grid_constant__ StageJobs jobs) {
  constexpr int kElem = sizeof(T), W = 2 * kElem, V = W / 4 + 1;   // words of eight columns; pieces that they can lie in
  constexpr int U = kUnits<T>;
  after_previous();
  const int lane = threadIdx.x & 31;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < jobs.end[jobs.count - 1]; i += (int64_t)gridDim.x * 8) {
    int j = 0;
    while (i >= jobs.end[j]) ++j;
    const StageJob& job = jobs.job[j];
    const int cols = (int)job.dst.cols, pieces = (int)(job.dst.pitch / 8);
    const char* end = reinterpret_cast<const char*>(reinterpret_cast<const T*>(job.src) + (job.rows - 1) * job.ld + cols);
    const int64_t first = (i - (j ? jobs.end[j - 1] : 0)) * (32 * U), row0 = first / pieces;
    const uint32_t rest = (uint32_t)(first - row0 * pieces);
    uint32_t w[U][4 * V];
    int64_t row[U];
    int piece[U];
    uint32_t off[U];   // bytes before its eight columns
    auto load = [&](int64_t row, int piece, uint32_t (&x)[4 * V], uint32_t& off) {
      const T* src = reinterpret_cast<const T*>(job.src) + row * job.ld;
      off = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15);
      const int there = min(cols - 8 * piece, 8);   // columns of this piece (at least one)
      const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(src) - off) + piece * (V - 1);
      const int used = ((int)off + there * kElem + 15) / 16;   // pieces that hold something of the row
      if (reinterpret_cast<const char*>(from + used) <= end) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (v < used) {
            const uint4 q = from[v];
            x[4 * v] = q.x;
            x[4 * v + 1] = q.y;
            x[4 * v + 2] = q.z;
            x[4 * v + 3] = q.w;
          }
      } else {
        // nothing is read behind the matrix's end
        T t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = e < there ? src[8 * piece + e] : from_f32<T>(0.f);
        memcpy(x, t, sizeof(t));
        off = 0;
      }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t t = rest + u * 32 + lane, rr = t / (uint32_t)pieces;
      piece[u] = (int)(t - rr * pieces);
      row[u] = row0 + rr;
#pragma unroll
      for (int k = 0; k < 4 * V; ++k) w[u][k] = 0;
      off[u] = 0;
      if (row[u] < job.rows) load(row[u], piece[u], w[u], off[u]);
    }
    auto put = [&](int64_t row, int piece, uint32_t (&x)[4 * V], uint32_t off) {
      const int there = min(cols - 8 * piece, 8);
#pragma unroll
      for (int k = 0; k < 4 * V; ++k) {
        const uint32_t far = k + 2 < 4 * V ? x[k + 2] : 0;
        x[k] = off & 8 ? far : x[k];
      }
#pragma unroll
      for (int k = 0; k < 4 * V; ++k) {
        const uint32_t next = k + 1 < 4 * V ? x[k + 1] : 0;
        x[k] = off & 4 ? next : x[k];
      }
      if (kElem == 2)
#pragma unroll
        for (int k = 0; k < W; ++k) x[k] = off & 2 ? __funnelshift_r(x[k], x[k + 1], 16) : x[k];
      uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(job.dst.p) + row * job.dst.pitch) + piece;
      if constexpr (kElem == 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = 2 * k + 1 < there ? x[k] : 2 * k < there ? x[k] & 0xffffu : 0u;
        *out = make_uint4(x[0], x[1], x[2], x[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = k < there ? x[k] : 0u;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          uint32_t b[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            b[k] = __byte_perm(x[2 * k], x[2 * k + 1], 0x7632);
#pragma unroll
            for (int h = 0; h < 2; ++h)
              x[2 * k + h] = __float_as_uint(__uint_as_float(x[2 * k + h]) - __uint_as_float(x[2 * k + h] & 0xffff0000u));
          }
          out[q * (job.dst.plane / 8)] = make_uint4(b[0], b[1], b[2], b[3]);
        }
      }
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row[u] < job.rows) put(row[u], piece[u], w[u], off[u]);
  }
}

// A block's eight warps are groups of `parts`, which take a share of the splits each, in order; their sums are added in
// order, all in fp32.  A thread makes four neighbours of a row.
struct Results {
  void* dst[3];
  int64_t end[3];      // pieces of four up to and with each product
  int cols[3], pieces[3];
};
template <typename T>
__global__ void __launch_bounds__(256) sum_partials_kernel(const float* __restrict__ partials, int splits, int64_t stride, int parts, Results r) {
  __shared__ float4 sum[8][32];
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % parts;
  const int64_t i = ((int64_t)blockIdx.x * (8 / parts) + warp / parts) * 32 + lane;
  const int lo = splits * part / parts, hi = splits * (part + 1) / parts;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < r.end[2]) {
#pragma unroll 4
    for (int k = lo; k < hi; ++k) {
      const float4 v = reinterpret_cast<const float4*>(partials + k * stride)[i];
      s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
    }
  }
  sum[warp][lane] = s;
  __syncthreads();
  if (part != 0 || i >= r.end[2]) return;
  for (int w = 1; w < parts; ++w) {
    const float4 v = sum[warp + w][lane];
    s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
  }
  const int j = i < r.end[0] ? 0 : i < r.end[1] ? 1 : 2;
  const int64_t at = i - (j == 0 ? 0 : j == 1 ? r.end[0] : r.end[1]);
  const int pieces = j == 2 ? r.pieces[2] : r.pieces[0], cols = j == 2 ? r.cols[2] : r.cols[0];
  const int64_t row = at / pieces;
  const int c = (int)(at - row * pieces) * 4;
  T* dst = reinterpret_cast<T*>(j == 0 ? r.dst[0] : j == 1 ? r.dst[1] : r.dst[2]) + row * cols + c;
  const float f[4] = {s.x, s.y, s.z, s.w};
  if (cols % 4 == 0) {
    if constexpr (std::is_same<T, float>::value)
      *reinterpret_cast<float4*>(dst) = s;
    else
      *reinterpret_cast<uint2*>(dst) = make_uint2(tc::pack2<T>(s.x, s.y), tc::pack2<T>(s.z, s.w));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < cols) dst[e] = from_f32<T>(f[e]);
  }
}

dim3 grid_for(int64_t threads) {
  const int64_t b = (threads + 255) / 256, most = (int64_t)sm_count() * 16;
  return dim3((unsigned)(b < most ? b : most));
}

}  // namespace

cudaError_t stage(const StageJob* jobs, int count, int dtype, cudaStream_t s) {
  StageJobs a = {};
  const int64_t per = 32 * (dtype == TRIFAST_F32 ? kUnits<float> : kUnits<__half>);
  for (int j = 0; j < count; ++j) {
    a.job[j] = jobs[j];
    a.end[j] = (j ? a.end[j - 1] : 0) + (jobs[j].rows * (jobs[j].dst.pitch / 8) + per - 1) / per;
  }
  a.count = count;
  if (count == 0) return cudaSuccess;
  const dim3 g = grid_for(a.end[count - 1] * 32);
  return dtype == TRIFAST_F32 ? launch_early(stage_kernel<float>, g, 256, 0, s, a) : launch_early(stage_kernel<__half>, g, 256, 0, s, a);
}

cudaError_t sum_partials(const float* partials, int splits, int64_t stride, void* const (&dst)[3], const int64_t (&rows)[3],
                         const int64_t (&cols)[3], int dtype, cudaStream_t s) {
  Results r = {};
  for (int j = 0; j < 3; ++j) {
    r.dst[j] = dst[j];
    r.cols[j] = (int)cols[j];
    r.pieces[j] = (int)(partial_pitch(cols[j]) / 4);
    r.end[j] = (j ? r.end[j - 1] : 0) + rows[j] * r.pieces[j];
  }
  const int parts = splits >= 8 ? 8 : splits >= 4 ? 4 : splits >= 2 ? 2 : 1, per = 32 * (8 / parts);
  const dim3 g((unsigned)((r.end[2] + per - 1) / per));
  switch (dtype) {
    case TRIFAST_F32: return launch_early(sum_partials_kernel<float>, g, 256, 0, s, partials, splits, stride, parts, r);
    case TRIFAST_BF16: return launch_early(sum_partials_kernel<__nv_bfloat16>, g, 256, 0, s, partials, splits, stride, parts, r);
    default: return launch_early(sum_partials_kernel<__half>, g, 256, 0, s, partials, splits, stride, parts, r);
  }
}

}  // namespace ff
}  // namespace trifast
