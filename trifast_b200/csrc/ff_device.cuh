// Device helpers of the feed-forward block's kernels (ff_gemm.cu, ff_fused.cu) and the tensor maps of their operands.
#pragma once

#include "ff_gemm.cuh"
#include "tc_common.cuh"

namespace trifast {
namespace ff {
using namespace tc;

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// block_gave_up(), and the host word is told again.  (No measurable cost: 8192 x 512, hidden 2048, forward and backward 207 us, 208
// without the barrier.)
__device__ __forceinline__ bool device_gave_up(unsigned int* status) {
  const bool up = block_gave_up(status, threadIdx.x == 0);
  if (up && blockIdx.x == 0 && threadIdx.x == 0) repeat_status(status);
  return up;
}

// ------------------------------------------------------------------ pairs of CTAs (cta_group::2)
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of another CTA's shared memory at this CTA's address `local`.
__device__ __forceinline__ uint32_t in_cta(uint32_t local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t load_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// An arrival at a barrier of either CTA.  (What it tells of is TMEM, read or written, which the tcgen05 fences order; the
// arrival and the wait need no more than the scope of a CTA.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Into this CTA's memory, counted by a barrier of either CTA of the pair (plain per-CTA loads).
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void umma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ts_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One arrival at this barrier of both CTAs when every MMA issued so far by this thread is done.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((uint16_t)3)
               : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t smem_result, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_result), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// The same tile as tma_load_3d's into L2 alone.
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// A barrier of `threads` threads that tells whether all of them came with `ok`.
__device__ __forceinline__ bool group_all(int id, int threads, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void group_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + e^-a): 0 and 1 at the ends, NaN for NaN
__device__ __forceinline__ float sigmoid(float a) { return rcp(1.f + ex2(-kLog2e * a)); }

// The same of two units, the arithmetic around the approximations packed.
__device__ __forceinline__ void sigmoid2(float a0, float a1, float& s0, float& s1) {
  fmul2(s0, s1, a0, a1, -kLog2e, -kLog2e);
  fadd2(s0, s1, ex2(s0), ex2(s1), 1.f, 1.f);
  s0 = rcp(s0);
  s1 = rcp(s1);
}

// h = silu(a) b of N units, packed: rounded to the call's 16-bit type, since the tensor cores take the next product's operand
// in that.  So are da and db below.  The results' error against 64 bits is 1.4 times that of one rounding at the end (bf16 2.35e-3
// for 1.66e-3, fp16 2.9e-4 for 2.1e-4).  fp16: h beyond 65504 is infinite, and da and db below 2^-25 are 0.  (One reciprocal for two units, 1/u = v / (u v), and every other exponential by a
// polynomial on the FMA pipe left the special-function unit half idle and the kernels of ff_fused.cu no faster: 344-360 us
// against 350 forward, 559-586 against 557 for dX.)
template <typename T, int N>
__device__ __forceinline__ void gate_units(const float* a, const float* b, uint32_t* h) {
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    float s0, s1;
    sigmoid2(a[e], a[e + 1], s0, s1);
    fmul2(s0, s1, a[e], a[e + 1], s0, s1);
    fmul2(s0, s1, s0, s1, b[e], b[e + 1]);
    h[e >> 1] = pack2<T>(s0, s1);
  }
}

// da = dh b silu'(a), db = dh silu(a) (and h) of N units, packed.
template <typename T, int N, bool H>
__device__ __forceinline__ void grad_units(const float* a, const float* b, const float* dh, uint32_t* da, uint32_t* db, uint32_t* h) {
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    float s0, s1, v0, v1, w0, w1, q0, q1, r0, r1;
    sigmoid2(a[e], a[e + 1], s0, s1);
    fmul2(v0, v1, a[e], a[e + 1], s0, s1);                   // silu
    ffma2(q0, q1, s0, s1, -1.f, -1.f, 1.f, 1.f);
    ffma2(q0, q1, v0, v1, q0, q1, s0, s1);                   // its slope, s + silu (1 - s)
    fmul2(w0, w1, dh[e], dh[e + 1], b[e], b[e + 1]);
    fmul2(w0, w1, w0, w1, q0, q1);
    fmul2(r0, r1, dh[e], dh[e + 1], v0, v1);
    da[e >> 1] = pack2<T>(w0, w1);
    db[e >> 1] = pack2<T>(r0, r1);
    if constexpr (H) {
      fmul2(v0, v1, v0, v1, b[e], b[e + 1]);
      h[e >> 1] = pack2<T>(v0, v1);
    }
  }
}

// 32 columns of a row of partial sums, of which `there` (a multiple of 4, or beyond 32) lie in the row.  They are added
// where they lie: reading them first waits for each row of the warp in turn (50 MB of a second chunk of rows took 240 us).  An
// entry gets one addition a turn, always the same thread's or the next kernel's: the order is fixed.  (A sum below 2^-126 may
// be 0.)
__device__ __forceinline__ void add_partials(float* dst, const float* v, int there, bool add) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (4 * i >= there) continue;
    if (add)
      asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(dst + 4 * i), "f"(v[4 * i]), "f"(v[4 * i + 1]),
                   "f"(v[4 * i + 2]), "f"(v[4 * i + 3])
                   : "memory");
    else
      reinterpret_cast<float4*>(dst)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  }
}

// `box_cols` x `box_rows` tiles of a matrix
inline bool map_of(CUtensorMap* map, bool bf16, const Matrix& m, int box_cols, int box_rows) {   // (128-byte swizzle; 64 for 32 columns)
  const uint64_t dims[3] = {(uint64_t)m.cols, (uint64_t)m.rows, (uint64_t)m.planes};
  const uint64_t st[2] = {(uint64_t)m.pitch * 2, (uint64_t)m.plane * 2};
  const uint32_t box[3] = {(uint32_t)box_cols, (uint32_t)box_rows, 1};
  return make_tensor_map(map, bf16, 3, m.p, dims, st, box, box_cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace ff
}  // namespace trifast
