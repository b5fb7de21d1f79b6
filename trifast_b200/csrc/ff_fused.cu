// The gated feed-forward block in one kernel, and its backward pass in two, for rows of up to 128 elements
// (16-bit types): the hidden values never leave the multiprocessor.
//
// All three walk the hidden units in chunks of 64.  With S = X [Wg; Wu]^T of a chunk (128 rows x (64 a | 64 b), fp32
// in TMEM),
//   forward:  h = silu(a) b -> TMEM as the 16-bit A operand,  Y += h Wd^T          (512 + 256 cycles of the tensor pipe)
//   dX:       dH = dY Wd;  da | db -> TMEM,                   dX += da Wg + db Wu   (512 + 256 + 512)
//   dW:       dH;  da | db | h -> shared memory, whose rows are then the contraction:
//             [dWg; dWu] += [da | db]^T X,  dWd += dY^T h                          (512 + 256 + 512 + 256)
// at 128 rows.  A weight tile in shared memory serves two products, along its rows (K-major) in one and
// across them (MN-major) in the other; so do the X and dY tiles of dW.
//
// The first two keep rows and stream the weights (rings of chunks); dW keeps a chunk of the weights and its
// gradients' fp32 sums (192 columns of TMEM) and streams the rows, a share of them per CTA, whose sums a second
// kernel adds up.  S is computed three times in all (forward, dX, dW) and dH twice, five products of fourteen, against six
// hidden-sized tensors through memory.
//
// 1,048,576 rows, width 128, hidden 512, bf16: forward 335 us, dX 549, dW 767, 1.23, 1.25 and 1.08 PFLOP/s of what they
// run, on a chip that was idle before; under load 389, 639 and 862.  Forward and dX are near what the chip sustains (cuBLAS: 1.36).
// dW: operands, rows fetched and gradients staged are 336 KB of shared memory per 128 rows, which at 128 bytes a cycle would be
// 2,625 of its 2,900 cycles.  The counters show no unit at its limit: reads of operands 55 % of the wavefronts, tensor pipe
// 47 %.
//
// All waits are bounded.

#include <type_traits>

#include "ff_device.cuh"
#include "ff_fused.cuh"

namespace trifast {
namespace ff {
namespace {

constexpr int kChunk = 64;               // hidden units
constexpr int kThreads = 352;            // of dW
constexpr int kSmemLimit = 232448;
constexpr int kTile = 128 * 64 * 2;      // 128 rows x 64 columns

struct Params {
  CUtensorMap x, dy, wg, wu, wd, out;
  CUtensorMap wg_across, wu_across;   // dX: half the width of 64 units
  int64_t rows;
  int tiles, chunks;   // row tiles; chunks of hidden units
  void* y;                  // result rows for stores that TMA cannot make
  int64_t ldy;
  int cols, y_tma;
  // dW
  float* partials;
  int64_t partial_stride;
  int splits, add, width, hidden, width_out;
  unsigned int* status;
};

// Shared memory: barriers, then the tiles.
struct Smem {
  uint8_t* g;
  uint32_t base;
  __device__ __forceinline__ uint32_t bar(int i) const { return base + 8u * i; }
  __device__ __forceinline__ volatile int* abort_flag() const { return reinterpret_cast<volatile int*>(g + 256); }
  __device__ __forceinline__ uint32_t* tmem_slot() const { return reinterpret_cast<uint32_t*>(g + 260); }
};
__device__ __forceinline__ Smem smem_of(uint8_t* raw) {
  const uint32_t r = smem_u32(raw), b = (r + 1023u) & ~1023u;
  return {raw + (b - r), b};
}

// After the barriers have been set up: TMEM, and with pairs of CTAs (CG = 2) whether both go on (`go`).
template <int CG>
__device__ __forceinline__ uint32_t start(const Smem& sm, bool owner, bool given_up, bool* go) {
  if (threadIdx.x == 0) *reinterpret_cast<volatile uint32_t*>(sm.g + 264) = given_up;
  if (owner) {
    if (CG == 2) {
      tmem_alloc_pair(smem_u32(sm.tmem_slot()), 512);
    } else {
      tmem_alloc(smem_u32(sm.tmem_slot()), 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tc_fence_after();
  *go = CG == 2 ? (load_cluster(in_cta(sm.base + 264, 0)) | load_cluster(in_cta(sm.base + 264, 1))) == 0 : !given_up;
  return *sm.tmem_slot();
}

template <int CG>
__device__ __forceinline__ void finish(const Smem& sm, bool owner, uint32_t tmem, unsigned int* status) {
  tc_fence_before();
  __syncthreads();
  if (*sm.abort_flag()) {
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000LL) {
    }
    if (threadIdx.x == 0) set_status(status, kStatusTimeoutFeedForward);
    __syncthreads();
  }
  // (neither CTA of a pair goes before the other's last access to it)
  if (CG == 2) cluster_sync();
  if (owner) {
    tc_fence_after();
    if (CG == 2)
      tmem_dealloc_pair(tmem, 512);
    else
      tmem_dealloc(tmem, 512);
  }
}

// 64 columns of 128 result rows (u: a row of them, packed): registers -> a swizzled tile in shared memory -> memory.
// Called by the 128 threads of barrier `id`.
__device__ __forceinline__ void store_tile(const Params& p, const Smem& sm, uint32_t off, int id, const uint32_t* u, int m0, int col) {
  const int row = threadIdx.x & 127, lane = threadIdx.x & 31, wq = (threadIdx.x >> 5) & 3;
  if (row == 0) bulk_wait_read();
  group_sync(id, 128);
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<uint4*>(sm.g + off + row * 128 + ((c ^ (row & 7)) << 4)) = make_uint4(u[4 * c], u[4 * c + 1], u[4 * c + 2], u[4 * c + 3]);
  if (p.y_tma) fence_async_smem();
  group_sync(id, 128);
  if (p.y_tma) {
    if (row == 0 && col < p.cols && m0 < p.rows) {
      tma_store_3d(&p.out, sm.base + off, col, m0, 0);
      bulk_commit();
    }
  } else {
    const int c = col + 2 * lane;
    for (int r = wq; r < 128 && (int64_t)m0 + r < p.rows; r += 4) {
      const uint32_t two = *reinterpret_cast<const uint32_t*>(sm.g + off + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2)));
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.y) + ((int64_t)m0 + r) * p.ldy + c;
      if (c < p.cols) dst[0] = (uint16_t)two;
      if (c + 1 < p.cols) dst[1] = (uint16_t)(two >> 16);
    }
  }
}

template <int CP>
__device__ __forceinline__ void load_rows(const CUtensorMap* map, uint32_t dst, uint32_t bar, int m0) {
#pragma unroll
  for (int kb = 0; kb < CP / 64; ++kb) tma_load_3d(dst + kb * kTile, map, bar, kb * 64, m0, 0);
}

// ------------------------------------------------------------------ the kernels that keep rows
// Two CTAs share every MMA, M = 256: each has a row tile of its own, its half of the weights' tiles (Wg's rows in the
// first, Wu's in the second; half of what the other products have for columns) and its part of the results.  With one
// CTA an MMA, each fetched all weights, 3.2 GB from L2 in 345 us for 1,048,576 rows forward, and read them from its
// shared memory, which set the pace of dX (566 us).
//
// Warps: 0-7 elementwise, 8-11 results, 12 and 13 TMA (rows, Wg and Wu; Wd), 14 and 15, of the pair's first CTA, MMA
// issuers (S and dH; the products of h, da and db).  A wait costs an issuer or producer about 100 cycles even for what is
// there, so the two kinds of each do not share a warp.
constexpr int kRowThreads = 512, kOutWarp = 8, kTmaWarp = 12, kTmaDWarp = 13, kSWarp = 14, kMmaWarp = 15;

// Shared memory by kernel: rows (two X tiles, or X and dY), rings of chunks, result tiles.
template <int CP, bool DX>
struct Rows {
  static constexpr int kBlocks = CP / 64, kHalf = CP / 2;
  static constexpr int kX = kBlocks * kTile;
  static constexpr int kSBytes = kBlocks * (kTile / 2);            // 64 rows of Wg or Wu, along their width
  static constexpr int kAcross = kChunk * kHalf * 2;               // half the width of 64 rows of Wg (then of Wu), for dX
  static constexpr int kGuBytes = kSBytes + (DX ? 2 * kAcross : 0);
  static constexpr int kDBytes = DX ? CP * 64 : kHalf * 128;       // Wd: 32 units of all rows; 64 units of half the rows
  static constexpr int kGU = DX ? 3 : 4, kD = DX ? 3 : 4;
  static constexpr int kXOff = 1024, kGuOff = kXOff + 2 * kX, kDOff = kGuOff + kGU * kGuBytes, kOutOff = kDOff + kD * kDBytes;
  static constexpr int smem_bytes() { return 1024 + kOutOff + 2 * kTile; }
  static_assert(smem_bytes() <= kSmemLimit && kGuBytes % 1024 == 0 && kDBytes % 1024 == 0, "shared memory");
};

// The row tiles of a CTA, and the chunks of hidden units that it walks over all of them.
struct Walk {
  int rank, first, stride, items, total;
  __device__ __forceinline__ Walk(const Params& p) {
    rank = (int)cluster_rank();
    first = blockIdx.x / 2;
    stride = gridDim.x / 2;
    const int pairs = (p.tiles + 1) / 2;
    items = first < pairs ? (pairs - 1 - first) / stride + 1 : 0;
    total = items * p.chunks;
  }
  __device__ __forceinline__ int row(int it) const { return ((first + it * stride) * 2 + rank) * 128; }
};

// Producers: this CTA's part, counted by the first CTA's barrier, which expects both parts.
struct Filler {
  uint32_t base, counted;   // this CTA's barriers, the first CTA's
  int rank;
  __device__ __forceinline__ uint32_t expect(int bar, int bytes) const {
    if (rank == 0) mbar_arrive_expect_tx(base + 8u * bar, 2 * bytes);
    return counted + 8u * bar;
  }
};

// S = X [Wg; Wu]^T, 256 x 128
template <bool BF16, int CP>
__device__ __forceinline__ void pair_s(uint32_t d, uint32_t x, uint32_t gu) {
  const uint64_t ad = make_smem_desc(x, 16, 1024, kSwizzle128), bd = make_smem_desc(gu, 16, 1024, kSwizzle128);
#pragma unroll
  for (int k = 0; k < CP / 16; ++k)
    umma_ss_pair(d, ad + (k >> 2) * (kTile >> 4) + (k & 3) * 2, bd + (k >> 2) * (kTile >> 5) + (k & 3) * 2,
                 make_idesc(256, 128, BF16, false, false), k > 0);
}

// The 128 x CP sums of an item at column `acc` of TMEM, as result rows: warps 8-11, once per item.
template <typename T, int CP>
__device__ __forceinline__ void write_results(const Params& p, const Smem& sm, const Walk& walk, uint32_t acc, uint32_t out_off, int done,
                                              uint32_t free) {
  const int lane = threadIdx.x & 31, wq = (threadIdx.x >> 5) & 3;
  const uint32_t at = acc + ((uint32_t)(wq * 32) << 16);
  for (int it = 0; it < walk.items; ++it) {
    // all go on or none: store_tile has barriers
    if (!group_all(1, 128, mbar_wait(sm.bar(done), it & 1, sm.abort_flag()))) break;
    tc_fence_after();
    uint32_t u[CP / 2];
#pragma unroll
    for (int c = 0; c < CP; c += 32) {
      float v[32];
      tmem_ld32(at + c, reinterpret_cast<uint32_t*>(v));
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; e += 2) u[(c + e) >> 1] = pack2<T>(v[e], v[e + 1]);
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive_cluster(free);
#pragma unroll
    for (int c = 0; c < CP; c += 64) store_tile(p, sm, out_off + (c >> 6) * kTile, 1, u + (c >> 1), walk.row(it), c);
  }
  bulk_wait();
}

// ------------------------------------------------------------------ forward
// TMEM: three S of 128 columns, which the chunks take in turn (h over a's first columns), so that the tensor pipe is two
// chunks ahead of the gates; Y [384, 384 + CP).
template <typename T, int CP>
__global__ void __launch_bounds__(kRowThreads, 1) ff_forward_kernel(const __grid_constant__ Params p) {
  using L = Rows<CP, false>;
  constexpr int kGU = L::kGU, kD = L::kD;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int X_FULL = 0, X_EMPTY = 2, GU_FULL = 4, GU_EMPTY = GU_FULL + kGU, D_FULL = GU_EMPTY + kGU, D_EMPTY = D_FULL + kD,
                S_FULL = D_EMPTY + kD, H_READY = S_FULL + 3, H_FREE = H_READY + 3, Y_DONE = H_FREE + 3, Y_FREE = Y_DONE + 1, NBARS = Y_FREE + 1;
  static_assert(NBARS * 8 <= 256, "barrier area");
  extern __shared__ uint8_t smem_raw[];
  const Smem sm = smem_of(smem_raw);
  volatile int* abort_flag = sm.abort_flag();
  after_previous();
  const bool given_up = device_gave_up(p.status);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NBARS; ++i) mbar_init(sm.bar(i), (i >= H_READY && i < H_READY + 3) || i == Y_FREE ? 8 : 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  bool go;
  const uint32_t tmem = start<2>(sm, warp == kMmaWarp, given_up, &go);
  const Walk walk(p);
  const int n = p.chunks, total = go ? walk.total : 0;
  const uint32_t first = in_cta(sm.base, 0);   // the first CTA's barriers
  const Filler fill{sm.base, first, walk.rank};
  auto wait = [&](int b, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(sm.bar(b), parity, abort_flag)); };
  auto x_tile = [&](int it) { return sm.base + L::kXOff + (it & 1) * L::kX; };
  auto gu_tile = [&](int g) { return sm.base + L::kGuOff + (g % kGU) * L::kGuBytes; };
  auto d_tile = [&](int g) { return sm.base + L::kDOff + (g % kD) * L::kDBytes; };

  if (!go) {
  } else if (warp == kTmaWarp) {
    bool ok = true;
    const CUtensorMap* own = walk.rank == 0 ? &p.wg : &p.wu;
    for (int g = 0, c = 0, it = 0; g < total && ok; ++g, c = c + 1 == n ? 0 : c + 1) {
      if (c == 0) {
        if (it >= 2) ok = wait(X_EMPTY + (it & 1), (it / 2 - 1) & 1);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t f = fill.expect(X_FULL + (it & 1), L::kX);
#pragma unroll
          for (int kb = 0; kb < L::kBlocks; ++kb) tma_load_3d_pair(x_tile(it) + kb * kTile, &p.x, f, kb * 64, walk.row(it), 0);
        }
        __syncwarp();
        ++it;
      }
      if (g >= kGU) ok = wait(GU_EMPTY + g % kGU, (g / kGU - 1) & 1);
      if (!ok) break;
      if (elect_one()) {
        const uint32_t f = fill.expect(GU_FULL + g % kGU, L::kGuBytes);
#pragma unroll
        for (int kb = 0; kb < L::kBlocks; ++kb) tma_load_3d_pair(gu_tile(g) + kb * (kTile / 2), own, f, kb * 64, c * kChunk, 0);
      }
      __syncwarp();
    }
  } else if (warp == kTmaDWarp) {
    bool ok = true;
    for (int g = 0, c = 0; g < total && ok; ++g, c = c + 1 == n ? 0 : c + 1) {
      if (g >= kD) ok = wait(D_EMPTY + g % kD, (g / kD - 1) & 1);
      if (!ok) break;
      if (elect_one()) tma_load_3d_pair(d_tile(g), &p.wd, fill.expect(D_FULL + g % kD, L::kDBytes), c * kChunk, walk.rank * L::kHalf, 0);
      __syncwarp();
    }
  } else if (warp == kSWarp) {
    bool ok = true;
    for (int g = 0, c = 0, it = 0; g < total && ok && walk.rank == 0; ++g) {
      if (c == 0) ok = wait(X_FULL + (it & 1), (it >> 1) & 1);
      ok = ok && wait(GU_FULL + g % kGU, (g / kGU) & 1);
      if (ok && g >= 3) ok = wait(H_FREE + g % 3, (g / 3 - 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        pair_s<kBf16, CP>(tmem + (g % 3) * 128, x_tile(it), gu_tile(g));
        umma_commit_pair(sm.bar(S_FULL + g % 3));
        umma_commit_pair(sm.bar(GU_EMPTY + g % kGU));
        if (c == n - 1) umma_commit_pair(sm.bar(X_EMPTY + (it & 1)));
      }
      __syncwarp();
      if (++c == n) {
        c = 0;
        ++it;
      }
    }
  } else if (warp == kMmaWarp) {
    bool ok = true;
    for (int g = 0, c = 0, it = 0; g < total && ok && walk.rank == 0; ++g) {
      ok = wait(D_FULL + g % kD, (g / kD) & 1) && wait(H_READY + g % 3, (g / 3) & 1);
      if (ok && c == 0 && it > 0) ok = wait(Y_FREE, (it - 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t bd = make_smem_desc(d_tile(g), 16, 1024, kSwizzle128);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_ts_pair(tmem + 384, tmem + (g % 3) * 128 + k * 8, bd + k * 2, make_idesc(256, CP, kBf16, false, false), (c > 0 || k > 0) ? 1u : 0u);
        umma_commit_pair(sm.bar(H_FREE + g % 3));
        umma_commit_pair(sm.bar(D_EMPTY + g % kD));
        if (c == n - 1) umma_commit_pair(sm.bar(Y_DONE));
      }
      __syncwarp();
      if (++c == n) {
        c = 0;
        ++it;
      }
    }
  } else if (warp >= kOutWarp) {
    write_results<T, CP>(p, sm, walk, tmem + 384, L::kOutOff, Y_DONE, first + 8u * Y_FREE);
  } else {
    // (the warpgroups take the chunks in turn; half of every chunk each made a shorter chain from one use of a buffer to
    // the next and 361 us of 336)
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    for (int g = warp >> 2; g < total; g += 2) {
      if (!wait(S_FULL + g % 3, (g / 3) & 1)) break;
      tc_fence_after();
      const uint32_t ts = lanes + (g % 3) * 128;
      float a[2][16], b[2][16];
      auto load = [&](int i) {
        tmem_ld16(ts + 16 * i, reinterpret_cast<uint32_t*>(a[i & 1]));
        tmem_ld16(ts + 64 + 16 * i, reinterpret_cast<uint32_t*>(b[i & 1]));
      };
      load(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // 16 units at a time, the next ones on their way
        tmem_wait_ld();
        if (i < 3) load(i + 1);
        uint32_t h[8];
        gate_units<T, 16>(a[i & 1], b[i & 1], h);
        tmem_st8(ts + 8 * i, h);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(first + 8u * (H_READY + g % 3));
    }
  }
  finish<2>(sm, warp == kMmaWarp, tmem, p.status);
}

// ------------------------------------------------------------------ dX
// The chunks alternate between two buffers of TMEM, [0, 192) and [192, 384): S and dH, with da and db over dH's columns (16
// and 16 of each 32), so that the next S only waits for a and b to be read; dX [384, 384 + CP).
template <typename T, int CP>
__global__ void __launch_bounds__(kRowThreads, 1) ff_dx_kernel(const __grid_constant__ Params p) {
  using L = Rows<CP, true>;
  constexpr int kGU = L::kGU, kD = L::kD;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int XY_FULL = 0, XY_EMPTY = 1, GU_FULL = 2, GU_EMPTY = GU_FULL + kGU, D_FULL = GU_EMPTY + kGU, D_EMPTY = D_FULL + kD,
                S_FULL = D_EMPTY + kD, P_READY = S_FULL + 2, P_FREE = P_READY + 2, DX_DONE = P_FREE + 2, DX_FREE = DX_DONE + 1, NBARS = DX_FREE + 1;
  static_assert(NBARS * 8 <= 256, "barrier area");
  extern __shared__ uint8_t smem_raw[];
  const Smem sm = smem_of(smem_raw);
  volatile int* abort_flag = sm.abort_flag();
  after_previous();
  const bool given_up = device_gave_up(p.status);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NBARS; ++i) mbar_init(sm.bar(i), i == DX_FREE ? 8 : (i >= P_READY && i < P_READY + 2) ? 16 : 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  bool go;
  const uint32_t tmem = start<2>(sm, warp == kMmaWarp, given_up, &go);
  const Walk walk(p);
  const int n = p.chunks, total = go ? walk.total : 0;
  const uint32_t first = in_cta(sm.base, 0);   // the first CTA's barriers
  const Filler fill{sm.base, first, walk.rank};
  const uint32_t x_tile = sm.base + L::kXOff, dy_tile = x_tile + L::kX;
  auto wait = [&](int b, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(sm.bar(b), parity, abort_flag)); };
  auto gu_tile = [&](int g) { return sm.base + L::kGuOff + (g % kGU) * L::kGuBytes; };
  auto d_tile = [&](int g) { return sm.base + L::kDOff + (g % kD) * L::kDBytes; };

  if (!go) {
  } else if (warp == kTmaWarp) {
    bool ok = true;
    const CUtensorMap* own = walk.rank == 0 ? &p.wg : &p.wu;
    for (int g = 0, c = 0, it = 0; g < total && ok; ++g, c = c + 1 == n ? 0 : c + 1) {
      if (c == 0) {
        if (it > 0) ok = wait(XY_EMPTY, (it - 1) & 1);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t f = fill.expect(XY_FULL, 2 * L::kX);
#pragma unroll
          for (int kb = 0; kb < L::kBlocks; ++kb) {
            tma_load_3d_pair(x_tile + kb * kTile, &p.x, f, kb * 64, walk.row(it), 0);
            tma_load_3d_pair(dy_tile + kb * kTile, &p.dy, f, kb * 64, walk.row(it), 0);
            // (one buffer of rows: the next ones are fetched from L2)
            if (it + 1 < walk.items) {
              tma_prefetch_3d(&p.x, kb * 64, walk.row(it + 1), 0);
              tma_prefetch_3d(&p.dy, kb * 64, walk.row(it + 1), 0);
            }
          }
        }
        __syncwarp();
        ++it;
      }
      if (g >= kGU) ok = wait(GU_EMPTY + g % kGU, (g / kGU - 1) & 1);
      if (!ok) break;
      if (elect_one()) {
        const uint32_t f = fill.expect(GU_FULL + g % kGU, L::kGuBytes), across = gu_tile(g) + L::kSBytes;
#pragma unroll
        for (int kb = 0; kb < L::kBlocks; ++kb) tma_load_3d_pair(gu_tile(g) + kb * (kTile / 2), own, f, kb * 64, c * kChunk, 0);
        tma_load_3d_pair(across, &p.wg_across, f, walk.rank * L::kHalf, c * kChunk, 0);
        tma_load_3d_pair(across + L::kAcross, &p.wu_across, f, walk.rank * L::kHalf, c * kChunk, 0);
      }
      __syncwarp();
    }
  } else if (warp == kTmaDWarp) {
    bool ok = true;
    for (int g = 0, c = 0; g < total && ok; ++g, c = c + 1 == n ? 0 : c + 1) {
      if (g >= kD) ok = wait(D_EMPTY + g % kD, (g / kD - 1) & 1);
      if (!ok) break;
      if (elect_one()) tma_load_3d_pair(d_tile(g), &p.wd, fill.expect(D_FULL + g % kD, L::kDBytes), c * kChunk + walk.rank * 32, 0, 0);
      __syncwarp();
    }
  } else if (warp == kSWarp) {
    bool ok = true;
    for (int g = 0, c = 0, it = 0; g < total && ok && walk.rank == 0; ++g) {
      if (c == 0) ok = wait(XY_FULL, it & 1);
      ok = ok && wait(GU_FULL + g % kGU, (g / kGU) & 1);
      if (ok && g >= 2) ok = wait(P_READY + (g & 1), ((g >> 1) - 1) & 1);   // (a and b have been read)
      if (!ok) break;
      tc_fence_after();
      const uint32_t d = tmem + (g & 1) * 192;
      if (elect_one()) pair_s<kBf16, CP>(d, x_tile, gu_tile(g));
      __syncwarp();
      ok = wait(D_FULL + g % kD, (g / kD) & 1);
      if (ok && g >= 2) ok = wait(P_FREE + (g & 1), ((g >> 1) - 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        // dH = dY Wd, 256 x 64; Wd across, halves of 32 units (rows of 64 bytes)
        const uint64_t ad = make_smem_desc(dy_tile, 16, 1024, kSwizzle128), bd = make_smem_desc(d_tile(g), 512, 512, kSwizzle64);
#pragma unroll
        for (int k = 0; k < CP / 16; ++k)
          umma_ss_pair(d + 128, ad + (k >> 2) * (kTile >> 4) + (k & 3) * 2, bd + k * (1024 >> 4), make_idesc(256, 64, kBf16, false, true), k > 0);
        umma_commit_pair(sm.bar(S_FULL + (g & 1)));
        umma_commit_pair(sm.bar(D_EMPTY + g % kD));
        if (c == n - 1) umma_commit_pair(sm.bar(XY_EMPTY));
      }
      __syncwarp();
      if (++c == n) {
        c = 0;
        ++it;
      }
    }
  } else if (warp == kMmaWarp) {
    bool ok = true;
    for (int g = 0, c = 0, it = 0; g < total && ok && walk.rank == 0; ++g) {
      // (its Wg and Wu are there: they came with those that S was made of)
      ok = wait(P_READY + (g & 1), (g >> 1) & 1);
      if (ok && c == 0 && it > 0) ok = wait(DX_FREE, (it - 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        // B: units down, half the width across
        constexpr uint32_t kRow = L::kHalf * 2;
        constexpr uint64_t kSwz = L::kHalf == 64 ? kSwizzle128 : kSwizzle64;
        constexpr uint32_t idesc = make_idesc(256, CP, kBf16, false, true);
        const uint32_t a = tmem + (g & 1) * 192 + 128, w = gu_tile(g) + L::kSBytes;
        const uint64_t bg = make_smem_desc(w, 8 * kRow, 8 * kRow, kSwz), bu = make_smem_desc(w + L::kAcross, 8 * kRow, 8 * kRow, kSwz);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_ts_pair(tmem + 384, a + (k >> 1) * 32 + (k & 1) * 8, bg + k * (16 * kRow >> 4), idesc, (c > 0 || k > 0) ? 1u : 0u);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_ts_pair(tmem + 384, a + 16 + (k >> 1) * 32 + (k & 1) * 8, bu + k * (16 * kRow >> 4), idesc, 1u);
        umma_commit_pair(sm.bar(P_FREE + (g & 1)));
        umma_commit_pair(sm.bar(GU_EMPTY + g % kGU));
        if (c == n - 1) umma_commit_pair(sm.bar(DX_DONE));
      }
      __syncwarp();
      if (++c == n) {
        c = 0;
        ++it;
      }
    }
  } else if (warp >= kOutWarp) {
    write_results<T, CP>(p, sm, walk, tmem + 384, L::kOutOff, DX_DONE, first + 8u * DX_FREE);
  } else {
    // both warpgroups take half the units of every chunk: its gradients are the longest link of the chain from one
    // use of a buffer to the next
    const int grp = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    for (int g = 0; g < total; ++g) {
      if (!wait(S_FULL + (g & 1), (g >> 1) & 1)) break;
      tc_fence_after();
      const uint32_t ts = lanes + (g & 1) * 192;
      float a[2][16], b[2][16], dh[2][16];
      auto load = [&](int i) {
        const int c = grp * 32 + i * 16;
        tmem_ld16(ts + c, reinterpret_cast<uint32_t*>(a[i]));
        tmem_ld16(ts + 64 + c, reinterpret_cast<uint32_t*>(b[i]));
        tmem_ld16(ts + 128 + c, reinterpret_cast<uint32_t*>(dh[i]));
      };
      load(0);
      tmem_wait_ld();
      load(1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t da[8], db[8];
        grad_units<T, 16, false>(a[i], b[i], dh[i], da, db, nullptr);
        if (i == 0) tmem_wait_ld();
        // (over columns of dH that this warp has read)
        tmem_st8(ts + 128 + grp * 32 + 8 * i, da);
        tmem_st8(ts + 128 + grp * 32 + 16 + 8 * i, db);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(first + 8u * (P_READY + (g & 1)));
    }
  }
  finish<2>(sm, warp == kMmaWarp, tmem, p.status);
}

// ------------------------------------------------------------------ dWg, dWu, dWd
// A CTA has a chunk of hidden units and a share of the row tiles, in runs of at most kRunTiles, after each of which its sums
// go to memory.  TMEM: S [0, 128) and [128, 256), dH [256, 320), [dWg; dWu] [320, 320 + CP), dWd [448, 512).
template <int CP>
struct Weights {   // (warps of this kernel: 0-7 elementwise, 8 TMA, 9 and 10 MMA issuers: S and dH; the gradients)
  static constexpr int kX = CP / 64 * kTile, kStage = 2 * kX;
  static constexpr int kGuBytes = CP / 64 * kTile, kDBytes = CP * 128;
  static constexpr int kXyOff = 1024, kWOff = kXyOff + 2 * kStage, kStgOff = kWOff + kGuBytes + kDBytes;
  static constexpr int smem_bytes() { return 1024 + kStgOff + 3 * kTile; }
  static_assert(smem_bytes() <= kSmemLimit, "shared memory");
};

// S = X [Wg; Wu]^T, 128 x 128, and dH = dY Wd, 128 x 64, of one CTA
template <bool BF16, int CP>
__device__ __forceinline__ void mma_s(uint32_t d, uint32_t x, uint32_t gu) {
  const uint64_t ad = make_smem_desc(x, 16, 1024, kSwizzle128), bd = make_smem_desc(gu, 16, 1024, kSwizzle128);
#pragma unroll
  for (int k = 0; k < CP / 16; ++k) {
    const uint32_t off = (k >> 2) * (kTile >> 4) + (k & 3) * 2;
    umma_ss(d, ad + off, bd + off, make_idesc(128, 128, BF16, false, false), k > 0);
  }
}
template <bool BF16, int CP>
__device__ __forceinline__ void mma_dh(uint32_t d, uint32_t dy, uint32_t wd) {
  const uint64_t ad = make_smem_desc(dy, 16, 1024, kSwizzle128), bd = make_smem_desc(wd, 16, 1024, kSwizzle128);
#pragma unroll
  for (int k = 0; k < CP / 16; ++k)
    umma_ss(d, ad + (k >> 2) * (kTile >> 4) + (k & 3) * 2, bd + k * (2048 >> 4), make_idesc(128, 64, BF16, false, true), k > 0);
}

template <typename T, int CP>
__global__ void __launch_bounds__(kThreads, 1) ff_dw_kernel(const __grid_constant__ Params p) {
  using L = Weights<CP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int X_FULL = 0, X_EMPTY = 2, DY_FULL = 4, DY_EMPTY = 6, W_FULL = 8, S_FULL = 9, DH_FREE = 11, STG_READY = 12, STG_FREE = 13,
                ACC_DONE = 14, ACC_FREE = 15, NBARS = 16;
  extern __shared__ uint8_t smem_raw[];
  const Smem sm = smem_of(smem_raw);
  volatile int* abort_flag = sm.abort_flag();
  after_previous();
  if (device_gave_up(p.status)) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NBARS; ++i) mbar_init(sm.bar(i), i == DH_FREE || i == STG_READY || i == ACC_FREE ? 8 : 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  bool go;
  const uint32_t tmem = start<1>(sm, warp == 9, false, &go);
  const int chunk = blockIdx.x % p.chunks, split = blockIdx.x / p.chunks;
  const int lo = (int)((int64_t)p.tiles * split / p.splits), hi = (int)((int64_t)p.tiles * (split + 1) / p.splits);
  const uint32_t gu = sm.base + L::kWOff, wd = gu + L::kGuBytes, stg = sm.base + L::kStgOff;
  auto xy = [&](int t) { return sm.base + L::kXyOff + (t & 1) * L::kStage; };
  auto wait = [&](int b, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(sm.bar(b), parity, abort_flag)); };
  const int count = hi - lo;   // at least one: there are no more shares than tiles

  if (warp == 8) {
    if (elect_one()) {
      mbar_arrive_expect_tx(sm.bar(W_FULL), L::kGuBytes + L::kDBytes);
#pragma unroll
      for (int kb = 0; kb < CP / 64; ++kb) {
        tma_load_3d(gu + kb * kTile, &p.wg, sm.bar(W_FULL), kb * 64, chunk * kChunk, 0);
        tma_load_3d(gu + kb * kTile + kTile / 2, &p.wu, sm.bar(W_FULL), kb * 64, chunk * kChunk, 0);
      }
      tma_load_3d(wd, &p.wd, sm.bar(W_FULL), chunk * kChunk, 0, 0);
    }
    __syncwarp();
    // x and dy of two tiles, each let go of as soon as its last product is done; the tile after them comes to L2
    bool ok = true;
    for (int t = 0; t < count && ok; ++t) {
      const int row = (lo + t) * 128, next = row + 256;
      if (t >= 2) ok = wait(X_EMPTY + (t & 1), (t / 2 - 1) & 1);
      if (!ok) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(sm.bar(X_FULL + (t & 1)), L::kX);
        load_rows<CP>(&p.x, xy(t), sm.bar(X_FULL + (t & 1)), row);
        if (t + 2 < count)
#pragma unroll
          for (int kb = 0; kb < CP / 64; ++kb) {
            tma_prefetch_3d(&p.x, kb * 64, next, 0);
            tma_prefetch_3d(&p.dy, kb * 64, next, 0);
          }
      }
      __syncwarp();
      if (t >= 2) ok = wait(DY_EMPTY + (t & 1), (t / 2 - 1) & 1);
      if (!ok) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(sm.bar(DY_FULL + (t & 1)), L::kX);
        load_rows<CP>(&p.dy, xy(t) + L::kX, sm.bar(DY_FULL + (t & 1)), row);
      }
      __syncwarp();
    }
  } else if (warp == 9) {
    bool ok = wait(W_FULL, 0);
    for (int t = 0; t < count && ok; ++t) {
      // (S of t - 2, in the same buffer, was read when the elementwise warps let go of its dH)
      ok = wait(X_FULL + (t & 1), (t / 2) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) mma_s<kBf16, CP>(tmem + (t & 1) * 128, xy(t), gu);
      __syncwarp();
      ok = wait(DY_FULL + (t & 1), (t / 2) & 1);
      if (ok && t > 0) ok = wait(DH_FREE, (t - 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        mma_dh<kBf16, CP>(tmem + 256, xy(t) + L::kX, wd);
        umma_commit(sm.bar(S_FULL + (t & 1)));
      }
      __syncwarp();
    }
  } else if (warp == 10) {
    bool ok = true;
    for (int t = 0; t < count && ok; ++t) {
      // (the rows are there: S and dH have read them)
      ok = wait(STG_READY, t & 1);
      const int in_run = t % kRunTiles;
      if (ok && in_run == 0 && t > 0) ok = wait(ACC_FREE, (t / kRunTiles - 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = make_smem_desc(stg, kTile, 1024, kSwizzle128), h = make_smem_desc(stg + 2 * kTile, 16, 1024, kSwizzle128);
        const uint64_t x = make_smem_desc(xy(t), kTile, 1024, kSwizzle128), dy = make_smem_desc(xy(t) + L::kX, kTile, 1024, kSwizzle128);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_ss(tmem + 320, a + k * (2048 >> 4), x + k * (2048 >> 4), make_idesc(128, CP, kBf16, true, true), (in_run > 0 || k > 0) ? 1u : 0u);
        umma_commit(sm.bar(X_EMPTY + (t & 1)));
        // (CP = 64: rows 64-127 of this product read what lies behind the tile and are not used)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_ss(tmem + 448, dy + k * (2048 >> 4), h + k * (2048 >> 4), make_idesc(128, 64, kBf16, true, true), (in_run > 0 || k > 0) ? 1u : 0u);
        umma_commit(sm.bar(DY_EMPTY + (t & 1)));
        umma_commit(sm.bar(STG_FREE));
        if (in_run == kRunTiles - 1 || t == count - 1) umma_commit(sm.bar(ACC_DONE));
      }
      __syncwarp();
    }
  } else {
    const int grp = warp >> 2, wq = warp & 3, row = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)(wq * 32) << 16);
    bool ok = true;
    float* part = p.partials + (int64_t)split * p.partial_stride;
    const int pitch = (int)partial_pitch(p.width), pitch_d = (int)partial_pitch(p.hidden);
    const int64_t in = (int64_t)p.hidden * pitch;
    // this group's half of the columns of the sums; unit: this thread's row of [dWg; dWu]
    auto flush = [&](bool add) {
      const int unit = chunk * kChunk + (row & 63);
#pragma unroll 1
      for (int c = 0; c < CP / 2; c += 32) {
        const int col = grp * (CP / 2) + c;
        float v[32];
        tmem_ld32(lanes + 320 + col, reinterpret_cast<uint32_t*>(v));
        tmem_wait_ld();
        if (unit < p.hidden) add_partials(part + (row >= 64 ? in : 0) + (int64_t)unit * pitch + col, v, pitch - col, add);
      }
      float v[32];
      tmem_ld32(lanes + 448 + grp * 32, reinterpret_cast<uint32_t*>(v));
      tmem_wait_ld();
      const int col = chunk * kChunk + grp * 32;
      if (row < p.width_out) add_partials(part + 2 * in + (int64_t)row * pitch_d + col, v, pitch_d - col, add);
    };
    // 16-byte piece of this thread's row in staged tile `tile`
    auto piece = [&](int tile, int c16) -> uint4* {
      return reinterpret_cast<uint4*>(sm.g + L::kStgOff + tile * kTile + row * 128 + ((c16 ^ (row & 7)) << 4));
    };
    for (int t = 0; t < count && ok; ++t) {
      ok = wait(S_FULL + (t & 1), (t / 2) & 1);
      if (!ok) break;
      tc_fence_after();
      float a[32], b[32], dh[32];
      uint32_t da[16], db[16], h[16];
      const uint32_t ts = lanes + (t & 1) * 128 + grp * 32;
      tmem_ld32(ts, reinterpret_cast<uint32_t*>(a));
      tmem_ld32(ts + 64, reinterpret_cast<uint32_t*>(b));
      tmem_ld32(lanes + 256 + grp * 32, reinterpret_cast<uint32_t*>(dh));
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(DH_FREE));
      grad_units<T, 32, true>(a, b, dh, da, db, h);
      if (t > 0) ok = wait(STG_FREE, (t - 1) & 1);
      if (!ok) break;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        *piece(0, grp * 4 + c) = make_uint4(da[4 * c], da[4 * c + 1], da[4 * c + 2], da[4 * c + 3]);
        *piece(1, grp * 4 + c) = make_uint4(db[4 * c], db[4 * c + 1], db[4 * c + 2], db[4 * c + 3]);
        *piece(2, grp * 4 + c) = make_uint4(h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(STG_READY));
      if (t % kRunTiles == kRunTiles - 1 || t == count - 1) {
        ok = wait(ACC_DONE, (t / kRunTiles) & 1);
        if (!ok) break;
        tc_fence_after();
        flush(t >= kRunTiles || p.add);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.bar(ACC_FREE));
      }
    }
  }
  finish<1>(sm, warp == 9, tmem, p.status);
}

int64_t tiles_of(int64_t x, int tile) { return (x + tile - 1) / tile; }

template <typename T, int CP>
cudaError_t launch(const FusedArgs& g, cudaStream_t stream) {
  Params p = {};
  p.rows = g.x.rows;
  p.tiles = (int)tiles_of(g.x.rows, 128);
  p.chunks = (int)tiles_of(g.wg.rows, kChunk);
  p.y = g.out.p;
  p.ldy = g.out.pitch;
  p.cols = (int)g.out.cols;
  p.y_tma = g.y_tma;
  p.partials = g.partials;
  p.partial_stride = g.partial_stride;
  p.splits = g.splits < p.tiles ? g.splits : p.tiles;
  p.add = g.add;
  p.width = (int)g.wg.cols;
  p.hidden = (int)g.wg.rows;
  p.width_out = (int)g.wd.rows;
  p.status = g.status;
  bool ok = map_of(&p.x, g.bf16, g.x, 64, 128) && map_of(&p.wg, g.bf16, g.wg, 64, 64) && map_of(&p.wu, g.bf16, g.wu, 64, 64) &&
            map_of(&p.wd, g.bf16, g.wd, g.what == kDx ? 32 : 64, g.what == kForward ? CP / 2 : CP);
  if (g.what == kDx) ok = ok && map_of(&p.wg_across, g.bf16, g.wg, CP / 2, 64) && map_of(&p.wu_across, g.bf16, g.wu, CP / 2, 64);
  if (g.what != kForward) ok = ok && map_of(&p.dy, g.bf16, g.dy, 64, 128);
  if (g.what != kDw && g.y_tma) ok = ok && map_of(&p.out, g.bf16, g.out, 64, 128);
  if (!ok) return cudaErrorInvalidValue;
  const int sms = sm_count();
  cudaError_t e;
  if (g.what == kDw) {
    if ((e = opt_in_smem<ff_dw_kernel<T, CP>>(Weights<CP>::smem_bytes())) != cudaSuccess) return e;
    return launch_early(ff_dw_kernel<T, CP>, dim3((unsigned)(p.chunks * p.splits)), kThreads, Weights<CP>::smem_bytes(), stream, p);
  }
  const int pairs = (p.tiles + 1) / 2;
  const dim3 grid(2 * (pairs < sms / 2 ? pairs : sms / 2));
  if (g.what == kDx) {
    if ((e = opt_in_smem<ff_dx_kernel<T, CP>>(Rows<CP, true>::smem_bytes())) != cudaSuccess) return e;
    return launch_clusters(ff_dx_kernel<T, CP>, grid, kRowThreads, Rows<CP, true>::smem_bytes(), stream, 2, p);
  }
  if ((e = opt_in_smem<ff_forward_kernel<T, CP>>(Rows<CP, false>::smem_bytes())) != cudaSuccess) return e;
  return launch_clusters(ff_forward_kernel<T, CP>, grid, kRowThreads, Rows<CP, false>::smem_bytes(), stream, 2, p);
}

template <typename T>
cudaError_t launch_width(const FusedArgs& g, cudaStream_t s) {
  return g.wg.cols <= 64 && g.wd.rows <= 64 ? launch<T, 64>(g, s) : launch<T, 128>(g, s);
}

}  // namespace

cudaError_t fused(const FusedArgs& g, cudaStream_t s) {
  return g.bf16 ? launch_width<__nv_bfloat16>(g, s) : launch_width<__half>(g, s);
}

int fused_weight_splits(int64_t rows, int64_t hidden, int sms) {
  const int64_t chunks = tiles_of(hidden, kChunk), tiles = tiles_of(rows, 128);
  int64_t s = sms / chunks;
  if (s > tiles) s = tiles;
  return s < 1 ? 1 : (int)s;
}

}  // namespace ff
}  // namespace trifast
