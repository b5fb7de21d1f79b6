// The matrix products of the gated feed-forward block
//     a = X Wg^T,  b = X Wu^T,  h = silu(a) * b,  y = h Wd^T
// and of its backward pass
//     dh = dY Wd,  db = dh silu(a),  da = dh b silu'(a),
//     dX = da Wg + db Wu,  dWg = da^T X,  dWu = db^T X,  dWd = dY^T h
// on the tensor cores, as one kernel with four epilogues (Mode in ff_gemm.cuh).
//
// A tile has 128 rows and up to 256 fp32 columns in TMEM, twice, so that the epilogue of one tile runs under the MMAs of
// the next.  Where there is more than one row tile, two CTAs share an MMA (CG = 2): each has its 128 rows of A and of
// the result, and half of B's tile, which the tensor cores of both read.  kHidden has 128 units a tile: a and b once, 256
// columns, dH twice, so that the next dH runs under the epilogue (64 units, all of them twice, fetched X and dY twice as
// often: 72 us of 58 for 8192 rows, width 512, hidden 2048).
//
// Operands come in blocks of 64 along the contraction, through a ring of stages that TMA fills (128-byte swizzle).
// Both majors are read as they lie: where the contraction runs along a matrix's rows the tile is an MN-major operand of
// 64-element columns.  CTAs are persistent, one per SM, the tiles of one row block next to one another.
// Warps 0-7: epilogue (two warpgroups, each half of a tile's columns), 8: TMA, 9: MMA issuer (of the pair's first CTA).
//
// fp32: every value is the sum of three bf16 ones (ff_support.cu), and a product is the six products of parts that are not
// below 2^-22 of it.  A stage holds all three parts of both operands.  The accumulators in TMEM round towards zero, so
// that a long sum drifts (1.0e-7 of a sum of positive terms with every MMA): a sum takes one stage, the smallest products first, and
// the epilogue adds the sums up in fp32 registers, rounded to nearest.
//
// What bounds it: the tiles' way from L2.  A pair's 256 x 256 tile takes 32 KB a CTA per 64 of the contraction, which the
// tensor pipe works on for 512 cycles: 64 bytes a cycle, of which about 41 arrive (9.4 TB/s on all SMs).  65,536 rows of
// 512, hidden 1024, bf16: 110 us for the gate, 56 for the result, 1.25 PFLOP/s.

#include <initializer_list>
#include <type_traits>

#include "ff_device.cuh"

namespace trifast {
namespace ff {
namespace {
using namespace tc;

constexpr int kBK = 64;                  // contraction per stage
constexpr int kTileA = 128 * kBK * 2;    // bytes of an operand tile of 128 rows
constexpr int kThreads = 320;
constexpr int kSmemLimit = 232448;

// Columns per B matrix (NT), accumulator columns, stages and staging of results by mode.
template <int PARTS, int MODE, int NT, int CG>
struct Cfg {
  static constexpr int kAccCols = MODE == kGate || MODE == kHidden ? 2 * NT : NT;
  static constexpr int kBRows = MODE == kGate || MODE == kHidden ? 2 * NT : NT;   // largest of a stage, in all
  static constexpr int kTileB = kBRows / CG * kBK * 2;
  static constexpr int kStageBytes = PARTS * (kTileA + kTileB);   // all planes of A, then of B
  // result tiles of 128 rows x 64 columns
  static constexpr int kOutTiles = MODE == kGate ? NT / 64 : MODE == kHidden ? (PARTS == 3 ? 1 : 3) : MODE == kLinear && PARTS == 1 ? 2 : 0;
  static constexpr int kStages = (kSmemLimit - 2048 - kOutTiles * kTileA) / kStageBytes;
  static constexpr int kBufCols = kAccCols > 128 ? 256 : 128;    // TMEM columns between the two buffers
  static constexpr int smem_bytes() { return 1024 + 1024 + kStages * kStageBytes + kOutTiles * kTileA; }
  static_assert(kAccCols <= 256 && kStages >= (PARTS == 3 ? 2 : 3) && smem_bytes() <= kSmemLimit, "tile configuration");
};

struct Params {
  CUtensorMap a[3], b[3], out[3];
  int64_t m[3], n[3], k[3];   // kWeight: of each product; else of product 0 (k: of each phase)
  int m_tiles[3], n_tiles[3], tiles;
  int phases;
  void* y;
  int64_t ldy;
  int y_tma;
  float* partials;
  int64_t partial_stride;
  int splits, split_tiles, add;
  unsigned int* status;
};

// Pairs of planes (of A, of B) whose products make up a product of fp32 values, the smallest first.
__device__ __forceinline__ int plane_a(int q) { return (0x001021 >> (4 * q)) & 15; }   // 1 2 0 1 0 0
__device__ __forceinline__ int plane_b(int q) { return (0x010201 >> (4 * q)) & 15; }   // 1 0 2 0 1 0

// One bf16 part of two values, cut and not rounded, and what is left of them: three parts hold all 24 bits.
__device__ __forceinline__ uint32_t take_part(float& v0, float& v1) {
  const uint32_t a = __float_as_uint(v0), b = __float_as_uint(v1);
  v0 -= __uint_as_float(a & 0xffff0000u);
  v1 -= __uint_as_float(b & 0xffff0000u);
  return __byte_perm(a, b, 0x7632);
}

// Sums in TMEM that a contraction of so many stages takes when PARTS is 3 (an empty one takes one all the same).
__device__ __forceinline__ int sums_of(int blocks) { return blocks < 1 ? 1 : blocks; }

struct TileAt {
  int m0, n0;     // first row and column
  int job, split;
};

template <int MODE, int NT, int CG>
__device__ __forceinline__ TileAt tile_at(const Params& p, int t, int rank) {
  TileAt r;
  r.job = 0;
  r.split = 0;
  if constexpr (MODE == kWeight) {
    // (one split after the other: its rows of the operands stay in L2 for all of its tiles.  The splits of a tile side by
    // side read all rows anew in every round, 235 MB of 8192 rows, width 1024, hidden 4096)
    r.split = t / p.split_tiles;
    t -= r.split * p.split_tiles;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (r.job == j && t >= p.m_tiles[j] * p.n_tiles[j]) {
        t -= p.m_tiles[j] * p.n_tiles[j];
        r.job = j + 1;
      }
  }
  const int nt = p.n_tiles[r.job];
  r.m0 = (t / nt) * 128 * CG + rank * 128;
  r.n0 = (t % nt) * NT;
  return r;
}

// T: type of the operands; PARTS: planes of each (1, or 3 for fp32); OUT: type of kLinear's result.
template <typename T, int PARTS, typename OUT, int MODE, int NT, bool B_MN, int CG>
__global__ void __launch_bounds__(kThreads, 1) ff_gemm_kernel(const __grid_constant__ Params p) {
  using C = Cfg<PARTS, MODE, NT, CG>;
  constexpr int S = C::kStages;
  constexpr int FULL = 0, EMPTY = S, ACC_FULL = 2 * S, ACC_EMPTY = 2 * S + 2, NBARS = 2 * S + 4;
  static_assert(NBARS * 8 <= 240, "barrier area");
  constexpr int kPairs = PARTS == 1 ? 1 : 6;
  constexpr bool kAMn = MODE == kWeight;
  constexpr bool kOneAB = MODE == kHidden && PARTS == 1;   // a and b have one place in TMEM, dH two
  constexpr int kDhCol = 256;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + 256);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + 260);
  auto bar = [&](int i) -> uint32_t { return base + 8u * i; };
  const int rank = CG == 2 ? (int)cluster_rank() : 0;
  // (the pair's first CTA counts what arrives, issues the MMAs and is told when results have been read)
  auto first_bar = [&](int i) -> uint32_t { return CG == 2 ? in_cta(bar(i), 0) : bar(i); };
  auto a_tile = [&](int s) -> uint32_t { return base + 1024 + s * C::kStageBytes; };
  auto b_tile = [&](int s) -> uint32_t { return a_tile(s) + PARTS * kTileA; };
  constexpr uint32_t out_off = 1024 + S * C::kStageBytes;

  after_previous();
  const bool given_up = device_gave_up(p.status);
  if (CG == 1 && given_up) return;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(bar(FULL + s), 1);
      mbar_init(bar(EMPTY + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(ACC_FULL + i), 1);
      mbar_init(bar(ACC_EMPTY + i), 8 * CG);
    }
    *abort_flag = 0;
    if (CG == 2) *reinterpret_cast<volatile uint32_t*>(gbase + 264) = given_up;
    mbar_fence_init();
  }
  if (warp == 9) {
    if (CG == 2) {
      tmem_alloc_pair(smem_u32(tmem_slot), 512);
    } else {
      tmem_alloc(smem_u32(tmem_slot), 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // both CTAs of a pair go on, or neither
  bool go = true;
  if (CG == 2) go = (load_cluster(in_cta(base + 264, 0)) | load_cluster(in_cta(base + 264, 1))) == 0;

  // blocks of the contraction of phase ph of a tile
  auto k_range = [&](const TileAt& t, int ph, int& lo, int& hi) {
    const int blocks = (int)((p.k[MODE == kWeight ? 0 : ph] + kBK - 1) / kBK);
    lo = 0;
    hi = blocks;
    if (MODE == kWeight) {
      lo = (int)((int64_t)blocks * t.split / p.splits);
      hi = (int)((int64_t)blocks * (t.split + 1) / p.splits);
    }
  };
  const int phases = MODE == kHidden ? 2 : MODE == kLinear ? p.phases : 1;

  if (!go) {
  } else if (warp == 8) {
    // ------------------------------------------------------------ TMA producer
    int g = 0;
    bool ok = true;
    for (int w = blockIdx.x / CG; w < p.tiles && ok; w += gridDim.x / CG) {
      const TileAt t = tile_at<MODE, NT, CG>(p, w, rank);
      for (int ph = 0; ph < phases && ok; ++ph) {
        int lo, hi;
        k_range(t, ph, lo, hi);
        const CUtensorMap* ma = &p.a[MODE == kWeight ? t.job : ph];
        for (int kb = lo; kb < hi; ++kb, ++g) {
          const int s = g % S;
          if (g >= S) ok = mbar_wait(bar(EMPTY + s), ((g / S) - 1) & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (elect_one()) {
            const uint32_t f = first_bar(FULL + s);
            const int kc = kb * kBK;
            // (the first CTA's arrival, with the bytes of both)
            auto expect = [&](int bytes) {
              if (rank == 0) mbar_arrive_expect_tx(bar(FULL + s), CG * bytes);
            };
            auto load = [&](uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2) {
              if (CG == 2)
                tma_load_3d_pair(dst, map, f, c0, c1, c2);
              else
                tma_load_3d(dst, map, f, c0, c1, c2);
            };
            if constexpr (MODE == kHidden)
              expect(PARTS * (kTileA + (ph == 0 ? 1 : 2) * NT / CG * kBK * 2));
            else
              expect(C::kStageBytes);
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
              const uint32_t at = a_tile(s) + q * kTileA, bt = b_tile(s) + q * C::kTileB;
              const int n0 = t.n0 + rank * (NT / CG);   // this CTA's part of B's tile
              if constexpr (kAMn) {
#pragma unroll
                for (int i = 0; i < 2; ++i) load(at + i * 8192, ma, t.m0 + 64 * i, kc, q);
              } else {
                load(at, ma, kc, t.m0, q);
              }
              if (MODE == kGate || (MODE == kHidden && ph == 1)) {
                // Wg and Wu: one each of a pair
                load(bt, &p.b[rank], kc, t.n0, q);
                if (CG == 1) load(bt + NT * kBK * 2, &p.b[1], kc, t.n0, q);
              } else {
                const CUtensorMap* mb = &p.b[MODE == kHidden ? 2 : MODE == kWeight ? t.job : ph];
                if constexpr (MODE == kHidden || B_MN) {
#pragma unroll
                  for (int i = 0; i < NT / CG / 64; ++i) load(bt + i * 8192, mb, n0 + 64 * i, kc, q);
                } else {
                  load(bt, mb, kc, n0, q);
                }
              }
            }
          }
          __syncwarp();
        }
      }
    }
  } else if (warp == 9 && rank == 0) {
    // ------------------------------------------------------------ MMA issuer
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    int g = 0, it = 0;   // running stage, and running sum (a buffer of TMEM)
    bool ok = true;
    uint32_t acc = tmem_base;
    auto wait_read = [&](int sum) {   // until the epilogue has read this sum
      const int e = ACC_EMPTY + (sum & 1), parity = (sum >> 1) & 1;
      if (sum >= 0) ok = mbar_wait(bar(e), parity, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    };
    auto open_sum = [&] {
      acc = tmem_base + (it & 1) * C::kBufCols;
      // (kHidden's dH goes where that of the sum before the last was, which has been read: a and b of the last sum
      // waited for it)
      if (!kOneAB) wait_read(it - 2);
    };
    auto commit = [&](int b) {
      if (CG == 2)
        umma_commit_pair(bar(b));
      else
        umma_commit(bar(b));
    };
    auto close_sum = [&] {
      if (elect_one()) commit(ACC_FULL + (it & 1));
      __syncwarp();
      ++it;
    };
    for (int w = blockIdx.x / CG; w < p.tiles && ok; w += gridDim.x / CG) {
      const TileAt t = tile_at<MODE, NT, CG>(p, w, rank);
      open_sum();
      for (int ph = 0; ph < phases && ok; ++ph) {
        int lo, hi;
        k_range(t, ph, lo, hi);
        const int steps = hi - lo;
        if (PARTS == 3 && ph > 0) {
          close_sum();
          open_sum();
        }
        if (kOneAB && ph == 1) {
          wait_read(it - 1);
          if (!ok) break;
        }
        // (kLinear's two products add up in one accumulator; kHidden's phases have their own)
        bool first = PARTS == 3 || MODE != kLinear || ph == 0;
        for (int i = 0; i < steps && ok; ++i, ++g) {
          if (PARTS == 3 && i > 0) {
            close_sum();
            open_sum();
            if (!ok) break;
            first = true;
          }
          const int s = g % S;
          ok = mbar_wait(bar(FULL + s), (g / S) & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const bool dh = MODE == kHidden && ph == 0;
            const bool bmn = dh || B_MN;
            const uint32_t idesc = dh ? make_idesc(128 * CG, NT, kBf16, false, true)
                                      : make_idesc(128 * CG, C::kBRows, kBf16, kAMn, B_MN);
            const uint32_t d = !kOneAB ? acc : dh ? tmem_base + kDhCol + (it & 1) * NT : tmem_base;
            const uint64_t ad = make_smem_desc(a_tile(s), kAMn ? 8192 : 16, 1024, kSwizzle128);
            const uint64_t bd = make_smem_desc(b_tile(s), bmn ? 8192 : 16, 1024, kSwizzle128);
            // 16 of the contraction: 32 bytes along a row, or 16 rows of an MN-major tile
            const uint32_t sa = kAMn ? 2048 >> 4 : 32 >> 4, sb = bmn ? 2048 >> 4 : 32 >> 4;
#pragma unroll
            for (int q = 0; q < kPairs; ++q) {
              const uint32_t qa = PARTS == 3 ? plane_a(q) * (kTileA >> 4) : 0, qb = PARTS == 3 ? plane_b(q) * (C::kTileB >> 4) : 0;
#pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk) {
                const uint32_t add = (q > 0 || kk > 0 || !first) ? 1u : 0u;
                if (CG == 2)
                  umma_ss_pair(d, ad + kk * sa, bd + kk * sb, idesc, add);
                else
                  umma_ss(d, ad + qa + kk * sa, bd + qb + kk * sb, idesc, add);
              }
            }
            commit(EMPTY + s);
          }
          __syncwarp();
          first = false;
        }
      }
      if (!ok) break;
      close_sum();
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ epilogue
    const int grp = warp >> 2, wq = warp & 3, row = tid & 127;
    const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
    int it = 0;   // running sum
    bool ok = true;
    // 16-byte piece `c16` of this thread's row in a 128 x 64 result tile (128-byte swizzle)
    auto out_piece = [&](int tile, int c16) -> uint4* {
      return reinterpret_cast<uint4*>(gbase + out_off + tile * kTileA + row * 128 + ((c16 ^ (row & 7)) << 4));
    };
    // kHidden's result tiles, and kGate's of 64 columns, are written by both groups
    constexpr bool kShared = MODE == kHidden || (MODE == kGate && NT == 64);
    const int bar_id = kShared ? 3 : 1 + grp;
    constexpr int kBarThreads = kShared ? 256 : 128;
    const bool leader = kShared ? tid == 0 : row == 0;
    uint32_t acc = tmem_base;
    // (all warps of a barrier go on, or none: the barriers below count on it)
    auto wait_sum = [&] {
      ok = mbar_wait(bar(ACC_FULL + (it & 1)), (it >> 1) & 1, abort_flag);
      ok = group_all(bar_id, kBarThreads, ok);
      tc_fence_after();
      acc = tmem_base + lane_base + (it & 1) * C::kBufCols;
    };
    auto release = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2)
          mbar_arrive_cluster(first_bar(ACC_EMPTY + (it & 1)));
        else
          mbar_arrive(bar(ACC_EMPTY + (it & 1)));
      }
      ++it;
    };
    // PARTS = 3: this thread's columns of each matrix, added up over the sums
    constexpr int kCols = NT / 2, kSets = MODE == kGate ? 2 : MODE == kHidden ? 3 : 1;
    float total[PARTS == 3 ? kSets : 1][PARTS == 3 ? kCols : 1];
    for (int w = blockIdx.x / CG; w < p.tiles; w += gridDim.x / CG) {
      const TileAt t = tile_at<MODE, NT, CG>(p, w, rank);
      bool none = false;   // an empty contraction: its sum is 0, and nothing wrote TMEM
      if constexpr (MODE == kWeight) {
        int lo, hi;
        k_range(t, 0, lo, hi);
        none = hi <= lo;
      }
      if constexpr (PARTS == 1) {
        wait_sum();
      } else {
#pragma unroll
        for (int m = 0; m < kSets; ++m)
#pragma unroll
          for (int e = 0; e < kCols; ++e) total[m][e] = 0.f;
#pragma unroll
        for (int ph = 0; ph < 2; ++ph) {
          if (ph >= phases) continue;
          int lo, hi;
          k_range(t, ph, lo, hi);
          const int sums = sums_of(hi - lo);
          for (int i = 0; i < sums && ok; ++i) {
            wait_sum();
            if (!ok) break;
            constexpr int kLast = kSets;
            const int m0 = MODE == kHidden && ph == 0 ? 2 : 0, m1 = MODE == kHidden && ph == 1 ? 2 : kLast;
#pragma unroll
            for (int m = 0; m < kSets; ++m) {
              if (m < m0 || m >= m1) continue;
#pragma unroll
              for (int c = 0; c < kCols; c += 32) {
                float v[32];
                tmem_ld32(acc + (m - m0) * NT + grp * kCols + c, reinterpret_cast<uint32_t*>(v));
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) total[m][c + e] += none ? 0.f : v[e];
              }
            }
            release();
          }
        }
      }
      if (!ok) break;
      // columns [c, c + 32) of matrix m of this thread's half
      auto columns = [&](int m, int c, float* v) {
        if constexpr (PARTS == 3) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = total[m][c + e];
        } else {
          tmem_ld32(acc + m * NT + grp * kCols + c, reinterpret_cast<uint32_t*>(v));
        }
      };
      auto loaded = [&](bool last) {
        if constexpr (PARTS == 1) {
          tmem_wait_ld();
          if (last) release();
        }
      };
      if constexpr (MODE == kGate) {
        float h[kCols];               // PARTS = 3; else packed
        uint32_t packed[kCols / 2];
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
          float a[32], b[32];
          columns(0, c, a);
          columns(1, c, b);
          loaded(c + 32 == kCols);
          if constexpr (PARTS == 1) {
            gate_units<T, 32>(a, b, packed + c / 2);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) h[c + e] = a[e] * sigmoid(a[e]) * b[e];
          }
        }
        const int tile = kShared ? 0 : grp, piece = kShared ? grp * (kCols / 8) : 0, col = t.n0 + tile * 64;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
          if (leader) bulk_wait_read();
          group_sync(bar_id, kBarThreads);
#pragma unroll
          for (int c = 0; c < kCols; c += 8) {
            if constexpr (PARTS == 3) {
#pragma unroll
              for (int e = 0; e < 8; e += 2) packed[(c + e) >> 1] = take_part(h[c + e], h[c + e + 1]);
            }
            const uint32_t* u = packed + c / 2;
            *out_piece(tile, piece + (c >> 3)) = make_uint4(u[0], u[1], u[2], u[3]);
          }
          fence_async_smem();
          group_sync(bar_id, kBarThreads);
          if (leader && col < p.n[0] && t.m0 < p.m[0]) {
            tma_store_3d(&p.out[0], base + out_off + tile * kTileA, col, t.m0, q);
            bulk_commit();
          }
        }
      } else if constexpr (MODE == kHidden) {
        static_assert(MODE != kHidden || NT == (PARTS == 1 ? 128 : 64), "units of a tile");
        // 64 units at a time, each group half of them
#pragma unroll 1
        for (int u0 = 0; u0 < NT; u0 += 64) {
          float r[3][32];               // PARTS = 3; else packed
          uint32_t packed[3][16];
          {
            float a[32], b[32], dh[32];
            if constexpr (PARTS == 1) {
              const uint32_t at = tmem_base + lane_base + u0 + grp * 32;
              tmem_ld32(at, reinterpret_cast<uint32_t*>(a));
              tmem_ld32(at + NT, reinterpret_cast<uint32_t*>(b));
              tmem_ld32(at + kDhCol + (it & 1) * NT, reinterpret_cast<uint32_t*>(dh));
              tmem_wait_ld();
              if (u0 + 64 == NT) release();
              grad_units<T, 32, true>(a, b, dh, packed[0], packed[1], packed[2]);
            } else {
              columns(0, 0, a);
              columns(1, 0, b);
              columns(2, 0, dh);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float s = sigmoid(a[e]), u = a[e] * s;
                r[0][e] = dh[e] * b[e] * fmaf(u, 1.f - s, s);
                r[1][e] = dh[e] * u;
                r[2][e] = u * b[e];
              }
            }
          }
          const int col = t.n0 + u0;
          const bool inside = t.m0 < p.m[0] && col < p.n[0];
          auto begin = [&] {
            if (leader) bulk_wait_read();
            group_sync(bar_id, kBarThreads);
          };
          auto put = [&](int tile, const uint32_t* u) {
#pragma unroll
            for (int c = 0; c < 4; ++c) *out_piece(tile, grp * 4 + c) = make_uint4(u[4 * c], u[4 * c + 1], u[4 * c + 2], u[4 * c + 3]);
          };
          auto end = [&] {
            fence_async_smem();
            group_sync(bar_id, kBarThreads);
          };
          if constexpr (PARTS == 1) {
            begin();
#pragma unroll
            for (int o = 0; o < 3; ++o) put(o, packed[o]);
            end();
            if (leader && inside) {
#pragma unroll
              for (int o = 0; o < 3; ++o) tma_store_3d(&p.out[o], base + out_off + o * kTileA, col, t.m0, 0);
              bulk_commit();
            }
          } else {
            // (one result tile in shared memory: the operands' planes take the rest)
#pragma unroll
            for (int o = 0; o < 3; ++o)
#pragma unroll
              for (int q = 0; q < PARTS; ++q) {
#pragma unroll
                for (int e = 0; e < 32; e += 2) packed[0][e >> 1] = take_part(r[o][e], r[o][e + 1]);
                begin();
                put(0, packed[0]);
                end();
                if (leader && inside) {
                  tma_store_3d(&p.out[o], base + out_off, col, t.m0, q);
                  bulk_commit();
                }
              }
          }
        }
      } else if constexpr (MODE == kLinear) {
        const int64_t gr = (int64_t)t.m0 + row;
        OUT* yr = reinterpret_cast<OUT*>(p.y) + gr * p.ldy;
        constexpr int kStep = kCols < 64 ? kCols : 64;
        static_assert(MODE != kLinear || PARTS == 3 || kStep == 64, "result tiles are 64 columns");
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += kStep) {
          const int col = t.n0 + grp * kCols + c0;
          float v[kStep];
#pragma unroll
          for (int c = 0; c < kStep; c += 32) columns(0, c0 + c, v + c);
          loaded(c0 + kStep == kCols);
          if constexpr (std::is_same<OUT, float>::value) {
            if (gr < p.m[0]) {
              if (p.ldy % 4 == 0 && col + kStep <= p.n[0] && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0) {
#pragma unroll
                for (int e = 0; e < kStep; e += 4)
                  *reinterpret_cast<float4*>(yr + col + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
              } else {
#pragma unroll
                for (int e = 0; e < kStep; ++e)
                  if (col + e < p.n[0]) yr[col + e] = v[e];
              }
            }
          } else {
            if (leader && p.y_tma) bulk_wait_read();
            group_sync(bar_id, kBarThreads);
#pragma unroll
            for (int c = 0; c < 64; c += 8) {
              uint4 u;
              u.x = pack2<T>(v[c], v[c + 1]);
              u.y = pack2<T>(v[c + 2], v[c + 3]);
              u.z = pack2<T>(v[c + 4], v[c + 5]);
              u.w = pack2<T>(v[c + 6], v[c + 7]);
              *out_piece(grp, c >> 3) = u;
            }
            if (p.y_tma) {
              fence_async_smem();
              group_sync(bar_id, kBarThreads);
              if (leader && col < p.n[0] && t.m0 < p.m[0]) {
                tma_store_3d(&p.out[0], base + out_off + grp * kTileA, col, t.m0, 0);
                bulk_commit();
              }
            } else {
              // rows that TMA cannot address: a warp writes one row at a time, two columns a lane
              group_sync(bar_id, kBarThreads);
              const int c = col + 2 * lane;
              for (int r = wq; r < 128 && t.m0 + r < p.m[0]; r += 4) {
                const uint32_t u = *reinterpret_cast<const uint32_t*>(
                    gbase + out_off + grp * kTileA + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2)));
                uint16_t* dst = reinterpret_cast<uint16_t*>(p.y) + ((int64_t)t.m0 + r) * p.ldy + c;
                if (c < p.n[0]) dst[0] = (uint16_t)u;
                if (c + 1 < p.n[0]) dst[1] = (uint16_t)(u >> 16);
              }
            }
          }
        }
      } else {
        // fp32 partial sums
        const int64_t n = p.n[t.job], gr = (int64_t)t.m0 + row;
        int64_t off = (int64_t)t.split * p.partial_stride;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (j < t.job) off += p.m[j] * partial_pitch(p.n[j]);
        const int pitch = (int)partial_pitch(n);
        float* dst = p.partials + off + gr * pitch;
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 32) {
          const int col = t.n0 + grp * kCols + c0;
          float v[32];
          columns(0, c0, v);
          loaded(c0 + 32 == kCols);
          if (none) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0.f;
          }
          if (gr < p.m[t.job]) add_partials(dst + col, v, pitch - col, p.add);
        }
      }
    }
    bulk_wait();
  }

  // -------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000LL) {
    }
    if (tid == 0) set_status(p.status, kStatusTimeoutFeedForward);
    __syncthreads();
  }
  // (neither CTA of a pair goes before the other's last access to it)
  if (CG == 2) cluster_sync();
  if (warp == 9) {
    tc_fence_after();
    if (CG == 2)
      tmem_dealloc_pair(tmem_base, 512);
    else
      tmem_dealloc(tmem_base, 512);
  }
}

int64_t tiles_of(int64_t x, int tile) { return (x + tile - 1) / tile; }

bool weight_pairs(bool f32, std::initializer_list<int64_t> m) {
  for (int64_t c : m)
    if (f32 || c <= 128) return false;
  return true;
}

template <typename T, int PARTS, typename OUT, int MODE, int NT, bool B_MN, int CG>
cudaError_t launch_group(const GemmArgs& g, cudaStream_t stream) {
  using C = Cfg<PARTS, MODE, NT, CG>;
  Params p = {};
  bool ok = true;
  int64_t tiles = 0;
  if (MODE == kWeight) {
    for (int j = 0; j < 3; ++j) {
      p.m[j] = g.a[j].cols;
      p.n[j] = g.b[j].cols;
      p.k[j] = g.a[j].rows;
      p.m_tiles[j] = (int)tiles_of(p.m[j], 128 * CG);
      p.n_tiles[j] = (int)tiles_of(p.n[j], NT);
      tiles += (int64_t)p.m_tiles[j] * p.n_tiles[j] * g.splits;
      ok = ok && map_of(&p.a[j], g.bf16, g.a[j], 64, kBK) && map_of(&p.b[j], g.bf16, g.b[j], 64, kBK);
    }
  } else {
    p.phases = MODE == kHidden ? 2 : MODE == kLinear ? g.products : 1;
    p.m[0] = g.a[0].rows;
    p.n[0] = MODE == kLinear && B_MN ? g.b[0].cols : g.b[0].rows;
    p.m_tiles[0] = (int)tiles_of(p.m[0], 128 * CG);
    p.n_tiles[0] = (int)tiles_of(p.n[0], NT);
    tiles = (int64_t)p.m_tiles[0] * p.n_tiles[0];
    for (int i = 0; i < p.phases; ++i) {
      p.k[i] = g.a[i].cols;
      ok = ok && map_of(&p.a[i], g.bf16, g.a[i], kBK, 128);
    }
    if (MODE == kLinear) {
      for (int i = 0; i < p.phases; ++i)
        ok = ok && (B_MN ? map_of(&p.b[i], g.bf16, g.b[i], 64, kBK) : map_of(&p.b[i], g.bf16, g.b[i], kBK, NT / CG));
      if (g.y_tma) ok = ok && map_of(&p.out[0], g.bf16, g.out[0], 64, 128);
    } else {
      for (int i = 0; i < 2; ++i) ok = ok && map_of(&p.b[i], g.bf16, g.b[i], kBK, NT);
      if (MODE == kHidden) ok = ok && map_of(&p.b[2], g.bf16, g.b[2], 64, kBK);
      for (int i = 0; i < (MODE == kHidden ? 3 : 1); ++i) ok = ok && map_of(&p.out[i], g.bf16, g.out[i], 64, 128);
    }
  }
  if (!ok || tiles > INT32_MAX / 2) return cudaErrorInvalidValue;
  if (tiles == 0) return cudaSuccess;
  p.tiles = (int)tiles;
  p.y = g.out[0].p;
  p.ldy = g.out[0].pitch;
  p.y_tma = g.y_tma;
  p.partials = g.partials;
  p.partial_stride = g.partial_stride;
  p.splits = g.splits;
  p.split_tiles = MODE == kWeight ? (int)(tiles / g.splits) : 0;
  p.add = g.add;
  p.status = g.status;
  constexpr auto kern = ff_gemm_kernel<T, PARTS, OUT, MODE, NT, B_MN, CG>;
  cudaError_t e = opt_in_smem<kern>(C::smem_bytes());
  if (e != cudaSuccess) return e;
  const int groups = sm_count() / CG, ctas = (p.tiles < groups ? p.tiles : groups) * CG;
  return launch_clusters(kern, dim3(ctas), kThreads, C::smem_bytes(), stream, CG, p);
}

template <typename T, int PARTS, typename OUT, int MODE, int NT, bool B_MN>
cudaError_t launch(const GemmArgs& g, cudaStream_t s) {
  // pairs where every result has more than one row tile (fp32, whose epilogues add up sums, gains nothing from them)
  if constexpr (PARTS == 1) {
    bool pairs = MODE != kWeight && g.a[0].rows > 128;
    if (MODE == kWeight) pairs = weight_pairs(false, {g.a[0].cols, g.a[1].cols, g.a[2].cols});
    if (pairs) return launch_group<T, PARTS, OUT, MODE, NT, B_MN, 2>(g, s);
  }
  return launch_group<T, PARTS, OUT, MODE, NT, B_MN, 1>(g, s);
}

// 256 columns a tile where every result has more than 128 (fp32: 128, for the sums in registers).
bool wide_tiles(bool f32, std::initializer_list<int64_t> n) {
  for (int64_t c : n)
    if (f32 || c <= 128) return false;
  return true;
}

template <typename T, int PARTS, typename OUT>
cudaError_t dispatch(const GemmArgs& g, cudaStream_t s) {
  constexpr int kWide = PARTS == 3 ? 128 : 256;
  switch (g.mode) {
    case kGate: return launch<T, PARTS, OUT, kGate, kWide / 2, false>(g, s);
    case kHidden: return launch<T, PARTS, OUT, kHidden, PARTS == 3 ? 64 : 128, false>(g, s);
    case kLinear: {
      const int64_t n = g.b_mn ? g.b[0].cols : g.b[0].rows;
      if constexpr (PARTS == 3) {
        // 64 columns where tiles of 128 leave multiprocessors without one (5041 rows, width 100, fp32: dX 22.2 us)
        if (tiles_of(g.a[0].rows, 128) * tiles_of(n, 128) < sm_count())
          return g.b_mn ? launch<T, PARTS, OUT, kLinear, 64, true>(g, s) : launch<T, PARTS, OUT, kLinear, 64, false>(g, s);
      }
      const bool wide = wide_tiles(PARTS == 3, {n});
      if (g.b_mn) return wide ? launch<T, PARTS, OUT, kLinear, kWide, true>(g, s) : launch<T, PARTS, OUT, kLinear, 128, true>(g, s);
      return wide ? launch<T, PARTS, OUT, kLinear, kWide, false>(g, s) : launch<T, PARTS, OUT, kLinear, 128, false>(g, s);
    }
    default:
      return wide_tiles(PARTS == 3, {g.b[0].cols, g.b[1].cols, g.b[2].cols}) ? launch<T, PARTS, OUT, kWeight, kWide, true>(g, s)
                                                                            : launch<T, PARTS, OUT, kWeight, 128, true>(g, s);
  }
}

}  // namespace

cudaError_t gemm(const GemmArgs& g, cudaStream_t s) {
  if (g.a[0].planes == 3) return dispatch<__nv_bfloat16, 3, float>(g, s);
  return g.bf16 ? dispatch<__nv_bfloat16, 1, __nv_bfloat16>(g, s) : dispatch<__half, 1, __half>(g, s);
}

// The number of splits whose rounds of tiles over the SMs cost least, at least 256 rows a split.  A round costs its rows,
// and as much as kTail rows more for writing its sums and reading them again: 74 pairs' 256 x 256 are 19 MB, both ways
// 6 us, in which they do about 1000 rows (fp32, six products a row: 170).  16-bit types: no split is longer than a run of
// sums (fp32 adds up in registers).
int weight_splits(const int64_t* m, const int64_t* n, int64_t rows, bool f32, int sms) {
  const bool wide = wide_tiles(f32, {n[0], n[1], n[2]});
  const int cg = weight_pairs(f32, {m[0], m[1], m[2]}) ? 2 : 1;
  int64_t tiles = 0;
  for (int j = 0; j < 3; ++j) tiles += tiles_of(m[j], 128 * cg) * tiles_of(n[j], wide ? 256 : 128);
  sms /= cg;
  const float kTail = f32 ? 170.f : 1000.f;
  const int64_t run = (int64_t)kRunTiles * 128, least = f32 ? 1 : (rows + run - 1) / run, most = least > 16 ? 2 * least : 32;
  int best = (int)least;
  float cost = 1e30f;
  for (int s = best; s <= most && (s == least || rows / s >= 256); ++s) {
    const float c = (float)tiles_of(tiles * s, sms) * ((float)rows / s + kTail);
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return best;
}

}  // namespace ff
}  // namespace trifast
