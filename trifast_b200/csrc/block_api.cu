// C ABI of the operators around the attention: argument checks, workspaces and the order of launches.
// Declared and documented in include/trifast_b200.h.

#include <math.h>

#include <initializer_list>

#include "block_kernels.h"
#include "ff_fused.cuh"
#include "kernels.h"

namespace trifast {
namespace {

constexpr int64_t kMostRows = (int64_t)1 << 40;

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool known_dtype(int d) { return d >= TRIFAST_F32 && d <= TRIFAST_F16; }
size_t elem(int dtype) { return dtype == TRIFAST_F32 ? 4 : 2; }

int check_pointers(std::initializer_list<const void*> required, std::initializer_list<const void*> optional) {
  for (const void* p : required) {
    if (!p) return TRIFAST_ERR_NULL;
    if (!aligned(p, 16)) return TRIFAST_ERR_ALIGN;
  }
  for (const void* p : optional)
    if (!aligned(p, 16)) return TRIFAST_ERR_ALIGN;
  return TRIFAST_OK;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  if (need == 0) return TRIFAST_OK;
  if (!ws || have < need) return TRIFAST_ERR_WORKSPACE;
  return aligned(ws, 256) ? TRIFAST_OK : TRIFAST_ERR_ALIGN;
}

// ------------------------------------------------------------------ layer norm
int check_norm(const trifast_norm* n, bool backward) {
  if (!n) return TRIFAST_ERR_NULL;
  if (n->rows < 0 || n->rows > kMostRows || n->width < 1 || n->width > 1 << 20) return TRIFAST_ERR_SHAPE;
  if (!known_dtype(n->dtype) || (n->affine_dtype != n->dtype && n->affine_dtype != TRIFAST_F32)) return TRIFAST_ERR_DTYPE;
  if (!(n->eps >= 0.f) || !isfinite(n->eps)) return TRIFAST_ERR_SHAPE;
  for (int64_t ld : {n->ld_x, backward ? n->ld_dy : n->ld_x})
    if (ld < n->width || (n->rows > 1 && !layer_norm_rows_fit(ld, n->width, n->dtype))) return TRIFAST_ERR_STRIDE;
  // (rows longer than a block's registers: their gradients' sums take 64 to a block along the grid's second dimension, and no
  // forward pass is taken whose backward would not be)
  if (layer_norm_in_passes(n->width, n->dtype) && n->rows > (int64_t)65535 * 64) return TRIFAST_ERR_TOO_LARGE;
  return TRIFAST_OK;
}

LayerNormArgs norm_args(const trifast_norm* n) {
  LayerNormArgs a = {};
  a.rows = n->rows;
  a.ld_x = n->ld_x;
  a.ld_dy = n->ld_dy;
  a.width = n->width;
  a.dtype = n->dtype;
  a.affine_dtype = n->affine_dtype;
  a.eps = n->eps;
  return a;
}

// ------------------------------------------------------------------ feed-forward
using ff::Matrix;

int check_ff(const trifast_ff* f, bool backward) {
  if (!f) return TRIFAST_ERR_NULL;
  if (f->rows < 0 || f->rows > kMostRows) return TRIFAST_ERR_SHAPE;
  for (int w : {f->width, f->hidden, f->width_out})
    if (w < 1 || w > 65536) return TRIFAST_ERR_SHAPE;
  if (!known_dtype(f->dtype)) return TRIFAST_ERR_DTYPE;
  if (f->ld_x < f->width || (backward && f->ld_dy < f->width_out)) return TRIFAST_ERR_STRIDE;
  return TRIFAST_OK;
}

int64_t round_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// Rows are worked on in chunks, whose hidden values (and, backward, their gradients) and operands laid out anew lie in the
// workspace, of at most this many bytes whatever the number of rows, but of 1024 rows at least (hidden 65536, backward: 403 MB in
// 16 bits, 1.2 GB in fp32).  (48 MB, which stay in L2 from one kernel to the next, lost more to the
// last rounds of tiles than they saved: 65,536 rows, width 512, hidden 1024 forward 198 us in three chunks.)
constexpr int64_t kChunkBytes = 256 << 20;

// The workspace of a call, carved in the order of the members.
struct FfPlan {
  bool few;                                // by the CUDA cores
  bool fused;                              // by the kernels that keep the hidden values on chip
  int planes;
  int64_t pitch_c, pitch_h, pitch_o;       // rows of staged operands and hidden values
  bool stage_c, stage_h, stage_x, stage_dy;  // the operands of that width have to be laid out anew
  int64_t chunk;                           // rows
  int splits;
  int64_t partial_stride;                  // floats
  size_t wg, wu, wd, x, dy, h, da, db, partials, total;
};

// Where the fused kernels run, of those calls that they can take: they walk the hidden units one chunk of 64 after the
// other, a tile of 128 rows to a multiprocessor, and are one kernel where the products are two or three.  Up to 512
// units that is faster for any number of rows (512 rows, width 128, hidden 512: 11.4 against 12.7 us forward, 13.9 against
// 15.7 for dX; hidden 256: 8.7 against 11.7 and 10.2 against 14.2), beyond, where there are tiles for half of the
// multiprocessors.
constexpr int kFusedHidden = 512;
constexpr int64_t kFusedRows = 148 / 2 * 128;

FfPlan plan_ff(const trifast_ff* f, bool backward, bool weights) {
  FfPlan p = {};
  const bool f32 = f->dtype == TRIFAST_F32;
  p.fused = !f32 && f->width <= ff::kFusedWidth && f->width_out <= ff::kFusedWidth && (f->hidden <= kFusedHidden || f->rows >= kFusedRows);
  p.pitch_h = round_up(f->hidden, 8);
  p.few = !backward && f->rows <= ff::kFewRows;
  if (p.few) {
    if (!ff::few_rows_in_cluster(f->rows, f->width, f->hidden, f->width_out, (int)elem(f->dtype)))
      p.total = (size_t)round_up(f->rows * p.pitch_h * 4, 256);
    return p;
  }
  p.planes = f32 ? 3 : 1;
  p.pitch_c = round_up(f->width, 8);
  p.pitch_o = round_up(f->width_out, 8);
  p.stage_c = f32 || f->width % 8;    // w_gate, w_up
  p.stage_h = f32 || f->hidden % 8;   // w_down
  p.stage_x = f32 || (f->rows > 1 && f->ld_x % 8);
  p.stage_dy = f32 || (f->rows > 1 && f->ld_dy % 8);
  const int64_t one = 2 * p.planes;
  int64_t per_row = p.fused ? 0 : p.pitch_h * one * (backward ? 3 : 1);
  if (p.stage_x) per_row += p.pitch_c * one;
  if (backward && p.stage_dy) per_row += p.pitch_o * one;
  int64_t most = per_row ? kChunkBytes / per_row / 128 * 128 : (int64_t)1 << 30;
  if (most < 1024) most = 1024;
  const int64_t chunks = (f->rows + most - 1) / most;
  p.chunk = chunks <= 1 ? round_up(f->rows, 128) : round_up((f->rows + chunks - 1) / chunks, 128);
  size_t off = 0;
  auto take = [&](bool wanted, int64_t bytes) {
    const size_t at = off;
    if (wanted) off += (size_t)round_up(bytes, 256);
    return at;
  };
  p.wg = take(p.stage_c, f->hidden * p.pitch_c * one);
  p.wu = take(p.stage_c, f->hidden * p.pitch_c * one);
  p.wd = take(p.stage_h, f->width_out * p.pitch_h * one);
  p.x = take(p.stage_x, p.chunk * p.pitch_c * one);
  p.dy = take(backward && p.stage_dy, p.chunk * p.pitch_o * one);
  p.h = take(!p.fused, p.chunk * p.pitch_h * one);
  p.da = take(backward && !p.fused, p.chunk * p.pitch_h * one);
  p.db = take(backward && !p.fused, p.chunk * p.pitch_h * one);
  if (backward && weights) {
    const int64_t m[3] = {f->hidden, f->hidden, f->width_out}, n[3] = {f->width, f->width, f->hidden};
    // (the plan is the same on every device: 148 multiprocessors)
    const int64_t rows = f->rows < p.chunk ? f->rows : p.chunk;
    p.splits = p.fused ? ff::fused_weight_splits(rows, f->hidden, 148) : ff::weight_splits(m, n, rows, f32, 148);
    p.partial_stride = 2 * f->hidden * ff::partial_pitch(f->width) + f->width_out * ff::partial_pitch(f->hidden);
    p.partials = take(true, p.splits * p.partial_stride * 4);
  }
  p.total = off;
  return p;
}

struct FfWeights {
  Matrix gate, up, down;
};

// Operands as the products read them: as they lie, or laid out anew by one kernel for all of a call's (the weights, then
// the rows of each chunk).
struct FfStage {
  const trifast_ff* f;
  const FfPlan* p;
  char* ws;
  ff::StageJob jobs[ff::kStageJobs];
  int count = 0;

  Matrix matrix(bool staged, const void* src, int64_t ld, int64_t rows, int64_t cols, int64_t pitch, int64_t padded, size_t off) {
    if (!staged) return Matrix{const_cast<void*>(src), rows, cols, ld, 1, rows * ld};
    const Matrix m{ws + off, rows, cols, pitch, p->planes, padded * pitch};
    jobs[count++] = {src, ld, rows, m};
    return m;
  }
  FfWeights weights(const void* wg, const void* wu, const void* wd) {
    const trifast_ff& s = *f;
    return {matrix(p->stage_c, wg, s.width, s.hidden, s.width, p->pitch_c, s.hidden, p->wg),
            matrix(p->stage_c, wu, s.width, s.hidden, s.width, p->pitch_c, s.hidden, p->wu),
            matrix(p->stage_h, wd, s.hidden, s.width_out, s.hidden, p->pitch_h, s.width_out, p->wd)};
  }
  // Rows [r0, r0 + rows) of x or dy.
  Matrix rows(bool staged, const void* src, int64_t ld, int64_t r0, int64_t rows, int64_t cols, int64_t pitch, size_t off) {
    return matrix(staged, reinterpret_cast<const char*>(src) + (size_t)r0 * ld * elem(f->dtype), ld, rows, cols, pitch, p->chunk, off);
  }
  int run(cudaStream_t s) {
    const int n = count;
    count = 0;
    return cuda_rc(ff::stage(jobs, n, f->dtype, s));
  }
};

ff::FusedArgs fused_args(const trifast_ff* f, const FfWeights& w, const Matrix& x, unsigned int* status) {
  ff::FusedArgs g = {};
  g.bf16 = f->dtype != TRIFAST_F16;
  g.x = x;
  g.wg = w.gate;
  g.wu = w.up;
  g.wd = w.down;
  g.status = status;
  return g;
}

// Rows [r0, r0 + rows) of y or dx, and whether TMA can write them.
Matrix ff_result(const trifast_ff* f, void* dst, int64_t r0, int64_t rows, int64_t cols, bool* tma) {
  char* y = reinterpret_cast<char*>(dst) + (size_t)r0 * cols * elem(f->dtype);
  *tma = f->dtype != TRIFAST_F32 && (cols % 8 == 0 || rows == 1) && aligned(y, 16);
  return Matrix{y, rows, cols, cols, 1, rows * cols};
}

}  // namespace
}  // namespace trifast

using namespace trifast;

extern "C" {

size_t trifast_layer_norm_workspace_bytes(const trifast_norm* norm) {
  if (check_norm(norm, false)) return 0;
  return (size_t)layer_norm_workspace_floats(norm->rows, norm->width, norm->dtype) * sizeof(float);
}

int trifast_layer_norm(const trifast_norm* norm, const void* x, const void* weight, const void* bias, void* y, void* stream) {
  int rc = check_norm(norm, false);
  if (rc) return rc;
  if (norm->rows == 0) return TRIFAST_OK;
  unsigned int* status;
  if ((rc = check_pointers({x, y}, {weight, bias})) || (rc = device_status(&status))) return rc;
  LayerNormArgs a = norm_args(norm);
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.y = y;
  return cuda_rc(layer_norm_forward(a, (cudaStream_t)stream));
}

int trifast_layer_norm_backward(const trifast_norm* norm, const void* dy, const void* x, const void* weight, void* dx,
                                void* dweight, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_norm(norm, true);
  if (rc) return rc;
  const bool affine = dweight || dbias;
  cudaStream_t s = (cudaStream_t)stream;
  unsigned int* status;
  if (norm->rows == 0) {
    const size_t bytes = norm->width * elem(norm->affine_dtype);
    if (dweight && (rc = cuda_rc(cudaMemsetAsync(dweight, 0, bytes, s)))) return rc;
    return dbias ? cuda_rc(cudaMemsetAsync(dbias, 0, bytes, s)) : TRIFAST_OK;
  }
  if ((rc = check_pointers({dy, x}, {weight, dx, dweight, dbias})) ||
      (rc = check_workspace(workspace, workspace_bytes, affine ? trifast_layer_norm_workspace_bytes(norm) : 0)) ||
      (rc = device_status(&status)))
    return rc;
  if (!dx && !affine) return TRIFAST_OK;
  LayerNormArgs a = norm_args(norm);
  a.x = x;
  a.dy = dy;
  a.weight = weight;
  a.dx = dx;
  a.dweight = dweight;
  a.dbias = dbias;
  a.partials = affine ? (float*)workspace : nullptr;
  return cuda_rc(layer_norm_backward(a, s));
}

size_t trifast_feed_forward_workspace_bytes(const trifast_ff* f) {
  if (check_ff(f, false)) return 0;
  return plan_ff(f, false, false).total;
}

size_t trifast_feed_forward_backward_workspace_bytes(const trifast_ff* f) {
  if (check_ff(f, true)) return 0;
  return plan_ff(f, true, true).total;
}

int trifast_feed_forward(const trifast_ff* f, const void* x, const void* w_gate, const void* w_up, const void* w_down, void* y,
                         void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_ff(f, false);
  if (rc) return rc;
  if (f->rows == 0) return TRIFAST_OK;
  const FfPlan p = plan_ff(f, false, false);
  unsigned int* status;
  if ((rc = check_pointers({x, w_gate, w_up, w_down, y}, {})) || (rc = check_workspace(workspace, workspace_bytes, p.total)) ||
      (rc = device_status(&status)))
    return rc;
  char* ws = (char*)workspace;
  cudaStream_t s = (cudaStream_t)stream;
  if (p.few)
    return cuda_rc(ff::few_rows({x, w_gate, w_up, w_down, y, (float*)ws, f->ld_x, (int)f->rows, f->width, f->hidden, f->width_out,
                                 (int)p.pitch_h, f->dtype}, s));
  FfStage stage{f, &p, ws};
  const FfWeights w = stage.weights(w_gate, w_up, w_down);
  for (int64_t r0 = 0; r0 < f->rows; r0 += p.chunk) {
    const int64_t rows = f->rows - r0 < p.chunk ? f->rows - r0 : p.chunk;
    const Matrix mx = stage.rows(p.stage_x, x, f->ld_x, r0, rows, f->width, p.pitch_c, p.x);
    if ((rc = stage.run(s))) return rc;
    if (p.fused) {
      ff::FusedArgs g = fused_args(f, w, mx, status);
      g.what = ff::kForward;
      g.out = ff_result(f, y, r0, rows, f->width_out, &g.y_tma);
      if ((rc = cuda_rc(ff::fused(g, s)))) return rc;
      continue;
    }
    const Matrix mh{ws + p.h, rows, f->hidden, p.pitch_h, p.planes, p.chunk * p.pitch_h};
    ff::GemmArgs g = {};
    g.mode = ff::kGate;
    g.bf16 = f->dtype != TRIFAST_F16;
    g.a[0] = mx;
    g.b[0] = w.gate;
    g.b[1] = w.up;
    g.out[0] = mh;
    g.status = status;
    if ((rc = cuda_rc(ff::gemm(g, s)))) return rc;
    g.mode = ff::kLinear;
    g.products = 1;
    g.a[0] = mh;
    g.b[0] = w.down;
    g.out[0] = ff_result(f, y, r0, rows, f->width_out, &g.y_tma);
    if ((rc = cuda_rc(ff::gemm(g, s)))) return rc;
  }
  return TRIFAST_OK;
}

int trifast_feed_forward_backward(const trifast_ff* f, const void* dy, const void* x, const void* w_gate, const void* w_up,
                                  const void* w_down, void* dx, void* dw_gate, void* dw_up, void* dw_down, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  int rc = check_ff(f, true);
  if (rc) return rc;
  const bool weights = dw_gate || dw_up || dw_down;
  if (weights && !(dw_gate && dw_up && dw_down)) return TRIFAST_ERR_NULL;
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t count_in = (int64_t)f->hidden * f->width, count_out = (int64_t)f->hidden * f->width_out;
  if (f->rows == 0) {
    if (!weights) return TRIFAST_OK;
    const size_t es = elem(f->dtype);
    if ((rc = cuda_rc(cudaMemsetAsync(dw_gate, 0, count_in * es, s))) || (rc = cuda_rc(cudaMemsetAsync(dw_up, 0, count_in * es, s))))
      return rc;
    return cuda_rc(cudaMemsetAsync(dw_down, 0, count_out * es, s));
  }
  const FfPlan p = plan_ff(f, true, weights);
  unsigned int* status;
  if ((rc = check_pointers({dy, x, w_gate, w_up, w_down}, {dx, dw_gate, dw_up, dw_down})) ||
      (rc = check_workspace(workspace, workspace_bytes, p.total)) || (rc = device_status(&status)))
    return rc;
  if (!dx && !weights) return TRIFAST_OK;
  char* ws = (char*)workspace;
  FfStage stage{f, &p, ws};
  const FfWeights w = stage.weights(w_gate, w_up, w_down);
  float* partials = (float*)(ws + p.partials);
  for (int64_t r0 = 0; r0 < f->rows; r0 += p.chunk) {
    const int64_t rows = f->rows - r0 < p.chunk ? f->rows - r0 : p.chunk;
    const Matrix mx = stage.rows(p.stage_x, x, f->ld_x, r0, rows, f->width, p.pitch_c, p.x);
    const Matrix mdy = stage.rows(p.stage_dy, dy, f->ld_dy, r0, rows, f->width_out, p.pitch_o, p.dy);
    if ((rc = stage.run(s))) return rc;
    if (p.fused) {
      ff::FusedArgs g = fused_args(f, w, mx, status);
      g.dy = mdy;
      if (dx) {
        g.what = ff::kDx;
        g.out = ff_result(f, dx, r0, rows, f->width, &g.y_tma);
        if ((rc = cuda_rc(ff::fused(g, s)))) return rc;
      }
      if (weights) {
        g.what = ff::kDw;
        g.partials = partials;
        g.partial_stride = p.partial_stride;
        g.splits = p.splits;
        g.add = r0 > 0;
        if ((rc = cuda_rc(ff::fused(g, s)))) return rc;
      }
      continue;
    }
    auto hidden = [&](size_t off) { return Matrix{ws + off, rows, f->hidden, p.pitch_h, p.planes, p.chunk * p.pitch_h}; };
    const Matrix mda = hidden(p.da), mdb = hidden(p.db), mh = hidden(p.h);
    ff::GemmArgs g = {};
    g.bf16 = f->dtype != TRIFAST_F16;
    g.status = status;
    g.mode = ff::kHidden;
    g.a[0] = mdy;
    g.a[1] = mx;
    g.b[0] = w.gate;
    g.b[1] = w.up;
    g.b[2] = w.down;
    g.out[0] = mda;
    g.out[1] = mdb;
    g.out[2] = mh;
    if ((rc = cuda_rc(ff::gemm(g, s)))) return rc;
    if (dx) {
      g.mode = ff::kLinear;
      g.b_mn = true;
      g.products = 2;
      g.a[0] = mda;
      g.a[1] = mdb;
      g.out[0] = ff_result(f, dx, r0, rows, f->width, &g.y_tma);
      if ((rc = cuda_rc(ff::gemm(g, s)))) return rc;
    }
    if (weights) {
      g.mode = ff::kWeight;
      g.a[0] = mda;
      g.a[1] = mdb;
      g.a[2] = mdy;
      g.b[0] = mx;
      g.b[1] = mx;
      g.b[2] = mh;
      g.partials = partials;
      g.partial_stride = p.partial_stride;
      g.splits = p.splits;
      g.add = r0 > 0;
      if ((rc = cuda_rc(ff::gemm(g, s)))) return rc;
    }
  }
  if (!weights) return TRIFAST_OK;
  return cuda_rc(ff::sum_partials(partials, p.splits, p.partial_stride, {dw_gate, dw_up, dw_down}, {f->hidden, f->hidden, f->width_out},
                                  {f->width, f->width, f->hidden}, f->dtype, s));
}

int trifast_dropout_add(const trifast_dropout* d, const int64_t* seed_device, const void* x, const void* residual, void* y,
                        void* stream) {
  if (!d) return TRIFAST_ERR_NULL;
  if (d->outer < 0 || d->mid < 0 || d->inner < 0 || !(d->p >= 0.0 && d->p <= 1.0)) return TRIFAST_ERR_SHAPE;
  if (!known_dtype(d->dtype)) return TRIFAST_ERR_DTYPE;
  if (d->outer == 0 || d->mid == 0 || d->inner == 0) return TRIFAST_OK;
  if (d->outer > kMostRows / d->mid || d->outer * d->mid > kMostRows / d->inner) return TRIFAST_ERR_SHAPE;
  unsigned int* status;
  int rc;
  if ((rc = check_pointers({x, y}, {residual}))) return rc;
  if (!aligned(seed_device, 8)) return TRIFAST_ERR_ALIGN;
  if ((rc = device_status(&status))) return rc;
  DropoutArgs a = {};
  a.x = x;
  a.residual = residual;
  a.y = y;
  a.outer = d->outer;
  a.mid = d->mid;
  a.inner = d->inner;
  a.dtype = d->dtype;
  a.threshold = (uint64_t)nearbyint(d->p * 4294967296.0);
  a.scale = d->p < 1.0 ? (float)(1.0 / (1.0 - d->p)) : 0.f;
  a.seed = d->seed;
  a.offset = d->offset;
  a.seed_ptr = seed_device;
  return cuda_rc(dropout_add(a, (cudaStream_t)stream));
}

}  // extern "C"
