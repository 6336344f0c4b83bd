// C ABI of the feed-forward block's operators (momijo_hip.h): the gated MLP, the
// norms around a residual sum, and dropout.  Arguments are checked here; scratch
// memory is the caller's, so every call can be captured into a HIP graph.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/momijo_hip.h"
#include "abi_util.h"
#include "launch.h"

namespace {

using namespace mj_abi;

int32_t check_act(int32_t act) {
  if (act == MJ_EPI_NONE || act == MJ_EPI_RELU || act == MJ_EPI_GELU_TANH || act == MJ_EPI_SILU)
    return MJ_OK;
  if (valid_epi(act))
    return fail(MJ_ERR_UNSUPPORTED, "gated MLP: activation %d has no gradient here (NONE, RELU, "
                "GELU_TANH and SILU do)", act);
  return fail(MJ_ERR_ARG, "unknown activation %d", act);
}

int32_t check_dtype(int32_t dtype) {
  if (dtype == MJ_F32 || dtype == MJ_BF16) return MJ_OK;
  return fail(MJ_ERR_ARG, "unknown element type %d", dtype);
}

int32_t check_mlp(int32_t act, int64_t M, int64_t K, int64_t I, int64_t H) {
  if (int32_t s = check_act(act)) return s;
  if (int32_t s = check_dims(M, K, I)) return s;
  return check_dims(M, H, I);
}

// What the tile kernels need of the bf16 block: 16-byte rows, 32-bit offsets
// within 256 rows of a tile and 32-bit row numbers.
int32_t check_mlp_bf16(const char *what, int64_t M, int64_t K, int64_t I, int64_t H,
                       const void *const *ptrs, int n) {
  if (K % 8 || I % 8 || H % 8)
    return fail(MJ_ERR_UNSUPPORTED, "%s: K, I and H must be multiples of 8 (%lld, %lld, %lld)", what,
                (long long)K, (long long)I, (long long)H);
  const int64_t lim = (int64_t)1 << 22;
  if (K >= lim || I >= lim || H >= lim)
    return fail(MJ_ERR_UNSUPPORTED, "%s: widths must be below 2^22", what);
  if (M > mj::kMlpMaxRows)
    return fail(MJ_ERR_UNSUPPORTED, "%s: at most %lld rows", what, (long long)mj::kMlpMaxRows);
  for (int i = 0; i < n; ++i)
    if (!aligned16(ptrs[i]))
      return fail(MJ_ERR_UNSUPPORTED, "%s: every array must be 16-byte aligned", what);
  return MJ_OK;
}

// The threshold and scale of a drop probability.
int32_t make_dropout(float p, uint64_t seed, uint64_t counter, const uint64_t *state,
                     mj::Dropout &d) {
  if (!(p >= 0.0f && p <= 1.0f)) return fail(MJ_ERR_ARG, "drop probability %g outside [0, 1]", p);
  d.seed = seed;
  d.counter = counter;
  d.state = state;
  if (p == 0.0f) {
    d.thr = 0;
    d.scale = 1.0f;
  } else if (p == 1.0f) {
    d.thr = 65536;
    d.scale = 0.0f;
  } else {
    const long t = std::lrint((double)p * 65536.0);
    d.thr = (uint32_t)(t < 1 ? 1 : t > 65535 ? 65535 : t);
    d.scale = (float)(65536.0 / (65536.0 - (double)d.thr));
  }
  return MJ_OK;
}

// K slices of an fp32 product (`pair`: of two of one shape in one launch): as many as
// bring its 64 x 64 tiles to four a CU with 512 k each at least.  y of 1024 x 1024 with
// K = 2752 61 us whole, 48 and 5 for the sum in four slices; dx, two such products,
// 147 us one after the other, 78 and 5 in one launch of two slices each.
int64_t f32_slices(int64_t M, int64_t N, int64_t K, int64_t pair) {
  const int64_t tiles = ((M + 63) / 64) * ((N + 63) / 64) * pair;
  int64_t s = 1;
  while (s < 4 && tiles * s * 2 <= 1024 && K % (2 * s) == 0 && K / (2 * s) >= 512) s *= 2;
  return s;
}

// Whether two products' results may be slices of one sum: they fill the chip only
// together (beyond, adding into the first's result moves fewer bytes).
bool f32_sums_pair(int64_t M, int64_t N) {
  return ((M + 63) / 64) * ((N + 63) / 64) * 2 <= 1024;
}

int64_t words_between(const void *a, const void *b) {
  return ((intptr_t)b - (intptr_t)a) / (intptr_t)sizeof(float);
}

// `pair` (1 or 2) products of one shape, each in `slices` along K, in one launch: C
// [pair][slices][M][N]; the second product's operands lie at A1, B1.
int32_t f32_products(int64_t pair, int64_t slices, int64_t M, int64_t N, int64_t K, const float *A,
                     const float *A1, int64_t sAm, int64_t sAk, const float *B, const float *B1,
                     int64_t sBk, int64_t sBn, float *C, hipStream_t st, const char *what) {
  mj::BatchDesc bd;
  bd.rank = 2;
  bd.shape[0] = pair, bd.shape[1] = slices;
  bd.a_stride[0] = pair > 1 ? words_between(A, A1) : 0;
  bd.b_stride[0] = pair > 1 ? words_between(B, B1) : 0;
  const int64_t k = K / slices;
  bd.a_stride[1] = k * sAk, bd.b_stride[1] = k * sBk;
  return hip_status(mj::launch_gemm_f32_batched(M, N, k, A, sAm, sAk, B, sBk, sBn, C, bd,
                                                pair * slices, st),
                    what);
}

// The shared arguments of the residual norm and its backward.
int32_t make_norm(mj::ResNorm &r, int32_t dtype, int32_t norm, const void *x, const void *b,
                  const void *gate, int64_t gate_rows, const float *scale, const float *wp,
                  const float *bp, const float *wn, const float *bn, float eps, float p,
                  uint64_t seed, uint64_t counter, const uint64_t *state, int64_t rows,
                  int64_t dim) {
  if (int32_t s = check_dtype(dtype)) return s;
  if (norm != MJ_NORM_RMS && norm != MJ_NORM_LAYER) return fail(MJ_ERR_ARG, "unknown norm %d", norm);
  if (int32_t s = check_dims(rows, dim, 0)) return s;
  if (dim > mj::kResNormMaxDim)
    return fail(MJ_ERR_UNSUPPORTED, "residual norm: width %lld above %lld", (long long)dim,
                (long long)mj::kResNormMaxDim);
  // (an empty array's pointer may be null)
  if (rows > 0 && dim > 0 && !x) return fail(MJ_ERR_ARG, "null x");
  if (rows > 0 && dim > 0 && !b && (gate || wp || p != 0.0f))
    return fail(MJ_ERR_ARG, "gate, post norm and dropout need a branch");
  if ((bp && !wp) || (bn && !wn)) return fail(MJ_ERR_ARG, "a norm's bias needs its weight");
  if (!(eps >= 0.0f)) return fail(MJ_ERR_ARG, "eps must not be negative");
  if (gate && (gate_rows < 1 || rows % gate_rows))
    return fail(MJ_ERR_SHAPE, "%lld gate rows do not divide %lld rows", (long long)gate_rows,
                (long long)rows);
  r.x = x, r.b = b, r.gate = gate, r.scale = scale;
  r.wp = wp, r.bp = bp, r.wn = wn, r.bn = bn;
  r.rows = rows, r.dim = dim;
  r.per = gate && rows > 0 ? rows / gate_rows : (rows > 0 ? rows : 1);
  r.eps = eps;
  r.layer = norm == MJ_NORM_LAYER;
  return make_dropout(p, seed, counter, state, r.drop);
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------ dropout
int32_t mj_dropout(int32_t dtype, const void *x, void *y, int64_t n, float p, uint64_t seed,
                   uint64_t counter, const uint64_t *state, void *stream) {
  if (int32_t s = check_dtype(dtype)) return s;
  if (n < 0) return fail(MJ_ERR_ARG, "negative size");
  mj::Dropout d;
  if (int32_t s = make_dropout(p, seed, counter, state, d)) return s;
  if (n == 0) return MJ_OK;
  if (!x || !y) return fail(MJ_ERR_ARG, "null operand");
  return hip_status(mj::launch_dropout(dtype == MJ_BF16, x, y, n, d, S(stream)), "dropout launch");
}

// ------------------------------------------------------------------ residual norm
int32_t mj_residual_norm(int32_t dtype, int32_t norm, const void *x, const void *b,
                         const void *gate, int64_t gate_rows, const float *scale, const float *wp,
                         const float *bp, const float *wn, const float *bn, float eps, float p,
                         uint64_t seed, uint64_t counter, const uint64_t *state, void *y, void *n,
                         float *stats, int64_t rows, int64_t dim, void *stream) {
  mj::ResNorm r;
  if (int32_t s = make_norm(r, dtype, norm, x, b, gate, gate_rows, scale, wp, bp, wn, bn, eps, p,
                            seed, counter, state, rows, dim))
    return s;
  if (rows == 0 || dim == 0) return MJ_OK;
  if (!y && !n) return fail(MJ_ERR_ARG, "no output");
  if ((n != nullptr) != (wn != nullptr)) return fail(MJ_ERR_ARG, "n and its weight go together");
  if (y == x && !b && !scale) {  // y is x: not written
    if (!n) return MJ_OK;
    y = nullptr;
  }
  r.y = y, r.n = n, r.stats = stats;
  return hip_status(mj::launch_residual_norm(dtype == MJ_BF16, r, S(stream)),
                    "residual norm launch");
}

int64_t mj_residual_norm_work_bytes(int64_t rows, int64_t dim, int64_t gate_rows) {
  if (rows <= 0 || dim <= 0 || gate_rows < 0 || (gate_rows > 0 && rows % gate_rows)) return 0;
  mj::ResNorm r;
  r.rows = rows, r.dim = dim;
  r.per = gate_rows > 0 ? rows / gate_rows : rows;
  int64_t most = 0;  // with biases or without
  for (int bias = 0; bias < 2; ++bias) {
    mj::ResNormGrad g;
    mj::plan_residual_norm_bwd(r, g, bias != 0);
    const int64_t n = mj::residual_norm_part_floats(r, g);
    most = n > most ? n : most;
  }
  return most * (int64_t)sizeof(float);
}

int32_t mj_residual_norm_backward(int32_t dtype, int32_t norm, const void *x, const void *b,
                                  const void *gate, int64_t gate_rows, const float *scale,
                                  const float *wp, const float *bp, const float *wn, float p,
                                  uint64_t seed, uint64_t counter, const uint64_t *state,
                                  const float *stats, const void *dy, const void *dn, void *dx,
                                  void *db, void *dgate, float *dscale, float *dwp, float *dbp,
                                  float *dwn, float *dbn, int64_t rows, int64_t dim, void *work,
                                  int64_t work_bytes, void *stream) {
  mj::ResNorm r;
  if (int32_t s = make_norm(r, dtype, norm, x, b, gate, gate_rows, scale, wp, bp, wn, nullptr, 0.0f,
                            p, seed, counter, state, rows, dim))
    return s;
  if (rows == 0 || dim == 0) return MJ_OK;
  if (!stats) return fail(MJ_ERR_ARG, "null stats");
  if (dn && !wn) return fail(MJ_ERR_ARG, "dn without the next norm's weight");
  if (!dy && !dn) return fail(MJ_ERR_ARG, "neither dy nor dn");
  if ((db || dwp || dbp) && !b) return fail(MJ_ERR_ARG, "gradients of an absent branch");
  if ((dwp || dbp) && !wp) return fail(MJ_ERR_ARG, "gradients of an absent post norm");
  if ((dwn || dbn) && !dn) return fail(MJ_ERR_ARG, "gradients of the next norm need dn");
  if (dgate && !gate) return fail(MJ_ERR_ARG, "the gradient of an absent gate");
  if (dscale && !scale) return fail(MJ_ERR_ARG, "the gradient of an absent scale");
  r.stats = const_cast<float *>(stats);
  mj::ResNormGrad g;
  g.dy = dy, g.dn = dn, g.dx = dx, g.db = db, g.dgate = dgate;
  g.dscale = dscale, g.dwp = dwp, g.dbp = dbp, g.dwn = dwn, g.dbn = dbn;
  mj::plan_residual_norm_bwd(r, g, mj::residual_norm_bias(r, g));
  const int64_t need = mj::residual_norm_part_floats(r, g) * (int64_t)sizeof(float);
  if (!work || work_bytes < need || !aligned16(work))
    return fail(MJ_ERR_ARG, "residual norm backward: work must be 16-byte aligned with %lld bytes",
                (long long)need);
  g.part = (float *)work;
  return hip_status(mj::launch_residual_norm_bwd(dtype == MJ_BF16, r, g, S(stream)),
                    "residual norm backward launch");
}

// ------------------------------------------------------------------ gated MLP
int64_t mj_gated_mlp_work_bytes(int64_t M, int64_t K, int64_t I, int64_t H, int32_t backward) {
  // the sliced product's own sizes alone (y [M, H] or dx [M, K], sums over I): it is planned and
  // launched whether or not the width that it does not have is zero
  if (M <= 0 || I <= 0 || (backward ? K : H) <= 0) return 0;
  return mj::gated_mlp_part_floats(M, K, I, H, backward != 0) * (int64_t)sizeof(float);
}

const char *mj_gated_mlp_kernel(int64_t M, int64_t K, int64_t I, int64_t H, int32_t product) {
  const void *none = nullptr;
  if (M <= 0 || K <= 0 || I <= 0 || H <= 0 || product < 0 || product > 4 ||
      check_mlp(MJ_EPI_NONE, M, K, I, H) || check_mlp_bf16("gated MLP", M, K, I, H, &none, 1))
    return "";
  return mj::gated_mlp_kernel_name(M, K, I, H, product);
}

int32_t mj_copy_rows_bf16(int32_t n, const uint16_t *const *src, uint16_t *const *dst,
                          const int64_t *sizes, void *stream) {
  if (n < 1 || n > 4) return fail(MJ_ERR_ARG, "1 to 4 matrices, got %d", n);
  if (!src || !dst || !sizes) return fail(MJ_ERR_ARG, "null argument");
  mj::CopyRows c;
  c.n = n;
  for (int i = 0; i < n; ++i) {
    const int64_t *z = sizes + 6 * i;
    mj::CopyRows::Mat &m = c.m[i];
    m.src = src[i], m.dst = dst[i];
    m.rows = z[0], m.cols = z[1], m.src_ld = z[2];
    m.dst_rows = z[3], m.dst_cols = z[4], m.dst_ld = z[5];
    for (int k = 0; k < 6; ++k)
      if (z[k] < 0) return fail(MJ_ERR_ARG, "negative size");
    if (m.src_ld < m.cols || m.dst_ld < m.dst_cols)
      return fail(MJ_ERR_SHAPE, "rows overlap (leading dimension below the width)");
    if ((m.dst_rows > 0 && m.dst_cols > 0 && !m.dst) || (m.rows > 0 && m.cols > 0 && !m.src))
      return fail(MJ_ERR_ARG, "null matrix");
  }
  return hip_status(mj::launch_copy_rows_bf16(c, S(stream)), "row copy launch");
}

int32_t mj_gated_mlp_bf16(const uint16_t *x, const uint16_t *Wg, const uint16_t *Wu,
                          const uint16_t *Wd, int32_t act, uint16_t *h, float *g, float *u,
                          uint16_t *y, int64_t M, int64_t K, int64_t I, int64_t H, void *work,
                          int64_t work_bytes, void *stream) {
  if (int32_t s = check_mlp(act, M, K, I, H)) return s;
  const void *ptrs[] = {x, Wg, Wu, Wd, h, g, u, y, work};
  if (int32_t s = check_mlp_bf16("gated MLP", M, K, I, H, ptrs, 9)) return s;
  if (M == 0) return MJ_OK;
  if ((H > 0 && !y) || (I > 0 && (!h || (H > 0 && !Wd) || (K > 0 && (!x || !Wg || !Wu)))))
    return fail(MJ_ERR_ARG, "null operand");
  if ((g == nullptr) != (u == nullptr)) return fail(MJ_ERR_ARG, "g and u are kept together");
  const int64_t need = mj_gated_mlp_work_bytes(M, K, I, H, 0);
  if (need > 0 && (!work || work_bytes < need))
    return fail(MJ_ERR_ARG, "gated MLP: work must hold %lld bytes", (long long)need);
  mj::GatedMlp q;
  q.x = x, q.wg = Wg, q.wu = Wu, q.wd = Wd, q.act = act;
  q.h = h, q.g = g, q.u = u, q.y = y;
  q.M = M, q.K = K, q.I = I, q.H = H, q.part = (float *)work;
  return hip_status(mj::launch_gated_mlp(q, S(stream)), "gated MLP launch");
}

int32_t mj_gated_mlp_backward_bf16(const uint16_t *x, const uint16_t *Wg, const uint16_t *Wu,
                                   const uint16_t *Wd, int32_t act, const uint16_t *h,
                                   const float *g, const float *u, const uint16_t *dy,
                                   uint16_t *dg, uint16_t *du, uint16_t *dx, uint16_t *dWg,
                                   uint16_t *dWu, uint16_t *dWd, int64_t M, int64_t K, int64_t I,
                                   int64_t H, void *work, int64_t work_bytes, void *stream) {
  if (int32_t s = check_mlp(act, M, K, I, H)) return s;
  const void *ptrs[] = {x, Wg, Wu, Wd, h, g, u, dy, dg, du, dx, dWg, dWu, dWd, work};
  if (int32_t s = check_mlp_bf16("gated MLP backward", M, K, I, H, ptrs, 15)) return s;
  if (M > 0 && I > 0 && (dx || dWg || dWu) &&
      (!dg || !du || !g || !u || (H > 0 && (!dy || !Wd))))
    return fail(MJ_ERR_ARG, "null operand");
  if (M > 0 && I > 0 && K > 0 && dx && (!Wg || !Wu)) return fail(MJ_ERR_ARG, "null weights");
  if (M > 0 && I > 0 && K > 0 && (dWg || dWu) && !x) return fail(MJ_ERR_ARG, "null x");
  if (M > 0 && I > 0 && H > 0 && dWd && (!dy || !h)) return fail(MJ_ERR_ARG, "null dy or h");
  const int64_t need = dx ? mj_gated_mlp_work_bytes(M, K, I, H, 1) : 0;
  if (need > 0 && (!work || work_bytes < need))
    return fail(MJ_ERR_ARG, "gated MLP backward: work must hold %lld bytes", (long long)need);
  mj::GatedMlp q;
  q.x = x, q.wg = Wg, q.wu = Wu, q.wd = Wd, q.act = act;
  q.h = const_cast<uint16_t *>(h), q.g = const_cast<float *>(g), q.u = const_cast<float *>(u);
  q.M = M, q.K = K, q.I = I, q.H = H, q.part = (float *)work;
  mj::GatedMlpGrad o;
  o.dy = dy, o.dg = dg, o.du = du, o.dx = dx, o.dwg = dWg, o.dwu = dWu, o.dwd = dWd;
  return hip_status(mj::launch_gated_mlp_bwd(q, o, S(stream)), "gated MLP backward launch");
}

int64_t mj_gated_mlp_f32_work_bytes(int64_t M, int64_t K, int64_t I, int64_t H, int32_t backward) {
  if (M <= 0 || K <= 0 || I <= 0 || H <= 0) return 0;
  const int64_t N = backward ? K : H, n = f32_slices(M, N, I, backward ? 2 : 1) * (backward ? 2 : 1);
  return n == 1 || (backward && !f32_sums_pair(M, N)) ? 0 : n * M * N * (int64_t)sizeof(float);
}

int32_t mj_gated_mlp_f32(const float *x, const float *Wg, const float *Wu, const float *Wd,
                         int32_t act, float *h, float *g, float *u, float *y, int64_t M, int64_t K,
                         int64_t I, int64_t H, void *work, int64_t work_bytes, void *stream) {
  if (int32_t s = check_mlp(act, M, K, I, H)) return s;
  if (M == 0) return MJ_OK;
  if ((H > 0 && !y) || (I > 0 && (!h || !g || !u || (H > 0 && !Wd) || (K > 0 && (!x || !Wg || !Wu)))))
    return fail(MJ_ERR_ARG, "null operand");
  const void *el[] = {h, g, u, y, work};
  for (const void *e : el)
    if (!aligned16(e))
      return fail(MJ_ERR_UNSUPPORTED, "gated MLP: h, g, u, y and work must be 16-byte aligned");
  const int64_t need = mj_gated_mlp_f32_work_bytes(M, K, I, H, 0);
  if (need > 0 && (!work || work_bytes < need))
    return fail(MJ_ERR_ARG, "gated MLP: work must hold %lld bytes", (long long)need);
  const hipStream_t st = S(stream);
  if (I > 0) {
    // both projections in one launch where u follows g
    if (K > 0 && u == g + M * I) {
      if (int32_t e = f32_products(2, 1, M, I, K, x, x, K, 1, Wg, Wu, 1, K, g, st, "gate and up launch"))
        return e;
    } else {
      if (int32_t e = mj_linear_f32(x, Wg, nullptr, MJ_EPI_NONE, g, M, K, I, stream)) return e;
      if (int32_t e = mj_linear_f32(x, Wu, nullptr, MJ_EPI_NONE, u, M, K, I, stream)) return e;
    }
    if (int32_t e = hip_status(mj::launch_gate_f32(act, g, u, h, M * I, st), "gate launch")) return e;
  }
  if (need == 0) return mj_linear_f32(h, Wd, nullptr, MJ_EPI_NONE, y, M, I, H, stream);
  const int64_t s = f32_slices(M, H, I, 1);
  if (int32_t e = f32_products(1, s, M, H, I, h, h, I, 1, Wd, Wd, 1, I, (float *)work, st, "y launch"))
    return e;
  return hip_status(mj::launch_sum_f32((const float *)work, y, M * H, s, st), "y sum launch");
}

int32_t mj_gated_mlp_backward_f32(const float *x, const float *Wg, const float *Wu, const float *Wd,
                                  int32_t act, const float *h, const float *g, const float *u,
                                  const float *dy, float *dg, float *du, float *dx, float *dWg,
                                  float *dWu, float *dWd, int64_t M, int64_t K, int64_t I,
                                  int64_t H, void *work, int64_t work_bytes, void *stream) {
  if (int32_t s = check_mlp(act, M, K, I, H)) return s;
  const bool inner = M > 0 && I > 0 && (dx || dWg || dWu);
  if (inner && (!dg || !du || !g || !u || (H > 0 && (!dy || !Wd))))
    return fail(MJ_ERR_ARG, "null operand");
  if (M > 0 && I > 0 && K > 0 && dx && (!Wg || !Wu)) return fail(MJ_ERR_ARG, "null weights");
  if (M > 0 && I > 0 && K > 0 && (dWg || dWu) && !x) return fail(MJ_ERR_ARG, "null x");
  if (M > 0 && I > 0 && H > 0 && dWd && (!dy || !h)) return fail(MJ_ERR_ARG, "null dy or h");
  const void *el[] = {g, u, dg, du, dx, work};
  for (const void *e : el)
    if (!aligned16(e))
      return fail(MJ_ERR_UNSUPPORTED, "gated MLP: g, u, dg, du, dx and work must be 16-byte aligned");
  const int64_t need = dx ? mj_gated_mlp_f32_work_bytes(M, K, I, H, 1) : 0;
  if (need > 0 && (!work || work_bytes < need))
    return fail(MJ_ERR_ARG, "gated MLP backward: work must hold %lld bytes", (long long)need);
  const hipStream_t st = S(stream);
  // dh = dy Wd into dg, which the elementwise step then overwrites in place
  if (inner) {
    if (int32_t e = mj_matmul_f32(M, I, H, dy, H, 1, Wd, I, 1, nullptr, MJ_EPI_NONE, dg, I, stream))
      return e;
    if (int32_t e = hip_status(mj::launch_gate_bwd_f32(act, g, u, dg, dg, du, M * I, st),
                               "gate backward launch"))
      return e;
  }
  if (dx && M > 0 && K > 0) {
    if (need > 0) {
      const int64_t s = f32_slices(M, K, I, 2);
      if (int32_t e = f32_products(2, s, M, K, I, dg, du, I, 1, Wg, Wu, K, 1, (float *)work, st,
                                   "dx launch"))
        return e;
      if (int32_t e = hip_status(mj::launch_sum_f32((const float *)work, dx, M * K, 2 * s, st),
                                 "dx sum launch"))
        return e;
    } else {
      if (int32_t e = mj_matmul_f32(M, K, I, dg, I, 1, Wg, K, 1, nullptr, MJ_EPI_NONE, dx, K, stream))
        return e;
      if (int32_t e = hip_status(mj::launch_gemm_f32_accum(M, K, I, du, I, 1, Wu, K, 1, dx, K, 1, st),
                                 "dx launch"))
        return e;
    }
  }
  // dW = d^T x: the transposes are strides; both projections' in one launch where dWu
  // follows dWg
  if (dWg && dWu == dWg + I * K && M > 0 && I > 0 && K > 0) {
    if (int32_t e = f32_products(2, 1, I, K, M, dg, du, 1, I, x, x, K, 1, dWg, st, "dW launch"))
      return e;
  } else {
    if (dWg)
      if (int32_t e = mj_matmul_f32(I, K, M, dg, 1, I, x, K, 1, nullptr, MJ_EPI_NONE, dWg, K, stream))
        return e;
    if (dWu)
      if (int32_t e = mj_matmul_f32(I, K, M, du, 1, I, x, K, 1, nullptr, MJ_EPI_NONE, dWu, K, stream))
        return e;
  }
  if (dWd)
    if (int32_t e = mj_matmul_f32(H, I, M, dy, 1, H, h, I, 1, nullptr, MJ_EPI_NONE, dWd, I, stream))
      return e;
  return MJ_OK;
}

}  // extern "C"
