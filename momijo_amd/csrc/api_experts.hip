// C ABI of the mixture of experts and of the 8-bit floating point products
// (momijo_hip.h).  Arguments are checked here; scratch memory is the caller's, so every
// call can be captured into a HIP graph.
#include <hip/hip_runtime.h>

#include "../../include/momijo_hip.h"
#include "abi_util.h"
#include "launch.h"

namespace {

using namespace mj_abi;

int32_t check_dtype(int32_t dtype) {
  if (dtype == MJ_F32 || dtype == MJ_BF16) return MJ_OK;
  return fail(MJ_ERR_ARG, "unknown element type %d", dtype);
}

int32_t check_act(int32_t act) {
  if (act == MJ_EPI_NONE || act == MJ_EPI_RELU || act == MJ_EPI_GELU_TANH || act == MJ_EPI_SILU)
    return MJ_OK;
  if (valid_epi(act))
    return fail(MJ_ERR_UNSUPPORTED, "activation %d is not available here (NONE, RELU, GELU_TANH and "
                "SILU are)", act);
  return fail(MJ_ERR_ARG, "unknown activation %d", act);
}

int32_t check_experts(int64_t experts) {
  if (experts < 1 || experts > mj::kMaxExperts)
    return fail(MJ_ERR_ARG, "1 to %lld experts, got %lld", (long long)mj::kMaxExperts, (long long)experts);
  return MJ_OK;
}

// Rows are numbered in 32 bits, with room for the rows a tile looks ahead.
int32_t check_rows(const char *what, int64_t rows) {
  if (rows < 0) return fail(MJ_ERR_ARG, "%s: negative number of rows", what);
  if (rows > mj::kMlpMaxRows)
    return fail(MJ_ERR_UNSUPPORTED, "%s: at most %lld rows", what, (long long)mj::kMlpMaxRows);
  return MJ_OK;
}

int32_t check_width(const char *what, int64_t width, int64_t step) {
  if (width < 0) return fail(MJ_ERR_ARG, "%s: negative width", what);
  if (width % step)
    return fail(MJ_ERR_UNSUPPORTED, "%s: width %lld is not a multiple of %lld", what, (long long)width,
                (long long)step);
  if (width >= (int64_t)1 << 22) return fail(MJ_ERR_UNSUPPORTED, "%s: widths must be below 2^22", what);
  return MJ_OK;
}

int32_t check_aligned(const char *what, const void *const *ptrs, int n) {
  for (int i = 0; i < n; ++i)
    if (!aligned16(ptrs[i]))
      return fail(MJ_ERR_UNSUPPORTED, "%s: every array must be 16-byte aligned", what);
  return MJ_OK;
}

// The token arguments of dispatch and combine.
int32_t make_rows(const char *what, mj::ExpertRows &r, int32_t dtype, const int32_t *pos,
                  const int32_t *offsets, int64_t experts, int64_t tokens, int64_t topk, int64_t dim) {
  if (int32_t s = check_dtype(dtype)) return s;
  if (int32_t s = check_experts(experts)) return s;
  if (int32_t s = check_dims(tokens, topk, dim)) return s;
  if (topk > 0 && tokens > mj::kMlpMaxRows / topk)
    return fail(MJ_ERR_UNSUPPORTED, "%s: at most %lld slots", what, (long long)mj::kMlpMaxRows);
  if (tokens > 0 && dim > 0 && (!offsets || (topk > 0 && !pos)))
    return fail(MJ_ERR_ARG, "%s: null pos or offsets", what);
  r.pos = pos, r.kept = offsets ? offsets + experts : nullptr;
  r.tokens = tokens, r.topk = topk, r.dim = dim;
  return MJ_OK;
}

int32_t make_mlp(const char *what, mj::ExpertMlp &q, const uint16_t *xs, const int32_t *offsets,
                 int64_t experts, const uint16_t *Wg, const uint16_t *Wu, const uint16_t *Wd, int32_t act,
                 const float *weights, int64_t R, int64_t K, int64_t I, int64_t H) {
  if (int32_t s = check_act(act)) return s;
  if (int32_t s = check_experts(experts)) return s;
  if (int32_t s = check_rows(what, R)) return s;
  for (int64_t w : {K, I, H})
    if (int32_t s = check_width(what, w, 8)) return s;
  const void *ptrs[] = {xs, Wg, Wu, Wd};
  if (int32_t s = check_aligned(what, ptrs, 4)) return s;
  if (!offsets) return fail(MJ_ERR_ARG, "%s: null offsets", what);
  q.xs = xs, q.offsets = offsets, q.wg = Wg, q.wu = Wu, q.wd = Wd, q.act = act, q.rw = weights;
  q.R = R, q.E = experts, q.K = K, q.I = I, q.H = H;
  return MJ_OK;
}

int32_t make_f8(const char *what, mj::F8Product &q, const uint8_t *x, const float *sx, const uint8_t *w,
                const float *sw, int64_t M, int64_t N, int64_t K, int64_t n_step) {
  if (int32_t s = check_rows(what, M)) return s;
  if (int32_t s = check_width(what, N, n_step)) return s;
  if (int32_t s = check_width(what, K, 16)) return s;
  const void *ptrs[] = {x, w};
  if (int32_t s = check_aligned(what, ptrs, 2)) return s;
  if (M > 0 && N > 0 && K > 0 && (!x || !sx || !w || !sw)) return fail(MJ_ERR_ARG, "%s: null operand", what);
  q.x = x, q.sx = sx, q.w = w, q.sw = sw;
  q.M = M, q.N = N, q.K = K;
  return MJ_OK;
}

int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }
int64_t f8_blocks(int64_t k) { return (k + 127) / 128; }

}  // namespace

extern "C" {

// ------------------------------------------------------------------ experts' rows
int64_t mj_sort_experts_work_bytes(int64_t slots, int64_t experts) {
  if (slots <= 0 || experts < 1 || experts > mj::kMaxExperts) return 0;
  return mj::sort_experts_work_ints(slots, experts) * (int64_t)sizeof(int32_t);
}

int32_t mj_sort_experts(const void *ids, int32_t id_bytes, int64_t slots, int64_t experts, int32_t *pos,
                        int32_t *offsets, void *work, int64_t work_bytes, void *stream) {
  if (id_bytes != 4 && id_bytes != 8) return fail(MJ_ERR_ARG, "experts' numbers have 4 or 8 bytes");
  if (int32_t s = check_experts(experts)) return s;
  if (int32_t s = check_rows("expert sort", slots)) return s;
  if (!offsets || (slots > 0 && (!ids || !pos))) return fail(MJ_ERR_ARG, "null operand");
  const int64_t need = mj_sort_experts_work_bytes(slots, experts);
  if (need > 0 && (!work || work_bytes < need))
    return fail(MJ_ERR_ARG, "expert sort: work must hold %lld bytes", (long long)need);
  return hip_status(mj::launch_sort_experts(ids, id_bytes == 8, slots, experts, pos, offsets, (int *)work,
                                            S(stream)),
                    "expert sort launch");
}

int32_t mj_dispatch(int32_t dtype, const void *x, const float *weights, const int32_t *pos,
                    const int32_t *offsets, int64_t experts, void *xs, float *ws, int64_t tokens,
                    int64_t topk, int64_t dim, void *stream) {
  mj::ExpertRows r;
  if (int32_t s = make_rows("dispatch", r, dtype, pos, offsets, experts, tokens, topk, dim)) return s;
  if ((weights != nullptr) != (ws != nullptr)) return fail(MJ_ERR_ARG, "dispatch: weights and ws go together");
  if (tokens == 0 || topk == 0 || (dim == 0 && !ws)) return MJ_OK;
  if (!pos || !offsets || (dim > 0 && (!x || !xs))) return fail(MJ_ERR_ARG, "dispatch: null operand");
  r.x = const_cast<void *>(x), r.xs = xs, r.w = weights, r.ws = ws;
  return hip_status(mj::launch_dispatch(dtype == MJ_BF16, r, S(stream)), "dispatch launch");
}

int32_t mj_combine(int32_t dtype, int32_t y_dtype, const void *ys, const float *weights, const int32_t *pos,
                   const int32_t *offsets, int64_t experts, void *y, int64_t tokens, int64_t topk,
                   int64_t dim, void *stream) {
  mj::ExpertRows r;
  if (int32_t s = make_rows("combine", r, dtype, pos, offsets, experts, tokens, topk, dim)) return s;
  if (int32_t s = check_dtype(y_dtype)) return s;
  if (y_dtype != dtype && y_dtype != MJ_BF16)
    return fail(MJ_ERR_UNSUPPORTED, "combine: bf16 rows give bf16");
  if (tokens == 0 || dim == 0) return MJ_OK;
  if (!y || (topk > 0 && !ys)) return fail(MJ_ERR_ARG, "combine: null operand");
  r.x = y, r.xs = const_cast<void *>(ys), r.w = weights;
  return hip_status(mj::launch_combine(dtype == MJ_BF16, y_dtype == MJ_BF16, r, S(stream)), "combine launch");
}

int32_t mj_combine_backward(int32_t dtype, const void *dy, const void *ys, const float *weights,
                            const int32_t *pos, const int32_t *offsets, int64_t experts, void *dys, float *dw,
                            int64_t tokens, int64_t topk, int64_t dim, void *stream) {
  mj::ExpertRows r;
  if (int32_t s = make_rows("combine backward", r, dtype, pos, offsets, experts, tokens, topk, dim))
    return s;
  if (tokens == 0 || topk == 0) return MJ_OK;
  if (!pos || !offsets || !weights || !dw || (dim > 0 && (!dy || !ys || !dys)))
    return fail(MJ_ERR_ARG, "combine backward: null operand");
  r.x = const_cast<void *>(dy), r.ys = ys, r.w = weights, r.xs = dys, r.ws = dw;
  return hip_status(mj::launch_combine_bwd(dtype == MJ_BF16, r, S(stream)), "combine backward launch");
}

// ------------------------------------------------------------------ experts' block
int32_t mj_experts_mlp_bf16(const uint16_t *xs, const int32_t *offsets, int64_t experts, const uint16_t *Wg,
                            const uint16_t *Wu, const uint16_t *Wd, int32_t act, const float *weights,
                            uint16_t *h, float *g, float *u, float *ys, int64_t R, int64_t K, int64_t I,
                            int64_t H, void *stream) {
  mj::ExpertMlp q;
  if (int32_t s = make_mlp("experts", q, xs, offsets, experts, Wg, Wu, Wd, act, weights, R, K, I, H)) return s;
  const void *ptrs[] = {h, g, u, ys};
  if (int32_t s = check_aligned("experts", ptrs, 4)) return s;
  if (R == 0) return MJ_OK;
  if ((H > 0 && !ys) || (I > 0 && (!h || (H > 0 && !Wd) || (K > 0 && (!xs || !Wg || !Wu)))))
    return fail(MJ_ERR_ARG, "experts: null operand");
  if ((g == nullptr) != (u == nullptr)) return fail(MJ_ERR_ARG, "g and u are kept together");
  q.h = h, q.g = g, q.u = u, q.ys = ys;
  return hip_status(mj::launch_experts_mlp(q, S(stream)), "experts launch");
}

int64_t mj_experts_mlp_dots(int64_t R, int64_t experts, int64_t K, int64_t I, int64_t H) {
  if (R <= 0 || R > mj::kMlpMaxRows || experts < 1 || K < 0 || I <= 0 || H < 0) return 0;
  mj::ExpertMlp q;
  q.R = R, q.E = experts, q.K = K, q.I = I, q.H = H;
  return R * mj::expert_dots_ld(q);
}

int32_t mj_experts_mlp_backward_bf16(const uint16_t *xs, const int32_t *offsets, int64_t experts,
                                     const uint16_t *Wg, const uint16_t *Wu, const uint16_t *Wd, int32_t act,
                                     const float *weights, const uint16_t *h, const float *g, const float *u,
                                     const uint16_t *dys, uint16_t *dg, uint16_t *du, float *dxs,
                                     uint16_t *dWg, uint16_t *dWu, uint16_t *dWd, const int32_t *pos,
                                     int64_t slots, float *dots, float *dw, int64_t R, int64_t K, int64_t I,
                                     int64_t H, void *stream) {
  mj::ExpertMlp q;
  if (int32_t s = make_mlp("experts backward", q, xs, offsets, experts, Wg, Wu, Wd, act, weights, R, K, I, H))
    return s;
  const void *ptrs[] = {h, g, u, dys, dg, du, dxs, dWg, dWu, dWd};
  if (int32_t s = check_aligned("experts backward", ptrs, 10)) return s;
  if (slots < 0) return fail(MJ_ERR_ARG, "experts backward: negative number of slots");
  if (dw && slots > 0 && (!pos || (R > 0 && I > 0 && !dots)))
    return fail(MJ_ERR_ARG, "experts backward: dw needs pos and dots");
  if (R > 0 && I > 0 && (dxs || dWg || dWu || dw) && (!dg || !du || !g || !u || (H > 0 && (!dys || !Wd))))
    return fail(MJ_ERR_ARG, "experts backward: null operand");
  if (R > 0 && I > 0 && K > 0 && dxs && (!Wg || !Wu)) return fail(MJ_ERR_ARG, "experts backward: null weights");
  if (R > 0 && I > 0 && K > 0 && (dWg || dWu) && !xs) return fail(MJ_ERR_ARG, "experts backward: null xs");
  if (R > 0 && I > 0 && H > 0 && dWd && (!dys || !h)) return fail(MJ_ERR_ARG, "experts backward: null dys or h");
  q.h = const_cast<uint16_t *>(h), q.g = const_cast<float *>(g), q.u = const_cast<float *>(u);
  mj::ExpertMlpGrad o;
  o.dys = dys, o.dg = dg, o.du = du, o.dxs = dxs, o.dwg = dWg, o.dwu = dWu, o.dwd = dWd;
  o.dots = dw ? dots : nullptr, o.dw = dw, o.pos = pos, o.slots = slots;
  return hip_status(mj::launch_experts_mlp_bwd(q, o, S(stream)), "experts backward launch");
}

const char *mj_experts_mlp_kernel(int64_t R, int64_t experts, int64_t K, int64_t I, int64_t H, int32_t product) {
  if (R <= 0 || R > mj::kMlpMaxRows || check_experts(experts) || product < 0 || product > 4) return "";
  for (int64_t w : {K, I, H})
    if (w == 0 || check_width("experts", w, 8)) return "";
  mj::ExpertMlp q;
  q.R = R, q.E = experts, q.K = K, q.I = I, q.H = H;
  return mj::experts_kernel_name(q, product);
}

// ------------------------------------------------------------------ 8-bit floating point
const char *mj_gemm_f8_kernel(int64_t M, int64_t N, int64_t K, int64_t experts, int32_t gate) {
  if (M <= 0 || M > mj::kMlpMaxRows || N <= 0 || K <= 0 || check_width("fp8", N, 1) || check_width("fp8", K, 16) ||
      (experts != 0 && check_experts(experts)) || (gate && experts == 0))
    return "";
  mj::F8Product q;
  const uint8_t none = 0;
  const int32_t row = 0;
  q.M = M, q.N = N, q.K = K, q.experts = (int)experts;
  q.offsets = experts ? &row : nullptr, q.w2 = gate ? &none : nullptr;
  return mj::gemm_f8_kernel_name(q);
}

int32_t mj_quantize_rows_f8(int32_t dtype, const void *x, uint8_t *q, float *scales, int64_t rows, int64_t K,
                            void *stream) {
  if (int32_t s = check_dtype(dtype)) return s;
  if (int32_t s = check_rows("fp8 rows", rows)) return s;
  if (int32_t s = check_width("fp8 rows", K, 16)) return s;
  if (rows == 0 || K == 0) return MJ_OK;
  if (!x || !q || !scales) return fail(MJ_ERR_ARG, "fp8 rows: null operand");
  const void *ptrs[] = {x, q};
  if (int32_t s = check_aligned("fp8 rows", ptrs, 2)) return s;
  mj::F8Rows a;
  a.x = x, a.q = q, a.scales = scales, a.tokens = a.rows = rows, a.dim = K;
  return hip_status(mj::launch_quantize_rows_f8(dtype == MJ_BF16, a, S(stream)), "fp8 rows launch");
}

int32_t mj_dispatch_f8(int32_t dtype, const void *x, const int32_t *pos, const int32_t *offsets,
                       int64_t experts, uint8_t *q, float *scales, int64_t tokens, int64_t topk, int64_t K,
                       void *stream) {
  mj::ExpertRows r;
  if (int32_t s = make_rows("fp8 dispatch", r, dtype, pos, offsets, experts, tokens, topk, K)) return s;
  if (int32_t s = check_width("fp8 dispatch", K, 16)) return s;
  if (tokens == 0 || topk == 0 || K == 0) return MJ_OK;
  if (!x || !q || !scales) return fail(MJ_ERR_ARG, "fp8 dispatch: null operand");
  const void *ptrs[] = {x, q};
  if (int32_t s = check_aligned("fp8 dispatch", ptrs, 2)) return s;
  mj::F8Rows a;
  a.x = x, a.q = q, a.scales = scales, a.tokens = tokens, a.topk = topk, a.rows = tokens * topk, a.dim = K;
  a.pos = r.pos, a.kept = r.kept;
  return hip_status(mj::launch_quantize_rows_f8(dtype == MJ_BF16, a, S(stream)), "fp8 dispatch launch");
}

int32_t mj_quantize_blocks_f8(int32_t dtype, const void *W, uint8_t *q, float *scales, int64_t mats, int64_t N,
                              int64_t K, void *stream) {
  if (int32_t s = check_dtype(dtype)) return s;
  if (mats < 0) return fail(MJ_ERR_ARG, "fp8 blocks: negative number of matrices");
  if (int32_t s = check_width("fp8 blocks", N, 1)) return s;
  if (int32_t s = check_width("fp8 blocks", K, 16)) return s;
  if (mats == 0 || N == 0 || K == 0) return MJ_OK;
  if (!W || !q || !scales) return fail(MJ_ERR_ARG, "fp8 blocks: null operand");
  const void *ptrs[] = {W, q};
  if (int32_t s = check_aligned("fp8 blocks", ptrs, 2)) return s;
  mj::F8Blocks a;
  a.w = W, a.q = q, a.scales = scales, a.mats = mats, a.n = N, a.k = K;
  return hip_status(mj::launch_quantize_blocks_f8(dtype == MJ_BF16, a, S(stream)), "fp8 blocks launch");
}

int64_t mj_gemm_f8_work_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return mj::gemm_f8_part_floats(M, N, K) * (int64_t)sizeof(float);
}

int32_t mj_gemm_f8(const uint8_t *xq, const float *sx, const uint8_t *Wq, const float *sw, const float *bias,
                   int32_t act, uint16_t *y, int64_t M, int64_t N, int64_t K, void *work, int64_t work_bytes,
                   void *stream) {
  mj::F8Product q;
  if (int32_t s = check_act(act)) return s;
  if (int32_t s = make_f8("fp8 product", q, xq, sx, Wq, sw, M, N, K, 1)) return s;
  const void *ptrs[] = {y, work};
  if (int32_t s = check_aligned("fp8 product", ptrs, 2)) return s;
  if (M == 0 || N == 0) return MJ_OK;
  if (!y) return fail(MJ_ERR_ARG, "fp8 product: null operand");
  const int64_t need = mj_gemm_f8_work_bytes(M, N, K);
  if (need > 0 && (!work || work_bytes < need))
    return fail(MJ_ERR_ARG, "fp8 product: work must hold %lld bytes", (long long)need);
  q.bias = bias, q.epi = act, q.y = y, q.part = (float *)work;
  return hip_status(mj::launch_gemm_f8(q, S(stream)), "fp8 product launch");
}

int64_t mj_linear_f8_work_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const int64_t part = mj_gemm_f8_work_bytes(M, N, K);
  return mj::gemm_f8_quantizes(M, N, K) ? part : up16(M * K) + up16(4 * M * f8_blocks(K)) + part;
}

int32_t mj_linear_f8(int32_t dtype, const void *x, const uint8_t *Wq, const float *sw, const float *bias,
                     int32_t act, uint16_t *y, int64_t M, int64_t N, int64_t K, void *work, int64_t work_bytes,
                     void *stream) {
  if (int32_t s = check_dtype(dtype)) return s;
  if (int32_t s = check_act(act)) return s;
  if (int32_t s = check_rows("fp8 Linear", M)) return s;
  if (int32_t s = check_width("fp8 Linear", N, 1)) return s;
  if (int32_t s = check_width("fp8 Linear", K, 16)) return s;
  const void *ptrs[] = {x, Wq, y, work};
  if (int32_t s = check_aligned("fp8 Linear", ptrs, 4)) return s;
  if (M == 0 || N == 0) return MJ_OK;
  if (!y || (K > 0 && (!x || !Wq || !sw))) return fail(MJ_ERR_ARG, "fp8 Linear: null operand");
  const int64_t need = mj_linear_f8_work_bytes(M, N, K);
  if (need > 0 && (!work || work_bytes < need))
    return fail(MJ_ERR_ARG, "fp8 Linear: work must hold %lld bytes", (long long)need);
  mj::F8Product q;
  q.w = Wq, q.sw = sw, q.bias = bias, q.epi = act, q.y = y, q.M = M, q.N = N, q.K = K;
  char *rest = (char *)work;
  if (mj::gemm_f8_quantizes(M, N, K)) {
    q.xf = x, q.xf_bf16 = dtype == MJ_BF16;
  } else if (K > 0) {
    mj::F8Rows a;
    a.x = x, a.tokens = a.rows = M, a.dim = K;
    a.q = (uint8_t *)work, a.scales = (float *)(rest + up16(M * K));
    rest = (char *)a.scales + up16(4 * M * f8_blocks(K));
    if (int32_t s = hip_status(mj::launch_quantize_rows_f8(dtype == MJ_BF16, a, S(stream)), "fp8 rows launch"))
      return s;
    q.x = a.q, q.sx = a.scales;
  }
  q.part = (float *)rest;
  return hip_status(mj::launch_gemm_f8(q, S(stream)), "fp8 Linear launch");
}

int32_t mj_experts_gemm_f8(const uint8_t *xq, const float *sx, const int32_t *offsets, int64_t experts,
                           const uint8_t *Wq, const float *sw, float *y, int64_t R, int64_t N, int64_t K,
                           void *stream) {
  mj::F8Product q;
  if (int32_t s = check_experts(experts)) return s;
  if (int32_t s = make_f8("fp8 experts", q, xq, sx, Wq, sw, R, N, K, 1)) return s;
  if (!aligned16(y)) return fail(MJ_ERR_UNSUPPORTED, "fp8 experts: every array must be 16-byte aligned");
  if (R == 0 || N == 0) return MJ_OK;
  if (!y || !offsets) return fail(MJ_ERR_ARG, "fp8 experts: null operand");
  q.offsets = offsets, q.experts = (int)experts, q.tail = 1, q.h = y;
  return hip_status(mj::launch_gemm_f8(q, S(stream)), "fp8 experts launch");
}

int64_t mj_experts_gate_f8_work_bytes(int64_t R, int64_t experts, int64_t I, int64_t K) {
  if (R <= 0 || experts < 1 || experts > mj::kMaxExperts || I <= 0 || K < 0) return 0;
  mj::F8Product q;
  const uint8_t none = 0;
  q.w2 = &none, q.M = R, q.N = I, q.K = K, q.experts = (int)experts;
  return mj::gemm_f8_fuses(q) ? 0 : 4 * R * I;
}

int32_t mj_experts_gate_f8(const uint8_t *xq, const float *sx, const int32_t *offsets, int64_t experts,
                           const uint8_t *Wg, const float *sg, const uint8_t *Wu, const float *su, int32_t act,
                           uint8_t *hq, float *sh, int64_t R, int64_t I, int64_t K, void *work,
                           int64_t work_bytes, void *stream) {
  mj::F8Product q;
  if (int32_t s = check_act(act)) return s;
  if (int32_t s = check_experts(experts)) return s;
  if (int32_t s = make_f8("fp8 gate", q, xq, sx, Wg, sg, R, I, K, 16)) return s;
  const void *ptrs[] = {Wu, hq, work};
  if (int32_t s = check_aligned("fp8 gate", ptrs, 3)) return s;
  if (R == 0 || I == 0) return MJ_OK;
  if (!Wu || !su || !hq || !sh || !offsets) return fail(MJ_ERR_ARG, "fp8 gate: null operand");
  const int64_t need = mj_experts_gate_f8_work_bytes(R, experts, I, K);
  if (need > 0 && (!work || work_bytes < need))
    return fail(MJ_ERR_ARG, "fp8 gate: work must hold %lld bytes", (long long)need);
  q.w2 = Wu, q.sw2 = su, q.epi = act, q.h = (float *)work, q.hq = hq, q.sh = sh;
  q.offsets = offsets, q.experts = (int)experts, q.tail = 1;
  if (int32_t s = hip_status(mj::launch_gemm_f8(q, S(stream)), "fp8 gate launch")) return s;
  if (need == 0) return MJ_OK;
  return mj_quantize_rows_f8(MJ_F32, work, hq, sh, R, I, stream);
}

}  // extern "C"
