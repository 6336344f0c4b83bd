/*
 * momijo_hip.h -- C ABI of the MI355X (gfx950) backend for momijo's
 * tensor-engine hot path: dense matmul / Linear, the int8 weight path and the
 * bias + activation epilogue.
 *
 * Every entry point is `extern "C"`, takes plain pointers and sizes, returns
 * an int32 status (MJ_OK = 0) and never throws.  Unless a name ends in `_h`
 * (or is one of the memory-copy entry points), pointers are DEVICE pointers (HIP global memory of the current device) and
 * the call is asynchronous on `stream` (a hipStream_t; NULL = the null
 * stream).  `_h` variants take HOST pointers, copy in, run and copy out
 * synchronously, which is the ownership model of the reference's own device
 * seam (tensor/gpu/runtime.mojo:539-631).
 *
 * Layout conventions: row-major with explicit leading dimensions / strides in
 * ELEMENTS.  bf16 values travel as uint16_t bit patterns.  Weights follow the
 * reference's Linear layout [out_features, in_features] (learn/nn/layers.mojo:
 * 347-348), so y = x W^T is an "NT" product.
 *
 * Workspace.  Calls that need scratch device memory (the split-K W8A16 and
 * bf16 GEMMs, the FFN when it splits K, QuantLinear, the W8A8 Linear,
 * Linear.backward's column sums for N > 1024, the min/max observer) take it
 * from one buffer per (device, stream) that the library keeps and grows;
 * hipStreamPerThread gets one per (device, host thread).  A call holds that
 * buffer from its first to its last enqueue, so host threads may share a
 * stream.  While `stream` is being captured into a HIP graph these calls
 * return MJ_ERR_UNSUPPORTED and enqueue nothing: the library never allocates
 * on a capturing stream.  Everything else (the GEMV, GEMMs without a K split,
 * quantizers, mj_quant_linear_f32_noalloc) can be captured.  For the bf16 GEMM
 * the shape alone decides: one whose larger tiles would split K is refused also
 * where the tile that serves it does not (the error says which of the two it is).
 *
 * Reference citations are relative to /root/reference/legacy/src/momijo/.
 */
#ifndef MOMIJO_HIP_H
#define MOMIJO_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes --------------------------------------------------- */
#define MJ_OK 0
#define MJ_ERR_ARG 1         /* null pointer, bad enum, negative size       */
#define MJ_ERR_SHAPE 2       /* operand shapes disagree                     */
#define MJ_ERR_UNSUPPORTED 3 /* alignment / divisibility the kernels need   */
#define MJ_ERR_DEVICE 4      /* a HIP runtime error (launch, copy, sync)    */
#define MJ_ERR_NO_DEVICE 5   /* no gfx950 device is visible                 */
#define MJ_ERR_ALLOC 6       /* device allocation failed                    */

/* ---- epilogues: applied to the fp32 result after scale and bias ----- */
#define MJ_EPI_NONE 0
#define MJ_EPI_RELU 1              /* ReLU.forward: v > 0 ? v : 0 (layers.mojo:117-137)      */
#define MJ_EPI_GELU_TANH 2         /* gelu32 (tensor/math.mojo:288-295), finite past x~10.06 */
#define MJ_EPI_SILU 3              /* silu32 (tensor/math.mojo:283-285)                      */
#define MJ_EPI_GELU_TANH_APPROX 4  /* learn.nn gelu via _exp_approx (activations.mojo:158-163) */
#define MJ_EPI_SILU_APPROX 5       /* learn.nn silu via _exp_approx (activations.mojo:137-152) */
/* Entry points with fp32 outputs evaluate GELU_TANH and SILU literally (expf,
 * IEEE division).  Entry points with bf16 outputs (the bf16 and W8A16 GEMMs,
 * GEMVs and the FFN) evaluate the same functions as x / (1 + 2^(-2t log2 e))
 * and x / (1 + 2^(-x log2 e)) with the hardware exp2 and reciprocal: the bf16
 * bits differ from the literal form's in a few outputs in 10^4 (near a
 * rounding boundary) and, for GELU at x < -2, where the literal form's
 * 1 + tanh cancels; every output stays within one bf16 step or 1e-6. */
#define MJ_EPI_RELU_UNARY 6        /* Tensor.relu, apply_unary op 8 (tensor/math.mojo:582-585) */

/* ---- int8 rounding rules -------------------------------------------- */
#define MJ_ROUND_RHE 0     /* round half to even, clamp [-127,127] (per-channel spec)   */
#define MJ_ROUND_LEGACY 1  /* fp32 v +- 0.5 then truncate, clamp [-128,127]
                              (functional.mojo:208-217)                                 */

/* ---- runtime ---------------------------------------------------------- */

/* ABI version (major*100 + minor). */
int32_t mj_version(void);

/* 1 if a gfx950 device is usable, else 0.  Replaces gpu_available()
 * (tensor/gpu/runtime.mojo:29-36), which is a compile-time probe there. */
int32_t mj_device_available(void);

/* Message for the last non-OK status returned on this host thread. */
const char *mj_last_error(void);

/* Waits for all work queued on `stream`. */
int32_t mj_stream_synchronize(void *stream);

/* ---- fp32 engine ------------------------------------------------------ */

/* C[M,N] = epi(A @ B + bias) for fp32 operands given as (pointer, row stride,
 * column stride), so transposed views (stride swaps, tensor/transform.mojo:
 * 1248-1294, 2107-2136) need no copy.  bias may be NULL; C has leading
 * dimension ldc.  Replaces matmul_core_mm (tensor/broadcast.mojo:1612-1673),
 * reached from Tensor.matmul (tensor/tensor.mojo:3168-3169) and
 * tensor.matmul (tensor/__init__.mojo:123). */
int32_t mj_matmul_f32(int64_t M, int64_t N, int64_t K,
                      const float *A, int64_t sAm, int64_t sAk,
                      const float *B, int64_t sBk, int64_t sBn,
                      const float *bias, int32_t epilogue,
                      float *C, int64_t ldc, void *stream);

/* The bits of an fp32 result.  Products of up to 256^3 multiply-adds with K <= 1024,
 * and all with K <= 16, are summed in the reference's strict k order on the fp32
 * MFMA, one product's rounding after another.  Larger ones run on bf16 MFMA with
 * every operand split in three bf16 parts: blocks of 32 k, six terms each, added in
 * k order; closer to the exact sum from K = 17 on, and an output that the parts
 * cannot hold (infinities, magnitudes that round to infinity in bf16, elements below
 * 2^-110 where they matter) is computed on the fp32 MFMA.  Within each of the two,
 * the bits do not depend on the tile, the layout or the batch, and a convolution has
 * the bits of the matmul on its im2col; but which of the two runs depends on M, N
 * and K, so a row's bits can change with the number of rows in the call.
 *
 * The kernel that such a call runs, by name ("" for an empty or refused one).
 * Host only; for tests and profiles. */
const char *mj_matmul_f32_kernel(int64_t M, int64_t N, int64_t K, int64_t batches, int64_t sAm,
                                 int64_t sBn);
const char *mj_conv2d_f32_kernel(int64_t N, int64_t C, int64_t H, int64_t W, int64_t OC,
                                 int64_t kH, int64_t kW, int64_t sH, int64_t sW, int64_t pH,
                                 int64_t pW);
const char *mj_gemm_bf16_kernel(int64_t M, int64_t N, int64_t K);

/* y[M] = A[M,N] x[N] with strides.  Replaces matmul_core_vec
 * (tensor/broadcast.mojo:1543-1608), Tensor.matmul_vec (tensor.mojo:3180). */
int32_t mj_matvec_f32(int64_t M, int64_t N, const float *A, int64_t sAm, int64_t sAn,
                      const float *x, int64_t sx, float *y, void *stream);

/* y[N,OutF] = epi(x[N,InF] W^T + b), W [OutF,InF] row-major, b [OutF] or
 * NULL.  Replaces Linear.forward / forward_auto (learn/nn/layers.mojo:
 * 383-433, 510-516) with the activation layer that follows it fused in. */
int32_t mj_linear_f32(const float *x, const float *W, const float *bias, int32_t epilogue,
                      float *y, int64_t N, int64_t InF, int64_t OutF, void *stream);

/* fp64 C[M,N] = A @ B with strides, on v_mfma_f64_16x16x4f64.  Replaces the
 * Float64 overloads of matmul_core_mm / matmul (tensor/broadcast.mojo:
 * 1466-1538) and matmul2d (tensor/math.mojo:7838-7880), which autograd's
 * matmul backward calls (tensor/autograd.mojo:1542-1555). */
int32_t mj_matmul_f64(int64_t M, int64_t N, int64_t K,
                      const double *A, int64_t sAm, int64_t sAk,
                      const double *B, int64_t sBk, int64_t sBn,
                      double *C, int64_t ldc, void *stream);

/* fp64 y[M] = A[M,N] x[N].  Replaces matmul_core_vec Float64
 * (tensor/broadcast.mojo:1397-1464). */
int32_t mj_matvec_f64(int64_t M, int64_t N, const double *A, int64_t sAm, int64_t sAn,
                      const double *x, int64_t sx, double *y, void *stream);

/* tensordot(A, B, axes=1) for fp32 (tensor/broadcast.mojo:1694-1900):
 * C[b, :, :] = A[b] @ B[b] over batch_rank <= 5 broadcast batch dimensions
 * of extent batch_shape[d]; the element strides of A's and B's batch
 * dimensions are a_batch_strides[d], b_batch_strides[d] (0 where the operand
 * is broadcast), and A[b], B[b] are (row stride, column stride) views as in
 * mj_matmul_f32.  C is contiguous [batch..., M, N].  The three arrays are
 * host memory. */
int32_t mj_tensordot_f32(int32_t batch_rank, const int64_t *batch_shape,
                         const int64_t *a_batch_strides, const int64_t *b_batch_strides,
                         int64_t M, int64_t N, int64_t K,
                         const float *A, int64_t sAm, int64_t sAk,
                         const float *B, int64_t sBk, int64_t sBn,
                         float *C, void *stream);

/* The MATMUL2D rule of the autograd tape (tensor/autograd.mojo:1542-1555)
 * for y = A @ B, A [M,K], B [K,N], upstream gradient G [M,N], all Float64
 * row-major device arrays:
 *   dA [M,K] (+)= G @ B^T      dB [K,N] (+)= A^T @ G
 * With accumulate != 0 the products are added to the existing dA / dB (the
 * tape's grads[p] = grads[p].add(g)); otherwise they overwrite them.  The
 * transposes are stride views; either output may be NULL. */
int32_t mj_matmul_backward_f64(int64_t M, int64_t N, int64_t K, const double *A, const double *B,
                               const double *G, double *dA, double *dB, int32_t accumulate,
                               void *stream);

/* The same MATMUL2D rule in Float32, the value type of the reference tape
 * (Tape.values / grads are List[Tensor[Float32]], tensor/autograd.mojo:
 * 214-216; GradTensor.matmul / matmul2d record the node, :930-939 and
 * :995-1017): dA (+)= G @ B^T, dB (+)= A^T @ G on the fp32 MFMA engine, the
 * products summed in fp32 and added to the old gradient with one rounding
 * (grads[p].add(g)).  Either output may be NULL. */
int32_t mj_matmul_backward_f32(int64_t M, int64_t N, int64_t K, const float *A, const float *B,
                               const float *G, float *dA, float *dB, int32_t accumulate,
                               void *stream);

/* Host-pointer seam with the signature of launch_1d_linear_fw
 * (tensor/gpu/runtime.mojo:539-631): x [N,InF], wT [InF,OutF] (the layout
 * Linear.forward_gpu builds, layers.mojo:489-497), b [OutF], y [N,OutF];
 * y[n,o] = sum_k x[n,k] wT[k,o] + b[o] as the seam's CPU kernel
 * _kernel_linear_fw (layers.mojo:436-475) defines it.  Synchronous. */
int32_t mj_launch_linear_fw_h(const float *x, const float *wT, const float *b, float *y,
                              int64_t N, int64_t InF, int64_t OutF, int32_t has_bias);

/* Linear.backward (learn/nn/layers.mojo:519-618, 785-787) for x [N,InF],
 * W [OutF,InF], dy [N,OutF] (device pointers, row-major):
 *   dW[o,i] = sum_n dy[n,o] x[n,i]   (dW [OutF,InF], the layer's layout)
 *   db[o]   = sum_n dy[n,o]          (strict ascending n for N <= 1024,
 *                                     else ascending within row segments)
 *   dx[n,i] = sum_o dy[n,o] W[o,i]   (dx [N,InF])
 * dx and dW run on the fp32 MFMA engine over stride views (no transposed
 * copies).  Any output may be NULL to skip it. */
int32_t mj_linear_backward_f32(const float *x, const float *W, const float *dy, float *dW,
                               float *db, float *dx, int64_t N, int64_t InF, int64_t OutF,
                               void *stream);

/* Host-pointer seams with the signatures of launch_1d_linear_bw_dx / _dw /
 * _db (tensor/gpu/runtime.mojo:636-713, 714-832, 834-903).  Layouts follow
 * the seam's CPU kernels _kernel_linear_bw_dx/_dw/_db (layers.mojo:624-729):
 * w and dW are [OutF,InF].  (The seam's GPU kernels, runtime.mojo:75-119,
 * index w and dW as [InF,OutF]; that layout is not reproduced.)  Synchronous. */
int32_t mj_launch_linear_bw_dx_h(const float *dy, const float *w, float *dx, int64_t N,
                                 int64_t InF, int64_t OutF);
int32_t mj_launch_linear_bw_dw_h(const float *dy, const float *x, float *dW, int64_t N,
                                 int64_t InF, int64_t OutF);
int32_t mj_launch_linear_bw_db_h(const float *dy, float *db, int64_t N, int64_t OutF);

/* Elementwise fp32 activation y = epi(x) over n elements (may alias).
 * Replaces Tensor.relu / silu / gelu (tensor/tensor.mojo:3848,4003,4020 ->
 * apply_unary, tensor/math.mojo:566-638) and ReLU.forward (layers.mojo:134). */
int32_t mj_activation_f32(int32_t epilogue, const float *x, float *y, int64_t n, void *stream);

/* ---- conv2d ------------------------------------------------------------- */

/* Conv2d.forward, NCHW fp32 (learn/nn/conv.mojo:600-681, the naive GPU kernel
 * _gpu_conv2d_fw_kernel, tensor/gpu/runtime.mojo:159-200): x [N,C,H,W],
 * w [OC,C,kH,kW], b [OC] or NULL, y [N,OC,OH,OW] with
 * OH = (H + 2 pH - kH) // sH + 1 (floor), OW likewise; zero padding, the
 * bias after the sum, then `epilogue` (MJ_EPI_NONE for the reference's
 * layer).  One implicit GEMM per image on fp32 MFMA: y[n] = w [OC, C kH kW]
 * @ im2col(x[n]), the im2col gathered by the kernel's loader, nothing
 * materialised.  An empty output (OH or OW <= 0) is MJ_OK with nothing
 * written.  Padded taps are multiplied as zeros where the reference skips
 * them: the same sums for finite weights. */
int32_t mj_conv2d_f32(const float *x, const float *w, const float *b, int32_t epilogue, float *y,
                      int64_t N, int64_t C, int64_t H, int64_t W, int64_t OC, int64_t kH,
                      int64_t kW, int64_t sH, int64_t sW, int64_t pH, int64_t pW, void *stream);

/* Host-pointer seam of launch_1d_conv2d_fw (tensor/gpu/runtime.mojo:376-470):
 * the same arguments (OH, OW as the caller computed them, checked against
 * the geometry: MJ_ERR_SHAPE if they disagree), copy in, mj_conv2d_f32,
 * copy out into y; has_bias = 0 ignores b. */
int32_t mj_launch_conv2d_fw_h(const float *x, const float *w, const float *b, float *y, int64_t N,
                              int64_t C, int64_t H, int64_t W, int64_t OH, int64_t OW, int64_t OC,
                              int64_t kH, int64_t kW, int64_t sH, int64_t sW, int64_t pH,
                              int64_t pW, int32_t has_bias);

/* y = x >= s ? x : s over n fp32 elements (may alias): -0 stays -0 at s = 0,
 * NaN gives s.  Replaces Tensor[Float32].maximum_scalar(s) =
 * where_f32(ge_t(self, s), self, s) (tensor/tensor.mojo:4232), which
 * Converted.forward applies between the quantized layers
 * (learn/api/sequential.mojo:423). */
int32_t mj_maximum_scalar_f32(const float *x, float s, float *y, int64_t n, void *stream);

/* y = Float32(x) over n int64 elements, rounded to nearest even.  Replaces
 * astype_f32_from_int (tensor/cast.mojo:5431-5437), the upcast of
 * Tensor[Int].matmul / matmul_vec (tensor/tensor.mojo:3161-3165,3174-3178). */
int32_t mj_cast_i64_f32(const int64_t *x, float *y, int64_t n, void *stream);

/* ---- bf16 -------------------------------------------------------------- */

/* C[M,N] = bf16(epi(A[M,K] B[N,K]^T + bias)), fp32 accumulation on bf16
 * MFMA.  No reference counterpart: momijo has no bf16 matmul (broadcast.mojo
 * has f64/f32 overloads only, :1531,1677); its result is defined as the fp32
 * engine on exactly upcast bf16 inputs.  Needs K % 8 == 0, lda/ldb/ldc % 8
 * == 0 and 16-byte aligned A, B, C. */
int32_t mj_gemm_bf16_nt(int64_t M, int64_t N, int64_t K,
                        const uint16_t *A, int64_t lda, const uint16_t *B, int64_t ldb,
                        const float *bias, int32_t epilogue,
                        uint16_t *C, int64_t ldc, void *stream);

/* ---- int8: legacy per-tensor W8A8 (QuantLinear) ------------------------- */

/* q[i] = clamp(round(x[i]/scale)) with the MJ_ROUND_LEGACY rule; scale 0 is
 * replaced by 1.  Replaces quantize_symmetric_int8 (learn/api/functional.mojo:
 * 231-247). */
int32_t mj_quantize_symmetric_int8(const float *x, int64_t n, float scale, int8_t *q, void *stream);

/* minmax_out (device fp32 [2]) = {min x, max x} over n > 0 elements: the
 * reduction of MinMaxObserver.observe (learn/api/sequential.mojo:232-250). */
int32_t mj_minmax_f32(const float *x, int64_t n, float *minmax_out, void *stream);

/* *scale_out (device fp32) = max(|min x|, |max x|) / max_q, or 1.0 when n == 0,
 * max_q <= 0 or the magnitude is 0.  Replaces MinMaxObserver.observe +
 * scale_symmetric (learn/api/sequential.mojo:232-263). */
int32_t mj_minmax_scale_symmetric(const float *x, int64_t n, float max_q, float *scale_out,
                                  void *stream);

/* C[M,N] int32 = A[M,K] int8 * B^T, B = w_q [N,K] int8, exact int32
 * accumulation on int8 MFMA.  legacy_literal = 1 instead reads B as
 * reshape(w_q.flat, [K,N]) exactly as matmul_i8_i8_to_i32 does when handed
 * the stride view w_q.transpose() (learn/api/functional.mojo:249-279, :274).
 * Runs on int8 MFMA for every K and alignment (K % 16 == 0 with 16-byte aligned
 * A and B on the larger tiles); the literal read is one thread per output. */
int32_t mj_matmul_i8_i8_to_i32(const int8_t *A, const int8_t *B, int32_t *C,
                               int64_t M, int64_t N, int64_t K, int32_t legacy_literal,
                               void *stream);

/* y[M,N] = float(acc) * sf + b[N] (rounded multiply, then rounded add).
 * Replaces dequantize_i32_to_f32_add_bias (learn/api/functional.mojo:281-302). */
int32_t mj_dequantize_i32_to_f32_add_bias(const int32_t *acc, float sf, const float *b, float *y,
                                          int64_t M, int64_t N, void *stream);

/* y[M,N] = float(acc) * (sx[m] * sw[n]) + b[n], each fp32 operation rounded
 * on its own (sx * sw first); sx may be NULL (the factor is then sw[n]) and
 * b may be NULL.  The per-channel (and per-row) form of
 * dequantize_i32_to_f32_add_bias (learn/api/functional.mojo:281-302), for
 * int32 sums from mj_matmul_i8_i8_to_i32 with per-channel weight scales; it
 * is the epilogue of mj_linear_w8a8 as a separate operator. */
int32_t mj_dequantize_i32_scaled_f32(const int32_t *acc, const float *sx, const float *sw,
                                     const float *b, float *y, int64_t M, int64_t N,
                                     void *stream);

/* QuantLinear.forward (learn/nn/layers.mojo:1681-1685): quantize x [M,K]
 * with s_x, int8 GEMM against w_q [N,K], y = float(acc)*(s_x*s_w) + b.
 * The dequantize is fused into the GEMM epilogue; the int8 copy of x lives in
 * a device workspace the library owns. */
int32_t mj_quant_linear_f32(const float *x, const int8_t *Wq, const float *b,
                            float s_w, float s_x, float *y,
                            int64_t M, int64_t N, int64_t K, int32_t legacy_literal,
                            void *stream);

/* mj_quant_linear_f32 without any device allocation.  No counterpart in the
 * reference: it is for callers that cannot allocate -- code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc.  The int8
 * copy of x lives in a static 16 MiB device array owned by the library (one
 * per GPU, held until the process ends), so M*K must be at most 16 MiB - 16
 * bytes (MJ_ERR_UNSUPPORTED otherwise).  Results equal mj_quant_linear_f32's.
 * Every call on a GPU shares that GPU's array: calls that overlap on one GPU
 * (different streams, or host threads without ordering) race. */
int32_t mj_quant_linear_f32_noalloc(const float *x, const int8_t *Wq, const float *b,
                                    float s_w, float s_x, float *y,
                                    int64_t M, int64_t N, int64_t K, int32_t legacy_literal,
                                    void *stream);

/* ---- int8: per-output-channel weight-only (BASELINE spec) -------------- */

/* Q[N,K] int8 and scales[N] from W[N,K] fp32, one scale per output row.
 * MJ_ROUND_RHE: scale = max|row|/127 (1.0 for an all-zero row),
 *               q = clamp(rne(w/scale), -127, 127).
 * MJ_ROUND_LEGACY: scale = MinMax rule per row (sequential.mojo:252-263),
 *               q by functional.mojo:214-217.
 * The per-tensor reference path is quantize_symmetric_int8 + convert
 * (sequential.mojo:436-450); this is its per-row generalisation. */
int32_t mj_quantize_rowwise_i8(const float *W, int64_t N, int64_t K, int32_t rounding,
                               int8_t *Q, float *scales, void *stream);

/* y[M,N] = bf16(epi((x[M,K] . Q[N,K]^T) * scales[N] + bias[N])) with x bf16,
 * fp32 accumulation.  M <= 16 (and M <= 48 when K is a multiple of 1024 up
 * to 4096) runs the GEMV kernels, larger M the MFMA GEMM with int8 -> bf16
 * conversion in registers.  bias may be NULL.  Needs K % 16 == 0 and 16-byte
 * aligned x, Q, y. */
int32_t mj_linear_w8a16(const uint16_t *x, const int8_t *Q, const float *scales,
                        const float *bias, int32_t epilogue, uint16_t *y,
                        int64_t M, int64_t N, int64_t K, void *stream);

/* Dynamic per-row activation quantize: xq[M,K] int8 and sx[M] fp32 from
 * x[M,K] bf16 by the MJ_ROUND_RHE rule of mj_quantize_rowwise_i8 applied to
 * each row of x (sx[m] = max|x[m,:]|/127, 1.0 for an all-zero row;
 * xq = clamp(rne(x/sx[m]), -127, 127); NaN -> 0).  The activation half of
 * mj_linear_w8a8; the per-tensor reference step it generalises is
 * quantize_symmetric_int8 with the observer's scale (learn/api/
 * functional.mojo:231-247, sequential.mojo:232-263). */
int32_t mj_quantize_rows_bf16_i8(const uint16_t *x, int64_t M, int64_t K, int8_t *xq, float *sx,
                                 void *stream);

/* W8A8 Linear with dynamic activation scales:
 *   sx, xq = mj_quantize_rows_bf16_i8(x)
 *   y[m,n] = bf16(epi(float(xq[m,:] . Q[n,:]) * (sx[m] * scales[n]) + bias[n]))
 * with the int32 dot product exact on int8 MFMA and the epilogue rounded
 * step by step in fp32 (sx*scales, then the product, then the bias).  It is
 * QuantLinear.forward (learn/nn/layers.mojo:1681-1685: quantize x, int8
 * matmul, dequantize + bias) with per-row scales for x and per-channel scales
 * for the weights instead of two per-tensor scales.  Same arguments as
 * mj_linear_w8a16; bias may be NULL; xq and sx live in the stream's
 * workspace.  Needs K % 16 == 0, K <= 131072 (the int32 sums cannot
 * overflow) and 16-byte aligned x, Q. */
int32_t mj_linear_w8a8(const uint16_t *x, const int8_t *Q, const float *scales,
                       const float *bias, int32_t epilogue, uint16_t *y,
                       int64_t M, int64_t N, int64_t K, void *stream);

/* Llama-style FFN on W8A16 weights (composition of Linear, silu32 and the
 * elementwise product, tensor/tensor.mojo:4373):
 *   h[M,I] = bf16(silu(x Wg^T * sg) * (x Wu^T * su))   (one fused GEMM; bf16-output silu)
 *   y[M,H] = bf16((h Wd^T) * sd)
 * Wg, Wu [I,K]; Wd [H,I]; h is a caller-owned [M,I] buffer.  The gate/up
 * runs as a GEMV at 1-4 x rows (K <= 16384) and at 5-32 rows when K = 1024 j
 * <= 4096, the down projection as mj_linear_w8a16 runs [M,I] x [H,I]^T; with
 * both as GEMVs the call needs no workspace and can be captured into a HIP
 * graph. */
int32_t mj_mlp_w8a16(const uint16_t *x, const int8_t *Wg, const float *sg,
                     const int8_t *Wu, const float *su, const int8_t *Wd, const float *sd,
                     uint16_t *h, uint16_t *y, int64_t M, int64_t K, int64_t I, int64_t H,
                     void *stream);

/* ---- device memory and streams (api_host.hip) -------------------------- */
/* For a caller that keeps tensors resident across calls (e.g. QuantLinear's
 * w_q uploaded once).  momijo itself has no device-resident tensors
 * (tensor/device.mojo:258-302: to_device round-trips through the host); the
 * reference seam allocates per call with DeviceContext.enqueue_create_buffer
 * (tensor/gpu/runtime.mojo:563-570), which these replace. */

/* *ptr = device allocation of `bytes` bytes (NULL for 0). */
int32_t mj_malloc(void **ptr, int64_t bytes);
/* Frees an mj_malloc allocation (NULL is a no-op). */
int32_t mj_free(void *ptr);
/* Synchronous copies: ordered after the work queued on `stream` (NULL = the
 * null stream) and complete when they return, like the reference's
 * enqueue_copy + synchronize (runtime.mojo:586-598). */
int32_t mj_memcpy_htod(void *dst_device, const void *src_host, int64_t bytes, void *stream);
int32_t mj_memcpy_dtoh(void *dst_host, const void *src_device, int64_t bytes, void *stream);
/* Asynchronous device-to-device copy on `stream`. */
int32_t mj_memcpy_dtod(void *dst_device, const void *src_device, int64_t bytes, void *stream);
/* Non-blocking stream at the default priority; destroy NULL is a no-op.
 * The reference has no stream concept (one DeviceContext per call,
 * runtime.mojo:556). */
int32_t mj_stream_create(void **stream);
int32_t mj_stream_destroy(void *stream);
/* Waits for all work on the device (DeviceContext.synchronize,
 * runtime.mojo:596). */
int32_t mj_device_synchronize(void);

/* ---- host-pointer variants (api_host.hip) -------------------------------- */
/* Same arguments and results as the device entry point without the `_h`
 * suffix, with every pointer a HOST pointer: inputs are copied to one device
 * block, the operator runs, and outputs are copied back before the call
 * returns (the reference seam's copy-in / copy-out contract,
 * tensor/gpu/runtime.mojo:556-604).  Strided operands are copied over the
 * extent their strides span; outputs with a leading dimension are written
 * row by row, leaving padding untouched.  This is what a momijo Tensor[T],
 * whose storage is a host List[T] (tensor/tensor.mojo:776-905), binds. */

/* Tensor.matmul / tensor.matmul Float32 (tensor/tensor.mojo:3168-3169,
 * tensor/__init__.mojo:123 -> matmul_core_mm, tensor/broadcast.mojo:
 * 1612-1673), with the tensor's _strides. */
int32_t mj_matmul_f32_h(int64_t M, int64_t N, int64_t K,
                        const float *A, int64_t sAm, int64_t sAk,
                        const float *B, int64_t sBk, int64_t sBn,
                        const float *bias, int32_t epilogue, float *C, int64_t ldc);
/* Tensor.matmul_vec Float32 (tensor/tensor.mojo:3180 -> matmul_core_vec,
 * tensor/broadcast.mojo:1543-1608). */
int32_t mj_matvec_f32_h(int64_t M, int64_t N, const float *A, int64_t sAm, int64_t sAn,
                        const float *x, int64_t sx, float *y);
/* Float64 matmul / matmul2d (tensor/broadcast.mojo:1466-1538,
 * tensor/math.mojo:7838-7880). */
int32_t mj_matmul_f64_h(int64_t M, int64_t N, int64_t K,
                        const double *A, int64_t sAm, int64_t sAk,
                        const double *B, int64_t sBk, int64_t sBn, double *C, int64_t ldc);
/* Float64 matmul_core_vec (tensor/broadcast.mojo:1397-1464). */
int32_t mj_matvec_f64_h(int64_t M, int64_t N, const double *A, int64_t sAm, int64_t sAn,
                        const double *x, int64_t sx, double *y);
/* tensordot(A, B, axes=1) Float32 (tensor/broadcast.mojo:1694-1900). */
int32_t mj_tensordot_f32_h(int32_t batch_rank, const int64_t *batch_shape,
                           const int64_t *a_batch_strides, const int64_t *b_batch_strides,
                           int64_t M, int64_t N, int64_t K,
                           const float *A, int64_t sAm, int64_t sAk,
                           const float *B, int64_t sBk, int64_t sBn, float *C);
/* Linear.forward (learn/nn/layers.mojo:383-433, 510-516) + fused activation. */
int32_t mj_linear_f32_h(const float *x, const float *W, const float *bias, int32_t epilogue,
                        float *y, int64_t N, int64_t InF, int64_t OutF);
/* Linear.backward (learn/nn/layers.mojo:519-618, 785-787). */
int32_t mj_linear_backward_f32_h(const float *x, const float *W, const float *dy, float *dW,
                                 float *db, float *dx, int64_t N, int64_t InF, int64_t OutF);
/* The MATMUL2D tape rule in Float64 (tensor/autograd.mojo:1542-1555); with
 * accumulate != 0 dA / dB are read as well as written. */
int32_t mj_matmul_backward_f64_h(int64_t M, int64_t N, int64_t K, const double *A,
                                 const double *B, const double *G, double *dA, double *dB,
                                 int32_t accumulate);
/* The MATMUL2D tape rule in Float32 (tensor/autograd.mojo:1542-1555). */
int32_t mj_matmul_backward_f32_h(int64_t M, int64_t N, int64_t K, const float *A,
                                 const float *B, const float *G, float *dA, float *dB,
                                 int32_t accumulate);
/* Tensor.relu / gelu / silu (tensor/tensor.mojo:3848,4003,4020). */
int32_t mj_activation_f32_h(int32_t epilogue, const float *x, float *y, int64_t n);
/* bf16 NT GEMM (no reference counterpart; see mj_gemm_bf16_nt). */
int32_t mj_gemm_bf16_nt_h(int64_t M, int64_t N, int64_t K,
                          const uint16_t *A, int64_t lda, const uint16_t *B, int64_t ldb,
                          const float *bias, int32_t epilogue, uint16_t *C, int64_t ldc);
/* quantize_symmetric_int8 (learn/api/functional.mojo:231-247). */
int32_t mj_quantize_symmetric_int8_h(const float *x, int64_t n, float scale, int8_t *q);
/* MinMaxObserver.observe reduction (learn/api/sequential.mojo:232-250);
 * minmax_out is host float[2]. */
int32_t mj_minmax_f32_h(const float *x, int64_t n, float *minmax_out);
/* MinMaxObserver.observe + scale_symmetric (learn/api/sequential.mojo:
 * 232-263); scale_out is a host float. */
int32_t mj_minmax_scale_symmetric_h(const float *x, int64_t n, float max_q, float *scale_out);
/* matmul_i8_i8_to_i32 (learn/api/functional.mojo:249-279). */
int32_t mj_matmul_i8_i8_to_i32_h(const int8_t *A, const int8_t *B, int32_t *C,
                                 int64_t M, int64_t N, int64_t K, int32_t legacy_literal);
/* dequantize_i32_to_f32_add_bias (learn/api/functional.mojo:281-302). */
int32_t mj_dequantize_i32_to_f32_add_bias_h(const int32_t *acc, float sf, const float *b,
                                            float *y, int64_t M, int64_t N);
/* Per-channel dequantize (see mj_dequantize_i32_scaled_f32); sx and b may be
 * NULL. */
int32_t mj_dequantize_i32_scaled_f32_h(const int32_t *acc, const float *sx, const float *sw,
                                       const float *b, float *y, int64_t M, int64_t N);
/* QuantLinear.forward (learn/nn/layers.mojo:1681-1685). */
int32_t mj_quant_linear_f32_h(const float *x, const int8_t *Wq, const float *b,
                              float s_w, float s_x, float *y,
                              int64_t M, int64_t N, int64_t K, int32_t legacy_literal);
/* Per-row quantize/pack (generalises quantize_symmetric_int8 + convert,
 * learn/api/sequential.mojo:436-450). */
int32_t mj_quantize_rowwise_i8_h(const float *W, int64_t N, int64_t K, int32_t rounding,
                                 int8_t *Q, float *scales);
/* W8A16 Linear (no reference counterpart; see mj_linear_w8a16). */
int32_t mj_linear_w8a16_h(const uint16_t *x, const int8_t *Q, const float *scales,
                          const float *bias, int32_t epilogue, uint16_t *y,
                          int64_t M, int64_t N, int64_t K);
/* W8A8 Linear with dynamic activation scales (see mj_linear_w8a8). */
int32_t mj_linear_w8a8_h(const uint16_t *x, const int8_t *Q, const float *scales,
                         const float *bias, int32_t epilogue, uint16_t *y,
                         int64_t M, int64_t N, int64_t K);
/* W8A16 FFN (no reference counterpart; see mj_mlp_w8a16); h may be NULL,
 * then the intermediate stays on the device. */
int32_t mj_mlp_w8a16_h(const uint16_t *x, const int8_t *Wg, const float *sg,
                       const int8_t *Wu, const float *su, const int8_t *Wd, const float *sd,
                       uint16_t *h, uint16_t *y, int64_t M, int64_t K, int64_t I, int64_t H);

/* ---- feed-forward block --------------------------------------------------
 * Operators of a transformer's feed-forward block, forward and backward (no
 * reference counterpart; Linear, the activations and the elementwise product
 * compose them there).  Device pointers only.  Scratch memory is the caller's:
 * these calls allocate nothing, take no library workspace and can be captured
 * into a HIP graph. */
#define MJ_F32 0
#define MJ_BF16 1
#define MJ_NORM_RMS 0
#define MJ_NORM_LAYER 1

/* Dropout with a mask from a counter-based generator, never stored:
 *   y[e] = keep(e) ? x[e] * 65536 / (65536 - T) : 0
 * T = round(65536 p), at least 1 for p > 0 and at most 65535 for p < 1.  Element
 * e = 8 b + i is kept where 16-bit half i (low half of word i / 2 for even i) of
 * Philox4x32-10 of counter words (b, b >> 32, counter, counter >> 32) with key
 * `seed` is >= T.  A dropped element gives 0 whatever it holds; p = 1 drops all,
 * p = 0 copies.  The backward pass is the same call on dy.  state (or NULL): a
 * device array {seed, counter}, whose seed replaces `seed` and whose counter is
 * added to `counter`, so a captured graph can draw a new mask each replay.  x and
 * y may be the same array. */
int32_t mj_dropout(int32_t dtype, const void *x, void *y, int64_t n, float p, uint64_t seed,
                   uint64_t counter, const uint64_t *state, void *stream);

/* The norms around a residual sum, rows of `dim` (at most 16384):
 *   c = norm(b) wp + bp (c = b without wp)
 *   y = scale x + dropout(gate c)
 *   n = norm(y) wn + bn (computed from the unrounded y; with wn)
 * norm(v) = v / sqrt(mean(v^2) + eps) (MJ_NORM_RMS) or (v - mean) / sqrt(var + eps)
 * (MJ_NORM_LAYER), in fp32.  x, b, gate, y, n have element type dtype; scale, wp,
 * bp, wn, bn are fp32 [dim].  Every operand but x may be NULL (b NULL: y = scale
 * x); gate has gate_rows rows, each for rows / gate_rows rows of x.  y may be NULL, or
 * x itself where b and scale are NULL (it is not written then).
 * Dropout as mj_dropout over the [rows, dim] array.  stats (or NULL) takes what the
 * backward needs: fp32 [4][rows]. */
int32_t mj_residual_norm(int32_t dtype, int32_t norm, const void *x, const void *b,
                         const void *gate, int64_t gate_rows, const float *scale, const float *wp,
                         const float *bp, const float *wn, const float *bn, float eps, float p,
                         uint64_t seed, uint64_t counter, const uint64_t *state, void *y, void *n,
                         float *stats, int64_t rows, int64_t dim, void *stream);

/* Bytes of `work` for mj_residual_norm_backward (gate_rows 0: no gate). */
int64_t mj_residual_norm_work_bytes(int64_t rows, int64_t dim, int64_t gate_rows);

/* Gradients of mj_residual_norm from dy, dn (either may be NULL) and the forward's
 * arguments and stats.  dx, db, dgate have element type dtype; dscale, dwp, dbp,
 * dwn, dbn are fp32 [dim]; any may be NULL.  A dropped element of gate c adds nothing to
 * dgate and its dc is 0, whatever c and the gate hold.  Sums run in a fixed order: the
 * same inputs give the same bits.  rows == 0 writes nothing. */
int32_t mj_residual_norm_backward(int32_t dtype, int32_t norm, const void *x, const void *b,
                                  const void *gate, int64_t gate_rows, const float *scale,
                                  const float *wp, const float *bp, const float *wn, float p,
                                  uint64_t seed, uint64_t counter, const uint64_t *state,
                                  const float *stats, const void *dy, const void *dn, void *dx,
                                  void *db, void *dgate, float *dscale, float *dwp, float *dbp,
                                  float *dwn, float *dbn, int64_t rows, int64_t dim, void *work,
                                  int64_t work_bytes, void *stream);

/* Gated feed-forward block:
 *   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
 * x [M,K], Wg and Wu [I,K], Wd [H,I], h [M,I], y [M,H], all contiguous; act is
 * MJ_EPI_NONE, RELU, GELU_TANH or SILU.
 * bf16: K, I, H multiples of 8 (mj_copy_rows_bf16 pads other widths) below 2^22, M at most 2^31 -
 * 1024, 16-byte aligned arrays;
 * h is rounded to bf16; g, u fp32 [M,I] are written for the backward, or both NULL;
 * `work` as mj_gated_mlp_work_bytes says (NULL where that is 0).
 * fp32: any widths; h, g, u are required (u right behind g saves a launch), and `work`
 * as mj_gated_mlp_f32_work_bytes says; these and y are 16-byte aligned. */
int64_t mj_gated_mlp_work_bytes(int64_t M, int64_t K, int64_t I, int64_t H, int32_t backward);
int32_t mj_gated_mlp_bf16(const uint16_t *x, const uint16_t *Wg, const uint16_t *Wu,
                          const uint16_t *Wd, int32_t act, uint16_t *h, float *g, float *u,
                          uint16_t *y, int64_t M, int64_t K, int64_t I, int64_t H, void *work,
                          int64_t work_bytes, void *stream);
int64_t mj_gated_mlp_f32_work_bytes(int64_t M, int64_t K, int64_t I, int64_t H, int32_t backward);
int32_t mj_gated_mlp_f32(const float *x, const float *Wg, const float *Wu, const float *Wd,
                         int32_t act, float *h, float *g, float *u, float *y, int64_t M, int64_t K,
                         int64_t I, int64_t H, void *work, int64_t work_bytes, void *stream);

/* The kernel of a product of the bf16 block, by name ("" for an empty or refused one):
 * product 0 gate and up, 1 y, 2 dg and du, 3 dx, 4 dWg, dWu and dWd.  Host only; for
 * tests and profiles. */
const char *mj_gated_mlp_kernel(int64_t M, int64_t K, int64_t I, int64_t H, int32_t product);

/* Row copies between a width and its zero-padded form, n (1..4) matrices in one
 * launch: dst[i] [dst_rows, dst_cols] (rows dst_ld apart) takes src[i] [rows, cols] (rows
 * src_ld apart) and zeros where that ends; dst_rows, dst_cols below rows, cols cut.
 * bf16, any alignment; the arrays of pointers and sizes are host memory, six sizes for
 * each matrix: rows, cols, src_ld, dst_rows, dst_cols, dst_ld. */
int32_t mj_copy_rows_bf16(int32_t n, const uint16_t *const *src, uint16_t *const *dst,
                          const int64_t *sizes, void *stream);

/* Gradients of the gated block from dy [M,H] and the forward's h, g, u:
 *   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
 *   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
 * dg, du [M,I] are scratch (bf16 in the bf16 form); any of dx, dWg, dWu, dWd may be
 * NULL.  relu'(0) = 0.  `work` as the forward's, with backward = 1.  fp32: dWu
 * right behind dWg saves a launch; g, u, dg, du, dx and work are 16-byte aligned. */
int32_t mj_gated_mlp_backward_bf16(const uint16_t *x, const uint16_t *Wg, const uint16_t *Wu,
                                   const uint16_t *Wd, int32_t act, const uint16_t *h,
                                   const float *g, const float *u, const uint16_t *dy,
                                   uint16_t *dg, uint16_t *du, uint16_t *dx, uint16_t *dWg,
                                   uint16_t *dWu, uint16_t *dWd, int64_t M, int64_t K, int64_t I,
                                   int64_t H, void *work, int64_t work_bytes, void *stream);
int32_t mj_gated_mlp_backward_f32(const float *x, const float *Wg, const float *Wu, const float *Wd,
                                  int32_t act, const float *h, const float *g, const float *u,
                                  const float *dy, float *dg, float *du, float *dx, float *dWg,
                                  float *dWu, float *dWd, int64_t M, int64_t K, int64_t I,
                                  int64_t H, void *work, int64_t work_bytes, void *stream);

/* ---- mixture of experts --------------------------------------------------
 * Tokens sorted by expert and back, and the experts' gated blocks over the sorted rows (no
 * reference counterpart).  Device pointers only; these calls allocate nothing, take no
 * library workspace and can be captured into a HIP graph.  Nothing is read back: how many
 * rows an expert has stays on the device.
 *
 * `tokens` tokens with `topk` experts each are tokens * topk slots (slot t * topk + j),
 * at most 2^31 - 1024; 1 to 1024 experts. */

/* The sort: pos [slots] is each slot's row among the rows sorted by expert, in the order of
 * the slots within an expert; offsets [experts + 1] the experts' first rows.  ids [slots]
 * are int32 or int64 (id_bytes 4, 8); a slot whose id is outside 0 .. experts - 1 is dropped:
 * such slots come last, in their order, from row offsets[experts] on.  (The entry points that
 * take pos and offsets keep inside their arrays whatever these hold.) */
int64_t mj_sort_experts_work_bytes(int64_t slots, int64_t experts);
int32_t mj_sort_experts(const void *ids, int32_t id_bytes, int64_t slots, int64_t experts, int32_t *pos,
                        int32_t *offsets, void *work, int64_t work_bytes, void *stream);

/* xs[pos[t, j]] = x[t], zeros for a dropped slot: x [tokens, dim] and xs [slots, dim] of
 * dtype (MJ_F32, MJ_BF16), any alignment of the elements.  With weights [tokens, topk] their
 * sorted form goes to ws [slots] (0 for a dropped slot); both NULL: none. */
int32_t mj_dispatch(int32_t dtype, const void *x, const float *weights, const int32_t *pos,
                    const int32_t *offsets, int64_t experts, void *xs, float *ws, int64_t tokens,
                    int64_t topk, int64_t dim, void *stream);

/* y[t] = the sum over j of weights[t, j] ys[pos[t, j]] (weights NULL: ones), in fp32 in the
 * order of j; dropped slots are left out, whatever they hold.  ys is of dtype, y of y_dtype:
 * the same, or MJ_BF16 from MJ_F32.  Without weights this is mj_dispatch's gradient. */
int32_t mj_combine(int32_t dtype, int32_t y_dtype, const void *ys, const float *weights, const int32_t *pos,
                   const int32_t *offsets, int64_t experts, void *y, int64_t tokens, int64_t topk,
                   int64_t dim, void *stream);

/* mj_combine's gradients: dys[pos[t, j]] = weights[t, j] dy[t] and dw[t, j] = <dy[t],
 * ys[pos[t, j]]>, both 0 for a dropped slot. */
int32_t mj_combine_backward(int32_t dtype, const void *dy, const void *ys, const float *weights,
                            const int32_t *pos, const int32_t *offsets, int64_t experts, void *dys, float *dw,
                            int64_t tokens, int64_t topk, int64_t dim, void *stream);

/* The experts' gated blocks over R sorted rows (mj_gated_mlp_bf16 with a matrix for each
 * expert); row r of expert e:
 *   g = x Wg_e^T, u = x Wu_e^T, h = weights[r] act(g) u, y = h Wd_e^T
 * xs [R,K], Wg and Wu [experts,I,K], Wd [experts,H,I], h [R,I], ys [R,H] fp32 (a token's rows
 * are added before they are rounded), weights [R] fp32 or NULL (ones); g, u fp32 [R,I] are
 * written for the backward, or both NULL.  K, I, H multiples of 8 below 2^22, arrays 16-byte
 * aligned.  ys's rows from offsets[experts] on become zeros; h, g and u's stay as they were. */
int32_t mj_experts_mlp_bf16(const uint16_t *xs, const int32_t *offsets, int64_t experts, const uint16_t *Wg,
                            const uint16_t *Wu, const uint16_t *Wd, int32_t act, const float *weights,
                            uint16_t *h, float *g, float *u, float *ys, int64_t R, int64_t K, int64_t I,
                            int64_t H, void *stream);

/* Its gradients from dys [R,H] and the forward's h, g, u:
 *   dh = dy Wd_e, dg = weights[r] dh u act'(g), du = weights[r] dh act(g)
 *   dx = dg Wg_e + du Wu_e, dWg_e = dg^T x, dWu_e = du^T x, dWd_e = dy^T h
 *   dw[slot] = <dh, act(g) u> of row pos[slot], 0 for a dropped slot
 * dxs [R,K] is fp32, as ys.  dg, du [R,I] are scratch, and with dw dots of
 * mj_experts_mlp_dots floats; any of dxs, dWg, dWu, dWd, dw may be NULL.  An expert without
 * rows gets zeros, and so do dxs's rows from offsets[experts] on. */
int64_t mj_experts_mlp_dots(int64_t R, int64_t experts, int64_t K, int64_t I, int64_t H);
int32_t mj_experts_mlp_backward_bf16(const uint16_t *xs, const int32_t *offsets, int64_t experts,
                                     const uint16_t *Wg, const uint16_t *Wu, const uint16_t *Wd, int32_t act,
                                     const float *weights, const uint16_t *h, const float *g, const float *u,
                                     const uint16_t *dys, uint16_t *dg, uint16_t *du, float *dxs,
                                     uint16_t *dWg, uint16_t *dWu, uint16_t *dWd, const int32_t *pos,
                                     int64_t slots, float *dots, float *dw, int64_t R, int64_t K, int64_t I,
                                     int64_t H, void *stream);

/* The kernel of a product of the experts' block, by name ("" for an empty or refused one):
 * product 0 gate and up, 1 y, 2 dg and du, 3 dx, 4 the weight gradients.  Host only; for tests
 * and profiles. */
const char *mj_experts_mlp_kernel(int64_t R, int64_t experts, int64_t K, int64_t I, int64_t H, int32_t product);

/* ---- 8-bit floating point ------------------------------------------------
 * Products of e4m3 values (largest 448) with a scale for each block of 128 features of a
 * row (x) or 128 x 128 elements (W), for inference (no reference counterpart).  A block of
 * largest magnitude m is quantized with a = max(m, 2^-100): scale a * (1 / 448), values
 * e4m3(v * (448 * (1 / a))) to the nearest even, each operation rounded to fp32.  A NaN stays a
 * NaN; an infinity becomes one, with an infinite scale.  A block's sum is multiplied by its two
 * scales' product, rounded to fp32: where the blocks' largest magnitudes multiply to less than
 * 2^-108 it loses bits, and from 2^145 on it is infinite.  Widths K are multiples of 16, widths
 * below 2^22, rows at most 2^31 - 1024, arrays of values 16-byte aligned.  Scales of x lie block
 * by block, [ceil(K / 128)][rows], those of W as [ceil(N / 128)][ceil(K / 128)].  Scratch memory
 * is the caller's. */
int32_t mj_quantize_rows_f8(int32_t dtype, const void *x, uint8_t *q, float *scales, int64_t rows, int64_t K,
                            void *stream);
int32_t mj_quantize_blocks_f8(int32_t dtype, const void *W, uint8_t *q, float *scales, int64_t mats, int64_t N,
                              int64_t K, void *stream);

/* The kernel of an 8-bit product, by name ("" for an empty or refused one): of one matrix
 * (experts 0), or of sorted rows with their experts' (gate: the gated block's first half).
 * Host only; for tests and profiles. */
const char *mj_gemm_f8_kernel(int64_t M, int64_t N, int64_t K, int64_t experts, int32_t gate);

/* y [M,N] bf16 = act(x W^T + bias); the sum of a block's products is scaled and added in
 * fp32.  bias fp32 [N] or NULL; act MJ_EPI_NONE, RELU, GELU_TANH or SILU.  mj_linear_f8
 * quantizes x [M,K] of dtype first. */
int64_t mj_gemm_f8_work_bytes(int64_t M, int64_t N, int64_t K);
int32_t mj_gemm_f8(const uint8_t *xq, const float *sx, const uint8_t *Wq, const float *sw, const float *bias,
                   int32_t act, uint16_t *y, int64_t M, int64_t N, int64_t K, void *work, int64_t work_bytes,
                   void *stream);
int64_t mj_linear_f8_work_bytes(int64_t M, int64_t N, int64_t K);
int32_t mj_linear_f8(int32_t dtype, const void *x, const uint8_t *Wq, const float *sw, const float *bias,
                     int32_t act, uint16_t *y, int64_t M, int64_t N, int64_t K, void *work, int64_t work_bytes,
                     void *stream);

/* mj_dispatch of quantized rows: each token's row is quantized once and goes to its topk
 * sorted rows of q [slots,K], scales [ceil(K / 128)][slots]; zeros for a dropped slot. */
int32_t mj_dispatch_f8(int32_t dtype, const void *x, const int32_t *pos, const int32_t *offsets,
                       int64_t experts, uint8_t *q, float *scales, int64_t tokens, int64_t topk, int64_t K,
                       void *stream);

/* Sorted rows times their expert's matrix: y [R,N] fp32 = x W_e^T, zeros from row
 * offsets[experts] on.  Wq [experts,N,K], sw [experts][ceil(N / 128)][ceil(K / 128)]. */
int32_t mj_experts_gemm_f8(const uint8_t *xq, const float *sx, const int32_t *offsets, int64_t experts,
                           const uint8_t *Wq, const float *sw, float *y, int64_t R, int64_t N, int64_t K,
                           void *stream);

/* The gated block's first half: h = act(x Wg_e^T) (x Wu_e^T) in fp32, quantized to hq
 * [R,I], sh [ceil(I / 128)][R] as rows of the next product (zeros from row offsets[experts]
 * on).  I a multiple of 16. */
int64_t mj_experts_gate_f8_work_bytes(int64_t R, int64_t experts, int64_t I, int64_t K);
int32_t mj_experts_gate_f8(const uint8_t *xq, const float *sx, const int32_t *offsets, int64_t experts,
                           const uint8_t *Wg, const float *sg, const uint8_t *Wu, const float *su, int32_t act,
                           uint8_t *hq, float *sh, int64_t R, int64_t I, int64_t K, void *work,
                           int64_t work_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MOMIJO_HIP_H */
