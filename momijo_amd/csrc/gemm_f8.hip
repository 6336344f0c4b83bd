// Products in 8-bit floating point with block scales on gfx950:
//
//   y[m, n] = sum_b sx[b, m] sw[n / 128, b] (sum of the 128 k of block b: xq[m, k] wq[n, k])
//
// The inner sum of a block is one v_mfma_f32_16x16x128_f8f6f4 (two e4m3 operands, fp32 sum,
// twice the bf16 rate); its four outputs a lane are scaled and added in fp32.  x is the
// instruction's column operand, so that a lane's outputs belong to one row of x and four
// consecutive weight rows: one scale a lane, sx sw, multiplies all of them, and the
// scaling costs an fma an output and block, half the issue slots of its MFMA.
//
// Precision: the matrix cores' 8-bit products are exact, but 8 consecutive ones are added
// as multiples of 2^-13 of the largest one's power of two (the rest cut off), and the sums
// of 8 then in fp32; both 8-bit instructions do this.  On normal data that is 1.3e-5 of y,
// without a bias, a hundredth of y's rounding to bf16 and 1/2000 of what the quantization
// loses; products of the values widened to bf16, which avoid it, have half the rate.
//
// A stage is one block of 128 k: rows of 128 bytes, the same bytes as 64 bf16, so the
// loads, the LDS layout and its swizzle are those of the bf16 tiles (mlp_tile.h, whose
// elements are pairs of values here).
#include <algorithm>
#include <atomic>

#include "expert_tile.h"
#include "fp8.h"
#include "launch.h"
#include "mlp_tile.h"

namespace mj {

namespace {

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8;

enum : int {
  F8_STORE = 0,  // y = bf16(epi(acc + bias))
  F8_PART,       // fp32 partial sums of a K slice
  F8_ROWS,       // experts: h = acc in fp32
  F8_GATE,       // experts: h = act(g) u in fp32
  F8_GATEQ,      // experts: h quantized (tiles whose columns are a block)
};

struct F8Tiles {
  F8Product p;
  int splits = 1, tiles_m = 0, tiles_n = 0;
};

// What a workgroup multiplies: rows [row0, row0 + M) of x, one matrix.
struct F8Prob {
  const uint8_t *x, *w, *w2;
  const float *sx, *sw, *sw2;
  int64_t row0;
  int M, N, K, kbs;  // K blocks; none for rows of no expert
};

__device__ __forceinline__ f32x4 mfma_f8(const i32x8 &w, const i32x8 &x) {
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, zero, 0, 0, 0, 0, 0, 0);
}

// Block j's fragment: chunks lane / 16 and 4 + lane / 16 of a row.  The restrict gives the
// reads alias information of their own, without which the compiler waits for every direct
// load into LDS in flight before them (mlp_tile.h).
__device__ __forceinline__ i32x4 f8_chunk(const char *__restrict__ p) { return *(const i32x4 *)p; }
__device__ __forceinline__ float f8_float(const float *__restrict__ p) { return *p; }

__device__ __forceinline__ i32x8 f8_frag(const uint16_t *stage, const int (&base)[2], int j) {
  const i32x4 a = f8_chunk((const char *)stage + base[0] + j * 2048);
  const i32x4 b = f8_chunk((const char *)stage + base[1] + j * 2048);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ void f8_operands(const F8Product &q, int expert, int row0, int rows, F8Prob &p) {
  const bool none = q.offsets && expert == q.experts;
  const int64_t e = none ? 0 : expert, mat = e * q.N * q.K;
  p.kbs = (int)((q.K + 127) / 128);
  const int64_t scales = e * ((q.N + 127) / 128) * p.kbs;
  if (none) p.kbs = 0;
  p.x = q.x + (int64_t)row0 * q.K;
  p.w = q.w + mat;
  p.w2 = q.w2 ? q.w2 + mat : p.w;
  p.sx = q.sx + row0;
  p.sw = q.sw + scales;
  p.sw2 = q.w2 ? q.sw2 + scales : p.sw;
  p.row0 = row0;
  p.M = rows, p.N = (int)q.N, p.K = (int)q.K;
}

// The tile's operands and place; false past the last tile.
template <bool EX, int BM>
__device__ __forceinline__ bool f8_locate(const F8Tiles &a, F8Prob &p, TileAt &at) {
  at.prob = 0, at.split = 0;
  if constexpr (EX) {
    ExpertTile t;
    if (!expert_tile<true>(a.p.offsets, a.p.experts, (int)a.p.M, a.p.tail, BM, a.tiles_n, blockIdx.x, t))
      return false;
    f8_operands(a.p, t.expert, t.row0, t.rows, p);
    at.m = t.m, at.n = t.n;
  } else {
    split_tile_coords(blockIdx.x, a.tiles_m, a.tiles_n, a.splits, 4, at.split, at.m, at.n);
    f8_operands(a.p, 0, 0, (int)a.p.M, p);
  }
  return true;
}

// y of a wave's blocks: a lane's block (i, j) holds row 16 i + (lane & 15) at columns 16 j +
// 4 (lane >> 4) + q; with N % 8 == 0 pairs of blocks are traded between lane rows for
// stores of 16 bytes.
template <int E, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void f8_store(const F8Product &q, const F8Prob &p, f32x4 (&acc)[TM][TN], int m0,
                                         int n0, int wm, int wn, int lane) {
  const int fr = lane & 15, fh = lane >> 4;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + wn * WN + j * 16 + 4 * fh;
    float b[4] = {};
    if (q.bias) {
#pragma unroll
      for (int r = 0; r < 4; ++r) b[r] = n + r < p.N ? q.bias[n + r] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = apply_epi_b16(E, acc[i][j][r] + b[r]);
  }
  uint16_t *y = q.y + p.row0 * p.N;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + fr;
    if (p.N % 8 == 0) {
#pragma unroll
      for (int j = 0; j < TN; j += 2) {
        const f32x4 &u = acc[i][j], &v = acc[i][j + 1];
        const auto a = __builtin_amdgcn_permlane16_swap(pack_bf16x2(u[0], u[1]), pack_bf16x2(v[0], v[1]),
                                                        false, false);
        const auto b = __builtin_amdgcn_permlane16_swap(pack_bf16x2(u[2], u[3]), pack_bf16x2(v[2], v[3]),
                                                        false, false);
        const int n = n0 + wn * WN + (j + (fh & 1)) * 16 + 8 * (fh >> 1);
        if (m < p.M && n < p.N)
          *(uint4 *)(y + (size_t)m * p.N + n) = make_uint4(a[0], b[0], a[1], b[1]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = n0 + wn * WN + j * 16 + 4 * fh;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m < p.M && n + r < p.N) y[(size_t)m * p.N + n + r] = (uint16_t)f32_to_bf16_bits(acc[i][j][r]);
      }
    }
  }
}

template <int TM, int TN, int WM, int WN>
__device__ __forceinline__ void f8_part(float *part, const F8Prob &p, f32x4 (&acc)[TM][TN], int m0, int n0,
                                        int wm, int wn, int lane) {
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + wn * WN + j * 16 + 4 * (lane >> 4);
      const f32x4 &v = acc[i][j];
      if (m >= p.M) continue;
      float *o = part + (size_t)m * p.N + n;
      if (p.N % 4 == 0) {
        if (n < p.N) *(float4 *)o = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < p.N) o[r] = v[r];
      }
    }
  }
}

// h = act(g) u: a wave's first half of blocks is the gate's, the second the up
// projection's (N % 16 == 0: it is the next product's K).
template <int E, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void f8_gate(const F8Product &q, const F8Prob &p, f32x4 (&acc)[TM][TN], int m0,
                                        int n0, int wm, int wn, int lane) {
  constexpr int TH = TN / 2;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < TH; ++j) {
      const int n = n0 + wn * (WN / 2) + j * 16 + 4 * (lane >> 4);
      float h[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) h[r] = apply_epi_b16(E, acc[i][j][r]) * acc[i][j + TH][r];
      if (m < p.M && n < p.N)
        *(float4 *)(q.h + (p.row0 + m) * p.N + n) = make_float4(h[0], h[1], h[2], h[3]);
    }
  }
}

// h of a tile of 128 columns, which is a block of the next product's rows: quantized from
// the accumulators, the rows' largest values of the two waves that share them traded
// through LDS.  A lane's 4 x 4 bytes of a row are traded between lane rows for one store.
template <int E, int BM, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void f8_gateq(float *lds, const F8Product &q, const F8Prob &p,
                                         f32x4 (&acc)[TM][TN], int m0, int n0, int wm, int wn, int lane) {
  static_assert(TN == 8 && WN == 128, "two waves of 64 columns");
  const int fr = lane & 15, fh = lane >> 4;
  float top[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    float a = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float h = apply_epi_b16(E, acc[i][j][r]) * acc[i][j + 4][r];
        acc[i][j][r] = h;
        a = fmaxf(a, fabsf(h));
      }
    a = fmaxf(a, __shfl_xor(a, 16, 64));
    a = fmaxf(a, __shfl_xor(a, 32, 64));
    top[i] = a;
    if (fh == 0) lds[wn * BM + wm * WM + i * 16 + fr] = a;
  }
  __syncthreads();
  const int64_t row0 = p.row0;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int ml = wm * WM + i * 16 + fr, m = m0 + ml;
    const F8Scale sc = f8_scale(fmaxf(top[i], lds[(wn ^ 1) * BM + ml]));
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = f8_pack4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], sc.inv);
    const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    const int n = n0 + wn * 64 + fh * 16;
    if (m < p.M && n < p.N)
      *(uint4 *)(q.hq + (row0 + m) * p.N + n) = make_uint4(c[0], c[1], d[0], d[1]);
    if (m < p.M && wn == 0 && fh == 0) q.sh[(int64_t)(n0 / 128) * q.M + row0 + m] = sc.scale;
  }
}

template <int OUT, int BM, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void f8_out(uint16_t *lds, const F8Product &q, const F8Prob &p,
                                       f32x4 (&acc)[TM][TN], int m0, int n0, int wm, int wn, int lane,
                                       int split) {
  if constexpr (OUT == F8_PART) {
    f8_part<TM, TN, WM, WN>(q.part + (size_t)split * p.M * p.N, p, acc, m0, n0, wm, wn, lane);
  } else if constexpr (OUT == F8_ROWS) {
    f8_part<TM, TN, WM, WN>(q.h + p.row0 * p.N, p, acc, m0, n0, wm, wn, lane);
  } else {
    switch (q.epi) {
#define MJ_OUT(E)                                                          \
  case E:                                                                  \
    if constexpr (OUT == F8_STORE)                                         \
      f8_store<E, TM, TN, WM, WN>(q, p, acc, m0, n0, wm, wn, lane);        \
    else if constexpr (OUT == F8_GATEQ)                                    \
      f8_gateq<E, BM, TM, TN, WM, WN>((float *)lds, q, p, acc, m0, n0, wm, wn, lane); \
    else                                                                   \
      f8_gate<E, TM, TN, WM, WN>(q, p, acc, m0, n0, wm, wn, lane);         \
    break;
      MJ_OUT(EPI_RELU)
      MJ_OUT(EPI_GELU_TANH)
      MJ_OUT(EPI_SILU)
      MJ_OUT(EPI_NONE)
#undef MJ_OUT
    }
  }
}

// Tiles of four waves (2 x 2) on a ring of S stages, loads S - 1 stages ahead.  A stage's
// scales come with it: wave w loads 64 floats, of the rows' scales first, then the
// block's (and the up projection's).  For few rows: 64 x 4096 x 11008 columns 17.9 us on 64 x
// 64 tiles of four stages.
template <int BM, int BN, int S, int OUT, bool EX>
__global__ __launch_bounds__(256) void f8_ring_kernel(F8Tiles args) {
  constexpr int NW = 4, WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
  constexpr bool GATE = OUT == F8_GATE;
  constexpr int BN_OUT = GATE ? BN / 2 : BN;
  using OA = Operand<BM, NW, true>;
  using OB = Operand<BN, NW, true>;
  constexpr int STAGE = OA::STAGE + OB::STAGE + 512;  // and 256 floats of scales
  constexpr int NDMA = OA::LOADS + OB::LOADS + 1, FLY = (S - 2) * NDMA;
  static_assert(S >= 3 && FLY < 64, "vmcnt range");
  constexpr int NX = BM / 64;  // waves that load row scales
  static_assert(NX + 2 <= NW, "scales of a stage");
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  F8Prob p;
  TileAt at;
  if (!f8_locate<EX, BM>(args, p, at)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1, fr = lane & 15;
  const int m0 = at.m * BM, n0 = at.n * BN_OUT;
  const int ld = p.K / 2, per = (p.kbs + args.splits - 1) / args.splits;
  const int kt0 = at.split * per, kt1 = std::min(kt0 + per, p.kbs);

  OA oa;
  oa.init(ld, wave, lane);
  OB ob;
  ob.init(ld, wave, lane);
  uint32_t aoff[OA::LOADS], boff[OB::LOADS];
#pragma unroll
  for (int i = 0; i < OA::LOADS; ++i) {
    const int r = OA::row_of(i, wave);
    aoff[i] = m0 + r + (lane >> 3) < p.M ? oa.off + (uint32_t)r * ld * 2 : kOobOffset;
  }
#pragma unroll
  for (int i = 0; i < OB::LOADS; ++i) {
    int r = OB::row_of(i, wave);
    if constexpr (GATE) r = (r / WN) * (WN / 2) + r % (WN / 2);
    boff[i] = n0 + r + (lane >> 3) < p.N ? ob.off + (uint32_t)r * ld * 2 : kOobOffset;
  }
  auto is_up = [&](int i) { return GATE && OB::row_of(i, wave) % WN >= WN / 2; };
  const auto ra = make_rsrc(p.x + (size_t)m0 * p.K, (int64_t)(p.M - m0) * p.K);
  const auto rb = make_rsrc(p.w + (size_t)n0 * p.K, (int64_t)(p.N - n0) * p.K);
  const auto rb2 = make_rsrc(p.w2 + (size_t)n0 * p.K, (int64_t)(p.N - n0) * p.K);
  // this wave's scales of stage kt: `count` floats from sp + kt * step
  const int64_t block = (int64_t)(n0 / 128) * p.kbs;
  const float *sp = wave < NX ? p.sx + m0 + wave * 64 : (wave == NX ? p.sw : p.sw2) + block;
  const int64_t step = wave < NX ? args.p.M : 1;
  const int left = p.M - m0 - wave * 64;
  const int count = wave < NX ? (left < 0 ? 0 : left > 64 ? 64 : left) : (wave == NX || (GATE && wave == NX + 1));
  auto issue = [&](int kt) __attribute__((always_inline)) {
    const int k0 = kt * kBK, Kin = kt < kt1 ? ld : 0;
    uint16_t *as = lds + (kt % S) * STAGE, *bs = as + OA::STAGE;
#pragma unroll
    for (int i = 0; i < OA::LOADS; ++i)
      dma16(ra, OA::dst(as, i, wave), k0 + oa.kc < Kin ? aoff[i] + k0 * 2 : kOobOffset);
#pragma unroll
    for (int i = 0; i < OB::LOADS; ++i) {
      const uint32_t o = k0 + ob.kc < Kin ? boff[i] + k0 * 2 : kOobOffset;
      if (is_up(i)) dma16(rb2, OB::dst(bs, i, wave), o);
      else dma16(rb, OB::dst(bs, i, wave), o);
    }
    const auto rs = make_rsrc(sp + kt * step, kt < kt1 ? count * 4 : 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void *)(bs + OB::STAGE + wave * 128), 4, lane * 4, 0, 0, 0);
  };
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  int abase[2], bbase[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    abase[ks] = OA::lane_base(wm * WM, ks, lane);
    bbase[ks] = OB::lane_base(wn * WN, ks, lane);
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s) issue(kt0 + s);
  for (int kt = kt0; kt < kt1; ++kt) {
    // stage kt has landed in every wave, and every wave holds the last stage's fragments
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070 | (FLY & 0xF) | ((FLY >> 4) << 14));
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    issue(kt + S - 1);
    const uint16_t *as = lds + (kt % S) * STAGE, *bs = as + OA::STAGE;
    const float *sc = (const float *)(bs + OB::STAGE);
    i32x8 fa[TM], fb[TN];
    float s[TM], s2[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[i] = f8_frag(as, abase, i);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = f8_frag(bs, bbase, j);
    const float w = f8_float(sc + NX * 64), w2 = GATE ? f8_float(sc + (NX + 1) * 64) : 0.0f;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const float x = f8_float(sc + wm * WM + i * 16 + fr);
      s[i] = x * w;
      s2[i] = x * w2;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const f32x4 d = mfma_f8(fb[j], fa[i]);
        const float f = GATE && j >= TN / 2 ? s2[i] : s[i];
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(d[r], f, acc[i][j][r]);
      }
  }
  // loads past the slice must not land in a later workgroup's LDS
  __builtin_amdgcn_s_waitcnt(0x0F70);
  f8_out<OUT, BM, TM, TN, WM, WN>(lds, args.p, p, acc, m0, n0, wm, wn, lane, at.split);
}

// The pipelined tiles: 256 x 256 of 8 waves (4 x 2, 64 x 128 outputs each), one workgroup a
// CU, or 128 x 128 of 4 (2 x 2, 64 x 64), two a CU; two waves a SIMD.  A wave keeps a
// stage's x fragments (32 registers) and streams the weights', 32 rows at a time and as
// many ahead.  The results of four MFMAs are in flight: before each MFMA come the fmas of
// the result that its registers held, four MFMAs old, so that neither waits for the other.
// The fmas' row scales come straight into registers (4 a lane), with a stage's loads.
//
// LDS holds two stages of x and three of weights, all 160 (80) KB.  x's buffer is free when
// every wave has its fragments, the weights' when every wave is a stage further; one
// barrier a stage, behind its first eight MFMAs, says both and that the next stage has
// landed, and the loads of the stage after next go out right behind it.
//
// Bound by the matrix cores under the power limit, and by the fmas: 8192^3 470 us (2338
// TFLOP/s; 3163 on zeros), 2048 x 4096 x 11008 columns 92 on 192 x 256 (2010).  8192 rows of 8
// experts, 4096 and 5504 wide: h 471 to 495 (1530), y 252 (1460).
template <int BM, int BN, int NW, int OUT, bool EX>
__global__ __launch_bounds__(NW * 64, 2) void f8_tile_kernel(F8Tiles args) {
  constexpr int WM = BM / (NW / 2), WN = BN / 2, TM = WM / 16, TN = WN / 16, MF = TM * TN;
  constexpr bool GATE = OUT == F8_GATE || OUT == F8_GATEQ;
  constexpr int BN_OUT = GATE ? BN / 2 : BN, WN_OUT = GATE ? WN / 2 : WN;
  using OA = Operand<BM, NW, true>;
  using OB = Operand<BN, NW, true>;
  constexpr int LOADS = OA::LOADS + OB::LOADS;
  static_assert(OB::LOADS == 4 && OA::LOADS <= 4 && LOADS <= MF - 2 * TM && TN % 4 == 0 && MF % 4 == 0, "");
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  uint16_t *As = lds, *Bs = lds + 2 * OA::STAGE;  // stage kt in buffers kt % 2, kt % 3
  F8Prob p;
  TileAt at;
  if (!f8_locate<EX, BM>(args, p, at)) return;
  const int lane = threadIdx.x & 63, fr = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int m0 = at.m * BM, n0 = at.n * BN_OUT, K = p.K, kbs = p.kbs;
  const int per = (kbs + args.splits - 1) / args.splits;
  const int kt0 = at.split * per, kt1 = std::min(kt0 + per, kbs);
  OB o;  // (both operands have rows of K bytes)
  o.init(K / 2, wave, lane);
  const int kc = o.kc * 2;  // first byte of this lane's chunk
  // Load i of x or of the weights covers tile rows (i NW + wave) 8 on, at the same offsets in
  // both; of gate/up tiles, whose rows are 8 NW of the gate's, then 8 NW of the up projection's,
  // in turn, i / 2 counts in each.  Rows past the edge lie past the resource's end and read
  // zeros, as do chunks past K.
  uint32_t off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) off[i] = o.off + (uint32_t)(OB::row_of(i, wave) * K);
  const uint8_t *px = p.x + (int64_t)m0 * K + kt0 * 128, *pw = p.w + (int64_t)n0 * K + kt0 * 128,
                *pw2 = p.w2 + (int64_t)n0 * K + kt0 * 128;
  int nx = std::min(p.M - m0, BM) * K - kt0 * 128, nw = std::min(p.N - n0, BN_OUT) * K - kt0 * 128;
  int next = kt0;  // the stage that these are at
  __amdgpu_buffer_rsrc_t rx, rw, rw2;
  bool past;
  auto load_stage = [&]() __attribute__((always_inline)) {
    const bool in = next < kt1;
    rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(px), (short)0, in ? nx : 0, 0x00020000);
    rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(pw), (short)0, in ? nw : 0, 0x00020000);
    if constexpr (GATE)
      rw2 = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(pw2), (short)0, in ? nw : 0, 0x00020000);
    past = next * 128 + kc >= K;
    ++next;
    px += 128, pw += 128, pw2 += 128, nx -= 128, nw -= 128;
  };
  auto load = [&](int abuf, int bbuf, int d) __attribute__((always_inline)) {
    const int i = d < OA::LOADS ? d : d - OA::LOADS;
    if (d < OA::LOADS)
      dma16(rx, OA::dst(As + abuf * OA::STAGE, i, wave), past ? kOobOffset : off[i]);
    else if (GATE)
      dma16(i & 1 ? rw2 : rw, OB::dst(Bs + bbuf * OB::STAGE, i, wave), past ? kOobOffset : off[i >> 1]);
    else
      dma16(rw, OB::dst(Bs + bbuf * OB::STAGE, i, wave), past ? kOobOffset : off[i]);
  };
  // the scales of stage kt
  const int nb = (n0 + wn * WN_OUT) / 128, nbs = (p.N + 127) / 128;
  const auto rsw = make_rsrc(p.sw, (int64_t)nbs * kbs * 4), rsw2 = make_rsrc(p.sw2, (int64_t)nbs * kbs * 4);
  const int rows = std::min(p.M - m0, BM);
  const float *psx = p.sx + m0 + (int64_t)kt0 * args.p.M;
  const uint32_t soff = (wm * WM + fr) * 4;
  float xs[TM], ws, ws2 = 0.0f;           // .. being loaded
  float s[TM], x[TM], up = 0.0f;          // .. of the result registers' next fmas
  auto load_scales = [&](int kt) __attribute__((always_inline)) {
    const auto rsx = make_rsrc(psx, kt < kt1 ? rows * 4 : 0);
    psx += args.p.M;
#pragma unroll
    for (int i = 0; i < TM; ++i)
      xs[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsx, soff + i * 64, 0, 0));
    const int at = kt < kt1 ? (nb * kbs + kt) * 4 : (int)kOobOffset;
    ws = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsw, at, 0, 0));
    if constexpr (GATE) ws2 = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsw2, at, 0, 0));
  };

  int abase[2], bbase[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    abase[ks] = OA::lane_base(wm * WM, ks, lane);
    bbase[ks] = OB::lane_base(wn * WN, ks, lane);
  }
  f32x4 acc[TM][TN], d[4];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    s[i] = x[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  load_scales(kt0);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    load_stage();
#pragma unroll
    for (int l = 0; l < LOADS; ++l) load(t, t, l);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70 | LOADS);  // the first stage
  asm volatile("s_barrier" ::: "memory");
  i32x8 fa[TM], fb[4];
#pragma unroll
  for (int i = 0; i < TM; ++i) {  // (in the order in which the loop reads them: its waits count on it)
    if (i < 2) fb[i] = f8_frag(Bs, bbase, i);
    __builtin_amdgcn_sched_barrier(0);
    fa[i] = f8_frag(As, abase, i);
    __builtin_amdgcn_sched_barrier(0);
  }

  // MFMA m of a stage: two blocks of weight rows at a time, x block by x block
  auto block_i = [](int m) constexpr { return m % (2 * TM) / 2; };
  auto block_j = [](int m) constexpr { return m / (2 * TM) * 2 + m % 2; };
  auto scale = [&](int m) __attribute__((always_inline)) {  // and add result m
    f32x4 &c = acc[block_i(m)][block_j(m)];
#pragma unroll
    for (int r = 0; r < 4; ++r) c[r] = __builtin_fmaf(d[m & 3][r], s[block_i(m)], c[r]);
  };
  int ab = 0, bb = 0;
  for (int kt = kt0; kt < kt1; ++kt) {
    const int bn = bb == 2 ? 0 : bb + 1, bl = bn == 2 ? 0 : bn + 1;
    const uint16_t *an = As + (ab ^ 1) * OA::STAGE, *bs = Bs + bb * OB::STAGE, *bsn = Bs + bn * OB::STAGE;
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const int pair = m / (2 * TM), w = m % (2 * TM);
      __builtin_amdgcn_sched_barrier(0);
      scale((m + MF - 4) % MF);
      __builtin_amdgcn_sched_barrier(0);
      d[m & 3] = mfma_f8(fb[(pair & 1) * 2 + (m & 1)], fa[block_i(m)]);
      __builtin_amdgcn_sched_barrier(0);
      // the next pair's fragments, and behind their last use the next stage's of x
      if (w == 0 || w == 2) {
        const int j = 2 * pair + 2 + w / 2;
        fb[(~pair & 1) * 2 + w / 2] = j < TN ? f8_frag(bs, bbase, j) : f8_frag(bsn, bbase, j - TN);
      }
      if (m >= MF - 2 * TM && (m & 1)) fa[block_i(m)] = f8_frag(an, abase, block_i(m));
      if (m == 3) {  // results of this stage follow
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if constexpr (GATE) x[i] = xs[i];
          s[i] = xs[i] * ws;
        }
        if constexpr (GATE) up = ws2;
      }
      if constexpr (GATE) {
        if (m == MF / 2 + 3) {  // .. and of the up projection
#pragma unroll
          for (int i = 0; i < TM; ++i) s[i] = x[i] * up;
        }
      }
      if (m == 2 * TM - 1) {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // stage kt + 1
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        load_scales(kt + 1);
        load_stage();  // kt + 2
      }
      if (m >= 2 * TM && m < 2 * TM + LOADS) load(ab, bl, m - 2 * TM);
    }
    ab ^= 1, bb = bn;
  }
#pragma unroll
  for (int m = MF - 4; m < MF; ++m) scale(m);
  // loads past the slice must not land in what follows in LDS
  __builtin_amdgcn_s_waitcnt(0x0F70);
  if constexpr (OUT == F8_GATEQ) __syncthreads();
  f8_out<OUT, BM, TM, TN, WM, WN>(lds, args.p, p, acc, m0, n0, wm, wn, lane, at.split);
}

// y = bf16(epi(sum of the K slices' partials + bias)), in slice order.
__global__ __launch_bounds__(256) void f8_sum_kernel(F8Product q, int splits) {
  const int64_t n = q.M * q.N, e = (grid_block<256>() * 256 + threadIdx.x) * 4;
  float v[4] = {};
  if (n % 4 == 0) {
    if (e >= n) return;
    for (int s = 0; s < splits; ++s) {
      const float4 a = *(const float4 *)(q.part + s * n + e);
      v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
    }
  } else {
    for (int s = 0; s < splits; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e + i < n) v[i] += q.part[s * n + e + i];
  }
  int64_t c = e % q.N;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (q.bias && e + i < n) v[i] += q.bias[c];
    v[i] = apply_epi_b16(q.epi, v[i]);
    if (++c == q.N) c = 0;
  }
  if (n % 4 == 0) {
    *(uint2 *)(q.y + e) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e + i < n) q.y[e + i] = (uint16_t)f32_to_bf16_bits(v[i]);
  }
}

// ---------------------------------------------------------------- few rows
// At most 16 MB rows: bound by reading the weights once.  A workgroup of NW waves owns 16
// weight rows (gate/up: of each) and deals the K blocks to its waves in turn; a lane's 32
// bytes of a row's 128 are its fragment as they are.  A wave has U blocks' loads in
// flight.  The waves' sums are added in wave order.  One row, 4096 x 11008 columns, x quantized
// in it: 11.8 us (3.8 TB/s) where the weights come from memory, 8.8 (5.1) where the last-level
// cache holds them, launch behind launch; 96 rows of 8 experts, 4096 and 11008 wide: h 158 (4.6), y
// 90 (4.0).
//
// XT: x comes quantized (X_F8), or in its own type: then each workgroup quantizes it into
// LDS (32 lanes a block) while its first weights are on their way, which saves a launch.
enum : int { X_F8 = 0, X_BF16, X_F32 };

// LDS for M quantized rows of K and their scales.
constexpr int64_t few_rows_lds(int64_t M, int64_t K) { return M * ((K + 127) / 128) * 132; }

// Four values of a block of a row; item i is block i % kbs of row i / kbs.
template <int XT>
struct FourOf {
  uint4 w;  // (bf16: two of it)
  __device__ __forceinline__ void load(const void *x, int i, int items, int K, int kbs) {
    const int m = i / kbs, k = (i - m * kbs) * 128 + (threadIdx.x & 31) * 4;
    w = make_uint4(0, 0, 0, 0);
    if (i >= items || k >= K) return;
    if constexpr (XT == X_BF16) {
      const uint2 v = *(const uint2 *)((const uint16_t *)x + (int64_t)m * K + k);
      w.x = v.x, w.y = v.y;
    } else {
      w = *(const uint4 *)((const float *)x + (int64_t)m * K + k);
    }
  }
  __device__ __forceinline__ void quantize(int i, int items, char *q, float *scales) const {
    const int l = threadIdx.x & 31;
    float v[4];
    if constexpr (XT == X_BF16) {
      v[0] = __uint_as_float(w.x << 16), v[1] = __uint_as_float(w.x & 0xFFFF0000u);
      v[2] = __uint_as_float(w.y << 16), v[3] = __uint_as_float(w.y & 0xFFFF0000u);
    } else {
      v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y);
      v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    }
    float a = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    a = f8_max16(a);
    a = fmaxf(a, __shfl_xor(a, 16, 64));
    const F8Scale s = f8_scale(a);
    if (i >= items) return;
    *(uint32_t *)(q + i * 128 + l * 4) = f8_pack4(v[0], v[1], v[2], v[3], s.inv);
    if (l == 0) scales[i] = s.scale;
  }
};

// Weight rows of a workgroup (gate/up: of each).  With 32 rows of x, 32 weight rows: with 16 it
// reads up to twice as much of x from L2 as of the weights from memory (96 rows of 8 experts,
// 11008 features, 4096 columns: 90 us, 99 with 16).
constexpr int skinny_cols(int out, int mb) { return out == F8_ROWS && mb == 2 ? 32 : 16; }

template <int OUT, int MB, int NW, int U, bool EX, int XT>
__global__ __launch_bounds__(NW * 64) void f8_skinny_kernel(F8Tiles args) {
  constexpr bool GATE = OUT == F8_GATE;
  constexpr int COLS = skinny_cols(OUT, MB), G = GATE ? 2 : COLS / 16;
  static_assert(XT == X_F8 || (MB == 1 && !EX), "rows in LDS");
  __shared__ float red[NW][G][MB][16][17];
  extern __shared__ __attribute__((aligned(16))) char xlds[];
  F8Prob p;
  int n0;
  if constexpr (EX) {
    ExpertTile t;
    const int bid = (int)grid_block<NW * 64>();  // (below 2^30: 2^18 column tiles of 2048 segments)
    if (!expert_tile<false>(args.p.offsets, args.p.experts, (int)args.p.M, args.p.tail, 16 * MB, args.tiles_n,
                            bid, t))
      return;
    f8_operands(args.p, t.expert, t.row0 + t.m * 16 * MB, t.rows - t.m * 16 * MB, p);
    n0 = t.n * COLS;
  } else {
    f8_operands(args.p, 0, 0, (int)args.p.M, p);
    n0 = blockIdx.x * COLS;
  }
  const int lane = threadIdx.x & 63, fr = lane & 15, fh = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = p.N - n0 < 16 ? p.N - n0 : 16, K = p.K, kbs = p.kbs;
  // (the second 16: the up projection's, or the next ones)
  const int rows2 = GATE ? rows : std::min(std::max(p.N - n0 - 16, 0), 16);
  const auto rw = make_rsrc(p.w + (size_t)n0 * K, (int64_t)rows * K);
  const auto rw2 = make_rsrc(GATE ? p.w2 + (size_t)n0 * K : p.w + (size_t)(n0 + 16) * K, (int64_t)rows2 * K);
  const int xr = p.M < 16 * MB ? p.M : 16 * MB;
  const auto rx = make_rsrc(p.x, (int64_t)xr * K);
  const int64_t block = (int64_t)(n0 / 128) * kbs;
  const auto rs = make_rsrc(p.sw + block, kbs * 4);
  const auto rs2 = make_rsrc(p.sw2 + block, kbs * 4);
  f32x4 acc[G][MB];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[g][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  uint4 wv[U][G][2], xv[U][MB][2];
  float ws[U][G], xs[U][MB];
  auto load = [&](int kb0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * NW;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kb * 128 + fh * 32 + h * 16;
        const uint32_t wo = k < K && fr < rows ? (uint32_t)(fr * K + k) : kOobOffset;
        wv[u][0][h] = buffer_load16(rw, wo);
        if constexpr (G == 2)
          wv[u][1][h] = buffer_load16(rw2, k < K && fr < rows2 ? (uint32_t)(fr * K + k) : kOobOffset);
        if constexpr (XT == X_F8) {
#pragma unroll
          for (int b = 0; b < MB; ++b)
            xv[u][b][h] = buffer_load16(rx, k < K && b * 16 + fr < xr ? (uint32_t)((b * 16 + fr) * K + k) : kOobOffset);
        }
      }
      const uint32_t so = kb < kbs ? (uint32_t)kb * 4 : kOobOffset;
      ws[u][0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, so, 0, 0));
      if constexpr (GATE) ws[u][1] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs2, so, 0, 0));
      else if constexpr (G == 2) ws[u][1] = ws[u][0];  // (32 columns from a multiple of 32: one block)
      if constexpr (XT == X_F8) {
#pragma unroll
        for (int b = 0; b < MB; ++b)
          xs[u][b] = kb < kbs && b * 16 + fr < xr ? p.sx[(int64_t)kb * args.p.M + b * 16 + fr] : 0.0f;
      }
    }
  };
  float *xscale = (float *)(xlds + (int64_t)xr * kbs * 128);
  if constexpr (XT != X_F8) {
    // (x's loads go out before the weights': waiting for them does not wait for those)
    constexpr int PRE = 3, STEP = NW * 2;
    const int items = xr * kbs, i0 = threadIdx.x >> 5;
    FourOf<XT> four[PRE];
#pragma unroll
    for (int j = 0; j < PRE; ++j) four[j].load(args.p.xf, i0 + j * STEP, items, K, kbs);
    __builtin_amdgcn_sched_barrier(0);
    load(wave);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < PRE; ++j)
      if (j == 0 || j * STEP < items) four[j].quantize(i0 + j * STEP, items, xlds, xscale);
    for (int i = PRE * STEP; i < items; i += STEP) {
      four[0].load(args.p.xf, i0 + i, items, K, kbs);
      four[0].quantize(i0 + i, items, xlds, xscale);
    }
    __syncthreads();
  } else {
    load(wave);
  }
  for (int kb0 = wave; kb0 < kbs; kb0 += NW * U) {
    if constexpr (XT != X_F8) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = fr * kbs + kb0 + u * NW;
        const bool on = kb0 + u * NW < kbs && fr < xr;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        xv[u][0][0] = on ? *(const uint4 *)(xlds + at * 128 + fh * 32) : zero;
        xv[u][0][1] = on ? *(const uint4 *)(xlds + at * 128 + fh * 32 + 16) : zero;
        xs[u][0] = on ? xscale[at] : 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          auto frag = [](const uint4 (&v)[2]) {
            return i32x8{(int)v[0].x, (int)v[0].y, (int)v[0].z, (int)v[0].w,
                         (int)v[1].x, (int)v[1].y, (int)v[1].z, (int)v[1].w};
          };
          const f32x4 d = mfma_f8(frag(wv[u][g]), frag(xv[u][b]));
          const float s = xs[u][b] * ws[u][g];
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[g][b][r] = __builtin_fmaf(d[r], s, acc[g][b][r]);
        }
    if (kb0 + NW * U < kbs) load(kb0 + NW * U);
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[wave][g][b][fr][4 * fh + r] = acc[g][b][r];
  __syncthreads();
  for (int e = threadIdx.x; e < MB * 256; e += NW * 64) {
    const int b = e >> 8, r = (e >> 4) & 15, c = e & 15, m = b * 16 + r, n = n0 + c;
    if (m >= p.M || n >= p.N) continue;  // (N ends the second 16 in the store)
    float v[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      v[g] = red[0][g][b][r][c];
#pragma unroll
      for (int w = 1; w < NW; ++w) v[g] += red[w][g][b][r][c];
    }
    const size_t o = (size_t)(p.row0 + m) * p.N + n;
    if constexpr (GATE) {
      args.p.h[o] = apply_epi_b16(args.p.epi, v[0]) * v[1];
    } else if constexpr (OUT == F8_ROWS) {
      args.p.h[o] = v[0];
      if (G == 2 && n + 16 < p.N) args.p.h[o + 16] = v[G - 1];
    } else {
      const float y = v[0] + (args.p.bias ? args.p.bias[n] : 0.0f);
      args.p.y[o] = (uint16_t)f32_to_bf16_bits(apply_epi_b16(args.p.epi, y));
    }
  }
}

// ---------------------------------------------------------------- launch
template <int BM, int BN, int S, int OUT, bool EX>
hipError_t launch_ring(F8Tiles a, int64_t grid, hipStream_t stream) {
  constexpr size_t lds = size_t(S) * ((BM + BN) * 128 + 1024);
  static_assert(lds <= 160 * 1024, "LDS budget");
  auto kern = f8_ring_kernel<BM, BN, S, OUT, EX>;
  static std::atomic<uint64_t> done{0};
  if (hipError_t e = raise_lds((const void *)kern, lds, done); e != hipSuccess) return e;
  if (!grid_fits(grid, 256)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <int BM, int BN, int NW, int OUT, bool EX>
hipError_t launch_pipe(F8Tiles a, int64_t grid, hipStream_t stream) {
  constexpr size_t lds = size_t(2 * BM + 3 * BN) * 128;  // 160, 144 or 80 KB
  auto kern = f8_tile_kernel<BM, BN, NW, OUT, EX>;
  static std::atomic<uint64_t> done{0};
  if (hipError_t e = raise_lds((const void *)kern, lds, done); e != hipSuccess) return e;
  if (!grid_fits(grid, NW * 64)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(NW * 64), lds, stream, a);
  return hipGetLastError();
}

template <int OUT, int MB, int NW, int U, bool EX, int XT>
hipError_t launch_skinny(const F8Tiles &a, int64_t grid, hipStream_t stream) {
  const size_t lds = XT == X_F8 ? 0 : few_rows_lds(a.p.M, a.p.K);
  hipLaunchKernelGGL((f8_skinny_kernel<OUT, MB, NW, U, EX, XT>), grid_rows<NW * 64>(grid), dim3(NW * 64), lds, stream,
                     a);
  return hipGetLastError();
}

// At most 16 rows.  The number of waves orders the sums, so it goes by the sizes alone and a
// product has the same bits whether x was quantized before or by the workgroups.  Those
// (where gemm_f8_quantizes says) hold one block in flight, on 16 waves where there is much to
// quantize or K is long (one row, K = 11008, 4096 columns: 14.1 us, 17.1 on 8; K = 4096, 11008
// columns: 12.7 and 11.8).  With x quantized before: as many blocks in flight as a wave has, up to three (16
// rows, us of both launches with 8 waves and one block, 16 and two, 16 and three: K = 1040,
// 3000 columns 5.1, 5.7, 6.2; 4096, 11008 17.4, 16.8, -; 11008, 4096 18.2, 17.8, 17.6).
template <int XT>
hipError_t launch_16_rows(const F8Tiles &a, hipStream_t stream) {
  const int64_t kbs = (a.p.K + 127) / 128;
  const bool fuses = gemm_f8_quantizes(a.p.M, a.p.N, a.p.K);
  const bool wide = fuses ? kbs > 32 || a.p.M * kbs >= 64 : kbs > 16;
  if constexpr (XT != X_F8) {
    if (wide) return launch_skinny<F8_STORE, 1, 16, 1, false, XT>(a, a.tiles_n, stream);
    return launch_skinny<F8_STORE, 1, 8, 1, false, XT>(a, a.tiles_n, stream);
  } else {
    if (wide && kbs > 32) return launch_skinny<F8_STORE, 1, 16, 3, false, XT>(a, a.tiles_n, stream);
    if (wide) return launch_skinny<F8_STORE, 1, 16, 2, false, XT>(a, a.tiles_n, stream);
    if (kbs > 8) return launch_skinny<F8_STORE, 1, 8, 2, false, XT>(a, a.tiles_n, stream);
    return launch_skinny<F8_STORE, 1, 8, 1, false, XT>(a, a.tiles_n, stream);
  }
}

// The tiles (h: half the columns) and their times on MI355X (us), as in mlp_tile.h: rounds of the
// workgroups that the CUs hold, each the stages (of one block of K) at the time of a stage
// with 1 or 2 workgroups a CU, and a fixed part; a round that leaves CUs idle runs a
// little faster.  Fits to products of 64 to 4096 rows, e.g. 2048 x 4096 x 11008 columns: 256 x
// 256 111, 192 x 256 98, 128 x 128 115, 64 x 64 201; 512 rows 54, 47, 43, 59; 64 rows (64 x
// 64) 17.9; 1000 x 1040 x 3000 19.0, 16.2, 11.1, 15.8.
enum : int { F8_256 = 0, F8_192, F8_128, F8_64, F8_COUNT };
struct F8Cost {
  int rows, cols, threads, per_cu;
  double stage[2], fixed;
};
constexpr F8Cost kF8Cost[F8_COUNT] = {
    {256, 256, 512, 1, {1.65, 0}, 2.5},
    {192, 256, 512, 1, {1.40, 0}, 2.0},
    {128, 128, 256, 2, {0.95, 1.15}, 1.0},
    {64, 64, 256, 2, {0.465, 0.56}, 0.8},
};

double f8_time_us(const F8Cost &c, double wgs, double stages) {
  const int64_t slots = kCUs * c.per_cu, n = (int64_t)(wgs + 0.5), rest = n % slots;
  double us = 2.0 + (double)(n / slots) * (c.fixed + stages * c.stage[c.per_cu - 1]);
  if (rest)
    us += c.fixed + stages * c.stage[(rest + kCUs - 1) / kCUs - 1] * (0.7 + 0.3 * (double)rest / (double)slots);
  return us;
}

template <int OUT, bool EX>
hipError_t launch_tiles(int tile, const F8Tiles &a, int64_t grid, hipStream_t stream) {
  switch (tile) {
    case F8_256: return launch_pipe<256, 256, 8, OUT, EX>(a, grid, stream);
    case F8_192: return launch_pipe<192, 256, 8, OUT, EX>(a, grid, stream);
    case F8_128: return launch_pipe<128, 128, 4, OUT, EX>(a, grid, stream);
    default: return launch_ring<64, 64, 4, OUT, EX>(a, grid, stream);
  }
}

// ---- one matrix
struct F8Plan {
  int tile = F8_64, splits = 1;
};

// K slices where tiles leave CUs idle: their partials are written and read once (mostly by the
// caches), by one more launch.  48 x 11008 x 4096: 64 x 64 tiles 40.9 us whole, 20.9 in four
// slices; 1024 rows 83 on 256 x 256, 63 in four; 2048 rows 129, 97 in two.
F8Plan plan_f8(int64_t M, int64_t N, int64_t K) {
  F8Plan best;
  double best_us = 1e30;
  const int64_t kbs = (K + 127) / 128;
  for (int t = 0; t < F8_COUNT; ++t) {
    const F8Cost &c = kF8Cost[t];
    const int64_t tiles = ((M + c.rows - 1) / c.rows) * ((N + c.cols - 1) / c.cols);
    for (int s = 1; s <= 8; ++s) {
      if (s > 1 && (kbs / s < 4 || tiles * s > 2 * kCUs * c.per_cu)) break;
      if (!grid_fits(tiles * s, c.threads)) break;
      double us = f8_time_us(c, (double)(tiles * s), (double)((kbs + s - 1) / s));
      if (s > 1) us += 2.2 + (8.0 * s + 2.0) * (double)M * (double)N / 7.0e6;
      if (us < best_us) best_us = us, best.tile = t, best.splits = s;
    }
  }
  return best;
}

// Rows of the few-row kernel: 16, and up to 64 where the weights are small and latency counts
// (x is read again for every 16 weight rows): 64 x 1040 x 3000 4.7 us, 7.1 on tiles; 64 x 1024 x
// 1024 4.3 and 6.5; but 48 x 4096 x 4096 19 and 12.
bool f8_few_rows(int64_t M, int64_t N, int64_t K) { return M <= 16 || (M <= 64 && N * K <= 8000000); }

// ---- experts
// The tiles to expect, as experts_mlp.hip does.
double likely_tiles(const F8Product &q, int64_t bm) {
  const double b = (double)std::min<int64_t>(q.M, q.experts), per = (double)q.M / b;
  if (per >= (double)bm) return (double)q.M / (double)bm + b / 2;
  return b * (1.0 + std::max(0.0, (1.6 * per - (double)bm) / (1.2 * per)));
}

// Rows of one expert, if they are even, up to which the few-row kernel is taken.
bool few_rows(const F8Product &q) { return q.M <= 16 * std::min<int64_t>(q.M, q.experts); }

// The gate's tiles of 256 columns quantize h; others leave it in fp32, to be written, read and
// quantized by one more launch.
int plan_experts(const F8Product &q, bool gate) {
  int best = F8_64;
  double best_us = 1e30;
  const double kbs = (double)((q.K + 127) / 128);
  for (int t = 0; t < F8_COUNT; ++t) {
    const F8Cost &c = kF8Cost[t];
    const int64_t cols = gate ? c.cols / 2 : c.cols, tn = (q.N + cols - 1) / cols;
    if (!grid_fits(tn * expert_tiles_most(q.M, q.experts + 1, c.rows), c.threads)) continue;
    double us = f8_time_us(c, (double)tn * likely_tiles(q, c.rows), kbs);
    if (gate && c.cols != 256) us += 3.0 + 8.0 * (double)q.M * (double)q.N / 5.0e6;
    if (us < best_us) best_us = us, best = t;
  }
  return best;
}

// Few rows an expert: segments of 32 rows where 16 would often split an expert (and read its
// weights twice): 96 rows of 8 experts, 4096 and 11008 wide, gate and up 156 us, 162 with 16;
// more waves or blocks in flight were slower (16 waves 186, two blocks 176).
template <int OUT>
hipError_t launch_few_rows(F8Tiles &a, hipStream_t stream) {
  const F8Product &q = a.p;
  const int64_t groups = q.experts + q.tail;
  const bool two = q.M > 8 * std::min<int64_t>(q.M, q.experts);
  const int cols = skinny_cols(OUT, two ? 2 : 1);
  a.tiles_n = (int)((q.N + cols - 1) / cols);
  if (two)
    return launch_skinny<OUT, 2, 8, 1, true, X_F8>(a, a.tiles_n * expert_tiles_most(q.M, groups, 32), stream);
  return launch_skinny<OUT, 1, 8, 1, true, X_F8>(a, a.tiles_n * expert_tiles_most(q.M, groups, 16), stream);
}

hipError_t launch_gate(F8Tiles &a, hipStream_t stream) {
  const F8Product &q = a.p;
  if (few_rows(q)) return launch_few_rows<F8_GATE>(a, stream);
  const int tile = plan_experts(q, true), cols = kF8Cost[tile].cols / 2;
  a.tiles_n = (int)((q.N + cols - 1) / cols);
  const int64_t grid = a.tiles_n * expert_tiles_most(q.M, q.experts + q.tail, kF8Cost[tile].rows);
  switch (tile) {
    case F8_256: return launch_pipe<256, 256, 8, F8_GATEQ, true>(a, grid, stream);
    case F8_192: return launch_pipe<192, 256, 8, F8_GATEQ, true>(a, grid, stream);
    case F8_128: return launch_pipe<128, 128, 4, F8_GATE, true>(a, grid, stream);
    default: return launch_ring<64, 64, 4, F8_GATE, true>(a, grid, stream);
  }
}

hipError_t launch_rows(F8Tiles &a, hipStream_t stream) {
  const F8Product &q = a.p;
  if (few_rows(q)) return launch_few_rows<F8_ROWS>(a, stream);
  const int tile = plan_experts(q, false), cols = kF8Cost[tile].cols;
  a.tiles_n = (int)((q.N + cols - 1) / cols);
  return launch_tiles<F8_ROWS, true>(
      tile, a, a.tiles_n * expert_tiles_most(q.M, q.experts + q.tail, kF8Cost[tile].rows), stream);
}

}  // namespace

bool gemm_f8_fuses(const F8Product &q) {
  return q.w2 && !few_rows(q) && kF8Cost[plan_experts(q, true)].cols == 256;
}

// Every workgroup of the few-row kernel quantizes all of x, which a launch of its own (1.7 us
// between others) does once: few blocks, fewer where a CU has several workgroups.  K =
// 4096, 11008 columns, one row 11.8 us, 12.8 with that launch, 4 rows 15.4 and 14.1; 4096, 4096 4
// rows 7.7 and 8.1, 8 rows 10.1 and 8.3; 1040, 3000 8 rows 4.1 and 5.0, 16 rows 5.4 and 5.1.
constexpr int64_t kQuantizeBlocks = 192;
static_assert(few_rows_lds(1, 128 * kQuantizeBlocks) + sizeof(float) * 16 * 16 * 17 <= 64 * 1024,
              "x's blocks and the sums of 16 waves");
bool gemm_f8_quantizes(int64_t M, int64_t N, int64_t K) {
  return M <= 16 && N > 0 && M * ((K + 127) / 128) * ((N + 4095) / 4096) <= kQuantizeBlocks;
}

int64_t gemm_f8_part_floats(int64_t M, int64_t N, int64_t K) {
  if (f8_few_rows(M, N, K)) return 0;
  const int s = plan_f8(M, N, K).splits;
  return s > 1 ? s * M * N : 0;
}

const char *gemm_f8_kernel_name(const F8Product &q) {
  static const char *const names[F8_COUNT][2] = {{"256x256", "256x256, K slices"},
                                                 {"192x256", "192x256, K slices"},
                                                 {"128x128", "128x128, K slices"},
                                                 {"64x64", "64x64, K slices"}};
  if (q.offsets || q.w2) {
    if (few_rows(q)) return q.M > 8 * std::min<int64_t>(q.M, q.experts) ? "32 rows" : "16 rows";
    return names[plan_experts(q, q.w2 != nullptr)][0];
  }
  if (f8_few_rows(q.M, q.N, q.K))
    return q.M > 32 ? "64 rows" : q.M > 16 ? "32 rows" : gemm_f8_quantizes(q.M, q.N, q.K) ? "16 rows, quantizing" : "16 rows";
  const F8Plan pl = plan_f8(q.M, q.N, q.K);
  return names[pl.tile][pl.splits > 1];
}

hipError_t launch_gemm_f8(const F8Product &q, hipStream_t stream) {
  if (q.M == 0 || q.N == 0) return hipSuccess;
  F8Tiles a;
  a.p = q;
  if (q.w2) return launch_gate(a, stream);
  if (q.offsets) return launch_rows(a, stream);
  if (f8_few_rows(q.M, q.N, q.K)) {
    a.tiles_n = (int)((q.N + 15) / 16);
    if (q.xf && q.xf_bf16) return launch_16_rows<X_BF16>(a, stream);
    if (q.xf) return launch_16_rows<X_F32>(a, stream);
    if (q.M <= 16) return launch_16_rows<X_F8>(a, stream);
    if (q.M <= 32) return launch_skinny<F8_STORE, 2, 8, 1, false, X_F8>(a, a.tiles_n, stream);
    return launch_skinny<F8_STORE, 4, 8, 1, false, X_F8>(a, a.tiles_n, stream);
  }
  const F8Plan pl = plan_f8(q.M, q.N, q.K);
  const F8Cost &c = kF8Cost[pl.tile];
  a.tiles_m = (int)((q.M + c.rows - 1) / c.rows);
  a.tiles_n = (int)((q.N + c.cols - 1) / c.cols);
  a.splits = pl.splits;
  const int64_t grid = (int64_t)a.tiles_m * a.tiles_n * a.splits;
  if (a.splits == 1) return launch_tiles<F8_STORE, false>(pl.tile, a, grid, stream);
  if (!q.part) return hipErrorInvalidValue;
  if (hipError_t e = launch_tiles<F8_PART, false>(pl.tile, a, grid, stream); e != hipSuccess) return e;
  const int64_t n = q.M * q.N;
  hipLaunchKernelGGL(f8_sum_kernel, grid_rows<256>((n + 1023) / 1024), dim3(256), 0, stream, q, a.splits);
  return hipGetLastError();
}

}  // namespace mj
