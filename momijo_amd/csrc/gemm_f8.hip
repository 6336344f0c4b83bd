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

__device__ __forceinline__ i32x8 f8_frag(const uint16_t *stage, const int (&base)[2], int j) {
  const char *s = (const char *)stage;
  const uint4 a = *(const uint4 *)(s + base[0] + j * 2048), b = *(const uint4 *)(s + base[1] + j * 2048);
  return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
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

template <int OUT, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void f8_out(const F8Product &q, const F8Prob &p, f32x4 (&acc)[TM][TN], int m0,
                                       int n0, int wm, int wn, int lane, int split) {
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
// block's (and the up projection's).
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
    const float w = sc[NX * 64], w2 = GATE ? sc[(NX + 1) * 64] : 0.0f;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const float x = sc[wm * WM + i * 16 + fr];
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
  f8_out<OUT, TM, TN, WM, WN>(args.p, p, acc, m0, n0, wm, wn, lane, at.split);
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
// weight rows (gate/up: of each) and deals the K blocks to its waves in turn; a lane's two
// 16-byte pieces of a row's 128 are its fragment as they are.  A wave has U blocks'
// loads in flight; no LDS in the loop.  The waves' sums are added in wave order.
template <int OUT, int MB, int NW, int U, bool EX>
__global__ __launch_bounds__(NW * 64) void f8_skinny_kernel(F8Tiles args) {
  constexpr bool GATE = OUT == F8_GATE;
  constexpr int G = GATE ? 2 : 1;
  __shared__ float red[NW][G][MB][16][17];
  F8Prob p;
  int n0, row0 = 0;
  if constexpr (EX) {
    ExpertTile t;
    if (!expert_tile<false>(args.p.offsets, args.p.experts, (int)args.p.M, args.p.tail, 16 * MB, args.tiles_n,
                            blockIdx.x, t))
      return;
    f8_operands(args.p, t.expert, t.row0 + t.m * 16 * MB, t.rows - t.m * 16 * MB, p);
    n0 = t.n * 16;
  } else {
    const int tm = blockIdx.x / args.tiles_n;
    row0 = tm * 16 * MB;
    n0 = (blockIdx.x - tm * args.tiles_n) * 16;
    f8_operands(args.p, 0, row0, (int)args.p.M - row0, p);
  }
  const int lane = threadIdx.x & 63, fr = lane & 15, fh = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = p.N - n0 < 16 ? p.N - n0 : 16, K = p.K, kbs = p.kbs;
  const auto rw = make_rsrc(p.w + (size_t)n0 * K, (int64_t)rows * K);
  const auto rw2 = make_rsrc(p.w2 + (size_t)n0 * K, (int64_t)rows * K);
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
  for (int kb0 = wave; kb0 < kbs; kb0 += NW * U) {
    uint4 wv[U][G][2], xv[U][MB][2];
    float ws[U][G], xs[U][MB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * NW;
      const bool on = kb < kbs;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kb * 128 + h * 64 + fh * 16;
        const bool in = on && k < K;
        const uint32_t wo = in && fr < rows ? (uint32_t)(fr * K + k) : kOobOffset;
        wv[u][0][h] = buffer_load16(rw, wo);
        if constexpr (GATE) wv[u][1][h] = buffer_load16(rw2, wo);
#pragma unroll
        for (int b = 0; b < MB; ++b)
          xv[u][b][h] = buffer_load16(rx, in && b * 16 + fr < xr ? (uint32_t)((b * 16 + fr) * K + k) : kOobOffset);
      }
      const uint32_t so = on ? (uint32_t)kb * 4 : kOobOffset;
      ws[u][0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, so, 0, 0));
      if constexpr (GATE) ws[u][1] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs2, so, 0, 0));
#pragma unroll
      for (int b = 0; b < MB; ++b)
        xs[u][b] = on && b * 16 + fr < xr ? p.sx[(int64_t)kb * args.p.M + b * 16 + fr] : 0.0f;
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
    if (m >= p.M || n >= p.N) continue;
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

template <int OUT, int MB, int NW, int U, bool EX>
hipError_t launch_skinny(F8Tiles a, int64_t grid, hipStream_t stream) {
  if (!grid_fits(grid, NW * 64)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((f8_skinny_kernel<OUT, MB, NW, U, EX>), dim3((unsigned)grid), dim3(NW * 64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

int64_t gemm_f8_part_floats(int64_t M, int64_t N, int64_t K) { return 0; }

namespace {

// The gate and up projections have offsets.
template <int OUT>
hipError_t launch_experts(F8Tiles a, hipStream_t stream) {
  const F8Product &q = a.p;
  const int64_t groups = q.experts + q.tail, bn = OUT == F8_GATE ? 64 : 128;
  if (q.M <= 16 * std::min<int64_t>(q.M, q.experts)) {
    a.tiles_n = (int)((q.N + 15) / 16);
    return launch_skinny<OUT, 1, 8, 2, true>(a, a.tiles_n * expert_tiles_most(q.M, groups, 16), stream);
  }
  a.tiles_n = (int)((q.N + bn - 1) / bn);
  return launch_ring<128, 128, 3, OUT, true>(a, a.tiles_n * expert_tiles_most(q.M, groups, 128), stream);
}

}  // namespace

hipError_t launch_gemm_f8(const F8Product &q, hipStream_t stream) {
  if (q.M == 0 || q.N == 0) return hipSuccess;
  F8Tiles a;
  a.p = q;
  if (q.w2) return launch_experts<F8_GATE>(a, stream);
  if (q.offsets) return launch_experts<F8_ROWS>(a, stream);
  if (q.M <= 16) {
    a.tiles_n = (int)((q.N + 15) / 16);
    return launch_skinny<F8_STORE, 1, 8, 2, false>(a, a.tiles_n, stream);
  }
  a.tiles_m = (int)((q.M + 127) / 128);
  a.tiles_n = (int)((q.N + 127) / 128);
  return launch_ring<128, 128, 3, F8_STORE, false>(a, (int64_t)a.tiles_m * a.tiles_n, stream);
}

}  // namespace mj
