// Gated feed-forward block on gfx950 bf16 MFMA, forward and backward:
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Every product is one kernel family over tiles of C[m, n] = sum_k A(m, k) B(n, k):
//  * each operand is either K-contiguous ([rows][k], as x and W in x W^T) or
//    K-strided ([k][rows]: W in dy W, both operands of dg^T x), so no matrix is
//    ever transposed in memory.  A K-contiguous stage lies in LDS as rows of 64 k;
//    a K-strided one as 64 rows of k, whose fragments are read with
//    ds_read_b64_tr_b16, which hands each lane four k of one column;
//  * the gate and up projections share one tile: half its B rows are Wg's, half
//    the same rows of Wu, so a lane holds g and u of the same outputs and writes h
//    (and g, u in fp32 for the backward) without another pass;
//  * dh never reaches memory: its tile's epilogue reads g and u and writes dg, du;
//  * dx sums two products in one accumulator (two K segments), and the three weight
//    gradients run as one launch.
//
// Roundings to bf16: h, dg, du (they feed the next product's matrix cores) and the
// outputs; g and u are kept in fp32, so that act and act' see unrounded inputs and
// every gradient carries one rounding of an operand and one of its own.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.h"
#include "gemm_tile.h"
#include "launch.h"
#include "philox.h"

namespace mj {

typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

namespace {

// What a tile's accumulators become.
enum : int {
  OUT_STORE = 0,  // C = bf16(acc)
  OUT_PART,       // fp32 partial sums of a K slice
  OUT_GATE,       // h = act(g) u, optionally g and u in fp32
  OUT_DGATE,      // dg, du from dh = acc and the stored g, u
};

struct TileProb {
  const uint16_t *A[2] = {nullptr, nullptr}, *B[2] = {nullptr, nullptr};  // K segments; gate/up: B[1] = Wu
  int64_t lda = 0, ldb = 0;
  int M = 0, N = 0, K = 0, segs = 1;  // K of one segment
  int tiles_m = 0, tiles_n = 0, first = 0;
  uint16_t *C = nullptr, *C2 = nullptr;  // C2: du
  float *F = nullptr, *F2 = nullptr;     // g, u
  float *part = nullptr;
  int64_t ldc = 0;                       // of C, C2, F, F2
};

struct TileArgs {
  TileProb p[3];
  int n = 1, tiles = 0, splits = 1, act = 0;
};

// act(g) and act'(g) (1 + 1e-6 relative, as silu_b16: the results are rounded to bf16).
// Where the sigmoid saturates its derivative's term is 0, not 0 x overflow.
__device__ __forceinline__ float act_b16(int act, float g) { return apply_epi_b16(act, g); }

__device__ __forceinline__ float2 act_grad_b16(int act, float g) {
  if (act == EPI_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g));
    const float t = s * (1.0f - s);
    return make_float2(g * s, s + (t == 0.0f ? 0.0f : g * t));
  }
  if (act == EPI_GELU_TANH) {
    constexpr float c = 0.7978845608028654f, k = 0.044715f;
    constexpr float a = (float)(-2.0 * 0.7978845608028654 * 1.4426950408889634);
    const float g2 = g * g;
    const float s =
        __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * __builtin_fmaf(g2, a * k, a)));
    const float t = s * (1.0f - s);
    return make_float2(g * s, s + (t == 0.0f ? 0.0f : 2.0f * c * g * t * (1.0f + 3.0f * k * g2)));
  }
  if (act == EPI_RELU) return make_float2(g > 0.0f ? g : 0.0f, g > 0.0f ? 1.0f : 0.0f);
  return make_float2(g, 1.0f);
}

// Four k of one column for each lane of 16: lanes 4 r + c of a group read 8 bytes each
// (columns 4 c on of row r) and get column (lane % 16) of the group's four rows.  The
// restrict on the address gives the read alias information of its own; without any,
// the compiler holds it to depend on every direct load into LDS in flight and waits
// for them all (a whole memory latency a fragment).
__device__ __forceinline__ bf16x4 read_tr(const uint16_t *__restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4 *)p);
}

// One operand of a tile: BR rows of a 64-deep stage, NW waves loading 1 KB each a
// load, LOADS loads a wave.
//
// K-contiguous (KC): LDS row r holds 64 k (128 bytes), chunk c of 8 k at
// c ^ (r / 2 % 8): a load covers 8 rows.
//
// K-strided: LDS row k holds BR columns (2 BR bytes) and a load covers 512 / BR of
// them.  A transposed read serves 32 lanes at a time: 32-byte pieces of the 8 rows
// {0-3, 8-11} + 4 h + 16 i, which would all start at one bank (rows are a multiple
// of the 256-byte bank window); XOR-ing the piece with (k % 4) + 4 (k / 8 % 2) gives
// them 8 different places in the window.  BR = 64: two rows share a window, so two
// bits (k / 2 % 2, k / 8 % 2) suffice.
template <int BR, int NW, bool KC>
struct Operand {
  static constexpr int LOADS = BR / (8 * NW);
  static constexpr int STAGE = BR * kBK;  // elements of a stage buffer
  static constexpr int UNIT = KC ? 8 : 512 / BR;  // LDS rows of a load
  uint32_t off;  // this lane's byte offset from the load's first row
  int kc;        // KC: the first k of this lane's chunk

  static __device__ __forceinline__ int piece(int k) {
    return BR == 64 ? ((k >> 1) & 1) | ((k >> 2) & 2) : (k & 3) | ((k >> 1) & 4);
  }

  // The swizzles repeat after the NW loads of a round, so a lane's offset is the
  // same for all its loads; what differs is uniform and goes into the resource.
  __device__ __forceinline__ void init(int64_t ld, int wave, int lane) {
    if constexpr (KC) {
      kc = ((lane & 7) ^ (((wave * 8 + (lane >> 3)) >> 1) & 7)) * 8;
      off = (uint32_t)((lane >> 3) * ld + kc) * 2;
    } else {
      constexpr int CH = BR / 8;  // 16-byte chunks of an LDS row
      const int k = lane / CH, c = lane % CH;
      kc = 0;
      off = (uint32_t)(k * ld + ((((c >> 1) ^ piece(wave * UNIT + k)) << 1) | (c & 1)) * 8) * 2;
    }
  }

  // First LDS row of load i.
  static __device__ __forceinline__ int row_of(int i, int wave) { return (i * NW + wave) * UNIT; }

  // The resource of a load from `rows` memory rows (clamped to the load's own; none:
  // it reads zeros) whose first begins at p, `skip` elements into its row.
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const uint16_t *p, int rows, int ld,
                                                                int skip) {
    rows = rows < 0 ? 0 : rows > UNIT ? UNIT : rows;
    const int bytes = rows == 0 ? 0 : (rows * ld - skip) * 2;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(p), (short)0, bytes, 0x00020000);
  }

  static __device__ __forceinline__ uint16_t *dst(uint16_t *stage, int i, int wave) {
    return stage + (i * NW + wave) * 512;
  }

  // The lane's part of a fragment's LDS address in bytes: block j of 16 rows at base +
  // j * 2048 (KC) or base ^ (j * 32) (K-strided: j < 8, and the bits of j are clear in
  // base before the XOR with the piece), step ks of 32 k.
  static __device__ __forceinline__ int lane_base(int row0, int ks, int lane) {
    const int fr = lane & 15, fh = lane >> 4;
    if constexpr (KC) return (row0 + fr) * 128 + (((ks * 4 + fh) ^ ((fr >> 1) & 7)) * 16);
    const int k = 8 * fh + (fr >> 2);
    return (ks * 32 + k) * (2 * BR) + ((row0 >> 4) ^ piece(k)) * 32 + (fr & 3) * 8;
  }

  // Block j's fragment.  The K-strided address is formed where it is used (in asm, which
  // the compiler cannot move out of the loop): eight of them kept in registers spill.
  static __device__ __forceinline__ void read(bf16x8 &f, const uint16_t *stage, int base, int j) {
    const char *s = (const char *)stage;
    if constexpr (KC) {
      f = *(const bf16x8 *)(s + base + j * 2048);
    } else {
      int at;
      asm volatile("v_xor_b32 %0, %1, %2" : "=v"(at) : "i"(j * 32), "v"(base));
      const bf16x4 lo = read_tr((const uint16_t *)(s + at));
      const bf16x4 hi = read_tr((const uint16_t *)(s + at + 8 * BR));
      f = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Load i of an operand's stage at k0 (of K segment seg) of the tile rows from row0 of
// R into LDS.  FAST: the stage is whole; else chunks past K read zeros, and all do
// where !in.  PAIR (gate/up): tile rows are WN / 2 of P0's, then the same WN / 2 of
// P1's, in turn.
template <typename O, bool KC, bool FAST, bool PAIR, int WN = 1>
__device__ __forceinline__ void load_block(const O &o, const uint16_t *P0, const uint16_t *P1, int ld,
                                           int row0, int R, int K, int seg, int k0, bool in,
                                           uint16_t *dst, int i, int wave) {
  int r = O::row_of(i, wave);
  if constexpr (KC) {
    bool second = seg != 0;
    if constexpr (PAIR) {
      second = r % WN >= WN / 2;
      r = (r / WN) * (WN / 2) + r % (WN / 2);
    }
    const uint16_t *p = (second ? P1 : P0) + (int64_t)(row0 + r) * ld + k0;
    if constexpr (FAST) {
      dma16(O::rsrc(p, R - row0 - r, ld, k0), dst, o.off);
    } else {
      dma16(O::rsrc(p, in ? R - row0 - r : 0, ld, k0), dst, k0 + o.kc < K ? o.off : kOobOffset);
    }
  } else {
    const uint16_t *p = (seg ? P1 : P0) + (int64_t)(k0 + r) * ld + row0;
    dma16(O::rsrc(p, FAST || in ? K - k0 - r : 0, ld, row0), dst, o.off);
  }
}

// Which problem, K slice and tile a workgroup computes.  The problems' tiles form
// one list, of which each XCD takes a contiguous run (neighbouring tiles share
// operand panels in its L2).
struct TileAt {
  int prob, split, m, n;
};
__device__ __forceinline__ TileAt locate(const TileArgs &a) {
  const int total = a.tiles * a.splits, x = blockIdx.x & 7, q = total >> 3, r = total & 7;
  int logical = x * q + (x < r ? x : r) + ((int)blockIdx.x >> 3);
  TileAt t;
  t.split = logical / a.tiles;
  logical -= t.split * a.tiles;
  t.prob = 0;
  if (a.n > 1 && logical >= a.p[1].first) t.prob = 1;
  if (a.n > 2 && logical >= a.p[2].first) t.prob = 2;
  const TileProb &p = a.p[t.prob];
  group_coords(logical - p.first, p.tiles_m, p.tiles_n, 4, t.m, t.n);
  return t;
}

// The outputs of a tile.  A lane's block (i, j) holds row 16 i + (lane & 15) at columns
// 16 j + 4 (lane >> 4) + q; pairs of blocks are traded between lane rows so that a lane
// stores 16 bytes.
template <int ACT, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void out_gate(const TileProb &p, const f32x4 (&acc)[TM][TN], int m0,
                                         int n0, int wm, int wn, int lane) {
  constexpr int TH = TN / 2;
  const int fr = lane & 15, fh = lane >> 4;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + fr;
    uint32_t w[TH][2];
#pragma unroll
    for (int j = 0; j < TH; ++j) {
      const int n = n0 + wn * (WN / 2) + j * 16 + 4 * fh;
      float h[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) h[q] = act_b16(ACT, acc[i][j][q]) * acc[i][j + TH][q];
      w[j][0] = pack_bf16x2(h[0], h[1]);
      w[j][1] = pack_bf16x2(h[2], h[3]);
      if (p.F && m < p.M && n < p.N) {
        const f32x4 &g = acc[i][j], &u = acc[i][j + TH];
        *(float4 *)(p.F + (size_t)m * p.ldc + n) = make_float4(g[0], g[1], g[2], g[3]);
        *(float4 *)(p.F2 + (size_t)m * p.ldc + n) = make_float4(u[0], u[1], u[2], u[3]);
      }
    }
    if constexpr (TH == 2) {
      const auto a = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
      const auto b = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
      const int n = n0 + wn * (WN / 2) + (fh & 1) * 16 + 8 * (fh >> 1);
      if (m < p.M && n < p.N)
        *(uint4 *)(p.C + (size_t)m * p.ldc + n) = make_uint4(a[0], b[0], a[1], b[1]);
    } else {
      const int n = n0 + wn * (WN / 2) + 4 * fh;
      if (m < p.M && n < p.N) *(uint2 *)(p.C + (size_t)m * p.ldc + n) = make_uint2(w[0][0], w[0][1]);
    }
  }
}

template <int ACT, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void out_dgate(const TileProb &p, const f32x4 (&acc)[TM][TN], int m0,
                                          int n0, int wm, int wn, int lane) {
  const int fr = lane & 15, fh = lane >> 4;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + fr;
    uint32_t wg[TN][2], wu[TN][2];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + wn * WN + j * 16 + 4 * fh;
      float4 g = make_float4(0, 0, 0, 0), u = g;
      if (m < p.M && n < p.N) {
        g = *(const float4 *)(p.F + (size_t)m * p.ldc + n);
        u = *(const float4 *)(p.F2 + (size_t)m * p.ldc + n);
      }
      const float gv[4] = {g.x, g.y, g.z, g.w}, uv[4] = {u.x, u.y, u.z, u.w};
      float dg[4], du[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 a = act_grad_b16(ACT, gv[q]);
        du[q] = acc[i][j][q] * a.x;
        dg[q] = acc[i][j][q] * uv[q] * a.y;
      }
      wg[j][0] = pack_bf16x2(dg[0], dg[1]);
      wg[j][1] = pack_bf16x2(dg[2], dg[3]);
      wu[j][0] = pack_bf16x2(du[0], du[1]);
      wu[j][1] = pack_bf16x2(du[2], du[3]);
    }
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      const int n = n0 + wn * WN + (j + (fh & 1)) * 16 + 8 * (fh >> 1);
      const auto a = __builtin_amdgcn_permlane16_swap(wg[j][0], wg[j + 1][0], false, false);
      const auto b = __builtin_amdgcn_permlane16_swap(wg[j][1], wg[j + 1][1], false, false);
      const auto c = __builtin_amdgcn_permlane16_swap(wu[j][0], wu[j + 1][0], false, false);
      const auto d = __builtin_amdgcn_permlane16_swap(wu[j][1], wu[j + 1][1], false, false);
      if (m < p.M && n < p.N) {
        *(uint4 *)(p.C + (size_t)m * p.ldc + n) = make_uint4(a[0], b[0], a[1], b[1]);
        *(uint4 *)(p.C2 + (size_t)m * p.ldc + n) = make_uint4(c[0], d[0], c[1], d[1]);
      }
    }
  }
}

template <int TM, int TN, int WM, int WN>
__device__ __forceinline__ void out_store(const TileProb &p, const f32x4 (&acc)[TM][TN], int m0,
                                          int n0, int wm, int wn, int lane) {
  const int fr = lane & 15, fh = lane >> 4;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + fr;
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      const f32x4 &x = acc[i][j], &y = acc[i][j + 1];
      const auto a = __builtin_amdgcn_permlane16_swap(pack_bf16x2(x[0], x[1]),
                                                      pack_bf16x2(y[0], y[1]), false, false);
      const auto b = __builtin_amdgcn_permlane16_swap(pack_bf16x2(x[2], x[3]),
                                                      pack_bf16x2(y[2], y[3]), false, false);
      const int n = n0 + wn * WN + (j + (fh & 1)) * 16 + 8 * (fh >> 1);
      if (m < p.M && n < p.N)
        *(uint4 *)(p.C + (size_t)m * p.ldc + n) = make_uint4(a[0], b[0], a[1], b[1]);
    }
  }
}

template <int TM, int TN, int WM, int WN>
__device__ __forceinline__ void out_part(const TileProb &p, const f32x4 (&acc)[TM][TN], int m0,
                                         int n0, int wm, int wn, int lane, int split) {
  float *part = p.part + (size_t)split * p.M * p.N;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + wn * WN + j * 16 + 4 * (lane >> 4);
      const f32x4 &v = acc[i][j];
      if (m < p.M && n < p.N)
        *(float4 *)(part + (size_t)m * p.N + n) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
}

template <int OUT, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void tile_out(const TileArgs &a, const TileProb &p,
                                         const f32x4 (&acc)[TM][TN], int m0, int n0, int wm,
                                         int wn, int lane, int split) {
  if constexpr (OUT == OUT_STORE) {
    out_store<TM, TN, WM, WN>(p, acc, m0, n0, wm, wn, lane);
  } else if constexpr (OUT == OUT_PART) {
    out_part<TM, TN, WM, WN>(p, acc, m0, n0, wm, wn, lane, split);
  } else {
    switch (a.act) {
#define MJ_OUT(E)                                                              \
  if constexpr (OUT == OUT_GATE)                                               \
    out_gate<E, TM, TN, WM, WN>(p, acc, m0, n0, wm, wn, lane);                 \
  else                                                                         \
    out_dgate<E, TM, TN, WM, WN>(p, acc, m0, n0, wm, wn, lane);                \
  break;
      case EPI_RELU: MJ_OUT(EPI_RELU)
      case EPI_GELU_TANH: MJ_OUT(EPI_GELU_TANH)
      case EPI_SILU: MJ_OUT(EPI_SILU)
      default: MJ_OUT(EPI_NONE)
#undef MJ_OUT
    }
  }
}

// Tiles of four waves (2 x 2) on a ring of S 64-deep stages, the direct loads
// S - 2 stages ahead and a wave's fragments half a stage: the stage's one barrier
// sits between its two 32-deep steps, where the next stage has landed.
template <int BM, int BN, int S, bool AKC, bool BKC, int OUT>
__global__ __launch_bounds__(256) void mlp_ring_kernel(TileArgs args) {
  constexpr int NW = 4, WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
  constexpr int BN_OUT = OUT == OUT_GATE ? BN / 2 : BN;
  using OA = Operand<BM, NW, AKC>;
  using OB = Operand<BN, NW, BKC>;
  constexpr int NDMA = OA::LOADS + OB::LOADS, FLY = (S - 3) * NDMA;
  static_assert(S >= 3 && FLY < 64, "vmcnt range");
  static_assert(OUT != OUT_GATE || BKC, "gate and up rows are K-contiguous");
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const TileAt at = locate(args);
  const TileProb &p = args.p[at.prob];
  const int m0 = at.m * BM, n0 = at.n * BN_OUT;
  const int M = p.M, N = p.N, K = p.K;
  const int lda = (int)p.lda, ldb = (int)p.ldb;
  const uint16_t *const A0 = p.A[0], *const A1 = p.A[1], *const B0 = p.B[0], *const B1 = p.B[1];
  const int nk = (K + kBK - 1) / kBK, stages = nk * p.segs;
  const int per = (stages + args.splits - 1) / args.splits;
  const int kt0 = at.split * per, kt1 = std::min(kt0 + per, stages);

  OA oa;
  oa.init(lda, wave, lane);
  OB ob;
  ob.init(ldb, wave, lane);
  // byte offsets of each load's rows from the tile's (K-contiguous: rows past the edge
  // read zeros) or the stage's first
  uint32_t aoff[OA::LOADS], boff[OB::LOADS];
#pragma unroll
  for (int i = 0; i < OA::LOADS; ++i) {
    const int r = OA::row_of(i, wave);
    aoff[i] = !AKC || m0 + r + (lane >> 3) < M ? oa.off + (uint32_t)r * lda * 2 : kOobOffset;
  }
#pragma unroll
  for (int i = 0; i < OB::LOADS; ++i) {
    int r = OB::row_of(i, wave);
    if constexpr (OUT == OUT_GATE) r = (r / WN) * (WN / 2) + r % (WN / 2);
    boff[i] = !BKC || n0 + r + (lane >> 3) < N ? ob.off + (uint32_t)r * ldb * 2 : kOobOffset;
  }
  // whether load i fetches up rows (gate/up tiles)
  auto is_up = [&](int i) { return OUT == OUT_GATE && OB::row_of(i, wave) % WN >= WN / 2; };
  auto tile_rsrc = [&](const uint16_t *P, int row0, int R, int ld) {
    return make_rsrc(P + (size_t)row0 * ld, (int64_t)(R - row0) * ld * 2);
  };
  auto stage_rsrc = [&](const uint16_t *P, int row0, int k0, int left, int ld) {
    const int rows = left < 0 ? 0 : left > kBK ? kBK : left;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(P + (int64_t)k0 * ld + row0),
                                             (short)0, rows ? (rows * ld - row0) * 2 : 0, 0x00020000);
  };
  // stage kt into its ring buffer; past the slice it reads zeros
  auto issue = [&](int kt) __attribute__((always_inline)) {
    const int seg = kt >= nk ? 1 : 0, k0 = (kt - seg * nk) * kBK;
    const int Kin = kt < kt1 ? K : 0;
    uint16_t *as = lds + (kt % S) * (OA::STAGE + OB::STAGE), *bs = as + OA::STAGE;
    if constexpr (AKC) {
      const auto r = tile_rsrc(seg ? A1 : A0, m0, M, lda);
#pragma unroll
      for (int i = 0; i < OA::LOADS; ++i)
        dma16(r, OA::dst(as, i, wave), k0 + oa.kc < Kin ? aoff[i] + k0 * 2 : kOobOffset);
    } else {
      const auto r = stage_rsrc(seg ? A1 : A0, m0, k0, Kin - k0, lda);
#pragma unroll
      for (int i = 0; i < OA::LOADS; ++i) dma16(r, OA::dst(as, i, wave), aoff[i]);
    }
    if constexpr (BKC) {
      const auto r = tile_rsrc(OUT != OUT_GATE && seg ? B1 : B0, n0, N, ldb);
      const auto r2 = tile_rsrc(OUT == OUT_GATE ? B1 : B0, n0, N, ldb);
#pragma unroll
      for (int i = 0; i < OB::LOADS; ++i) {
        const uint32_t o = k0 + ob.kc < Kin ? boff[i] + k0 * 2 : kOobOffset;
        if (is_up(i)) dma16(r2, OB::dst(bs, i, wave), o);
        else dma16(r, OB::dst(bs, i, wave), o);
      }
    } else {
      const auto r = stage_rsrc(seg ? B1 : B0, n0, k0, Kin - k0, ldb);
#pragma unroll
      for (int i = 0; i < OB::LOADS; ++i) dma16(r, OB::dst(bs, i, wave), boff[i]);
    }
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
  bf16x8 fa[2][TM], fb[2][TN];
  auto read_frags = [&](int kt, int ks) __attribute__((always_inline)) {
    const uint16_t *as = lds + (kt % S) * (OA::STAGE + OB::STAGE), *bs = as + OA::STAGE;
#pragma unroll
    for (int i = 0; i < TM; ++i) OA::read(fa[ks][i], as, abase[ks], i);
#pragma unroll
    for (int j = 0; j < TN; ++j) OB::read(fb[ks][j], bs, bbase[ks], j);
  };
  auto mma = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[ks][j], fa[ks][i], acc[i][j], 0, 0,
                                                            0);
  };
  // the loads of all but the FLY youngest have landed, in every wave, and every
  // wave holds the fragments that it read before
  auto landed = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070 | (FLY & 0xF) | ((FLY >> 4) << 14));  // and lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int s = 0; s < S - 2; ++s) issue(kt0 + s);
  landed();  // stage kt0
  issue(kt0 + S - 2);
  read_frags(kt0, 0);
  for (int kt = kt0; kt < kt1; ++kt) {
    read_frags(kt, 1);
    mma(0);
    landed();  // stage kt + 1
    issue(kt + S - 1);
    read_frags(kt + 1, 0);
    mma(1);
  }
  // loads past the slice must not land in a later workgroup's LDS
  __builtin_amdgcn_s_waitcnt(0x0F70);
  tile_out<OUT, TM, TN, WM, WN>(args, p, acc, m0, n0, wm, wn, lane, at.split);
}

// The pipelined tiles: 256 x 256 of 8 waves (2 x 4, 128 x 64 outputs each), one
// workgroup a CU, or 128 x 128 of 4 waves (2 x 2, 64 x 64 each), two a CU, where 256 x
// 256 tiles leave CUs idle (twice the operand traffic and a third more LDS reads a
// flop: in whole layers 0.98 us for two 64-deep stages of 128 x 128, 1.47 for one of 256 x
// 256, twice the work of the two).  Both put two waves on a SIMD, and run the pipeline of the
// framework's large bf16 product (gemm_nt_w8_kernel): two A and three B stage buffers,
// a stage of two 32-deep steps with one barrier between them, each step's fragment
// reads for the next spread between its MFMAs, four direct loads a step for the stage
// after next.  A K-strided operand has two 8-byte transposed reads a fragment in place
// of one of 16 bytes; its resource moves along K with the stage, so its loads need no
// bounds selects at any K.
template <int BM, int NW, bool AKC, bool BKC, int OUT>
__global__ __launch_bounds__(NW * 64, 2) void mlp_tile_kernel(TileArgs args) {
  constexpr int BN = BM, WGN = NW / 2, WM = BM / 2, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr int BN_OUT = OUT == OUT_GATE ? BN / 2 : BN;
  using OA = Operand<BM, NW, AKC>;
  using OB = Operand<BN, NW, BKC>;
  constexpr int DPO = 4;  // direct loads per wave per operand per stage
  static_assert(OA::LOADS == DPO && OB::LOADS == DPO && TN == DPO, "a load per group");
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  uint16_t *As = lds;                   // stage kt in buffer kt % 2
  uint16_t *Bs = lds + 2 * OA::STAGE;   // stage kt in buffer kt % 3
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const TileAt at = locate(args);
  const TileProb &p = args.p[at.prob];
  const int m0 = at.m * BM, n0 = at.n * BN_OUT;
  const int M = p.M, N = p.N, K = p.K;
  const int lda = (int)p.lda, ldb = (int)p.ldb;
  const uint16_t *const A0 = p.A[0], *const A1 = p.A[1], *const B0 = p.B[0], *const B1 = p.B[1];
  const int nk = (K + kBK - 1) / kBK, stages = nk * p.segs;
  const int per = (stages + args.splits - 1) / args.splits;
  const int kt0 = at.split * per, kt1 = std::min(kt0 + per, stages);

  OA oa;
  oa.init(lda, wave, lane);
  OB ob;
  ob.init(ldb, wave, lane);
  // direct load d of stage kt into buffer buf: d < 4 is A block d, else B block d - 4
  auto load = [&](auto fast, int kt, int buf, int d) __attribute__((always_inline)) {
    constexpr bool FAST = decltype(fast)::value;
    const int seg = kt >= nk ? 1 : 0, k0 = (kt - seg * nk) * kBK;
    const bool in = kt < kt1;
    const int i = d & 3;
    if (d < DPO)
      load_block<OA, AKC, FAST, false>(oa, A0, A1, lda, m0, M, K, seg, k0, in,
                                       OA::dst(As + buf * OA::STAGE, i, wave), i, wave);
    else
      load_block<OB, BKC, FAST, OUT == OUT_GATE, WN>(ob, B0, B1, ldb, n0, N, K, seg, k0, in,
                                                     OB::dst(Bs + buf * OB::STAGE, i, wave), i,
                                                     wave);
  };

  int abase[2], bbase[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    abase[ks] = OA::lane_base(wm * WM, ks, lane);
    bbase[ks] = OB::lane_base(wn * WN, ks, lane);
  }
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  bf16x8 fa[2][TM], fb[2][TN];
  // the fragments of a step: A's blocks, then B's, PER a group
  constexpr int PER = (TM + TN) / TN;
  auto read_frag = [&](int t, int dst, int abuf, int bbuf) __attribute__((always_inline)) {
    if (t < TM) OA::read(fa[dst][t], As + abuf * OA::STAGE, abase[dst], t);
    else OB::read(fb[dst][t - TM], Bs + bbuf * OB::STAGE, bbase[dst], t - TM);
  };

#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int d = 0; d < 2 * DPO; ++d) load(std::false_type(), kt0 + s, s, d);
  __builtin_amdgcn_s_waitcnt(0x0F70 | (2 * DPO));  // stage 0
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int t = 0; t < TM + TN; ++t) read_frag(t, 0, 0, 0);
  __builtin_amdgcn_s_waitcnt(kLgkm0);
  asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");  // zero fill -> first MFMAs

  auto stage = [&](auto ab_c, auto bb_c, auto fast, int kt) __attribute__((always_inline)) {
    constexpr int AB = decltype(ab_c)::value;
    constexpr int BB = decltype(bb_c)::value;
    auto group = [&](int j, int src, int dst, int abuf, int bbuf, int load_d,
                     int load_buf) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        __builtin_amdgcn_sched_barrier(0);
        read_frag(PER * j + u, dst, abuf, bbuf);
        __builtin_amdgcn_sched_barrier(0);
        mfma_16x16x32_tied(acc[u][j], fb[src][j], fa[src][u]);
      }
      __builtin_amdgcn_sched_barrier(0);
      load(fast, kt + 2, load_buf, load_d);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = PER; i < TM; ++i) mfma_16x16x32_tied(acc[i][j], fb[src][j], fa[src][i]);
    };
    // step 0; B loads of stage kt+2 into B buffer (BB + 2) % 3
#pragma unroll
    for (int j = 0; j < TN; ++j) group(j, 0, 1, AB, BB, DPO + j, (BB + 2) % 3);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kLgkm0);
    __builtin_amdgcn_s_waitcnt(0x0F70 | DPO);  // all but this step's B loads
    asm volatile("s_barrier" ::: "memory");
    // step 1; A loads of stage kt+2 into A buffer AB
#pragma unroll
    for (int j = 0; j < TN; ++j) group(j, 1, 0, AB ^ 1, (BB + 1) % 3, j, AB);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kLgkm0);
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using F = std::true_type;
  using S = std::false_type;
  // stages up to here are whole; K-strided operands end by their resource alone
  const int whole = std::min(kt1, K % kBK == 0 ? stages : (p.segs == 1 ? K / kBK : 0));
  int kt = kt0;
  for (; kt + 8 <= whole; kt += 6) {
    stage(I0(), I0(), F(), kt);
    stage(I1(), I1(), F(), kt + 1);
    stage(I0(), I2(), F(), kt + 2);
    stage(I1(), I0(), F(), kt + 3);
    stage(I0(), I1(), F(), kt + 4);
    stage(I1(), I2(), F(), kt + 5);
  }
  for (; kt < kt1; kt += 6) {
    stage(I0(), I0(), S(), kt);
    if (kt + 1 < kt1) stage(I1(), I1(), S(), kt + 1);
    if (kt + 2 < kt1) stage(I0(), I2(), S(), kt + 2);
    if (kt + 3 < kt1) stage(I1(), I0(), S(), kt + 3);
    if (kt + 4 < kt1) stage(I0(), I1(), S(), kt + 4);
    if (kt + 5 < kt1) stage(I1(), I2(), S(), kt + 5);
  }
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);
  tile_out<OUT, TM, TN, WM, WN>(args, p, acc, m0, n0, wm, wn, lane, at.split);
}

// C = bf16(sum of the K slices' partials, in slice order), 8 elements a thread.
__global__ __launch_bounds__(256) void mlp_reduce_kernel(const float *part, uint16_t *C, int64_t n,
                                                         int splits) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (e >= n) return;
  float v[8] = {};
  for (int s = 0; s < splits; ++s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 q = *(const float4 *)(part + (size_t)s * n + e + 4 * h);
      v[4 * h] += q.x, v[4 * h + 1] += q.y, v[4 * h + 2] += q.z, v[4 * h + 3] += q.w;
    }
  }
  *(uint4 *)(C + e) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                 pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// ---------------------------------------------------------------- few rows
// Products of at most 16 MB rows: bound by reading the weights once.  A workgroup of NW
// waves owns 16 weight rows (gate/up: 16 of each) and splits K, 64 at a time dealt to
// the waves in turn, so each 128-byte line of a weight row is read by two loads of one
// wave; a lane's 16 bytes are a row's 8 k, which is a fragment of
// v_mfma_f32_16x16x32_bf16 as it is.  x comes from the caches the same way (rows past M
// are zeros).  A wave loads its next slice of 64 as it multiplies one; no LDS in the
// loop.  The waves' sums are added in wave order and act, g, u, h (or y) follow in the
// same launch.
struct SkinnyArgs {
  const uint16_t *x = nullptr, *w = nullptr, *w2 = nullptr;
  uint16_t *C = nullptr;
  float *F = nullptr, *F2 = nullptr;
  int M = 0, N = 0, K = 0, act = 0;
};

template <bool GATE, int MB, int NW = 8>
__global__ __launch_bounds__(NW * 64) void mlp_skinny_kernel(SkinnyArgs p) {
  constexpr int G = GATE ? 2 : 1;
  __shared__ float red[NW][G][MB][16][17];
  const int lane = threadIdx.x & 63, fr = lane & 15, fh = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, M = p.M, N = p.N, K = p.K;
  const int rows = N - n0 < 16 ? N - n0 : 16;
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w + (size_t)n0 * K, (int64_t)rows * K * 2);
  const __amdgpu_buffer_rsrc_t rw2 =
      make_rsrc((GATE ? p.w2 : p.w) + (size_t)n0 * K, (int64_t)rows * K * 2);
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x, (int64_t)M * K * 2);
  const uint32_t wo = fr < rows ? (uint32_t)(fr * K) * 2 : kOobOffset;
  uint32_t xo[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) xo[b] = b * 16 + fr < M ? (uint32_t)((b * 16 + fr) * K) * 2 : kOobOffset;
  f32x4 acc[G][MB];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[g][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  uint4 wv[2][G], xv[2][MB];  // a slice of 64
  auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + 32 * h + 8 * fh;
      const bool in = k < K;
      wv[h][0] = buffer_load16(rw, in && wo != kOobOffset ? wo + k * 2 : kOobOffset);
      if constexpr (GATE)
        wv[h][1] = buffer_load16(rw2, in && wo != kOobOffset ? wo + k * 2 : kOobOffset);
#pragma unroll
      for (int b = 0; b < MB; ++b)
        xv[h][b] = buffer_load16(rx, in && xo[b] != kOobOffset ? xo[b] + k * 2 : kOobOffset);
    }
  };
  const int step = NW * 64;
  load(wave * 64);
  for (int k0 = wave * 64; k0 < K; k0 += step) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int b = 0; b < MB; ++b)
          acc[g][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[h][g]),
                                                              __builtin_bit_cast(bf16x8, xv[h][b]),
                                                              acc[g][b], 0, 0, 0);
    load(k0 + step);
  }
  // block (g, b): weight row 4 fh + q, x row 16 b + fr
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q) red[wave][g][b][fr][4 * fh + q] = acc[g][b][q];
  __syncthreads();
  for (int e = threadIdx.x; e < MB * 256; e += NW * 64) {
    const int b = e >> 8, r = (e >> 4) & 15, c = e & 15, m = b * 16 + r, n = n0 + c;
    if (m >= M || n >= N) continue;
    float v[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      v[g] = red[0][g][b][r][c];
#pragma unroll
      for (int w = 1; w < NW; ++w) v[g] += red[w][g][b][r][c];
    }
    const size_t at = (size_t)m * N + n;
    if constexpr (GATE) {
      if (p.F) p.F[at] = v[0], p.F2[at] = v[1];
      p.C[at] = (uint16_t)f32_to_bf16_bits(act_b16(p.act, v[0]) * v[1]);
    } else {
      p.C[at] = (uint16_t)f32_to_bf16_bits(v[0]);
    }
  }
}

// ---------------------------------------------------------------- odd widths
// 8 columns a thread: 16-byte loads and stores at the elements' own alignment.
__global__ __launch_bounds__(256) void copy_rows_kernel(CopyRows c) {
  const CopyRows::Mat &m = c.m[blockIdx.y];
  const int64_t per_row = (m.dst_cols + 7) / 8, total = m.dst_rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row, col = (i - r * per_row) * 8;
    const int64_t have = r < m.rows ? m.cols - col : 0, want = m.dst_cols - col;
    uint32_t w[4] = {0, 0, 0, 0};
    const uint16_t *s = m.src + r * m.src_ld + col;
    if (have >= 8) {
      const u32x4_a2 q = *(const u32x4_a2 *)s;
      w[0] = q[0], w[1] = q[1], w[2] = q[2], w[3] = q[3];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < have) w[j >> 1] |= (uint32_t)s[j] << (16 * (j & 1));
    }
    uint16_t *d = m.dst + r * m.dst_ld + col;
    if (want >= 8) {
      *(u32x4_a2 *)d = u32x4_a2{w[0], w[1], w[2], w[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < want) d[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// ---------------------------------------------------------------- fp32 block
__device__ __forceinline__ float2 act_grad_f32(int act, float g) {
  if (act == EPI_SILU) {
    const float s = sigmoid32(g), t = s * (1.0f - s);
    return make_float2(g * s, s + (t == 0.0f ? 0.0f : g * t));
  }
  if (act == EPI_GELU_TANH) {
    const float c = 0.7978845608028654f, k = 0.044715f;
    const float s = sigmoid32(2.0f * c * (g + k * g * g * g)), t = s * (1.0f - s);
    return make_float2(g * s, s + (t == 0.0f ? 0.0f : 2.0f * c * g * t * (1.0f + 3.0f * k * g * g)));
  }
  if (act == EPI_RELU) return make_float2(g > 0.0f ? g : 0.0f, g > 0.0f ? 1.0f : 0.0f);
  return make_float2(g, 1.0f);
}

// 4 elements a thread; the last few singly.
__global__ __launch_bounds__(256) void gate_f32_kernel(int act, const float *g, const float *u,
                                                       float *h, int64_t n) {
  const int64_t e = (grid_block<256>() * 256 + threadIdx.x) * 4;
  if (e + 4 <= n) {
    const float4 a = *(const float4 *)(g + e), b = *(const float4 *)(u + e);
    *(float4 *)(h + e) =
        make_float4(act_grad_f32(act, a.x).x * b.x, act_grad_f32(act, a.y).x * b.y,
                    act_grad_f32(act, a.z).x * b.z, act_grad_f32(act, a.w).x * b.w);
  } else {
    for (int64_t i = e; i < n; ++i) h[i] = act_grad_f32(act, g[i]).x * u[i];
  }
}

__global__ __launch_bounds__(256) void gate_bwd_f32_kernel(int act, const float *g, const float *u,
                                                           const float *dh, float *dg, float *du,
                                                           int64_t n) {
  const int64_t e = (grid_block<256>() * 256 + threadIdx.x) * 4;
  if (e + 4 <= n) {
    const float4 gv = *(const float4 *)(g + e), uv = *(const float4 *)(u + e),
                 dv = *(const float4 *)(dh + e);
    const float2 a = act_grad_f32(act, gv.x), b = act_grad_f32(act, gv.y),
                 c = act_grad_f32(act, gv.z), d = act_grad_f32(act, gv.w);
    *(float4 *)(dg + e) = make_float4(dv.x * uv.x * a.y, dv.y * uv.y * b.y, dv.z * uv.z * c.y,
                                      dv.w * uv.w * d.y);
    *(float4 *)(du + e) = make_float4(dv.x * a.x, dv.y * b.x, dv.z * c.x, dv.w * d.x);
  } else {
    for (int64_t i = e; i < n; ++i) {
      const float2 a = act_grad_f32(act, g[i]);
      const float d = dh[i];
      dg[i] = d * u[i] * a.y;
      du[i] = d * a.x;
    }
  }
}

// The sum of an fp32 product's K slices, in slice order; the buffers are 16-byte aligned
// where n is a multiple of 4.
__global__ __launch_bounds__(256) void sum_f32_kernel(const float *part, float *out, int64_t n,
                                                      int parts) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (n % 4 == 0 && e < n) {
    float4 s = *(const float4 *)(part + e);
    for (int k = 1; k < parts; ++k) {
      const float4 q = *(const float4 *)(part + k * n + e);
      s.x += q.x, s.y += q.y, s.z += q.z, s.w += q.w;
    }
    *(float4 *)(out + e) = s;
  } else {
    for (int64_t i = e; i < n && i < e + 4; ++i) {
      float s = part[i];
      for (int k = 1; k < parts; ++k) s += part[k * n + i];
      out[i] = s;
    }
  }
}

// ---------------------------------------------------------------- launch
void set_tiles(TileArgs &a, int bm, int bn_out) {
  a.tiles = 0;
  for (int i = 0; i < a.n; ++i) {
    a.p[i].tiles_m = (a.p[i].M + bm - 1) / bm;
    a.p[i].tiles_n = (a.p[i].N + bn_out - 1) / bn_out;
    a.p[i].first = a.tiles;
    a.tiles += a.p[i].tiles_m * a.p[i].tiles_n;
  }
}

template <int BM, int BN, int S, bool AKC, bool BKC, int OUT>
hipError_t launch_ring(TileArgs a, hipStream_t stream) {
  constexpr size_t lds = size_t(S) * (BM + BN) * kBK * sizeof(uint16_t);
  static_assert(lds <= 160 * 1024, "LDS budget");
  auto kern = mlp_ring_kernel<BM, BN, S, AKC, BKC, OUT>;
  static std::atomic<uint64_t> done{0};
  if (hipError_t e = raise_lds((const void *)kern, lds, done); e != hipSuccess) return e;
  set_tiles(a, BM, OUT == OUT_GATE ? BN / 2 : BN);
  const int64_t grid = (int64_t)a.tiles * a.splits;
  if (grid == 0) return hipSuccess;
  if (!grid_fits(grid, 256)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <int BM, int NW, bool AKC, bool BKC, int OUT>
hipError_t launch_w(TileArgs a, hipStream_t stream) {
  constexpr size_t lds = size_t(5 * BM) * kBK * sizeof(uint16_t);  // 160 or 80 KB
  auto kern = mlp_tile_kernel<BM, NW, AKC, BKC, OUT>;
  static std::atomic<uint64_t> done{0};
  if (hipError_t e = raise_lds((const void *)kern, lds, done); e != hipSuccess) return e;
  set_tiles(a, BM, OUT == OUT_GATE ? BM / 2 : BM);
  const int64_t grid = (int64_t)a.tiles * a.splits;
  if (grid == 0) return hipSuccess;
  if (!grid_fits(grid, NW * 64)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(NW * 64), lds, stream, a);
  return hipGetLastError();
}

// The tile kernels' times on MI355X (us): a launch, then for each round of workgroups
// that the CUs hold (per_cu each) the stages at the time of a 64-deep stage with 1, 2,
// .. workgroups per CU and the fixed part of a round (first loads and, by kind,
// output).  Fits to products of 48 to 4096 rows, widths 512 to 11008, e.g. the gradients
// dg, du of 4096 rows (K = 4096, 11008 columns): 256 x 256 395, 128 x 128 445, 128 x 64
// 641, 64 x 64 771; of 512 rows 105, 67, 90, 87; h of 300 rows (K = 1024, 2816
// columns) 37, 15.3, 16.4, 13.1; of 48 rows (11008) 82, -, 45, and 64 x 64 40.2
// with three stages, 34.1 with five (one or two workgroups a CU wait on memory).
// 128 x 128 and the fixed part of 256 x 256 gate/up are taken from whole layers, whose power
// lowers the clock: with 0.48, 0.86 and 8, which products alone give, the forward of 1024
// rows, 4096 and 11008 wide, took 293 us against 273, of 1536 434 against 401, of 6000, 1500
// and 4000 wide, 254 against 235; 200 rows, 2560 and 6912 wide, 53.8 against 57.2.
enum : int { T_256 = 0, T_128, T_64S3, T_64S5, T_128X64, T_COUNT };
struct TileCost {
  int bm, bn, threads, per_cu;
  double stage[3], fixed[4];  // fixed by OUT_*
};
constexpr TileCost kTileCost[T_COUNT] = {
    {256, 256, 512, 1, {1.47, 0, 0}, {7, 7, 10, 14}},
    {128, 128, 256, 2, {0.52, 0.98, 0}, {4, 3, 6, 9}},
    {64, 64, 256, 3, {0.48, 0.52, 0.62}, {2.1, 2.1, 3, 4}},
    {64, 64, 256, 2, {0.31, 0.48, 0}, {2.1, 2.1, 3, 4}},
    {128, 64, 256, 2, {0.45, 0.70, 0}, {2.5, 2.5, 4, 6}},
};
constexpr int64_t kCUs = 256;

int64_t tiles_of(const TileArgs &a, int bm, int bn) {
  int64_t t = 0;
  for (int i = 0; i < a.n; ++i)
    t += (int64_t)((a.p[i].M + bm - 1) / bm) * ((a.p[i].N + bn - 1) / bn);
  return t;
}

double tile_time_us(const TileCost &c, int out, int64_t wgs, int64_t stages) {
  const int64_t slots = kCUs * c.per_cu, rest = wgs % slots;
  double us = 3.0 + (double)(wgs / slots) * (c.fixed[out] + (double)stages * c.stage[c.per_cu - 1]);
  if (rest) us += c.fixed[out] + (double)stages * c.stage[(rest + kCUs - 1) / kCUs - 1];
  return us;
}

struct TilePlan {
  int tile = T_64S3, splits = 1;
};

// The tile, and for a plain product the K slices, of the least predicted time.  The
// slices' partials (fp32, written and read once, and their launch) pay where the
// tiles leave CUs idle: 512 x 4096 with K = 11008 is 32 tiles of 256 x 256, 58 us in 8
// slices; 67 on 128 x 64 tiles in 2, the best of the smaller tiles.  A number of slices
// that is no power of two has to win by 8 %, about what the predictions are off: 200 rows,
// 2560 and 6912 wide (y and dx in 6 slices, predicted 15 and 21 % below 4) step
// 183 -> 177 us, but 48 rows, 4096 and 11008 (y in 12 for 8, by 2 %) forward 73.7 -> 76.7.
TilePlan plan_tiles(const TileArgs &a, int out) {
  TilePlan best;
  double best_us = 1e30;
  const TileProb &p = a.p[0];
  const int64_t stages = (int64_t)((p.K + kBK - 1) / kBK) * p.segs;
  for (int t = 0; t < T_COUNT; ++t) {
    const TileCost &c = kTileCost[t];
    const int64_t tiles = tiles_of(a, c.bm, out == OUT_GATE ? c.bn / 2 : c.bn);
    if (!grid_fits(tiles, c.threads)) continue;
    for (int s = 1; s <= (out == OUT_STORE && a.n == 1 ? 16 : 1); ++s) {
      if (s > 1 && (stages / s < 4 || tiles * s > 2 * kCUs * c.per_cu)) break;
      double us = tile_time_us(c, s > 1 ? OUT_PART : out, tiles * s, (stages + s - 1) / s);
      if (s > 1) us += 2.5 + (8.0 * s + 2.0) * (double)p.M * (double)p.N / 8.0e6;
      if (s & (s - 1)) us *= 1.08;
      if (us < best_us) {
        best_us = us;
        best.tile = t;
        best.splits = s;
      }
    }
  }
  return best;
}

template <bool AKC, bool BKC, int OUT>
hipError_t launch_tile_kernel(int tile, const TileArgs &a, hipStream_t stream) {
  switch (tile) {
    case T_256: return launch_w<256, 8, AKC, BKC, OUT>(a, stream);
    case T_128: return launch_w<128, 4, AKC, BKC, OUT>(a, stream);
    case T_64S3: return launch_ring<64, 64, 3, AKC, BKC, OUT>(a, stream);
    case T_64S5: return launch_ring<64, 64, 5, AKC, BKC, OUT>(a, stream);
    default: return launch_ring<128, 64, 3, AKC, BKC, OUT>(a, stream);
  }
}

template <bool AKC, bool BKC, int OUT>
hipError_t launch_tiles(const TileArgs &a, hipStream_t stream) {
  return launch_tile_kernel<AKC, BKC, OUT>(plan_tiles(a, OUT).tile, a, stream);
}

// Up to 16 rows always; 17 to 32 where the weights are small (one launch instead of a K
// split's two, and latency counts): K = 1024, 2816 gate/up columns 6.4 us against 8.8 on
// tiles, K = 1408, 512 columns 5.8 against 7.9; at K = 2048, 5504 columns 18.7 against
// 13.9 (x is read again for every 16 weight rows).
bool skinny_takes(int64_t M, int64_t N, int64_t K) {
  return M <= 16 || (M <= 32 && N * K <= 3000000);
}

// Sixteen waves for a long sum of few rows (below).
bool few_rows_deep(int64_t M, int64_t K) { return M <= 4 && K >= 8192; }

// Waves: 4096 x 11008 gate/up of one row 34.6 us with eight (5.2 TB/s) and one slice of
// 64 k in flight each, 36.3, 37.1, 37.5 with two, three, four in flight (a wave's eight
// slices end sooner with one, and more workgroups fit a CU).  Sixteen waves for one long row: K = 11008, 4096 columns
// 20.6 us against 22.2 at one row (256 workgroups, one a CU), but 26.5 against 24.7 at
// 16 rows and 8.3 against 8.1 at K = 5504.
template <bool GATE>
hipError_t launch_skinny(const SkinnyArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.N + 15) / 16));
  if (a.N == 0) return hipSuccess;
  if (a.M > 16)
    hipLaunchKernelGGL((mlp_skinny_kernel<GATE, 2>), grid, dim3(512), 0, stream, a);
  else if (!GATE && few_rows_deep(a.M, a.K))
    hipLaunchKernelGGL((mlp_skinny_kernel<false, 1, 16>), grid, dim3(1024), 0, stream, a);
  else
    hipLaunchKernelGGL((mlp_skinny_kernel<GATE, 1>), grid, dim3(512), 0, stream, a);
  return hipGetLastError();
}

// A plain product, its K split where the plan says; `part` holds splits * M * N floats.
template <bool AKC, bool BKC>
hipError_t launch_plain(TileArgs a, float *part, hipStream_t stream) {
  const TileProb &p = a.p[0];
  if (p.M == 0 || p.N == 0) return hipSuccess;
  const TilePlan pl = plan_tiles(a, OUT_STORE);
  if (pl.splits == 1) return launch_tile_kernel<AKC, BKC, OUT_STORE>(pl.tile, a, stream);
  if (!part) return hipErrorInvalidValue;
  a.splits = pl.splits;
  a.p[0].part = part;
  if (hipError_t e = launch_tile_kernel<AKC, BKC, OUT_PART>(pl.tile, a, stream); e != hipSuccess)
    return e;
  const int64_t n = (int64_t)p.M * p.N;
  hipLaunchKernelGGL(mlp_reduce_kernel, dim3((unsigned)((n / 8 + 255) / 256)), dim3(256), 0, stream,
                     part, p.C, n, pl.splits);
  return hipGetLastError();
}

// The products' operands.  y, and dx with its two segments, may split K.
TileArgs gate_args(const GatedMlp &q) {
  TileArgs a;
  a.act = q.act;
  TileProb &p = a.p[0];
  p.A[0] = q.x, p.lda = q.K;
  p.B[0] = q.wg, p.B[1] = q.wu, p.ldb = q.K;
  p.M = (int)q.M, p.N = (int)q.I, p.K = (int)q.K;
  p.C = q.h, p.F = q.g, p.F2 = q.u, p.ldc = q.I;
  return a;
}

TileArgs down_args(const GatedMlp &q) {
  TileArgs a;
  TileProb &p = a.p[0];
  p.A[0] = q.h, p.lda = q.I;
  p.B[0] = q.wd, p.ldb = q.I;
  p.M = (int)q.M, p.N = (int)q.H, p.K = (int)q.I;
  p.C = q.y, p.ldc = q.H;
  return a;
}

TileArgs dx_args(const GatedMlp &q, const GatedMlpGrad &o) {
  TileArgs a;
  TileProb &p = a.p[0];
  p.A[0] = o.dg, p.A[1] = o.du, p.lda = q.I;
  p.B[0] = q.wg, p.B[1] = q.wu, p.ldb = q.K;
  p.M = (int)q.M, p.N = (int)q.K, p.K = (int)q.I, p.segs = 2;
  p.C = o.dx, p.ldc = q.K;
  return a;
}

TileArgs dgate_args(const GatedMlp &q, const GatedMlpGrad &o) {
  TileArgs a;
  a.act = q.act;
  TileProb &p = a.p[0];
  p.A[0] = o.dy, p.lda = q.H;
  p.B[0] = q.wd, p.ldb = q.I;
  p.M = (int)q.M, p.N = (int)q.I, p.K = (int)q.H;
  p.C = o.dg, p.C2 = o.du, p.F = q.g, p.F2 = q.u, p.ldc = q.I;
  return a;
}

// The wanted weight gradients (n: how many).
TileArgs dw_args(const GatedMlp &q, const GatedMlpGrad &o, bool dwg, bool dwu, bool dwd) {
  TileArgs w;
  w.n = 0;
  auto add = [&](const uint16_t *A, int64_t rows, const uint16_t *B, int64_t cols, uint16_t *C) {
    TileProb &p = w.p[w.n++];
    p.A[0] = A, p.lda = rows;
    p.B[0] = B, p.ldb = cols;
    p.M = (int)rows, p.N = (int)cols, p.K = (int)q.M;
    p.C = C, p.ldc = cols;
  };
  if (dwg) add(o.dg, q.I, q.x, q.K, o.dwg);
  if (dwu) add(o.du, q.I, q.x, q.K, o.dwu);
  if (dwd) add(o.dy, q.H, q.h, q.I, o.dwd);
  return w;
}

}  // namespace

const char *gated_mlp_kernel_name(int64_t M, int64_t K, int64_t I, int64_t H, int product) {
  GatedMlp q;
  q.M = M, q.K = K, q.I = I, q.H = H;
  const GatedMlpGrad o;
  if (product == 0 && skinny_takes(M, I, K)) return M > 16 ? "32 rows" : "16 rows";
  if (product == 1 && skinny_takes(M, H, I))
    return M > 16 ? "32 rows" : few_rows_deep(M, I) ? "4 rows, 16 waves" : "16 rows";
  const bool plain = product == 1 || product == 3;
  const TileArgs a = product == 0   ? gate_args(q)
                     : product == 1 ? down_args(q)
                     : product == 2 ? dgate_args(q, o)
                     : product == 3 ? dx_args(q, o)
                                    : dw_args(q, o, true, true, true);
  const TilePlan pl = plan_tiles(a, plain         ? OUT_STORE
                                    : product == 0 ? OUT_GATE
                                    : product == 2 ? OUT_DGATE
                                                   : OUT_STORE);
  static const char *const names[T_COUNT][2] = {
      {"256x256", "256x256, K slices"},
      {"128x128", "128x128, K slices"},
      {"64x64, 3 stages", "64x64, 3 stages, K slices"},
      {"64x64, 5 stages", "64x64, 5 stages, K slices"},
      {"128x64", "128x64, K slices"}};
  return names[pl.tile][pl.splits > 1];
}

int64_t gated_mlp_part_floats(int64_t M, int64_t K, int64_t I, int64_t H, bool backward) {
  GatedMlp q;
  q.M = M, q.K = K, q.I = I, q.H = H;
  if (!backward && skinny_takes(M, H, I)) return 0;
  const TileArgs a = backward ? dx_args(q, GatedMlpGrad()) : down_args(q);
  const int s = plan_tiles(a, OUT_STORE).splits;
  return s > 1 ? (int64_t)s * a.p[0].M * a.p[0].N : 0;
}

hipError_t launch_gated_mlp(const GatedMlp &q, hipStream_t stream) {
  if (q.M == 0) return hipSuccess;
  if (skinny_takes(q.M, q.I, q.K)) {
    SkinnyArgs a;
    a.x = q.x, a.w = q.wg, a.w2 = q.wu, a.C = q.h, a.F = q.g, a.F2 = q.u;
    a.M = (int)q.M, a.N = (int)q.I, a.K = (int)q.K, a.act = q.act;
    if (hipError_t e = launch_skinny<true>(a, stream); e != hipSuccess) return e;
  } else {
    if (hipError_t e = launch_tiles<true, true, OUT_GATE>(gate_args(q), stream); e != hipSuccess)
      return e;
  }
  if (!skinny_takes(q.M, q.H, q.I)) return launch_plain<true, true>(down_args(q), q.part, stream);
  SkinnyArgs a;
  a.x = q.h, a.w = q.wd, a.C = q.y;
  a.M = (int)q.M, a.N = (int)q.H, a.K = (int)q.I;
  return launch_skinny<false>(a, stream);
}

hipError_t launch_gated_mlp_bwd(const GatedMlp &q, const GatedMlpGrad &o, hipStream_t stream) {
  if (o.dx || o.dwg || o.dwu)
    if (hipError_t e = launch_tiles<true, false, OUT_DGATE>(dgate_args(q, o), stream); e != hipSuccess)
      return e;
  if (o.dx)
    if (hipError_t e = launch_plain<true, false>(dx_args(q, o), q.part, stream); e != hipSuccess)
      return e;
  const TileArgs w = dw_args(q, o, o.dwg, o.dwu, o.dwd);
  return w.n ? launch_tiles<false, false, OUT_STORE>(w, stream) : hipSuccess;
}

hipError_t launch_copy_rows_bf16(const CopyRows &c, hipStream_t stream) {
  int64_t most = 0;
  for (int i = 0; i < c.n; ++i)
    most = std::max(most, c.m[i].dst_rows * ((c.m[i].dst_cols + 7) / 8));
  if (most == 0) return hipSuccess;
  const int64_t blocks = std::min<int64_t>((most + 255) / 256, 4096);
  hipLaunchKernelGGL(copy_rows_kernel, dim3((unsigned)blocks, (unsigned)c.n), dim3(256), 0, stream,
                     c);
  return hipGetLastError();
}

hipError_t launch_gate_f32(int act, const float *g, const float *u, float *h, int64_t n,
                           hipStream_t stream) {
  if (n <= 0) return hipSuccess;
  hipLaunchKernelGGL(gate_f32_kernel, grid_rows<256>((n + 1023) / 1024), dim3(256), 0, stream, act, g,
                     u, h, n);
  return hipGetLastError();
}

hipError_t launch_sum_f32(const float *part, float *out, int64_t n, int64_t parts,
                          hipStream_t stream) {
  if (n <= 0) return hipSuccess;
  const int64_t grid = (n + 1023) / 1024;
  if (!grid_fits(grid, 256)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(sum_f32_kernel, dim3((unsigned)grid), dim3(256), 0, stream, part, out, n,
                     (int)parts);
  return hipGetLastError();
}

hipError_t launch_gate_bwd_f32(int act, const float *g, const float *u, const float *dh, float *dg,
                               float *du, int64_t n, hipStream_t stream) {
  if (n <= 0) return hipSuccess;
  hipLaunchKernelGGL(gate_bwd_f32_kernel, grid_rows<256>((n + 1023) / 1024), dim3(256), 0, stream, act,
                     g, u, dh, dg, du, n);
  return hipGetLastError();
}

}  // namespace mj
