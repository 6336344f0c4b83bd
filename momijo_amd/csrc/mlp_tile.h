// Tiles of bf16 products on gfx950 MFMA, with the gated feed-forward block's epilogues:
// the device side that the block (gated_mlp.hip) and the experts' block
// (experts_mlp.hip, EX: rows of many experts in one launch) share.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gemm_tile.h"

namespace mj {

typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

// What a tile's accumulators become.
enum : int {
  OUT_STORE = 0,  // C = bf16(acc)
  OUT_PART,       // fp32 partial sums of a K slice; EX: the output
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
  // experts' products (EX): the rows' weights, or null for ones, and where the gate
  // gradient's tiles leave their parts of the weights' gradients ([rows][dots_ld], or null)
  const float *rw = nullptr;
  float *dots = nullptr;
  int dots_ld = 0;
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
// The problem, K slice and tile that a workgroup computes.  The tile functions below read
// the operands of their TileProb and ask `out` for the one with the outputs only when the
// sums are there: where it has to be computed (an expert's rows), it costs no registers
// in the K loop.
struct TileAt {
  int prob, split, m, n;
};

// The outputs of a tile.  A lane's block (i, j) holds row 16 i + (lane & 15) at columns
// 16 j + 4 (lane >> 4) + q; pairs of blocks are traded between lane rows so that a lane
// stores 16 bytes.
template <int ACT, bool EX, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void out_gate(const TileProb &p, const f32x4 (&acc)[TM][TN], int m0,
                                         int n0, int wm, int wn, int lane) {
  constexpr int TH = TN / 2;
  const int fr = lane & 15, fh = lane >> 4;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + fr;
    const float rw = EX && p.rw && m < p.M ? p.rw[m] : 1.0f;
    uint32_t w[TH][2];
#pragma unroll
    for (int j = 0; j < TH; ++j) {
      const int n = n0 + wn * (WN / 2) + j * 16 + 4 * fh;
      float h[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        h[q] = act_b16(ACT, acc[i][j][q]) * acc[i][j + TH][q];
        if constexpr (EX) h[q] *= rw;
      }
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

//
// EX: acc is the gradient of the weighted h = rw act(g) u, so g and u take rw of it, and
// the weight the row's product of acc with act(g) u: each wave leaves its columns' part.
template <int ACT, bool EX, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void out_dgate(const TileProb &p, const f32x4 (&acc)[TM][TN], int m0,
                                          int n0, int wm, int wn, int lane) {
  const int fr = lane & 15, fh = lane >> 4;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm * WM + i * 16 + fr;
    const float rw = EX && p.rw && m < p.M ? p.rw[m] : 1.0f;
    float dot = 0.0f;
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
        if constexpr (EX) {
          if (n < p.N) dot = __builtin_fmaf(du[q], uv[q], dot);
          du[q] *= rw;
          dg[q] *= rw;
        }
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
    if constexpr (EX) {
      dot += __shfl_xor(dot, 16, 64);
      dot += __shfl_xor(dot, 32, 64);
      if (p.dots && fh == 0 && m < p.M && n0 + wn * WN < p.N) p.dots[(size_t)m * p.dots_ld + (n0 + wn * WN) / WN] = dot;
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

template <int OUT, bool EX, int TM, int TN, int WM, int WN>
__device__ __forceinline__ void tile_out(int act, const TileProb &p, const f32x4 (&acc)[TM][TN],
                                         int m0, int n0, int wm, int wn, int lane, int split) {
  if constexpr (OUT == OUT_STORE) {
    out_store<TM, TN, WM, WN>(p, acc, m0, n0, wm, wn, lane);
  } else if constexpr (OUT == OUT_PART) {
    out_part<TM, TN, WM, WN>(p, acc, m0, n0, wm, wn, lane, split);
  } else {
    switch (act) {
#define MJ_OUT(E)                                                              \
  if constexpr (OUT == OUT_GATE)                                               \
    out_gate<E, EX, TM, TN, WM, WN>(p, acc, m0, n0, wm, wn, lane);             \
  else                                                                         \
    out_dgate<E, EX, TM, TN, WM, WN>(p, acc, m0, n0, wm, wn, lane);            \
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
template <int BM, int BN, int S, bool AKC, bool BKC, int OUT, bool EX, typename Out>
__device__ __forceinline__ void ring_tile(uint16_t *lds, const TileProb &p, TileAt at, int splits,
                                          int act, Out out) {
  constexpr int NW = 4, WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
  constexpr int BN_OUT = OUT == OUT_GATE ? BN / 2 : BN;
  using OA = Operand<BM, NW, AKC>;
  using OB = Operand<BN, NW, BKC>;
  constexpr int NDMA = OA::LOADS + OB::LOADS, FLY = (S - 3) * NDMA;
  static_assert(S >= 3 && FLY < 64, "vmcnt range");
  static_assert(OUT != OUT_GATE || BKC, "gate and up rows are K-contiguous");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int m0 = at.m * BM, n0 = at.n * BN_OUT;
  const int M = p.M, N = p.N, K = p.K;
  const int lda = (int)p.lda, ldb = (int)p.ldb;
  const uint16_t *const A0 = p.A[0], *const A1 = p.A[1], *const B0 = p.B[0], *const B1 = p.B[1];
  const int nk = (K + kBK - 1) / kBK, stages = nk * p.segs;
  const int per = (stages + splits - 1) / splits;
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
  tile_out<OUT, EX, TM, TN, WM, WN>(act, out(), acc, m0, n0, wm, wn, lane, at.split);
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
template <int BM, int NW, bool AKC, bool BKC, int OUT, bool EX, typename Out>
__device__ __forceinline__ void pipe_tile(uint16_t *lds, const TileProb &p, TileAt at, int splits,
                                          int act, Out out) {
  constexpr int BN = BM, WGN = NW / 2, WM = BM / 2, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr int BN_OUT = OUT == OUT_GATE ? BN / 2 : BN;
  using OA = Operand<BM, NW, AKC>;
  using OB = Operand<BN, NW, BKC>;
  constexpr int DPO = 4;  // direct loads per wave per operand per stage
  static_assert(OA::LOADS == DPO && OB::LOADS == DPO && TN == DPO, "a load per group");
  uint16_t *As = lds;                   // stage kt in buffer kt % 2
  uint16_t *Bs = lds + 2 * OA::STAGE;   // stage kt in buffer kt % 3
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const int m0 = at.m * BM, n0 = at.n * BN_OUT;
  const int M = p.M, N = p.N, K = p.K;
  const int lda = (int)p.lda, ldb = (int)p.ldb;
  const uint16_t *const A0 = p.A[0], *const A1 = p.A[1], *const B0 = p.B[0], *const B1 = p.B[1];
  const int nk = (K + kBK - 1) / kBK, stages = nk * p.segs;
  const int per = (stages + splits - 1) / splits;
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
  tile_out<OUT, EX, TM, TN, WM, WN>(act, out(), acc, m0, n0, wm, wn, lane, at.split);
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
  float *F = nullptr, *F2 = nullptr;  // g, u; EX without a gate: the output
  int M = 0, N = 0, K = 0, act = 0;
  const float *rw = nullptr;  // EX: the rows' weights, or null for ones
};

template <bool GATE, int MB, int NW>
struct SkinnySums {
  float red[NW][GATE ? 2 : 1][MB][16][17];
};

template <bool GATE, int MB, int NW, bool EX>
__device__ __forceinline__ void skinny_rows(SkinnySums<GATE, MB, NW> &sums, const SkinnyArgs &p, int n0) {
  constexpr int G = GATE ? 2 : 1;
  auto &red = sums.red;
  const int lane = threadIdx.x & 63, fr = lane & 15, fh = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int M = p.M, N = p.N, K = p.K;
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
      float h = act_b16(p.act, v[0]) * v[1];
      if constexpr (EX) h *= p.rw ? p.rw[m] : 1.0f;
      p.C[at] = (uint16_t)f32_to_bf16_bits(h);
    } else if constexpr (EX) {
      p.F[at] = v[0];
    } else {
      p.C[at] = (uint16_t)f32_to_bf16_bits(v[0]);
    }
  }
}

// ---------------------------------------------------------------- cost
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

inline double tile_time_us(const TileCost &c, int out, int64_t wgs, int64_t stages) {
  const int64_t slots = kCUs * c.per_cu, rest = wgs % slots;
  double us = 3.0 + (double)(wgs / slots) * (c.fixed[out] + (double)stages * c.stage[c.per_cu - 1]);
  if (rest) us += c.fixed[out] + (double)stages * c.stage[(rest + kCUs - 1) / kCUs - 1];
  return us;
}

}  // namespace mj
