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

#include "common.h"
#include "launch.h"
#include "mlp_tile.h"
#include "philox.h"

namespace mj {

namespace {

struct TileArgs {
  TileProb p[3];
  int n = 1, tiles = 0, splits = 1, act = 0;
};

// Which problem, K slice and tile a workgroup computes.  The problems' tiles form
// one list, of which each XCD takes a contiguous run (neighbouring tiles share
// operand panels in its L2).
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

template <int BM, int BN, int S, bool AKC, bool BKC, int OUT>
__global__ __launch_bounds__(256) void mlp_ring_kernel(TileArgs args) {
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  const TileAt at = locate(args);
  const TileProb &p = args.p[at.prob];
  ring_tile<BM, BN, S, AKC, BKC, OUT, false>(lds, p, at, args.splits, args.act,
                                             [&]() -> const TileProb & { return p; });
}

template <int BM, int NW, bool AKC, bool BKC, int OUT>
__global__ __launch_bounds__(NW * 64, 2) void mlp_tile_kernel(TileArgs args) {
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  const TileAt at = locate(args);
  const TileProb &p = args.p[at.prob];
  pipe_tile<BM, NW, AKC, BKC, OUT, false>(lds, p, at, args.splits, args.act,
                                          [&]() -> const TileProb & { return p; });
}

template <bool GATE, int MB, int NW = 8>
__global__ __launch_bounds__(NW * 64) void mlp_skinny_kernel(SkinnyArgs p) {
  __shared__ SkinnySums<GATE, MB, NW> sums;
  skinny_rows<GATE, MB, NW, false>(sums, p, blockIdx.x * 16);
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

int64_t tiles_of(const TileArgs &a, int bm, int bn) {
  int64_t t = 0;
  for (int i = 0; i < a.n; ++i)
    t += (int64_t)((a.p[i].M + bm - 1) / bm) * ((a.p[i].N + bn - 1) / bn);
  return t;
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
