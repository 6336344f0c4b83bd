// The gated feed-forward block of a mixture of experts on gfx950 bf16 MFMA, forward and
// backward, over rows sorted by expert (experts.hip).  Row r of expert e, with weight w_r:
//
//   g = x Wg_e^T, u = x Wu_e^T, h = w_r act(g) u, y = h Wd_e^T
//   dh = dy Wd_e, dg = w_r dh u act'(g), du = w_r dh act(g), dw_r = <dh, act(g) u>
//   dx = dg Wg_e + du Wu_e, dWg_e = dg^T x, dWu_e = du^T x, dWd_e = dy^T h
//
// The weight is applied to h and not to y, so that the layer's output is a plain sum of
// rows, the backward needs no y (dw comes from the fp32 g and u, with the error of an fp32
// sum and not of a rounded y), and dy's rows are copies of the tokens' gradients.  y and dx
// stay in fp32: a token's rows are still to be added, and rounded once then.
// h, dg and du are rounded to bf16, as in the block without experts: they are the next products'
// operands, and the matrix cores take bf16 at full rate (outputs off by 0.0023 against 64 bits;
// 0.0017 with these in fp32).
//
// The tiles are the gated block's (mlp_tile.h).  What differs is where a tile's operands
// are: the rows of all experts run as one launch, each workgroup finding its expert from
// the offsets (expert_tile.h).  The weight gradients' K is the expert's rows, so their grid
// is known; an expert without rows gets zeros.  With few rows an expert the weights' reading
// bounds, and the few-row kernel takes the segments of 16 rows.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "expert_tile.h"
#include "launch.h"
#include "mlp_tile.h"

namespace mj {

namespace {

struct ExpertArgs {
  TileProb p[3];
  int64_t b_expert = 0;       // elements of an expert's B matrix (row products)
  int64_t c_expert[3] = {};   // .. of its gradient (weight gradients)
  const int *offsets = nullptr;
  int experts = 0, rows = 0, n = 1, tail = 0, act = 0;
  int tiles_n = 0, cut = CUT_NONE;  // row products
  int tiles = 0;              // weight gradients: of one expert
};

// A product over the rows: the tile's expert and its operands.  SEGS: two K segments.
template <int BM, int BN_OUT, int OUT, bool SEGS>
__device__ __forceinline__ bool row_product(const ExpertArgs &a, TileProb &p, TileAt &at, ExpertTile &t) {
  const TileProb &q = a.p[0];
  const int bm = a.cut == CUT_REST ? 2 * BM : BM;
  if (!expert_tile<true>(a.offsets, a.experts, a.rows, a.tail, bm, a.tiles_n, blockIdx.x, t, a.cut)) return false;
  if (a.cut == CUT_REST && (t.m * BM >= t.rows || t.n * BN_OUT >= q.N)) return false;
  const int64_t row = (int64_t)t.row0 * q.lda;
  const bool none = t.expert == a.experts;  // rows of no expert: zeros
  const int64_t mat = none ? 0 : t.expert * a.b_expert;
  p.A[0] = q.A[0] + row;
  p.A[1] = SEGS ? q.A[1] + row : p.A[0];
  p.B[0] = q.B[0] + mat;
  p.B[1] = SEGS || OUT == OUT_GATE ? q.B[1] + mat : p.B[0];
  p.lda = q.lda, p.ldb = q.ldb;
  p.M = t.rows, p.N = q.N, p.K = none ? 0 : q.K, p.segs = SEGS ? 2 : 1;
  at = {0, 0, t.m, t.n};
  return true;
}

// Its outputs.
template <int OUT>
__device__ __forceinline__ TileProb row_outputs(const ExpertArgs &a, int row0, int rows) {
  TileProb p = a.p[0];
  const int64_t at = (int64_t)row0 * p.ldc;
  p.M = rows;
  if constexpr (OUT == OUT_PART) {
    p.part += at;
    return p;
  }
  p.C += at;
  if constexpr (OUT == OUT_DGATE) {
    p.C2 += at;
    if (p.dots) p.dots += (int64_t)row0 * p.dots_ld;
  }
  if (p.F) p.F += at, p.F2 += at;
  if (p.rw) p.rw += row0;
  return p;
}

// A weight gradient: expert by expert, its matrices' tiles in turn, dealt to the XCDs in runs
// of 32 (a workgroup for each CU of an XCD, 4 x 8 tiles).  A contiguous eighth for each XCD,
// as in the row products, would give XCDs experts of different lengths: 8 experts with up
// to twice the rows of the average took 2285 us against 1310.
__device__ __forceinline__ void weight_product(const ExpertArgs &a, TileProb &p, TileAt &at, int &e) {
  const int total = a.tiles * a.experts, b = (int)blockIdx.x;
  int logical = b;
  if (b < (total & ~255)) logical = (b & ~255) + (b & 7) * 32 + ((b >> 3) & 31);
  e = logical / a.tiles;
  logical -= e * a.tiles;
  at.prob = 0, at.split = 0;
  if (a.n > 1 && logical >= a.p[1].first) at.prob = 1;
  if (a.n > 2 && logical >= a.p[2].first) at.prob = 2;
  const TileProb &s = a.p[at.prob];
  // (scalars: loaded values would be kept in vector registers)
  const int row = within(__builtin_amdgcn_readfirstlane(a.offsets[e]), a.rows);
  const int end = within(__builtin_amdgcn_readfirstlane(a.offsets[e + 1]), a.rows);
  p.lda = s.lda, p.ldb = s.ldb;
  p.A[0] = p.A[1] = s.A[0] + row * s.lda;
  p.B[0] = p.B[1] = s.B[0] + row * s.ldb;
  p.M = s.M, p.N = s.N, p.K = std::max(end - row, 0), p.segs = 1;
  group_coords(logical - s.first, s.tiles_m, s.tiles_n, 4, at.m, at.n);
}

__device__ __forceinline__ TileProb weight_outputs(const ExpertArgs &a, int prob, int e) {
  TileProb p = a.p[prob];
  p.C += e * a.c_expert[prob];
  return p;
}

// The block's small tiles, for few rows an expert: bound by the latency of short K loops.  3000
// rows of 16 experts, 1040 and 712 wide: y 21 us (200 TFLOP/s), dg and du 22.6, dx 36.
template <int BM, int BN, int S, bool AKC, bool BKC, int OUT>
__global__ __launch_bounds__(256) void experts_ring_kernel(ExpertArgs args) {
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  TileProb p;
  TileAt at;
  if constexpr (AKC) {
    ExpertTile t;
    if (!row_product<BM, OUT == OUT_GATE ? BN / 2 : BN, OUT, OUT == OUT_PART && !BKC>(args, p, at, t)) return;
    ring_tile<BM, BN, S, AKC, BKC, OUT, true>(lds, p, at, 1, args.act,
                                              [&]() { return row_outputs<OUT>(args, t.row0, t.rows); });
  } else {
    int e;
    weight_product(args, p, at, e);
    ring_tile<BM, BN, S, AKC, BKC, OUT, true>(lds, p, at, 1, args.act,
                                              [&]() { return weight_outputs(args, at.prob, e); });
  }
}

// The pipelined tiles, bound by the matrix cores under the power limit.  8192 rows of 8 experts,
// 4096 and 5504 wide, with what the whole rounds leave: h 797 us (927 TFLOP/s with g and u
// kept), y 370 (1000), dg and du 473 (780: g and u read, dg and du written), dx 723 (1020), the
// weight gradients 1190 (930: 16 stages a tile, 1.08 GB written).
template <int BM, int NW, bool AKC, bool BKC, int OUT>
__global__ __launch_bounds__(NW * 64, 2) void experts_tile_kernel(ExpertArgs args) {
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  TileProb p;
  TileAt at;
  if constexpr (AKC) {
    ExpertTile t;
    if (!row_product<BM, OUT == OUT_GATE ? BM / 2 : BM, OUT, OUT == OUT_PART && !BKC>(args, p, at, t)) return;
    pipe_tile<BM, NW, AKC, BKC, OUT, true>(lds, p, at, 1, args.act,
                                           [&]() { return row_outputs<OUT>(args, t.row0, t.rows); });
  } else {
    int e;
    weight_product(args, p, at, e);
    pipe_tile<BM, NW, AKC, BKC, OUT, true>(lds, p, at, 1, args.act,
                                           [&]() { return weight_outputs(args, at.prob, e); });
  }
}

// Few rows an expert: 16 MB of them and 16 weight rows a workgroup, bound by reading the busy
// experts' weights once.  One token, 2 experts, 4096 and 11008 wide: h 65 us (5.5 TB/s), y 39.6
// (4.6).
struct ExpertSkinny {
  SkinnyArgs p;
  const int *offsets = nullptr;
  int experts = 0, rows = 0, tail = 0, tiles_n = 0;
};

template <bool GATE, int MB, int NW>
__global__ __launch_bounds__(NW * 64) void experts_skinny_kernel(ExpertSkinny a) {
  __shared__ SkinnySums<GATE, MB, NW> sums;
  ExpertTile t;
  const int bid = (int)grid_block<NW * 64>();  // (below 2^30: 2^18 column tiles of 2048 segments)
  if (!expert_tile<false>(a.offsets, a.experts, a.rows, a.tail, 16 * MB, a.tiles_n, bid, t)) return;
  SkinnyArgs p = a.p;
  const int64_t row = t.row0 + t.m * 16 * MB, weights = (int64_t)p.N * p.K;
  p.M = t.rows - t.m * 16 * MB;
  p.x += row * p.K;
  if (GATE) p.C += row * p.N;
  if (p.F) p.F += row * p.N;
  if (GATE && p.F2) p.F2 += row * p.N;
  if (p.rw) p.rw += row;
  if (t.expert < a.experts) {
    p.w += t.expert * weights;
    if (GATE) p.w2 += t.expert * weights;
  } else {
    p.K = 0;
  }
  skinny_rows<GATE, MB, NW, true>(sums, p, t.n * 16);
}

// dw of a slot: its row's parts, one wave a slot, in a fixed order; 0 for a dropped slot.
__global__ __launch_bounds__(256) void expert_dots_kernel(const int *pos, const int *kept,
                                                          const float *dots, int ld, float *dw,
                                                          int64_t slots, int rows) {
  const int64_t slot = grid_block<256>() * 4 + (threadIdx.x >> 6);
  if (slot >= slots) return;
  const int lane = threadIdx.x & 63, p = pos[slot];
  float sum = 0.0f;
  if (p >= 0 && p < within(*kept, rows))
    for (int c = lane; c < ld; c += 64) sum += dots[(int64_t)p * ld + c];
  sum = wave_sum_dpp(sum);
  if (lane == 0) dw[slot] = sum;
}

// ---------------------------------------------------------------- launch
template <int BM, int BN, int S, bool AKC, bool BKC, int OUT>
hipError_t launch_ring(const ExpertArgs &a, int64_t grid, hipStream_t stream) {
  constexpr size_t lds = size_t(S) * (BM + BN) * kBK * sizeof(uint16_t);
  auto kern = experts_ring_kernel<BM, BN, S, AKC, BKC, OUT>;
  static std::atomic<uint64_t> done{0};
  if (hipError_t e = raise_lds((const void *)kern, lds, done); e != hipSuccess) return e;
  if (!grid_fits(grid, 256)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <int BM, int NW, bool AKC, bool BKC, int OUT>
hipError_t launch_pipe(const ExpertArgs &a, int64_t grid, hipStream_t stream) {
  constexpr size_t lds = size_t(5 * BM) * kBK * sizeof(uint16_t);
  auto kern = experts_tile_kernel<BM, NW, AKC, BKC, OUT>;
  static std::atomic<uint64_t> done{0};
  if (hipError_t e = raise_lds((const void *)kern, lds, done); e != hipSuccess) return e;
  if (!grid_fits(grid, NW * 64)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(NW * 64), lds, stream, a);
  return hipGetLastError();
}

template <bool AKC, bool BKC, int OUT>
hipError_t launch_kernel(int tile, const ExpertArgs &a, int64_t grid, hipStream_t stream) {
  if (grid == 0) return hipSuccess;
  switch (tile) {
    case T_256: return launch_pipe<256, 8, AKC, BKC, OUT>(a, grid, stream);
    case T_128: return launch_pipe<128, 4, AKC, BKC, OUT>(a, grid, stream);
    case T_64S3: return launch_ring<64, 64, 3, AKC, BKC, OUT>(a, grid, stream);
    case T_64S5: return launch_ring<64, 64, 5, AKC, BKC, OUT>(a, grid, stream);
    default: return launch_ring<128, 64, 3, AKC, BKC, OUT>(a, grid, stream);
  }
}

// The experts that the rows reach, at most.
int64_t busy_experts(const ExpertMlp &q) { return std::min(q.R, q.E); }

// The tiles of bm rows to expect: an expert's rows are taken to be spread over 0.4 to 1.6 of the
// average, so one of several tiles leaves half a tile empty, and one of about a tile's
// rows takes one or two.
double likely_tiles(const ExpertMlp &q, int64_t bm) {
  const double b = (double)busy_experts(q), per = (double)q.R / b;
  if (per >= (double)bm) return (double)q.R / (double)bm + b / 2;
  return b * (1.0 + std::max(0.0, (1.6 * per - (double)bm) / (1.2 * per)));
}

// The block's tile costs (mlp_tile.h) hold for the experts too, but for 128 x 128: in the large
// products of 8192 rows and 8 experts, 4096 and 5504 wide, it fell 8 to 12 % behind its
// prediction (y 446 us, 408 on 256 x 256; dx 867 and 792; h 901 and 831); 8192 rows of 32
// experts, 2048 and 1408 wide, h 158 us and 177 on 256 x 256.
double expert_time_us(int tile, int out, double tiles, int64_t stages) {
  return tile_time_us(kTileCost[tile], out, (int64_t)(tiles + 0.5), stages) * (tile == T_128 ? 1.08 : 1.0);
}

// Whether what 256 x 256 tiles leave over their whole rounds goes to 128 x 128 ones (expert_tile.h).
// A last round of few tiles takes 1.2 to 1.6 us a stage, the quarters 0.75 to 0.98, and a
// launch that finds nothing left 3 to 4: 8192 rows of 8 experts, 4096 and 5504 wide, h 826 -> 794
// us (64 stages), dg, du 515 -> 473, y 403 -> 370 (86), dx 761 -> 721 (172).  With 32 stages (32
// experts, 2048 and 1408 wide) h took 165 us so, 177 whole and 156 on 128 x 128 alone.
bool cuts(int tile, int64_t stages) { return tile == T_256 && stages >= 48; }

double rows_time_us(int tile, int out, double tiles, int64_t stages) {
  if (!cuts(tile, stages)) return expert_time_us(tile, out, tiles, stages);
  const double rest = tiles - std::floor(tiles / kTileRound) * kTileRound;
  if (rest < 1 || rest > CUT_REST_MOST) return expert_time_us(tile, out, tiles, stages) + 3.0;
  return expert_time_us(tile, out, tiles - rest, stages) + expert_time_us(T_128, out, 4 * CUT_REST_MOST, stages);
}

int plan_rows(const ExpertMlp &q, int64_t N, int64_t stages, int out) {
  int best = T_64S3;
  double best_us = 1e30;
  for (int t = 0; t < T_COUNT; ++t) {
    const TileCost &c = kTileCost[t];
    const int64_t bn = out == OUT_GATE ? c.bn / 2 : c.bn, tn = (N + bn - 1) / bn;
    if (!grid_fits(tn * expert_tiles_most(q.R, q.E + 1, c.bm), c.threads)) continue;
    const double us = rows_time_us(t, out, (double)tn * likely_tiles(q, c.bm), stages);
    if (us < best_us) best_us = us, best = t;
  }
  return best;
}

template <bool BKC, int OUT>
hipError_t launch_rows(const ExpertMlp &q, ExpertArgs &a, hipStream_t stream) {
  TileProb &p = a.p[0];
  if (q.R == 0 || p.N == 0) return hipSuccess;
  const int64_t stages = (int64_t)((p.K + kBK - 1) / kBK) * p.segs;
  const int tile = plan_rows(q, p.N, stages, OUT);
  const int64_t bm = kTileCost[tile].bm, bn = OUT == OUT_GATE ? kTileCost[tile].bn / 2 : kTileCost[tile].bn;
  a.offsets = q.offsets, a.experts = (int)q.E, a.rows = (int)q.R, a.act = q.act;
  a.tiles_n = (int)((p.N + bn - 1) / bn);
  const int64_t most = a.tiles_n * expert_tiles_most(q.R, q.E + a.tail, bm);
  const bool cut = cuts(tile, stages);
  a.cut = cut ? CUT_ROUNDS : CUT_NONE;
  if (hipError_t e = launch_kernel<true, BKC, OUT>(tile, a, most, stream); e != hipSuccess || !cut) return e;
  a.cut = CUT_REST;
  return launch_kernel<true, BKC, OUT>(T_128, a, 4 * std::min<int64_t>(most, CUT_REST_MOST), stream);
}

int plan_weights(const ExpertMlp &q, const ExpertArgs &a) {
  const int64_t per = q.R / q.E, stages = std::max<int64_t>((per + kBK - 1) / kBK, 1);
  int best = T_64S3;
  double best_us = 1e30;
  for (int t = 0; t < T_COUNT; ++t) {
    const TileCost &c = kTileCost[t];
    int64_t tiles = 0;
    for (int i = 0; i < a.n; ++i)
      tiles += (int64_t)((a.p[i].M + c.bm - 1) / c.bm) * ((a.p[i].N + c.bn - 1) / c.bn);
    if (!grid_fits(tiles * q.E, c.threads)) continue;
    const double us = expert_time_us(t, OUT_STORE, (double)(tiles * q.E), stages);
    if (us < best_us) best_us = us, best = t;
  }
  return best;
}

hipError_t launch_weights(const ExpertMlp &q, ExpertArgs &a, hipStream_t stream) {
  if (a.n == 0) return hipSuccess;
  const int tile = plan_weights(q, a);
  const TileCost &c = kTileCost[tile];
  for (int i = 0; i < a.n; ++i) {
    TileProb &p = a.p[i];
    p.tiles_m = (p.M + c.bm - 1) / c.bm;
    p.tiles_n = (p.N + c.bn - 1) / c.bn;
    p.first = a.tiles;
    a.tiles += p.tiles_m * p.tiles_n;
  }
  a.offsets = q.offsets, a.experts = (int)q.E, a.rows = (int)q.R;
  return launch_kernel<false, false, OUT_STORE>(tile, a, (int64_t)a.tiles * q.E, stream);
}

// The wanted weight gradients.
ExpertArgs weight_args(const ExpertMlp &q, const ExpertMlpGrad &o, bool dwg, bool dwu, bool dwd) {
  ExpertArgs w;
  w.n = 0;
  auto add = [&](const uint16_t *A, int64_t rows, const uint16_t *B, int64_t cols, uint16_t *C) {
    if (rows == 0 || cols == 0) return;
    w.c_expert[w.n] = rows * cols;
    TileProb &p = w.p[w.n++];
    p.A[0] = p.A[1] = A, p.lda = rows;
    p.B[0] = p.B[1] = B, p.ldb = cols;
    p.M = (int)rows, p.N = (int)cols;
    p.C = C, p.ldc = cols;
  };
  if (dwg) add(o.dg, q.I, q.xs, q.K, o.dwg);
  if (dwu) add(o.du, q.I, q.xs, q.K, o.dwu);
  if (dwd) add(o.dys, q.H, q.h, q.I, o.dwd);
  return w;
}

// Rows of one expert, if they are even, up to which the few-row kernel is taken.
bool few_rows(const ExpertMlp &q) { return q.R <= 16 * busy_experts(q); }

template <bool GATE>
hipError_t launch_few(const ExpertMlp &q, ExpertSkinny &a, hipStream_t stream) {
  a.offsets = q.offsets, a.experts = (int)q.E, a.rows = (int)q.R;
  a.tiles_n = (a.p.N + 15) / 16;
  const int64_t grid = a.tiles_n * expert_tiles_most(q.R, q.E + a.tail, 16);
  if (grid == 0) return hipSuccess;
  hipLaunchKernelGGL((experts_skinny_kernel<GATE, 1, 8>), grid_rows<512>(grid), dim3(512), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

const char *experts_kernel_name(const ExpertMlp &q, int product) {
  static const char *const names[T_COUNT] = {"256x256", "128x128", "64x64, 3 stages", "64x64, 5 stages", "128x64"};
  if (product < 2 && few_rows(q)) return "16 rows";
  auto stages = [](int64_t k) { return (k + kBK - 1) / kBK; };
  switch (product) {
    case 0: return names[plan_rows(q, q.I, stages(q.K), OUT_GATE)];
    case 1: return names[plan_rows(q, q.H, stages(q.I), OUT_PART)];
    case 2: return names[plan_rows(q, q.I, stages(q.H), OUT_DGATE)];
    case 3: return names[plan_rows(q, q.K, 2 * stages(q.I), OUT_PART)];
    default: return names[plan_weights(q, weight_args(q, ExpertMlpGrad(), true, true, true))];
  }
}

int64_t expert_dots_ld(const ExpertMlp &q) {
  if (q.R == 0 || q.I == 0) return 0;
  const TileCost &c = kTileCost[plan_rows(q, q.I, (q.H + kBK - 1) / kBK, OUT_DGATE)];
  const int64_t wn = c.bn == 256 ? 64 : c.bn / 2;  // columns of a wave
  return (q.I + wn - 1) / wn;
}

hipError_t launch_experts_mlp(const ExpertMlp &q, hipStream_t stream) {
  if (q.R == 0) return hipSuccess;
  if (few_rows(q)) {
    ExpertSkinny a;
    a.p.x = q.xs, a.p.w = q.wg, a.p.w2 = q.wu, a.p.C = q.h, a.p.F = q.g, a.p.F2 = q.u, a.p.rw = q.rw;
    a.p.N = (int)q.I, a.p.K = (int)q.K, a.p.act = q.act;
    if (hipError_t e = launch_few<true>(q, a, stream); e != hipSuccess) return e;
    ExpertSkinny d;
    d.p.x = q.h, d.p.w = q.wd, d.p.F = q.ys;
    d.p.N = (int)q.H, d.p.K = (int)q.I, d.tail = 1;
    return launch_few<false>(q, d, stream);
  }
  ExpertArgs a;
  TileProb &p = a.p[0];
  p.A[0] = p.A[1] = q.xs, p.lda = q.K;
  p.B[0] = q.wg, p.B[1] = q.wu, p.ldb = q.K;
  p.N = (int)q.I, p.K = (int)q.K;
  p.C = q.h, p.F = q.g, p.F2 = q.u, p.ldc = q.I, p.rw = q.rw;
  a.b_expert = q.I * q.K;
  if (hipError_t e = launch_rows<true, OUT_GATE>(q, a, stream); e != hipSuccess) return e;
  ExpertArgs d;
  TileProb &y = d.p[0];
  y.A[0] = y.A[1] = q.h, y.lda = q.I;
  y.B[0] = y.B[1] = q.wd, y.ldb = q.I;
  y.N = (int)q.H, y.K = (int)q.I;
  y.part = q.ys, y.ldc = q.H;
  d.b_expert = q.H * q.I, d.tail = 1;
  return launch_rows<true, OUT_PART>(q, d, stream);
}

hipError_t launch_experts_mlp_bwd(const ExpertMlp &q, const ExpertMlpGrad &o, hipStream_t stream) {
  if (o.dxs || o.dwg || o.dwu || o.dw) {
    ExpertArgs a;
    TileProb &p = a.p[0];
    p.A[0] = p.A[1] = o.dys, p.lda = q.H;
    p.B[0] = p.B[1] = q.wd, p.ldb = q.I;
    p.N = (int)q.I, p.K = (int)q.H;
    p.C = o.dg, p.C2 = o.du, p.F = q.g, p.F2 = q.u, p.ldc = q.I, p.rw = q.rw;
    p.dots = o.dots, p.dots_ld = (int)expert_dots_ld(q);
    a.b_expert = q.H * q.I;
    if (hipError_t e = launch_rows<false, OUT_DGATE>(q, a, stream); e != hipSuccess) return e;
  }
  if (o.dw && o.slots > 0) {
    const dim3 grid = grid_rows<256>((o.slots + 3) / 4);
    hipLaunchKernelGGL(expert_dots_kernel, grid, dim3(256), 0, stream, o.pos, q.offsets + q.E, o.dots,
                       (int)expert_dots_ld(q), o.dw, o.slots, (int)q.R);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (o.dxs) {
    ExpertArgs a;
    TileProb &p = a.p[0];
    p.A[0] = o.dg, p.A[1] = o.du, p.lda = q.I;
    p.B[0] = q.wg, p.B[1] = q.wu, p.ldb = q.K;
    p.N = (int)q.K, p.K = (int)q.I, p.segs = 2;
    p.part = o.dxs, p.ldc = q.K;
    a.b_expert = q.I * q.K, a.tail = 1;
    if (hipError_t e = launch_rows<false, OUT_PART>(q, a, stream); e != hipSuccess) return e;
  }
  ExpertArgs w = weight_args(q, o, o.dwg, o.dwu, o.dwd);
  return launch_weights(q, w, stream);
}

}  // namespace mj
