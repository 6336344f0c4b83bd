// The boundary between two blocks of a transformer in one pass: the norm after
// a block, its gate, dropout, the residual sum and the norm before the next block.
//
//   c = norm(b) wp + bp   (or b where there is no post norm)
//   y = s x + drop(g c)
//   n = norm(y) wn + bn   (where there is a next norm)
//
// norm(v) = (v - mean) / sqrt(var + eps) (layer) or v / sqrt(mean(v^2) + eps)
// (rms).  s, wp, bp, wn, bn are fp32 vectors, each optional; g is one row for
// every `per` rows of x.  All arithmetic is fp32; y and n are each rounded once
// (n comes from the unrounded y).
//
// Bound by memory: forward reads x, b and writes y, n; backward reads x, b, dy,
// dn and writes dx, db.  A row lives in the registers of a team of TPR threads,
// 8 columns (one 16-byte bf16 access) a thread and VPT such chunks, so every
// value is read once however many sums its row needs.  Teams of one wave to 16
// by width, so that a row's chunks just fit the team.
#include <type_traits>

#include "launch.h"
#include "philox.h"

namespace mj {

// Sums of NV values over a team of TPR threads, the same bits in every thread.
// Larger teams add their waves' sums in wave order through LDS; two LDS slots
// taken in turn, so a sum costs one barrier.
template <int TPR, int NV>
__device__ __forceinline__ void team_sum(float (&v)[NV], float *lds, int &slot) {
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = wave_sum_dpp(v[k]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int team = threadIdx.x / TPR, wave = (threadIdx.x % TPR) / 64;
    float *s = lds + (slot * 16 + team * W) * 2;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < NV; ++k) s[wave * 2 + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float t = s[k];
#pragma unroll
      for (int w = 1; w < W; ++w) t += s[w * 2 + k];
      v[k] = t;
    }
  }
}

template <int VPT>
struct Cols {
  float v[VPT][8];
};

template <int TPR, int VPT, bool ALIGNED, typename T>
__device__ __forceinline__ void load_cols(Cols<VPT> &o, const T *p, int lane, int dim) {
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    const int c = (u * TPR + lane) * 8;
    if (c < dim) load8<ALIGNED>(p + c, dim - c, o.v[u]);
    else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[u][i] = 0.0f;
    }
  }
}

template <int TPR, int VPT, bool ALIGNED, typename T>
__device__ __forceinline__ void store_cols(const Cols<VPT> &o, T *p, int lane, int dim) {
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    const int c = (u * TPR + lane) * 8;
    if (c < dim) store8<ALIGNED>(p + c, dim - c, o.v[u]);
  }
}

// Vectors that may be absent: `fill` in their place.
template <int TPR, int VPT, bool ALIGNED>
__device__ __forceinline__ void load_vec(Cols<VPT> &o, const float *p, float fill, int lane,
                                         int dim) {
  if (p) {
    load_cols<TPR, VPT, ALIGNED>(o, p, lane, dim);
  } else {
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[u][i] = fill;
  }
}

// Row statistics of v: mean (0 for rms) and 1 / std or 1 / rms.  The variance is
// the mean of squared differences from the mean, not a difference of large sums.
template <int TPR, int VPT>
__device__ __forceinline__ void row_stats(const Cols<VPT> &v, bool layer, float eps, int lane,
                                          int dim, float *lds, int &slot, float &mean,
                                          float &rstd) {
  const float inv = 1.0f / (float)dim;
  mean = 0.0f;
  if (layer) {
    float s[1] = {0.0f};
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] += v.v[u][i];  // columns past dim hold zeros
    team_sum<TPR, 1>(s, lds, slot);
    mean = s[0] * inv;
  }
  float q[1] = {0.0f};
#pragma unroll
  for (int u = 0; u < VPT; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = v.v[u][i] - mean;
      if ((u * TPR + lane) * 8 + i < dim) q[0] = __builtin_fmaf(d, d, q[0]);
    }
  team_sum<TPR, 1>(q, lds, slot);
  rstd = 1.0f / sqrtf(q[0] * inv + eps);
}

// The keep factor (0 or scale) of every column of row m.
template <int TPR, int VPT, bool ALIGNED>
__device__ __forceinline__ void keep_bits(uint32_t (&w)[VPT][4], int64_t m, int lane, int dim,
                                          uint64_t seed, uint64_t counter) {
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    const int c = (u * TPR + lane) * 8;
    if (c < dim) draws8<ALIGNED>((uint64_t)m * (uint64_t)dim + c, counter, seed, w[u]);
    else w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0;
  }
}

template <typename T, int TPR, int VPT, bool ALIGNED>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void residual_norm_kernel(ResNorm p) {
  constexpr int TEAMS = (TPR > 256 ? TPR : 256) / TPR;
  __shared__ float lds[64];
  int slot = 0;
  const int lane = threadIdx.x % TPR, dim = (int)p.dim;
  int64_t m = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TPR;
  // a team past the last row computes it again (its barriers are everyone's) and writes nothing
  const bool live = m < p.rows;
  if (!live) m = p.rows - 1;
  const T *x = (const T *)p.x + m * p.dim, *b = p.b ? (const T *)p.b + m * p.dim : nullptr;

  Cols<VPT> y, c;
  load_cols<TPR, VPT, ALIGNED>(y, x, lane, dim);
  if (b) load_cols<TPR, VPT, ALIGNED>(c, b, lane, dim);
  if (p.scale) {
    Cols<VPT> s;
    load_cols<TPR, VPT, ALIGNED>(s, p.scale, lane, dim);
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) y.v[u][i] *= s.v[u][i];
  }
  float mean_p = 0.0f, rstd_p = 1.0f;
  if (b) {
    if (p.wp) {
      row_stats<TPR, VPT>(c, p.layer, p.eps, lane, dim, lds, slot, mean_p, rstd_p);
      Cols<VPT> w, o;
      load_cols<TPR, VPT, ALIGNED>(w, p.wp, lane, dim);
      load_vec<TPR, VPT, ALIGNED>(o, p.bp, 0.0f, lane, dim);
#pragma unroll
      for (int u = 0; u < VPT; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          c.v[u][i] = (c.v[u][i] - mean_p) * rstd_p * w.v[u][i] + o.v[u][i];
    }
    if (p.gate) {
      Cols<VPT> g;
      load_cols<TPR, VPT, ALIGNED>(g, (const T *)p.gate + (m / p.per) * p.dim, lane, dim);
#pragma unroll
      for (int u = 0; u < VPT; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) c.v[u][i] *= g.v[u][i];
    }
    if (p.drop.thr) {
      uint64_t seed, counter;
      dropout_key(p.drop, seed, counter);
      uint32_t w[VPT][4];
      keep_bits<TPR, VPT, ALIGNED>(w, m, lane, dim, seed, counter);
#pragma unroll
      for (int u = 0; u < VPT; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          c.v[u][i] = keep_of(w[u], i, p.drop.thr) ? c.v[u][i] * p.drop.scale : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((u * TPR + lane) * 8 + i < dim) y.v[u][i] += c.v[u][i];
  }
  if (p.y && live) store_cols<TPR, VPT, ALIGNED>(y, (T *)p.y + m * p.dim, lane, dim);
  float mean_n = 0.0f, rstd_n = 1.0f;
  if (p.n) {
    row_stats<TPR, VPT>(y, p.layer, p.eps, lane, dim, lds, slot, mean_n, rstd_n);
    Cols<VPT> w, o;
    load_cols<TPR, VPT, ALIGNED>(w, p.wn, lane, dim);
    load_vec<TPR, VPT, ALIGNED>(o, p.bn, 0.0f, lane, dim);
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        y.v[u][i] = (y.v[u][i] - mean_n) * rstd_n * w.v[u][i] + o.v[u][i];
    if (live) store_cols<TPR, VPT, ALIGNED>(y, (T *)p.n + m * p.dim, lane, dim);
  }
  if (p.stats && live && lane == 0) {
    p.stats[m] = mean_p;
    p.stats[p.rows + m] = rstd_p;
    p.stats[2 * p.rows + m] = mean_n;
    p.stats[3 * p.rows + m] = rstd_n;
  }
}

// Backward.  A team walks a segment of consecutive rows with the columns' sums
// (the gradients of the vectors, and of the gate's row) in its registers:
//   dyt = dy + rn (dn wn - yhat mean(dn wn yhat) - [layer] mean(dn wn))
//   dx = s dyt, ds += x dyt, dz = keep dyt, dgate += dz c, dc = dz g
//   dwn += dn yhat, dbn += dn, dwp += dc bhat, dbp += dc
//   db = rp (dc wp - bhat mean(dc wp bhat) - [layer] mean(dc wp))
// with bhat, c, y and yhat computed again from x, b and the saved statistics, in
// the forward's order, so y is the unrounded one.  A segment lies inside one gate
// row's rows (its dgate goes to the partials) or holds whole groups of them
// (dgate written as it is finished).  No atomics: sums are added in a fixed order.
enum : int { SUM_WN = 0, SUM_BN, SUM_S, SUM_WP, SUM_BP, SUM_G, SUMS };

template <typename T, int TPR, int VPT, bool ALIGNED>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void residual_norm_bwd_kernel(ResNorm p,
                                                                                  ResNormGrad g) {
  constexpr int TEAMS = (TPR > 256 ? TPR : 256) / TPR;
  __shared__ float lds[64];
  int slot = 0;
  const int lane = threadIdx.x % TPR, dim = (int)p.dim;
  const int64_t team = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TPR;
  const bool live = team < g.teams;
  // rows [r0, r1) of groups [g0, g1)
  const int64_t t = live ? team : 0;
  const int64_t g0 = (t / g.segs) * g.groups_per_team;
  int64_t g1 = g0 + g.groups_per_team;
  if (g1 > g.groups) g1 = g.groups;
  const int64_t s0 = (t % g.segs) * g.seg_rows;
  int64_t s1 = s0 + g.seg_rows;
  if (s1 > p.per) s1 = p.per;
  const bool post = p.wp != nullptr, has_b = p.b != nullptr;
  const float inv = 1.0f / (float)dim;
  uint64_t seed = 0, counter = 0;
  if (p.drop.thr) dropout_key(p.drop, seed, counter);

  Cols<VPT> wp, bp, wn, sc, acc[SUMS];
  load_vec<TPR, VPT, ALIGNED>(wp, p.wp, 1.0f, lane, dim);
  load_vec<TPR, VPT, ALIGNED>(bp, p.bp, 0.0f, lane, dim);
  load_vec<TPR, VPT, ALIGNED>(wn, g.dn ? p.wn : nullptr, 0.0f, lane, dim);
  load_vec<TPR, VPT, ALIGNED>(sc, p.scale, 1.0f, lane, dim);
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[k].v[u][i] = 0.0f;

  // every team of a workgroup makes the same number of rounds (barriers inside)
  const int64_t rounds = g.groups_per_team * g.seg_rows;
  int64_t gr = g0, s = s0;
  Cols<VPT> gate;
  load_vec<TPR, VPT, ALIGNED>(gate, nullptr, 1.0f, lane, dim);
  bool fresh = true;
  for (int64_t k = 0; k < rounds; ++k) {
    const bool on = live && gr < g1 && s < s1;
    const int64_t m = on ? gr * p.per + s : 0;
    if (on && fresh && p.gate)
      load_cols<TPR, VPT, ALIGNED>(gate, (const T *)p.gate + gr * p.dim, lane, dim);
    fresh = false;
    Cols<VPT> x, b, dy, dn;
    load_cols<TPR, VPT, ALIGNED>(x, (const T *)p.x + m * p.dim, lane, dim);
    if (has_b) load_cols<TPR, VPT, ALIGNED>(b, (const T *)p.b + m * p.dim, lane, dim);
    else load_vec<TPR, VPT, ALIGNED>(b, nullptr, 0.0f, lane, dim);
    if (g.dy) load_cols<TPR, VPT, ALIGNED>(dy, (const T *)g.dy + m * p.dim, lane, dim);
    else load_vec<TPR, VPT, ALIGNED>(dy, nullptr, 0.0f, lane, dim);
    if (g.dn) load_cols<TPR, VPT, ALIGNED>(dn, (const T *)g.dn + m * p.dim, lane, dim);
    else load_vec<TPR, VPT, ALIGNED>(dn, nullptr, 0.0f, lane, dim);
    const float mean_p = p.stats[m], rstd_p = p.stats[p.rows + m];
    const float mean_n = p.stats[2 * p.rows + m], rstd_n = p.stats[3 * p.rows + m];
    uint32_t w[VPT][4];
    if (p.drop.thr) keep_bits<TPR, VPT, ALIGNED>(w, m, lane, dim, seed, counter);

    // b -> bhat; yhat from x and c
    Cols<VPT> yh;
    float a[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float c = b.v[u][i];
        if (post) {
          b.v[u][i] = (b.v[u][i] - mean_p) * rstd_p;
          c = b.v[u][i] * wp.v[u][i] + bp.v[u][i];
        }
        float z = c * gate.v[u][i];
        if (p.drop.thr) z = keep_of(w[u], i, p.drop.thr) ? z * p.drop.scale : 0.0f;
        const float y = x.v[u][i] * sc.v[u][i] + (has_b ? z : 0.0f);
        yh.v[u][i] = (y - mean_n) * rstd_n;
        const float d = dn.v[u][i] * wn.v[u][i];
        a[0] = __builtin_fmaf(d, yh.v[u][i], a[0]);
        a[1] += d;
      }
    if (g.dn) team_sum<TPR, 2>(a, lds, slot);
    const float ma = a[0] * inv, mb = p.layer ? a[1] * inv : 0.0f;
    float q[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float d = dy.v[u][i];
        if (g.dn) d += rstd_n * (dn.v[u][i] * wn.v[u][i] - yh.v[u][i] * ma - mb);
        if (on) {
          acc[SUM_WN].v[u][i] = __builtin_fmaf(dn.v[u][i], yh.v[u][i], acc[SUM_WN].v[u][i]);
          acc[SUM_BN].v[u][i] += dn.v[u][i];
          acc[SUM_S].v[u][i] = __builtin_fmaf(d, x.v[u][i], acc[SUM_S].v[u][i]);
        }
        x.v[u][i] = d * sc.v[u][i];  // dx
        if (p.drop.thr) d = keep_of(w[u], i, p.drop.thr) ? d * p.drop.scale : 0.0f;
        const float c = post ? b.v[u][i] * wp.v[u][i] + bp.v[u][i] : b.v[u][i];
        const float dc = d * gate.v[u][i];
        if (on) {
          acc[SUM_G].v[u][i] = __builtin_fmaf(d, c, acc[SUM_G].v[u][i]);
          acc[SUM_WP].v[u][i] = __builtin_fmaf(dc, b.v[u][i], acc[SUM_WP].v[u][i]);
          acc[SUM_BP].v[u][i] += dc;
        }
        dn.v[u][i] = dc * wp.v[u][i];
        const bool in = (u * TPR + lane) * 8 + i < dim;
        q[0] = __builtin_fmaf(in ? dn.v[u][i] : 0.0f, in ? b.v[u][i] : 0.0f, q[0]);
        q[1] += in ? dn.v[u][i] : 0.0f;
      }
    if (on && g.dx) store_cols<TPR, VPT, ALIGNED>(x, (T *)g.dx + m * p.dim, lane, dim);
    if (has_b) {
      if (post) {
        team_sum<TPR, 2>(q, lds, slot);
        const float mq = q[0] * inv, mr = p.layer ? q[1] * inv : 0.0f;
#pragma unroll
        for (int u = 0; u < VPT; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dn.v[u][i] = rstd_p * (dn.v[u][i] - b.v[u][i] * mq - mr);
      }
      if (on && g.db) store_cols<TPR, VPT, ALIGNED>(dn, (T *)g.db + m * p.dim, lane, dim);
    }
    if (on && ++s == s1) {
      if (g.dgate && g.segs == 1) {
        store_cols<TPR, VPT, ALIGNED>(acc[SUM_G], (T *)g.dgate + gr * p.dim, lane, dim);
#pragma unroll
        for (int u = 0; u < VPT; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[SUM_G].v[u][i] = 0.0f;
      }
      s = s0;
      ++gr;
      fresh = true;
    }
  }
  if (!live) return;
  float *out[SUMS] = {g.dwn, g.dbn, g.dscale, g.dwp, g.dbp, g.segs > 1 ? (float *)g.dgate : nullptr};
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
    if (out[k])
      store_cols<TPR, VPT, ALIGNED>(acc[k], g.part + ((int64_t)k * g.teams + team) * p.dim, lane,
                                    dim);
}

// Column sums of the teams' partials: 64 columns a workgroup, 16 threads a column
// over the teams in turn, their sums added in order.  blockIdx.y: one of the
// vectors, or SUM_G + a gate row (that row's `segs` teams).
template <typename T>
__global__ __launch_bounds__(1024) void residual_norm_sum_kernel(ResNormGrad g, int64_t dim) {
  __shared__ float red[16][64];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + c;
  const int set = blockIdx.y < SUM_G ? (int)blockIdx.y : (int)SUM_G;
  const int64_t row = (int64_t)blockIdx.y - SUM_G;
  float *const vec[SUM_G] = {g.dwn, g.dbn, g.dscale, g.dwp, g.dbp};
  if (set < SUM_G && !vec[set]) return;
  const int64_t first = set == SUM_G ? row * g.segs : 0, count = set == SUM_G ? g.segs : g.teams;
  const float *part = g.part + ((int64_t)set * g.teams + first) * dim + col;
  float s = 0.0f;
  if (col < dim)
    for (int64_t t = r; t < count; t += 16) s += part[t * dim];
  red[r][c] = s;
  __syncthreads();
  if (r != 0 || col >= dim) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += red[k][c];
  if (set < SUM_G) {
    vec[set][col] = s;
  } else if constexpr (sizeof(T) == 2) {
    ((uint16_t *)g.dgate)[row * dim + col] = (uint16_t)f32_to_bf16_bits(s);
  } else {
    ((float *)g.dgate)[row * dim + col] = s;
  }
}

namespace {

// Whether every row and vector starts on a 16-byte boundary.
bool all_aligned(const ResNorm &p, const ResNormGrad *g) {
  uintptr_t a = (uintptr_t)p.x | (uintptr_t)p.b | (uintptr_t)p.gate | (uintptr_t)p.scale |
                (uintptr_t)p.wp | (uintptr_t)p.bp | (uintptr_t)p.wn | (uintptr_t)p.bn |
                (uintptr_t)p.y | (uintptr_t)p.n;
  if (g) a |= (uintptr_t)g->dy | (uintptr_t)g->dn | (uintptr_t)g->dx | (uintptr_t)g->db |
              (uintptr_t)g->dgate | (uintptr_t)g->part;
  return (a & 15) == 0 && p.dim % 8 == 0;
}

template <typename T, int TPR, int VPT>
hipError_t launch_fwd(const ResNorm &p, hipStream_t stream) {
  constexpr int NT = TPR > 256 ? TPR : 256;
  const int64_t grid = (p.rows + NT / TPR - 1) / (NT / TPR);
  if (grid > INT32_MAX) return hipErrorInvalidValue;
  const dim3 gr((unsigned)grid), bl(NT);
  if (all_aligned(p, nullptr))
    hipLaunchKernelGGL((residual_norm_kernel<T, TPR, VPT, true>), gr, bl, 0, stream, p);
  else
    hipLaunchKernelGGL((residual_norm_kernel<T, TPR, VPT, false>), gr, bl, 0, stream, p);
  return hipGetLastError();
}

template <typename T, int TPR, int VPT>
hipError_t launch_bwd(const ResNorm &p, const ResNormGrad &g, hipStream_t stream) {
  constexpr int NT = TPR > 256 ? TPR : 256;
  const int64_t grid = (g.teams + NT / TPR - 1) / (NT / TPR);
  if (grid > INT32_MAX) return hipErrorInvalidValue;
  const dim3 gr((unsigned)grid), bl(NT);
  if (all_aligned(p, &g))
    hipLaunchKernelGGL((residual_norm_bwd_kernel<T, TPR, VPT, true>), gr, bl, 0, stream, p, g);
  else
    hipLaunchKernelGGL((residual_norm_bwd_kernel<T, TPR, VPT, false>), gr, bl, 0, stream, p, g);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const bool sums = g.dwn || g.dbn || g.dscale || g.dwp || g.dbp;
  const bool gates = g.dgate && g.segs > 1;
  if (!sums && !gates) return hipSuccess;
  const int64_t ny = SUM_G + (gates ? g.groups : 0);
  hipLaunchKernelGGL(residual_norm_sum_kernel<T>, dim3((unsigned)((p.dim + 63) / 64), (unsigned)ny),
                     dim3(1024), 0, stream, g, p.dim);
  return hipGetLastError();
}

// The team that a row's chunks of 8 fit.
template <typename T, typename F>
hipError_t by_width(int64_t dim, F f) {
  if (dim <= 512) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
  if (dim <= 1024) return f(std::integral_constant<int, 128>(), std::integral_constant<int, 1>());
  if (dim <= 2048) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
  if (dim <= 4096) return f(std::integral_constant<int, 512>(), std::integral_constant<int, 1>());
  if (dim <= 8192) return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 1>());
  return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
}

template <typename T>
hipError_t fwd_typed(const ResNorm &p, hipStream_t stream) {
  return by_width<T>(p.dim, [&](auto tpr, auto vpt) {
    return launch_fwd<T, decltype(tpr)::value, decltype(vpt)::value>(p, stream);
  });
}

template <typename T>
hipError_t bwd_typed(const ResNorm &p, const ResNormGrad &g, hipStream_t stream) {
  return by_width<T>(p.dim, [&](auto tpr, auto vpt) {
    return launch_bwd<T, decltype(tpr)::value, decltype(vpt)::value>(p, g, stream);
  });
}

}  // namespace

// Segments of rows for about `kTeams` teams: inside a gate row's group of `per`
// rows where the groups are large, else whole groups.
void plan_residual_norm_bwd(const ResNorm &p, ResNormGrad &g) {
  constexpr int64_t kTeams = 512;
  g.groups = p.rows / p.per;
  const int64_t want = (p.rows + kTeams - 1) / kTeams;  // rows per team
  if (p.per >= want) {
    g.segs = (p.per + want - 1) / want;
    g.seg_rows = (p.per + g.segs - 1) / g.segs;
    g.groups_per_team = 1;
    g.teams = g.groups * g.segs;
  } else {
    g.segs = 1;
    g.seg_rows = p.per;
    g.groups_per_team = want / p.per;
    g.teams = (g.groups + g.groups_per_team - 1) / g.groups_per_team;
  }
}

int64_t residual_norm_part_floats(const ResNormGrad &g, int64_t dim) {
  return (int64_t)SUMS * g.teams * dim;
}

hipError_t launch_residual_norm(bool bf16, const ResNorm &p, hipStream_t stream) {
  if (p.rows <= 0) return hipSuccess;
  return bf16 ? fwd_typed<uint16_t>(p, stream) : fwd_typed<float>(p, stream);
}

hipError_t launch_residual_norm_bwd(bool bf16, const ResNorm &p, const ResNormGrad &g,
                                    hipStream_t stream) {
  if (p.rows <= 0) return hipSuccess;
  return bf16 ? bwd_typed<uint16_t>(p, g, stream) : bwd_typed<float>(p, g, stream);
}

}  // namespace mj
