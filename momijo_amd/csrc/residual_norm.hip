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
#include <algorithm>
#include <atomic>
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

// The 16-bit draws of every column of row m, two a word (keep_of).
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
  constexpr int NT = TPR > 256 ? TPR : 256, TEAMS = NT / TPR;
  __shared__ float lds[64];
  int slot = 0;
  const int lane = threadIdx.x % TPR, dim = (int)p.dim;
  // (a wave is of one team, so its row is uniform)
  const int64_t first = grid_block<NT>() * TEAMS;
  int64_t m = first + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
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

// Backward:
//   dyt = dy + rn (dn wn - yhat mean(dn wn yhat) - [layer] mean(dn wn))
//   dx = s dyt, ds += x dyt, dz = keep dyt, dgate += dz c, dc = dz g
//   (a dropped element: dgate and dc take 0 without looking at c and g, which may be inf or NaN)
//   dwn += dn yhat, dbn += dn, dwp += dc bhat, dbp += dc
//   db = rp (dc wp - bhat mean(dc wp bhat) - [layer] mean(dc wp))
// with bhat, c, y and yhat computed again from x, b and the saved statistics, in
// the forward's order, so y is the unrounded one.
//
// A workgroup of 512 threads (512 / TPR teams) walks a segment of rows, its teams in
// turn, with the columns' sums in registers; the teams' sums are added through LDS at
// the end and the workgroup writes one partial row for each vector.  A segment lies
// inside one gate row's rows (its dgate goes to the partials too), or, where the groups
// are small, is a run of whole groups dealt to the teams, which write dgate as they
// finish one.  No atomics: sums are added in a fixed order.
//
// Rows of more than 8192 columns have no registers for the columns' sums: there one kernel
// takes the rows' four means, and a second one, eight columns a thread and nothing to
// reduce, walks the rows again and does the rest: 2048 x 16384 bf16 with dropout 99 + 98 us
// and 13 for the partials' sums, 611 with all in one kernel (spills).
//
// What bounds it is latency (a row's loads, then two sums over it, one after the
// other) and, near the memory rate, the vector unit (some 60 operations an element).
// Two workgroups on a CU cover each other's waits, so a thread has 128 registers: they
// go to the sums; what a row needs again is computed again from its packed values, and
// the vectors wait in LDS, each thread's own columns in its own slots (no barrier, no
// bank conflicts).  8192 x 4096 bf16 with dropout and four gate rows: 111 us with the
// partials' sums (403 MB, 3.6 TB/s).  Built otherwise, while those sums took 7 us more
// (118): with the next row's loads ahead 202 (spills at 128 registers) or 141 (one
// workgroup a CU); with the vectors in registers, one workgroup a CU, 182.
enum : int { SUM_WN = 0, SUM_BN, SUM_S, SUM_WP, SUM_BP, SUM_G, SUMS };
enum : int { V_WN = 0, V_WP, V_GATE, V_SCALE, V_BP, VECS };
constexpr int kBwdThreads = 512;

// 8 consecutive elements as they are stored.
template <typename T>
struct Pack8;
template <>
struct Pack8<uint16_t> {
  uint32_t w[4];
  template <bool ALIGNED>
  __device__ __forceinline__ void load(const uint16_t *p, int n) {
    if (ALIGNED || n >= 8) {
      if constexpr (ALIGNED) {
        const uint4 q = *(const uint4 *)p;
        w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
      } else {
        const u32x4_a2 q = *(const u32x4_a2 *)p;
        w[0] = q[0], w[1] = q[1], w[2] = q[2], w[3] = q[3];
      }
    } else {
      w[0] = w[1] = w[2] = w[3] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    }
  }
  __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0; }
  __device__ __forceinline__ float get(int i) const {
    return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
  }
};
template <>
struct Pack8<float> {
  float v[8];
  template <bool ALIGNED>
  __device__ __forceinline__ void load(const float *p, int n) { load8<ALIGNED>(p, n, v); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  }
  __device__ __forceinline__ float get(int i) const { return v[i]; }
};

template <typename T, int VPT>
struct RowIn {  // x, b, dy, dn of a row's columns
  Pack8<T> x[VPT], b[VPT], dy[VPT], dn[VPT];
  float mean_p, rstd_p, mean_n, rstd_n;
};

// A row's address for a lane: the row uniform, the lane's byte offset 32 bits.
template <typename T>
__device__ __forceinline__ T *lane_at(T *row, uint32_t bytes) {
  return (T *)((char *)row + bytes);
}
template <typename T>
__device__ __forceinline__ const T *lane_at(const T *row, uint32_t bytes) {
  return (const T *)((const char *)row + bytes);
}

// The vectors that wait in LDS (slots of 16 KB VPT); the others are read from memory
// for every row.
constexpr bool vec_in_lds(int v, int vpt, bool bias) {
  return v < V_BP || (vpt == 1 && bias);
}
constexpr int lds_vecs(int vpt, bool bias) {
  int n = 0;
  for (int v = 0; v < VECS; ++v) n += vec_in_lds(v, vpt, bias);
  return n;
}

// BIAS: the biases are there (their gradients' sums, and bp in c).
template <typename T, int TPR, int VPT, bool ALIGNED, bool BIAS>
__global__ __launch_bounds__(kBwdThreads, (VPT == 1 && !BIAS ? 4 : 2)) void
residual_norm_bwd_kernel(ResNorm p, ResNormGrad g) {
  constexpr int TEAMS = kBwdThreads / TPR;
  __shared__ float lds[64];
  extern __shared__ __attribute__((aligned(16))) float vecs[];
  int slot = 0;
  const int tid = threadIdx.x, dim = (int)p.dim;
  const uint32_t lane = (uint32_t)tid % TPR;
  const int team = __builtin_amdgcn_readfirstlane(tid / TPR);  // a wave is of one team
  const bool inside = g.segs > 0;  // segments inside groups, else whole groups
  // this workgroup's ns rows of group g0, or ng whole groups; row numbers count from m0
  // (the last segments may lie past their group's end: no rows)
  const int per = (int)p.per;
  int64_t g0, m0;
  int ng, ns, rounds;
  if (inside) {
    g0 = blockIdx.x / (uint32_t)g.segs;
    const uint32_t s0 = (blockIdx.x % (uint32_t)g.segs) * (uint32_t)g.seg_rows;
    m0 = g0 * per + s0;
    ng = 1;
    ns = s0 < (uint32_t)per ? (int)std::min((uint32_t)g.seg_rows, (uint32_t)per - s0) : 0;
    rounds = ((int)g.seg_rows + TEAMS - 1) / TEAMS;
  } else {
    g0 = (int64_t)blockIdx.x * g.groups_per_block;
    m0 = g0 * per;
    ng = (int)std::min(g.groups_per_block, g.groups - g0);
    ns = per;
    rounds = ((int)g.groups_per_block + TEAMS - 1) / TEAMS * per;
  }
  const bool post = p.wp != nullptr, has_b = p.b != nullptr, drop = p.drop.thr != 0;
  const bool next = g.dn != nullptr;
  const float inv = 1.0f / (float)dim;
  uint64_t seed = 0, counter = 0;
  if (drop) dropout_key(p.drop, seed, counter);

  auto col = [&](int u) { return (int)(u * TPR + lane) * 8; };
  // the vectors: this thread's columns in its own LDS slots
  auto at = [&](int v, int u, int h) { return vecs + (((v * VPT + u) * 2 + h) * kBwdThreads + tid) * 4; };
  auto keep_vec = [&](int v, const auto *src, float fill) __attribute__((always_inline)) {
    if (!vec_in_lds(v, VPT, BIAS)) return;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = fill;
      if (src && col(u) < dim) load8<ALIGNED>(src + col(u), dim - col(u), t);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *(float4 *)at(v, u, h) = make_float4(t[4 * h], t[4 * h + 1], t[4 * h + 2], t[4 * h + 3]);
    }
  };
  auto get_vec = [&](float (&t)[4], int v, const auto *src, float fill, int u, int h)
      __attribute__((always_inline)) {
    if (vec_in_lds(v, VPT, BIAS)) {
      const float4 q = *(const float4 *)at(v, u, h);
      t[0] = q.x, t[1] = q.y, t[2] = q.z, t[3] = q.w;
    } else {
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = fill;
      if (src && col(u) < dim) load8<ALIGNED>(src + col(u), dim - col(u), o);
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = o[4 * h + i];
    }
  };
  const float *const wn = next ? p.wn : nullptr;
  keep_vec(V_WN, wn, 0.0f);
  keep_vec(V_WP, p.wp, 1.0f);
  keep_vec(V_SCALE, p.scale, 1.0f);
  keep_vec(V_BP, p.bp, 0.0f);
  if (!p.gate) keep_vec(V_GATE, (const T *)nullptr, 1.0f);

  int gr = inside ? 0 : team, s = inside ? team : 0;
  auto alive = [&](int gr_, int s_) { return gr_ < ng && s_ < ns; };
  auto step = [&](int &gr_, int &s_) {
    if (inside) s_ += TEAMS;
    else if (++s_ == per) s_ = 0, gr_ += TEAMS;
  };
  auto load_row = [&](RowIn<T, VPT> &r, int gr_, int s_) __attribute__((always_inline)) {
    const int64_t m = alive(gr_, s_) ? m0 + gr_ * per + s_ : 0, base = m * dim;
    const T *x = (const T *)p.x + base, *b = (const T *)p.b + base;
    const T *dy = (const T *)g.dy + base, *dn = (const T *)g.dn + base;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const uint32_t o = (u * TPR + lane) * 8 * (uint32_t)sizeof(T);
      const int left = dim - col(u);
      r.x[u].clear(), r.b[u].clear(), r.dy[u].clear(), r.dn[u].clear();
      if (left > 0) {
        r.x[u].template load<ALIGNED>(lane_at(x, o), left);
        if (has_b) r.b[u].template load<ALIGNED>(lane_at(b, o), left);
        if (g.dy) r.dy[u].template load<ALIGNED>(lane_at(dy, o), left);
        if (next) r.dn[u].template load<ALIGNED>(lane_at(dn, o), left);
      }
    }
    r.mean_p = p.stats[m], r.rstd_p = p.stats[p.rows + m];
    r.mean_n = p.stats[2 * p.rows + m], r.rstd_n = p.stats[3 * p.rows + m];
  };

  Cols<VPT> acc[SUMS];
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[k].v[u][i] = 0.0f;

  bool fresh = true;
  RowIn<T, VPT> r;
  for (int k = 0; k < rounds; ++k) {
    const bool on = alive(gr, s);
    const int64_t m = on ? m0 + gr * per + s : 0;
    const T *const gate = p.gate ? (const T *)p.gate + (on ? g0 + gr : 0) * dim : nullptr;
    if (fresh && gate) keep_vec(V_GATE, gate, 1.0f);
    fresh = false;
    load_row(r, gr, s);
    uint32_t w[VPT][4];
    if (drop) keep_bits<TPR, VPT, ALIGNED>(w, m, lane, dim, seed, counter);

    // yhat from x and c, four columns at a time (the vectors' registers)
    Cols<VPT> yh;
    float a[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float vwp[4], vbp[4], vg[4], vs[4], vn[4];
        get_vec(vwp, V_WP, p.wp, 1.0f, u, h);
        get_vec(vbp, V_BP, p.bp, 0.0f, u, h);
        get_vec(vg, V_GATE, gate, 1.0f, u, h);
        get_vec(vs, V_SCALE, p.scale, 1.0f, u, h);
        get_vec(vn, V_WN, wn, 0.0f, u, h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * h + j;
          const float c = (r.b[u].get(i) - r.mean_p) * r.rstd_p * vwp[j] + vbp[j];
          float z = c * vg[j];
          if (drop) z = keep_of(w[u], i, p.drop.thr) ? z * p.drop.scale : 0.0f;
          const float y = r.x[u].get(i) * vs[j] + (has_b ? z : 0.0f);
          yh.v[u][i] = (y - r.mean_n) * r.rstd_n;
          const float d = r.dn[u].get(i) * vn[j];
          a[0] = __builtin_fmaf(d, yh.v[u][i], a[0]);
          a[1] += d;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    if (next) team_sum<TPR, 2>(a, lds, slot);
    const float ma = a[0] * inv, mb = p.layer ? a[1] * inv : 0.0f;
    float q[2] = {0.0f, 0.0f};
    Cols<VPT> e;
    T *const dx = on && g.dx ? (T *)g.dx + m * dim : nullptr;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int c0 = col(u);
      float out[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float vwp[4], vbp[4], vg[4], vs[4], vn[4];
        get_vec(vwp, V_WP, p.wp, 1.0f, u, h);
        get_vec(vbp, V_BP, p.bp, 0.0f, u, h);
        get_vec(vg, V_GATE, gate, 1.0f, u, h);
        get_vec(vs, V_SCALE, p.scale, 1.0f, u, h);
        get_vec(vn, V_WN, wn, 0.0f, u, h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * h + j;
          const float dn = r.dn[u].get(i), bh = (r.b[u].get(i) - r.mean_p) * r.rstd_p;
          float d = r.dy[u].get(i);
          if (next) d += r.rstd_n * (dn * vn[j] - yh.v[u][i] * ma - mb);
          out[i] = d * vs[j];
          // a dropped element's gradients are 0 whatever c and the gate hold
          float dk = d;
          if (drop) dk = d * p.drop.scale;
          const bool kept = !drop || keep_of(w[u], i, p.drop.thr);
          const float dc = kept ? dk * vg[j] : 0.0f;
          if (on) {
            acc[SUM_WN].v[u][i] = __builtin_fmaf(dn, yh.v[u][i], acc[SUM_WN].v[u][i]);
            acc[SUM_S].v[u][i] = __builtin_fmaf(d, r.x[u].get(i), acc[SUM_S].v[u][i]);
            if (kept)
              acc[SUM_G].v[u][i] = __builtin_fmaf(dk, bh * vwp[j] + vbp[j], acc[SUM_G].v[u][i]);
            acc[SUM_WP].v[u][i] = __builtin_fmaf(dc, bh, acc[SUM_WP].v[u][i]);
            if constexpr (BIAS) {
              acc[SUM_BN].v[u][i] += dn;
              acc[SUM_BP].v[u][i] += dc;
            }
          }
          e.v[u][i] = c0 + i < dim ? dc * vwp[j] : 0.0f;
          q[0] = __builtin_fmaf(e.v[u][i], c0 + i < dim ? bh : 0.0f, q[0]);
          q[1] += e.v[u][i];
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (dx && c0 < dim)
        store8<ALIGNED>(lane_at(dx, (uint32_t)c0 * (uint32_t)sizeof(T)), dim - c0, out);
    }
    if (has_b) {
      if (post) {
        team_sum<TPR, 2>(q, lds, slot);
        const float mq = q[0] * inv, mr = p.layer ? q[1] * inv : 0.0f;
#pragma unroll
        for (int u = 0; u < VPT; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float bh = (r.b[u].get(i) - r.mean_p) * r.rstd_p;
            e.v[u][i] = r.rstd_p * (e.v[u][i] - bh * mq - mr);
          }
      }
      if (on && g.db) {
        T *const db = (T *)g.db + m * dim;
#pragma unroll
        for (int u = 0; u < VPT; ++u)
          if (col(u) < dim)
            store8<ALIGNED>(lane_at(db, (uint32_t)col(u) * (uint32_t)sizeof(T)), dim - col(u),
                            e.v[u]);
      }
    }
    if (on && !inside && s == per - 1) {
      if (g.dgate)
        store_cols<TPR, VPT, ALIGNED>(acc[SUM_G], (T *)g.dgate + (g0 + gr) * dim, lane, dim);
#pragma unroll
      for (int u = 0; u < VPT; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[SUM_G].v[u][i] = 0.0f;
      fresh = true;
    }
    step(gr, s);
  }
  float *const out[SUMS] = {g.dwn, g.dbn, g.dscale, g.dwp, g.dbp, inside ? (float *)g.dgate : nullptr};
#pragma unroll
  for (int k = 0; k < SUMS; ++k) {
    if (!BIAS && (k == SUM_BN || k == SUM_BP)) continue;
    if (!out[k]) continue;
    if constexpr (TEAMS > 1) {
      // thread tid of team 0 adds its columns of every team
      __syncthreads();
#pragma unroll
      for (int u = 0; u < VPT; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *(float4 *)at(0, u, h) = make_float4(acc[k].v[u][4 * h], acc[k].v[u][4 * h + 1],
                                               acc[k].v[u][4 * h + 2], acc[k].v[u][4 * h + 3]);
      __syncthreads();
      if (team == 0) {
#pragma unroll
        for (int t = 1; t < TEAMS; ++t)
#pragma unroll
          for (int u = 0; u < VPT; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float4 f = *(const float4 *)(at(0, u, h) + t * TPR * 4);
              acc[k].v[u][4 * h] += f.x, acc[k].v[u][4 * h + 1] += f.y;
              acc[k].v[u][4 * h + 2] += f.z, acc[k].v[u][4 * h + 3] += f.w;
            }
      }
    }
    if (team == 0)
      store_cols<TPR, VPT, ALIGNED>(acc[k], g.part + ((int64_t)k * g.blocks + blockIdx.x) * p.dim,
                                    lane, dim);
  }
}

// The rows' means of dn wn yhat, dn wn, dc wp bhat and dc wp, [4][rows] behind the partials
// (rows of more than 8192 columns).
__device__ __forceinline__ float *row_means(const ResNorm &p, const ResNormGrad &g) {
  return g.part + (int64_t)SUMS * g.blocks * p.dim;
}

// A workgroup a row.  The products of the row's columns that both passes need stay in
// registers (88 of 128 with the gradients).
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(1024) void residual_norm_means_kernel(ResNorm p, ResNormGrad g) {
  constexpr int TPR = 1024, VPT = 2;
  __shared__ float lds[64];
  int slot = 0;
  const int lane = threadIdx.x, dim = (int)p.dim;
  const int64_t m = grid_block<TPR>(), base = m * dim;
  if (m >= p.rows) return;
  const float mean_p = p.stats[m], rstd_p = p.stats[p.rows + m];
  const float mean_n = p.stats[2 * p.rows + m], rstd_n = p.stats[3 * p.rows + m];
  const bool drop = p.drop.thr != 0;
  uint32_t w[VPT][4];
  if (drop) {
    uint64_t seed, counter;
    dropout_key(p.drop, seed, counter);
    keep_bits<TPR, VPT, ALIGNED>(w, m, lane, dim, seed, counter);
  }
  Cols<VPT> yh, bh, gw, t;  // y, then yhat; b, then bhat; gate wp
  load_cols<TPR, VPT, ALIGNED>(yh, (const T *)p.x + base, lane, dim);
  load_vec<TPR, VPT, ALIGNED>(t, p.scale, 1.0f, lane, dim);
#pragma unroll
  for (int u = 0; u < VPT; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      yh.v[u][i] *= t.v[u][i];
      bh.v[u][i] = 0.0f;
    }
  load_vec<TPR, VPT, ALIGNED>(gw, p.wp, 1.0f, lane, dim);
  if (p.b) {
    Cols<VPT> gate;
    load_cols<TPR, VPT, ALIGNED>(bh, (const T *)p.b + base, lane, dim);
    load_vec<TPR, VPT, ALIGNED>(t, p.bp, 0.0f, lane, dim);
    if (p.gate) {
      load_cols<TPR, VPT, ALIGNED>(gate, (const T *)p.gate + m / p.per * dim, lane, dim);
    } else {
#pragma unroll
      for (int u = 0; u < VPT; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) gate.v[u][i] = 1.0f;
    }
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bh.v[u][i] = (bh.v[u][i] - mean_p) * rstd_p;
        float z = (bh.v[u][i] * gw.v[u][i] + t.v[u][i]) * gate.v[u][i];
        if (drop) z = keep_of(w[u], i, p.drop.thr) ? z * p.drop.scale : 0.0f;
        yh.v[u][i] += z;
        gw.v[u][i] *= gate.v[u][i];
      }
  }
#pragma unroll
  for (int u = 0; u < VPT; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) yh.v[u][i] = (yh.v[u][i] - mean_n) * rstd_n;
  Cols<VPT> d;  // dn wn, then dy of the row's sum
  float a[2] = {0.0f, 0.0f}, q[2] = {0.0f, 0.0f};
  const float inv = 1.0f / (float)dim;
  if (g.dn) {
    load_cols<TPR, VPT, ALIGNED>(d, (const T *)g.dn + base, lane, dim);
    load_cols<TPR, VPT, ALIGNED>(t, p.wn, lane, dim);
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        d.v[u][i] *= t.v[u][i];
        a[0] = __builtin_fmaf(d.v[u][i], yh.v[u][i], a[0]);
        a[1] += d.v[u][i];
      }
    team_sum<TPR, 2>(a, lds, slot);
    a[0] *= inv;
    a[1] = p.layer ? a[1] * inv : 0.0f;
  }
  if (p.wp) {
    if (g.dy) load_cols<TPR, VPT, ALIGNED>(t, (const T *)g.dy + base, lane, dim);
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = g.dy ? t.v[u][i] : 0.0f;
        if (g.dn) v += rstd_n * (d.v[u][i] - yh.v[u][i] * a[0] - a[1]);
        if (drop) v *= p.drop.scale;
        const bool in = (u * TPR + lane) * 8 + i < dim;
        const bool kept = !drop || keep_of(w[u], i, p.drop.thr);
        const float e = in && kept ? v * gw.v[u][i] : 0.0f;
        q[0] = __builtin_fmaf(e, in ? bh.v[u][i] : 0.0f, q[0]);
        q[1] += e;
      }
    team_sum<TPR, 2>(q, lds, slot);
  }
  if (lane == 0) {
    float *const means = row_means(p, g);
    means[m] = a[0];
    means[p.rows + m] = a[1];
    means[2 * p.rows + m] = q[0] * inv;
    means[3 * p.rows + m] = p.layer ? q[1] * inv : 0.0f;
  }
}

// Wide rows' gradients and their columns' sums from the rows' means: eight columns a
// thread, the workgroup's rows in turn (blockIdx.x as in residual_norm_bwd_kernel,
// blockIdx.y a run of 2048 columns).
constexpr int kColThreads = 256;
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(kColThreads) void residual_norm_cols_kernel(ResNorm p, ResNormGrad g) {
  const int dim = (int)p.dim, c0 = ((int)blockIdx.y * kColThreads + (int)threadIdx.x) * 8;
  const int left = dim - c0;
  if (left <= 0) return;
  const bool inside = g.segs > 0, has_b = p.b != nullptr, drop = p.drop.thr != 0;
  const bool next = g.dn != nullptr, post = p.wp != nullptr;
  int64_t g0, g1, s0, s1;
  if (inside) {
    g0 = (int64_t)blockIdx.x / g.segs;
    g1 = g0 + 1;
    s0 = (int64_t)blockIdx.x % g.segs * g.seg_rows;
    s1 = std::min(s0 + g.seg_rows, p.per);
  } else {
    g0 = (int64_t)blockIdx.x * g.groups_per_block;
    g1 = std::min(g0 + g.groups_per_block, g.groups);
    s0 = 0;
    s1 = p.per;
  }
  uint64_t seed = 0, counter = 0;
  if (drop) dropout_key(p.drop, seed, counter);
  const float *const means = row_means(p, g);
  auto vec = [&](float (&v)[8], const auto *src, float fill) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fill;
    if (src) load8<ALIGNED>(src + c0, left, v);
  };
  float wn[8], wp[8], bp[8], gate[8], acc[SUMS][8];
  vec(wn, next ? p.wn : nullptr, 0.0f);
  vec(wp, p.wp, 1.0f);
  vec(bp, p.bp, 0.0f);
  float scale[8];
  vec(scale, p.scale, 1.0f);
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[k][i] = 0.0f;

  for (int64_t gr = g0; gr < g1; ++gr) {
    vec(gate, p.gate ? (const T *)p.gate + gr * dim : nullptr, 1.0f);
    for (int64_t r = s0; r < s1; ++r) {
      const int64_t m = gr * p.per + r, base = m * dim + c0;
      Pack8<T> x, b, dy, dn;
      b.clear(), dy.clear(), dn.clear();
      x.template load<ALIGNED>((const T *)p.x + base, left);
      if (has_b) b.template load<ALIGNED>((const T *)p.b + base, left);
      if (g.dy) dy.template load<ALIGNED>((const T *)g.dy + base, left);
      if (next) dn.template load<ALIGNED>((const T *)g.dn + base, left);
      uint32_t w[4];
      if (drop) draws8<ALIGNED>((uint64_t)base, counter, seed, w);
      const float mean_p = p.stats[m], rstd_p = p.stats[p.rows + m];
      const float mean_n = p.stats[2 * p.rows + m], rstd_n = p.stats[3 * p.rows + m];
      const float ma = means[m], mb = means[p.rows + m];
      const float mq = means[2 * p.rows + m], mr = means[3 * p.rows + m];
      float dx[8], db[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool kept = !drop || keep_of(w, i, p.drop.thr);
        const float bh = (b.get(i) - mean_p) * rstd_p, c = bh * wp[i] + bp[i];
        float z = c * gate[i];
        if (drop) z = kept ? z * p.drop.scale : 0.0f;
        const float y = x.get(i) * scale[i] + (has_b ? z : 0.0f);
        const float yh = (y - mean_n) * rstd_n;
        float d = dy.get(i);
        if (next) d += rstd_n * (dn.get(i) * wn[i] - yh * ma - mb);
        const float dk = drop ? d * p.drop.scale : d;
        const float dc = kept ? dk * gate[i] : 0.0f, e = dc * wp[i];
        dx[i] = d * scale[i];
        db[i] = post ? rstd_p * (e - bh * mq - mr) : e;
        acc[SUM_WN][i] = __builtin_fmaf(dn.get(i), yh, acc[SUM_WN][i]);
        acc[SUM_BN][i] += dn.get(i);
        acc[SUM_S][i] = __builtin_fmaf(d, x.get(i), acc[SUM_S][i]);
        acc[SUM_WP][i] = __builtin_fmaf(dc, bh, acc[SUM_WP][i]);
        acc[SUM_BP][i] += dc;
        if (kept) acc[SUM_G][i] = __builtin_fmaf(dk, c, acc[SUM_G][i]);
      }
      if (g.dx) store8<ALIGNED>((T *)g.dx + base, left, dx);
      if (g.db) store8<ALIGNED>((T *)g.db + base, left, db);
    }
    if (!inside) {
      if (g.dgate) store8<ALIGNED>((T *)g.dgate + gr * dim + c0, left, acc[SUM_G]);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[SUM_G][i] = 0.0f;
    }
  }
  float *const out[SUMS] = {g.dwn, g.dbn, g.dscale, g.dwp, g.dbp, inside ? (float *)g.dgate : nullptr};
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
    if (out[k])
      store8<ALIGNED>(g.part + ((int64_t)k * g.blocks + blockIdx.x) * dim + c0, left, acc[k]);
}

// Column sums of the workgroups' partials: 64 columns a workgroup, 16 threads a column
// over the partials in turn, their sums added in order.  blockIdx.y: one of the
// vectors, or SUM_G + a gate row (that row's `segs` partials).
template <typename T>
__global__ __launch_bounds__(1024) void residual_norm_sum_kernel(ResNormGrad g, int64_t dim) {
  __shared__ float red[16][64];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + c;
  const int set = blockIdx.y < SUM_G ? (int)blockIdx.y : (int)SUM_G;
  const int64_t row = (int64_t)blockIdx.y - SUM_G;
  float *const vec[SUM_G] = {g.dwn, g.dbn, g.dscale, g.dwp, g.dbp};
  if (set < SUM_G && !vec[set]) return;
  const int64_t first = set == SUM_G ? row * g.segs : 0, count = set == SUM_G ? g.segs : g.blocks;
  const float *part = g.part + ((int64_t)set * g.blocks + first) * dim + col;
  float s = 0.0f;
  if (col < dim) {
    int64_t t = r;
    for (; t + 7 * 16 < count; t += 8 * 16) {  // eight loads in flight
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[(t + 16 * k) * dim];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    for (; t < count; t += 16) s += part[t * dim];
  }
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
  const dim3 gr = grid_rows<NT>((p.rows + NT / TPR - 1) / (NT / TPR)), bl(NT);
  if (all_aligned(p, nullptr))
    hipLaunchKernelGGL((residual_norm_kernel<T, TPR, VPT, true>), gr, bl, 0, stream, p);
  else
    hipLaunchKernelGGL((residual_norm_kernel<T, TPR, VPT, false>), gr, bl, 0, stream, p);
  return hipGetLastError();
}

template <typename T, int TPR, int VPT, bool ALIGNED, bool BIAS>
hipError_t launch_bwd_kernel(const ResNorm &p, const ResNormGrad &g, hipStream_t stream) {
  constexpr size_t lds = (size_t)kBwdThreads * 8 * VPT * sizeof(float) * lds_vecs(VPT, BIAS);
  auto kern = residual_norm_bwd_kernel<T, TPR, VPT, ALIGNED, BIAS>;
  static std::atomic<uint64_t> done{0};
  if (hipError_t e = raise_lds((const void *)kern, lds, done); e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)g.blocks), dim3(kBwdThreads), lds, stream, p, g);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_bwd_sums(const ResNorm &p, const ResNormGrad &g, hipStream_t stream) {
  const bool sums = g.dwn || g.dbn || g.dscale || g.dwp || g.dbp;
  const bool gates = g.dgate && g.segs > 0;
  if (!sums && !gates) return hipSuccess;
  const int64_t ny = SUM_G + (gates ? g.groups : 0);
  hipLaunchKernelGGL(residual_norm_sum_kernel<T>, dim3((unsigned)((p.dim + 63) / 64), (unsigned)ny),
                     dim3(1024), 0, stream, g, p.dim);
  return hipGetLastError();
}

template <typename T, int TPR, int VPT>
hipError_t launch_bwd(const ResNorm &p, const ResNormGrad &g, hipStream_t stream) {
  const bool bias = residual_norm_bias(p, g);
  hipError_t e;
  if (all_aligned(p, &g))
    e = bias ? launch_bwd_kernel<T, TPR, VPT, true, true>(p, g, stream)
             : launch_bwd_kernel<T, TPR, VPT, true, false>(p, g, stream);
  else
    e = bias ? launch_bwd_kernel<T, TPR, VPT, false, true>(p, g, stream)
             : launch_bwd_kernel<T, TPR, VPT, false, false>(p, g, stream);
  return e != hipSuccess ? e : launch_bwd_sums<T>(p, g, stream);
}

template <typename T, bool ALIGNED>
hipError_t launch_bwd_wide(const ResNorm &p, const ResNormGrad &g, hipStream_t stream) {
  hipLaunchKernelGGL((residual_norm_means_kernel<T, ALIGNED>), grid_rows<1024>(p.rows), dim3(1024), 0,
                     stream, p, g);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const dim3 grid((unsigned)g.blocks, (unsigned)((p.dim + 8 * kColThreads - 1) / (8 * kColThreads)));
  hipLaunchKernelGGL((residual_norm_cols_kernel<T, ALIGNED>), grid, dim3(kColThreads), 0, stream, p, g);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_bwd_sums<T>(p, g, stream);
}

// The team that a row's chunks of 8 fit.
template <typename F>
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
  return by_width(p.dim, [&](auto tpr, auto vpt) {
    return launch_fwd<T, decltype(tpr)::value, decltype(vpt)::value>(p, stream);
  });
}

// Backward teams: one to eight waves of a workgroup of 512 threads.
int bwd_team(int64_t dim) { return dim <= 512 ? 64 : dim <= 1024 ? 128 : dim <= 2048 ? 256 : 512; }

template <typename T>
hipError_t bwd_typed(const ResNorm &p, const ResNormGrad &g, hipStream_t stream) {
  switch (bwd_team(p.dim)) {
    case 64: return launch_bwd<T, 64, 1>(p, g, stream);
    case 128: return launch_bwd<T, 128, 1>(p, g, stream);
    case 256: return launch_bwd<T, 256, 1>(p, g, stream);
    default: break;
  }
  if (p.dim <= 4096) return launch_bwd<T, 512, 1>(p, g, stream);
  if (p.dim <= 8192) return launch_bwd<T, 512, 2>(p, g, stream);
  return all_aligned(p, &g) ? launch_bwd_wide<T, true>(p, g, stream)
                            : launch_bwd_wide<T, false>(p, g, stream);
}

}  // namespace

// Rows for about as many workgroups as the chip holds at once (512 where two fit a
// CU, else 256), a row for each team of one at least: segments inside a gate row's
// group of `per` rows where the groups are large, else whole groups.  More workgroups
// mean more partials and a last round half empty, fewer leave waits uncovered: 8192 x
// 4096 bf16 with 256 / 512 / 1024 138 / 111 / 121 us, 4096 x 1024 fp32 with biases
// (one a CU) 30 / 35 / 45.
void plan_residual_norm_bwd(const ResNorm &p, ResNormGrad &g, bool bias) {
  const int64_t kBlocks = p.dim <= 4096 && !bias ? 512 : 256;
  const int64_t teams = kBwdThreads / bwd_team(p.dim);
  g.groups = p.rows / p.per;
  const int64_t want = std::max(teams, (p.rows + kBlocks - 1) / kBlocks);  // rows per workgroup
  if (p.per >= want) {
    g.segs = (p.per + want - 1) / want;
    g.seg_rows = (p.per + g.segs - 1) / g.segs;
    g.groups_per_block = 1;
    g.blocks = g.groups * g.segs;
  } else {
    g.segs = 0;
    g.seg_rows = p.per;
    g.groups_per_block = std::max(teams, want / p.per);
    g.blocks = (g.groups + g.groups_per_block - 1) / g.groups_per_block;
  }
}

bool residual_norm_bias(const ResNorm &p, const ResNormGrad &g) { return g.dbn || g.dbp || p.bp; }

int64_t residual_norm_part_floats(const ResNorm &p, const ResNormGrad &g) {
  return (int64_t)SUMS * g.blocks * p.dim + (p.dim > 8192 ? 4 * p.rows : 0);
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
