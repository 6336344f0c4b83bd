// Tokens of a mixture of experts, sorted by expert and back.
//
// T tokens with k experts each are T k slots, slot t k + j.  The sort is a counting
// sort, stable in the slots: pos[slot] is its row among the sorted ones, offsets[e] the
// first row of expert e, and slots whose expert is outside [0, E) come last, from
// offsets[E] on (dropped).  Then, token by token:
//
//   dispatch          xs[pos[t, j]] = x[t]                     (0 for a dropped slot)
//   combine           y[t] = sum_j w[t, j] ys[pos[t, j]]       (dropped slots left out)
//   combine backward  dys[pos[t, j]] = w[t, j] dy[t], dw[t, j] = <dy[t], ys[pos[t, j]]>
//
// and dispatch's gradient is combine without weights.  All of it is bound by memory:
// going by tokens, each row of x and dy is read once and written k times, each row of ys
// read once.  Sums run in fp32 in the order of j (dot products: in a fixed order), so
// the same inputs give the same bits; the only atomics are the sort's counts in LDS, whole
// numbers whose order changes nothing.
#include <algorithm>
#include <atomic>

#include "common.h"
#include "expert_tile.h"  // within
#include "launch.h"
#include "philox.h"  // u32x4_a2

namespace mj {

namespace {

// ---------------------------------------------------------------- sort
// A workgroup of 16 waves sorts 1024 S consecutive slots, each wave 64 S of them, 64 at a
// time: the lanes of one key find each other by a ballot for each bit of the key, so a
// lane's place among its wave's earlier ones needs no atomics, and the order is that of
// the slots.  Counts stay in LDS for each wave and key.
//
// Up to 8192 slots each workgroup counts the keys of all other slots itself, earlier ones
// and later ones, by integer atomics on LDS (their order is of no matter): one launch.
// Beyond, the counts of every workgroup are written, summed over the workgroups by one
// more launch and read again.  8192 slots of 32 experts 7.3 us (11 in one workgroup), 3000 of
// 16 4.7 (5.8), 65536 of 64 in three launches 18.
enum : int { SORT_WHOLE = 0, SORT_COUNT, SORT_PLACE };

struct SortArgs {
  const void *ids = nullptr;
  int wide = 0;           // ids are int64
  int64_t slots = 0;
  int experts = 0, bits = 0;
  int *pos = nullptr, *offsets = nullptr, *work = nullptr;  // work [blocks + 1][experts + 1]
  int64_t blocks = 1;
};

constexpr int kSortWaves = 16;
constexpr int kSortWhole = 8;  // most workgroups of one launch

template <int S, int MODE>
__global__ __launch_bounds__(1024) void sort_kernel(SortArgs a) {
  extern __shared__ int lds[];
  const int E1 = a.experts + 1;
  int *base = lds, *before = base + E1, *after = before + E1, *wsum = after + E1;
  volatile uint16_t *hist = (volatile uint16_t *)(wsum + kSortWaves);  // [waves][E1]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = (int64_t)blockIdx.x * (1024 * S) + wave * (64 * S) + lane;
  int key[S], place[S];
  auto key_of = [&](int64_t slot) __attribute__((always_inline)) {
    int64_t id = -1;
    if (slot < a.slots) id = a.wide ? ((const int64_t *)a.ids)[slot] : ((const int *)a.ids)[slot];
    return id >= 0 && id < a.experts ? (int)id : a.experts;
  };
#pragma unroll
  for (int s = 0; s < S; ++s) key[s] = key_of(first + s * 64);
  int others[kSortWhole];
  const bool more = MODE == SORT_WHOLE && a.blocks > 1;
  if (more) {
#pragma unroll
    for (int b = 0; b < kSortWhole; ++b) others[b] = key_of(b * 1024 + tid);
  }
  for (int i = tid; i < kSortWaves * E1; i += 1024) hist[i] = 0;
  for (int i = tid; i < 2 * E1; i += 1024) before[i] = 0;
  __syncthreads();
  if (more) {
#pragma unroll
    for (int b = 0; b < kSortWhole; ++b)
      if (b != (int)blockIdx.x && b * 1024 + tid < a.slots)
        atomicAdd((b < (int)blockIdx.x ? before : after) + others[b], 1);
  }
  volatile uint16_t *mine = hist + wave * E1;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const bool in = first + s * 64 < a.slots;
    uint64_t same = __ballot(in);
    for (int b = 0; b < a.bits; ++b) {
      const bool bit = (key[s] >> b) & 1;
      const uint64_t set = __ballot(bit);
      same &= bit ? set : ~set;
    }
    const int rank = __popcll(same & (((uint64_t)1 << lane) - 1));
    const int before = mine[key[s]];  // read by every lane before its first lane adds to it
    place[s] = before + rank;
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) mine[key[s]] = (uint16_t)(before + __popcll(same));
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // counts -> places within the workgroup; totals of the keys
  for (int e = tid; e < E1; e += 1024) {
    int run = 0;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = hist[w * E1 + e];
      hist[w * E1 + e] = (uint16_t)run;
      run += c;
    }
    base[e] = run;
    if (MODE == SORT_WHOLE) base[e] += before[e] + after[e];
    if (MODE == SORT_COUNT) a.work[(int64_t)blockIdx.x * E1 + e] = run;
  }
  if constexpr (MODE == SORT_COUNT) return;
  __syncthreads();
  // offsets: an exclusive scan of the keys' totals (one thread each, experts <= 1024)
  const int *total = MODE == SORT_PLACE ? a.work + a.blocks * E1 : base;
  const int v = tid < a.experts ? total[tid] : 0;
  int sum = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(sum, d, 64);
    if (lane >= d) sum += o;
  }
  if (lane == 63) wsum[wave] = sum;
  __syncthreads();
  int lower = 0, all = 0;
  for (int w = 0; w < kSortWaves; ++w) {
    if (w < wave) lower += wsum[w];
    all += wsum[w];
  }
  const int64_t row = (int64_t)blockIdx.x * E1;
  if (tid < a.experts) {
    const int off = lower + sum - v;
    base[tid] = off + (MODE == SORT_PLACE ? a.work[row + tid] : before[tid]);
    if (blockIdx.x == 0) a.offsets[tid] = off;
  }
  if (tid == 0) {
    base[a.experts] = all + (MODE == SORT_PLACE ? a.work[row + a.experts] : before[a.experts]);
    if (blockIdx.x == 0) a.offsets[a.experts] = all;
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (first + s * 64 < a.slots) a.pos[first + s * 64] = base[key[s]] + mine[key[s]] + place[s];
}

// For each key the counts of the workgroups become sums over the earlier ones; their total
// goes behind.  One workgroup a key.
__global__ __launch_bounds__(256) void sort_sums_kernel(int *work, int64_t blocks, int E1) {
  __shared__ int wsum[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x;
  int carry = 0;
  for (int64_t b0 = 0; b0 < blocks; b0 += 256) {
    const int64_t b = b0 + threadIdx.x;
    const int v = b < blocks ? work[b * E1 + e] : 0;
    int sum = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(sum, d, 64);
      if (lane >= d) sum += o;
    }
    if (lane == 63) wsum[wave] = sum;
    __syncthreads();
    int lower = carry;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) lower += wsum[w];
      carry += wsum[w];
    }
    if (b < blocks) work[b * E1 + e] = lower + sum - v;
    __syncthreads();
  }
  if (threadIdx.x == 0) work[blocks * E1 + e] = carry;
}

// ---------------------------------------------------------------- rows
// 16 bytes of a row a thread, at the elements' own alignment; `have` of its elements are
// inside the row.
template <bool BF>
struct Unit {
  static constexpr int N = BF ? 8 : 4;
  static constexpr int SIZE = BF ? 2 : 4;
  u32x4_a2 w;
  // NT: nontemporal
  template <bool NT = false>
  __device__ __forceinline__ void load(const void *row, int64_t e, int have) {
    const char *p = (const char *)row + e * SIZE;
    if (have >= N) {
      if constexpr (NT) w = __builtin_nontemporal_load((const u32x4_a2 *)p);
      else w = *(const u32x4_a2 *)p;
    } else {
      w = u32x4_a2{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < have) {
          if constexpr (BF) w[i >> 1] |= (uint32_t)((const uint16_t *)p)[i] << (16 * (i & 1));
          else w[i] = ((const uint32_t *)p)[i];
        }
    }
  }
  template <bool NT = false>
  __device__ __forceinline__ void store(void *row, int64_t e, int have) const {
    char *p = (char *)row + e * SIZE;
    if (have >= N) {
      if constexpr (NT) __builtin_nontemporal_store(w, (u32x4_a2 *)p);
      else *(u32x4_a2 *)p = w;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < have) {
          if constexpr (BF) ((uint16_t *)p)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
          else ((uint32_t *)p)[i] = w[i];
        }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (BF) return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
    else return __uint_as_float(w[i]);
  }
  __device__ __forceinline__ void set(const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (BF) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      else w[i] = __float_as_uint(v[i]);
    }
  }
};

// The token and the unit of a row that a thread handles; false past the last token.
__device__ __forceinline__ bool unit_of(int64_t i, int64_t units, int64_t tokens, int64_t &t, int64_t &u) {
  if (i < ((int64_t)1 << 32)) {  // (a division in 32 bits)
    t = (uint32_t)i / (uint32_t)units;
  } else {
    t = i / units;
  }
  u = i - t * units;
  return t < tokens;
}

// The rows of slots that are not dropped.
__device__ __forceinline__ int kept_rows(const ExpertRows &a) {
  return within(*a.kept, (int)(a.tokens * a.topk));
}

// A thread copies 16 bytes of a token's row to its k sorted rows: one read, k writes, whole
// lines either way.  8192 tokens, 8 experts each, 4096 bf16: 111 us, 5.4 TB/s.
template <bool BF>
__global__ __launch_bounds__(256) void dispatch_kernel(ExpertRows a) {
  using U = Unit<BF>;
  int64_t t, u;
  if (!unit_of(grid_block<256>() * 256 + threadIdx.x, a.units, a.tokens, t, u)) return;
  const int64_t e = u * U::N;
  const int have = (int)std::min<int64_t>(a.dim - e, U::N), kept = kept_rows(a), k = (int)a.topk;
  const uint32_t rows = (uint32_t)(a.tokens * a.topk);
  U x, zero;
  x.load((const char *)a.x + t * a.dim * U::SIZE, e, have);
  zero.w = u32x4_a2{0, 0, 0, 0};
  const int *pos = a.pos + t * k;
#pragma unroll 4
  for (int j = 0; j < k; ++j) {
    const int p = pos[j];
    if ((uint32_t)p >= rows) continue;
    char *row = (char *)a.xs + (int64_t)p * a.dim * U::SIZE;
    if (p < kept) x.store(row, e, have);
    else zero.store(row, e, have);
    if (a.ws && u == 0) a.ws[p] = p < kept ? a.w[t * k + j] : 0.0f;
  }
}

// BI, BO: the rows' and the sum's type; a thread's 16 bytes of the sum are one or two units
// of a row, and up to eight loads are in flight (the rows lie anywhere, so latency counts).
// 8192 tokens, 8 experts each, 4096 bf16: 105 us, 5.8 TB/s.
template <bool BI, bool BO, bool NT>
__global__ __launch_bounds__(256) void combine_kernel(ExpertRows a) {
  using UI = Unit<BI>;
  using UO = Unit<BO>;
  constexpr int N = UO::N, P = N / UI::N;
  int64_t t, u;
  if (!unit_of(grid_block<256>() * 256 + threadIdx.x, a.units, a.tokens, t, u)) return;
  const int64_t e = u * N;
  const int have = (int)std::min<int64_t>(a.dim - e, N), k = (int)a.topk;
  const uint32_t kept = kept_rows(a);
  const int *pos = a.pos + t * k;
  float acc[N] = {};
  auto load = [&](UI (&v)[P], int p) __attribute__((always_inline)) {
    const char *row = (const char *)a.xs + (int64_t)p * a.dim * UI::SIZE;
#pragma unroll
    for (int q = 0; q < P; ++q) v[q].template load<NT>(row, e + q * UI::N, have - q * UI::N);
  };
  auto add = [&](const UI (&v)[P], int j) __attribute__((always_inline)) {
    const float w = a.w ? a.w[t * k + j] : 1.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = __builtin_fmaf(w, v[i / UI::N].get(i % UI::N), acc[i]);
  };
  constexpr int FLY = 8 / P;  // rows' loads in flight
  for (int j0 = 0; j0 < k; j0 += FLY) {
    UI v[FLY][P];
    uint32_t p[FLY];
#pragma unroll
    for (int q = 0; q < FLY; ++q) p[q] = j0 + q < k ? pos[j0 + q] : 0x7FFFFFFF;
#pragma unroll
    for (int q = 0; q < FLY; ++q)
      if (p[q] < kept) load(v[q], p[q]);
#pragma unroll
    for (int q = 0; q < FLY; ++q)
      if (p[q] < kept) add(v[q], j0 + q);
  }
  UO y;
  y.set(acc);
  y.template store<NT>((char *)a.x + t * a.dim * UO::SIZE, e, have);
}

// One workgroup a token (one wave where a row is short), four slots at a time: for each the row
// of dys and the product of dy with the row of ys, its lanes' and waves' sums added in order.
// dy comes from the caches after the first four.  8192 tokens, 8 experts each, 4096 bf16: 236
// us, 4.8 TB/s (a read and a write an element of the sorted rows, and dy once).
constexpr int kDotSlots = 4;

template <bool BF, int NW, bool NT>
__global__ __launch_bounds__(NW * 64) void combine_bwd_kernel(ExpertRows a) {
  using U = Unit<BF>;
  __shared__ float red[2][kDotSlots][NW];
  const int64_t t = grid_block<NW * 64>();
  if (t >= a.tokens) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kept = kept_rows(a), k = (int)a.topk;
  const uint32_t rows = (uint32_t)(a.tokens * a.topk);
  const char *dy = (const char *)a.x + t * a.dim * U::SIZE;
  for (int j0 = 0, half = 0; j0 < k; j0 += kDotSlots, half ^= 1) {
    const int n = std::min(k - j0, kDotSlots);
    int64_t row[kDotSlots];
    bool in[kDotSlots], is[kDotSlots];
    float w[kDotSlots], sum[kDotSlots];
#pragma unroll
    for (int q = 0; q < kDotSlots; ++q) {
      const int64_t slot = t * k + j0 + (q < n ? q : 0);
      const int p = a.pos[slot];
      row[q] = (int64_t)p * a.dim * U::SIZE;
      is[q] = q < n && (uint32_t)p < rows;
      in[q] = is[q] && p < kept;
      w[q] = a.w[slot];
      sum[q] = 0.0f;
    }
    for (int64_t e = (int64_t)threadIdx.x * U::N; e < a.dim; e += NW * 64 * U::N) {
      const int have = (int)std::min<int64_t>(a.dim - e, U::N);
      U d, y[kDotSlots];
      d.load(dy, e, have);
#pragma unroll
      for (int q = 0; q < kDotSlots; ++q)
        if (in[q]) y[q].template load<NT>((const char *)a.ys + row[q], e, have);
#pragma unroll
      for (int q = 0; q < kDotSlots; ++q) {
        if (!is[q]) continue;
        U o;
        float v[U::N];
        if (in[q]) {
#pragma unroll
          for (int i = 0; i < U::N; ++i) sum[q] = __builtin_fmaf(d.get(i), y[q].get(i), sum[q]);
        }
#pragma unroll
        for (int i = 0; i < U::N; ++i) v[i] = in[q] ? w[q] * d.get(i) : 0.0f;
        o.set(v);
        o.template store<NT>((char *)a.xs + row[q], e, have);
      }
    }
#pragma unroll
    for (int q = 0; q < kDotSlots; ++q) {
      sum[q] = wave_sum_dpp(sum[q]);
      if (lane == 0) red[half][q][wave] = sum[q];
    }
    __syncthreads();  // (two buffers: the next four wait only for these to be read)
    if ((int)threadIdx.x < n) {
      float s = red[half][threadIdx.x][0];
#pragma unroll
      for (int v = 1; v < NW; ++v) s += red[half][threadIdx.x][v];
      a.ws[t * k + j0 + threadIdx.x] = s;
    }
  }
}

// Slots of a workgroup: as few as can be in one launch, else 4096.
constexpr int64_t kSortOnce = 1024 * kSortWhole, kSortSteps = 4;

int64_t sort_blocks(int64_t slots) {
  const int64_t per = slots <= kSortOnce ? 1024 : 1024 * kSortSteps;
  return (slots + per - 1) / per;
}

// 16-byte units of a row; one for an empty row (its token's weights are sorted all the same).
template <bool BF>
int64_t units_of(int64_t dim) {
  return std::max<int64_t>((dim + Unit<BF>::N - 1) / Unit<BF>::N, 1);
}

// Rows that the XCDs' caches do not hold are read (and written) past them.  Combine, 8 x 8192
// rows of 4096 bf16: 122 -> 110 us, right behind the kernel that wrote them 120 -> 85; 3000 x
// 1001 fp32 5.0 -> 6.0.  Its backward 254 -> 235.  Dispatch, which only writes them, loses by it
// (106 -> 114).
bool past_caches(bool bf16, const ExpertRows &a) {
  return a.tokens * a.topk * a.dim * (bf16 ? 2 : 4) > (32 << 20);
}

}  // namespace

int64_t sort_experts_work_ints(int64_t slots, int64_t experts) {
  return slots <= kSortOnce ? 0 : (sort_blocks(slots) + 1) * (experts + 1);
}

hipError_t launch_sort_experts(const void *ids, bool wide, int64_t slots, int64_t experts, int *pos,
                               int *offsets, int *work, hipStream_t stream) {
  SortArgs a;
  a.ids = ids, a.wide = wide, a.slots = slots, a.experts = (int)experts;
  while ((1 << a.bits) < experts + 1) ++a.bits;
  a.pos = pos, a.offsets = offsets, a.work = work;
  a.blocks = std::max<int64_t>(sort_blocks(slots), 1);  // (no slots: the offsets are zeros)
  const size_t lds = (size_t)(3 * (experts + 1) + kSortWaves) * 4 + (size_t)kSortWaves * (experts + 1) * 2;
  const dim3 grid((unsigned)a.blocks), block(1024);
  if (slots <= kSortOnce) {
    hipLaunchKernelGGL((sort_kernel<1, SORT_WHOLE>), grid, block, lds, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((sort_kernel<kSortSteps, SORT_COUNT>), grid, block, lds, stream, a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  hipLaunchKernelGGL(sort_sums_kernel, dim3((unsigned)(experts + 1)), dim3(256), 0, stream, work, a.blocks,
                     (int)experts + 1);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  hipLaunchKernelGGL((sort_kernel<kSortSteps, SORT_PLACE>), grid, block, lds, stream, a);
  return hipGetLastError();
}

hipError_t launch_dispatch(bool bf16, ExpertRows a, hipStream_t stream) {
  a.units = bf16 ? units_of<true>(a.dim) : units_of<false>(a.dim);
  const int64_t n = a.tokens * a.units;
  if (n == 0 || a.topk == 0) return hipSuccess;
  const dim3 grid = grid_rows<256>((n + 255) / 256);
  if (bf16) hipLaunchKernelGGL(dispatch_kernel<true>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(dispatch_kernel<false>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_combine(bool bf16, bool y_bf16, ExpertRows a, hipStream_t stream) {
  a.units = y_bf16 ? units_of<true>(a.dim) : units_of<false>(a.dim);
  const int64_t n = a.tokens * a.units;
  if (n == 0) return hipSuccess;
  const dim3 grid = grid_rows<256>((n + 255) / 256);
  const bool nt = past_caches(bf16, a);
#define MJ_COMBINE(BI, BO)                                                                       \
  do {                                                                                           \
    if (nt) hipLaunchKernelGGL((combine_kernel<BI, BO, true>), grid, dim3(256), 0, stream, a);   \
    else hipLaunchKernelGGL((combine_kernel<BI, BO, false>), grid, dim3(256), 0, stream, a);     \
  } while (0)
  if (bf16) MJ_COMBINE(true, true);
  else if (y_bf16) MJ_COMBINE(false, true);
  else MJ_COMBINE(false, false);
#undef MJ_COMBINE
  return hipGetLastError();
}

hipError_t launch_combine_bwd(bool bf16, const ExpertRows &a, hipStream_t stream) {
  if (a.tokens == 0 || a.topk == 0) return hipSuccess;
  const bool one = (bf16 ? units_of<true>(a.dim) : units_of<false>(a.dim)) <= 64;
  const dim3 grid = one ? grid_rows<64>(a.tokens) : grid_rows<256>(a.tokens);
  const bool nt = past_caches(bf16, a);
#define MJ_BWD(BF, NW, NT) \
  hipLaunchKernelGGL((combine_bwd_kernel<BF, NW, NT>), grid, dim3(NW * 64), 0, stream, a)
  if (bf16) {
    if (one) MJ_BWD(true, 1, false);
    else if (nt) MJ_BWD(true, 4, true);
    else MJ_BWD(true, 4, false);
  } else {
    if (one) MJ_BWD(false, 1, false);
    else if (nt) MJ_BWD(false, 4, true);
    else MJ_BWD(false, 4, false);
  }
#undef MJ_BWD
  return hipGetLastError();
}

}  // namespace mj
