// Quantization to 8-bit floating point (e4m3: 448 is the largest value) with a scale for
// each block: 128 features of a row (activations) or 128 x 128 elements (weights).
//
//   a = max(2^-100, the block's largest magnitude), scale = a (1 / 448),
//   q = e4m3(v (448 (1 / a))), ties to even, each operation rounded to fp32
//
// The floor keeps the factor finite (a block of zeros gives zeros).  A NaN gives a NaN, and a
// block that holds an infinity gives NaNs there and an infinite scale.
//
// Rows go token by token as in experts.hip: with a sort, a token's row is quantized once
// and written to each of its sorted rows (zeros for a dropped slot).  The rows' scales
// lie block by block, scale[k / 128][row], so that a tile of the product reads the scales of
// its rows for one K step as one piece.  Bound by memory: 2 (or 4) bytes read, one
// written an element.
#include <algorithm>

#include "common.h"
#include "expert_tile.h"  // within
#include "fp8.h"
#include "launch.h"

namespace mj {

namespace {

// Eight values of a row; bf16 or fp32, rows 16-byte aligned.
template <bool BF>
__device__ __forceinline__ void load8(const void *p, int64_t e, float (&v)[8]) {
  if constexpr (BF) {
    const uint4 w = *(const uint4 *)((const uint16_t *)p + e);
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(q[i] << 16);
      v[2 * i + 1] = __uint_as_float(q[i] & 0xFFFF0000u);
    }
  } else {
    const float4 a = *(const float4 *)((const float *)p + e), b = *(const float4 *)((const float *)p + e + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}

__device__ __forceinline__ float max8(const float (&v)[8]) {
  float a = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) a = fmaxf(a, fabsf(v[i]));
  return a;
}

// 16 lanes a block of a row, 8 elements a lane (K % 16 == 0: a lane has all or none).  2048 x
// 4096 bf16 6.3 us (4 TB/s); 4096 x 4096 to two sorted rows each 18 us.
template <bool BF>
__global__ __launch_bounds__(256) void quantize_rows_kernel(F8Rows a) {
  const int64_t i = grid_block<256>() * 16 + (threadIdx.x >> 4);
  const int64_t kbs = (a.dim + 127) / 128;
  const int64_t t = i < ((int64_t)1 << 32) ? (int64_t)((uint32_t)i / (uint32_t)kbs) : i / kbs;
  if (t >= a.tokens) return;
  const int64_t kb = i - t * kbs, e = kb * 128 + (threadIdx.x & 15) * 8;
  const bool in = e < a.dim;
  float v[8] = {};
  if (in) load8<BF>(a.x, t * a.dim + e, v);
  const F8Scale s = f8_scale(f8_max16(max8(v)));
  const uint2 q = f8_pack8(v, s.inv);
  auto put = [&](int64_t p, uint2 w, float scale) __attribute__((always_inline)) {
    if (in) *(uint2 *)(a.q + p * a.dim + e) = w;
    if ((threadIdx.x & 15) == 0) a.scales[kb * a.rows + p] = scale;
  };
  if (!a.pos) {
    put(t, q, s.scale);
    return;
  }
  const int kept = within(*a.kept, (int)a.rows), k = (int)a.topk;
#pragma unroll 4
  for (int j = 0; j < k; ++j) {
    const int p = a.pos[t * k + j];
    if ((uint32_t)p >= (uint32_t)a.rows) continue;
    const bool on = p < kept;
    put(p, on ? q : make_uint2(0, 0), on ? s.scale : 0.0f);
  }
}

// One workgroup a 128 x 128 block of one of `mats` matrices [N, K]: 16 lanes a row, 8 rows
// of each thread in registers, so the matrix is read once.  Not in a model's step: weights
// are quantized when they are loaded.  11008 x 4096 bf16 25 us (5.4 TB/s), 8 x 5504 x 4096 102
// (5.3), fp32 157 (5.8).
template <bool BF>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(F8Blocks a) {
  __shared__ float red[4];
  const int64_t nbs = (a.n + 127) / 128, kbs = (a.k + 127) / 128;
  const int64_t b = grid_block<256>();
  if (b >= a.mats * nbs * kbs) return;
  const int64_t mat = b / (nbs * kbs), at = b - mat * (nbs * kbs), nb = at / kbs, kb = at - nb * kbs;
  const int64_t e = kb * 128 + (threadIdx.x & 15) * 8, base = mat * a.n * a.k;
  const int64_t row0 = nb * 128 + (threadIdx.x >> 4);
  float v[8][8], most = 0.0f;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t n = row0 + r * 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[r][i] = 0.0f;
    if (n < a.n && e < a.k) load8<BF>(a.w, base + n * a.k + e, v[r]);
    most = fmaxf(most, max8(v[r]));
  }
  most = wave_max(most);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
  __syncthreads();
  most = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const F8Scale s = f8_scale(most);
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t n = row0 + r * 16;
    if (n < a.n && e < a.k) *(uint2 *)(a.q + base + n * a.k + e) = f8_pack8(v[r], s.inv);
  }
  if (threadIdx.x == 0) a.scales[b] = s.scale;
}

}  // namespace

hipError_t launch_quantize_rows_f8(bool bf16, const F8Rows &a, hipStream_t stream) {
  const int64_t n = a.tokens * ((a.dim + 127) / 128);
  if (n == 0) return hipSuccess;
  const dim3 grid = grid_rows<256>((n + 15) / 16);
  if (bf16) hipLaunchKernelGGL(quantize_rows_kernel<true>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(quantize_rows_kernel<false>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_quantize_blocks_f8(bool bf16, const F8Blocks &a, hipStream_t stream) {
  const int64_t n = a.mats * ((a.n + 127) / 128) * ((a.k + 127) / 128);
  if (n == 0) return hipSuccess;
  const dim3 grid = grid_rows<256>(n);
  if (bf16) hipLaunchKernelGGL(quantize_blocks_kernel<true>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(quantize_blocks_kernel<false>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mj
