// The keep mask of the dropout operators, drawn where it is used and never
// stored, and 8-element row accesses of the elementwise block kernels.
//
// Random words: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011): ten rounds of two 32 x 32 -> 64 bit
// products over a 128-bit counter, keyed by the seed.  Any block of the stream
// is computed from its number alone, so the backward pass draws the forward's
// mask again and a thread needs no state.  A block's four words serve 8
// elements, 16 bits each: one draw per element would make the generator, not
// memory, the bound of a bf16 dropout (a block is 20 multiplies of quarter rate
// and about 40 other operations).
#pragma once

#include "common.h"
#include "launch.h"

namespace mj {

// The key and counter of a launch (the device state replaces seed and moves counter).
__device__ __forceinline__ void dropout_key(const Dropout &d, uint64_t &seed, uint64_t &counter) {
  seed = d.state ? d.state[0] : d.seed;
  counter = d.state ? d.state[1] + d.counter : d.counter;
}

__device__ __forceinline__ uint4 philox4x32(uint64_t block, uint64_t counter, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32);
  uint32_t c2 = (uint32_t)counter, c3 = (uint32_t)(counter >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The 16-bit draws of the 8 elements from flat index e on, two a word.
// ALIGNED: e is a multiple of 8, one block; otherwise the window over two blocks.
template <bool ALIGNED>
__device__ __forceinline__ void draws8(uint64_t e, uint64_t counter, uint64_t seed,
                                       uint32_t (&w)[4]) {
  const uint4 a = philox4x32(e >> 3, counter, seed);
  if constexpr (ALIGNED) {
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
  } else {
    const uint4 b = philox4x32((e >> 3) + 1, counter, seed);
    uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const uint32_t s = (uint32_t)e & 7;
    if (s & 4) {
#pragma unroll
      for (int i = 0; i < 6; ++i) v[i] = v[i + 2];
    }
    if (s & 2) {
#pragma unroll
      for (int i = 0; i < 5; ++i) v[i] = v[i + 1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = s & 1 ? (v[i] >> 16) | (v[i + 1] << 16) : v[i];
  }
}

// Whether element i of the 8 is kept.  A dropped element's value is not looked at (0,
// whatever it holds): callers select by this, they do not multiply by 0.
__device__ __forceinline__ bool keep_of(const uint32_t (&w)[4], int i, uint32_t thr) {
  return ((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu) >= thr;
}

// ---- 8 consecutive elements of a row as floats.  ALIGNED: a 16-byte aligned
// address.  Otherwise the same load at the elements' own alignment, which the
// memory unit takes at any address.  n < 8: only the first n exist.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void unpack8(const uint32_t (&w)[4], float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

template <bool ALIGNED>
__device__ __forceinline__ void load8(const uint16_t *p, int n, float (&v)[8]) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (ALIGNED || n >= 8) {
    if constexpr (ALIGNED) {
      const uint4 q = *(const uint4 *)p;
      w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    } else {
      const u32x4_a2 q = *(const u32x4_a2 *)p;
      w[0] = q[0], w[1] = q[1], w[2] = q[2], w[3] = q[3];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
  }
  unpack8(w, v);
}

template <bool ALIGNED>
__device__ __forceinline__ void load8(const float *p, int n, float (&v)[8]) {
  if (ALIGNED || n >= 8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (ALIGNED) {
        const float4 q = *(const float4 *)(p + 4 * h);
        v[4 * h] = q.x, v[4 * h + 1] = q.y, v[4 * h + 2] = q.z, v[4 * h + 3] = q.w;
      } else {
        const f32x4_a4 q = *(const f32x4_a4 *)(p + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * h + i] = q[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
  }
}

template <bool ALIGNED>
__device__ __forceinline__ void store8(uint16_t *p, int n, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  if (ALIGNED || n >= 8) {
    if constexpr (ALIGNED) *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
    else *(u32x4_a2 *)p = u32x4_a2{w[0], w[1], w[2], w[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
  }
}

template <bool ALIGNED>
__device__ __forceinline__ void store8(float *p, int n, const float (&v)[8]) {
  if (ALIGNED || n >= 8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (ALIGNED)
        *(float4 *)(p + 4 * h) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
      else
        *(f32x4_a4 *)(p + 4 * h) = f32x4_a4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = v[i];
  }
}

}  // namespace mj
