// The quantization of a block to e4m3 (fp8.hip, gemm_f8.hip).
#pragma once

#include "common.h"

namespace mj {

constexpr int kF8Block = 128;
constexpr float kF8Max = 448.0f;
constexpr float kF8Floor = 0x1p-100f;  // keeps the factor finite

struct F8Scale {
  float scale, inv;
};
__device__ __forceinline__ F8Scale f8_scale(float most) {
  const float a = fmaxf(most, kF8Floor);
  return {a * (1.0f / kF8Max), kF8Max * (1.0f / a)};
}

// v_cvt_pk_fp8_f32 rounds to the nearest even; its inputs are at most 448 (1 + 2^-20).
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d, float inv) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
}

__device__ __forceinline__ uint2 f8_pack8(const float (&v)[8], float inv) {
  return make_uint2(f8_pack4(v[0], v[1], v[2], v[3], inv), f8_pack4(v[4], v[5], v[6], v[7], inv));
}

// The largest of 16 lanes (magnitudes), in each of them.
__device__ __forceinline__ float f8_max16(float v) {
#define MJ_MAX(ctrl) \
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, false)))
  MJ_MAX(0xB1);   // quad_perm [1,0,3,2]
  MJ_MAX(0x4E);   // quad_perm [2,3,0,1]
  MJ_MAX(0x124);  // row_ror:4
  MJ_MAX(0x128);  // row_ror:8
#undef MJ_MAX
  return v;
}

}  // namespace mj
