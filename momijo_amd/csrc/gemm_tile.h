// Building blocks of the bf16 MFMA tile kernels (gemm_nt.hip, gated_mlp.hip).
#pragma once

#include "common.h"

namespace mj {

constexpr int kBK = 64;  // K per pipeline stage

typedef __attribute__((address_space(3))) void lds_void;

// 16 bytes a lane straight from memory into LDS (lane i at lds_dst + 16 i bytes).
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint16_t *lds_dst, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)lds_dst, 16, off, 0, 0, 0);
}

// The same with a scalar offset: the K advance costs no vector instruction.
__device__ __forceinline__ void dma16s(__amdgpu_buffer_rsrc_t r, uint16_t *lds_dst,
                                       uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)lds_dst, 16, voff, soff, 0, 0);
}

// s_waitcnt lgkmcnt(0) as the builtin (vmcnt and expcnt left open): unlike the
// same text in inline asm, the compiler's wait-count pass sees it, so it does
// not add a wait of its own for fragments this one already covered (such a
// wait, placed after the next step's first read, stalled every stage for a
// full LDS round trip).
constexpr int kLgkm0 = 0xC07F;

__device__ __forceinline__ void mfma_16x16x32_tied(f32x4 &acc, const bf16x8 &a, const bf16x8 &b) {
  asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

}  // namespace mj
