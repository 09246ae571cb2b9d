// Shared pieces of the attention kernels: the two 16-bit operand types, transposed reads from shared
// memory and reductions over the lanes that hold a query's scores.
#pragma once

#include "kv_cache.h"

constexpr float kLog2e = 1.4426950408889634f;
#define OMNI_LDS __attribute__((address_space(3)))

// An operand type's MFMA, conversion and the power of two that a softmax weight is held in: weights are
// 2^kBias exp2(score - maximum), so that float16, whose numbers end at 2^-24, keeps those far below the
// largest one. The sum of the weights carries the same factor and the quotient is free of it.
template <typename T>
struct Op;

template <>
struct Op<__bf16> {
  typedef bf16x8 x8;
  typedef bf16x4 x4;
  static constexpr float kBias = 0.f;
  static OMNI_DEVICE f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static OMNI_DEVICE f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Op<_Float16> {
  typedef f16x8 x8;
  typedef f16x4 x4;
  static constexpr float kBias = 7.f;
  static OMNI_DEVICE f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static OMNI_DEVICE f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// Two transposed reads side by side: a row of the result is a column of shared memory. Of each 16
// lanes, lane i gives the address of 4 values of row i / 4 (columns 4 (i % 4) ..) and receives column
// i's values of the four rows.
OMNI_DEVICE s16x8 read_transposed(const uint8_t OMNI_LDS* first, const uint8_t OMNI_LDS* second) {
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 OMNI_LDS*)first);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 OMNI_LDS*)second);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The other half-wave's v beside this one's.
OMNI_DEVICE float other_half(float v, float* mine) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  *mine = __builtin_bit_cast(float, (uint32_t)r[0]);
  return __builtin_bit_cast(float, (uint32_t)r[1]);
}
OMNI_DEVICE float half_max(float v) {
  float mine;
  const float other = other_half(v, &mine);
  return fmaxf(mine, other);
}
OMNI_DEVICE float half_sum(float v) {
  float mine;
  const float other = other_half(v, &mine);
  return mine + other;
}

// 64 pieces of 16 bytes, a lane's at base + off, into shared memory from `to` on, in the lanes' order; an
// offset past the buffer's bytes gives zeros. Written out because the compiler, which knows of its own
// such loads, waits for all of them before every transposed read, also where they fill another tile:
// nothing but the caller's s_waitcnt vmcnt waits for these. M0 holds the address, and nothing else in these
// kernels uses it. The wait states, which the compiler does not add here: one after M0, five where a vector
// instruction (a readfirstlane, a spilled scalar's return) has just written the buffer's registers.
OMNI_DEVICE u32x4 dma_rsrc(const uint8_t* base, uint32_t bytes) {
  const uint64_t at = (uint64_t)base;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)) & 0xffffu,
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
OMNI_DEVICE void dma_rows(u32x4 rsrc, uint32_t to, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)to)), "v"(off), "s"(rsrc)
               : "memory");
}
