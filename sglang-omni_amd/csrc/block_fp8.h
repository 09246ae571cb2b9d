// Shared pieces of the 8-bit block-scaled kernels: element loads of any alignment, the group
// quantizer, the MFMA of one K block and the output store.
#pragma once

#include "common.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kBlock = 128;                  // elements that share a scale
constexpr int64_t kMaxFeatures = 1 << 20;    // of a row
constexpr float kE4m3Max = 448.f;
// Groups whose largest magnitude is below this hold zeros with scale 1: 448 / amax stays finite
// and amax / 448 a normal number for every other.
constexpr float kTinyGroup = 7.8886090522101181e-31f;  // 2^-100

inline bool aligned_to(const void* ptr, int bytes) {
  return (reinterpret_cast<uintptr_t>(ptr) & (uintptr_t)(bytes - 1)) == 0;
}

// N values from src as float32, those from `valid` on zero. One wide load where all are valid: its
// address needs the element's alignment only (global memory takes unaligned vector accesses).
template <typename T, int N>
OMNI_DEVICE void load_values(const T* src, int64_t valid, float (&v)[N]) {
  typedef T vec __attribute__((ext_vector_type(N)));
  if (valid >= N) {
    vec t;
    __builtin_memcpy(&t, src, sizeof(t));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < valid ? (float)src[i] : 0.f;
  }
}

template <typename T, int N>
OMNI_DEVICE void store_values(T* dst, int64_t valid, const float (&v)[N]) {
  typedef T vec __attribute__((ext_vector_type(N)));
  if (valid >= N) {
    vec t;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = (T)v[i];
    __builtin_memcpy(dst, &t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < valid) dst[i] = (T)v[i];
  }
}

// A group's scale from its largest magnitude, and the factor its values take. NaN stays NaN through
// them; an infinity makes the scale infinite, so the group's products are NaN.
OMNI_DEVICE float group_scale(float amax, float* unit) {
  const bool tiny = amax < kTinyGroup;
  *unit = tiny ? 1.f : kE4m3Max / amax;
  return tiny ? 1.f : amax / kE4m3Max;
}

// 8 values of a group of 128 held by 16 consecutive lanes, 8 each: their E4M3 bytes and the group's
// scale.
OMNI_DEVICE float quantize_group(const float (&v)[8], u32x2* packed) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
  for (int off = 1; off < 16; off <<= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 16));
  float unit;
  const float scale = group_scale(amax, &unit);
  u32x2 p = {0u, 0u};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    p[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * unit, v[4 * h + 1] * unit, p[h], false);
    p[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * unit, v[4 * h + 3] * unit, p[h], true);
  }
  *packed = p;
  return scale;
}

OMNI_DEVICE i32x8 read_operand(const uint8_t* row, int slot0, int slot1) {
  const i32x4 a = *reinterpret_cast<const i32x4*>(row + slot0);
  const i32x4 b = *reinterpret_cast<const i32x4*>(row + slot1);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The 16 x 16 product of one K block, from zero.
//
// The 8-bit matrix instruction (here with no scale operands) cuts each product towards zero to a
// multiple of 2^(E - 13), 2^E the largest product of operand binades among the 8 consecutive features
// it is added with (zeros and subnormals count as 2^-6). A group's sum so loses up to 7 * 2^(E - 13),
// however small it is: beside +p and -p, what lies below p / 2^13 is gone. Without such cancelling the
// loss is far below a bf16 rounding (1.65e-3 of the results in the mean square): 1.3e-5 for Gaussian
// rows and weights, 1.6e-5 for operands over six binades, 5.2e-5 over all. So bf16 outputs take it
// (8192 x 4096 -> 8192 280 us; an operand's own E4M3 rounding is up to 2^-4); f16 and float32 outputs
// keep more bits than it does and take EXACT, the same bytes widened to bf16 (exactly) for four
// v_mfma_f32_16x16x32_bf16 at half its rate, whose sums are float32 throughout.
OMNI_DEVICE bf16x8 widen8(int lo, int hi) {
  const i32x4 w = {
      __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false)),
      __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true)),
      __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false)),
      __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true))};
  return __builtin_bit_cast(bf16x8, w);
}

template <bool EXACT>
struct Operand {
  i32x8 v;
  OMNI_DEVICE Operand() {}
  OMNI_DEVICE explicit Operand(i32x8 bytes) : v(bytes) {}
};
template <>
struct Operand<true> {
  bf16x8 v[4];
  OMNI_DEVICE Operand() {}
  OMNI_DEVICE explicit Operand(i32x8 bytes) {
#pragma unroll
    for (int s = 0; s < 4; ++s) v[s] = widen8(bytes[2 * s], bytes[2 * s + 1]);
  }
};

OMNI_DEVICE f32x4 block_product(const Operand<false>& a, const Operand<false>& b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0,
                                                          0, 0, 0, 0);
}
OMNI_DEVICE f32x4 block_product(const Operand<true>& a, const Operand<true>& b) {
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[s], b.v[s], c, 0, 0, 0);
  return c;
}
