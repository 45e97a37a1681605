// Shared pieces of the decoding kernels (block cache, cached attention, 4-bit
// linear): the 16 x 16 x 32 matrix instruction by element type, and the
// conversion of e4m3 bytes to its operands.
#pragma once

#include <type_traits>

#include "sah_common.hpp"

namespace sah {

// C[m][n] += sum_k A[m][k] B[k][n], m and n of 16, k of 32.  Lane l holds row
// (column) l % 16 of A (B) at k = 8 (l / 16) + 0..7, and of C column l % 16, rows
// 4 (l / 16) + 0..3.  Any order of k is right that A and B share.
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Eight e4m3 bytes, in order, times a power of two, as one operand: exact in both
// types for the scales used here (1; 1/2 on whole numbers up to 7 * 2^-9; and from 1 down
// to 2^-15 in fp16, whose smallest subnormal is the smallest code's then).
template <typename T>
__device__ __forceinline__ typename Vec8<T>::type e4m3_operand(uint32_t lo, uint32_t hi, float scale);
template <>
__device__ __forceinline__ bf16x8 e4m3_operand<bf16>(uint32_t lo, uint32_t hi, float scale) {
  const u32x4 v = {
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
  return __builtin_bit_cast(bf16x8, v);
}
template <>
__device__ __forceinline__ f16x8 e4m3_operand<f16>(uint32_t lo, uint32_t hi, float scale) {
  const u32x4 v = {
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true))};
  return __builtin_bit_cast(f16x8, v);
}

// fp32 in T, where rounded codes times their scale may have left T's range though the
// values that they stand for did not (within half a code's step of its largest, which
// is taken then).  NaN stays.
template <typename T>
__device__ __forceinline__ T in_range(float v) {
  constexpr float kMost = std::is_same<T, f16>::value ? 65504.0f : 3.38953139e38f;
  return from_f32<T>(v != v ? v : fminf(fmaxf(v, -kMost), kMost));
}

// Tokens of one block of the key/value cache.
constexpr int kBlockTokens = 64;

}  // namespace sah
