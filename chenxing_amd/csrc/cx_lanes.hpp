// cx_lanes.hpp -- what the attention kernels do with lane groups and with elements that
// are NaN or infinite (cx_attend.hip, cx_tree.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cx_kv.hpp"

namespace cx {

// A value that every lane holds, in scalar registers.
__device__ __forceinline__ uint64_t scalar64(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}

// Lane groups of two registers change places: of groups 0 1 2 3, [a0 a1 a2 a3] and
// [b0 b1 b2 b3] become [a0 a1 b0 b1] and [a2 a3 b2 b3], or [a0 b0 a2 b2] and [a1 b1 a3 b3].
__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ void swap_rows(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
// The largest of the four lane groups' values, or their sum, in every group.
__device__ __forceinline__ float groups_max(float x) {
  uint32_t a = __float_as_uint(x), b = a;
  swap_halves(a, b);
  x = fmaxf(__uint_as_float(a), __uint_as_float(b));
  a = b = __float_as_uint(x);
  swap_rows(a, b);
  return fmaxf(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float groups_sum(float x) {
  uint32_t a = __float_as_uint(x), b = a;
  swap_halves(a, b);
  x = __uint_as_float(a) + __uint_as_float(b);
  a = b = __float_as_uint(x);
  swap_rows(a, b);
  return __uint_as_float(a) + __uint_as_float(b);
}
// The sign bits of the result say which bf16 or e4m3 elements of x are NaN or
// infinite (exponent all ones; code 0x7F or 0xFF).
template <bool F8>
__device__ __forceinline__ uint32_t nonfinite_sign(uint32_t x) {
  return F8 ? (x & 0x7F7F7F7Fu) + 0x01010101u : (x & 0x7F807F80u) + 0x00800080u;
}
// A mask of the other elements.
template <bool F8>
__device__ __forceinline__ uint32_t finite_mask(uint32_t x) {
  const uint32_t m = nonfinite_sign<F8>(x) & (F8 ? 0x80808080u : 0x80008000u);
  return ~(m | (m - (m >> (F8 ? 7 : 15))));
}

// Eight e4m3 codes as bf16.
__device__ __forceinline__ bf16x8 e4m3x8(uint32_t a, uint32_t b) {
  const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
  const bf16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
  const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
  const bf16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
  return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

}  // namespace cx
