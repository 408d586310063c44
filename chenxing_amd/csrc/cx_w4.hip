// cx_w4.hip -- products of few rows with 4-bit weights and group scales, for gfx950.
//
// y[m, n] = sum_k x[m, k] W[n, k], W[n, k] = s q + t of row n and k's group.  With
// v = 1 + q / 16, whose bf16 form is the code's bits in the mantissa of 1,
//
//   y[m, n] = sum over groups of 16 s (sum_k x v) + (t - 16 s) (sum_k x):
//
// the codes enter the products as they are, the second sum comes from the same matrix
// instruction with ones for weights, and a group's two sums are scaled in fp32.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cx_device.hpp"
#include "cx_internal.hpp"
#include "cx_sampler.h"
#include "cx_timing.hpp"

namespace cx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct W4Args {
  const uint16_t* x;          // [M, ldx] bf16 bits
  int64_t ldx;
  const uint32_t* tiles;
  const uint16_t* scales;
  int M, N, K, steps;         // steps: of 32 k in a group
  void* out;
  int64_t ldo;
};

// 8 codes as bf16 1 + q / 16.
__device__ __forceinline__ bf16x8 w4_values(uint32_t w) {
  constexpr uint32_t ONE = 0x3F803F80u, BITS = 0x00780078u;
  return __builtin_bit_cast(bf16x8, u32x4{(w << 3 & BITS) | ONE, (w >> 1 & BITS) | ONE,
                                          (w >> 5 & BITS) | ONE, (w >> 9 & BITS) | ONE});
}
__device__ __forceinline__ float half_value(uint16_t h) {
  return (float)__builtin_bit_cast(_Float16, h);
}

// Wave: 16 rows of W and 16 MT of x.
template <int MT, bool SHIFT, bool BF16>
__global__ __launch_bounds__(256) void w4_rows(W4Args A) {
  const int l = lane_id(), g = l >> 4, c = l & 15;
  const int nt = blockIdx.x * 4 + wave_id(), m0 = blockIdx.y * 16 * MT;
  if (nt * 16 >= A.N) return;
  const int KT = (A.K + 127) / 128, groups = A.K / (32 * A.steps);
  const uint32_t* tile = A.tiles + ((int64_t)nt * KT * 64 + l) * 4;
  const uint16_t* sc = A.scales + ((int64_t)nt * groups * 16 + c) * (SHIFT ? 2 : 1);
  const uint16_t* xp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xp[i] = A.x + (int64_t)min(m0 + 16 * i + c, A.M - 1) * A.ldx + 8 * g;
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0, 0, 0, 0};
  for (int gr = 0; gr < groups; ++gr) {
    f32x4 p[MT], h[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) p[i] = h[i] = f32x4{0, 0, 0, 0};
    for (int k = gr * A.steps; k < (gr + 1) * A.steps; ++k) {
      const bf16x8 w = w4_values(tile[(k >> 2) * 256 + (k & 3)]);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const bf16x8 x = __builtin_bit_cast(bf16x8, *(const u32x4*)(xp[i] + 32 * k));
        p[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, w, p[i], 0, 0, 0);
        h[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, ones, h[i], 0, 0, 0);
      }
    }
    const float s = half_value(sc[gr * 16 * (SHIFT ? 2 : 1)]);
    const float f = 16.f * s, t = SHIFT ? half_value(sc[gr * 32 + 1]) - f : -24.f * s;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(f, p[i][j], fmaf(t, h[i][j], acc[i][j]));
  }
  const int n = nt * 16 + c;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + 16 * i + 4 * g + j;
      if (m >= A.M || n >= A.N) continue;
      if (BF16) ((__bf16*)A.out)[m * A.ldo + n] = (__bf16)acc[i][j];
      else ((float*)A.out)[m * A.ldo + n] = acc[i][j];
    }
}

}  // namespace cx

extern "C" int cx_w4_linear_bf16(const uint16_t* x, int64_t ldx, const uint32_t* tiles,
                                 const uint16_t* scales, int32_t shifts, int32_t group, int32_t M,
                                 int32_t N, int32_t K, void* out, int64_t ldo, int32_t out_bf16,
                                 void* stream) {
  if (M < 0 || N < 1 || K < 1 || ldx < K || ldo < N) return cx::api_fail(CX_EINVAL, "bad shape");
  if (group != 32 && group != 64 && group != 128)
    return cx::api_fail(CX_EINVAL, "group (%d) must be 32, 64 or 128", group);
  if (K % group) return cx::api_fail(CX_EINVAL, "K (%d) must be a multiple of the group (%d)", K, group);
  if (M == 0) return CX_OK;
  if (!x || !tiles || !scales || !out) return cx::api_fail(CX_EINVAL, "null pointer argument");
  if ((((uintptr_t)x | (uintptr_t)tiles | (uintptr_t)scales) & 15) || (ldx & 7))
    return cx::api_fail(CX_EINVAL, "rows of x, tiles and scales must be 16-byte aligned");
  if ((uintptr_t)out & (out_bf16 ? 1 : 3)) return cx::api_fail(CX_EINVAL, "out must be aligned to its type");
  cx::W4Args A = {x, ldx, tiles, scales, M, N, K, group / 32, out, ldo};
  using Kernel = void (*)(cx::W4Args);
  static const Kernel kernels[2][2] = {{cx::w4_rows<1, false, false>, cx::w4_rows<1, false, true>},
                                       {cx::w4_rows<1, true, false>, cx::w4_rows<1, true, true>}};
  const Kernel k = kernels[shifts != 0][out_bf16 != 0];
  cx::timed_launch(CX_KERNEL_W4, k, dim3((N + 63) / 64, (M + 15) / 16), dim3(256), 0, (hipStream_t)stream, A);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "w4 launch: %s", hipGetErrorString(e));
  return CX_OK;
}
