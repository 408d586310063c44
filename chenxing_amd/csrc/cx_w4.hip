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
  int M, N, K;
  int wk;                     // waves that share rows of W
  void* out;
  int64_t ldo;
  int bf16;                   // out is
};

constexpr int W4_WAVES = 4096;

// 8 codes as bf16 1 + q / 16.
__device__ __forceinline__ bf16x8 w4_values(uint32_t w) {
  constexpr uint32_t ONE = 0x3F803F80u, BITS = 0x00780078u;
  return __builtin_bit_cast(bf16x8, u32x4{(w << 3 & BITS) | ONE, (w >> 1 & BITS) | ONE,
                                          (w >> 5 & BITS) | ONE, (w >> 9 & BITS) | ONE});
}
__device__ __forceinline__ float half_value(uint16_t h) {
  return (float)__builtin_bit_cast(_Float16, h);
}

// Few rows: a wave takes 16 NTW rows of W and, of their K, every WK-th tile of 128; the
// WK waves of the same rows add up through LDS.  All loads go straight to registers,
// codes and scales two tiles ahead, x (from the caches: a few rows) one.
template <int MT, int NTW, int STEPS, bool SHIFT>
__global__ __launch_bounds__(512) void w4_stream(W4Args A) {
  constexpr int GROUPS = 4 / STEPS;          // of a tile
  __shared__ f32x4 s_sum[7][MT * NTW * 64];
  const int w = wave_id(), l = lane_id(), g = l >> 4, c = l & 15;
  const int wk = w % A.wk, pair = (int)blockIdx.x * (8 / A.wk) + w / A.wk;
  const int m0 = blockIdx.y * 16 * MT;
  const int KT = (A.K + 127) / 128, groups = A.K / (32 * STEPS), steps = A.K / 32;
  const int NTILES = (A.N + 15) / 16;
  const uint16_t* xp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xp[i] = A.x + (int64_t)min(m0 + 16 * i + c, A.M - 1) * A.ldx + 8 * g;
  const u32x4* tp[NTW];
  const char* sp[NTW];
#pragma unroll
  for (int n = 0; n < NTW; ++n) {
    const int t = min(pair * NTW + n, NTILES - 1);
    tp[n] = (const u32x4*)A.tiles + (int64_t)t * KT * 64 + l;
    sp[n] = (const char*)A.scales + (int64_t)t * groups * 16 * (SHIFT ? 4 : 2);
  }
  struct Tile {
    u32x4 code[NTW];
    uint32_t scale[NTW];                     // of group g / STEPS, row c
  };
  struct Rows {
    u32x4 x[MT][4];
  };
  auto load = [&](Tile& t, int kt) {
    kt = min(kt, KT - 1);
    const int gr = min(kt * GROUPS + g / STEPS, groups - 1) * 16 + c;
#pragma unroll
    for (int n = 0; n < NTW; ++n) {
      t.code[n] = __builtin_nontemporal_load(tp[n] + kt * 64);
      t.scale[n] = SHIFT ? ((const uint32_t*)sp[n])[gr] : ((const uint16_t*)sp[n])[gr];
    }
  };
  auto load_x = [&](Rows& r, int kt) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) r.x[i][k] = *(const u32x4*)(xp[i] + 32 * min(kt * 4 + k, steps - 1));
  };
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
  f32x4 acc[MT][NTW];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NTW; ++n) acc[i][n] = f32x4{0, 0, 0, 0};
  auto multiply = [&](const Tile& t, const Rows& r, int kt) {
    // the scales of the tile's groups, in every lane group
    uint32_t sc[NTW][4];
#pragma unroll
    for (int n = 0; n < NTW; ++n) {
      if (GROUPS == 1) {
        sc[n][0] = t.scale[n];
        continue;
      }
      const auto h = __builtin_amdgcn_permlane32_swap(t.scale[n], t.scale[n], false, false);
      if (GROUPS == 2) {
        sc[n][0] = h[0];
        sc[n][1] = h[1];
        continue;
      }
      const auto a = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false);
      const auto b = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);
      sc[n][0] = a[0];
      sc[n][1] = a[1];
      sc[n][2] = b[0];
      sc[n][3] = b[1];
    }
#pragma unroll
    for (int q = 0; q < GROUPS; ++q) {
      if (kt * GROUPS + q >= groups) break;  // (uniform: the last tile of a K that is no multiple of 128)
      f32x4 p[MT][NTW], h[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        h[i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < NTW; ++n) p[i][n] = f32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int k = q * STEPS; k < (q + 1) * STEPS; ++k) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
          h[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, r.x[i][k]), ones, h[i], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NTW; ++n) {
          const bf16x8 v = w4_values(t.code[n][k]);
#pragma unroll
          for (int i = 0; i < MT; ++i)
            p[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, r.x[i][k]), v, p[i][n], 0, 0, 0);
        }
      }
#pragma unroll
      for (int n = 0; n < NTW; ++n) {
        const float f = 16.f * half_value((uint16_t)sc[n][q]);
        const float s = SHIFT ? half_value((uint16_t)(sc[n][q] >> 16)) - f : -1.5f * f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][n][j] = fmaf(f, p[i][n][j], fmaf(s, h[i][j], acc[i][n][j]));
      }
    }
  };
  Tile t0, t1;
  Rows r0, r1;
  load(t0, wk);
  load_x(r0, wk);
  load(t1, wk + A.wk);
  for (int kt = wk; kt < KT; kt += 2 * A.wk) {
    load_x(r1, kt + A.wk);
    multiply(t0, r0, kt);
    load(t0, kt + 2 * A.wk);
    if (kt + A.wk >= KT) break;
    load_x(r0, kt + 2 * A.wk);
    multiply(t1, r1, kt + A.wk);
    load(t1, kt + 3 * A.wk);
  }
  // the waves' sums, in the order of wk
  if (A.wk > 1) {
    f32x4* const mine = s_sum[0] + ((w / A.wk) * (A.wk - 1) + wk - 1) * (MT * NTW * 64) + l;
    if (wk > 0) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NTW; ++n) mine[(i * NTW + n) * 64] = acc[i][n];
    }
    __syncthreads();
    if (wk > 0) return;
    for (int k = 1; k < A.wk; ++k) {
      const f32x4* at = s_sum[0] + ((w / A.wk) * (A.wk - 1) + k - 1) * (MT * NTW * 64) + l;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NTW; ++n) acc[i][n] += at[(i * NTW + n) * 64];
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NTW; ++n) {
      const int col = (pair * NTW + n) * 16 + c;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + 16 * i + 4 * g + j;
        if (m >= A.M || col >= A.N) continue;
        if (A.bf16) ((__bf16*)A.out)[m * A.ldo + col] = (__bf16)acc[i][n][j];
        else ((float*)A.out)[m * A.ldo + col] = acc[i][n][j];
      }
    }
}

template <int MT, int NTW>
static void launch_w4(W4Args A, int group, bool shifts, hipStream_t s) {
  const int pairs = (A.N + 16 * NTW - 1) / (16 * NTW), KT = (A.K + 127) / 128;
  // waves enough for the chip's 256 CUs, of two tiles at least
  int wk = 1;
  while (wk < 8 && pairs * wk < W4_WAVES && KT >= 4 * wk) wk *= 2;
  A.wk = wk;
  using Kernel = void (*)(W4Args);
  static const Kernel kernels[3][2] = {{w4_stream<MT, NTW, 1, false>, w4_stream<MT, NTW, 1, true>},
                                       {w4_stream<MT, NTW, 2, false>, w4_stream<MT, NTW, 2, true>},
                                       {w4_stream<MT, NTW, 4, false>, w4_stream<MT, NTW, 4, true>}};
  timed_launch(CX_KERNEL_W4, kernels[group == 32 ? 0 : group == 64 ? 1 : 2][shifts],
               dim3((pairs * wk + 7) / 8, (A.M + 16 * MT - 1) / (16 * MT)), dim3(512), 0, s, A);
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
  const cx::W4Args A = {x, ldx, tiles, scales, M, N, K, 1, out, ldo, out_bf16 != 0};
  const hipStream_t st = (hipStream_t)stream;
  if (M <= 16) cx::launch_w4<1, 2>(A, group, shifts != 0, st);
  else if (M <= 32) cx::launch_w4<2, 2>(A, group, shifts != 0, st);
  else cx::launch_w4<4, 2>(A, group, shifts != 0, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "w4 launch: %s", hipGetErrorString(e));
  return CX_OK;
}
