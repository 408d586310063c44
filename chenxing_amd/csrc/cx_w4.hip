// cx_w4.hip -- products of few rows with 4-bit weights and group scales, for gfx950.
//
// y[m, n] = sum_k x[m, k] W[n, k], W[n, k] = s q + t of row n and k's group.  With
// v = 1 + q / 16, whose bf16 form is the code's bits in the mantissa of 1,
//
//   y[m, n] / 16 = sum over groups of s (sum_k x v - sum_k x) + t (sum_k x / 16)
//
// (without shifts of s (sum_k x v - 1.5 sum_k x)): the codes enter the products as they
// are, beginning from what the sums of x take away, which come from the same matrix
// instruction with a constant for weights; a group's two sums are scaled in fp32 by the
// half-precision s and t as they are.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cx_device.hpp"
#include "cx_dma.hpp"
#include "cx_internal.hpp"
#include "cx_lds.hpp"
#include "cx_sampler.h"
#include "cx_timing.hpp"

namespace cx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));

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

// Tiles of codes that a wave has asked for, 2 and 4 (K = 4096, us, weights from memory): 1 row
// N = 4096 7.9 and 8.0, N = 14336 11.0 and 12.3; 16 rows N = 14336 12.8 and 14.5, N = 128256
// 71.3 and 72.8; 61 rows N = 14336 21.7 and 23.0.
constexpr int W4_AHEAD = 2;
// The waves that a product should have, of the chip's 8192: two of a SIMD keep enough loads
// in flight, and each further one has less work for its x and its sums.  K = 4096, us, with
// half as many, these and twice as many (weights from memory): 16 rows, N = 6144 11.4, 9.1,
// 12.9; N = 14336 17.3, 12.8, 15.2; N = 50257 56, 35, 40; N = 128256 71, 71, 77; 61 rows, N =
// 14336 30.6, 21.7, 21.6; 30 rows, N = 50257 56, 40, 36.
constexpr int W4_WAVES = 1536;
constexpr int W4_CUS = 256;
// Rows of x so far apart that 16 of them pass 32 bits take the other kernel.
constexpr int64_t W4_STRIDE = 1 << 26;

// 8 codes as bf16 1 + q / 16.
// bits, one: 0x00780078 in a scalar register, 0x3F803F80 in a vector one, so that each two
// codes are a shift and a v_and_or.
__device__ __forceinline__ bf16x8 w4_values(uint32_t w, uint32_t bits, uint32_t one) {
  return __builtin_bit_cast(bf16x8, u32x4{(w << 3 & bits) | one, (w >> 1 & bits) | one,
                                          (w >> 5 & bits) | one, (w >> 9 & bits) | one});
}

// Where a wave's 16 NTW rows of W are.
template <int NTW, int GROUPS, bool SHIFT>
struct W4Rows {
  const char* code[NTW];
  const char* scale[NTW];
  int KT, groups;
  __device__ __forceinline__ W4Rows(const W4Args& A, int pair) {
    KT = (A.K + 127) / 128;
    groups = A.K / (128 / GROUPS);
#pragma unroll
    for (int n = 0; n < NTW; ++n) {
      const int t = min(pair * NTW + n, (A.N + 15) / 16 - 1);
      code[n] = (const char*)A.tiles + (int64_t)t * KT * 1024;
      scale[n] = (const char*)A.scales + (int64_t)t * groups * (SHIFT ? 64 : 32);
    }
  }
};
// A wave's part of a tile of 128 k: the codes of 16 NTW rows of W, row c's scales.
template <int NTW, int GROUPS>
struct W4Tile {
  u32x4 code[NTW];
  uint32_t scale[NTW][GROUPS];
  template <bool SHIFT>
  __device__ __forceinline__ void load(const W4Rows<NTW, GROUPS, SHIFT>& W, int kt) {
    kt = min(kt, W.KT - 1);
#pragma unroll
    for (int n = 0; n < NTW; ++n) {
      code[n] = __builtin_nontemporal_load((const u32x4*)(W.code[n] + (int64_t)kt * 1024 + 16 * lane_id()));
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) {
        const char* p = W.scale[n] + (int64_t)min(kt * GROUPS + q, W.groups - 1) * (SHIFT ? 64 : 32);
        const uint32_t c = lane_id() & 15;
        scale[n][q] = SHIFT ? ((const uint32_t*)p)[c] : ((const uint16_t*)p)[c];
      }
    }
  }
};
struct W4Constants {
  uint32_t bits, one;
  bf16x8 less, sixteenth;                    // weights of x's sums
};
template <bool SHIFT>
__device__ __forceinline__ W4Constants w4_constants() {
  W4Constants C;
  C.bits = 0x00780078u;
  C.one = 0x3F803F80u;
  asm("" : "+s"(C.bits), "+v"(C.one));
  auto constant = [](uint32_t two) { return __builtin_bit_cast(bf16x8, u32x4{two, two, two, two}); };
  C.less = constant(SHIFT ? 0xBF80BF80u : 0xBFC0BFC0u);                  // -1, -1.5
  C.sixteenth = constant(0x3D803D80u);
  return C;
}
// acc += the tile's products with x(i, k): rows 16 i .. of x, k 32 k .. of the tile; left:
// the groups that K has from the tile on.
template <int MT, int NTW, int STEPS, bool SHIFT, class X>
__device__ __forceinline__ void w4_multiply(const W4Constants& C, const W4Tile<NTW, 4 / STEPS>& t, int left,
                                            X x, f32x4 (&acc)[MT][NTW]) {
#pragma unroll
  for (int q = 0; q < 4 / STEPS; ++q) {
    if (q >= left) break;                    // (uniform: K may be no multiple of 128)
    // x of the group in registers where they are free, else read twice
    constexpr bool KEEP = MT * STEPS <= 8;
    bf16x8 xs[MT][KEEP ? STEPS : 1];
#pragma unroll
    for (int k = 0; k < (KEEP ? STEPS : 0); ++k)
#pragma unroll
      for (int i = 0; i < MT; ++i) xs[i][k] = __builtin_bit_cast(bf16x8, x(i, q * STEPS + k));
    auto row = [&](int i, int k) { return KEEP ? xs[i][k] : __builtin_bit_cast(bf16x8, x(i, q * STEPS + k)); };
    f32x4 p[MT][NTW], h[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      f32x4 from = {0, 0, 0, 0};
      h[i] = from;
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {
        if (!SHIFT || MT == 1) from = __builtin_amdgcn_mfma_f32_16x16x32_bf16(row(i, k), C.less, from, 0, 0, 0);
        if (SHIFT) h[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(row(i, k), C.sixteenth, h[i], 0, 0, 0);
      }
      // (few rows do not wait for h)
      if (SHIFT && MT > 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) from[j] = -16.f * h[i][j];
#pragma unroll
      for (int n = 0; n < NTW; ++n) p[i][n] = from;
    }
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      if (!KEEP) asm volatile("" ::: "memory");  // (not kept all the same)
#pragma unroll
      for (int n = 0; n < NTW; ++n) {
        const bf16x8 v = w4_values(t.code[n][q * STEPS + k], C.bits, C.one);
#pragma unroll
        for (int i = 0; i < MT; ++i) p[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(row(i, k), v, p[i][n], 0, 0, 0);
      }
    }
#pragma unroll
    for (int n = 0; n < NTW; ++n) {
      const half2 st = __builtin_bit_cast(half2, t.scale[n][q]);
      float f = (float)st[0], u = SHIFT ? (float)st[1] : 0.f;
      asm("" : "+v"(f), "+v"(u));            // converted once: no mixed-precision products
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (SHIFT) acc[i][n][j] = fmaf(u, h[i][j], acc[i][n][j]);
          acc[i][n][j] = fmaf(f, p[i][n][j], acc[i][n][j]);
        }
    }
  }
}
// acc out: rows m0 .., columns n0 ...
template <int MT, int NTW>
__device__ __forceinline__ void w4_out(const W4Args& A, const f32x4 (&acc)[MT][NTW], int m0, int n0) {
  const int l = lane_id(), g = l >> 4, c = l & 15;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NTW; ++n) {
      const int col = n0 + 16 * n + c;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + 16 * i + 4 * g + j;
        if (m >= A.M || col >= A.N) continue;
        if (A.bf16) ((__bf16*)A.out)[m * A.ldo + col] = (__bf16)(16.f * acc[i][n][j]);
        else ((float*)A.out)[m * A.ldo + col] = 16.f * acc[i][n][j];
      }
    }
}

// Few rows: a wave takes 16 NTW rows of W and, of their K, every WK-th tile of 128; the
// WK waves of the same rows add up through LDS.  All loads go straight to registers,
// codes and scales two tiles ahead, x (from the caches: a few rows) one.  Every wave
// reads all of x's part: at 16 rows that is as much as 64 rows of W, so that NTW = 4
// takes 65 us where 2 and 1 take 81 and 138 (N = 128256, K = 4096, groups of 32 with
// shifts: 337 MB, 5.2 TB/s, where reads reach 6.9); a lane's loads of the scales bring 4 bytes
// each.  One row, N = K = 4096: 4.8 us, of which about 3 are a launch's.
template <int NTW, int STEPS, bool SHIFT>
__global__ __launch_bounds__(512) void w4_stream(W4Args A) {
  constexpr int GROUPS = 4 / STEPS;          // of a tile
  __shared__ f32x4 s_sum[7][NTW * 64];
  const int w = __builtin_amdgcn_readfirstlane(wave_id()), l = lane_id(), g = l >> 4, c = l & 15;
  const int wk = w & (A.wk - 1), pair = (int)blockIdx.x * (8 / A.wk) + w / A.wk;
  const int KT = (A.K + 127) / 128, groups = A.K / (32 * STEPS), steps = A.K / 32;
  const uint32_t xo = (uint32_t)((min(c, A.M - 1) * A.ldx + 8 * g) * 2);  // (below 2^32: W4_STRIDE)
  const W4Rows<NTW, GROUPS, SHIFT> W(A, pair);
  using Tile = W4Tile<NTW, GROUPS>;
  struct Rows {
    u32x4 x[4];
  };
  auto load = [&](Tile& t, int kt) { t.load(W, kt); };
  auto load_x = [&](Rows& r, int kt) {
#pragma unroll
    for (int k = 0; k < 4; ++k) r.x[k] = *(const u32x4*)((const char*)A.x + 64 * (int64_t)min(kt * 4 + k, steps - 1) + xo);
  };
  f32x4 acc[1][NTW];
#pragma unroll
  for (int n = 0; n < NTW; ++n) acc[0][n] = f32x4{0, 0, 0, 0};
  const W4Constants C = w4_constants<SHIFT>();
  Tile t[W4_AHEAD];
  Rows r[2];
  load(t[0], wk);
  load_x(r[0], wk);
#pragma unroll
  for (int u = 1; u < W4_AHEAD; ++u) load(t[u], wk + u * A.wk);
  for (int k0 = wk; k0 < KT; k0 += W4_AHEAD * A.wk)
#pragma unroll
    for (int u = 0; u < W4_AHEAD; ++u) {
      const int kt = k0 + u * A.wk;
      if (u > 0 && kt >= KT) break;
      load_x(r[(u + 1) & 1], kt + A.wk);
      w4_multiply<1, NTW, STEPS, SHIFT>(C, t[u], groups - kt * GROUPS, [&](int, int k) { return r[u & 1].x[k]; }, acc);
      load(t[u], kt + W4_AHEAD * A.wk);
    }
  // the waves' sums, in the order of wk
  if (A.wk > 1) {
    f32x4* const at = s_sum[0] + (w / A.wk) * (A.wk - 1) * (NTW * 64) + l;
    if (wk > 0) {
#pragma unroll
      for (int n = 0; n < NTW; ++n) at[((wk - 1) * NTW + n) * 64] = acc[0][n];
    }
    __syncthreads();
    if (wk > 0) return;
    for (int k = 0; k < A.wk - 1; ++k)
#pragma unroll
      for (int n = 0; n < NTW; ++n) acc[0][n] += at[(k * NTW + n) * 64];
  }
  w4_out<1, NTW>(A, acc, 0, pair * NTW * 16);
}

// More rows: x passes through LDS, for all waves of a workgroup.  8 / WK waves side by side
// take 16 NTW rows of W each, WK waves every WK-th tile of K; a step is a tile of each,
// its x sent to LDS a step ahead, past the registers (through them 22.4 us, not 20.1), its
// codes two ahead.  A row's 16 chunks of 8 k stand in the order of their number ^ the row's,
// so that the 16 rows that a lane group reads are in different banks.  61 rows, N = 14336, K =
// 4096: 20.1 us, 37 with every wave's own loads of x; 30 rows 13.9 us.  A step is 2.1 us, with
// 0.75 of matrix instructions: x in and out of LDS (192 KB a CU), conversions and scales are
// beside them.
template <int MT, int NTW, int WK, int STEPS, bool SHIFT>
__global__ __launch_bounds__(512) void w4_tile(W4Args A) {
  constexpr int GROUPS = 4 / STEPS, ROWS = 16 * MT, CHUNKS = ROWS * 16;  // 16-byte chunks of a tile's x
  constexpr int XL = WK * CHUNKS / 512;      // of a thread
  static_assert(WK * CHUNKS % 512 == 0, "whole loads");
  extern __shared__ __align__(16) char w4_lds[];
  CX_LDS u32x4* const s_x = (CX_LDS u32x4*)to_lds(w4_lds);               // [2][WK][ROWS][16]
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(wave_id()), l = lane_id();
  const int g = l >> 4, c = l & 15;
  const int wk = w % WK, pair = (int)blockIdx.x * (8 / WK) + w / WK;
  const int m0 = blockIdx.y * ROWS;
  const int KT = (A.K + 127) / 128, groups = A.K / (32 * STEPS), chunks = A.K / 8;
  const int iters = (KT + WK - 1) / WK;
  const W4Rows<NTW, GROUPS, SHIFT> W(A, pair);
  using Tile = W4Tile<NTW, GROUPS>;
  auto load = [&](Tile& t, int it) { t.load(W, it * WK + wk); };
  // this thread's chunks of x: place 512 j + tid is (wave k, row, place in the row)
  auto load_x = [&](int it) {
#pragma unroll
    for (int j = 0; j < XL; ++j) {
      const int at = 512 * j + tid, row = at / 16 % ROWS, kt = min(it * WK + at / CHUNKS, KT - 1);
      const int k = min(kt * 16 + (at % 16 ^ (row & 15)), chunks - 1);
      load_lds16((const char*)(A.x + min(m0 + row, A.M - 1) * A.ldx + 8 * (int64_t)k),
                 (uint32_t)(uintptr_t)s_x + 16 * ((it & 1) * WK * CHUNKS + 512 * j + 64 * w));
    }
  };
  const W4Constants C = w4_constants<SHIFT>();
  f32x4 acc[MT][NTW];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NTW; ++n) acc[i][n] = f32x4{0, 0, 0, 0};
  auto step = [&](int it, Tile& t) {
    // this step's x and codes are there (the next codes alone are on their way), in all waves,
    // and the step before has been read
    wave_vm<NTW * (1 + GROUPS)>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // (the compiler's own wait for the codes: behind the loads of x it would take in those)
#pragma unroll
    for (int n = 0; n < NTW; ++n) {
      asm volatile("" : "+v"(t.code[n]));
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) asm volatile("" : "+v"(t.scale[n][q]));
    }
    load_x(it + 1);
    const CX_LDS u32x4* xs = s_x + ((it & 1) * WK + wk) * CHUNKS;
    w4_multiply<MT, NTW, STEPS, SHIFT>(
        C, t, groups - (it * WK + wk) * GROUPS,
        [&](int i, int k) { return xs[(16 * i + c) * 16 + ((4 * k + g) ^ c)]; }, acc);
    load(t, it + W4_AHEAD);
  };
  Tile t[W4_AHEAD];
  load(t[0], 0);
  load_x(0);
#pragma unroll
  for (int u = 1; u < W4_AHEAD; ++u) load(t[u], u);
  for (int i0 = 0; i0 < iters; i0 += W4_AHEAD)
#pragma unroll
    for (int u = 0; u < W4_AHEAD; ++u) {
      if (u > 0 && i0 + u >= iters) break;
      step(i0 + u, t[u]);
    }
  wave_vm<0>();                              // the last loads write LDS
  // the waves' sums, in the order of wk
  if (WK > 1) {
    __syncthreads();
    CX_LDS f32x4* const at = (CX_LDS f32x4*)s_x + (w / WK) * (WK - 1) * MT * NTW * 64 + l;
    if (wk > 0) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NTW; ++n) at[((wk - 1) * MT * NTW + i * NTW + n) * 64] = acc[i][n];
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int k = 0; k < WK - 1; ++k)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NTW; ++n) acc[i][n] += at[(k * MT * NTW + i * NTW + n) * 64];
  }
  w4_out<MT, NTW>(A, acc, m0, pair * NTW * 16);
}
template <int MT, int NTW, int WK>
constexpr int w4_lds_bytes() {
  const int x = 2 * WK * 16 * MT * 256, sums = 8 / WK * (WK - 1) * MT * NTW * 1024;
  return x > sums ? x : sums;
}

using W4Kernel = void (*)(W4Args);
template <int NTW>
static void launch_stream(W4Args A, int group, bool shifts, hipStream_t s) {
  const int pairs = (A.N + 16 * NTW - 1) / (16 * NTW);
  static const W4Kernel kernels[3][2] = {{w4_stream<NTW, 1, false>, w4_stream<NTW, 1, true>},
                                         {w4_stream<NTW, 2, false>, w4_stream<NTW, 2, true>},
                                         {w4_stream<NTW, 4, false>, w4_stream<NTW, 4, true>}};
  A.wk = 1;
  while (A.wk < 8 && (int64_t)pairs * A.wk < W4_WAVES && (A.K + 127) / 128 >= 4 * A.wk) A.wk *= 2;
  timed_launch(CX_KERNEL_W4, kernels[group / 64][shifts], dim3((pairs * (int64_t)A.wk + 7) / 8), dim3(512), 0, s, A);
}
template <int MT, int NTW, int WK>
static hipError_t launch_tile(const W4Args& A, int group, bool shifts, hipStream_t s) {
  const int pairs = (A.N + 16 * NTW - 1) / (16 * NTW);
  static const W4Kernel kernels[3][2] = {{w4_tile<MT, NTW, WK, 1, false>, w4_tile<MT, NTW, WK, 1, true>},
                                         {w4_tile<MT, NTW, WK, 2, false>, w4_tile<MT, NTW, WK, 2, true>},
                                         {w4_tile<MT, NTW, WK, 4, false>, w4_tile<MT, NTW, WK, 4, true>}};
  static LdsLimit limits[3][2];
  constexpr int lds = w4_lds_bytes<MT, NTW, WK>();
  const W4Kernel k = kernels[group / 64][shifts];
  if (int e = limits[group / 64][shifts].raise((const void*)k, lds)) return (hipError_t)e;
  timed_launch(CX_KERNEL_W4, k, dim3((pairs * (int64_t)WK + 7) / 8, (A.M + 16 * MT - 1) / (16 * MT)), dim3(512), lds, s, A);
  return hipSuccess;
}
// Rows of W a wave, waves that share them: few and many while the workgroups are on the chip
// at once, then as many rows as leave W4_WAVES waves.  K = 4096, 30 and 61 rows, with 16
// rows of W a wave and with 32: N = 4096 8.2 and 14.6, 9.9 and 19.5 us; N = 14336 26.5 and
// 27.4, 13.9 and 20.1 us; N = 6144, 32 rows, 15.2 and 11.0 us.  30 rows with 32 and with 64:
// N = 50257 38.9 and 55.8 us, N = 128256 67.2 and 61.2.
template <int MT>
static hipError_t launch_tiles(const W4Args& A, int group, bool shifts, hipStream_t s) {
  const int pairs = (A.N + 31) / 32;
  if (pairs <= W4_CUS) {
    if constexpr (MT == 2)
      if (pairs * 2 > W4_CUS) return launch_tile<MT, 2, 8>(A, group, shifts, s);
    return launch_tile<MT, 1, 16 / MT>(A, group, shifts, s);
  }
  if (pairs * 2 < W4_WAVES) return launch_tile<MT, 2, 4>(A, group, shifts, s);
  if (pairs < W4_WAVES) return launch_tile<MT, 2, 2>(A, group, shifts, s);
  if constexpr (MT == 2)                     // (64 of 64 rows do not fit the registers)
    if (pairs / 2 >= W4_WAVES) return launch_tile<MT, 4, 1>(A, group, shifts, s);
  return launch_tile<MT, 2, 1>(A, group, shifts, s);
}
static hipError_t launch_w4(const W4Args& A, int group, bool shifts, hipStream_t s) {
  const int tiles = (A.N + 15) / 16;
  // 32 rows a workgroup also where these are all on the chip at once (64 rows, N = 512, K =
  // 14336: 18 us, 45 with 64 rows a workgroup; 128 rows, N = 1024, K = 4096: 8.0 and 15.8)
  if (A.M > 32 && tiles * (int64_t)((A.M + 31) / 32) > W4_CUS) return launch_tiles<4>(A, group, shifts, s);
  if (A.M > 16 || A.ldx > W4_STRIDE) return launch_tiles<2>(A, group, shifts, s);
  if (tiles * (8 / 4) >= W4_WAVES) launch_stream<4>(A, group, shifts, s);
  else if (tiles * (8 / 2) >= W4_WAVES) launch_stream<2>(A, group, shifts, s);
  else launch_stream<1>(A, group, shifts, s);
  return hipSuccess;
}

}  // namespace cx

extern "C" int cx_w4_linear_bf16(const uint16_t* x, int64_t ldx, const uint32_t* tiles,
                                 const uint16_t* scales, int32_t shifts, int32_t group, int32_t M,
                                 int32_t N, int32_t K, void* out, int64_t ldo, int32_t out_bf16,
                                 void* stream) {
  // (65535 workgroups of 64 rows; the kernels' counts are ints)
  if (M < 0 || N < 1 || K < 1 || M >= 1 << 21 || N >= 1 << 28 || K >= 1 << 28 || ldx < K || ldo < N)
    return cx::api_fail(CX_EINVAL, "bad shape (%d, %d, %d)", M, N, K);
  if (group != 32 && group != 64 && group != 128)
    return cx::api_fail(CX_EINVAL, "group (%d) must be 32, 64 or 128", group);
  if (K % group) return cx::api_fail(CX_EINVAL, "K (%d) must be a multiple of the group (%d)", K, group);
  if (M == 0) return CX_OK;
  if (!x || !tiles || !scales || !out) return cx::api_fail(CX_EINVAL, "null pointer argument");
  if ((((uintptr_t)x | (uintptr_t)tiles | (uintptr_t)scales) & 15) || (ldx & 7))
    return cx::api_fail(CX_EINVAL, "rows of x, tiles and scales must be 16-byte aligned");
  if ((uintptr_t)out & (out_bf16 ? 1 : 3)) return cx::api_fail(CX_EINVAL, "out must be aligned to its type");
  const cx::W4Args A = {x, ldx, tiles, scales, M, N, K, 1, out, ldo, out_bf16 != 0};
  hipError_t e = cx::launch_w4(A, group, shifts != 0, (hipStream_t)stream);
  if (e == hipSuccess) e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "w4 launch: %s", hipGetErrorString(e));
  return CX_OK;
}
