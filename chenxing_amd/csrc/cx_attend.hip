// cx_attend.hip -- attention of the new tokens over the paged KV cache, for
// gfx950 (layout: cx_kv.hpp).
//
// out[t, h] = sum over the allowed positions s of softmax(scale q.k_s) v_s, in
// one pass over K and V with the running maximum m and sum l of the softmax's
// terms: a block of scores raises m to m', and l and the output so far are
// scaled by exp(m - m').  Two stream-ordered launches:
//
//   1. attend_split  workgroups of 4 waves, each with an equal share of all the
//                    batch's units (32 tokens of bf16, 64 of e4m3, for one kv
//                    head and row block); a row block that ends inside the share
//                    it began in is written out, the others' parts (m, l, sums)
//                    go to the workspace.
//   2. attend_join   one workgroup per split row block: its parts, in the order
//                    of its tokens.
//
// Bound: HBM, every page read once.  A row block is 16 NT rows of (new token, q
// head of the kv head's group); 16 rows of one unit are 24 MFMAs (head_dim 128)
// for 16 KB.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <mutex>
#include <type_traits>

#include "cx_device.hpp"
#include "cx_internal.hpp"
#include "cx_kv.hpp"
#include "cx_sampler.h"
#include "cx_timing.hpp"

namespace cx {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int ATT_WAVES = 4, ATT_WG = 64 * ATT_WAVES;
constexpr int ATT_MIN_UNITS = ATT_WAVES;     // of a workgroup's share: one per wave
constexpr float ATT_LOW = -3e38f;            // running maximum of a row that attends to something

struct AttendArgs {
  KvArgs kv;
  const uint16_t* q;
  int64_t q_token, q_head;
  int q_heads, G;             // G: q heads per kv head
  float s1, s2;               // score in powers of 2: s1 qk, or s2 tanh(s1 / 2 qk)
  int cap;                    // the latter
  int window;                 // 0: none
  uint16_t* out;
  struct AttendJoin* join;    // [grid]
  float* ml;                  // [2 grid, ROWS, 2]: a part's maxima and sums
  float* part;                // [2 grid, ROWS, D]
};

// A row block whose units lie in several workgroups' shares: those of
// workgroups first .. last.  Written by the first; none: last = -1.
struct AttendJoin {
  int first, last;
  int tok0, row0, rows, head;
  int pad[2];
};

// What a workgroup needs of a sequence: its rows among the new tokens, the
// length, and its units of TOK tokens (those in some row's window).
struct AttendSeq {
  int tok0, q, len, lim, first, n;
};
template <int TOK>
__device__ __forceinline__ AttendSeq attend_seq(const AttendArgs& A, int b) {
  const KvArgs& C = A.kv;
  AttendSeq s;
  const int2 r = kv_rows(C, b);
  s.tok0 = r.x;
  s.q = r.y - r.x;
  s.len = max(C.kv_len[b], 0);               // no position is reached by a shorter one
  s.lim = C.n_pages ? min(s.len, C.M << C.logP) : 0;
  const int lowest = s.len - s.q;
  s.first = A.window && lowest >= A.window ? (lowest - A.window + 1) / TOK : 0;
  s.n = s.q > 0 ? max((s.lim + TOK - 1) / TOK - s.first, 0) : 0;
  return s;
}

// A value that every lane holds, in scalar registers.
__device__ __forceinline__ uint64_t scalar64(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}

__device__ __forceinline__ bf16x8 e4m3x8(uint32_t a, uint32_t b) {
  const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
  const bf16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
  const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
  const bf16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
  return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

template <int D, int NT, bool F8>
struct AttendShape {
  static constexpr int TOK = F8 ? 64 : 32;   // tokens of a unit
  static constexpr int ROWS = 16 * NT;
  static constexpr int E = F8 ? 16 : 8;      // elements of a 16-byte chunk
  static constexpr int PAD = D + 4;          // floats of a row of s_o
  static constexpr int WAVES = NT == 1 && D < 256 ? 2 : 1;   // per SIMD
  static constexpr int OFF_O = ROWS * D * 2;
  static constexpr int OFF_ML = OFF_O + ATT_WAVES * 16 * PAD * 4;
  static constexpr int OFF_SCALE = OFF_ML + ATT_WAVES * ROWS * 8;
  static constexpr int OFF_PREF = OFF_SCALE + (F8 ? ATT_WAVES * 512 : 0) + ATT_WAVES * 8;
  static int lds(int B) { return OFF_PREF + 8 * (B + 1); }
};

// The lengths are on the device, so each workgroup finds its share itself: the
// units of every sequence summed up in LDS, and its range of the total.  Its
// waves take the units of a row block in turn and merge through LDS at its end.
//
//  * S^T = K Q^T, so a lane holds scores of 4 neighbouring tokens a tile for its
//    row (column) and the softmax's statistics need two shuffles; tile y's row
//    4 g + j is the unit's token (TOK / 4) g + 4 y + j, which makes a lane's
//    terms the very operand of O^T = V^T P^T, and its part of V 16 contiguous
//    bytes of a page: neither passes through LDS.
//  * The next unit's K is requested when this unit's scores are taken, its V
//    after this unit's products: half of a unit's 16 KB is always in flight.
//  * Softmax terms enter the products as two bf16 parts (16 bits): one part's
//    rounding would add as much error as the result's own.
template <int D, int NT, bool F8>
__global__ __launch_bounds__(ATT_WG, (AttendShape<D, NT, F8>::WAVES)) void attend_split(AttendArgs A) {
  using Sh = AttendShape<D, NT, F8>;
  constexpr int TOK = Sh::TOK, ROWS = Sh::ROWS, E = Sh::E, PAD = Sh::PAD;
  constexpr int KT = TOK / 16;               // score tiles of a unit, and its 16-token groups
  constexpr int KL = D / (4 * E);            // K loads of a tile
  constexpr int DT = D / 16, KH = TOK / 32;
  constexpr int BATCH = 64 / KT;             // units whose page ids a wave holds
  extern __shared__ __align__(16) char lds[];
  CX_LDS u32x4* const s_q = to_lds((u32x4*)lds);
  CX_LDS float* const s_o = to_lds((float*)(lds + Sh::OFF_O));
  CX_LDS float* const s_ml = to_lds((float*)(lds + Sh::OFF_ML));
  CX_LDS float* const s_scale = to_lds((float*)(lds + Sh::OFF_SCALE)) + wave_id() * 128;
  CX_LDS uint64_t* const s_sum = to_lds((uint64_t*)(lds + Sh::OFF_PREF)) - ATT_WAVES;
  CX_LDS uint64_t* const s_pref = to_lds((uint64_t*)(lds + Sh::OFF_PREF));
  const KvArgs& C = A.kv;
  const int tid = threadIdx.x, w = wave_id(), l = lane_id(), g = l >> 4, c = l & 15;
  const int P = 1 << C.logP;

  // units before each sequence, over its kv heads and row blocks
  if (tid == 0) s_pref[0] = 0;
  uint64_t run = 0;
  for (int b0 = 0; b0 < C.B; b0 += ATT_WG) {
    const int b = b0 + tid;
    uint64_t x = 0;
    if (b < C.B) {
      const AttendSeq s = attend_seq<TOK>(A, b);
      x = (uint64_t)s.n * C.heads * ((s.q * A.G + ROWS - 1) / ROWS);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t y = __shfl_up(x, o);
      if (l >= o) x += y;
    }
    if (l == 63) s_sum[w] = x;
    __syncthreads();
    for (int k = 0; k < w; ++k) x += s_sum[k];
    if (b < C.B) s_pref[b + 1] = run + x;
    __syncthreads();
    run = s_pref[min(b0 + ATT_WG, C.B)];
  }
  const uint64_t total = run;

  // tokens that attend to nothing
  for (int b = blockIdx.x; b < C.B; b += gridDim.x)
    if (s_pref[b + 1] == s_pref[b]) {
      const int2 r = kv_rows(C, b);
      const int64_t n = (int64_t)(r.y - r.x) * A.q_heads * (D / 8);
      u32x4* o = (u32x4*)(A.out + (int64_t)r.x * A.q_heads * D);
      for (int64_t i = tid; i < n; i += ATT_WG) o[i] = u32x4{0, 0, 0, 0};
    }

  // this workgroup's share of the units: as many workgroups as have
  // ATT_MIN_UNITS, the first ones with one unit more
  const uint64_t shares = min((uint64_t)gridDim.x, (total + ATT_MIN_UNITS - 1) / ATT_MIN_UNITS);
  bool joined = false;
  if (blockIdx.x < shares) {
    const uint64_t per = total / shares, more = total % shares;
    uint64_t u = scalar64(blockIdx.x * per + min((uint64_t)blockIdx.x, more));
    const uint64_t end = scalar64(u + per + (blockIdx.x < more));
    int b = 0;
    for (int hi = C.B - 1; b < hi;) {        // the last b with s_pref[b] <= u
      const int mid = (b + hi + 1) >> 1;
      if (s_pref[mid] <= u) b = mid;
      else hi = mid - 1;
    }
    while (u < end) {
      while (s_pref[b + 1] <= u) ++b;
      b = __builtin_amdgcn_readfirstlane(b);
      const AttendSeq s = attend_seq<TOK>(A, b);
      const uint64_t rem = scalar64(u - s_pref[b]);
      const int blocks = (s.q * A.G + ROWS - 1) / ROWS;
      const unsigned row = rem >> 32 ? (unsigned)(rem / (unsigned)s.n)
                                     : (unsigned)rem / (unsigned)s.n;
      const int ua = (int)(rem - (uint64_t)row * (unsigned)s.n);
      const int ub = (int)min((uint64_t)s.n, ua + (end - u));
      const int h = __builtin_amdgcn_readfirstlane((int)(row / (unsigned)blocks));
      const int r0 = __builtin_amdgcn_readfirstlane((int)(row % (unsigned)blocks)) * ROWS;
      const int R = min(ROWS, s.q * A.G - r0);
      const bool whole = ua == 0 && ub == s.n;
      const int slot = 2 * blockIdx.x + (ua == 0);
      if (ua == 0 && !whole) {
        joined = true;
        if (tid == 0) {
          const uint64_t lastu = u + s.n - 1, cut = more * (per + 1);
          AttendJoin j;
          j.first = blockIdx.x;
          j.last = (int)(lastu < cut ? lastu / (per + 1) : more + (lastu - cut) / per);
          j.tok0 = s.tok0; j.row0 = r0; j.rows = R; j.head = h;
          j.pad[0] = j.pad[1] = 0;
          A.join[blockIdx.x] = j;
        }
      }
      u += ub - ua;

      __syncthreads();                       // the last segment's reads of LDS are done
      for (int i = tid; i < ROWS * (D / 8); i += ATT_WG) {
        const int r = i % ROWS, ch = i / ROWS;
        u32x4 x = {0, 0, 0, 0};
        if (r < R)
          x = *(const u32x4*)(A.q + (s.tok0 + (r0 + r) / A.G) * A.q_token +
                              (h * A.G + (r0 + r) % A.G) * A.q_head + 8 * ch);
        s_q[i] = x;
      }

      const int lowest = s.len - s.q;
      int pos[NT];                           // this lane's rows
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) pos[nt] = lowest + min(r0 + 16 * nt + c, r0 + R - 1) / A.G;
      const int pmin = lowest + r0 / A.G, pmax = lowest + (r0 + R - 1) / A.G;

      const int cnt = (ub - ua - w + ATT_WAVES - 1) / ATT_WAVES;   // this wave's units
      const int unit0 = s.first + ua + w;
      // ids of BATCH units from the k-th: lane KT k + group
      auto load_ids = [&](int k) {
        const int t16 = (unit0 + ATT_WAVES * (k + l / KT)) * KT + l % KT;
        int id = -1;
        if (t16 < (s.lim + 15) >> 4) id = C.table[b * C.ld_table + (t16 >> (C.logP - 4))];
        return (unsigned)id < (unsigned)C.n_pages ? id : -1;
      };
      // this lane's one of a unit's page ids: of its row of K, or of its tokens
      auto pick = [&](int ids, int k, int group) {
        int id = lane_read(ids, k * KT);
#pragma unroll
        for (int x = 1; x < KT; ++x) {
          const int y = lane_read(ids, k * KT + x);
          id = group == x ? y : id;
        }
        return id;
      };
      const int kgroup = F8 ? c >> 2 : c >> 3, vgroup = F8 ? g : g >> 1;
      // place in the page of a unit's 16-token group
      auto place = [&](int unit, int group) { return ((unit * KT + group) << 4) & (P - 1); };

      u32x4 kr[KT][KL], vr[DT];
      float ks = 1.f, vs = 1.f;              // e4m3: the scales of the unit's token l
      const char* const head0 = C.pages + (int64_t)h * C.head_bytes;
      const char *vp = nullptr, *vnext = nullptr;
      bool held = false, hnext = false;
      auto load_k = [&](int ids, int k, int unit) {
        const int id = pick(ids, k, kgroup), vid = pick(ids, k, vgroup);
        const char* p = head0 + max(id, 0) * C.page_stride +
                        ((place(unit, kgroup) + (F8 ? c & 3 : (c & 3) + 2 * (c & 4))) << 4) +
                        (g << (C.logP + 4));
#pragma unroll
        for (int x = 0; x < KL; ++x)
#pragma unroll
          for (int y = 0; y < KT; ++y)
            kr[y][x] = *(const u32x4*)(p + 64 * y + ((int64_t)x << (C.logP + 6)));
        vnext = head0 + max(vid, 0) * C.page_stride;
        hnext = vid >= 0;
        if (F8) ks = *(const float*)(vnext + k_scale<D>(place(unit, g) + c, C.logP));
      };
      auto load_v = [&](int unit) {
        vp = vnext;
        held = hnext;
        const char* p = vp + v_chunk<E, D>(c, place(unit, vgroup) + (F8 ? 0 : 8 * (g & 1)), C.logP);
#pragma unroll
        for (int n = 0; n < DT; ++n) vr[n] = *(const u32x4*)(p + 256 * n);
        if (F8) vs = *(const float*)(vp + v_scale<D>(place(unit, g) + c, C.logP));
      };

      f32x4 acc[NT][DT];
      float m[NT], sum[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        sum[nt] = 0;
#pragma unroll
        for (int n = 0; n < DT; ++n) acc[nt][n] = f32x4{0, 0, 0, 0};
      }
      int ids = -1, idn = -1;
      if (cnt > 0) {
        ids = load_ids(0);
        idn = load_ids(BATCH);
        load_k(ids, 0, unit0);
        load_v(unit0);
      }
      __syncthreads();                       // s_q
      for (int i = 0; i < cnt; ++i) {
        const int unit = unit0 + ATT_WAVES * i, t0 = unit * TOK;
        // a unit is open where all its tokens are held, at or before the first
        // row and inside the last row's window
        const bool masked = t0 + TOK - 1 > pmin || t0 + TOK > s.lim ||
                            (A.window && t0 <= pmax - A.window) || __any(!held);
        const int tl = t0 + (TOK / 4) * g;   // this lane's first token
        const bool more_units = i + 1 < cnt;
        u32x4 ph[NT][KH], pl[NT][KH];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // scores: tile y's row 4 g + j is token t0 + (TOK / 4) g + 4 y + j
          f32x4 v[KT];
#pragma unroll
          for (int y = 0; y < KT; ++y) v[y] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int x = 0; x < KL; ++x)
#pragma unroll
            for (int e = 0; e < (F8 ? 2 : 1); ++e) {
              const u32x4 qv = s_q[(F8 ? 2 * (4 * x + g) + e : 4 * x + g) * ROWS + 16 * nt + c];
#pragma unroll
              for (int y = 0; y < KT; ++y) {
                const bf16x8 ka = F8 ? e4m3x8(kr[y][x][2 * e], kr[y][x][2 * e + 1])
                                     : __builtin_bit_cast(bf16x8, kr[y][x]);
                v[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, __builtin_bit_cast(bf16x8, qv),
                                                               v[y], 0, 0, 0);
              }
            }
          if (F8) {
            if (nt == 0) {                   // the wave's own words: no barrier
              s_scale[l] = ks;
              s_scale[64 + l] = vs;
              asm volatile("" ::: "memory");
            }
#pragma unroll
            for (int y = 0; y < KT; ++y) v[y] *= *(const CX_LDS f32x4*)(s_scale + 16 * g + 4 * y);
          }
          if (nt == NT - 1 && more_units) {  // K is used up: the next unit's
            const int k = (i + 1) % BATCH;
            if (k == 0) {
              ids = idn;
              idn = load_ids(i + 1 + BATCH);
            }
            load_k(ids, k, unit + ATT_WAVES);
          }
#pragma unroll
          for (int y = 0; y < KT; ++y) v[y] *= A.s1;
          if (A.cap) {                       // tanh(z) = 1 - 2 / (exp(2 z) + 1)
#pragma unroll
            for (int y = 0; y < KT; ++y)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                v[y][j] = fmaf(-2.f * A.s2,
                               __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(v[y][j]) + 1.f), A.s2);
          }
          // a row's running maximum is at least ATT_LOW once it has attended to
          // a token, whatever its score: -inf says that it has not
          float top = ATT_LOW;
          if (masked) {
            top = -INFINITY;
#pragma unroll
            for (int y = 0; y < KT; ++y)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int t = tl + 4 * y + j;
                const bool in = held && t <= pos[nt] && t < s.lim &&
                                !(A.window && t <= pos[nt] - A.window);
                v[y][j] = in ? v[y][j] : -INFINITY;
                top = in ? ATT_LOW : top;
              }
          }
#pragma unroll
          for (int y = 0; y < KT; ++y)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, v[y][j]);
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float m1 = fmaxf(m[nt], top);
          const float base = m1 == -INFINITY ? 0.f : m1;
          const float alpha = __builtin_amdgcn_exp2f(m[nt] - base);
          m[nt] = m1;
          float add = 0;
#pragma unroll
          for (int k = 0; k < KH; ++k) {
            float term[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int y = 2 * k + e / 4, j = e % 4;
              float p = __builtin_amdgcn_exp2f(v[y][j] - base);
              add += p;
              if (F8) p = v[y][j] == -INFINITY ? 0.f : p * s_scale[64 + 16 * g + 4 * y + j];
              term[e] = p;
            }
            // the terms as two bf16 parts each, 16 bits of them.  The first is
            // cut off and the second kept above 0, so an infinite value keeps
            // its sign in both products
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const uint32_t x0 = __float_as_uint(term[2 * d]), x1 = __float_as_uint(term[2 * d + 1]);
              ph[nt][k][d] = __builtin_amdgcn_perm(x1, x0, 0x07060302);
              pl[nt][k][d] = pack_bf16(
                  fmaxf(term[2 * d] - __uint_as_float(x0 & 0xFFFF0000u), term[2 * d] * 0x1p-24f),
                  fmaxf(term[2 * d + 1] - __uint_as_float(x1 & 0xFFFF0000u),
                        term[2 * d + 1] * 0x1p-24f));
            }
          }
          sum[nt] = fmaf(sum[nt], alpha, add);
          if (__any(alpha != 1.f)) {
#pragma unroll
            for (int n = 0; n < DT; ++n) acc[nt][n] *= alpha;
          }
        }
        // V's tokens from after lo through hi that are held, as a mask of each of
        // the lane's dwords: the others count as zeros, whatever is there (a
        // product with a zero term would not)
        uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
        auto keep_bits = [&](int lo, int hi) {
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            keep[d] = 0;
#pragma unroll
            for (int e = 0; e < E / 4; ++e) {
              const int t = tl + E / 4 * d + e;
              keep[d] |= held && t < s.lim && t <= hi && t > lo
                             ? (F8 ? 0xFFu << 8 * e : 0xFFFFu << 16 * e) : 0;
            }
          }
        };
        // NaN or infinity that only some rows may attend to: one position's rows
        // after the other, each with its own tokens of V
        bool fix = false;
        if (masked) {
          keep_bits(A.window ? pmin - A.window : -1, pmax);
          bool bad = false;
#pragma unroll
          for (int n = 0; n < DT; ++n)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const uint32_t x = vr[n][d] & keep[d];
              if (F8) bad |= (((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
              else bad |= (x & 0x7F80u) == 0x7F80u || (x & 0x7F800000u) == 0x7F800000u;
            }
          fix = pmin != pmax && __any(bad);
        }
        int q = fix ? pmin : pmax;
        do {
          if (fix) keep_bits(A.window ? q - A.window : -1, q);
#pragma unroll
          for (int n = 0; n < DT; ++n)
#pragma unroll
            for (int k = 0; k < KH; ++k) {
              u32x4 x = vr[n];
#pragma unroll
              for (int d = 0; d < 4; ++d) x[d] &= keep[d];
              const bf16x8 va = F8 ? e4m3x8(x[2 * k], x[2 * k + 1]) : __builtin_bit_cast(bf16x8, x);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                f32x4 o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    va, __builtin_bit_cast(bf16x8, ph[nt][k]), acc[nt][n], 0, 0, 0);
                o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8, pl[nt][k]), o,
                                                            0, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  acc[nt][n][j] = !fix || pos[nt] == q ? o[j] : acc[nt][n][j];
              }
            }
        } while (++q <= pmax);
        if (more_units) load_v(unit + ATT_WAVES);
      }

      // the waves' parts added in their order
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sum[nt] += __shfl_xor(sum[nt], 16);
        sum[nt] += __shfl_xor(sum[nt], 32);
        if (g == 0) {
          s_ml[2 * (w * ROWS + 16 * nt + c)] = m[nt];
          s_ml[2 * (w * ROWS + 16 * nt + c) + 1] = sum[nt];
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < DT; ++n)
          *(CX_LDS f32x4*)(s_o + (w * 16 + c) * PAD + 16 * n + 4 * g) = acc[nt][n];
        __syncthreads();
        for (int i = tid; i < 16 * (D / 8); i += ATT_WG) {
          const int r = i / (D / 8), d = 8 * (i % (D / 8)), rr = 16 * nt + r;
          if (rr >= R) continue;
          float top = -INFINITY, L = 0;
#pragma unroll
          for (int k = 0; k < ATT_WAVES; ++k) top = fmaxf(top, s_ml[2 * (k * ROWS + rr)]);
          const float base = top == -INFINITY ? 0.f : top;
          f32x4 o0 = {0, 0, 0, 0}, o1 = {0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < ATT_WAVES; ++k) {
            const float f = __builtin_amdgcn_exp2f(s_ml[2 * (k * ROWS + rr)] - base);
            L = fmaf(f, s_ml[2 * (k * ROWS + rr) + 1], L);
            const CX_LDS float* o = s_o + (k * 16 + r) * PAD + d;
            o0 += f * *(const CX_LDS f32x4*)o;
            o1 += f * *(const CX_LDS f32x4*)(o + 4);
          }
          if (whole) {
            const float f = top == -INFINITY ? 0.f : 1.f / L;
            const u32x4 x = {pack_bf16(o0[0] * f, o0[1] * f), pack_bf16(o0[2] * f, o0[3] * f),
                             pack_bf16(o1[0] * f, o1[1] * f), pack_bf16(o1[2] * f, o1[3] * f)};
            *(u32x4*)(A.out + ((int64_t)(s.tok0 + (r0 + rr) / A.G) * A.q_heads + h * A.G +
                               (r0 + rr) % A.G) * D + d) = x;
          } else {
            float* o = A.part + ((int64_t)slot * ROWS + rr) * D + d;
            *(f32x4*)o = o0;
            *(f32x4*)(o + 4) = o1;
            if (d == 0) {
              A.ml[2 * (slot * ROWS + rr)] = top;
              A.ml[2 * (slot * ROWS + rr) + 1] = L;
            }
          }
        }
      }
    }
  }
  if (!joined && tid == 0) A.join[blockIdx.x].last = -1;
}

// A row block's parts joined, in the order of its tokens: 256 threads over
// (part group, row, 8 dims).
template <int D, int ROWS>
__global__ __launch_bounds__(256) void attend_join(AttendArgs A) {
  __shared__ float s_m[ROWS], s_l[ROWS];
  __shared__ f32x4 s_acc[256][2];
  const AttendJoin J = const_load(A.join + blockIdx.x);
  if (J.last < 0) return;
  const int n = J.last - J.first + 1, tid = threadIdx.x, w = wave_id(), l = lane_id();
  auto slot = [&](int p) { return 2 * (J.first + p) + (p == 0); };
  for (int r = w; r < J.rows; r += 4) {
    float top = -INFINITY, L = 0;
    for (int p = l; p < n; p += 64) {
      const float* x = A.ml + 2 * (slot(p) * ROWS + r);
      const float m1 = fmaxf(top, x[0]), base = m1 == -INFINITY ? 0.f : m1;
      L = L * __builtin_amdgcn_exp2f(top - base) + x[1] * __builtin_amdgcn_exp2f(x[0] - base);
      top = m1;
    }
    const float all = wave_max(top), base = all == -INFINITY ? 0.f : all;
    L = wave_sum(L * __builtin_amdgcn_exp2f(top - base));
    if (l == 0) { s_m[r] = all; s_l[r] = L; }
  }
  __syncthreads();
  const int items = J.rows * (D / 8);
  int lg = 0;                                // items of a pass: the power of two above, to 256
  while ((1 << lg) < items && lg < 8) ++lg;
  const int groups = 256 >> lg, grp = tid >> lg;
  for (int i0 = 0; i0 < items; i0 += 1 << lg) {
    const int i = i0 + (tid & ((1 << lg) - 1));
    const int r = min(i, items - 1) / (D / 8), d = 8 * (i % (D / 8));
    const float top = s_m[r], base = top == -INFINITY ? 0.f : top;
    f32x4 o0 = {0, 0, 0, 0}, o1 = {0, 0, 0, 0};
#pragma unroll 4
    for (int p = grp; p < n; p += groups) {
      const float f = __builtin_amdgcn_exp2f(A.ml[2 * (slot(p) * ROWS + r)] - base);
      const float* x = A.part + ((int64_t)slot(p) * ROWS + r) * D + d;
      o0 += f * *(const f32x4*)x;
      o1 += f * *(const f32x4*)(x + 4);
    }
    __syncthreads();
    s_acc[tid][0] = o0;
    s_acc[tid][1] = o1;
    __syncthreads();
    if (grp == 0 && i < items) {
      for (int k = 1; k < groups; ++k) {
        o0 += s_acc[tid + (k << lg)][0];
        o1 += s_acc[tid + (k << lg)][1];
      }
      const float f = top == -INFINITY ? 0.f : 1.f / s_l[r];
      const u32x4 x = {pack_bf16(o0[0] * f, o0[1] * f), pack_bf16(o0[2] * f, o0[3] * f),
                       pack_bf16(o1[0] * f, o1[1] * f), pack_bf16(o1[2] * f, o1[3] * f)};
      const int row = J.row0 + r;
      *(u32x4*)(A.out + ((int64_t)(J.tok0 + row / A.G) * A.q_heads + J.head * A.G + row % A.G) * D +
                d) = x;
    }
  }
}

// The rows of a sequence that share a kv head, at most: the tile of 16, 32 or
// 64, as far as their sums fit the registers.
static int row_tiles(int64_t rows, int D, int dtype) {
  if (rows <= 16 || (D == 256 && dtype == CX_KV_E4M3)) return 1;
  return rows <= 32 || D == 256 || dtype == CX_KV_E4M3 ? 2 : 4;
}
static int workgroups(int nt) { return nt == 1 ? 512 : 256; }

struct AttendWork {
  size_t off_ml, off_part, total;
};
static AttendWork attend_workspace(int nt, int D) {
  const size_t W = workgroups(nt), rows = 16 * (size_t)nt;
  AttendWork x;
  x.off_ml = align_up(W * sizeof(AttendJoin), 256);
  x.off_part = x.off_ml + align_up(2 * W * rows * 8, 256);
  x.total = x.off_part + 2 * W * rows * D * 4;
  return x;
}

template <int D, int NT, bool F8>
static int launch_tile(const AttendArgs& A, hipStream_t s) {
  using Sh = AttendShape<D, NT, F8>;
  static std::once_flag once;
  hipError_t err = hipSuccess;
  std::call_once(once, [&] {
    err = hipFuncSetAttribute((const void*)attend_split<D, NT, F8>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, Sh::lds(CX_KV_MAX_BATCH));
  });
  if (err != hipSuccess) return (int)err;
  const dim3 grid((unsigned)workgroups(NT));
  timed_launch(CX_KERNEL_ATTEND, attend_split<D, NT, F8>, grid, dim3(ATT_WG),
               (uint32_t)Sh::lds(A.kv.B), s, A);
  timed_launch(CX_KERNEL_ATTEND_JOIN, attend_join<D, 16 * NT>, grid, dim3(256), 0, s, A);
  return (int)hipGetLastError();
}

template <int D>
static int launch_attend(const AttendArgs& A, int dtype, int nt, hipStream_t s) {
  const bool f8 = dtype == CX_KV_E4M3;
  if (nt == 1) return f8 ? launch_tile<D, 1, true>(A, s) : launch_tile<D, 1, false>(A, s);
  if constexpr (D < 256) {
    if (nt == 4) return launch_tile<D, 4, false>(A, s);
    if (f8) return launch_tile<D, 2, true>(A, s);
  }
  if (nt == 2 && !f8) return launch_tile<D, 2, false>(A, s);
  return (int)hipErrorInvalidValue;
}

}  // namespace cx

extern "C" {

size_t cx_paged_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                          int32_t max_new) {
  if (q_heads < 1 || kv_heads < 1 || head_dim < 1 || max_new < 1) return 256;
  const int64_t rows = (int64_t)(q_heads / kv_heads) * max_new;
  const size_t bf16 = cx::attend_workspace(cx::row_tiles(rows, head_dim, CX_KV_BF16), head_dim).total;
  const size_t e4m3 = cx::attend_workspace(cx::row_tiles(rows, head_dim, CX_KV_E4M3), head_dim).total;
  return bf16 > e4m3 ? bf16 : e4m3;
}

int cx_paged_attention_bf16(const cx_kv_batch* kv, const uint16_t* q, int64_t q_token,
                            int64_t q_head, int32_t q_heads, int32_t max_new, double scale,
                            int32_t window, double softcap, uint16_t* out, void* workspace,
                            size_t ws_bytes, void* stream) {
  cx::AttendArgs A;
  const int rc = cx::kv_args(kv, q_heads, &A.kv);
  if (rc != CX_OK) return rc;
  if (max_new < 1) return cx::api_fail(CX_EINVAL, "max_new must be >= 1");
  if (window < 0) return cx::api_fail(CX_EINVAL, "window must be >= 0");
  if (!(softcap >= 0)) return cx::api_fail(CX_EINVAL, "softcap must be >= 0");
  if (!(scale > 0)) return cx::api_fail(CX_EINVAL, "scale must be > 0");
  if (kv->T == 0 || kv->B == 0) return CX_OK;
  if (!q || !out || !workspace) return cx::api_fail(CX_EINVAL, "null pointer argument");
  if ((((uintptr_t)q | (uintptr_t)out) & 15) || ((q_token | q_head) & 7))
    return cx::api_fail(CX_EINVAL, "rows must be 16-byte aligned");
  if ((int64_t)kv->T * q_heads > INT32_MAX) return cx::api_fail(CX_EINVAL, "too many rows");
  const size_t need = cx_paged_attention_workspace_bytes(q_heads, kv->kv_heads, kv->head_dim,
                                                         max_new);
  if (ws_bytes < need)
    return cx::api_fail(CX_ENOSPACE, "workspace holds %zu bytes, needs %zu", ws_bytes, need);
  A.q = q; A.q_token = q_token; A.q_head = q_head;
  A.q_heads = q_heads; A.G = q_heads / kv->kv_heads;
  A.cap = softcap > 0;
  A.s1 = (float)((A.cap ? 2 * scale / softcap : scale) * 1.4426950408889634);
  A.s2 = (float)(softcap * 1.4426950408889634);
  A.window = window < INT32_MAX - cx::KV_MAX_NEW ? window : INT32_MAX - cx::KV_MAX_NEW;
  A.out = out;
  const int64_t rows = (int64_t)A.G * max_new;
  const int D = kv->head_dim, nt = cx::row_tiles(rows, D, kv->dtype);
  const cx::AttendWork lay = cx::attend_workspace(nt, D);
  A.join = (cx::AttendJoin*)workspace;
  A.ml = (float*)((char*)workspace + lay.off_ml);
  A.part = (float*)((char*)workspace + lay.off_part);
  const hipStream_t s = (hipStream_t)stream;
  const int e = D == 64    ? cx::launch_attend<64>(A, kv->dtype, nt, s)
                : D == 128 ? cx::launch_attend<128>(A, kv->dtype, nt, s)
                           : cx::launch_attend<256>(A, kv->dtype, nt, s);
  if (e != 0) return cx::api_fail(CX_EHIP, "attention launch: %s", hipGetErrorString((hipError_t)e));
  return CX_OK;
}

}  // extern "C"
