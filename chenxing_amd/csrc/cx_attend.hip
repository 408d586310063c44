// cx_attend.hip -- attention of the new tokens over the paged KV cache, for
// gfx950 (layout: cx_kv.hpp).
//
// out[t, h] = sum over the allowed positions s of softmax(scale q.k_s) v_s, in
// one pass over K and V with the running maximum m and sum l of the softmax's
// terms: a block of scores raises m to m', and l and the output so far are
// scaled by exp(m - m').  Two stream-ordered launches:
//
//   1. attend_split  independent waves, each with an equal share of all the
//                    batch's units (32 tokens of bf16, 64 of e4m3, for one kv
//                    head and row block); a row block that ends inside the share
//                    it began in is written out, the others' parts (m, l, sums)
//                    go to the workspace.
//   2. attend_join   one workgroup per split row block: its parts, in the order
//                    of its tokens.
//
// or, for short tables, attend_split<BLOCK> alone.
//
// Bound: HBM, every page read once a row block.  A row block is 16 NT rows of (new
// token, q head of the kv head's group); 16 rows of one unit are 24 MFMAs (head_dim
// 128) for 16 KB.  64 ragged requests of up to 8192 tokens, 8 kv heads of 128, 560
// MB: 95 us and 5 us of join, 5.9 TB/s in the first; 2 of 131072, 1018 MB: 164 and
// 6.5 us, 6.2 TB/s.  A prompt of 4096 tokens, 32 / 8 heads of 128: 452 us, 304
// TFLOP/s, bound by one wave a SIMD (products, softmax and loads of 48 rows one after
// the other) and by its reads: every wave's own, 2.6 GB past the L2s.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "cx_device.hpp"
#include "cx_internal.hpp"
#include "cx_kv.hpp"
#include "cx_lanes.hpp"
#include "cx_sampler.h"
#include "cx_share.hpp"
#include "cx_timing.hpp"

namespace cx {

constexpr int ATT_WG = 64 * ATT_WAVES;
// Terms are relative to a maximum that lags by up to this, in powers of 2: they
// reach 256 instead of 1, and the sums are rarely scaled.
constexpr float ATT_SLACK = 8.f;
// Caps up to this take tanh from the exponential alone, which is off by 6e-5 at most;
// larger ones a kernel of their own with tanh's series too (in the one kernel 118
// requests of 1008..2017 tokens, e4m3, 12 / 4 heads of 64, cap 30: 25.2 -> 25.8 us).
constexpr double ATT_CAP = 256;
constexpr float ATT_LOW = -3e38f;            // running maximum of a row that attends to something

struct AttendArgs {
  KvArgs kv;
  const uint16_t* q;
  int64_t q_token, q_head;
  int q_heads, G;             // G: q heads per kv head
  // score in powers of 2: s1 qk, or s2 tanh(s4 qk), where exp(2 s4 qk) = 2 ^ (s3 qk)
  float s1, s2, s3, s4;
  int cap;                    // the latter; 2: by more than ATT_CAP
  int window;                 // 0: none
  uint16_t* out;
  int workers;
  int* entries;               // number of entries of join
  AttendJoin* join;           // [workers]
  float* ml;                  // [2 workers, ROWS, 2]: a part's maxima and sums
  float* part;                // [2 workers, ROWS, D]
};

// 16 bytes of a page, read once: past the caches (131072 tokens 181 -> 161 us)
__device__ __forceinline__ u32x4 ld_page(const char* p) {
  return __builtin_nontemporal_load((const u32x4*)p);
}

// What the split of the work needs of the call.
__device__ __forceinline__ ShareBatch share_batch(const AttendArgs& A) {
  return {A.G, A.kv.heads, A.window, A.kv.n_pages ? A.kv.M << A.kv.logP : 0};
}

// The kernel's arguments in memory (its first, at the segment's start), for the
// parts of it that run once a piece: what they need is read there again, so the
// loop keeps its scalar registers.
__device__ __forceinline__ const AttendArgs& launch_args() {
  uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttendArgs*)(const CX_CONST AttendArgs*)p;
}

// Lane groups and registers change places.  Four registers: x[y] of group g
// becomes x[g] of group y.  Two: the registers of groups 0 1 2 3, [a0 a1 a2 a3]
// and [b0 b1 b2 b3], become [a0 a2 b0 b2] and [a1 a3 b1 b3].
__device__ __forceinline__ void regroup(uint32_t (&x)[4][2]) {
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    swap_halves(x[0][d], x[2][d]);
    swap_halves(x[1][d], x[3][d]);
    swap_rows(x[0][d], x[1][d]);
    swap_rows(x[2][d], x[3][d]);
  }
}
__device__ __forceinline__ void regroup(uint32_t (&x)[2][2]) {
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    swap_halves(x[0][d], x[1][d]);
    swap_rows(x[0][d], x[1][d]);
  }
}

template <int D, int NT, bool F8>
struct AttendShape {
  static constexpr int TOK = F8 ? 64 : 32;   // tokens of a unit
  static constexpr int ROWS = 16 * NT;
  using Line = AttendLine<TOK, NT>;
  using Seqs = AttendSeqs<CX_LDS uint64_t*, CX_LDS int*>;
  static constexpr int E = F8 ? 16 : 8;      // elements of a 16-byte chunk
  // A wave's scratch: its 16 rows, whole where the waves join their sums (BLOCK),
  // else a quarter of their dims (a large batch's lengths take the rest).
  static constexpr int PAD = D + 4, FIX = D / 4, FPAD = FIX + 4;   // floats of a row
  static constexpr int scratch(bool block) { return 16 * (block ? PAD : FPAD); }
  // waves per SIMD, as many as the registers hold
  static constexpr int WAVES = D * NT == 64                      ? (F8 ? 3 : 4)
                               : D * NT < 256 || (NT == 2 && !F8) ? 2
                                                                  : 1;
  // units of the longest context that BLOCK takes: a unit's time in a wave grows
  // with D NT (0.8 us at 128, 1.9 at 384; e4m3 twice as many tokens, 1.5 at 128)
  static constexpr int BLOCK_UNITS = 4096 / (D * NT < 128 ? 128 : D * NT) / (F8 ? 2 : 1);
  static constexpr int off_scale(bool block) { return ATT_WAVES * scratch(block) * 4; }
  static constexpr int off_seqs(bool block) {
    return off_scale(block) + (F8 ? ATT_WAVES * 512 : 0) + ATT_WAVES * 8;
  }
  static int lds_shares(int B, bool starts) { return off_seqs(false) + Seqs::bytes(B, starts); }
  static int lds_block() { return off_seqs(true); }
};

// The lengths are on the device, so each worker (a wave) finds its share itself:
// the units of every sequence summed up in LDS, and its range of the total.
//
//  * S^T = K Q^T, tile y being the unit's tokens 16 y .. 16 y + 15 of one page:
//    a lane holds scores of tokens 16 y + 4 g + j for its row (column), and the
//    softmax's statistics need two lane swaps.  O^T = V^T P^T wants a lane's terms
//    of the TOK / 4 tokens whose V it loaded as 16 contiguous bytes: lane groups
//    and tiles change places by lane swaps.  Nothing passes through LDS but the
//    e4m3 scales.
//  * The next unit's K is requested when this unit's scores are taken, its V
//    after this unit's products: half of a unit's 16 KB is always in flight, also
//    from one piece to the next.  The requests are unconditional (a branch on
//    them would make the waits of the loop drain them); after the last unit they
//    all name one place.
//  * Softmax terms enter the products as two bf16 parts (16 bits): one part's
//    rounding would add as much error as the result's own.
//
// BLOCK: short tables.  A workgroup takes a row block whole, each wave a quarter of
// its units, and the waves join through LDS: no share to find, no second launch.
// launch_tile says when.  WIDE: scores capped by more than ATT_CAP.
template <int D, int NT, bool F8, bool BLOCK, bool WIDE>
__global__ __launch_bounds__(ATT_WG, (AttendShape<D, NT, F8>::WAVES)) void attend_split(AttendArgs A) {
  using Sh = AttendShape<D, NT, F8>;
  constexpr int TOK = Sh::TOK, ROWS = Sh::ROWS, E = Sh::E, PAD = Sh::PAD;
  constexpr int KT = TOK / 16;               // score tiles of a unit, and its 16-token groups
  constexpr int KL = D / (4 * E);            // K loads of a tile
  constexpr int QL = D / 32;                 // Q loads of 16 rows
  constexpr int DT = D / 16, KH = TOK / 32;
  constexpr int BATCH = 64 / KT;             // units whose page ids a wave holds
  using Line = typename Sh::Line;
  constexpr uint32_t ALL = (1u << KT) - 1;
  extern __shared__ __align__(16) char lds[];
  __shared__ float s_ml[BLOCK ? ATT_WAVES * ROWS * 2 : 1];
  const KvArgs& C = A.kv;
  const int tid = threadIdx.x, w = wave_id(), l = lane_id(), g = l >> 4, c = l & 15;
  const int P = 1 << C.logP;
  CX_LDS float* const s_o = to_lds((float*)lds) + w * Sh::scratch(BLOCK);
  CX_LDS float* const s_scale = to_lds((float*)(lds + Sh::off_scale(BLOCK))) + w * 128;
  CX_LDS uint64_t* const s_pref = to_lds((uint64_t*)(lds + Sh::off_seqs(BLOCK)));
  CX_LDS uint64_t* const s_sum = s_pref - ATT_WAVES;
  CX_LDS int* const s_len = (CX_LDS int*)(s_pref + C.B + 1);
  const typename Sh::Seqs seqs = {s_pref, s_len, s_len + C.B, C.q_start != nullptr};

  // the line before each sequence, and its whole
  uint64_t line = 0;
  if constexpr (!BLOCK) {
    if (tid == 0) s_pref[0] = 0;
    seqs.read(C.kv_len, C.q_start, C.B, C.T, tid, ATT_WG);
    __syncthreads();
    for (int b0 = 0; b0 < C.B; b0 += ATT_WG) {
      const int b = b0 + tid;
      uint64_t x = 0;
      if (b < C.B) {
        const ShareBatch batch = share_batch(A);
        x = Line::length(batch, Line::seq(batch, seqs.first(b), seqs.end(b), s_len[b]));
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up(x, o);
        if (l >= o) x += y;
      }
      if (l == 63) s_sum[w] = x;
      __syncthreads();
      for (int k = 0; k < w; ++k) x += s_sum[k];
      if (b < C.B) s_pref[b + 1] = line + x;
      __syncthreads();
      line = s_pref[min(b0 + ATT_WG, C.B)];
    }
  }
  line = scalar64(line);
  ShareSplit split = share_split(line, gridDim.x * ATT_WAVES);
  split.per = scalar64(split.per);
  split.more = scalar64(split.more);
  const bool by_block = split.by_block;
  if (!BLOCK && blockIdx.x == 0 && tid == 0)
    *A.entries = by_block ? (int)line_blocks(line) : gridDim.x * ATT_WAVES;

  // tokens that attend to nothing
  for (int b = BLOCK ? C.B : blockIdx.x; b < C.B; b += gridDim.x)
    if (s_pref[b + 1] == s_pref[b]) {
      const int r0 = seqs.first(b);
      const int64_t n = (int64_t)(seqs.end(b) - r0) * A.q_heads * (D / 8);
      u32x4* o = (u32x4*)(A.out + (int64_t)r0 * A.q_heads * D);
      for (int64_t i = tid; i < n; i += ATT_WG) o[i] = u32x4{0, 0, 0, 0};
    }

  // this worker's share; neighbouring workers are on different CUs
  const unsigned worker = __builtin_amdgcn_readfirstlane(blockIdx.x + gridDim.x * w);
  if (!BLOCK && worker >= split.shares) {
    if (l == 0 && !by_block) A.join[worker].last = -1;
    return;
  }
  uint64_t u = share_begin(split, worker);
  const uint64_t end = u + split.per + (worker < split.more);
  int b = 0;
  for (int hi = BLOCK ? 0 : C.B - 1; b < hi;) {   // the last b with its units at or before u
    const int mid = (b + hi + 1) >> 1;
    if (line_units(s_pref[mid]) <= u) b = mid;
    else hi = mid - 1;
  }
  bool joined = false;
  // the piece that begins at u, and u past it; b: the sequence of the one before
  auto piece = [&]() {
    const auto& A = launch_args();
    while (line_units(s_pref[b + 1]) <= u) ++b;
    b = __builtin_amdgcn_readfirstlane(b);
    const ShareBatch batch = share_batch(A);
    const AttendSeq s = Line::seq(batch, seqs.first(b), seqs.end(b), s_len[b]);
    return Line::piece(batch, s, b, s_pref[b], split, worker, end, u,
                       [&](unsigned entry, const AttendJoin& j) {
                         joined |= j.last >= 0;
                         if (l == 0) A.join[entry] = j;
                       });
  };

  // ids of BATCH units of a piece from its k-th: lane KT k + group
  auto load_ids = [&](const AttendPiece& p, int k) {
    const auto& C = launch_args().kv;
    const int t16 = (p.unit + k) * KT + l;
    return t16 < (p.lim + 15) >> 4 ? C.table[p.b * C.ld_table + (t16 >> (C.logP - 4))] : -1;
  };
  u32x4 qr[NT][QL], kr[KT][KL], vr[DT];
  float ks = 1.f, vs = 1.f;                  // e4m3: the scales of the unit's token l
  auto load_q = [&](const AttendPiece& p) {
    const auto& A = launch_args();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = p.r0 + min(16 * nt + c, p.R - 1);
      const uint16_t* q = A.q + (p.tok0 + row / A.G) * A.q_token + (p.h * A.G + row % A.G) * A.q_head;
#pragma unroll
      for (int x = 0; x < QL; ++x)           // e4m3: the dims of a 16-element chunk in two
        qr[nt][x] = *(const u32x4*)(q + (F8 ? 64 * (x / 2) + 16 * g + 8 * (x % 2) : 32 * x + 8 * g));
    }
  };
  const int vgroup = F8 ? g : g >> 1;        // the group of this lane's tokens of V
  // place in the page of a unit's 16-token group
  auto place = [&](int unit, int group) { return ((unit * KT + group) << 4) & (P - 1); };
  uint32_t koff[KL];                         // this lane's place in K, from chunk 4 x
#pragma unroll
  for (int x = 0; x < KL; ++x) koff[x] = (uint32_t)(c + ((4 * x + g) << C.logP)) * 16;
  // the unit's pages: which are in the pool (bit y: 16-token group y), and where
  // this lane's V is
  uint32_t held = 0, hnext = 0;
  const char* vnext = nullptr;
  auto load_k = [&](int ids, int k, int unit, int h, bool live) {
    const char* const head0 = C.pages + (int64_t)h * C.head_bytes;
    const uint32_t on = live ? ~0u : 0;
    hnext = 0;
#pragma unroll
    for (int y = 0; y < KT; ++y) {
      const int id = lane_read(ids, k * KT + y);
      const bool in = (unsigned)id < (unsigned)C.n_pages;
      hnext |= (uint32_t)in << y;
      const char* p = head0 + (in ? id : 0) * C.page_stride + place(unit, y) * 16;
#pragma unroll
      for (int x = 0; x < KL; ++x)
        kr[y][x] = ld_page(p + (koff[x] & on));
    }
    const int id = __shfl(ids, k * KT + vgroup);
    const char* p = head0 + ((unsigned)id < (unsigned)C.n_pages ? id : 0) * C.page_stride;
    vnext = p + (live ? v_chunk<E, D>(c, place(unit, vgroup) + (F8 ? 0 : 8 * (g & 1)), C.logP) : 0);
    if (F8) {
      const float* sc = (const float*)(p + k_scale<D>(place(unit, g) + c, C.logP));
      ks = sc[0];
      vs = sc[P];
    }
    __builtin_amdgcn_sched_barrier(0);       // the loop's waits count on this order
  };
  auto load_v = [&]() {
    held = hnext;
#pragma unroll
    for (int n = 0; n < DT; ++n) vr[n] = ld_page(vnext + 256 * n);
    __builtin_amdgcn_sched_barrier(0);
  };

  f32x4 acc[NT][DT];
  float m[NT], sum[NT];
  int hi[NT], lo[NT];                        // the row attends to lo < t <= hi
  int pmin = 0, pmax = 0;                    // positions of the piece's first and last row
  bool again = false;
  auto begin = [&](const AttendPiece& p) {
    const auto& A = launch_args();
    pmin = p.lowest + p.r0 / A.G;
    pmax = p.lowest + (p.r0 + p.R - 1) / A.G;
    again = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int pos = p.lowest + (p.r0 + min(16 * nt + c, p.R - 1)) / A.G;
      hi[nt] = min(pos, p.lim - 1);
      lo[nt] = A.window ? pos - A.window : -1;
      m[nt] = -INFINITY;
      sum[nt] = 0;
#pragma unroll
      for (int n = 0; n < DT; ++n) acc[nt][n] = f32x4{0, 0, 0, 0};
    }
  };

  AttendPiece cur, nxt;
  int ids = -1, idn = -1, idq = -1;
  bool last = true;
  // the piece after the current one, if the share holds one
  auto follow = [&]() {
    last = true;
    if (u < end) {
      nxt = piece();
      last = nxt.cnt == 0;
    }
    if (last) nxt = cur;
    idq = load_ids(nxt, 0);
  };
  int rb = BLOCK ? (int)(blockIdx.x / (unsigned)C.heads) : 0, blocks = 1;
  do {
  if constexpr (BLOCK) {
    // this wave's quarter of row block rb of a sequence and kv head
    const auto& A = launch_args();
    const int sb = blockIdx.y;
    const int2 rows = kv_rows(A.kv, sb);
    const AttendSeq s = Line::seq(share_batch(A), rows.x, rows.y, A.kv.kv_len[sb]);
    blocks = Line::row_blocks(share_batch(A), s);
    if (rb >= blocks) return;
    cur.b = sb;
    cur.h = (int)(blockIdx.x % (unsigned)A.kv.heads);
    cur.tok0 = s.tok0;
    cur.r0 = rb * ROWS;
    cur.R = min(ROWS, s.q * A.G - cur.r0);
    cur.lowest = s.len - s.q;
    cur.lim = s.lim;
    // the units of its rows' windows, up to its last row
    const int low = cur.lowest + cur.r0 / A.G, high = cur.lowest + (cur.r0 + cur.R - 1) / A.G;
    const int first = A.window ? max(low - A.window + 1, 0) / TOK : 0;
    const int n = max((min(s.lim, high + 1) + TOK - 1) / TOK - first, 0);
    const int quarter = (n + ATT_WAVES - 1) / ATT_WAVES;
    cur.unit = __builtin_amdgcn_readfirstlane(first + w * quarter);
    cur.cnt = __builtin_amdgcn_readfirstlane(min(max(n - w * quarter, 0), quarter));
    cur.slot = -1;
  } else {
    cur = piece();
    if (cur.cnt == 0) {
      if (l == 0 && !by_block) A.join[worker].last = -1;
      return;
    }
  }
  if (!BLOCK || cur.cnt > 0) {
    load_q(cur);
    ids = load_ids(cur, 0);
    idn = load_ids(cur, BATCH);
    load_k(ids, 0, cur.unit, cur.h, true);
    load_v();
    if (!BLOCK) follow();
  }
  begin(cur);
  if (!BLOCK || cur.cnt > 0) for (int i = 0;;) {
    const int unit = cur.unit + i, t0 = unit * TOK;
    // scores: tile y's row 4 g + j is token t0 + 16 y + 4 g + j
    f32x4 v[NT][KT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int y = 0; y < KT; ++y) v[nt][y] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int x = 0; x < QL; ++x)
#pragma unroll
      for (int y = 0; y < KT; ++y) {
        const bf16x8 ka = F8 ? e4m3x8(kr[y][x / 2][2 * (x % 2)], kr[y][x / 2][2 * (x % 2) + 1])
                             : __builtin_bit_cast(bf16x8, kr[y][x]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          v[nt][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              ka, __builtin_bit_cast(bf16x8, qr[nt][x]), v[nt][y], 0, 0, 0);
      }
    f32x4 vscale[F8 ? KT : 1];
    if (F8) {
      s_scale[l] = ks;                       // the wave's own words: no barrier
      s_scale[64 + l] = vs;
      asm volatile("" ::: "memory");
#pragma unroll
      for (int y = 0; y < KT; ++y) {
        const f32x4 kscale = *(const CX_LDS f32x4*)(s_scale + 16 * y + 4 * g);
        vscale[y] = *(const CX_LDS f32x4*)(s_scale + 64 + 16 * y + 4 * g);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) v[nt][y] *= kscale;
      }
    }
    // K and Q are used up: those of the next unit, in this piece or the next
    const bool turn = i + 1 == cur.cnt;
    int k = (i + 1) % BATCH;
    if (turn) {
      if (!BLOCK) {
        ids = idq;
        load_q(nxt);
      }
      k = 0;
    } else if (k == 0) {
      ids = idn;
      idn = load_ids(cur, i + 1 + BATCH);
    }
    load_k(ids, k, turn && !BLOCK ? nxt.unit : unit + 1, turn && !BLOCK ? nxt.h : cur.h, !(turn && last));

    // scores in powers of 2 are to2 * v
    const float to2 = WIDE || A.cap ? 1.f : A.s1;
    if constexpr (WIDE) {
      // that is off by 2^-23 of the cap, whatever the score: too much of a large one.
      // Below z = 1/16 the series, to z^5
      const auto& A = launch_args();
      const float s1 = A.s1, s2 = A.s2, s3 = A.s3, s4 = A.s4;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int y = 0; y < KT; ++y)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = v[nt][y][j], z = s4 * x, zz = z * z, sx = s1 * x;
            const float far = fmaf(-2.f * s2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s3 * x) + 1.f), s2);
            v[nt][y][j] = zz < 1.f / 256.f ? fmaf(sx * zz, fmaf(zz, 2.f / 15.f, -1.f / 3.f), sx) : far;
          }
    } else if (A.cap) {                      // tanh(z) = 1 - 2 / (exp(2 z) + 1)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int y = 0; y < KT; ++y)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[nt][y][j] = fmaf(-2.f * A.s2,
                               __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(A.s3 * v[nt][y][j]) + 1.f),
                               A.s2);
    }
    // a row's running maximum is at least ATT_LOW once it has attended to a
    // token, whatever its score: -inf says that it has not
    float low[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) low[nt] = ATT_LOW;
    // a unit is open where all its tokens are held, at or before the first row
    // and inside the last row's window
    const uint32_t here = held;
    const bool masked = t0 + TOK - 1 > pmin || t0 + TOK > cur.lim ||
                        (A.window && t0 <= pmax - A.window) || here != ALL;
    if (masked) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        bool some = false;
#pragma unroll
        for (int y = 0; y < KT; ++y) {
          const int ty = t0 + 16 * y;
          const bool in = here >> y & 1;
          some |= in && max(ty, lo[nt] + 1) <= min(ty + 15, hi[nt]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int t = ty + 4 * g + j;
            v[nt][y][j] = in && t <= hi[nt] && t > lo[nt] ? v[nt][y][j] : -INFINITY;
          }
        }
        low[nt] = some ? ATT_LOW : -INFINITY;
      }
    }
    float alpha[NT];
    bool moved = false;
    u32x4 ph[NT][KH], pl[NT][KH];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top = -INFINITY;
#pragma unroll
      for (int y = 0; y < KT; ++y)
        top = fmaxf(top, fmaxf(fmaxf(v[nt][y][0], v[nt][y][1]), fmaxf(v[nt][y][2], v[nt][y][3])));
      const float m1 = fmaxf(low[nt], to2 * groups_max(top));
      const bool up = m1 > m[nt] + ATT_SLACK;
      const float base = up ? m1 : m[nt] == -INFINITY ? 0.f : m[nt];
      alpha[nt] = up ? __builtin_amdgcn_exp2f(m[nt] - m1) : 1.f;
      moved |= up;
      m[nt] = up ? m1 : m[nt];
      uint32_t th[KT][2], tl[KT][2];
      float add = 0;
#pragma unroll
      for (int y = 0; y < KT; ++y) {
        f32x4 p;
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(to2, v[nt][y][j], -base));
        add += (p[0] + p[1]) + (p[2] + p[3]);
        if (F8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = v[nt][y][j] == -INFINITY ? 0.f : p[j] * vscale[y][j];
        }
        // the terms as two bf16 parts each, 16 bits of them.  The first is cut
        // off and the second kept above 0, so an infinite value keeps its sign
        // in both products
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const float p0 = p[2 * d], p1 = p[2 * d + 1];
          const uint32_t x0 = __float_as_uint(p0), x1 = __float_as_uint(p1);
          th[y][d] = __builtin_amdgcn_perm(x1, x0, 0x07060302);
          tl[y][d] = pack_bf16(fmaxf(p0 - __uint_as_float(x0 & 0xFFFF0000u), p0 * 0x1p-24f),
                               fmaxf(p1 - __uint_as_float(x1 & 0xFFFF0000u), p1 * 0x1p-24f));
        }
      }
      sum[nt] = fmaf(sum[nt], alpha[nt], add);
      // lane group G gets the terms of the tokens whose V it holds
      regroup(th);
      regroup(tl);
#pragma unroll
      for (int x = 0; x < KH; ++x) {
        ph[nt][x] = u32x4{th[2 * x][0], th[2 * x][1], th[2 * x + 1][0], th[2 * x + 1][1]};
        pl[nt][x] = u32x4{tl[2 * x][0], tl[2 * x][1], tl[2 * x + 1][0], tl[2 * x + 1][1]};
      }
    }
    if (__any(moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int n = 0; n < DT; ++n) acc[nt][n] *= alpha[nt];
    }
    if (masked) {
      // V of tokens that no row attends to counts as zeros, whatever is there
      // (a product with a zero term would not)
      const bool vheld = here >> vgroup & 1;
      const int tv = t0 + (TOK / 4) * g;     // the first of this lane's tokens of V
      const int from = A.window ? pmin - A.window : -1, to = min(pmax, cur.lim - 1);
      uint32_t keep[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        keep[d] = 0;
#pragma unroll
        for (int e = 0; e < E / 4; ++e) {
          const int t = tv + E / 4 * d + e;
          keep[d] |= vheld && t > from && t <= to ? (F8 ? 0xFFu << 8 * e : 0xFFFFu << 16 * e) : 0;
        }
      }
#pragma unroll
      for (int n = 0; n < DT; ++n)
#pragma unroll
        for (int d = 0; d < 4; ++d) vr[n][d] &= keep[d];
      if (pmin != pmax) {
        // nor may NaN or infinity reach the rows that do not attend to it: left
        // out here, added row by row at the piece's end
        uint32_t bad = 0;
#pragma unroll
        for (int n = 0; n < DT; ++n)
#pragma unroll
          for (int d = 0; d < 4; ++d) bad |= nonfinite_sign<F8>(vr[n][d]);
        if (__any((bad & (F8 ? 0x80808080u : 0x80008000u)) != 0)) {
          again = true;
#pragma unroll
          for (int n = 0; n < DT; ++n)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              // hidden: the sums above are not kept for this
              asm volatile("" : "+v"(vr[n][d]));
              vr[n][d] &= finite_mask<F8>(vr[n][d]);
            }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < DT; ++n)
#pragma unroll
      for (int x = 0; x < KH; ++x) {
        const bf16x8 va = F8 ? e4m3x8(vr[n][2 * x], vr[n][2 * x + 1])
                             : __builtin_bit_cast(bf16x8, vr[n]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          acc[nt][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              va, __builtin_bit_cast(bf16x8, ph[nt][x]), acc[nt][n], 0, 0, 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          acc[nt][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              va, __builtin_bit_cast(bf16x8, pl[nt][x]), acc[nt][n], 0, 0, 0);
      }
    load_v();
    if (!turn) {
      ++i;
      continue;
    }

    // the piece ends
    const auto& A = launch_args();
    const auto& C = A.kv;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (again) {
        // each row's own NaN and infinite values (their terms' size does not
        // matter), token by token, FIX dims of all 16 rows at a time
        constexpr int FIX = BLOCK ? 64 : Sh::FIX, FPAD = FIX + 4, NQ = FIX / 16;
        const int fd = l % FIX;
#pragma unroll
        for (int x = 0; x < D / FIX; ++x) {
#pragma unroll
          for (int n = 0; n < NQ; ++n)
            *(CX_LDS f32x4*)(s_o + c * FPAD + 16 * n + 4 * g) = acc[nt][NQ * x + n];
          asm volatile("" ::: "memory");
          for (int t = cur.unit * TOK; t < (cur.unit + cur.cnt) * TOK && t < cur.lim; ++t) {
            const int id = C.table[cur.b * C.ld_table + (t >> C.logP)], o = t & (P - 1);
            if ((unsigned)id >= (unsigned)C.n_pages) continue;
            const char* p = C.pages + id * C.page_stride + (int64_t)cur.h * C.head_bytes +
                            v_chunk<E, D>(FIX * x + fd, o, C.logP) + o % E * (16 / E);
            const float v = F8 ? e4m3_value(*(const uint8_t*)p) : bf16_lo(*(const uint16_t*)p);
            if (fabsf(v) < INFINITY) continue;
#pragma unroll 1
            for (int r = l / FIX; r < 16; r += 64 / FIX) {
              const int at = cur.lowest + (cur.r0 + min(16 * nt + r, cur.R - 1)) / A.G;
              if (t <= at && !(A.window && t <= at - A.window)) s_o[r * FPAD + fd] += v;
            }
          }
          asm volatile("" ::: "memory");
#pragma unroll
          for (int n = 0; n < NQ; ++n)
            acc[nt][NQ * x + n] = *(const CX_LDS f32x4*)(s_o + c * FPAD + 16 * n + 4 * g);
        }
      }
      const int r = 16 * nt + c;
      const float L = groups_sum(sum[nt]);
      sum[nt] = L;
      if (!BLOCK && r < cur.R) {
        if (cur.slot < 0) {
          const float f = m[nt] == -INFINITY ? 0.f : 1.f / L;
          const int row = cur.r0 + r;
          uint16_t* o = A.out + ((int64_t)(cur.tok0 + row / A.G) * A.q_heads + cur.h * A.G +
                                 row % A.G) * D + 4 * g;
#pragma unroll
          for (int n = 0; n < DT; ++n)
            *(u32x2*)(o + 16 * n) = u32x2{pack_bf16(acc[nt][n][0] * f, acc[nt][n][1] * f),
                                          pack_bf16(acc[nt][n][2] * f, acc[nt][n][3] * f)};
        } else {
          float* o = A.part + ((int64_t)cur.slot * ROWS + r) * D + 4 * g;
#pragma unroll
          for (int n = 0; n < DT; ++n) *(f32x4*)(o + 16 * n) = acc[nt][n];
          if (g == 0) {
            A.ml[2 * ((int64_t)cur.slot * ROWS + r)] = m[nt];
            A.ml[2 * ((int64_t)cur.slot * ROWS + r) + 1] = L;
          }
        }
      }
    }
    if (BLOCK || last) break;
    cur = nxt;
    idn = load_ids(cur, BATCH);
    follow();
    begin(cur);
    i = 0;
  }
  if constexpr (BLOCK) {
    // the waves' sums, in their order
    const auto& A = launch_args();
    CX_LDS float* const s_all = to_lds((float*)lds);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (g == 0) {
        s_ml[2 * (w * ROWS + 16 * nt + c)] = m[nt];
        s_ml[2 * (w * ROWS + 16 * nt + c) + 1] = sum[nt];
      }
      if (nt > 0) __syncthreads();
#pragma unroll
      for (int n = 0; n < DT; ++n) *(CX_LDS f32x4*)(s_o + c * PAD + 16 * n + 4 * g) = acc[nt][n];
      __syncthreads();
      for (int i = tid; i < 16 * (D / 8); i += ATT_WG) {
        const int r = i / (D / 8), d = 8 * (i % (D / 8)), rr = 16 * nt + r;
        if (rr >= cur.R) continue;
        float top = -INFINITY, L = 0;
#pragma unroll
        for (int k = 0; k < ATT_WAVES; ++k) top = fmaxf(top, s_ml[2 * (k * ROWS + rr)]);
        const float base = top == -INFINITY ? 0.f : top;
        f32x4 o0 = {0, 0, 0, 0}, o1 = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < ATT_WAVES; ++k) {
          const float f = __builtin_amdgcn_exp2f(s_ml[2 * (k * ROWS + rr)] - base);
          const CX_LDS float* o = s_all + (k * 16 + r) * PAD + d;
          L = fmaf(f, s_ml[2 * (k * ROWS + rr) + 1], L);
          o0 += f * *(const CX_LDS f32x4*)o;
          o1 += f * *(const CX_LDS f32x4*)(o + 4);
        }
        const float f = top == -INFINITY ? 0.f : 1.f / L;
        const u32x4 x = {pack_bf16(o0[0] * f, o0[1] * f), pack_bf16(o0[2] * f, o0[3] * f),
                         pack_bf16(o1[0] * f, o1[1] * f), pack_bf16(o1[2] * f, o1[3] * f)};
        const int row = cur.r0 + rr;
        *(u32x4*)(A.out + ((int64_t)(cur.tok0 + row / A.G) * A.q_heads + cur.h * A.G + row % A.G) * D +
                  d) = x;
      }
    }
    rb += (int)(gridDim.x / (unsigned)A.kv.heads);
    if (rb < blocks) __syncthreads();        // the sums are read
  }
  } while (BLOCK && rb < blocks);
  if (!BLOCK && !joined && l == 0 && !by_block) A.join[worker].last = -1;
}

// The parts of rows joined, in an order that goes by their number alone.
struct JoinSum {
  float top, L;
  f32x4 o0, o1;
};
// Adds parts p, p + step, .. of row r at dims d .. d + 7, AHEAD of them together.
template <int D, int ROWS, int AHEAD>
__device__ __forceinline__ JoinSum join_parts(const AttendArgs& A, const AttendJoin& J, int n, int r,
                                              int d, int p, int step) {
  JoinSum S = {-INFINITY, 0.f, {0, 0, 0, 0}, {0, 0, 0, 0}};
  for (int p0 = p; p0 < n; p0 += AHEAD * step) {
    float m[AHEAD], s[AHEAD];
    f32x4 x0[AHEAD], x1[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {        // past the last: the last again, not added
      const int q = min(p0 + k * step, n - 1);
      const int64_t at = (int64_t)(2 * (J.first + q) + (q == 0)) * ROWS + r;
      const float2 ml = *(const float2*)(A.ml + 2 * at);
      m[k] = p0 + k * step < n ? ml.x : -INFINITY;
      s[k] = ml.y;
      x0[k] = *(const f32x4*)(A.part + at * D + d);
      x1[k] = *(const f32x4*)(A.part + at * D + d + 4);
    }
    float t = S.top;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) t = fmaxf(t, m[k]);
    const float base = t == -INFINITY ? 0.f : t, f0 = __builtin_amdgcn_exp2f(S.top - base);
    S.top = t;
    S.L *= f0;
    S.o0 *= f0;
    S.o1 *= f0;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (p0 + k * step >= n) continue;
      const float f = __builtin_amdgcn_exp2f(m[k] - base);
      S.L = fmaf(f, s[k], S.L);
      S.o0 += f * x0[k];
      S.o1 += f * x1[k];
    }
  }
  return S;
}
__device__ __forceinline__ void join_add(JoinSum& a, const JoinSum& b) {
  const float t = fmaxf(a.top, b.top), base = t == -INFINITY ? 0.f : t;
  const float fa = __builtin_amdgcn_exp2f(a.top - base), fb = __builtin_amdgcn_exp2f(b.top - base);
  a.top = t;
  a.L = fa * a.L + fb * b.L;
  a.o0 = fa * a.o0 + fb * b.o0;
  a.o1 = fa * a.o1 + fb * b.o1;
}
template <int D>
__device__ __forceinline__ void join_out(const AttendArgs& A, const AttendJoin& J, const JoinSum& S,
                                         int r, int d) {
  const float f = S.top == -INFINITY ? 0.f : 1.f / S.L;
  const u32x4 x = {pack_bf16(S.o0[0] * f, S.o0[1] * f), pack_bf16(S.o0[2] * f, S.o0[3] * f),
                   pack_bf16(S.o1[0] * f, S.o1[1] * f), pack_bf16(S.o1[2] * f, S.o1[3] * f)};
  const int row = J.row0 + r;
  *(u32x4*)(A.out + ((int64_t)(J.tok0 + row / A.G) * A.q_heads + J.head * A.G + row % A.G) * D + d) = x;
}

// An entry in range: those of a call are, unless its lengths change while it runs,
// when some are not written.
template <int ROWS>
__device__ __forceinline__ bool join_holds(const AttendArgs& A, const AttendJoin& J) {
  return J.first >= 0 && J.last >= J.first && J.last < A.workers && J.rows <= ROWS && J.row0 >= 0 &&
         (unsigned)J.head < (unsigned)A.kv.heads && J.tok0 >= 0 &&
         (int64_t)J.row0 + J.rows <= (int64_t)(A.kv.T - J.tok0) * A.G;
}

// Few row blocks, so perhaps of many parts: workgroup (entry, row), the row's
// parts over all its lane groups of D / 8 lanes.
template <int D, int ROWS>
__global__ __launch_bounds__(256) void attend_join_row(AttendArgs A) {
  constexpr int LANES = D / 8, GROUPS = 256 / LANES;
  __shared__ JoinSum s_sum[GROUPS][LANES];
  const int count = const_load(A.entries);
  const AttendJoin J = const_load(A.join + blockIdx.x);
  const int r = blockIdx.y;
  if ((int)blockIdx.x >= count || r >= J.rows || !join_holds<ROWS>(A, J)) return;
  const int n = J.last - J.first + 1, grp = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  JoinSum S = join_parts<D, ROWS, 8>(A, J, n, r, 8 * lane, grp, GROUPS);
  if (grp > 0) s_sum[grp][lane] = S;
  __syncthreads();
  if (grp > 0) return;
  for (int k = 1; k < min(n, GROUPS); ++k) join_add(S, s_sum[k][lane]);
  join_out<D>(A, J, S, r, 8 * lane);
}

// Many row blocks: workgroup (entry, 16 or 4 rows).  Each lane group of D / 8 lanes
// takes a row with all its parts; where there are few rows and many parts, each
// wave takes one with its groups' shares of them (32 verify rounds, 36 rows: 6 us
// with groups, 9 with waves; 11 requests of up to 7400 tokens, 8 rows: 20 and 9 us).
template <int D, int ROWS>
__global__ __launch_bounds__(256) void attend_join_block(AttendArgs A) {
  constexpr int LANES = D / 8, GROUPS = 256 / LANES;
  const int count = const_load(A.entries);
  const AttendJoin J = const_load(A.join + blockIdx.x);
  if ((int)blockIdx.x >= count || !join_holds<ROWS>(A, J)) return;
  const int n = J.last - J.first + 1, d = 8 * (threadIdx.x % LANES);
  const int per = ROWS / gridDim.y, r0 = per * blockIdx.y, end = min(J.rows, r0 + per);
  if (n <= 8 || end - r0 > 8) {
    for (int r = r0 + threadIdx.x / LANES; r < end; r += GROUPS)
      join_out<D>(A, J, join_parts<D, ROWS, 4>(A, J, n, r, d, 0, 1), r, d);
    return;
  }
  const int l = lane_id();
  for (int r = r0 + wave_id(); r < end; r += 4) {
    JoinSum S = join_parts<D, ROWS, 8>(A, J, n, r, d, l / LANES, GROUPS / 4);
#pragma unroll
    for (int x = LANES; x < 64; x <<= 1) {
      JoinSum T;
      T.top = __shfl_xor(S.top, x);
      T.L = __shfl_xor(S.L, x);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        T.o0[k] = __shfl_xor(S.o0[k], x);
        T.o1[k] = __shfl_xor(S.o1[k], x);
      }
      join_add(S, T);                        // a sum of two: in either order the same
    }
    if (l < LANES) join_out<D>(A, J, S, r, d);
  }
}

// The tile, in 16 rows, for at most that many rows of a sequence that share a kv
// head: as few row blocks as the registers allow, of one size.
static int row_tiles(int64_t rows, int most) {
  const int64_t tiles = (rows + 15) / 16, blocks = (tiles + most - 1) / most;
  return (int)((tiles + blocks - 1) / blocks);
}
// Four tiles of heads of 64 leave one wave a SIMD, three two: where four do not hold
// all rows, three are faster or no slower (28 / 4 heads, prompts of 1024 and 4096
// tokens: 29 and 228 us, with four 39 and 262; 32 new tokens of 2048, one request: 19
// and 20; 64 requests of 20 new of 2048, 16 / 2 heads: 58 and 68).  But where three
// fill at least an eighth more rows than four, calls that have many units are faster
// with four (64 requests of 32 new tokens of 512, 32 / 8 heads: 47 us, with three 61;
// of 8192: 506 and 557; 16 requests of 64 new of 512: 30 and 26), if all sequences have
// as many rows (42 of 16206 tokens, 1 to 15 new, 24 / 3 heads: 224 and 180).
// head_units: the units that one row block of each sequence and kv head may have, all
// together, or 0.
constexpr int64_t ATT_FOUR_UNITS = 24576;
static int attend_tiles(int64_t rows, int D, int dtype, int64_t head_units) {
  if (D == 256) return row_tiles(rows, 1);
  if (dtype == CX_KV_E4M3) return row_tiles(rows, 2);
  if (D == 128) return row_tiles(rows, 3);
  if (rows <= 64) return row_tiles(rows, 4);
  const int nt = row_tiles(rows, 4);
  const int64_t b3 = (rows + 47) / 48, b4 = (rows + 16 * nt - 1) / (16 * nt);
  return 8 * 48 * b3 >= 9 * 16 * nt * b4 && head_units * b3 >= ATT_FOUR_UNITS ? nt
                                                                            : row_tiles(rows, 3);
}
// Workers: as many waves as the chip's 256 CUs hold of the tile's kernel.
static int workgroups(int nt, int D, int dtype) {
  const bool f8 = dtype == CX_KV_E4M3;
  return 256 * (D * nt == 64 ? (f8 ? 3 : 4) : D * nt < 256 || (nt == 2 && !f8) ? 2 : 1);
}

// The join: a workgroup a row where a row block may have more than join_parts parts,
// as many as its share of the workers or as the longest context's units make; else a
// wave a row, unless that is many workgroups (4 rounds of 13 rows over 8014 tokens,
// heads of 64: 6 us, 16 rows a workgroup 15).  A wave adds 512 / D parts of 8 dims a
// lane together; a workgroup a row as many for each of its four waves, but then joins
// 2048 / D sums one after the other (a workgroup a row and a wave a row, heads of 64: 2
// new tokens of 30000, one request of 4 kv heads, 9 and 14 us; 32 of 3000: 12 and 5; 8
// requests of 2500: 9 and 5; of 128: one of 8000, 8 kv heads, 5 and 8; 12 new of 3000:
// 6.5 and 5.3; of 256: one of 3000, one kv head: 4.4 and 6.1).
constexpr int join_parts(int D) { return D == 64 ? 192 : D == 128 ? 64 : 20; }
constexpr int64_t ATT_JOIN_ROWS = 8192;

struct AttendWork {
  size_t off_join, off_ml, off_part, total;
};
static AttendWork attend_workspace(int nt, int D, int dtype) {
  const size_t W = ATT_WAVES * (size_t)workgroups(nt, D, dtype), rows = 16 * (size_t)nt;
  AttendWork x;
  x.off_join = 256;
  x.off_ml = x.off_join + align_up(W * sizeof(AttendJoin), 256);
  x.off_part = x.off_ml + align_up(2 * W * rows * 8, 256);
  x.total = x.off_part + 2 * W * rows * D * 4;
  return x;
}

template <int D, int NT, bool F8>
static int launch_tile(AttendArgs A, int64_t max_new, hipStream_t s) {
  using Sh = AttendShape<D, NT, F8>;
  constexpr int ROWS = Sh::ROWS;
  const unsigned grid = 256 * Sh::WAVES;
  A.workers = (int)grid * ATT_WAVES;
  const int64_t span = A.window ? std::min<int64_t>(A.window + max_new, (int64_t)A.kv.M << A.kv.logP)
                                : (int64_t)A.kv.M << A.kv.logP;
  const int64_t tiles = ((int64_t)A.G * max_new + ROWS - 1) / ROWS;
  const int64_t blocks = A.kv.heads * std::max(A.kv.B * tiles, (int64_t)A.kv.T * A.G / ROWS);
  // BLOCK, where a wave's quarter of the longest context takes less than finding
  // shares and joining them, unless workgroups would queue three deep (heads of 128,
  // 8 kv heads, 1 and 32 requests, BLOCK and shares: 256 tokens 5.7 and 9.4, 6.3 and
  // 13.2 us; 1024 tokens 10.4 and 11.2, 21 and 31; 2048 tokens 17 and 12, 43 and 52.
  // 256 requests of 64 tokens: 21 and 17).  Row blocks that fill half the chip gain
  // from twice the length; max_new is a hint only, so they are counted by T, too.
  const int most = Sh::BLOCK_UNITS * (2 * blocks >= grid ? 2 : 1);
  using Kernel = void (*)(AttendArgs);
  static const Kernel in_block[2] = {attend_split<D, NT, F8, true, false>,
                                     attend_split<D, NT, F8, true, true>},
                      in_shares[2] = {attend_split<D, NT, F8, false, false>,
                                      attend_split<D, NT, F8, false, true>};
  static LdsLimit limit_block[2], limit[2];
  const int wide = A.cap > 1;
  if (blocks <= 2 * grid && span <= most * Sh::TOK) {
    if (int e = limit_block[wide].raise((const void*)in_block[wide], Sh::lds_block())) return e;
    timed_launch(CX_KERNEL_ATTEND, in_block[wide],
                 dim3((unsigned)(A.kv.heads * tiles), A.kv.B), dim3(ATT_WG), (uint32_t)Sh::lds_block(), s,
                 A);
    return (int)hipGetLastError();
  }
  if (int e = limit[wide].raise((const void*)in_shares[wide],
                                Sh::lds_shares(CX_KV_MAX_BATCH, true)))
    return e;
  timed_launch(CX_KERNEL_ATTEND, in_shares[wide], dim3(grid), dim3(ATT_WG),
               (uint32_t)Sh::lds_shares(A.kv.B, A.kv.q_start != nullptr), s, A);
  // row blocks at most: every sequence's last one may hold fewer rows
  const int64_t entries = std::min<int64_t>(A.kv.heads * ((int64_t)A.kv.T * A.G / ROWS + A.kv.B),
                                            grid * ATT_WAVES);
  const int64_t parts = std::min<int64_t>(
      grid * ATT_WAVES / entries, ((span + Sh::TOK - 1) / Sh::TOK + Sh::Line::PIECE) / ATT_SHARE + 1);
  if (parts > join_parts(D))
    timed_launch(CX_KERNEL_ATTEND_JOIN, attend_join_row<D, ROWS>, dim3((unsigned)entries, ROWS),
                 dim3(256), 0, s, A);
  else
    timed_launch(CX_KERNEL_ATTEND_JOIN, attend_join_block<D, ROWS>,
                 dim3((unsigned)entries, entries * ROWS <= ATT_JOIN_ROWS ? ROWS / 4 : NT), dim3(256), 0, s,
                 A);
  return (int)hipGetLastError();
}

template <int D>
static int launch_attend(const AttendArgs& A, int dtype, int nt, int64_t max_new, hipStream_t s) {
  const bool f8 = dtype == CX_KV_E4M3;
  if (nt == 1) return f8 ? launch_tile<D, 1, true>(A, max_new, s) : launch_tile<D, 1, false>(A, max_new, s);
  if constexpr (D < 256) {
    if (nt == 2) return f8 ? launch_tile<D, 2, true>(A, max_new, s) : launch_tile<D, 2, false>(A, max_new, s);
    if (nt == 3 && !f8) return launch_tile<D, 3, false>(A, max_new, s);
  }
  if constexpr (D == 64)
    if (nt == 4 && !f8) return launch_tile<D, 4, false>(A, max_new, s);
  return (int)hipErrorInvalidValue;
}

}  // namespace cx

extern "C" {

size_t cx_paged_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                          int32_t max_new) {
  if (q_heads < 1 || kv_heads < 1 || head_dim < 1 || max_new < 1) return 256;
  // the most of any call of as many rows or fewer, whatever its cache and table;
  // more than 8 tiles take no tile that fewer do not
  const int64_t tiles = ((int64_t)(q_heads / kv_heads) * max_new + 15) / 16;
  size_t most = 0;
  for (int64_t t = 1; t <= std::min<int64_t>(tiles, 8); ++t)
    for (int dtype : {CX_KV_BF16, CX_KV_E4M3})
      for (int64_t units : {(int64_t)0, cx::ATT_FOUR_UNITS}) {
        const int nt = cx::attend_tiles(16 * t, head_dim, dtype, units);
        most = std::max(most, cx::attend_workspace(nt, head_dim, dtype).total);
      }
  return most;
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
  if ((uintptr_t)workspace & 15)
    return cx::api_fail(CX_EINVAL, "workspace must be 16-byte aligned");
  if ((int64_t)kv->T * q_heads > INT32_MAX) return cx::api_fail(CX_EINVAL, "too many rows");
  A.G = q_heads / kv->kv_heads;
  max_new = std::min(max_new, kv->T);        // no sequence has more
  const int D = kv->head_dim;
  const bool even = kv->T >= (int64_t)kv->B * max_new;
  const int64_t table_units = (int64_t)kv->max_pages * kv->page_tokens / 32;
  const int nt = cx::attend_tiles((int64_t)A.G * max_new, D, kv->dtype,
                                  even ? (int64_t)kv->B * kv->kv_heads * table_units : 0);
  const cx::AttendWork lay = cx::attend_workspace(nt, D, kv->dtype);
  if (ws_bytes < lay.total)
    return cx::api_fail(CX_ENOSPACE, "workspace holds %zu bytes, needs %zu", ws_bytes, lay.total);
  // the units and row blocks, at most, fit the share arithmetic's 38 bits
  const double units = (double)kv->max_pages * kv->page_tokens / 32 + 8;
  const double blocks = kv->kv_heads * ((double)kv->T * (q_heads / kv->kv_heads) / 16 + kv->B);
  if (units * blocks >= 0x1p38) return cx::api_fail(CX_EINVAL, "too many tokens for one call");
  A.q = q; A.q_token = q_token; A.q_head = q_head;
  A.q_heads = q_heads;
  A.cap = softcap > cx::ATT_CAP ? 2 : softcap > 0;
  const double log2e = 1.4426950408889634;
  // (0 times a masked score's infinity would be NaN)
  A.s1 = std::max((float)(scale * log2e), std::numeric_limits<float>::min());
  A.s2 = (float)(softcap * log2e);
  A.s3 = A.cap ? (float)(2 * scale / softcap * log2e) : 0.f;
  A.s4 = A.cap ? (float)(scale / softcap) : 0.f;
  if (!std::isfinite(A.s1) || !std::isfinite(A.s3))
    return cx::api_fail(CX_EINVAL, "scale (%g) and softcap (%g) pass the range of fp32", scale, softcap);
  A.window = window < INT32_MAX - cx::KV_MAX_NEW ? window : INT32_MAX - cx::KV_MAX_NEW;
  A.out = out;
  A.entries = (int*)workspace;
  A.join = (cx::AttendJoin*)((char*)workspace + lay.off_join);
  A.ml = (float*)((char*)workspace + lay.off_ml);
  A.part = (float*)((char*)workspace + lay.off_part);
  const hipStream_t s = (hipStream_t)stream;
  const int e = D == 64    ? cx::launch_attend<64>(A, kv->dtype, nt, max_new, s)
                : D == 128 ? cx::launch_attend<128>(A, kv->dtype, nt, max_new, s)
                           : cx::launch_attend<256>(A, kv->dtype, nt, max_new, s);
  if (e != 0) return cx::api_fail(CX_EHIP, "attention launch: %s", hipGetErrorString((hipError_t)e));
  return CX_OK;
}

}  // extern "C"
