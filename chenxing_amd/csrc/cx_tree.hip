// cx_tree.hip -- attention of trees of drafted tokens over the paged KV cache, for
// gfx950 (layout: cx_kv.hpp).
//
// out[t, h] = sum over the allowed slots s of softmax(scale q.k_s) v_s, in one pass
// over K and V with the running maximum m and sum l of the softmax's terms: a block of
// scores raises m to m', and l and the output so far are scaled by exp(m - m').  Two
// stream-ordered launches:
//
//   1. tree_split  workgroups of 8 waves, each with an equal share of all the batch's
//                  units (32 slots for one kv head and row block); a row block that
//                  ends inside the share it began in is written out, the others'
//                  parts (m, l, sums) go to the workspace.
//   2. tree_join   a workgroup per split row block and 16 rows: its parts, in the
//                  order of their slots.
//
// or, for short tables, a workgroup for a chunk of a row block's units, and the join of
// those that have more than one.
//
// K and V are read once for up to 256 rows, so trees of 64 nodes are bound by the matrix
// cores (with the terms in two parts half as much again as the formula's products) and by
// the softmax beside them: 2 sequences of 120001 .. 131072 tokens, 32 / 8 heads of 128,
// bf16, 445 us, 586 TFLOP/s of the formula's; 64 of up to 8192, e4m3, 433 us.  Few rows are
// bound by the start, a step's latency (1.2 us at D = 128) and a row block's own cost (about
// 5 us: its rows, the groups' meeting, its part): 32 ragged trees of up to 33 nodes 52 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "cx_device.hpp"
#include "cx_dma.hpp"
#include "cx_internal.hpp"
#include "cx_kv.hpp"
#include "cx_lanes.hpp"
#include "cx_sampler.h"
#include "cx_share.hpp"
#include "cx_timing.hpp"

namespace cx {

constexpr int TREE_WAVES = 8, TREE_WG = 64 * TREE_WAVES;
constexpr int TREE_WORKERS = 256;            // a workgroup a CU: they are on the chip at once
constexpr int TREE_UNIT = 32;                // slots of a unit
constexpr int TREE_LEAST = 2;                // the least share, in units
// Units of a workgroup's chunk at most, and workgroups of chunks that are aimed at: those
// that are on the chip at once.  32 q / 8 kv heads of 128, bf16, chunks and shares, us: one
// request, 16 nodes, of 700 tokens 13.8 and 17.2, of 6000 22 and 27; four of 1500 18.3 and
// 22.3; 16 of 700 22.8 and 28.5.  Past 16 units a chunk gains where lengths are alike (16
// requests of 1500, chunks of 24: 32 and 38) and loses more where they are not (16 of 50 ..
// 1500, 1 .. 64 nodes: 49 and 36).  Twice the workgroups, in two turns: 16 requests of 500 ..
// 1500, 1 .. 33 nodes, 64 us, in shares 39; one of 6000 36, not 22.  Row blocks, a chunk each,
// may be twice the workgroups, no more: requests of 20 .. 500 tokens, 64 of 1 .. 16 nodes
// (512 row blocks) 34 and 36, of 1 .. 33 nodes 24 (576) 28 and 29, 64 63 and 47, 256 232 and
// 131.
constexpr int TREE_CHUNK = 16;
constexpr int64_t TREE_SPREAD = TREE_WORKERS, TREE_BLOCKS = 2 * TREE_WORKERS;
constexpr int TREE_BATCH = 512;              // sequences of a launch: their lengths are in LDS
// A lane's terms of a unit sum to this before the running maximum is raised: it need not
// be the largest score, so most units look for none (64 trees of 64 nodes 440 us, with the
// maximum looked for in every unit 551).
constexpr float TREE_SLACK = 4096.f;
constexpr float TREE_LOW = -3e38f;           // running maximum of a row that attends to something

struct TreeArgs {
  KvArgs kv;
  const uint16_t* q;
  int64_t q_token, q_head;
  int q_heads, G;             // G: q heads per kv head
  const uint32_t* mask;       // [T, words] of 32 bits
  int words;
  const int32_t* depth;       // nullable
  // score in powers of 2: s1 qk, or s2 tanh(s4 qk), where exp(2 s4 qk) = 2 ^ (s3 qk)
  float s1, s2, s3, s4;
  int cap;                    // the latter
  int window;                 // 0: none
  uint16_t* out;
  int b0;                     // first sequence of the launch; kv.B: their number
  int tiles, chunks, chunk;   // row blocks of a sequence, their parts, units of a part
  int* entries;               // number of entries of join
  AttendJoin* join;           // [TREE_WORKERS]
  float* ml;                  // [slots, ROWS, 2]: a part's maxima and sums
  float* part;                // [slots, ROWS, D], in the order of join's lanes
};

// The kernel's arguments in memory (its first, at the segment's start), for the parts
// that run once a piece: what they need is read there again, so the loop keeps its
// scalar registers.
__device__ __forceinline__ const TreeArgs& tree_args() {
  uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const TreeArgs*)(const CX_CONST TreeArgs*)p;
}
// The lane's number, for rare code: what it makes of it is not kept for the loop.
__device__ __forceinline__ int rare_lane() {
  int l = lane_id();
  asm volatile("" : "+v"(l));
  return l;
}
// Sequence b of a launch, its lengths by scalar loads.
template <class Line>
__device__ __forceinline__ AttendSeq tree_seq(const TreeArgs& A, int b) {
  int s0 = A.b0 + b, s1 = s0 + 1;
  if (A.kv.q_start) {
    s0 = min(max(const_load(A.kv.q_start + b), 0), A.kv.T);
    s1 = min(max(const_load(A.kv.q_start + b + 1), s0), A.kv.T);
  }
  return Line::seq(ShareBatch{A.G, A.kv.heads, A.window, A.kv.n_pages ? A.kv.M << A.kv.logP : 0}, s0, s1,
                   const_load(A.kv.kv_len + b));
}
// load_lds16 from a scalar base, and 4 bytes a lane.
__device__ __forceinline__ void load_lds16_at(const char* base, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(to), "v"(at), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void load_lds4(const char* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               :: "s"(to), "v"(from) : "memory", "m0");
}
// 8 waves: WR of them share a unit's K and V, each for 16 NT rows; WT such groups take
// every WT-th unit.
template <int D, int NT, int WR, bool F8>
struct TreeShape {
  static constexpr int WT = TREE_WAVES / WR, ROWS = 16 * NT * WR;
  // e4m3: many waves share a unit, so its codes are made bf16 once (CONV), else by
  // each wave as it reads them (64 trees of 64 nodes 440 and 448 us; four waves' two units
  // of D = 256 in bf16 do not fit beside the ring)
  static constexpr bool CONV = F8 && WR >= 4 && !(D == 256 && WR == 4);
  static constexpr int KB = (F8 ? 1 : 2) * TREE_UNIT * D;       // bytes of a unit's K
  static constexpr int RAW = 2 * KB;
  static constexpr int LOADS = 2 * KB / 1024;                   // of 1 KB
  static constexpr int LW = (LOADS + WR - 1) / WR;              // of a wave, at most
  static constexpr int WIDE = 2 * TREE_UNIT * D * 2;            // a unit in bf16
  // stages of the ring
  static constexpr int S = WR == 8 ? (D == 256 ? 4 : 8)
                           : D == 64 ? 4
                           : F8      ? (D == 256 && WR == 2 ? 2 : 3)
                                     : (D == 128 && WR == 4 ? 3 : 2);
  // bytes of a group: the ring, e4m3 its scales (256 bytes, kept a step longer), CONV
  // two units in bf16
  static constexpr int SCALES = F8 ? 256 * (S + 1) : 0;
  static constexpr int GROUP = S * RAW + SCALES + (CONV ? 2 * WIDE : 0);
  // the groups' sums meet DR dims at a time
  static constexpr int DR = WT == 1 ? D : WR == 2 ? 32 : 64;
  static constexpr int SCRATCH = WT == 1 ? 0 : (WT - 1) * WR * 16 * (DR + 16) * 4;
  using Line = AttendLine<TREE_UNIT, NT * WR, true>;
  using Seqs = AttendSeqs<CX_LDS uint64_t*, CX_LDS int*>;
  static constexpr int QUEUE = TREE_WAVES * (S + 2) * 64;       // pieces on their way, by wave
  static constexpr int off_scratch() { return WT * GROUP; }
  static constexpr int off_queue() { return off_scratch() + SCRATCH; }
  static constexpr int off_seqs() { return off_queue() + QUEUE + TREE_WAVES * 8; }
  static constexpr int lds() { return off_seqs() + Seqs::bytes(TREE_BATCH, true); }
  static_assert(lds() <= 160 * 1024, "LDS");
};

//  * S^T = K Q^T: row 4 g + j of score tile y is slot 8 g + 4 y + j of the unit, so a
//    lane's terms of both tiles are those of the 8 slots whose V is one of its 16-byte
//    chunks: O^T = V^T P^T takes them as they are.  K's slots stand in LDS in that
//    order.
//  * K and V go from the pages to LDS without registers, S - 1 units ahead, from one
//    piece to the next; a barrier a unit.  Each wave counts its own loads: they are
//    unconditional, after the last unit all of one place.
//  * Softmax terms enter the products as two bf16 parts (16 bits): one part's rounding
//    would add as much error as the result's own.
//
// SHARES: each of TREE_WORKERS workgroups takes an equal stretch of the line of all the
// batch's units (cx_share.hpp).  Else a workgroup takes A.chunk units of one row block:
// no lengths to sum up, no places to find (launch_tree says when).
template <int D, int NT, int WR, bool F8, bool SHARES>
__global__ __launch_bounds__(TREE_WG) void tree_split(TreeArgs A) {
  using Sh = TreeShape<D, NT, WR, F8>;
  using Line = typename Sh::Line;
  constexpr int WT = Sh::WT, ROWS = Sh::ROWS, S = Sh::S, KB = Sh::KB, RAW = Sh::RAW;
  constexpr int E = F8 ? 16 : 8, QL = D / 32, DT = D / 16;
  constexpr bool CONV = Sh::CONV, NARROW = F8 && !CONV;         // operands from codes
  extern __shared__ __align__(16) char lds[];
  const KvArgs& C = A.kv;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(wave_id()), l = lane_id();
  const int g = l >> 4, c = l & 15;
  const int wr = w % WR, wt = w / WR;        // row wave, group
  const int P = 1 << C.logP;
  CX_LDS char* const ring = to_lds(lds) + wt * Sh::GROUP;
  CX_LDS char* const s_scale = ring + S * RAW;
  CX_LDS char* const wide = s_scale + Sh::SCALES;
  CX_LDS f32x4* const s_acc = (CX_LDS f32x4*)(to_lds(lds) + Sh::off_scratch());
  CX_LDS uint64_t* const s_pref = (CX_LDS uint64_t*)(to_lds(lds) + Sh::off_seqs());
  CX_LDS uint64_t* const s_sum = s_pref - TREE_WAVES;
  CX_LDS int* const s_len = (CX_LDS int*)(s_pref + C.B + 1);
  const typename Sh::Seqs seqs = {s_pref, s_len, s_len + C.B, C.q_start != nullptr};
  CX_LDS int* const s_queue = (CX_LDS int*)(to_lds(lds) + Sh::off_queue()) + w * (S + 2) * 16;
  auto share_batch = [&]() {
    const auto& A = tree_args();
    return ShareBatch{A.G, A.kv.heads, A.window, A.kv.n_pages ? A.kv.M << A.kv.logP : 0};
  };
  auto first = [&](int b) { return seqs.starts ? seqs.first(b) : tree_args().b0 + b; };
  auto seq = [&](const ShareBatch& batch, int b) {
    const int f = first(b);
    return Line::seq(batch, f, seqs.starts ? seqs.end(b) : f + 1, s_len[b]);
  };
  // tokens r0 .. end - 1 attend to nothing
  auto nothing = [&](int r0, int end) {
    const int64_t n = (int64_t)(end - r0) * A.q_heads * (D / 8);
    u32x4* o = (u32x4*)(A.out + (int64_t)r0 * A.q_heads * D);
    for (int64_t i = tid; i < n; i += TREE_WG) o[i] = u32x4{0, 0, 0, 0};
  };

  const unsigned worker = blockIdx.x;
  ShareSplit split = {};
  uint64_t end = 0;
  int blocks = 0;                            // the sequence's row blocks
  AttendSeq own = {};                        // the sequence
  if constexpr (SHARES) {
    // the line before each sequence, and its whole
    seqs.read(C.kv_len, C.q_start, C.B, C.T, tid, TREE_WG);
    __syncthreads();
    const int b = tid;                       // (a launch's sequences are no more)
    uint64_t x = 0;
    if (b < C.B) x = Line::length(share_batch(), seq(share_batch(), b));
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t y = __shfl_up(x, o);
      if (l >= o) x += y;
    }
    if (l == 63) s_sum[w] = x;
    __syncthreads();
    for (int k = 0; k < w; ++k) x += s_sum[k];
    if (b < C.B) s_pref[b + 1] = x;
    if (tid == 0) s_pref[0] = 0;
    __syncthreads();
    const uint64_t line = scalar64(s_pref[C.B]);
    split = share_split(line, TREE_WORKERS, TREE_LEAST);
    split.per = scalar64(split.per);
    split.more = scalar64(split.more);
    if (worker == 0 && tid == 0) *A.entries = split.by_block ? (int)line_blocks(line) : TREE_WORKERS;
    for (int b = blockIdx.x; b < C.B; b += TREE_WORKERS)
      if (s_pref[b + 1] == s_pref[b]) nothing(first(b), seqs.starts ? seqs.end(b) : first(b) + 1);
    if (worker >= split.shares) {
      if (tid == 0 && !split.by_block) A.join[worker].last = -1;
      return;
    }
    end = share_begin(split, worker) + split.per + (worker < split.more);
  } else {
    own = tree_seq<Line>(A, blockIdx.z);
    blocks = Line::row_blocks(share_batch(), own);
    if (own.n == 0) {
      if (blockIdx.x == 0 && blockIdx.y == 0) nothing(own.tok0, own.tok0 + own.q);
      return;
    }
  }

  // The workgroup's pieces, as they are loaded; what is computed takes them, up to S +
  // 1 later, from the wave's queue.
  struct {
    const int32_t* ids;       // of the sequence's pages
    const char* head;         // the head's part of page 0
    int groups, unit, cnt;    // groups of 16 slots
  } ahead = {nullptr, C.pages, 0, 0, 0};
  int step = 0, steps = 0;                   // of the piece that is loaded
  uint64_t u = 0;                            // SHARES: past it
  int b = 0;
  int rb = blockIdx.y, chunk = 0;            // else the row block and the part of its units
  if constexpr (SHARES) {
    u = share_begin(split, worker);
    for (int hi = C.B - 1; b < hi;) {        // the last b with its units at or before u
      const int mid = (b + hi + 1) >> 1;
      if (line_units(s_pref[mid]) <= u) b = mid;
      else hi = mid - 1;
    }
  } else {
    for (; rb >= A.tiles; rb -= A.tiles) ++chunk;               // (a few)
    if (rb >= blocks || chunk * A.chunk >= own.n) return;
  }
  bool joined = false;
  int pushed = 0;
  // The next piece, pushed to the queue, and whether there is one.
  auto next_piece = [&]() {
    const auto& A = tree_args();
    const ShareBatch batch = share_batch();
    AttendPiece p;
    if constexpr (SHARES) {
      if (u >= end) return false;
      while (line_units(s_pref[b + 1]) <= u) ++b;
      b = __builtin_amdgcn_readfirstlane(b);
      p = Line::piece(batch, seq(batch, b), b, s_pref[b], split, worker, end, u,
                      [&](unsigned entry, const AttendJoin& j) {
                        joined |= j.last >= 0;
                        if (tid == 0) A.join[entry] = j;
                      });
      u = scalar64(u);
      if (p.cnt == 0) return false;
    } else {
      // its chunk; then, where a sequence has more new tokens than the caller said, the
      // first chunk's workgroups take whole row blocks
      const bool whole = rb >= A.tiles;
      if (rb >= blocks || (whole && chunk > 0)) return false;
      p.b = blockIdx.z;
      p.h = blockIdx.x;
      p.tok0 = own.tok0;
      p.r0 = rb * ROWS;
      p.R = min(ROWS, own.q * A.G - p.r0);
      p.lowest = own.len - own.q;
      p.lim = own.lim;
      p.unit = own.first + (whole ? 0 : chunk * A.chunk);
      // (the last one what a longer context than the launch counts on has left)
      p.cnt = whole ? own.n : own.n - chunk * A.chunk;
      if (!whole && chunk + 1 < A.chunks) p.cnt = min(p.cnt, A.chunk);
      p.slot = p.cnt == own.n ? -1
                              : (p.b * A.kv.heads + p.h) * A.tiles * A.chunks + rb * A.chunks + chunk;
      rb += A.tiles;
    }
    ahead.ids = A.kv.table + __builtin_amdgcn_readfirstlane(p.b) * A.kv.ld_table;
    ahead.head = A.kv.pages + __builtin_amdgcn_readfirstlane(p.h) * (int64_t)A.kv.head_bytes;
    ahead.groups = (__builtin_amdgcn_readfirstlane(p.lim) + 15) >> 4;
    ahead.unit = __builtin_amdgcn_readfirstlane(p.unit);
    ahead.cnt = __builtin_amdgcn_readfirstlane(p.cnt);
    const int l = rare_lane();
    const int x = l == 0 ? p.h : l == 1 ? p.tok0 : l == 2 ? p.r0 : l == 3 ? p.R : l == 4 ? p.lowest
                  : l == 5 ? p.lim : l == 6 ? p.unit : l == 7 ? p.cnt : p.slot;
    if (l < 9) s_queue[16 * pushed + l] = x;
    pushed = pushed == S + 1 ? 0 : pushed + 1;
    step = 0;
    steps = (ahead.cnt + WT - 1) / WT;
    return true;
  };
  // ------------------------------------------------------------------ loads
  // The ids of a unit's two groups of 16 slots, asked for a step before they are used.
  bool more = true, live = false;            // pieces to load; a unit for this group's next stage
  int unit = 0, next0 = -1, next1 = -1;
  auto ask = [&]() {
    unit = ahead.unit + step * WT + wt;
    live = more && step * WT + wt < ahead.cnt;
    auto id = [&](int half) {
      const int s16 = 2 * unit + half;
      if (!live || s16 >= ahead.groups) return -1;
      return const_load(ahead.ids + (s16 >> (C.logP - 4)));
    };
    next0 = id(0);
    next1 = id(1);
  };
  // Load j of the wave is chunks 64 i .. of the stage, i = wr + WR j: of K, chunk rows 2 i
  // and 2 i + 1 of 32 slots, the lane's in group c / 8; of V (F8: 16 slots a chunk) of D
  // dims.  The lane's place in its page's part, but for the unit's:
  constexpr int NK = Sh::LOADS / 2;
  uint32_t place[Sh::LW];
#pragma unroll
  for (int j = 0; j < Sh::LW; ++j) {
    const int i = wr + WR * j, f = 64 * (i - NK), row = f / D;
    const int slot = 8 * (c >> 2 & 1) + 4 * (l >> 4 & 1) + (c & 3);
    place[j] = i < NK ? (((2 * i + (l >> 5)) << C.logP) + slot) * 16
                      : v_chunk<E, D>(f % D + l, F8 ? 0 : 8 * (row & 1), C.logP);
  }
  const uint32_t place_scale = k_scale<D>(l & 15, C.logP) + (l & 32 ? 4 * P : 0);
  uint32_t fill = 0, fill_scale = 0;         // the stage that is loaded next, its scales
  uint32_t held = 0, fill_held = 0;          // two bits a stage: its groups are in the pool
  auto request = [&]() {
    const bool in0 = (unsigned)next0 < (unsigned)C.n_pages, in1 = (unsigned)next1 < (unsigned)C.n_pages;
    held = (held & ~(3u << 2 * fill_held)) | ((in0 ? 1u : 0u) | (in1 ? 2u : 0u)) << 2 * fill_held;
    fill_held = (fill_held + 1) & 15;
    const char* p0 = ahead.head + (in0 ? next0 : 0) * C.page_stride;
    const char* p1 = ahead.head + (in1 ? next1 : 0) * C.page_stride;
    const int o0 = live ? (unit * 32) & (P - 1) : 0, o1 = live ? (unit * 32 + 16) & (P - 1) : 0;
    const uint32_t to = (uint32_t)(uintptr_t)ring + fill * RAW;
    const uint32_t on = live ? ~0u : 0;      // without a unit: page 0's first bytes, all lanes
    if (F8 && wr == 0) {
      // in their slots' order: keys' scales, then values'
      const char* p = l & 16 ? p1 + 4 * o1 : p0 + 4 * o0;
      load_lds4(p + (place_scale & on), (uint32_t)(uintptr_t)s_scale + 256 * fill_scale);
    }
    const char* pk = c & 8 ? p1 + 16 * o1 : p0 + 16 * o0;
    constexpr int VS = F8 ? D : 2 * D;       // bytes of V a slot
#pragma unroll
    for (int j = 0; j < Sh::LW; ++j) {
      const int i = wr + WR * j;
      if (i >= Sh::LOADS) break;             // (uniform)
      if (NK % WR == 0 ? WR * j < NK : i < NK) {
        load_lds16(pk + (place[j] & on), to + 1024 * i);
      } else {
        const int row = 64 * (i - NK) / D, half = F8 ? row : row >> 1;
        load_lds16_at(half ? p1 + (int64_t)o1 * VS : p0 + (int64_t)o0 * VS, place[j] & on, to + 1024 * i);
      }
    }
    fill = fill + 1 == S ? 0 : fill + 1;
    if (F8) fill_scale = fill_scale == S ? 0 : fill_scale + 1;
  };
  // until the oldest of the stages under way, all but the N newest, are in LDS
  auto arrive = [&](auto n) {
    constexpr int N = decltype(n)::value;
    if (F8 && wr == 0) wave_vm<N * (Sh::LW + 1)>();
    else wave_vm<N * Sh::LW>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  uint32_t take = 0;                         // the stage that is computed (CONV: converted) next
  uint32_t conv = 0;                         // CONV: the bf16 buffer that it goes to
  auto convert = [&]() {
    const CX_LDS char* raw = ring + take * RAW;
    CX_LDS char* to = wide + conv * Sh::WIDE;
#pragma unroll
    for (int j = 0; j < (2 * KB / 1024 + WR - 1) / WR; ++j) {
      if (wr + WR * j >= 2 * KB / 1024) break;                  // (uniform)
      const int f = (wr + WR * j) * 64 + l;
      const u32x4 x = *(const CX_LDS u32x4*)(raw + 16 * f);
      const bf16x8 lo = e4m3x8(x[0], x[1]), hi = e4m3x8(x[2], x[3]);
      // K: chunk rows of 32 slots; V: of D dims
      const int fv = f - KB / 16;
      const int at = fv < 0 ? (f / 32 * 2) * 32 + f % 32 : 2 * KB / 16 + fv / D * 2 * D + fv % D;
      *(CX_LDS bf16x8*)(to + 16 * at) = lo;
      *(CX_LDS bf16x8*)(to + 16 * (at + (fv < 0 ? 32 : D))) = hi;
    }
    take = take + 1 == S ? 0 : take + 1;
    conv ^= 1;
  };

  // ------------------------------------------------------------------ a piece's rows
  u32x4 qr[NT][QL];
  f32x4 acc[NT][DT];
  float m[NT], sum[NT];
  int lo[NT];                                // of the slots before the tree: those above
  const uint32_t* mrow[NT];                  // the row's mask
  uint32_t mlow[NT][2];                      // and its first 64 bits
  struct {
    int h, tok0, r0, R, lowest, lim, unit, cnt, slot;
  } cur;
  int popped = 0, i = 0, todo = 0;           // the step of the piece, and its steps
  int count = 0;                             // its units, 0 for a wave without rows
  auto begin = [&]() {
    const auto& A = tree_args();
    const int l = rare_lane(), g = l >> 4, c = l & 15;
    const int x = s_queue[16 * popped + c];
    popped = popped == S + 1 ? 0 : popped + 1;
    cur.h = lane_read(x, 0);
    cur.tok0 = lane_read(x, 1);
    cur.r0 = lane_read(x, 2);
    cur.R = lane_read(x, 3);
    cur.lowest = lane_read(x, 4);
    cur.lim = lane_read(x, 5);
    cur.unit = lane_read(x, 6);
    cur.cnt = lane_read(x, 7);
    cur.slot = lane_read(x, 8);
    i = 0;
    todo = (cur.cnt + WT - 1) / WT;
    count = 16 * NT * wr < cur.R ? cur.cnt : 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = cur.r0 + min(16 * (NT * wr + nt) + c, cur.R - 1);
      const int t = cur.tok0 + row / A.G;
      const uint16_t* q = A.q + t * A.q_token + (cur.h * A.G + row % A.G) * A.q_head;
#pragma unroll
      for (int x = 0; x < QL; ++x) qr[nt][x] = *(const u32x4*)(q + 32 * x + 8 * g);
      mrow[nt] = A.mask + (int64_t)t * A.words;
      mlow[nt][0] = mrow[nt][0];
      mlow[nt][1] = mrow[nt][1];
      lo[nt] = A.window ? cur.lowest - A.window + min(max(A.depth[t], 0), 1 << 28) : -1;
      m[nt] = -INFINITY;
      sum[nt] = 0;
#pragma unroll
      for (int n = 0; n < DT; ++n) acc[nt][n] = f32x4{0, 0, 0, 0};
    }
    // waited for here: at their first use the wait would be part of every step, and drain
    // the loads under way
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int x = 0; x < QL; ++x) asm volatile("" : "+v"(qr[nt][x]));
      asm volatile("" : "+v"(lo[nt]), "+v"(mlow[nt][0]), "+v"(mlow[nt][1]));
    }
  };
  // the bits of nodes i0 .. i0 + 31
  auto node_bits = [&](int nt, int i0) {
    auto word = [&](int k) -> uint32_t {
      return k < 0 || k >= A.words ? 0 : k == 0 ? mlow[nt][0] : k == 1 ? mlow[nt][1] : mrow[nt][k];
    };
    const int k = i0 >> 5, sh = i0 & 31;
    const uint64_t both = (uint64_t)word(k) | (uint64_t)word(k + 1) << 32;
    return (uint32_t)(both >> sh);
  };
  // What a unit's products with V need of its scores.
  u32x4 ph[NT], pl[NT];                      // the terms, in two parts
  bool masked = false;
  uint32_t valid = 0, bits[NT];              // slots that are held; that the row attends to
  const CX_LDS char* vb = nullptr;
  auto scores = [&](int unit, uint32_t here, const CX_LDS char* kv, const CX_LDS char* scales) {
    const int t0 = unit * TREE_UNIT;
    f32x4 v[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) v[nt][0] = v[nt][1] = f32x4{0, 0, 0, 0};
    auto key = [&](int x, int y) {
      if (NARROW) {
        const u32x2 r = *(const CX_LDS u32x2*)(kv + ((2 * x + (g >> 1)) * 32 + 16 * y + c) * 16 + 8 * (g & 1));
        return u32x4{r[0], r[1], 0, 0};
      }
      return *(const CX_LDS u32x4*)(kv + ((4 * x + g) * 32 + 16 * y + c) * 16);
    };
    // (four steps' keys at a time: as many as the registers hold)
#pragma unroll
    for (int x0 = 0; x0 < QL; x0 += 4) {
      constexpr int N = QL < 4 ? QL : 4;
      u32x4 ka[N][2];
#pragma unroll
      for (int x = 0; x < N; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) ka[x][y] = key(x0 + x, y);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < N; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const bf16x8 k = NARROW ? e4m3x8(ka[x][y][0], ka[x][y][1]) : __builtin_bit_cast(bf16x8, ka[x][y]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            v[nt][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, __builtin_bit_cast(bf16x8, qr[nt][x0 + x]),
                                                               v[nt][y], 0, 0, 0);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    vb = kv + (NARROW ? KB : 2 * TREE_UNIT * D);
    f32x4 vs[F8 ? 2 : 1];
    if (F8) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const f32x4 ks = *(const CX_LDS f32x4*)(scales + 4 * (8 * g + 4 * y));
        vs[y] = *(const CX_LDS f32x4*)(scales + 128 + 4 * (8 * g + 4 * y));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) v[nt][y] *= ks;
      }
    }
    const float to2 = A.cap ? 1.f : A.s1;
    if (A.cap) {                             // tanh(z) = 1 - 2 / (exp(2 z) + 1), near 0 its series
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = v[nt][y][j], z = A.s4 * x, zz = z * z, sx = A.s1 * x;
            const float far = fmaf(-2.f * A.s2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(A.s3 * x) + 1.f), A.s2);
            v[nt][y][j] = zz < 1.f / 256.f ? fmaf(sx * zz, fmaf(zz, 2.f / 15.f, -1.f / 3.f), sx) : far;
          }
    }
    // a unit is open where all its slots are held, before the tree and inside every
    // row's window
    masked = t0 + TREE_UNIT > min(cur.lowest, cur.lim) || here != 3;
    if (A.window) {
      bool out = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) out |= lo[nt] >= t0;
      masked |= __any(out);
    }
    valid = ~0u;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) bits[nt] = ~0u;
    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
    if (masked) {
      const int g = rare_lane() >> 4;
      valid = (here & 1 ? 0xFFFFu : 0u) | (here & 2 ? 0xFFFF0000u : 0u);
      valid &= below(cur.lim - t0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t x = below(cur.lowest - t0) & ~below(lo[nt] + 1 - t0);
        if (t0 + TREE_UNIT > cur.lowest) x |= node_bits(nt, t0 - cur.lowest);
        bits[nt] = x & valid;
        const uint32_t mine = bits[nt] >> (8 * g);
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[nt][y][j] = mine >> (4 * y + j) & 1 ? v[nt][y][j] : -INFINITY;
      }
    }
    // terms by the maximum so far, unless one is much above it (or there is none)
    float all = 0, add[NT];
    f32x4 p[NT][2];
    auto terms = [&](int nt, float base) {
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int j = 0; j < 4; ++j) p[nt][y][j] = __builtin_amdgcn_exp2f(fmaf(to2, v[nt][y][j], -base));
      add[nt] = ((p[nt][0][0] + p[nt][0][1]) + (p[nt][0][2] + p[nt][0][3])) +
                ((p[nt][1][0] + p[nt][1][1]) + (p[nt][1][2] + p[nt][1][3]));
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      terms(nt, m[nt]);
      all += add[nt];
    }
    if (masked || __any(!(all < TREE_SLACK))) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top = bits[nt] == 0 ? -INFINITY : TREE_LOW;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int j = 0; j < 4; ++j) top = fmaxf(top, to2 * v[nt][y][j]);
        const float m1 = fmaxf(m[nt], groups_max(top));
        const float alpha = m[nt] == m1 ? 1.f : __builtin_amdgcn_exp2f(m[nt] - m1);
        m[nt] = m1;
        sum[nt] *= alpha;
#pragma unroll
        for (int n = 0; n < DT; ++n) acc[nt][n] *= alpha;
        terms(nt, m1 == -INFINITY ? 0.f : m1);
      }
    }
    if (F8) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int y = 0; y < 2; ++y) p[nt][y] *= vs[y];
      if (masked) {                          // (0 times a scale that is NaN)
        const int g = rare_lane() >> 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int j = 0; j < 4; ++j) p[nt][y][j] = bits[nt] >> (8 * g + 4 * y + j) & 1 ? p[nt][y][j] : 0.f;
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      sum[nt] += add[nt];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        // two bf16 parts: the first cut off, the second never 0, so that an infinite
        // value keeps its sign in both products (2^-23 of a term too much).  That is 2^-16
        // of a term, and 0.2 to 0.5 % of the results are the other neighbour of what 64
        // bits round to, where a third part leaves 0.03 to 0.13 % and its products take 518
        // us for 2 documents of 131072 tokens, not 445, and 485 for 64 full trees, not 433
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const float p0 = p[nt][y][2 * d], p1 = p[nt][y][2 * d + 1];
          const uint32_t x0 = __float_as_uint(p0), x1 = __float_as_uint(p1);
          ph[nt][2 * y + d] = __builtin_amdgcn_perm(x1, x0, 0x07060302);
          pl[nt][2 * y + d] = pack_bf16(fmaf(p0, 1.f + 0x1p-23f, -__uint_as_float(x0 & 0xFFFF0000u)),
                                        fmaf(p1, 1.f + 0x1p-23f, -__uint_as_float(x1 & 0xFFFF0000u)));
        }
      }
    }
  };
  // The products with V.  V of slots that nobody holds counts as zeros, whatever is there,
  // and NaN and infinity reach the rows that attend to them only: left out of the
  // products and added one by one.
  auto values = [&](auto then) {
    auto value = [&](int n) {
      if (NARROW) {
        const u32x2 r = *(const CX_LDS u32x2*)(vb + ((g >> 1) * D + 16 * n + c) * 16 + 8 * (g & 1));
        return u32x4{r[0], r[1], 0, 0};
      }
      return *(const CX_LDS u32x4*)(vb + (g * D + 16 * n + c) * 16);
    };
    constexpr int EARLY = 4;                 // 16-dim tiles that are read together
    u32x4 va[EARLY];
#pragma unroll
    for (int n = 0; n < EARLY; ++n) va[n] = value(n);
    uint32_t bad = 0;
#pragma unroll
    for (int n0 = 0; n0 < DT; n0 += EARLY) {
      u32x4 x[EARLY];
#pragma unroll
      for (int n = 0; n < EARLY; ++n) {
        x[n] = va[n];
        if (NARROW) x[n] = __builtin_bit_cast(u32x4, e4m3x8(x[n][0], x[n][1]));
      }
      if (masked) {
        const int g = rare_lane() >> 4;
#pragma unroll
        for (int n = 0; n < EARLY; ++n)
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const uint32_t two = valid >> (8 * g + 2 * d);
            x[n][d] &= (two & 1 ? 0xFFFFu : 0) | (two & 2 ? 0xFFFF0000u : 0);
            bad |= nonfinite_sign<false>(x[n][d]);
            x[n][d] &= finite_mask<false>(x[n][d]);
          }
      }
      if (n0 + EARLY < DT) {
#pragma unroll
        for (int n = 0; n < EARLY; ++n) va[n] = value(n0 + EARLY + n);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        // its scalar loads would make LDS reads after them wait for all: there are none
        __builtin_amdgcn_sched_barrier(0);
        then();
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int n = 0; n < EARLY; ++n) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          acc[nt][n0 + n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, x[n]), __builtin_bit_cast(bf16x8, ph[nt]), acc[nt][n0 + n], 0, 0, 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          acc[nt][n0 + n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, x[n]), __builtin_bit_cast(bf16x8, pl[nt]), acc[nt][n0 + n], 0, 0, 0);
      }
    }
    const bool some = masked && __any((bad & 0x80008000u) != 0);
    if (!some) return;
    const int lane = rare_lane(), gr = lane >> 4;
#pragma unroll 1
    for (int k = 0; k < TREE_UNIT; ++k) {
      if (!(valid >> k & 1)) continue;
#pragma unroll
      for (int n = 0; n < DT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = 16 * n + 4 * gr + j;
          float x;
          if (NARROW) x = e4m3_value(*(const CX_LDS uint8_t*)(vb + ((k >> 4) * D + d) * 16 + (k & 15)));
          else x = bf16_lo(*(const CX_LDS uint16_t*)(vb + ((k >> 3) * D + d) * 16 + 2 * (k & 7)));
          const bool fine = fabsf(x) < INFINITY;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[nt][n][j] += !fine && (bits[nt] >> k & 1) ? x : 0.f;
        }
    }
  };

  // the groups' sums meet in the first one's registers
  auto meet = [&]() {
    if constexpr (WT > 1) {
      constexpr int ND = Sh::DR / 16;
      CX_LDS f32x4* const mine = s_acc + ((wt - 1) * WR + wr) * (ND + 1) * 64;
      auto barrier = [&]() {
        __builtin_amdgcn_s_waitcnt((15 | 3 << 14) | (7 << 4));  // LDS alone
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      };
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f0 = 1.f, f[WT];
#pragma unroll
        for (int x = 0; x < DT / ND; ++x) {
          if (wt > 0) {
#pragma unroll
            for (int n = 0; n < ND; ++n) mine[n * 64 + l] = acc[nt][ND * x + n];
            if (x == 0) mine[ND * 64 + l] = f32x4{m[nt], sum[nt], 0, 0};
          }
          barrier();
          if (wt == 0) {
            const CX_LDS f32x4* at = s_acc + wr * (ND + 1) * 64;
            if (x == 0) {
              float top = m[nt], other[WT];
#pragma unroll
              for (int k = 1; k < WT; ++k) {
                const f32x4 ml = at[((k - 1) * WR * (ND + 1) + ND) * 64 + l];
                other[k] = ml[0];
                f[k] = ml[1];
                top = fmaxf(top, ml[0]);
              }
              const float base = top == -INFINITY ? 0.f : top;
              f0 = __builtin_amdgcn_exp2f(m[nt] - base);
              sum[nt] *= f0;
              m[nt] = top;
#pragma unroll
              for (int k = 1; k < WT; ++k) {
                const float e = __builtin_amdgcn_exp2f(other[k] - base);
                sum[nt] = fmaf(e, f[k], sum[nt]);
                f[k] = e;
              }
            }
#pragma unroll
            for (int n = 0; n < ND; ++n) {
              f32x4 a = acc[nt][ND * x + n] * f0;
#pragma unroll
              for (int k = 1; k < WT; ++k) a += f[k] * at[((k - 1) * WR * (ND + 1) + n) * 64 + l];
              acc[nt][ND * x + n] = a;
            }
          }
          barrier();
        }
      }
    }
  };
  auto finish = [&]() {
    meet();
    if (wt > 0) return;
    const auto& A = tree_args();
    const int l = rare_lane(), g = l >> 4, c = l & 15;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float L = groups_sum(sum[nt]);
      const int r = 16 * (NT * wr + nt) + c;
      if (cur.slot < 0) {
        if (r >= cur.R) continue;
        const float f = m[nt] == -INFINITY ? 0.f : 1.f / L;
        const int row = cur.r0 + r;
        uint16_t* o = A.out + ((int64_t)(cur.tok0 + row / A.G) * A.q_heads + cur.h * A.G + row % A.G) * D + 4 * g;
#pragma unroll
        for (int n = 0; n < DT; ++n)
          *(u32x2*)(o + 16 * n) = u32x2{pack_bf16(acc[nt][n][0] * f, acc[nt][n][1] * f),
                                        pack_bf16(acc[nt][n][2] * f, acc[nt][n][3] * f)};
      } else if (16 * (NT * wr + nt) < cur.R) {
        const int64_t tile = (int64_t)cur.slot * (ROWS / 16) + NT * wr + nt;
        f32x4* o = (f32x4*)(A.part + tile * 16 * D) + l;
#pragma unroll
        for (int n = 0; n < DT; ++n) o[64 * n] = acc[nt][n];
        if (g == 0) *(float2*)(A.ml + 2 * (tile * 16 + c)) = make_float2(m[nt], L);
      }
    }
  };

  // ------------------------------------------------------------------ the steps
  // FIRST steps load only; then each computes what arrived and loads FIRST steps ahead
  constexpr int FIRST = S - 1 + CONV;
  uint32_t at = 0, at_scale = 0, at_wide = 0, at_held = 0;      // the stage that is computed
#pragma unroll 1
  for (int k = -FIRST;; ++k) {
    if (k >= 0) {
      if (i == todo) {
        if (k > 0) finish();
        if (popped == pushed) break;
        begin();
      }
      arrive(std::integral_constant<int, S - 2>());
    }
    if (step >= steps && more) {
      more = next_piece();
      ask();
    }
    request();
    auto next = [&]() {
      ++step;
      if (step < steps || !more) ask();
    };
    // (a wave without rows, and a group without a unit, only load)
    if (k >= 0 && i * WT + wt < count) {
      scores(cur.unit + i * WT + wt, held >> 2 * at_held & 3,
             CONV ? wide + at_wide * Sh::WIDE : ring + at * RAW, s_scale + 256 * at_scale);
      values(next);
    } else {
      next();
    }
    if (CONV && k >= -1) {
      if (k < 0) arrive(std::integral_constant<int, S - 1>());
      convert();
    }
    if (k >= 0) {
      ++i;
      at = at + 1 == S ? 0 : at + 1;
      at_held = (at_held + 1) & 15;
      if (F8) at_scale = at_scale == S ? 0 : at_scale + 1;
      if (CONV) at_wide ^= 1;
    }
  }
  wave_vm<0>();                              // the last loads write LDS: end them first
  if (SHARES && !joined && tid == 0 && !split.by_block) A.join[worker].last = -1;
}

// Part q's slot of a row block's: a thread's ITEMS times 4 of 16 rows' sums.
template <int D, int AHEAD, class Slot>
__device__ __forceinline__ void tree_join_parts(const TreeArgs& A, int rows, int n, int r0, Slot slot, int R,
                                               int row0, int tok0, int head) {
  constexpr int ITEMS = D / 64;              // 16-byte items of a thread
  const int l = lane_id(), c = l & 15, g = l >> 4;
  float top = -INFINITY, L = 0;
  f32x4 o[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) o[k] = f32x4{0, 0, 0, 0};
  for (int p0 = 0; p0 < n; p0 += AHEAD) {
    float m[AHEAD], s[AHEAD];
    f32x4 x[AHEAD][ITEMS];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {        // past the last: the last again, not added
      const int64_t tile = ((int64_t)slot(min(p0 + k, n - 1)) * rows + r0) / 16;
      const float2 ml = *(const float2*)(A.ml + 2 * (tile * 16 + c));
      m[k] = p0 + k < n ? ml.x : -INFINITY;
      s[k] = ml.y;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) x[k][i] = *((const f32x4*)(A.part + tile * 16 * D) + 256 * i + threadIdx.x);
    }
    float t = top;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) t = fmaxf(t, m[k]);
    const float base = t == -INFINITY ? 0.f : t, f0 = __builtin_amdgcn_exp2f(top - base);
    top = t;
    L *= f0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) o[i] *= f0;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (p0 + k >= n) continue;
      const float f = __builtin_amdgcn_exp2f(m[k] - base);
      L = fmaf(f, s[k], L);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) o[i] += f * x[k][i];
    }
  }
  if (r0 + c >= R) return;
  const float f = top == -INFINITY ? 0.f : 1.f / L;
  const int row = row0 + r0 + c;
  uint16_t* out = A.out + ((int64_t)(tok0 + row / A.G) * A.q_heads + head * A.G + row % A.G) * D + 4 * g;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int d = 16 * (4 * i + wave_id());
    *(u32x2*)(out + d) = u32x2{pack_bf16(o[i][0] * f, o[i][1] * f), pack_bf16(o[i][2] * f, o[i][3] * f)};
  }
}

// AHEAD parts are read at a time: about as many as there are (64 trees in row blocks of 256,
// two or three parts each: 16.7 us, 24 with 8 at all times).
template <int D, class Slot>
__device__ __forceinline__ void tree_join_rows(const TreeArgs& A, int rows, int n, int r0, Slot slot, int R,
                                               int row0, int tok0, int head) {
  if (n <= 2) tree_join_parts<D, 2>(A, rows, n, r0, slot, R, row0, tok0, head);
  else if (n <= 4) tree_join_parts<D, 4>(A, rows, n, r0, slot, R, row0, tok0, head);
  else tree_join_parts<D, 8>(A, rows, n, r0, slot, R, row0, tok0, head);
}

// A row block's parts joined, 16 rows to a workgroup, in the order of their slots: of
// shares, by its entry, ..
template <int D>
__global__ __launch_bounds__(256) void tree_join(TreeArgs A, int rows) {
  const int count = const_load(A.entries);
  const AttendJoin J = const_load(A.join + blockIdx.x);
  const int r0 = 16 * blockIdx.y;
  // (an entry of a call whose lengths change while it runs may not be in range)
  if ((int)blockIdx.x >= count || J.first < 0 || J.last < J.first || J.last >= TREE_WORKERS ||
      r0 >= J.rows || J.rows > rows || J.row0 < 0 || (unsigned)J.head >= (unsigned)A.kv.heads ||
      J.tok0 < 0 || (int64_t)J.row0 + J.rows > (int64_t)(A.kv.T - J.tok0) * A.G)
    return;
  tree_join_rows<D>(A, rows, J.last - J.first + 1, r0, [&](int q) { return 2 * (J.first + q) + (q == 0); },
                    J.rows, J.row0, J.tok0, J.head);
}
// .. or of chunks.
template <int D, class Line>
__global__ __launch_bounds__(256) void tree_join_chunks(TreeArgs A) {
  const AttendSeq s = tree_seq<Line>(A, blockIdx.z);
  const int n = (s.n + A.chunk - 1) / A.chunk, rows = Line::ROWS, r0 = 16 * blockIdx.y;
  const int head = (int)(blockIdx.x % (unsigned)A.kv.heads), rb = (int)(blockIdx.x / (unsigned)A.kv.heads);
  const int row0 = rb * rows, R = min(rows, s.q * A.G - row0);
  if (n < 2 || r0 >= R) return;
  const int slot0 = (((int)blockIdx.z * A.kv.heads + head) * A.tiles + rb) * A.chunks;
  tree_join_rows<D>(A, rows, min(n, A.chunks), r0, [&](int q) { return slot0 + q; }, R, row0, s.tok0, head);
}

// Rows of a row block: the least of those that hold a sequence's on average (32 ragged
// trees of 14 nodes, 4 heads a kv head: 64 us with 64 rows, 70 with 128).  D = 256, e4m3, 2
// heads a kv head, 4 kv heads, with 32 and with 64 rows: 64 requests up to 3000 tokens of 8
// rows a sequence on average 48 and 59, of 26 58 and 57, of 32 69 and 65, of 60 97 and 81;
// 19 up to 6000 of 13 34.5 and 38.4, of 60 50 and 53; four up to 20000, whose few row blocks
// leave the chip to their units' shares, 56 and 69, 41 and 65 of 32, 45 and 63 of 60.
static int tree_rows(int64_t rows, int D, bool f8) {
  if (D == 256) return rows <= 32 && f8 ? 32 : rows <= 64 ? 64 : 128;  // (32 of bf16: the ring passes LDS)
  return rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
}

// Parts that the workspace holds: two a worker, and no fewer of the smaller row blocks.
static int tree_slots(int rows) { return std::max(2 * TREE_WORKERS, 65536 / rows); }

struct TreeWork {
  size_t off_join, off_ml, off_part, total;
};
static TreeWork tree_workspace(int rows, int D) {
  TreeWork x;
  const size_t slots = tree_slots(rows);
  x.off_join = 256;
  x.off_ml = x.off_join + align_up(TREE_WORKERS * sizeof(AttendJoin), 256);
  x.off_part = x.off_ml + align_up(slots * rows * 8, 256);
  x.total = x.off_part + slots * rows * D * 4;
  return x;
}

template <int D, int NT, int WR, bool F8>
static int launch_tree(TreeArgs A, int64_t max_new, hipStream_t s) {
  using Sh = TreeShape<D, NT, WR, F8>;
  constexpr int ROWS = Sh::ROWS;
  const int64_t held = (int64_t)A.kv.M << A.kv.logP;
  const int64_t span = A.window ? std::min<int64_t>(A.window + max_new + TREE_UNIT, held) : held;
  // (a table without columns: one empty chunk, whose rows are 0)
  const int64_t units = std::max<int64_t>((span + TREE_UNIT - 1) / TREE_UNIT, 1);
  const int64_t tiles = (A.G * max_new + ROWS - 1) / ROWS, blocks = A.kv.B * A.kv.heads * tiles;
  // Chunks where the longest context is short for the workgroups that there are ..
  const int64_t most = tree_slots(ROWS) / blocks;               // parts of a row block at most
  int64_t chunks = std::max<int64_t>(std::min({TREE_SPREAD / blocks, most, (units + Sh::WT - 1) / Sh::WT}), 1);
  const int64_t chunk = (units + chunks - 1) / chunks;
  if (chunk <= TREE_CHUNK && blocks <= TREE_BLOCKS) {
    chunks = (units + chunk - 1) / chunk;
    A.tiles = (int)tiles;
    A.chunks = (int)chunks;
    A.chunk = (int)chunk;
    static LdsLimit limit;
    if (int e = limit.raise((const void*)tree_split<D, NT, WR, F8, false>, Sh::lds())) return e;
    timed_launch(CX_KERNEL_TREE, tree_split<D, NT, WR, F8, false>,
                 dim3(A.kv.heads, (unsigned)(tiles * chunks), A.kv.B), dim3(TREE_WG),
                 (uint32_t)Sh::off_seqs(), s, A);
    if (chunks > 1)
      timed_launch(CX_KERNEL_TREE_JOIN, tree_join_chunks<D, typename Sh::Line>,
                   dim3((unsigned)(A.kv.heads * tiles), ROWS / 16, A.kv.B), dim3(256), 0, s, A);
    return (int)hipGetLastError();
  }
  // .. else shares
  static LdsLimit limit;
  if (int e = limit.raise((const void*)tree_split<D, NT, WR, F8, true>, Sh::lds())) return e;
  timed_launch(CX_KERNEL_TREE, tree_split<D, NT, WR, F8, true>, dim3(TREE_WORKERS), dim3(TREE_WG),
               (uint32_t)(Sh::off_seqs() + Sh::Seqs::bytes(A.kv.B, A.kv.q_start != nullptr)), s, A);
  const int64_t entries =
      std::min<int64_t>(A.kv.heads * ((int64_t)A.kv.T * A.G / ROWS + A.kv.B), TREE_WORKERS);
  timed_launch(CX_KERNEL_TREE_JOIN, tree_join<D>, dim3((unsigned)entries, ROWS / 16), dim3(256), 0, s, A, ROWS);
  return (int)hipGetLastError();
}
template <int D, bool F8>
static int launch_tree(const TreeArgs& A, int rows, int64_t max_new, hipStream_t s) {
  if constexpr (D == 256) {
    if constexpr (F8) if (rows == 32) return launch_tree<D, 1, 2, F8>(A, max_new, s);
    if (rows == 64) return launch_tree<D, 1, 4, F8>(A, max_new, s);
    return launch_tree<D, 1, 8, F8>(A, max_new, s);
  } else {
    if (rows == 32) return launch_tree<D, 1, 2, F8>(A, max_new, s);
    if (rows == 64) return launch_tree<D, 1, 4, F8>(A, max_new, s);
    if (rows == 128) return launch_tree<D, 2, 4, F8>(A, max_new, s);
    return launch_tree<D, 2, 8, F8>(A, max_new, s);
  }
}

}  // namespace cx

extern "C" {

size_t cx_tree_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                         int32_t max_new) {
  if (q_heads < 1 || kv_heads < 1 || head_dim < 1 || max_new < 1) return 256;
  // the most of any call of as many rows or fewer
  const int64_t rows = (int64_t)(q_heads / kv_heads) * max_new;
  size_t most = 0;
  for (int64_t r : {32, 64, 128, 256})
    for (bool f8 : {false, true})
      most = std::max(most, cx::tree_workspace(cx::tree_rows(std::min(r, rows), head_dim, f8), head_dim).total);
  return most;
}

int cx_tree_attention_bf16(const cx_kv_batch* kv, const uint16_t* q, int64_t q_token,
                           int64_t q_head, int32_t q_heads, const uint64_t* mask,
                           int32_t mask_words, const int32_t* depth, int32_t max_new,
                           double scale, int32_t window, double softcap, uint16_t* out,
                           void* workspace, size_t ws_bytes, void* stream) {
  cx::TreeArgs A;
  const int rc = cx::kv_args(kv, q_heads, &A.kv);
  if (rc != CX_OK) return rc;
  if (max_new < 1) return cx::api_fail(CX_EINVAL, "max_new must be >= 1");
  if (mask_words < 1 || mask_words > CX_TREE_MAX_WORDS)
    return cx::api_fail(CX_EINVAL, "mask_words (%d) must be 1 .. %d", mask_words, CX_TREE_MAX_WORDS);
  if (window < 0) return cx::api_fail(CX_EINVAL, "window must be >= 0");
  if (!(softcap >= 0)) return cx::api_fail(CX_EINVAL, "softcap must be >= 0");
  if (!(scale > 0)) return cx::api_fail(CX_EINVAL, "scale must be > 0");
  if (kv->T == 0 || kv->B == 0) return CX_OK;
  if (!q || !out || !mask || !workspace) return cx::api_fail(CX_EINVAL, "null pointer argument");
  if (window && !depth) return cx::api_fail(CX_EINVAL, "a window needs the nodes' depths");
  if ((((uintptr_t)q | (uintptr_t)out) & 15) || ((q_token | q_head) & 7))
    return cx::api_fail(CX_EINVAL, "rows must be 16-byte aligned");
  if ((uintptr_t)workspace & 15)
    return cx::api_fail(CX_EINVAL, "workspace must be 16-byte aligned");
  if ((int64_t)kv->T * q_heads > INT32_MAX) return cx::api_fail(CX_EINVAL, "too many rows");
  A.q = q; A.q_token = q_token; A.q_head = q_head;
  A.q_heads = q_heads;
  A.G = q_heads / kv->kv_heads;
  max_new = std::min(max_new, kv->T);        // no sequence has more
  const int D = kv->head_dim;
  const int64_t each = std::min<int64_t>(max_new, (kv->T + kv->B - 1) / kv->B);
  const bool f8 = kv->dtype == CX_KV_E4M3;
  const int rows = cx::tree_rows(A.G * each, D, f8);
  const cx::TreeWork lay = cx::tree_workspace(rows, D);
  if (ws_bytes < lay.total)
    return cx::api_fail(CX_ENOSPACE, "workspace holds %zu bytes, needs %zu", ws_bytes, lay.total);
  // the units and row blocks, at most, fit the share arithmetic's 38 bits
  const double units = (double)kv->max_pages * kv->page_tokens / 32 + 16;
  const double blocks = kv->kv_heads * ((double)kv->T * A.G / 16 + kv->B);
  if (units * blocks >= 0x1p38) return cx::api_fail(CX_EINVAL, "too many tokens for one call");
  A.mask = (const uint32_t*)mask;
  A.words = 2 * mask_words;
  A.depth = depth;
  A.cap = softcap > 0 && !std::isinf(softcap);
  const double log2e = 1.4426950408889634;
  // (0 times a masked score's infinity would be NaN)
  A.s1 = std::max((float)(scale * log2e), std::numeric_limits<float>::min());
  A.s2 = A.cap ? (float)(softcap * log2e) : 0.f;
  A.s3 = A.cap ? (float)(2 * scale / softcap * log2e) : 0.f;
  A.s4 = A.cap ? (float)(scale / softcap) : 0.f;
  if (!std::isfinite(A.s1) || !std::isfinite(A.s2) || !std::isfinite(A.s3))
    return cx::api_fail(CX_EINVAL, "scale (%g) and softcap (%g) pass the range of fp32", scale, softcap);
  A.window = std::min(window, INT32_MAX - cx::KV_MAX_NEW);
  A.out = out;
  A.entries = (int*)workspace;
  A.join = (cx::AttendJoin*)((char*)workspace + lay.off_join);
  A.ml = (float*)((char*)workspace + lay.off_ml);
  A.part = (float*)((char*)workspace + lay.off_part);
  const hipStream_t s = (hipStream_t)stream;
  // one launch after the other where a call has more sequences than a launch takes
  for (int b0 = 0; b0 < kv->B; b0 += cx::TREE_BATCH) {
    cx::TreeArgs X = A;
    X.b0 = b0;
    X.kv.B = std::min(kv->B - b0, cx::TREE_BATCH);
    X.kv.table += b0 * kv->ld_table;
    X.kv.kv_len += b0;
    if (X.kv.q_start) X.kv.q_start += b0;
    const int e = D == 64    ? (f8 ? cx::launch_tree<64, true>(X, rows, max_new, s)
                                   : cx::launch_tree<64, false>(X, rows, max_new, s))
                  : D == 128 ? (f8 ? cx::launch_tree<128, true>(X, rows, max_new, s)
                                   : cx::launch_tree<128, false>(X, rows, max_new, s))
                             : (f8 ? cx::launch_tree<256, true>(X, rows, max_new, s)
                                   : cx::launch_tree<256, false>(X, rows, max_new, s));
    if (e != 0) return cx::api_fail(CX_EHIP, "tree attention launch: %s", hipGetErrorString((hipError_t)e));
  }
  return CX_OK;
}

}  // extern "C"
