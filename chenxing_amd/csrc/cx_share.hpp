// cx_share.hpp -- how a batch's attention is split over its workers (cx_attend.hip).
//
// A sequence's rows (new token, q head of a kv head's group) form row blocks of
// 16 NT for each kv head; a unit is TOK tokens for one row block.  All the batch's
// units lie on one line: sequence by sequence, kv head by head, row block by row
// block, each row block PIECE + its units long, what it costs beside them first.
// Each worker takes an equal stretch of the line, whatever row blocks it cuts.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cx {

// A value that every lane of a wave holds, in a scalar register.
#ifndef CX_UNIFORM
#define CX_UNIFORM(x) __builtin_amdgcn_readfirstlane(x)
#endif

constexpr int ATT_WAVES = 4;
constexpr int ATT_SHARE = 2;                 // the least share, in units
// A sequence's row blocks count as at most one more than the workers, 4096 at most.
constexpr unsigned ATT_COUNTED = 4097;

// What the arithmetic needs of a call.
struct ShareBatch {
  int G, heads;               // q heads per kv head, kv heads
  int window;                 // 0: none
  int held;                   // tokens that a table row's pages hold
};

// A sequence: its rows among the new tokens, the length, and its units (those in
// some row's window).
struct AttendSeq {
  int tok0, q, len, lim, first, n;
};

// A prompt's row blocks, in groups that span NT units of tokens: a group's n units
// are those that its last row may attend to, NT more than those of the group before,
// up to the most that a row's window or the sequence holds.  A sequence of one group
// (decode, verify) has its n.  Any n that holds a row block's units is right.  (All
// the sequence's units for each instead: 4096 new tokens 1015 us, not 446.)  A tree's
// row blocks have all its units.
struct AttendGroups {
  int size, count;                           // row blocks of a group, groups
  int n0, most;                              // units of the first group, of any
};

// Consecutive units of one row block in a worker's share: rows r0 .. r0 + R - 1
// of (new token, q head of the group) of kv head h of sequence b.
struct AttendPiece {
  int b, h, tok0, r0, R, lowest, lim;        // lowest: position of the first new token
  int unit, cnt;
  int slot;                                  // of its part, -1: the whole row block
};

// A row block whose units lie in several workers' shares: those of workers
// first .. last (last = -1: in one).  Written by the first; there is an entry for
// every row block, in their order, or, where they are more than the workers, for
// every worker.
struct AttendJoin {
  int first, last;
  int tok0, row0, rows, head;
  int pad[2];
};

// The line's length and its row blocks, of the batch or of the sequences before
// one: units above, row blocks below, in one word that sums both.
constexpr int RB = 25;
__device__ __forceinline__ uint64_t line_units(uint64_t x) { return x >> RB; }
__device__ __forceinline__ unsigned line_blocks(uint64_t x) {
  return (unsigned)(x & ((1u << RB) - 1));
}

// The line's split over the workers: shares of ``least`` units at least, the first
// ones a unit longer.
struct ShareSplit {
  bool by_block;              // a join entry for every row block
  uint64_t shares, per, more;
};
__device__ __forceinline__ ShareSplit share_split(uint64_t line, unsigned workers,
                                                  unsigned least = ATT_SHARE) {
  ShareSplit s;
  const uint64_t total = line_units(line);
  s.by_block = line_blocks(line) <= workers;
  s.shares = min((uint64_t)workers, (total + least - 1) / least);
  s.per = s.shares ? total / s.shares : 0;
  s.more = total - s.per * s.shares;
  return s;
}
// A share's first unit, and the worker that holds unit u.
__device__ __forceinline__ uint64_t share_begin(const ShareSplit& s, unsigned worker) {
  return worker * s.per + min((uint64_t)worker, s.more);
}
__device__ __forceinline__ int share_of(const ShareSplit& s, uint64_t u) {
  const uint64_t cut = s.more * (s.per + 1);
  return (int)(u < cut ? u / (s.per + 1) : s.more + (u - cut) / s.per);
}

// The sequences as one workgroup sees them.  They are read once: the lengths may
// change while the call runs (a graph's next inputs written too early), and a piece
// is in range only by the values that made its place on the line.
template <class Word, class Int>
struct AttendSeqs {
  Word line;                  // [B + 1] the line before each sequence
  Int len;                    // [B]
  Int start;                  // [B + 1] first rows; starts = false: one row each
  bool starts;

  // Bytes of the three, in this order.
  static constexpr int bytes(int B, bool starts) {
    return 8 * (B + 1) + 4 * B + (starts ? 4 * (B + 1) : 0);
  }
  // Thread tid's part of lengths and first rows, whatever q_start holds.
  __device__ __forceinline__ void read(const int32_t* kv_len, const int32_t* q_start, int B, int T,
                                       int tid, int threads) const {
    for (int b = tid; b <= B; b += threads) {
      if (b < B) len[b] = kv_len[b];
      if (starts) start[b] = min(max(q_start[b], 0), T);
    }
  }
  __device__ __forceinline__ int first(int b) const { return starts ? (int)start[b] : b; }
  __device__ __forceinline__ int end(int b) const {
    return starts ? max((int)start[b + 1], (int)start[b]) : b + 1;
  }
};

// TREE: new tokens may attend to any of the others.
template <int TOK, int NT, bool TREE = false>
struct AttendLine {
  static constexpr int ROWS = 16 * NT;
  // what a row block costs beside its units, in units (64 ragged requests 99, 94
  // and 93 us with 0, 1 and 2; 32 verify rounds 48, 42, 39 and 35 us with 0 .. 3).  Trees,
  // whose workgroups take a unit or more a step: 32 ragged ones 84, 64, 55, 54 and 58 us
  // with 2, 4, 6, 9 and 14, 64 full ones in row blocks of 256 484, 456, 439, 443 and 459.
  // Ragged ones of 1 .. 64 nodes with 4, 9 and 16: 8 up to 4096 tokens 40 in each, 32 of them
  // 84, 65 and 69, 16 up to 16000 126, 118 and 119, 100 up to 1500 114, 103 and 102
  static constexpr int PIECE = TREE ? (NT < 16 ? 9 : 6) : NT == 1 ? 2 : 4;

  // The sequence of new tokens tok0 .. end - 1 and len tokens in all.
  static __device__ __forceinline__ AttendSeq seq(const ShareBatch& A, int tok0, int end, int len) {
    AttendSeq s;
    s.tok0 = tok0;
    s.q = end - tok0;
    s.len = max(len, 0);                     // no position is reached by a shorter one
    s.lim = min(s.len, A.held);
    const int lowest = s.len - s.q;
    s.first = A.window && lowest >= A.window ? (lowest - A.window + 1) / TOK : 0;
    s.n = s.q > 0 ? max((s.lim + TOK - 1) / TOK - s.first, 0) : 0;
    return s;
  }
  static __device__ __forceinline__ int row_blocks(const ShareBatch& A, const AttendSeq& s) {
    return (s.q * A.G + ROWS - 1) / ROWS;
  }
  static __device__ __forceinline__ AttendGroups groups(const ShareBatch& A, const AttendSeq& s,
                                                        int blocks) {
    AttendGroups g;
    g.size = A.G * (TOK / 16);
    g.count = (blocks + g.size - 1) / g.size;
    if (TREE) {
      g.size = blocks;
      g.count = 1;
    }
    g.n0 = g.most = s.n;
    const int lowest = s.len - s.q;
    if (g.count > 1 && lowest >= 0) {
      g.n0 = min((int)(((unsigned)lowest + TOK - 1) / TOK) + NT - s.first, s.n);
      if (A.window) g.most = s.first > 0 ? g.n0 : min(s.n, A.window / TOK + NT + 3);
      g.n0 = min(g.n0, g.most);
    }
    return g;
  }
  // What the row blocks of the groups before the j-th cost, / size.
  static __device__ __forceinline__ uint64_t before(const AttendGroups& g, int j) {
    const int i = min(j, (g.most - g.n0 + NT - 1) / NT);
    return (uint64_t)i * (g.n0 + PIECE) + (uint64_t)i * (i - 1) / 2 * NT +
           (uint64_t)(j - i) * (g.most + PIECE);
  }
  // What a head's row blocks cost.
  static __device__ __forceinline__ uint64_t head_cost(const AttendGroups& g, int blocks) {
    const int j = g.count - 1;
    return before(g, j) * g.size +
           (uint64_t)(blocks - j * g.size) * (min(g.n0 + NT * j, g.most) + PIECE);
  }
  // A sequence's part of the line, as line_units and line_blocks read it.
  static __device__ __forceinline__ uint64_t length(const ShareBatch& A, const AttendSeq& s) {
    if (s.n <= 0) return 0;
    const int blocks = row_blocks(A, s);
    return head_cost(groups(A, s, blocks), blocks) * A.heads << RB |
           min((uint64_t)A.heads * blocks, (uint64_t)ATT_COUNTED);
  }

  // The piece of worker's share that begins at u, of sequence b, whose part of the
  // line begins at line; u moves past it.  A share may end before a row block's
  // first unit (cnt = 0).  enter(entry, join) where the piece is the first of a row
  // block that has an entry.
  template <class Enter>
  static __device__ __forceinline__ AttendPiece piece(const ShareBatch& A, const AttendSeq& s, int b,
                                                      uint64_t line, const ShareSplit& split,
                                                      unsigned worker, uint64_t end, uint64_t& u,
                                                      Enter enter) {
    AttendPiece p;
    uint64_t rem = u - line_units(line);
    rem = (uint64_t)(uint32_t)CX_UNIFORM((int)rem) |
          (uint64_t)(uint32_t)CX_UNIFORM((int)(rem >> 32)) << 32;
    const int blocks = row_blocks(A, s);
    const AttendGroups g = groups(A, s, blocks);
    int n = s.n, first = s.first;
    unsigned row;                            // of the sequence's row blocks by head
    int at;                                  // place in it
    if (g.count == 1) {
      const unsigned cost = n + PIECE;
      row = rem >> 32 ? (unsigned)(rem / cost) : (unsigned)rem / cost;
      at = (int)(rem - (uint64_t)row * cost);
    } else {
      const uint64_t head = head_cost(g, blocks);
      const unsigned h = (unsigned)(rem / head);
      uint64_t r = rem - h * head;
      int j = 0;
      for (int hi = g.count - 1; j < hi;) {
        const int mid = (j + hi + 1) >> 1;
        if (before(g, mid) * g.size <= r) j = mid;
        else hi = mid - 1;
      }
      r -= before(g, j) * g.size;
      n = min(g.n0 + NT * j, g.most);
      if (A.window) first = max(s.len - s.q + j * NT * TOK - A.window + 1, 0) / TOK;
      const unsigned cost = n + PIECE, i = r >> 32 ? (unsigned)(r / cost) : (unsigned)r / cost;
      row = h * (unsigned)blocks + j * g.size + i;
      at = (int)(r - (uint64_t)i * cost);
    }
    const unsigned cost = n + PIECE;
    const int ua = max(at - PIECE, 0);
    const int64_t room = (int64_t)(end - u) - max(PIECE - at, 0);
    p.b = b;
    p.h = CX_UNIFORM((int)(row / (unsigned)blocks));
    p.tok0 = s.tok0;
    p.r0 = CX_UNIFORM((int)(row % (unsigned)blocks)) * ROWS;
    p.R = min(ROWS, s.q * A.G - p.r0);
    p.lowest = s.len - s.q;
    p.lim = s.lim;
    p.unit = CX_UNIFORM(first + ua);
    p.cnt = CX_UNIFORM((int)min((int64_t)(n - ua), max(room, (int64_t)0)));
    p.slot = ua == 0 && p.cnt == n ? -1 : (int)(2 * worker + (ua == 0));
    p.slot = CX_UNIFORM(p.slot);
    if (ua == 0 && p.cnt > 0 && (split.by_block || p.cnt < n)) {
      AttendJoin J;
      J.first = (int)worker;
      J.last = p.cnt == n ? -1 : share_of(split, u - at + cost - 1);
      J.tok0 = p.tok0;
      J.row0 = p.r0;
      J.rows = p.R;
      J.head = p.h;
      J.pad[0] = J.pad[1] = 0;
      enter(split.by_block ? line_blocks(line) + row : worker, J);
    }
    u = p.cnt > 0 ? u + max(PIECE - at, 0) + p.cnt : end;
    return p;
  }
};

}  // namespace cx
