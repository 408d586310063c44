// cx_kv.hip -- the paged KV cache, for gfx950: new tokens normed, rotated and
// appended, pages copied (layout: cx_kv.hpp).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "cx_device.hpp"
#include "cx_internal.hpp"
#include "cx_kv.hpp"
#include "cx_sampler.h"
#include "cx_timing.hpp"

namespace cx {

int kv_args(const cx_kv_batch* kv, int q_heads, KvArgs* out) {
  if (!kv) return api_fail(CX_EINVAL, "null pointer argument");
  const int P = kv->page_tokens, D = kv->head_dim;
  if (kv->B < 0 || kv->T < 0 || kv->n_pages < 0 || kv->max_pages < 0 || kv->kv_heads < 1 ||
      kv->ld_table < kv->max_pages)
    return api_fail(CX_EINVAL, "bad shape");
  if (kv->T > KV_MAX_NEW) return api_fail(CX_EINVAL, "too many new tokens (%d)", kv->T);
  if (kv->B > CX_KV_MAX_BATCH)
    return api_fail(CX_EINVAL, "a call takes at most %d sequences (%d)", CX_KV_MAX_BATCH, kv->B);
  if (D != 64 && D != 128 && D != 256)
    return api_fail(CX_EINVAL, "head_dim (%d) must be 64, 128 or 256", D);
  if (P < 16 || P > 256 || (P & (P - 1)))
    return api_fail(CX_EINVAL, "page_tokens (%d) must be 16, 32, 64, 128 or 256", P);
  if (kv->dtype != CX_KV_BF16 && kv->dtype != CX_KV_E4M3)
    return api_fail(CX_EINVAL, "unknown cache dtype %d", kv->dtype);
  if (q_heads < 1 || q_heads % kv->kv_heads)
    return api_fail(CX_EINVAL, "q_heads (%d) must be a multiple of kv_heads (%d)", q_heads,
                    kv->kv_heads);
  if (!kv->q_start && kv->T != kv->B)
    return api_fail(CX_EINVAL, "without q_start there is one new token per sequence");
  const int64_t head = kv_head_bytes(D, P, kv->dtype);
  if (kv->page_stride % 16 || kv->page_stride < head * kv->kv_heads || ((uintptr_t)kv->pages & 15))
    return api_fail(CX_EINVAL, "pages must be 16-byte aligned and hold every head's part");
  if ((int64_t)kv->max_pages * P > INT32_MAX - 4096)
    return api_fail(CX_EINVAL, "a table row of %d pages passes 2^31 tokens", kv->max_pages);
  if (kv->B && (!kv->kv_len || (kv->max_pages && !kv->table) || (kv->n_pages && !kv->pages)))
    return api_fail(CX_EINVAL, "null pointer argument");
  out->pages = (char*)kv->pages;
  out->page_stride = kv->page_stride;
  out->table = kv->table;
  out->ld_table = kv->ld_table;
  out->kv_len = kv->kv_len;
  out->q_start = kv->q_start;
  out->n_pages = kv->n_pages;
  out->heads = kv->kv_heads;
  out->B = kv->B;
  out->M = kv->max_pages;
  out->T = kv->T;
  out->logP = __builtin_ctz(P);
  out->head_bytes = (int)head;
  return CX_OK;
}

struct AppendArgs {
  KvArgs kv;
  const uint16_t* x[3];       // q, k, v
  int64_t st[3], sh[3];       // elements from token to token, from head to head
  int q_heads;
  const float* rope;          // nullable [rope_rows, rdim]
  int rdim;
  int interleaved;
  const uint16_t* norm[2];    // nullable: q, k
  const int32_t* depth;       // nullable: positions from the first new one
  float eps;
  uint16_t* q_out;
};

// The sequence of new token t, its position and its sequence's first new one: the last
// b with q_start[b] <= t.  -1 for a token outside every sequence.
__device__ __forceinline__ int3 token_place(const KvArgs& A, int t) {
  int b = t, i = 0, n = 1;
  if (A.q_start) {
    int lo = 0, hi = A.B;                     // first b with q_start[b + 1] > t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (A.q_start[mid + 1] > t) hi = mid;
      else lo = mid + 1;
    }
    if (lo >= A.B) return make_int3(-1, -1, -1);
    b = lo;
    const int2 r = kv_rows(A, b);
    i = t - r.x;
    n = r.y - r.x;
  }
  const unsigned first = A.kv_len[b] - (unsigned)n;
  return make_int3(b, (int)(first + (unsigned)i), (int)first);
}

// A row's lane of 8 dims, d .., as floats.
struct Row8 {
  float x[8];
};
__device__ __forceinline__ Row8 widen(u32x4 in) {
  Row8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) { r.x[2 * i] = bf16_lo(in[i]); r.x[2 * i + 1] = bf16_hi(in[i]); }
  return r;
}

// A reduction over the D / 8 lanes of a row, in every one of them: neighbours,
// pairs, quads of a half row, half rows, and for 32 lanes the two rows.
template <int D, typename T, typename Op>
__device__ __forceinline__ T lanes_reduce(T v, Op op) {
  auto dpp = [](T x, auto ctrl) {
    return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x),
                                                          decltype(ctrl)::value, 0xF, 0xF, false));
  };
  v = op(v, dpp(v, std::integral_constant<int, 0xB1>()));    // quad_perm 1 0 3 2
  v = op(v, dpp(v, std::integral_constant<int, 0x4E>()));    // quad_perm 2 3 0 1
  v = op(v, dpp(v, std::integral_constant<int, 0x141>()));   // row_half_mirror
  if (D >= 128) v = op(v, dpp(v, std::integral_constant<int, 0x140>()));   // row_mirror
  if (D == 256) v = op(v, __shfl_xor(v, 16));
  return v;
}

// x * rsqrt(mean(x^2) + eps) * w over the row's D / 8 lanes; the root by v_rsq, within
// 1 ulp: with the sum's roundings it is not what the result's error comes from.
template <int D>
__device__ __forceinline__ void norm_row(Row8& r, u32x4 w, float eps) {
  float ss = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(r.x[i], r.x[i], ss);
  ss = lanes_reduce<D>(ss, [](float a, float b) { return a + b; });
  const float f = __builtin_amdgcn_rsqf(ss * (1.f / D) + eps);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.x[2 * i] = r.x[2 * i] * f * bf16_lo(w[i]);
    r.x[2 * i + 1] = r.x[2 * i + 1] * f * bf16_hi(w[i]);
  }
}

// The cosines and sines of a lane's pairs at one position: of dims d, d + 2 ..
// where the pair (2 j, 2 j + 1) is in the lane, of dims d .. d + 7 where it is
// (j, j + rdim / 2), rdim / 16 lanes away.
struct Turn8 {
  f32x4 c[2], s[2];
};
__device__ __forceinline__ Turn8 load_turn(const AppendArgs& A, int pos, int d) {
  Turn8 t = {};
  if (!A.rope || d >= A.rdim) return t;
  const int half = A.rdim / 2;
  const float* p = A.rope + (int64_t)pos * A.rdim +
                   (A.interleaved ? d / 2 : d < half ? d : d - half);
  t.c[0] = *(const f32x4*)p;
  t.s[0] = *(const f32x4*)(p + half);
  if (!A.interleaved) {
    t.c[1] = *(const f32x4*)(p + 4);
    t.s[1] = *(const f32x4*)(p + half + 4);
  }
  return t;
}
__device__ __forceinline__ void turn_row(const AppendArgs& A, Row8& r, const Turn8& t, int d) {
  if (!A.rope) return;
  if (A.interleaved) {
    if (d >= A.rdim) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = r.x[2 * i], b = r.x[2 * i + 1];
      r.x[2 * i] = fmaf(a, t.c[0][i], -(b * t.s[0][i]));
      r.x[2 * i + 1] = fmaf(b, t.c[0][i], a * t.s[0][i]);
    }
    return;
  }
  const int half = A.rdim / 2;
  const bool low = d < half;
  const int other = (threadIdx.x + (low ? half / 8 : -(half / 8))) & 63;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = __shfl(r.x[i], other), c = t.c[i / 4][i % 4], s = t.s[i / 4][i % 4];
    if (d < A.rdim) r.x[i] = fmaf(r.x[i], c, low ? -(y * s) : y * s);
  }
}
__device__ __forceinline__ u32x4 narrow(const Row8& r) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack_bf16(r.x[2 * i], r.x[2 * i + 1]);
  return o;
}

// A lane's 8 e4m3 codes and the row's scale; the largest |x| by its bits: NaN
// above inf above every number.
template <int D>
__device__ __forceinline__ u32x2 encode_row(const Row8& r, float* scale) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(r.x[i]) & 0x7FFFFFFFu);
  m = lanes_reduce<D>(m, [](uint32_t a, uint32_t b) { return max(a, b); });
  const bool fine = m < 0x7F800000u;
  // Quotients as a division rounds them (but perhaps for ties among denormal scales):
  // times a reciprocal, less what that is too much times it (in this order a zero
  // keeps its sign).  A scale too small for that (below 2^-126 it has no finite
  // reciprocal) is taken 2^80 times as large, as is x.
  auto quotient = [](float x, float f, float inv) {
    const float a = x * inv;
    return fmaf(-fmaf(a, f, -x), inv, a);
  };
  float f = quotient(__uint_as_float(m), E4M3_MAX, 1.f / E4M3_MAX);
  if (f == 0.f) f = 1.f;                     // a row of zeros, or of values whose scale rounds to 0
  *scale = fine ? f : __builtin_nanf("");
  const float by = f < 0x1p-60f ? 0x1p80f : 1.f, fs = f * by;
  float inv = __builtin_amdgcn_rcpf(fs);
  inv = fmaf(fmaf(-inv, fs, 1.f), inv, inv);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = __builtin_amdgcn_fmed3f(quotient(r.x[i] * by, fs, inv), -E4M3_MAX, E4M3_MAX);
  }
  u32x2 c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
    c[i] = fine ? __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], p, true) : 0;
  }
  return c;
}

// Where a new token goes: byte offset of its page (-1: nowhere) and its place
// in the page; pos: the position that it is rotated to.
struct Slot {
  int64_t page;
  int o, pos;
};
__device__ __forceinline__ Slot token_slot(const KvArgs& C, int t, const int32_t* depth) {
  const int3 at = token_place(C, t);
  Slot s = {-1, 0, 0};
  const int held = C.M << C.logP;
  if (at.x < 0 || at.y < 0 || at.y >= held) return s;
  s.pos = at.y;
  // (the sum in 64 bits: depths are the caller's)
  if (depth) s.pos = (int)min(max((int64_t)at.z + depth[t], (int64_t)0), (int64_t)held - 1);
  s.o = at.y & ((1 << C.logP) - 1);
  const int id = C.table[at.x * C.ld_table + (at.y >> C.logP)];
  if ((unsigned)id < (unsigned)C.n_pages) s.page = id * C.page_stride;
  return s;
}

// A lane's part of a row as the page holds it: 8 elements of bf16, or 8 e4m3 codes
// and the row's scale.
struct Part {
  u32x4 w;
  float scale;
};
template <int D, bool F8>
__device__ __forceinline__ Part page_part(const Row8& r) {
  Part p = {};
  if (F8) {
    const u32x2 c = encode_row<D>(r, &p.scale);
    p.w = u32x4{c[0], c[1], 0, 0};
  } else {
    p.w = narrow(r);
  }
  return p;
}
// A lane's part of a key row, to its page.
template <int D, bool F8>
__device__ __forceinline__ void put_key(const KvArgs& C, const Part& p, const Slot& s, int h, int d) {
  if (s.page < 0) return;
  char* base = C.pages + s.page + (int64_t)h * C.head_bytes;
  if (F8) {
    *(u32x2*)(base + k_chunk<16>(d, s.o, C.logP) + (d & 8)) = u32x2{p.w[0], p.w[1]};
    if (d == 0) *(float*)(base + k_scale<D>(s.o, C.logP)) = p.scale;
  } else {
    *(u32x4*)(base + k_chunk<8>(d, s.o, C.logP)) = p.w;
  }
}

// One row (token, head) of q, k or v to D / 8 lanes, every row of the call at
// once: q heads first, then k, then v.  A small call is one latency, launch and
// loads (1 token, 48 heads of 128: 3.7 us); a row's v leaves as one element a chunk,
// so in a large one the stores bound it (256 tokens of as many sequences 6.9 us, 256
// prompts of 64 tokens 251 us).
template <int D, bool F8>
__global__ __launch_bounds__(256) void append_rows(AppendArgs A) {
  constexpr int LR = D / 8, E = F8 ? 16 : 8;
  const KvArgs& C = A.kv;
  const unsigned heads = A.q_heads + 2 * C.heads;
  const unsigned row = blockIdx.x * (256 / LR) + threadIdx.x / LR;
  const int t = (int)(row / heads), hh = (int)(row % heads);
  if (t >= C.T) return;
  const int d = 8 * (threadIdx.x % LR);
  const int kind = hh < A.q_heads ? 0 : hh < A.q_heads + C.heads ? 1 : 2;
  const int h = kind == 0 ? hh : kind == 1 ? hh - A.q_heads : hh - A.q_heads - C.heads;
  const u32x4 in = *(const u32x4*)(A.x[kind] + t * A.st[kind] + h * A.sh[kind] + d);
  const uint16_t* w = kind < 2 ? A.norm[kind] : nullptr;
  u32x4 wv = {};
  if (w) wv = *(const u32x4*)(w + d);
  const Slot s = token_slot(C, t, A.depth);
  Row8 r = widen(in);
  if (kind < 2) {
    const Turn8 turn = load_turn(A, s.pos, d);
    if (w) norm_row<D>(r, wv, A.eps);
    turn_row(A, r, turn, d);
  }
  if (kind == 0) {
    *(u32x4*)(A.q_out + ((int64_t)t * A.q_heads + h) * D + d) = narrow(r);
    return;
  }
  Part y = page_part<D, F8>(r);
  if (kind == 1) {
    put_key<D, F8>(C, y, s, h, d);
    return;
  }
  if (s.page < 0) return;
  if (!F8) y.w = in;                         // as it came, NaN's bits too
  char* base = C.pages + s.page + (int64_t)h * C.head_bytes;
  char* p = base + v_chunk<E, D>(d, s.o, C.logP) + s.o % E * (16 / E);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (F8) *(uint8_t*)(p + 16 * i) = (uint8_t)(y.w[i / 4] >> 8 * (i % 4));
    else *(uint16_t*)(p + 16 * i) = (uint16_t)(y.w[i / 2] >> 16 * (i % 2));
  }
  if (F8 && d == 0) *(float*)(base + v_scale<D>(s.o, C.logP)) = y.scale;
}

// Prompts: neighbouring tokens share lines of the pages, so a workgroup takes
// neighbouring tokens (lines written in part by several XCDs go to memory in
// part, from each).
//
//  * Workgroups 0 .. qk - 1: 2048 / D tokens (a row of D / 8 lanes each) by
//    APPEND_HEADS heads of q or k, one after the other with the next one's row
//    requested; a token's cosines and sines are read once for them.
//  * The others: VT tokens of one head of v.  They pass through LDS, and the
//    tokens of a chunk that are all here leave as 16 bytes a dim.
//
// Bound: HBM.  5 prompts of 2500 tokens, 48 heads of 128, e4m3: 217 MB in 52 us,
// 4.2 TB/s where a copy reaches 4.75 (append_rows 125 us); bf16: 219 MB in 47 us.
constexpr int APPEND_HEADS = 8, APPEND_VT = 64;

template <int D, bool F8>
__global__ __launch_bounds__(256) void append_tiles(AppendArgs A, int qk, int groups) {
  constexpr int LR = D / 8, TT = 256 / LR, E = F8 ? 16 : 8, VT = APPEND_VT;
  constexpr int EL = F8 ? 1 : 2, PITCH = D * EL + 4;     // bytes of a token's row in LDS
  __shared__ __align__(16) char s_v[VT * PITCH];
  __shared__ int64_t s_page[VT];
  __shared__ int s_o[VT], s_run[VT], s_runs;
  const KvArgs& C = A.kv;
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < qk) {
    const int t = (int)(blockIdx.x / (unsigned)groups) * TT + tid / LR, d = 8 * (tid % LR);
    const int h0 = (int)(blockIdx.x % (unsigned)groups) * APPEND_HEADS;
    const int heads = A.q_heads + C.heads, end = min(h0 + APPEND_HEADS, heads);
    if (t >= C.T) return;
    auto load = [&](int hh) {
      const bool q = hh < A.q_heads;
      return *(const u32x4*)(q ? A.x[0] + t * A.st[0] + hh * A.sh[0] + d
                               : A.x[1] + t * A.st[1] + (hh - A.q_heads) * A.sh[1] + d);
    };
    u32x4 next = load(h0);
    u32x4 wq = {}, wk = {};
    if (A.norm[0]) wq = *(const u32x4*)(A.norm[0] + d);
    if (A.norm[1]) wk = *(const u32x4*)(A.norm[1] + d);
    const Slot s = token_slot(C, t, A.depth);
    const Turn8 turn = load_turn(A, s.pos, d);
    for (int hh = h0; hh < end; ++hh) {
      Row8 r = widen(next);
      if (hh + 1 < end) next = load(hh + 1);
      const bool q = hh < A.q_heads;
      if (A.norm[q ? 0 : 1]) norm_row<D>(r, q ? wq : wk, A.eps);
      turn_row(A, r, turn, d);
      if (q) *(u32x4*)(A.q_out + ((int64_t)t * A.q_heads + hh) * D + d) = narrow(r);
      else put_key<D, F8>(C, page_part<D, F8>(r), s, hh - A.q_heads, d);
    }
    return;
  }
  const unsigned v = blockIdx.x - (unsigned)qk;
  const int t0 = (int)(v / (unsigned)C.heads) * VT, h = (int)(v % (unsigned)C.heads);
  const int n = min(VT, C.T - t0);
  if (tid < VT) {                            // one wave
    Slot s = {-1, 0, 0};
    if (tid < n) s = token_slot(C, t0 + tid, nullptr);
    // runs: neighbouring tokens that go to neighbouring places of one chunk
    const int64_t before = __shfl_up(s.page, 1);
    const int at = __shfl_up(s.o, 1);
    const bool in = s.page >= 0;
    const bool first = in && (tid == 0 || s.page != before || s.o != at + 1 || s.o % E == 0);
    const uint64_t starts = ballot(first), breaks = starts | ~ballot(in);
    if (first) {
      const uint64_t later = tid < 63 ? breaks >> (tid + 1) : 0;
      const int len = later ? __builtin_ctzll(later) + 1 : 64 - tid;
      s_run[lanes_below(starts)] = tid | len << 8;
    }
    s_page[tid] = s.page;
    s_o[tid] = s.o;
    if (tid == 0) s_runs = __builtin_popcountll(starts);
  }
  constexpr int LOADS = VT * LR / 256;
  u32x4 in[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int r = min(i * TT + tid / LR, n - 1);
    in[i] = *(const u32x4*)(A.x[2] + (t0 + r) * A.st[2] + h * A.sh[2] + 8 * (tid % LR));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int r = i * TT + tid / LR, d = 8 * (tid % LR);
    uint32_t* p = (uint32_t*)(s_v + r * PITCH + d * EL);
    if (F8) {
      float scale;
      const u32x2 c = encode_row<D>(widen(in[i]), &scale);
      p[0] = c[0];
      p[1] = c[1];
      if (d == 0 && r < n && s_page[r] >= 0)
        *(float*)(C.pages + s_page[r] + (int64_t)h * C.head_bytes + v_scale<D>(s_o[r], C.logP)) = scale;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) p[k] = in[i][k];
    }
  }
  __syncthreads();
  // (run, 4 / EL dims) to a thread: a dword of each token's row
  constexpr int DW = D * EL / 4;             // dwords of a row
  for (int i = tid; i < s_runs * DW; i += 256) {
    const int run = s_run[i / DW], j = run & 255, len = run >> 8, dw = i % DW;
    const int d = dw * (4 / EL), o = s_o[j];
    char* base = C.pages + s_page[j] + (int64_t)h * C.head_bytes;
    auto word = [&](int k) { return *(const uint32_t*)(s_v + (j + k) * PITCH + 4 * dw); };
    if (len == E) {
      uint32_t x[E];
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] = word(k);
#pragma unroll
      for (int e = 0; e < 4 / EL; ++e) {     // element e of each dword, token by token
        u32x4 y;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (F8) {
            const uint32_t sel = 0x0C0C0400u + 0x0101u * e;      // byte e of two words
            const uint32_t a = __builtin_amdgcn_perm(x[(4 * k + 1) % E], x[4 * k % E], sel);
            const uint32_t b = __builtin_amdgcn_perm(x[(4 * k + 3) % E], x[(4 * k + 2) % E], sel);
            y[k] = a | b << 16;
          } else {
            y[k] = __builtin_amdgcn_perm(x[2 * k + 1], x[2 * k], e ? 0x07060302u : 0x05040100u);
          }
        }
        *(u32x4*)(base + v_chunk<E, D>(d + e, o, C.logP)) = y;
      }
    } else {
      for (int k = 0; k < len; ++k) {
        const uint32_t x = word(k);
        char* p = base + v_chunk<E, D>(d, o + k, C.logP) + (o + k) % E * EL;
#pragma unroll
        for (int e = 0; e < 4 / EL; ++e) {
          if (F8) *(uint8_t*)(p + 16 * e) = (uint8_t)(x >> 8 * e);
          else *(uint16_t*)(p + 16 * e) = (uint16_t)(x >> 16 * e);
        }
      }
    }
  }
}

struct CopyArgs {
  char* pages;
  int64_t layer_stride, page_stride, page_bytes;
  int n_layers, n_pages, parts;
  const int32_t* src;
  const int32_t* dst;
};

__device__ __forceinline__ u32x4 ld_copy(const char* p) { return *(const u32x4*)p; }
__device__ __forceinline__ void st_copy(char* p, u32x4 v) { __builtin_nontemporal_store(v, (u32x4*)p); }

constexpr int COPY_LOADS = 8;                // 16-byte loads of a thread, all in flight
constexpr int COPY_PART = COPY_LOADS * 4096; // bytes a workgroup copies

// Workgroup (pair, layer, part): COPY_PART bytes of the page.  Bound: HBM.  400
// pages of 64 KB in 32 layers, 1.68 GB read and written: 334 us, 5.0 TB/s (plain
// stores 343); 16 such pages, 67 MB: 7.1 us (plain stores 9.2, loads past the caches
// 10.6).
__global__ __launch_bounds__(256) void copy_pages(CopyArgs A) {
  const unsigned part = blockIdx.x % (unsigned)A.parts, x = blockIdx.x / (unsigned)A.parts;
  const unsigned layer = x % (unsigned)A.n_layers, pair = x / (unsigned)A.n_layers;
  const int s = A.src[pair], d = A.dst[pair];
  if ((unsigned)s >= (unsigned)A.n_pages || (unsigned)d >= (unsigned)A.n_pages) return;
  char* base = A.pages + layer * A.layer_stride;
  const int64_t at = (int64_t)part * COPY_PART + threadIdx.x * 16;
  const char* from = base + s * A.page_stride + at;
  char* to = base + d * A.page_stride + at;
  const int64_t left = A.page_bytes - at;
  u32x4 v[COPY_LOADS];
  if (left > (COPY_LOADS - 1) * 4096) {
#pragma unroll
    for (int i = 0; i < COPY_LOADS; ++i) v[i] = ld_copy(from + i * 4096);
#pragma unroll
    for (int i = 0; i < COPY_LOADS; ++i) st_copy(to + i * 4096, v[i]);
  } else {
    for (int i = 0; i * 4096 < left; ++i) st_copy(to + i * 4096, ld_copy(from + i * 4096));
  }
}

struct CommitArgs {
  KvArgs kv;
  int64_t layer_stride;
  int n_layers, width, heads; // heads of a workgroup
  int32_t* path;              // [B, width]
  const int32_t* count;       // nullable [B]
};
constexpr int COMMIT_PASS = 32;              // moves looked up at a time
constexpr int COMMIT_AHEAD = 8;              // and read before any of them is written
constexpr int COMMIT_GROUPS = 2048;          // workgroups that a call should have

// Workgroup (sequence, layer, a few heads): a thread a 16-byte chunk of the keys, a dim of
// the values, or a scale.  A token's values are 16 bytes apart and its chunks of keys 16 P:
// bound by the lines that hold them (48 sequences of 32 layers and 8 heads, e4m3: 23 MB of
// tokens, 112 MB of lines, 43 us from memory, 31 where the pool's lines are in the caches;
// there reads and writes in turn take 36, a head a workgroup 36; one sequence 4.3 us).
template <int D, bool F8>
__global__ __launch_bounds__(256) void commit_tokens(CommitArgs A) {
  constexpr int E = F8 ? 16 : 8, KC = D / E, ITEMS = KC + D + (F8 ? 2 : 0);
  __shared__ int64_t s_from[COMMIT_PASS], s_to[COMMIT_PASS];             // pages, in bytes
  __shared__ int s_slot[COMMIT_PASS], s_moves[2];                        // slots: from << 16 | to
  const KvArgs& C = A.kv;
  const unsigned parts = (C.heads + A.heads - 1) / A.heads, x = blockIdx.x / parts;
  const int h0 = (int)(blockIdx.x % parts) * A.heads, nh = min(A.heads, C.heads - h0);
  const int b = (int)(x / (unsigned)A.n_layers);
  const int2 rows = kv_rows(C, b);
  const int n = rows.y - rows.x, P = 1 << C.logP;
  const int64_t s0 = (int64_t)C.kv_len[b] - n;
  if (s0 < 0) return;
  char* const base = C.pages + (x % (unsigned)A.n_layers) * A.layer_stride + (int64_t)h0 * C.head_bytes;
  int32_t* path = A.path + (int64_t)b * A.width;
  const int m = A.count ? min(A.count[b], A.width) : A.width;
  for (int j0 = 0; j0 < m; j0 += COMMIT_PASS) {
    // the pass's moves: the first wave looks them up, side by side
    if (wave_id() == 0) {
      const int j = j0 + lane_id();
      const int p = lane_id() < COMMIT_PASS && j < m ? path[j] : -1;
      const int before = j > 0 && p >= 0 ? path[j - 1] : -1;
      const uint64_t ends = ballot(p <= before || p >= n);
      const int end = ends ? __builtin_ctzll(ends) : 64;                 // COMMIT_PASS at most
      int64_t page[2] = {-1, -1};
      if (lane_id() < end && p != j) {
        const int64_t slots[2] = {s0 + p, s0 + j};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int64_t at = slots[k] >> C.logP;
          if (at < C.M) page[k] = C.table[b * C.ld_table + at];
        }
      }
      const bool moves = page[0] >= 0 && page[0] < C.n_pages && page[1] >= 0 && page[1] < C.n_pages;
      const uint64_t all = ballot(moves);
      if (moves) {
        const int at = __builtin_popcountll(all & ((1ull << lane_id()) - 1));
        s_from[at] = page[0] * C.page_stride;
        s_to[at] = page[1] * C.page_stride;
        s_slot[at] = (int)((s0 + p) & (P - 1)) << 16 | (int)((s0 + j) & (P - 1));
      }
      if (lane_id() == 0) {
        s_moves[0] = __builtin_popcountll(all);
        s_moves[1] = end;
        // a row that ends too early says where; for those that read it later it ends there too
        if (blockIdx.x % (A.n_layers * parts) == 0 && end < min(m - j0, COMMIT_PASS)) path[j0 + end] = -1;
      }
    }
    __syncthreads();
    const int moves = s_moves[0], end = s_moves[1];
    // An element is one thread's for all moves, so that it may read COMMIT_AHEAD of them
    // before it writes: a path rises, and what is moved to is behind all that is yet to move.
    for (int i = threadIdx.x; i < nh * ITEMS; i += 256) {
      char* const head = base + i / ITEMS * C.head_bytes;
      const int e = i % ITEMS;
      for (int v0 = 0; v0 < moves; v0 += COMMIT_AHEAD) {
        auto move = [&](auto zero, auto where) {
          using T = decltype(zero);
          T t[COMMIT_AHEAD];
#pragma unroll
          for (int u = 0; u < COMMIT_AHEAD; ++u)
            if (v0 + u < moves) t[u] = *(const T*)(head + s_from[v0 + u] + where(s_slot[v0 + u] >> 16));
#pragma unroll
          for (int u = 0; u < COMMIT_AHEAD; ++u)
            if (v0 + u < moves) *(T*)(head + s_to[v0 + u] + where(s_slot[v0 + u] & 0xFFFF)) = t[u];
        };
        if (e < KC) {
          move(u32x4{}, [&](int slot) { return k_chunk<E>(e * E, slot, C.logP); });
        } else if (e < KC + D) {
          using V = typename std::conditional<F8, uint8_t, uint16_t>::type;
          move(V{}, [&](int slot) { return v_chunk<E, D>(e - KC, slot, C.logP) + slot % E * (16 / E); });
        } else {
          move(uint32_t{}, [&](int slot) {
            return e == KC + D ? k_scale<D>(slot, C.logP) : v_scale<D>(slot, C.logP);
          });
        }
      }
    }
    if (end < COMMIT_PASS) break;
    __syncthreads();
  }
}

template <int D, bool F8>
static void launch_append(const AppendArgs& A, hipStream_t s) {
  const unsigned per = 256 / (D / 8), heads = A.q_heads + A.kv.heads;
  // New tokens of a sequence share the pages' lines, which pays from 2 or 4 million
  // elements on; below that append_tiles' three dependent reads cost more (48 heads of
  // 128, bf16, rows and tiles: 1 sequence of 64 tokens 4.3 and 6.9 us, 32 of 9 7.6 and
  // 7.8, 256 of 2 10.0 and 9.0, 32 of 64 27 and 12; e4m3: 32 of 16 9.4 and 10.3, 256
  // of 4 17 and 15; heads of 64: 256 of 4 8.0 and 8.2, 256 of 9 14 and 10)
  const int64_t work = (int64_t)A.kv.T * (heads + A.kv.heads) * D;
  if (A.kv.q_start && A.kv.T >= 2 * (int64_t)A.kv.B && work >= (F8 ? 1 << 22 : 1 << 21)) {
    const unsigned groups = (heads + APPEND_HEADS - 1) / APPEND_HEADS;
    const unsigned qk = (A.kv.T + per - 1) / per * groups;
    const unsigned v = (A.kv.T + APPEND_VT - 1) / APPEND_VT * A.kv.heads;
    timed_launch(CX_KERNEL_KV_APPEND, append_tiles<D, F8>, dim3(qk + v), dim3(256), 0, s, A, (int)qk,
                 (int)groups);
    return;
  }
  const unsigned rows = (unsigned)A.kv.T * (heads + A.kv.heads);
  timed_launch(CX_KERNEL_KV_APPEND, append_rows<D, F8>, dim3((rows + per - 1) / per), dim3(256), 0,
               s, A);
}
template <int D>
static void launch_append(const AppendArgs& A, int dtype, hipStream_t s) {
  if (dtype == CX_KV_BF16) launch_append<D, false>(A, s);
  else launch_append<D, true>(A, s);
}

}  // namespace cx

extern "C" {

int cx_kv_append_bf16(const cx_kv_batch* kv, const uint16_t* q, int64_t q_token, int64_t q_head,
                      const uint16_t* k, int64_t k_token, int64_t k_head, const uint16_t* v,
                      int64_t v_token, int64_t v_head, int32_t q_heads, const float* rope,
                      int32_t rope_rows, int32_t rotary_dim, int32_t interleaved,
                      const uint16_t* q_norm, const uint16_t* k_norm, double eps,
                      uint16_t* q_out, void* stream) {
  return cx_kv_append_tree_bf16(kv, q, q_token, q_head, k, k_token, k_head, v, v_token, v_head,
                                q_heads, rope, rope_rows, rotary_dim, interleaved, q_norm, k_norm,
                                eps, nullptr, q_out, stream);
}

int cx_kv_append_tree_bf16(const cx_kv_batch* kv, const uint16_t* q, int64_t q_token,
                           int64_t q_head, const uint16_t* k, int64_t k_token, int64_t k_head,
                           const uint16_t* v, int64_t v_token, int64_t v_head, int32_t q_heads,
                           const float* rope, int32_t rope_rows, int32_t rotary_dim,
                           int32_t interleaved, const uint16_t* q_norm, const uint16_t* k_norm,
                           double eps, const int32_t* depth, uint16_t* q_out, void* stream) {
  cx::AppendArgs A;
  const int rc = cx::kv_args(kv, q_heads, &A.kv);
  if (rc != CX_OK) return rc;
  if (rope && (rotary_dim < 16 || rotary_dim % 16 || rotary_dim > kv->head_dim))
    return cx::api_fail(CX_EINVAL, "rotary_dim (%d) must be a multiple of 16 up to head_dim",
                        rotary_dim);
  if (rope && (int64_t)rope_rows < (int64_t)kv->max_pages * kv->page_tokens)
    return cx::api_fail(CX_EINVAL, "rope holds %d positions, the table's pages %lld", rope_rows,
                        (long long)kv->max_pages * kv->page_tokens);
  if (!(eps >= 0)) return cx::api_fail(CX_EINVAL, "eps must be >= 0");
  if (kv->T == 0 || kv->B == 0) return CX_OK;
  if (!q || !k || !v || !q_out) return cx::api_fail(CX_EINVAL, "null pointer argument");
  const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out |
                        (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)rope;
  if ((all & 15) || ((q_token | q_head | k_token | k_head | v_token | v_head) & 7))
    return cx::api_fail(CX_EINVAL, "rows must be 16-byte aligned");
  if ((int64_t)kv->T * (q_heads + 2 * (int64_t)kv->kv_heads) >= ((int64_t)1 << 31))
    return cx::api_fail(CX_EINVAL, "too many rows");
  A.x[0] = q; A.x[1] = k; A.x[2] = v;
  A.st[0] = q_token; A.st[1] = k_token; A.st[2] = v_token;
  A.sh[0] = q_head; A.sh[1] = k_head; A.sh[2] = v_head;
  A.q_heads = q_heads;
  // a rope without rows: no token has a position
  A.rope = rope_rows > 0 ? rope : nullptr;
  A.rdim = A.rope ? rotary_dim : 0;
  A.interleaved = interleaved;
  A.norm[0] = q_norm; A.norm[1] = k_norm;
  A.depth = depth;
  A.eps = (float)eps;
  A.q_out = q_out;
  const hipStream_t s = (hipStream_t)stream;
  switch (kv->head_dim) {
    case 64: cx::launch_append<64>(A, kv->dtype, s); break;
    case 128: cx::launch_append<128>(A, kv->dtype, s); break;
    default: cx::launch_append<256>(A, kv->dtype, s);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "append launch: %s", hipGetErrorString(e));
  return CX_OK;
}

int cx_kv_copy_pages(void* pages, int64_t layer_stride, int64_t page_stride, int64_t page_bytes,
                     int32_t n_layers, int32_t n_pages, const int32_t* src, const int32_t* dst,
                     int32_t n, void* stream) {
  if (n < 0 || n_layers < 0 || n_pages < 0 || page_bytes < 0 || page_stride < page_bytes ||
      layer_stride < 0)
    return cx::api_fail(CX_EINVAL, "bad shape");
  if (((uintptr_t)pages | page_bytes | page_stride | layer_stride) & 15)
    return cx::api_fail(CX_EINVAL, "pages must be 16-byte aligned");
  if (n == 0 || n_layers == 0 || n_pages == 0 || page_bytes == 0) return CX_OK;
  if (!pages || !src || !dst) return cx::api_fail(CX_EINVAL, "null pointer argument");
  cx::CopyArgs A;
  A.pages = (char*)pages;
  A.layer_stride = layer_stride; A.page_stride = page_stride; A.page_bytes = page_bytes;
  A.n_layers = n_layers; A.n_pages = n_pages;
  A.src = src; A.dst = dst;
  const int64_t parts = (page_bytes + cx::COPY_PART - 1) / cx::COPY_PART;
  if (parts * n_layers > INT32_MAX / n) return cx::api_fail(CX_EINVAL, "too many pages in one call");
  A.parts = (int)parts;
  cx::timed_launch(CX_KERNEL_KV_COPY, cx::copy_pages, dim3((unsigned)(parts * n_layers * n)),
                   dim3(256), 0, (hipStream_t)stream, A);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "page copy launch: %s", hipGetErrorString(e));
  return CX_OK;
}

int cx_kv_commit(const cx_kv_batch* kv, int64_t layer_stride, int32_t n_layers,
                 int32_t* path, int32_t width, const int32_t* count, void* stream) {
  cx::CommitArgs A;
  const int rc = cx::kv_args(kv, kv ? kv->kv_heads : 1, &A.kv);
  if (rc != CX_OK) return rc;
  if (n_layers < 0 || width < 0 || layer_stride < 0 || layer_stride % 16 ||
      (layer_stride == 0 && n_layers > 1))   // (all layers would move the same tokens)
    return cx::api_fail(CX_EINVAL, "bad shape");
  if (kv->T == 0 || kv->B == 0 || kv->n_pages == 0 || kv->max_pages == 0 || n_layers == 0 || width == 0)
    return CX_OK;
  if (!path) return cx::api_fail(CX_EINVAL, "null pointer argument");
  if ((int64_t)kv->B * n_layers > INT32_MAX / kv->kv_heads)
    return cx::api_fail(CX_EINVAL, "too many layers in one call");
  A.layer_stride = layer_stride;
  A.n_layers = n_layers;
  A.width = width;
  // heads together while the chip has workgroups enough
  A.heads = 1;
  while (A.heads < kv->kv_heads && (int64_t)kv->B * n_layers * kv->kv_heads >= 2ll * A.heads * cx::COMMIT_GROUPS)
    A.heads *= 2;
  A.path = path;
  A.count = count;
  using Kernel = void (*)(cx::CommitArgs);
  const bool f8 = kv->dtype == CX_KV_E4M3;
  const Kernel k = kv->head_dim == 64    ? (f8 ? (Kernel)cx::commit_tokens<64, true> : cx::commit_tokens<64, false>)
                   : kv->head_dim == 128 ? (f8 ? (Kernel)cx::commit_tokens<128, true> : cx::commit_tokens<128, false>)
                                         : (f8 ? (Kernel)cx::commit_tokens<256, true> : cx::commit_tokens<256, false>);
  cx::timed_launch(CX_KERNEL_KV_COMMIT, k, dim3((unsigned)(kv->B * n_layers * ((kv->kv_heads + A.heads - 1) / A.heads))),
                   dim3(256), 0, (hipStream_t)stream, A);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "commit launch: %s", hipGetErrorString(e));
  return CX_OK;
}

}  // extern "C"
