// cx_kv.hip -- the paged KV cache, for gfx950: new tokens normed, rotated and
// appended, pages copied (layout: cx_kv.hpp).
#include <hip/hip_runtime.h>
#include <stdint.h>

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
  float eps;
  uint16_t* q_out;
};

// The sequence of new token t and its position: the last b with
// q_start[b] <= t.  -1 for a token outside every sequence.
__device__ __forceinline__ int2 token_place(const KvArgs& A, int t) {
  int b = t, i = 0, n = 1;
  if (A.q_start) {
    int lo = 0, hi = A.B;                     // first b with q_start[b + 1] > t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (A.q_start[mid + 1] > t) hi = mid;
      else lo = mid + 1;
    }
    if (lo >= A.B) return make_int2(-1, -1);
    b = lo;
    const int2 r = kv_rows(A, b);
    i = t - r.x;
    n = r.y - r.x;
  }
  return make_int2(b, (int)(A.kv_len[b] - (unsigned)n + (unsigned)i));
}

// One row (token, head) of q, k or v to D / 8 lanes, 8 dims each, every row of
// the call at once: q heads first, then k, then v.  The mean square and, for
// e4m3, the largest magnitude go over the row's lanes; the other dim of a
// rotated pair is in the same lane (interleaved) or rdim / 16 lanes away.
template <int D, bool F8>
__global__ __launch_bounds__(256) void append_rows(AppendArgs A) {
  constexpr int LR = D / 8, E = F8 ? 16 : 8;
  const KvArgs& C = A.kv;
  const int heads = A.q_heads + 2 * C.heads;
  const int64_t row = (int64_t)blockIdx.x * (256 / LR) + threadIdx.x / LR;
  const int t = (int)(row / heads), hh = (int)(row % heads);
  if (t >= C.T) return;
  const int j = threadIdx.x % LR, d = 8 * j;
  const int kind = hh < A.q_heads ? 0 : hh < A.q_heads + C.heads ? 1 : 2;
  const int h = kind == 0 ? hh : kind == 1 ? hh - A.q_heads : hh - A.q_heads - C.heads;
  const u32x4 in = *(const u32x4*)(A.x[kind] + t * A.st[kind] + h * A.sh[kind] + d);
  const int2 place = token_place(C, t);
  const int pos = place.y;
  const bool held = place.x >= 0 && pos >= 0 && pos < (C.M << C.logP);
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = bf16_lo(in[i]); x[2 * i + 1] = bf16_hi(in[i]); }
  const uint16_t* w = kind < 2 ? A.norm[kind] : nullptr;
  if (w) {
    float ss = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = LR / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
    const float r = 1.f / sqrtf(ss * (1.f / D) + A.eps);
    const u32x4 wv = *(const u32x4*)(w + d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = x[2 * i] * r * bf16_lo(wv[i]);
      x[2 * i + 1] = x[2 * i + 1] * r * bf16_hi(wv[i]);
    }
  }
  if (kind < 2 && A.rope) {
    const float* cs = A.rope + (int64_t)(held ? pos : 0) * A.rdim;
    const int half = A.rdim / 2;
    if (A.interleaved) {
      if (d < A.rdim) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float c = cs[d / 2 + i], s = cs[half + d / 2 + i];
          const float a = x[2 * i], b = x[2 * i + 1];
          x[2 * i] = a * c - b * s;
          x[2 * i + 1] = b * c + a * s;
        }
      }
    } else {
      const bool low = d < half;
      const int other = threadIdx.x + (low ? half / 8 : -(half / 8));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __shfl(x[i], other & 63);
        if (d < A.rdim) {
          const int p = low ? d + i : d - half + i;
          const float c = cs[p], s = cs[half + p];
          x[i] = low ? x[i] * c - y * s : x[i] * c + y * s;
        }
      }
    }
  }
  if (kind == 0) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    *(u32x4*)(A.q_out + ((int64_t)t * A.q_heads + h) * D + d) = o;
    return;
  }
  float scale = 1.f;
  if (F8) {                                   // the largest |x| by its bits: NaN above inf above all
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = LR / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    const bool fine = m < 0x7F800000u;
    scale = !fine ? __builtin_nanf("") : m == 0 ? 1.f : __uint_as_float(m) / E4M3_MAX;
    // a row of denormals can round its scale to 0
    if (scale == 0.f) scale = 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = fine ? fminf(fmaxf(x[i] / scale, -E4M3_MAX), E4M3_MAX) : 0.f;
  }
  if (!held) return;
  const int page = C.table[place.x * C.ld_table + (pos >> C.logP)];
  if ((unsigned)page >= (unsigned)C.n_pages) return;
  const int o = pos & ((1 << C.logP) - 1);
  char* base = C.pages + page * C.page_stride + (int64_t)h * C.head_bytes;
  if (F8) {
    u32x2 c;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      c[i] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], p, true);
    }
    if (kind == 1) {
      *(u32x2*)(base + k_chunk<E>(d, o, C.logP) + (d & 8)) = c;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *(uint8_t*)(base + v_chunk<E, D>(d + i, o, C.logP) + o % E) = (uint8_t)(c[i / 4] >> 8 * (i % 4));
    }
    if (j == 0)
      *(float*)(base + (kind == 1 ? k_scale<D>(o, C.logP) : v_scale<D>(o, C.logP))) = scale;
    return;
  }
  if (kind == 1) {
    u32x4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    *(u32x4*)(base + k_chunk<E>(d, o, C.logP)) = c;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *(uint16_t*)(base + v_chunk<E, D>(d + i, o, C.logP) + o % E * 2) =
          (uint16_t)(in[i / 2] >> 16 * (i % 2));
  }
}

struct CopyArgs {
  char* pages;
  int64_t layer_stride, page_stride, page_bytes;
  int n_layers, n_pages, parts;
  const int32_t* src;
  const int32_t* dst;
};

constexpr int COPY_PART = 16384;              // bytes a workgroup copies

// Workgroup (pair, layer, part): 16 KB of the page.
__global__ __launch_bounds__(256) void copy_pages(CopyArgs A) {
  const unsigned part = blockIdx.x % (unsigned)A.parts, x = blockIdx.x / (unsigned)A.parts;
  const unsigned layer = x % (unsigned)A.n_layers, pair = x / (unsigned)A.n_layers;
  const int s = A.src[pair], d = A.dst[pair];
  if ((unsigned)s >= (unsigned)A.n_pages || (unsigned)d >= (unsigned)A.n_pages) return;
  char* base = A.pages + layer * A.layer_stride;
  const char* from = base + s * A.page_stride;
  char* to = base + d * A.page_stride;
  for (int i = 0; i < COPY_PART / 4096; ++i) {
    const int64_t at = (int64_t)part * COPY_PART + i * 4096 + threadIdx.x * 16;
    if (at < A.page_bytes) *(u32x4*)(to + at) = *(const u32x4*)(from + at);
  }
}

template <int D>
static void launch_append(const AppendArgs& A, int dtype, hipStream_t s) {
  const int64_t rows = (int64_t)A.kv.T * (A.q_heads + 2 * A.kv.heads), per = 256 / (D / 8);
  const dim3 grid((unsigned)((rows + per - 1) / per));
  timed_launch(CX_KERNEL_KV_APPEND, dtype == CX_KV_BF16 ? append_rows<D, false> : append_rows<D, true>,
               grid, dim3(256), 0, s, A);
}

}  // namespace cx

extern "C" {

int cx_kv_append_bf16(const cx_kv_batch* kv, const uint16_t* q, int64_t q_token, int64_t q_head,
                      const uint16_t* k, int64_t k_token, int64_t k_head, const uint16_t* v,
                      int64_t v_token, int64_t v_head, int32_t q_heads, const float* rope,
                      int32_t rope_rows, int32_t rotary_dim, int32_t interleaved,
                      const uint16_t* q_norm, const uint16_t* k_norm, double eps,
                      uint16_t* q_out, void* stream) {
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
  if ((int64_t)kv->T * (q_heads + 2 * (int64_t)kv->kv_heads) > ((int64_t)1 << 33))
    return cx::api_fail(CX_EINVAL, "too many rows");
  A.x[0] = q; A.x[1] = k; A.x[2] = v;
  A.st[0] = q_token; A.st[1] = k_token; A.st[2] = v_token;
  A.sh[0] = q_head; A.sh[1] = k_head; A.sh[2] = v_head;
  A.q_heads = q_heads;
  A.rope = rope; A.rdim = rope ? rotary_dim : 0;
  A.interleaved = interleaved;
  A.norm[0] = q_norm; A.norm[1] = k_norm;
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

}  // extern "C"
