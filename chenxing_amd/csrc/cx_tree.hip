// cx_tree.hip -- attention of trees of drafted tokens over the paged KV cache, for
// gfx950 (layout: cx_kv.hpp).
//
// out[t, h] = sum over the allowed slots s of softmax(scale q.k_s) v_s, in one pass
// over K and V with the running maximum and sum of the softmax's terms.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "cx_device.hpp"
#include "cx_internal.hpp"
#include "cx_kv.hpp"
#include "cx_sampler.h"
#include "cx_timing.hpp"

namespace cx {

struct TreeArgs {
  KvArgs kv;
  const uint16_t* q;
  int64_t q_token, q_head;
  int q_heads, G;             // G: q heads per kv head
  const uint64_t* mask;       // [T, words]
  int words;
  const int32_t* depth;       // nullable
  float scale, cap;           // cap 0: none
  int window;                 // 0: none
  uint16_t* out;
};

// Wave: a row (node, q head).  64 slots at a time: a lane's slot for the scores, a
// lane's dims for the sums.
template <int D, bool F8>
__global__ __launch_bounds__(64) void tree_rows(TreeArgs A) {
  constexpr int E = F8 ? 16 : 8, DL = D / 64;
  __shared__ float s_q[D], s_p[64];
  const KvArgs& C = A.kv;
  const int l = lane_id();
  const int t = (int)(blockIdx.x / (unsigned)A.q_heads), h = (int)(blockIdx.x % (unsigned)A.q_heads);
  int b = t;
  if (C.q_start) {
    int lo = 0, hi = C.B;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (C.q_start[mid + 1] > t) hi = mid;
      else lo = mid + 1;
    }
    b = lo;
    if (b >= C.B) return;
  }
  const int2 r = kv_rows(C, b);
  if (t < r.x || t >= r.y) return;
  const int P = 1 << C.logP, len = max(C.kv_len[b], 0), base = len - (r.y - r.x);
  const int lim = min(len, C.M << C.logP);
  const int lo = A.window ? base + max(A.depth[t], 0) - A.window : -1;
  for (int d = l; d < D; d += 64) s_q[d] = bf16_lo(A.q[t * A.q_token + h * A.q_head + d]);
  __syncthreads();
  float m = -INFINITY, sum = 0, acc[DL] = {};
  for (int s0 = A.window ? max(min(lo + 1, base), 0) & ~63 : 0; s0 < lim; s0 += 64) {
    const int s = s0 + l, o = s & (P - 1), node = s - base;
    const int id = s < lim ? C.table[b * C.ld_table + (s >> C.logP)] : -1;
    bool in = (unsigned)id < (unsigned)C.n_pages;
    if (node < 0) in &= s > lo;
    else in &= node < 64 * A.words && (A.mask[(int64_t)t * A.words + (node >> 6)] >> (node & 63) & 1);
    const char* base_h = C.pages + (int64_t)(in ? id : 0) * C.page_stride + (int64_t)(h / A.G) * C.head_bytes;
    float x = -INFINITY;
    if (in) {
      x = 0;
      for (int d = 0; d < D; ++d) {
        const char* p = base_h + k_chunk<E>(d, o, C.logP) + d % E * (16 / E);
        x = fmaf(s_q[d], F8 ? e4m3_value(*(const uint8_t*)p) : bf16_lo(*(const uint16_t*)p), x);
      }
      if (F8) x *= *(const float*)(base_h + k_scale<D>(o, C.logP));
      x *= A.scale;
      if (A.cap > 0) x = A.cap * tanhf(x / A.cap);
    }
    const uint64_t some = ballot(in);
    if (!some) continue;
    const float top = fmaxf(wave_max(x), -3e38f), m1 = fmaxf(m, top);
    const float f = expf(m - m1), p = in ? expf(x - m1) : 0.f;
    m = m1;
    sum = sum * f + wave_sum(p);
    s_p[l] = p;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DL; ++i) acc[i] *= f;
    for (int k = 0; k < 64; ++k) {
      if (!(some >> k & 1)) continue;
      const int sk = s0 + k, ok = sk & (P - 1);
      const char* bk = C.pages + (int64_t)lane_read(id, k) * C.page_stride + (int64_t)(h / A.G) * C.head_bytes;
      float pk = s_p[k];
      if (F8) pk *= *(const float*)(bk + v_scale<D>(ok, C.logP));
#pragma unroll
      for (int i = 0; i < DL; ++i) {
        const char* p = bk + v_chunk<E, D>(l + 64 * i, ok, C.logP) + ok % E * (16 / E);
        acc[i] = fmaf(pk, F8 ? e4m3_value(*(const uint8_t*)p) : bf16_lo(*(const uint16_t*)p), acc[i]);
      }
    }
    __syncthreads();
  }
  const float f = m == -INFINITY ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < DL; ++i)
    A.out[((int64_t)t * A.q_heads + h) * D + l + 64 * i] = (uint16_t)pack_bf16(acc[i] * f, 0.f);
}

}  // namespace cx

extern "C" {

size_t cx_tree_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                         int32_t max_new) {
  return 256;
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
  A.mask = mask;
  A.words = mask_words;
  A.depth = depth;
  A.scale = (float)scale;
  A.cap = std::isinf(softcap) ? 0.f : (float)softcap;
  if (!std::isfinite(A.scale) || !std::isfinite(A.cap) ||
      (A.cap > 0 && !std::isfinite((float)(scale / softcap))) || (softcap > 0 && A.cap == 0 && !std::isinf(softcap)))
    return cx::api_fail(CX_EINVAL, "scale (%g) and softcap (%g) pass the range of fp32", scale, softcap);
  A.window = window;
  A.out = out;
  using Kernel = void (*)(cx::TreeArgs);
  const bool f8 = kv->dtype == CX_KV_E4M3;
  const Kernel k = kv->head_dim == 64    ? (f8 ? (Kernel)cx::tree_rows<64, true> : cx::tree_rows<64, false>)
                   : kv->head_dim == 128 ? (f8 ? (Kernel)cx::tree_rows<128, true> : cx::tree_rows<128, false>)
                                         : (f8 ? (Kernel)cx::tree_rows<256, true> : cx::tree_rows<256, false>);
  cx::timed_launch(CX_KERNEL_TREE, k, dim3((unsigned)(kv->T * q_heads)), dim3(64), 0, (hipStream_t)stream, A);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "tree attention launch: %s", hipGetErrorString(e));
  return CX_OK;
}

}  // extern "C"
