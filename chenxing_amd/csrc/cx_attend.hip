// cx_attend.hip -- attention of the new tokens over the paged KV cache, for
// gfx950 (layout: cx_kv.hpp).
//
// out[t, h] = sum over the allowed positions s of softmax(scale q.k_s) v_s, with
// the running maximum m and sum l of the softmax's terms: a block of scores
// raises m to m', and l and the output so far are scaled by exp(m - m').
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cx_device.hpp"
#include "cx_internal.hpp"
#include "cx_kv.hpp"
#include "cx_sampler.h"
#include "cx_timing.hpp"

namespace cx {

constexpr float LOG2E = 1.4426950408889634f;

struct AttendArgs {
  KvArgs kv;
  const uint16_t* q;
  int64_t q_token, q_head;
  int q_heads, G;             // G: q heads per kv head
  float s1, s2;               // score in powers of 2: s1 qk, or s2 tanh(s1 qk)
  int cap;                    // the latter
  int window;                 // 0: none
  uint16_t* out;
};

__device__ __forceinline__ float score(const AttendArgs& A, float qk) {
  return A.cap ? A.s2 * tanhf(A.s1 * qk) : A.s1 * qk;
}

// One wave per (token, q head): 64 positions at a time, one to a lane, then
// the dims of the output D / 64 to a lane.
template <int D, bool F8>
__global__ __launch_bounds__(64) void attend_row(AttendArgs A) {
  constexpr int E = F8 ? 16 : 8, N = D / 64;
  __shared__ float s_q[D], s_p[64];
  __shared__ int64_t s_at[64];
  const KvArgs& C = A.kv;
  const int t = blockIdx.x / A.q_heads, hq = blockIdx.x % A.q_heads, h = hq / A.G;
  const int l = threadIdx.x;
  int b = t, n = 1, i = 0;
  if (C.q_start) {
    for (b = 0; b < C.B && C.q_start[b + 1] <= t; ++b) {}
    if (b == C.B) return;
    const int2 r = kv_rows(C, b);
    i = t - r.x; n = r.y - r.x;
  }
  const int pos = C.kv_len[b] - n + i, end = min(pos + 1, C.M << C.logP);
  const int first = A.window ? max(0, pos - A.window + 1) : 0;
  for (int d = l; d < D; d += 64)
    s_q[d] = __uint_as_float((uint32_t)A.q[t * A.q_token + hq * A.q_head + d] << 16);
  float m = -INFINITY, sum = 0, acc[N];
  bool any = false;
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0;
  for (int s0 = first; s0 < end; s0 += 64) {
    __syncthreads();
    const int s = s0 + l, o = s & ((1 << C.logP) - 1);
    const int page = s < end ? C.table[b * C.ld_table + (s >> C.logP)] : -1;
    const bool ok = (unsigned)page < (unsigned)C.n_pages;
    const char* base = C.pages + page * C.page_stride + (int64_t)h * C.head_bytes;
    float x = -INFINITY, vs = 1.f;
    if (ok) {
      float dot = 0;
      for (int d = 0; d < D; ++d) {
        const char* p = base + k_chunk<E>(d, o, C.logP);
        const float kv = F8 ? e4m3_value(*(const uint8_t*)(p + d % E))
                            : bf16_lo(*(const uint16_t*)(p + d % E * 2));
        dot = fmaf(s_q[d], kv, dot);
      }
      if (F8) {
        dot *= *(const float*)(base + k_scale<D>(o, C.logP));
        vs = *(const float*)(base + v_scale<D>(o, C.logP));
      }
      x = score(A, dot);
    }
    any |= __any(ok);
    const float m1 = fmaxf(m, wave_max(x));
    const float u = m1 == -INFINITY ? 0.f : m1;
    const float alpha = __builtin_amdgcn_exp2f(m - u);
    const float p = ok ? __builtin_amdgcn_exp2f(x - u) : 0.f;
    m = m1;
    sum = sum * alpha + wave_sum(p);
    s_p[l] = p * vs;
    s_at[l] = ok ? base - C.pages : -1;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] *= alpha;
    for (int j = 0; j < 64 && s0 + j < end; ++j) {
      if (s_at[j] < 0) continue;
      const char* vb = C.pages + s_at[j];
      const int oj = (s0 + j) & ((1 << C.logP) - 1);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const char* p = vb + v_chunk<E, D>(l + 64 * k, oj, C.logP);
        const float v = F8 ? e4m3_value(*(const uint8_t*)(p + oj % E))
                           : bf16_lo(*(const uint16_t*)(p + oj % E * 2));
        acc[k] = fmaf(s_p[j], v, acc[k]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    A.out[((int64_t)t * A.q_heads + hq) * D + l + 64 * k] =
        (uint16_t)pack_bf16(any ? acc[k] / sum : 0.f, 0.f);
}

template <int D>
static void launch_attend(const AttendArgs& A, int dtype, hipStream_t s) {
  timed_launch(CX_KERNEL_ATTEND, dtype == CX_KV_BF16 ? attend_row<D, false> : attend_row<D, true>,
               dim3((unsigned)(A.kv.T * A.q_heads)), dim3(64), 0, s, A);
}

}  // namespace cx

extern "C" {

size_t cx_paged_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                          int32_t max_new) {
  return 256;
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
  A.s1 = (float)(A.cap ? scale / softcap : scale * 1.4426950408889634);
  A.s2 = (float)(softcap * 1.4426950408889634);
  A.window = window;
  A.out = out;
  const hipStream_t s = (hipStream_t)stream;
  switch (kv->head_dim) {
    case 64: cx::launch_attend<64>(A, kv->dtype, s); break;
    case 128: cx::launch_attend<128>(A, kv->dtype, s); break;
    default: cx::launch_attend<256>(A, kv->dtype, s);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "attention launch: %s", hipGetErrorString(e));
  return CX_OK;
}

}  // extern "C"
