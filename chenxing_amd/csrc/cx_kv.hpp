// cx_kv.hpp -- the paged KV cache's layout and a batch's place in it, shared by
// the append, copy and attention kernels (cx_kv.hip, cx_attend.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cx_device.hpp"
#include "cx_sampler.h"

namespace cx {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float E4M3_MAX = 448.f;
constexpr int KV_MAX_NEW = 1 << 28;           // new tokens of a call: positions stay above -2^28

// cx_kv_batch with what the kernels derive from it.
struct KvArgs {
  char* pages;
  int64_t page_stride;        // bytes
  const int32_t* table;
  int64_t ld_table;
  const int32_t* kv_len;
  const int32_t* q_start;     // nullable
  int n_pages, heads, B, M, T;
  int logP;                   // page tokens = 1 << logP
  int head_bytes;             // one head's part of a page
};

// Bytes of one head's part of a page: K and V, and for e4m3 the scales.
inline int64_t kv_head_bytes(int D, int P, int dtype) {
  return dtype == CX_KV_BF16 ? (int64_t)4 * P * D : (int64_t)2 * P * D + 8 * P;
}

// Checks a cx_kv_batch and fills KvArgs; CX_OK or the failed entry point's
// return value (cx_kv.hip).
int kv_args(const cx_kv_batch* kv, int q_heads, KvArgs* out);

// [first, end) of sequence b's rows among the T new tokens, whatever q_start holds.
__device__ __forceinline__ int2 kv_rows(const KvArgs& A, int b) {
  if (!A.q_start) return make_int2(b, b + 1);
  const int s0 = min(max(A.q_start[b], 0), A.T);
  return make_int2(s0, min(max(A.q_start[b + 1], s0), A.T));
}

// Byte offsets inside a head's part of a page: the 16-byte chunk of K that
// holds dims d.. of the page's token o, and of V that holds dim d of token o's
// neighbours.  E: elements of a chunk.
template <int E>
__device__ __forceinline__ int k_chunk(int d, int o, int logP) { return ((d / E << logP) + o) * 16; }
template <int E, int D>
__device__ __forceinline__ int v_chunk(int d, int o, int logP) {
  return (D << logP) * (16 / E) + (o / E * D + d) * 16;
}
// The scales of the page's tokens (e4m3): K's, then V's.
template <int D>
__device__ __forceinline__ int k_scale(int o, int logP) { return (2 * D << logP) + 4 * o; }
template <int D>
__device__ __forceinline__ int v_scale(int o, int logP) {
  return (2 * D << logP) + (4 << logP) + 4 * o;
}

// Two floats as bf16 bits, rounded to nearest even.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const bf16x2 v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// The value of an e4m3 code (exact in bf16).
__device__ __forceinline__ float e4m3_value(uint32_t code) {
  return (float)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code, 1.0f, false)[0];
}

}  // namespace cx
