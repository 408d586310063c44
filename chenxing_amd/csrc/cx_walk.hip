// cx_walk.hip -- trees of drafted tokens, for gfx950: masks and depths from the
// parents, and the path that the sampled ids follow.
//
// Both are chains of dependent steps over a few dozen integers, bound by the launch
// and a step's latency: a tree's integers are read once, into LDS or registers (256 trees
// of up to 64 nodes: 4.0 us each, one tree 2.5 and 1.9).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cx_device.hpp"
#include "cx_internal.hpp"
#include "cx_sampler.h"
#include "cx_timing.hpp"

namespace cx {

struct WalkArgs {
  const int32_t* parents;
  const int32_t* tokens;
  const int32_t* sampled;
  const int32_t* q_start;     // nullable
  int B, T, words, width;
  int window;                 // 0: none
  uint64_t* mask;
  int32_t* depth;             // nullable
  int32_t* path;
  int32_t* count;
  int32_t* next;
};

// [first, end) of sequence b's nodes, whatever q_start holds.
__device__ __forceinline__ int2 walk_nodes(const WalkArgs& A, int b) {
  if (!A.q_start) return make_int2(b, b + 1);
  const int s0 = min(max(A.q_start[b], 0), A.T);
  return make_int2(s0, min(max(A.q_start[b + 1], s0), A.T));
}

constexpr int WALK_NODES = 2048;             // parents kept in LDS

// Workgroup: a sequence.  A thread a word of a node's mask: its way to the root.
__global__ __launch_bounds__(256) void tree_masks(WalkArgs A) {
  __shared__ int s_parent[WALK_NODES];
  const int b = blockIdx.x;
  const int2 r = walk_nodes(A, b);
  const int n = r.y - r.x;
  const bool kept = n <= WALK_NODES;
  if (kept) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) s_parent[i] = A.parents[r.x + i];
    __syncthreads();
  }
  const int64_t items = (int64_t)n * A.words;
  for (int64_t x = threadIdx.x; x < items; x += blockDim.x) {
    const int i = (int)(x / A.words), w = (int)(x % A.words);
    uint64_t m = 0;
    int d = -1;
    for (int a = i; a >= 0;) {               // parents lie below their children: it ends
      ++d;
      if (a >> 6 == w && (A.window == 0 || d < A.window)) m |= 1ull << (a & 63);
      const int p = kept ? s_parent[a] : A.parents[r.x + a];
      a = p < a ? p : -1;
    }
    A.mask[(int64_t)(r.x + i) * A.words + w] = m;
    if (w == 0 && A.depth) A.depth[r.x + i] = d;
  }
}

// Wave: a sequence.  The first 64 KEPT nodes are held by its lanes.
constexpr int WALK_KEPT = 4;
__global__ __launch_bounds__(64) void tree_accept(WalkArgs A) {
  const int b = blockIdx.x, l = lane_id();
  const int2 r = walk_nodes(A, b);
  const int n = r.y - r.x;
  int par[WALK_KEPT], tok[WALK_KEPT], out[WALK_KEPT];
#pragma unroll
  for (int c = 0; c < WALK_KEPT; ++c) {
    const int i = 64 * c + l;
    const bool in = i < n;
    par[c] = in ? A.parents[r.x + i] : -1;
    tok[c] = in ? A.tokens[r.x + i] : 0;
    out[c] = in ? A.sampled[r.x + i] : 0;
  }
  int32_t* path = A.path + (int64_t)b * A.width;
  int count = 0, cur = n > 0 ? 0 : -1, want = -1;
  while (cur >= 0) {
    if (l == 0) path[count] = cur;
    ++count;
    if (cur < 64 * WALK_KEPT) {
#pragma unroll
      for (int c = 0; c < WALK_KEPT; ++c)
        if (cur >> 6 == c) want = lane_read(out[c], cur & 63);
    } else {
      want = A.sampled[r.x + cur];
    }
    if (count == A.width) break;
    int next = -1;
#pragma unroll
    for (int c = 0; c < WALK_KEPT; ++c) {
      if (64 * c >= n) break;
      const uint64_t m = ballot(par[c] == cur && tok[c] == want && 64 * c + l > cur);
      if (next < 0 && m) next = 64 * c + __builtin_ctzll(m);
    }
    for (int i0 = 64 * WALK_KEPT; next < 0 && i0 < n; i0 += 64) {
      const int i = i0 + l;
      const bool hit = i < n && i > cur && A.parents[r.x + i] == cur && A.tokens[r.x + i] == want;
      const uint64_t m = ballot(hit);
      if (m) next = i0 + __builtin_ctzll(m);
    }
    cur = next;
  }
  for (int j = count + l; j < A.width; j += 64) path[j] = -1;
  if (l == 0) {
    A.count[b] = count;
    A.next[b] = want;
  }
}

}  // namespace cx

extern "C" {

int cx_tree_masks(const int32_t* parents, const int32_t* q_start, int32_t B, int32_t T,
                  uint64_t* mask, int32_t words, int32_t* depth, void* stream) {
  return cx_tree_masks_window(parents, q_start, B, T, mask, words, depth, 0, stream);
}

int cx_tree_masks_window(const int32_t* parents, const int32_t* q_start, int32_t B, int32_t T,
                         uint64_t* mask, int32_t words, int32_t* depth, int32_t window,
                         void* stream) {
  if (B < 0 || T < 0 || words < 1) return cx::api_fail(CX_EINVAL, "bad shape");
  if (window < 0) return cx::api_fail(CX_EINVAL, "window must be >= 0");
  if (!q_start && T != B)
    return cx::api_fail(CX_EINVAL, "without q_start there is one node per sequence");
  if (B == 0 || T == 0) return CX_OK;
  if (!parents || !mask) return cx::api_fail(CX_EINVAL, "null pointer argument");
  cx::WalkArgs A = {};
  A.parents = parents;
  A.q_start = q_start;
  A.B = B; A.T = T; A.words = words;
  A.mask = mask;
  A.depth = depth;
  A.window = window;
  cx::timed_launch(CX_KERNEL_TREE_WALK, cx::tree_masks, dim3(B), dim3(256), 0, (hipStream_t)stream, A);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "tree masks launch: %s", hipGetErrorString(e));
  return CX_OK;
}

int cx_tree_accept(const int32_t* parents, const int32_t* tokens, const int32_t* sampled,
                   const int32_t* q_start, int32_t B, int32_t T, int32_t width, int32_t* path,
                   int32_t* count, int32_t* next, void* stream) {
  if (B < 0 || T < 0 || width < 1) return cx::api_fail(CX_EINVAL, "bad shape");
  if (!q_start && T != B)
    return cx::api_fail(CX_EINVAL, "without q_start there is one node per sequence");
  if (B == 0) return CX_OK;
  if ((T && (!parents || !tokens || !sampled)) || !path || !count || !next)
    return cx::api_fail(CX_EINVAL, "null pointer argument");
  cx::WalkArgs A = {};
  A.parents = parents;
  A.tokens = tokens;
  A.sampled = sampled;
  A.q_start = q_start;
  A.B = B; A.T = T; A.width = width;
  A.path = path;
  A.count = count;
  A.next = next;
  cx::timed_launch(CX_KERNEL_TREE_WALK, cx::tree_accept, dim3(B), dim3(64), 0, (hipStream_t)stream, A);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cx::api_fail(CX_EHIP, "tree accept launch: %s", hipGetErrorString(e));
  return CX_OK;
}

}  // extern "C"
