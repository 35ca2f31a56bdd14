// Shared by the kernels of attention over a cache: their arguments, and what a row of a
// drafted tree, a chunk or a decode step may see.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace w8 {

static __device__ int g_tree_status = 0;  // each source file's own

constexpr int kTreeMaxSplits = 256;

struct TreeArgs {
  const uint16_t *q, *k, *v, *kn, *vn;
  uint16_t* o;
  const int* lens;
  const uint8_t* tree;   // [B, N, N] or null: causal
  const int* depth;      // [B, N] or null: the token's index
  int64_t q_b, q_h, q_t, k_b, k_h, k_s, v_b, v_h, v_s, kn_b, kn_h, kn_t, vn_b, vn_h, vn_t, o_b, o_h, o_t;
  int64_t tree_b, tree_i, depth_b;
  int batch, kv_heads, group, n, slots, window;
  float scale_log2;      // scale * log2(e): scores in log2 units
  int row_tiles, splits;
  float* part_o;         // [item][split][BM][D] fp32, item = (b * kv_heads + c) * row_tiles + rt
  float2* part_ml;       // [item][split][BM]
  float* lse;            // [b * kv_heads + c][R] (log2 units) when the weights are wanted
  float* scores;         // [b * kv_heads + c][R][score_pitch] (log2 units), slots then drafts
  int64_t score_pitch;
  const float* w_in;
  float* w_out;
  float* w_new;          // [B, KV, N]
  int64_t wi_b, wi_h, wo_b, wo_h;
};

__device__ __forceinline__ float ex2_tree(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The committed length of sequence b, kept inside the cache whatever the memory holds.
__device__ __forceinline__ int tree_len(const TreeArgs& a, int b) {
  const int n = a.lens[b];
  if (n < 0 || n > a.slots) {
    atomicExch(&g_tree_status, W8_ERR_INVALID_ARG);
    return n < 0 ? 0 : a.slots;
  }
  return n;
}

// First committed slot that token i at `depth` sees under the window (0: all of them).
__device__ __forceinline__ int tree_first(const TreeArgs& a, int len, int depth) {
  if (a.window <= 0) return 0;
  const int64_t f = static_cast<int64_t>(len) + depth - a.window + 1;
  return f <= 0 ? 0 : (f >= len ? len : static_cast<int>(f));
}

__device__ __forceinline__ int tree_depth(const TreeArgs& a, int b, int i) {
  return a.depth != nullptr ? max(a.depth[b * a.depth_b + i], 0) : i;
}

// Whether token i sees new token j (both < n).
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, int b, int i, int j, int depth_i) {
  const bool on = a.tree != nullptr ? a.tree[b * a.tree_b + i * a.tree_i + j] != 0 : j <= i;
  if (!on || a.window <= 0) return on;
  return static_cast<int64_t>(tree_depth(a, b, j)) > static_cast<int64_t>(depth_i) - a.window;
}

// Tiles of `bn` keys of one row tile of `bm` rows: committed tiles [c0, c1), then draft
// tiles [0, nd).
struct TreeSpan {
  int c0, c1, nd;
};
__device__ __forceinline__ TreeSpan tree_span(const TreeArgs& a, int len, int rt, int bm, int bn) {
  TreeSpan s;
  const int rows = a.group * a.n;
  const int i0 = rt * bm / a.group, i1 = min((rt + 1) * bm, rows) - 1;
  // Without given depths the first row's token is the shallowest; with them, 0 is a bound.
  s.c0 = tree_first(a, len, a.depth != nullptr ? 0 : i0) / bn;
  s.c1 = (len + bn - 1) / bn;
  // A causal chunk's row tile needs the new keys up to its last token only.
  const int last = a.tree != nullptr ? a.n - 1 : i1 / a.group;
  s.nd = last / bn + 1;
  if (s.c0 > s.c1) s.c0 = s.c1;
  return s;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&p);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&p);
}
template <typename T>
__device__ __forceinline__ float tree_f32(uint16_t bits);
template <>
__device__ __forceinline__ float tree_f32<__nv_bfloat16>(uint16_t bits) {
  return __uint_as_float(static_cast<uint32_t>(bits) << 16);
}
template <>
__device__ __forceinline__ float tree_f32<__half>(uint16_t bits) {
  return __half2float(__ushort_as_half(bits));
}
// Infinity or NaN: every exponent bit set.
template <typename T>
__device__ __forceinline__ bool tree_nonfinite(uint32_t bits) {
  constexpr uint32_t e = sizeof(T) == 2 && __is_same(T, __half) ? 0x7C00u : 0x7F80u;
  return (bits & e) == e;
}

}  // namespace w8
