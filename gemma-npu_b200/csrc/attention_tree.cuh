// Shared by the kernels of attention over a cache: their arguments, and what a row of a
// drafted tree, a chunk or a decode step may see.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace w8 {

static __device__ int g_tree_status = 0;  // each source file's own

constexpr int kTreeMaxPieces = 512;  // partial results of one item

struct TreeArgs {
  const uint16_t *q, *k, *v, *kn, *vn;
  uint16_t* o;
  const int* lens;
  const uint8_t* tree;   // [B, N, N] or null: causal
  const int* depth;      // [B, N] or null: the token's index
  int64_t q_b, q_h, q_t, k_b, k_h, k_s, v_b, v_h, v_s, kn_b, kn_h, kn_t, vn_b, vn_h, vn_t, o_b, o_h, o_t;
  int64_t tree_b, tree_i, depth_b;
  uint32_t group_rcp;    // floor(2^32 / group), for tree_row
  int q_tma;             // q's rows load as TMA boxes (tcgen05 schedule)
  int batch, kv_heads, group, n, slots, window;
  int sink;              // positions below it stay visible behind a window (0: none)
  float scale_log2;      // scale * log2(e): scores in log2 units
  int row_tiles, splits;  // splits: of each item, tcgen05 schedule only
  // Partial results of an item (item = (b * kv_heads + c) * row_tiles + rt): piece s in slot
  // item * splits + s, or where `info` gives (first CTA, pieces) as tree_slot says.
  float* part_o;         // [slot][BM][D] fp32
  float2* part_ml;       // [slot][BM]
  int2* info;            // [items], mma.sync schedule
  int direct;            // mma.sync schedule: CTA i takes item i whole
  float* lse;            // [b * kv_heads + c][R] (log2 units) when the weights are wanted
  float* scores;         // [b * kv_heads + c][R][score_pitch] (log2 units), new tokens from draft_at on
  int64_t score_pitch;
  int draft_at;
  int tma;               // the caches and new rows load as TMA boxes (mma.sync schedule)
  const float* w_in;
  float* w_out;
  float* w_new;          // [B, KV, N]
  int64_t wi_b, wi_h, wo_b, wo_h;
};

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
  constexpr uint32_t e = __is_same(T, __half) ? 0x7C00u : 0x7F80u;
  return (bits & e) == e;
}

// The softmax's running reference.  p = 2^(x - m) is rounded to the operands' type, in which fp16
// ends at 2^-24 (halves of it round to 0) and 65504: there m stands 2^7 below the row's maximum, so
// that what a long tail of small probabilities sums to is not lost beside one large one (each is at
// most 2^-25 off against a sum of 2^7 at least: 2^-32 of the output a key).  m moves only when a
// maximum exceeds it by more than 8 above that, so the output is seldom rescaled: p <= 2^15, 2^8 for
// bf16, which has fp32's exponents and needs no such room.
template <typename T>
struct TreeRef {
  static constexpr float kBelow = __is_same(T, __half) ? 7.f : 0.f;  // of m under the maximum it is set to
  static constexpr float kSlack = 8.f + kBelow;                     // a maximum this far above m moves it
};

// A CTA's range of tiles holds at most one piece that begins an item it does not finish (its
// last, slot 2 u + 1) and one that continues an item (its first, slot 2 u).
__device__ __forceinline__ int64_t tree_slot(int2 info, int s) {
  return s == 0 ? 2 * static_cast<int64_t>(info.x) + 1 : 2 * (static_cast<int64_t>(info.x) + s);
}

// Row r = i * group + g as (token i, head g of the group) without a division: the product with
// the truncated reciprocal is at most one short for r < 2^32.
__device__ __forceinline__ void tree_row(const TreeArgs& a, int r, int& i, int& g) {
  i = a.group == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), a.group_rcp));
  g = r - i * a.group;
  if (g >= a.group) ++i, g -= a.group;
}

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
// `sink_left`: a.sink less the committed length; new tokens of a smaller depth are sinks.
constexpr int kNoSinks = INT32_MIN;
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, int b, int i, int j, int depth_i, int sink_left = kNoSinks) {
  const bool on = a.tree != nullptr ? a.tree[b * a.tree_b + i * a.tree_i + j] != 0 : j <= i;
  if (!on || a.window <= 0) return on;
  const int dj = tree_depth(a, b, j);
  return static_cast<int64_t>(dj) > static_cast<int64_t>(depth_i) - a.window || dj < sink_left;
}

// The same for a packed pair: bit 15 / 31 set for a half that is not finite (the exponent
// field plus its lowest bit carries into the sign's place only from all ones).
template <typename T>
__device__ __forceinline__ uint32_t nonfinite_bits(uint32_t pair) {
  constexpr uint32_t e = __is_same(T, __half) ? 0x7C007C00u : 0x7F807F80u;
  constexpr uint32_t one = __is_same(T, __half) ? 0x04000400u : 0x00800080u;
  return ((pair & e) + one) & 0x80008000u;
}

// The bytes of a word that are not zero, as 4 bits.
__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t w) {
  const uint32_t m = __vcmpne4(w, 0u) & 0x08040201u;  // one distinct bit of each byte
  return (m | (m >> 8) | (m >> 16) | (m >> 24)) & 15u;
}

// tree_sees of the new tokens j0 .. j0 + 31 as bits (those behind n are 0).  A loop of byte
// loads would wait for each in turn: the row is read with 16-byte loads where it is aligned
// and with 32 independent ones where it is not.
__device__ __forceinline__ uint32_t tree_sees32(const TreeArgs& a, int b, int i, int j0, int depth_i,
                                                int sink_left = kNoSinks) {
  const int left = a.n - j0;
  if (left <= 0) return 0u;
  uint32_t bits = 0;
  if (a.tree == nullptr) {
    bits = i < j0 ? 0u : i - j0 >= 31 ? 0xFFFFFFFFu : (2u << (i - j0)) - 1u;
    if (a.depth == nullptr) {  // a plain chunk: the last `window` tokens up to i
      const int lo = a.window > 0 ? i - a.window + 1 - j0 : 0;
      const uint32_t sinks = sink_left <= j0 ? 0u : sink_left - j0 > 31 ? 0xFFFFFFFFu : (1u << (sink_left - j0)) - 1u;
      if (lo > 0) bits &= (lo > 31 ? 0u : 0xFFFFFFFFu << lo) | sinks;
      return left < 32 ? bits & ((1u << left) - 1u) : bits;
    }
  } else {
    const uint8_t* row = a.tree + b * a.tree_b + i * a.tree_i + j0;
    if (left >= 32 && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
      const uint4 lo = *reinterpret_cast<const uint4*>(row), hi = *reinterpret_cast<const uint4*>(row + 16);
      bits = nonzero_bytes(lo.x) | nonzero_bytes(lo.y) << 4 | nonzero_bytes(lo.z) << 8 | nonzero_bytes(lo.w) << 12 |
             nonzero_bytes(hi.x) << 16 | nonzero_bytes(hi.y) << 20 | nonzero_bytes(hi.z) << 24 |
             nonzero_bytes(hi.w) << 28;
    } else {
      uint8_t v[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] = e < left ? row[e] : 0;
#pragma unroll
      for (int e = 0; e < 32; ++e) bits |= v[e] != 0 ? 1u << e : 0u;
    }
  }
  if (left < 32) bits &= (1u << left) - 1u;
  if (a.window > 0 && bits != 0u) {
    int d[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) d[e] = e < left ? tree_depth(a, b, j0 + e) : 0;
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (static_cast<int64_t>(d[e]) <= static_cast<int64_t>(depth_i) - a.window && d[e] >= sink_left) bits &= ~(1u << e);
  }
  return bits;
}

// What a warp's rows see of the new tokens j0 .. j0 + 63, as bits: each lane brings its row's
// token (ascending over the lanes, -1 for none) and its depth.  The rows of a token share its
// line of the tree, which the warp reads once, a byte a lane (any alignment).  All lanes.
__device__ __forceinline__ void tree_sees64_rows(const TreeArgs& a, int b, int tok, int j0, int depth_i,
                                                 uint32_t (&keep)[2], int sink_left = kNoSinks) {
  const int lane = threadIdx.x & 31;
  keep[0] = keep[1] = 0u;
  const int j[2] = {j0 + lane, j0 + 32 + lane};
  int dj[2] = {0, 0};
  if (a.window > 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (j[h] < a.n) dj[h] = tree_depth(a, b, j[h]);
  }
  const int hi = __reduce_max_sync(0xffffffffu, tok);
  const int lo = __reduce_min_sync(0xffffffffu, tok < 0 ? INT32_MAX : tok);
#pragma unroll 4
  for (int t = lo; t <= hi; ++t) {  // (no row at all: lo > hi)
    const unsigned rows_of = __ballot_sync(0xffffffffu, tok == t);
    const int dt = __shfl_sync(0xffffffffu, depth_i, rows_of ? __ffs(rows_of) - 1 : 0);
    const uint8_t* line = a.tree != nullptr ? a.tree + b * a.tree_b + t * a.tree_i : nullptr;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bool on = j[h] < a.n;
      if (on) on = line != nullptr ? line[j[h]] != 0 : j[h] <= t;
      if (a.window > 0)
        on = on && (static_cast<int64_t>(dj[h]) > static_cast<int64_t>(dt) - a.window || dj[h] < sink_left);
      const uint32_t bits = __ballot_sync(0xffffffffu, on);
      if (tok == t) keep[h] = bits;
    }
  }
}

// The same for one row's new tokens j0 .. j0 + 15, in little code (it stands beside the common
// tiles, which have none of it).  All lanes, of the same j0.
__device__ __forceinline__ uint32_t tree_sees16(const TreeArgs& a, int b, int i, int j0, int depth_i,
                                                int sink_left = kNoSinks) {
  const int left = min(a.n - j0, 16);
  uint32_t bits = left <= 0 || i < 0 ? 0u : (1u << left) - 1u;
  if (a.tree == nullptr) {
    bits &= i < j0 ? 0u : (2u << min(i - j0, 15)) - 1u;
  } else if (bits != 0u) {
    const uint8_t* row = a.tree + b * a.tree_b + i * a.tree_i + j0;
    uint8_t v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = e < left ? row[e] : 0;
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (v[e] == 0) bits &= ~(1u << e);
  }
  if (a.window > 0) {
    const int e0 = threadIdx.x & 15;
    const int dj = e0 < left ? tree_depth(a, b, j0 + e0) : 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int d = __shfl_sync(0xffffffffu, dj, e);
      if (static_cast<int64_t>(d) <= static_cast<int64_t>(depth_i) - a.window && d >= sink_left) bits &= ~(1u << e);
    }
  }
  return bits;
}

// New tokens whose values are not all finite, one bit each; tokens 2048 apart share a bit, so
// a set bit only says that the token's values must be looked at.
constexpr int kPoisonWords = 64;
__device__ __forceinline__ uint32_t poison_of(const volatile uint32_t* words, int j0) {  // of j0 .. j0 + 31, j0 % 32 == 0
  return words[(j0 >> 5) & (kPoisonWords - 1)];
}

// Tiles of `bn` keys of one row tile of `bm` rows: committed tiles [c0, c1), then draft
// tiles [0, nd).
struct TreeSpan {
  int c0, c1, nd;
  int low;  // first committed slot that a row may see: what lies before it may hold anything
};
template <int bm, int bn>  // (powers of two)
__device__ __forceinline__ TreeSpan tree_span(const TreeArgs& a, int len, int rt) {
  TreeSpan s;
  const int rows = a.group * a.n;
  int i0, last, g;  // tokens of the first and last row
  tree_row(a, rt * bm, i0, g);
  tree_row(a, min((rt + 1) * bm, rows) - 1, last, g);
  // Without given depths the first row's token is the shallowest; with them, 0 is a bound.
  s.low = tree_first(a, len, a.depth != nullptr ? 0 : i0);
  s.c0 = static_cast<uint32_t>(s.low) / bn;
  s.c1 = static_cast<uint32_t>(len + bn - 1) / bn;
  // A causal chunk's row tile needs the new keys up to its last token only.
  if (a.tree != nullptr) last = a.n - 1;
  s.nd = static_cast<uint32_t>(last) / bn + 1;
  if (s.c0 > s.c1) s.c0 = s.c1;
  return s;
}

}  // namespace w8
