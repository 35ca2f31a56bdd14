// Shared by the kernels of attention over a paged 8-bit cache: their arguments, and the tiles
// of keys that a row tile reads.
//
// Position p of a sequence lies in page table[p / P] (P tokens of every cache head) while that
// page is full: 8-bit values of one scale for keys and one for values a page and head.  The
// positions of the last, partial page are 16-bit rows of the sequence's tail; then come the
// new tokens.
#pragma once

#include "attention_tree.cuh"

namespace w8 {

struct PagedArgs {
  TreeArgs t;  // q, new tokens, out, lengths, tree, window, sink, pieces; slots = table_pages * P
  const int* table;
  int64_t table_b;
  int table_pages, pages, shift;  // P = 1 << shift
  const float *ks, *vs;           // [pages, KV]
  int64_t ks_p, ks_h, vs_p, vs_h;
};

constexpr int kPagedMaxBoxes = 16;  // pages (or parts of one) of a tile

// The tiles of one row tile, in order: `ns` of pages that hold sinks before the window, pages
// [c0, c1) in tiles of bn keys, `tail` and `nd` of new tokens in tiles of bn16 keys.
struct PagedSpan {
  int ns, c0, c1, tail, nd;
  int full;  // positions in full pages
  int low;   // first committed position that a row may see under the window
  __device__ __forceinline__ int pages() const { return ns + c1 - c0; }
  __device__ __forceinline__ int tiles() const { return ns + c1 - c0 + tail + nd; }
};
template <int bm, int bn, int bn16>  // (bn, bn16 powers of two)
__device__ __forceinline__ PagedSpan paged_span(const PagedArgs& a, int len, int rt) {
  PagedSpan s;
  const TreeArgs& t = a.t;
  const int rows = t.group * t.n;
  int i0, last, g;  // tokens of the first and last row
  tree_row(t, rt * bm, i0, g);
  tree_row(t, min((rt + 1) * bm, rows) - 1, last, g);
  s.full = (len >> a.shift) << a.shift;
  // Without given depths the first row's token is the shallowest; with them, 0 is a bound.
  s.low = tree_first(t, len, t.depth != nullptr ? 0 : i0);
  s.c1 = static_cast<uint32_t>(s.full + bn - 1) / bn;
  s.c0 = min(static_cast<int>(static_cast<uint32_t>(s.low) / bn), s.c1);
  s.ns = t.window > 0 ? min(static_cast<int>(static_cast<uint32_t>(min(t.sink, s.full) + bn - 1) / bn), s.c0) : 0;
  s.tail = static_cast<uint32_t>(len - s.full + bn16 - 1) / bn16;
  // A causal chunk's row tile needs the new keys up to its last token only.
  if (t.tree != nullptr) last = t.n - 1;
  s.nd = static_cast<uint32_t>(last) / bn16 + 1;
  return s;
}

// Whether some row of the tile may see a position of [p0, p1) of the full pages.
__device__ __forceinline__ bool paged_needs(const PagedArgs& a, const PagedSpan& s, int p0, int p1) {
  return p0 < s.full && (p1 > s.low || p0 < a.t.sink);
}

// 4 values of 8 bits (two's complement) as two pairs of T, bytes 0 and 1, 2 and 3 (`kPairs` 0x4140,
// 0x4342) or 0 and 2, 1 and 3 (0x4240, 0x4341).  Exact.  fp16: the byte plus 128 as the low bits of
// 1024 + x, less 1152.  bf16 has 7 of those bits: 128 + (x mod 128), less 128 or, of a negative x, 256.
template <typename T>
__device__ __forceinline__ void paged_unpack(uint32_t x, uint32_t sel0, uint32_t sel1, uint32_t& p0, uint32_t& p1);
template <>
__device__ __forceinline__ void paged_unpack<__half>(uint32_t x, uint32_t sel0, uint32_t sel1, uint32_t& p0,
                                                     uint32_t& p1) {
  const uint32_t u = x ^ 0x80808080u;
  const uint32_t bias = 0x64806480u;
  const __half2 b = *reinterpret_cast<const __half2*>(&bias);
  uint32_t w0 = __byte_perm(u, 0x64646464u, sel0), w1 = __byte_perm(u, 0x64646464u, sel1);
  const __half2 h0 = __hsub2(*reinterpret_cast<__half2*>(&w0), b), h1 = __hsub2(*reinterpret_cast<__half2*>(&w1), b);
  p0 = *reinterpret_cast<const uint32_t*>(&h0);
  p1 = *reinterpret_cast<const uint32_t*>(&h1);
}
template <>
__device__ __forceinline__ void paged_unpack<__nv_bfloat16>(uint32_t x, uint32_t sel0, uint32_t sel1, uint32_t& p0,
                                                            uint32_t& p1) {
  auto one = [&](uint32_t sel) {
    const uint32_t w = __byte_perm(x, 0u, sel);
    const uint32_t up = (w & 0x007F007Fu) | 0x43004300u, down = (w & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&up),
                                     *reinterpret_cast<const __nv_bfloat162*>(&down));
    return *reinterpret_cast<const uint32_t*>(&h);
  };
  p0 = one(sel0);
  p1 = one(sel1);
}

// The same less 1152 still to be taken off, in fp16: 1024 + 128 + x.
__device__ __forceinline__ void paged_raise(uint32_t x, uint32_t sel0, uint32_t sel1, uint32_t& p0, uint32_t& p1) {
  const uint32_t u = x ^ 0x80808080u;
  p0 = __byte_perm(u, 0x64646464u, sel0);
  p1 = __byte_perm(u, 0x64646464u, sel1);
}

// The smallest power of two that is not below a scale (of 2^-126 to 2^126), and its reciprocal:
// the unit in which the sums of values are held while pages of different scales add to them.
__device__ __forceinline__ float paged_unit(float scale) {
  uint32_t e = (__float_as_uint(scale) + 0x007FFFFFu) & 0x7F800000u;
  e = min(max(e, 0x00800000u), 0x7E800000u);  // (a NaN or an infinity shows in the products)
  return __uint_as_float(e);
}
__device__ __forceinline__ float paged_unit_rcp(float unit) { return __uint_as_float(0x7F000000u - __float_as_uint(unit)); }

}  // namespace w8
