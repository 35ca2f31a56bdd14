// Attention of a tree of drafted tokens (or one token, or a causal chunk) over a cache:
// the decode counterpart of the prefill attention, replacing the cached-key calls of
// pipeline.py:133-180 and local_attn.py:44-83.
//
// Per sequence b and cache head c, the R = G N query rows (G = heads / kv_heads query heads
// of the group, N new tokens) share one stream of keys: the lens[b] committed slots of the
// cache, then the N new tokens' own keys:
//   x_rj = scale q_r . k_j,   p = softmax over the keys row r may see,   o_r = sum_j p_rj v_j
// with the softmax in one pass over the keys (running maximum m and sum l of each row, the
// output rescaled when m moves), fp32 scores, statistics and output sums; P is rounded to
// the operands' 16-bit type for the second product, as the prefill attention does (half a
// step of 2^-8 or 2^-11 on each weight, averaged over the keys).
//
// Decode reads every key once for few rows, so it is bound by HBM: R flops per byte for R
// rows against about 80 for the mma.sync rate over the copy rate.  One CTA of 8 warps owns
// a tile of 16 MT rows and a range of 64-key tiles.  K and V tiles stream through a
// cp.async ring (16-byte chunks, XOR-swizzled rows: ldmatrix without bank conflicts); in
// the S step each warp scores 8 keys for all rows, in the O step it owns D / 8 output
// columns, so both K and V fragments are read from shared memory once per row tile, and P
// and the row maxima cross warps through shared memory.
//
// The work is cut by what is there: all tiles of all sequences, in order, are dealt in equal
// contiguous ranges to as many CTAs as fit the GPU at once (every CTA adds up the lengths for
// itself), so ragged lengths leave no SM idle and a single long sequence fills them all.  A
// CTA writes the items that it holds whole, and partial (m, l, O) of at most two others, which
// attn_tree_combine_kernel joins.
#include "attention_tree.cuh"

#include <algorithm>

namespace w8 {

constexpr int kTreeThreads = 256;
constexpr int kTreeWarps = 8;
constexpr int kTreePPitch = 72;      // P row pitch (elements): 144 bytes, conflict-free ldmatrix

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x2_t(uint32_t addr, uint32_t (&r)[2]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(r[0]), "=r"(r[1])
               : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int D, int MT>
struct TreeCfg {
  static constexpr int kBM = 16 * MT;
  static constexpr int kBN = D == 512 ? 32 : 64;  // keys per tile: 16 to 64 KB of K and V each
  static constexpr int kSlotBytes = kBN * D * 2;
  static constexpr int kSlots = D == 512 ? 5 : D == 256 ? 3 : 6;
  static constexpr int kOffRing = kBM * D * 2;
  static constexpr int kOffP = kOffRing + kSlots * kSlotBytes;
  static constexpr int kOffRed = kOffP + kBM * kTreePPitch * 2;
  static constexpr int kOffPoison = kOffRed + kBM * kTreeWarps * 4;
  static constexpr int kSmem = kOffPoison + kPoisonWords * 4;
  static_assert(kSmem <= 232448, "shared memory budget exceeded");
};

// Sum over the block; `sm`: 16 words of shared memory, free again on return.
__device__ __forceinline__ long long block_sum(long long v, long long* sm) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  long long s = 0;
#pragma unroll
  for (int i = 0; i < kTreeWarps; ++i) s += sm[i];
  __syncthreads();
  return s;
}
// Exclusive prefix sum over the block and the block's sum.
__device__ __forceinline__ long long block_scan(long long v, long long* sm, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kTreeWarps; ++i) {
    if (i < warp) before += sm[i];
    total += sm[i];
  }
  __syncthreads();
  return before + x - v;
}

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kTreeThreads) attn_tree_kernel(const TreeArgs a) {
  using C = TreeCfg<D, MT>;
  constexpr int BM = C::kBM, BN = C::kBN, NS = C::kSlots, CH = D / 8;  // CH: 16-byte chunks per row
  constexpr int NT = D / 64;                              // n8 output tiles per warp
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sq = smem_u32(smem), ring = sq + C::kOffRing, sp = sq + C::kOffP;
  float* red = reinterpret_cast<float*>(smem + C::kOffRed);  // [BM][8]
  uint32_t* poison = reinterpret_cast<uint32_t*>(smem + C::kOffPoison);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = a.group * a.n;

  pdl_launch_dependents();
  pdl_wait();
  // ---- this CTA's range of all tiles.  A pair (sequence, row tile) has kv_heads items of
  // `tiles` tiles each; pairs and their heads follow one another.
  const int pairs = a.batch * a.row_tiles;
  auto pair_tiles = [&](int p) {
    const TreeSpan s = tree_span(a, tree_len(a, p / a.row_tiles), p % a.row_tiles, BM, BN);
    return s.c1 - s.c0 + s.nd;
  };
  long long* sched = reinterpret_cast<long long*>(smem + C::kOffRing);  // (the ring is not in use yet)
  long long mine = 0;
  for (int p = tid; p < pairs; p += kTreeThreads) mine += pair_tiles(p);
  const long long sum_tiles = block_sum(mine, sched);
  const long long total = sum_tiles * a.kv_heads;
  const long long ctas = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= ctas) return;
  long long pos = total * blockIdx.x / ctas;
  const long long stop = total * (blockIdx.x + 1) / ctas;
  // The pair that holds `pos`: a running sum over rounds of 256 pairs.
  long long before = 0;
  for (int p0 = 0;; p0 += kTreeThreads) {
    const int p = p0 + tid;
    const long long nt = p < pairs ? pair_tiles(p) : 0;
    long long round;
    const long long excl = before + block_scan(nt, sched, round);
    if (nt > 0 && excl * a.kv_heads <= pos && pos < (excl + nt) * a.kv_heads) {
      sched[16] = p;
      sched[17] = excl * a.kv_heads;
    }
    __syncthreads();
    before += round;
    if (pos < before * a.kv_heads) break;  // (every pair has tiles, and pos < total)
    if (p0 + kTreeThreads >= pairs) return;  // only if the lengths changed under the call
  }
  int pair = static_cast<int>(sched[16]);
  long long item_pos = sched[17];  // first tile of the current item
  __syncthreads();
  int b = pair / a.row_tiles, rt = pair % a.row_tiles;
  int len = tree_len(a, b);
  TreeSpan span = tree_span(a, len, rt, BM, BN);
  int nt = span.c1 - span.c0 + span.nd;
  int c = static_cast<int>((pos - item_pos) / nt);
  item_pos += static_cast<long long>(c) * nt;

  if (tid < kPoisonWords) poison[tid] = 0u;  // (ordered before its first use by the ring's barriers)
  while (true) {
    const int row0 = rt * BM, bc = b * a.kv_heads + c, nc = span.c1 - span.c0;
    const int t0 = static_cast<int>(pos - item_pos);
    const int t1 = static_cast<int>(stop - item_pos < nt ? stop - item_pos : nt);
    const bool whole = t0 == 0 && t1 == nt;
    const int64_t part_row = (2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0 ? 1 : 0)) * BM;
    if (t0 == 0 && tid == 0) {
      // The CTA that begins an item says where its pieces are: one in each CTA up to its last tile's.
      const long long last = ((item_pos + nt) * ctas - 1) / total;
      a.info[bc * a.row_tiles + rt] = make_int2(blockIdx.x, static_cast<int>(last - blockIdx.x) + 1);
    }

    // Row r = i * group + g: query head c * group + g of new token i.
    auto q_row = [&](int r) {
      int i, g;
      tree_row(a, r, i, g);
      return a.q + b * a.q_b + (static_cast<int64_t>(c) * a.group + g) * a.q_h + i * a.q_t;
    };
    for (int e = tid; e < BM * CH; e += kTreeThreads) {
      const int r = e / CH, ch = e % CH;
      const bool on = row0 + r < rows;
      cp_async16(sq + r * (D * 2) + ((ch ^ (r & 7)) << 4), (on ? q_row(row0 + r) : a.q) + ch * 8, on);
    }
    // Ring step g = 2 (tile - t0) + (0: K, 1: V).
    const int steps = 2 * (t1 - t0);
    auto load = [&](int g) {
      if (g < steps) {
        const int t = t0 + (g >> 1);
        const bool is_v = g & 1;
        const bool draft = t >= nc;
        const int key0 = (draft ? t - nc : span.c0 + t) * BN, end = draft ? a.n : len;
        const uint16_t* base;
        int64_t pitch;
        if (draft) {
          base = is_v ? a.vn + b * a.vn_b + c * a.vn_h : a.kn + b * a.kn_b + c * a.kn_h;
          pitch = is_v ? a.vn_t : a.kn_t;
        } else {
          base = is_v ? a.v + b * a.v_b + c * a.v_h : a.k + b * a.k_b + c * a.k_h;
          pitch = is_v ? a.v_s : a.k_s;
        }
        const uint32_t dst = ring + (g % NS) * C::kSlotBytes;
#pragma unroll
        for (int e = tid; e < BN * CH; e += kTreeThreads) {
          const int r = e / CH, ch = e % CH;
          const bool on = key0 + r < end;  // rows behind the end read as zeros
          cp_async16(dst + r * (D * 2) + ((ch ^ (r & 7)) << 4), base + (on ? (key0 + r) * pitch : 0) + ch * 8, on);
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int g = 0; g < NS - 1; ++g) load(g);

    // This thread's rows of each 16-row tile: lane / 4 and lane / 4 + 8.
    const int rl = lane >> 2;
    int tok[MT][2], first[MT][2], dep[MT][2];
    float m[MT][2], l[MT][2], corr[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row0 + mt * 16 + rl + 8 * h;
        tok[mt][h] = r < rows ? r / a.group : -1;
        dep[mt][h] = r < rows ? tree_depth(a, b, tok[mt][h]) : 0;
        first[mt][h] = r < rows ? tree_first(a, len, dep[mt][h]) : len;
        m[mt][h] = -INFINITY;
        l[mt][h] = 0.f;
        corr[mt][h] = 1.f;
      }
    float o[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;

    bool poisoned = false;  // a new token's V holds an infinity or NaN (in this CTA's tiles)
    for (int g = 0; g < steps; g += 2) {
      const int t = t0 + (g >> 1);
      const bool draft = t >= nc;
      const int key0 = (draft ? t - nc : span.c0 + t) * BN;
      // ---- S step
      cp_wait<NS - 2>();
      __syncthreads();
      load(g + NS - 1);
      const uint32_t sk = ring + (g % NS) * C::kSlotBytes;
      float s[MT][2][4];  // two chains of the reduction over D
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[mt][e >> 2][e & 3] = 0.f;
      const int krow = warp * 8 + (lane & 7), arow = lane & 15;
      const bool scores_here = warp < BN / 8;  // 8 keys a warp
      if (scores_here) {
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
        uint32_t kb[4];
        ldsm_x4(sk + krow * (D * 2) + (((4 * kk + (lane >> 3)) ^ (krow & 7)) << 4), kb);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t qa[4];
            const int r = mt * 16 + arow;
            ldsm_x4(sq + r * (D * 2) + (((4 * kk + 2 * h + (lane >> 4)) ^ (r & 7)) << 4), qa);
            mma16816<T>(s[mt][h], qa, kb[2 * h], kb[2 * h + 1]);
          }
      }
      }
      const int col = warp * 8 + (lane & 3) * 2;  // this thread's two keys of the tile
      float x[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1, key = key0 + col + (e & 1);
          bool on;
          if (!scores_here)
            on = false;
          else if (draft)
            on = tok[mt][h] >= 0 && key < a.n && tree_sees(a, b, tok[mt][h], key, dep[mt][h]);
          else
            on = key < len && key >= first[mt][h];
          x[mt][e] = on ? (s[mt][0][e] + s[mt][1][e]) * a.scale_log2 : -INFINITY;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(x[mt][2 * h], x[mt][2 * h + 1]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          if ((lane & 3) == 0) red[(mt * 16 + rl + 8 * h) * kTreeWarps + warp] = mx;
        }
      }
      if (a.scores != nullptr) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = row0 + mt * 16 + rl + 8 * h;
            if (r < rows && scores_here) {
              float* dst = a.scores + (static_cast<int64_t>(bc) * rows + r) * a.score_pitch +
                           (draft ? a.slots : 0) + key0 + col;
              const int left = (draft ? a.n : len) - key0 - col;
              if (left > 0) dst[0] = x[mt][2 * h];
              if (left > 1) dst[1] = x[mt][2 * h + 1];
            }
          }
      }
      __syncthreads();
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = mt * 16 + rl + 8 * h;
          const float4 lo = *reinterpret_cast<const float4*>(red + r * kTreeWarps);
          const float4 hi = *reinterpret_cast<const float4*>(red + r * kTreeWarps + 4);
          const float mx = fmaxf(fmaxf(fmaxf(lo.x, lo.y), fmaxf(lo.z, lo.w)),
                                 fmaxf(fmaxf(hi.x, hi.y), fmaxf(hi.z, hi.w)));
          const float mn = fmaxf(m[mt][h], mx);
          const float ref = mn == -INFINITY ? 0.f : mn;
          corr[mt][h] = ex2_tree(m[mt][h] - ref);
          m[mt][h] = mn;
          const float p0 = ex2_tree(x[mt][2 * h] - ref), p1 = ex2_tree(x[mt][2 * h + 1] - ref);
          l[mt][h] = l[mt][h] * corr[mt][h] + (p0 + p1);
          *reinterpret_cast<uint32_t*>(smem + C::kOffP + (r * kTreePPitch + col) * 2) = pack2<T>(p0, p1);
        }
      // ---- O step
      cp_wait<NS - 2>();
      __syncthreads();
      load(g + NS);
      const uint32_t sv = ring + ((g + 1) % NS) * C::kSlotBytes;
      if (draft) {
        // A new token's values may be infinite or NaN where some row must not see them, and
        // 0 * NaN is NaN in the product: take them out here, and add them at the end to the
        // rows that do see them.
        bool any = false;
        for (int e = tid; e < BN * CH; e += kTreeThreads) {
          bool bad = false;
          uint32_t* w = reinterpret_cast<uint32_t*>(smem + C::kOffRing + ((g + 1) % NS) * C::kSlotBytes) + e * 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t v = w[i];
            const bool lo = tree_nonfinite<T>(v), hi = tree_nonfinite<T>(v >> 16);
            if (lo || hi) {
              w[i] = (lo ? 0u : v & 0xFFFFu) | (hi ? 0u : v & 0xFFFF0000u);
              bad = true;
            }
          }
          if (bad) {
            poison_mark(poison, key0 + e / CH);
            any = true;
          }
        }
        if (__syncthreads_or(any)) poisoned = true;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (__any_sync(0xffffffffu, corr[mt][0] != 1.f || corr[mt][1] != 1.f)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[mt][n][0] *= corr[mt][0];
            o[mt][n][1] *= corr[mt][0];
            o[mt][n][2] *= corr[mt][1];
            o[mt][n][3] *= corr[mt][1];
          }
        }
      }
#pragma unroll
      for (int ks = 0; ks < BN / 16; ++ks) {
        uint32_t pa[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          ldsm_x4(sp + ((mt * 16 + arow) * kTreePPitch + ks * 16 + (lane >> 4) * 8) * 2, pa[mt]);
        const int vr = ks * 16 + (lane & 15);
        if constexpr (NT == 1) {
          uint32_t vb[2];
          ldsm_x2_t(sv + vr * (D * 2) + (((warp * NT) ^ (vr & 7)) << 4), vb);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mma16816<T>(o[mt][0], pa[mt], vb[0], vb[1]);
        } else {
#pragma unroll
          for (int n = 0; n < NT; n += 2) {
            uint32_t vb[4];
            ldsm_x4_t(sv + vr * (D * 2) + (((warp * NT + n + (lane >> 4)) ^ (vr & 7)) << 4), vb);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma16816<T>(o[mt][n], pa[mt], vb[0], vb[1]);
              mma16816<T>(o[mt][n + 1], pa[mt], vb[2], vb[3]);
            }
          }
        }
      }
    }
    cp_wait<0>();
    if (poisoned) {
      const int j0 = (max(t0, nc) - nc) * BN, j1 = min((t1 - nc) * BN, a.n);
#pragma unroll 1
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll 1
        for (int h = 0; h < 2; ++h)
          if (tok[mt][h] >= 0)
#pragma unroll 1
            for (int jw = j0; jw < j1; jw += 32) {
              uint32_t bits = poison_of(poison, jw);
              if (bits != 0u) bits &= tree_sees32(a, b, tok[mt][h], jw, dep[mt][h]);
#pragma unroll 1
              for (; bits != 0u; bits &= bits - 1u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const uint16_t v = a.vn[b * a.vn_b + c * a.vn_h + (jw + __ffs(bits) - 1) * a.vn_t + warp * (D / 8) +
                                            n * 8 + (lane & 3) * 2 + e];
                    // (static register indexes only: both rows are written under a select)
                    const float add = tree_nonfinite<T>(v) ? tree_f32<T>(v) : 0.f;
#pragma unroll
                    for (int mm = 0; mm < MT; ++mm) {
                      if (mm == mt && h == 0) o[mm][n][e] += add;
                      if (mm == mt && h == 1) o[mm][n][2 + e] += add;
                    }
                  }
            }
    }

    // ---- row sums over the warps, then the output or this split's partial
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v = l[mt][h];
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        if ((lane & 3) == 0) red[(mt * 16 + rl + 8 * h) * kTreeWarps + warp] = v;
      }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = mt * 16 + rl + 8 * h;
        if (row0 + r >= rows) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kTreeWarps; ++w) sum += red[r * kTreeWarps + w];
        const int cols = warp * (D / 8) + (lane & 3) * 2;
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing: zeros
          const int i = (row0 + r) / a.group, gq = (row0 + r) % a.group;
          uint16_t* dst = a.o + b * a.o_b + (static_cast<int64_t>(c) * a.group + gq) * a.o_h + i * a.o_t + cols;
#pragma unroll
          for (int n = 0; n < NT; ++n)
            *reinterpret_cast<uint32_t*>(dst + n * 8) = pack2<T>(o[mt][n][2 * h] * inv, o[mt][n][2 * h + 1] * inv);
          if (a.lse != nullptr && warp == 0 && (lane & 3) == 0)
            a.lse[static_cast<int64_t>(bc) * rows + row0 + r] = sum == 0.f ? INFINITY : m[mt][h] + log2f(sum);
        } else {
          float* dst = a.part_o + (part_row + r) * D + cols;
#pragma unroll
          for (int n = 0; n < NT; ++n)
            *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
          if (warp == 0 && (lane & 3) == 0) a.part_ml[part_row + r] = make_float2(m[mt][h], sum);
        }
      }
    pos += t1 - t0;
    if (pos >= stop) break;
    // ---- the next item: the next head, or the next pair's first
    item_pos += nt;
    if (++c == a.kv_heads) {
      c = 0;
      if (++rt == a.row_tiles) {
        rt = 0;
        ++b;
        len = tree_len(a, b);
      }
      span = tree_span(a, len, rt, BM, BN);
      nt = span.c1 - span.c0 + span.nd;
    }
    __syncthreads();  // everybody has left the ring, Q and the row sums
    if (poisoned && tid < kPoisonWords) poison[tid] = 0u;
  }
}

// Joins the pieces of one row: M = max m_s, o = sum 2^(m_s - M) O_s / sum 2^(m_s - M) l_s.
// One CTA per row and 128 (64) columns: 4 columns a thread, the pieces over thread groups.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_tree_combine_kernel(const TreeArgs a, int bm) {
  constexpr int kCols = D < 128 ? D : 128, kLanes = kCols / 4, kGroups = 256 / kLanes;
  __shared__ float w[kTreeMaxPieces];
  __shared__ float4 acc[kGroups][kLanes];
  __shared__ float wmax[8], wsum[8];
  const int rows = a.group * a.n;
  const int64_t row = blockIdx.x;
  const int bc = static_cast<int>(row / rows), r = static_cast<int>(row % rows);
  const int64_t item = static_cast<int64_t>(bc) * a.row_tiles + r / bm;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x;
  const bool dealt = a.info != nullptr;
  const int2 info = dealt ? a.info[item] : make_int2(0, a.splits);
  const int pieces = info.y;
  if (pieces <= 1) return;  // written whole
  auto slot = [&](int s) { return dealt ? tree_slot(info, s) : item * a.splits + s; };
  float2 ml[kTreeMaxPieces / 256];
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < kTreeMaxPieces / 256; ++i) {
    const int s = tid + 256 * i;
    ml[i] = s < pieces ? a.part_ml[slot(s) * bm + r % bm] : make_float2(-INFINITY, 0.f);
    mx = fmaxf(mx, ml[i].x);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  if ((tid & 31) == 0) wmax[tid >> 5] = mx;
  __syncthreads();
  mx = wmax[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) mx = fmaxf(mx, wmax[i]);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kTreeMaxPieces / 256; ++i) {
    const float f = ml[i].x == -INFINITY ? 0.f : ex2_tree(ml[i].x - mx);
    if (tid + 256 * i < pieces) {
      w[tid + 256 * i] = f;
      sum += f * ml[i].y;
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if ((tid & 31) == 0) wsum[tid >> 5] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += wsum[i];
  const int ln = tid % kLanes, grp = tid / kLanes;
  const int col = blockIdx.y * kCols + ln * 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = grp; s < pieces; s += kGroups) {
    const float ws = w[s];
    if (ws != 0.f) {  // a piece without keys left its rows unwritten (NaN weights pass)
      const float4 p = *reinterpret_cast<const float4*>(a.part_o + (slot(s) * bm + r % bm) * D + col);
      v.x += ws * p.x, v.y += ws * p.y, v.z += ws * p.z, v.w += ws * p.w;
    }
  }
  acc[grp][ln] = v;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int i = 1; i < kGroups; ++i) {
      const float4 p = acc[i][ln];
      v.x += p.x, v.y += p.y, v.z += p.z, v.w += p.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int b = bc / a.kv_heads, c = bc % a.kv_heads, i = r / a.group, gq = r % a.group;
    uint16_t* dst = a.o + b * a.o_b + (static_cast<int64_t>(c) * a.group + gq) * a.o_h + i * a.o_t + col;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
    if (a.lse != nullptr && tid == 0 && blockIdx.y == 0)
      a.lse[row] = sum == 0.f ? INFINITY : mx + log2f(sum);
  }
}

// Accumulated weights: slot j gets weights[j] + sum over the R rows of p_rj, p from the stored
// scores and the rows' log-sum-exp (the sums in the rows' order: the same bits every time).
__global__ void __launch_bounds__(256) attn_tree_weights_kernel(const TreeArgs a) {
  extern __shared__ float sm[];
  const int rows = a.group * a.n, bc = blockIdx.y, b = bc / a.kv_heads, c = bc % a.kv_heads;
  pdl_launch_dependents();
  pdl_wait();
  const int len = tree_len(a, b);
  const int j = blockIdx.x * 256 + threadIdx.x;  // slots [0, S), then drafts
  if (blockIdx.x * 256 >= len && (blockIdx.x + 1) * 256 <= a.slots) return;
  const bool draft = j >= a.slots;
  const bool on = draft ? j - a.slots < a.n : j < len;
  const float* x = a.scores + static_cast<int64_t>(bc) * rows * a.score_pitch + j;
  const float* lse = a.lse + static_cast<int64_t>(bc) * rows;
  float sum = 0.f;
  for (int r0 = 0; r0 < rows; r0 += 256) {
    // (lse, first visible slot) of up to 256 rows at a time
    __syncthreads();
    if (r0 + threadIdx.x < rows) {
      const int r = r0 + threadIdx.x, i = r / a.group;
      sm[threadIdx.x] = lse[r];
      reinterpret_cast<int*>(sm + 256)[threadIdx.x] = tree_first(a, len, tree_depth(a, b, i));
    }
    __syncthreads();
    if (on) {
      const int n = min(256, rows - r0);
#pragma unroll 4
      for (int q = 0; q < n; ++q) {
        const int i = (r0 + q) / a.group;
        // Keys that no tile of the row covered were never scored.
        const bool seen = draft ? (a.tree != nullptr || j - a.slots <= i)
                                : j >= reinterpret_cast<const int*>(sm + 256)[q];
        if (seen) sum += ex2_tree(x[static_cast<int64_t>(r0 + q) * a.score_pitch] - sm[q]);
      }
    }
  }
  if (!on) return;
  if (draft)
    a.w_new[static_cast<int64_t>(bc) * a.n + j - a.slots] = sum;
  else
    a.w_out[b * a.wo_b + c * a.wo_h + j] = a.w_in[b * a.wi_b + c * a.wi_h + j] + sum;
}

}  // namespace w8

namespace w8host {

int require_sm100(int* device);

int tree_tc(const w8::TreeArgs& a, bool half, int64_t d, int64_t items, int device, cudaStream_t stream);
int tree_tc_device_status(int clear, int* out);

// How a call is cut: rows per tile, row tiles, and over the keys a number of splits (tcgen05)
// or of CTAs that share all tiles (mma.sync).
struct TreePlan {
  bool tc;  // the tcgen05 schedule (attention_tree_tc.cu)
  int bm, row_tiles, splits, ctas;
  int64_t items;
};

// More than 32 rows a cache head at head_dim >= 128 go to the tcgen05 schedule (`tma`: its
// maps can describe the tensors), whose tiles take 256 rows; fewer to mma.sync tiles of 16
// or 32, which a split key axis spreads over more SMs.
static TreePlan tree_plan(int64_t batch, int64_t kv_heads, int64_t group, int64_t n, int64_t d, int64_t slots,
                          int64_t window, int sms, bool tma) {
  TreePlan p;
  const int64_t rows = group * n;
  p.tc = tma && rows > 32 && d >= 128;
  p.bm = p.tc ? 256 : rows > 16 && d <= 256 ? 32 : 16;
  p.row_tiles = static_cast<int>((rows + p.bm - 1) / p.bm);
  p.items = batch * kv_heads * p.row_tiles;
  // Keys of one row tile: with a window, those its tokens see.
  const int64_t bn = p.tc ? 128 : d == 512 ? 32 : 64;
  const int64_t tokens = std::min(n, p.bm / group + 2);
  const int64_t keys = window > 0 ? std::min(slots, window + tokens) : slots;
  const int64_t tiles = (keys + bn - 1) / bn + (n + bn - 1) / bn;
  p.splits = 1;
  if (p.tc) {
    // The number of splits with the least estimated time: waves of clusters, each 1.6 us a tile
    // and 8 us besides, then 4 us and the partials at 3 TB/s to join them (measured on trees
    // of 64 drafts at D 256).
    const int64_t width = d == 512 ? 2 : 1, pairs = sms / 2;
    double best = 0;
    for (int64_t s = 1; s <= std::min<int64_t>(tiles, 64); ++s) {
      const double waves = static_cast<double>((p.items * width * s + pairs - 1) / pairs);
      double us = waves * (1.6 * static_cast<double>((tiles + s - 1) / s) + 8);
      if (s > 1) us += 4 + static_cast<double>(p.items * p.bm * d) * 8 * static_cast<double>(s) / 3e6;
      if (s == 1 || us < best) best = us, p.splits = static_cast<int>(s);
    }
    p.ctas = 0;
  } else {
    // What fits at once by shared memory and registers (attn_tree_kernel).
    const int64_t per_sm = d == 512 || (d == 256 && p.bm == 32) ? 1 : d == 64 ? 3 : 2;
    p.ctas = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({sms * per_sm, p.items * tiles, w8::kTreeMaxPieces})));
  }
  return p;
}

struct TreeWs {
  int64_t part_o, part_ml, info, lse, scores, total, score_pitch;
};
static TreeWs tree_ws(const TreePlan& p, int64_t batch, int64_t kv_heads, int64_t group, int64_t n, int64_t d,
                      int64_t slots, bool weights) {
  TreeWs w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  const int64_t part_rows = p.tc ? (p.splits > 1 ? p.items * p.splits * p.bm : 0) : 2 * static_cast<int64_t>(p.ctas) * p.bm;
  w.part_o = take(part_rows * d * 4);
  w.part_ml = take(part_rows * 8);
  w.info = take(p.tc ? 0 : p.items * 8);
  const int64_t rows = batch * kv_heads * group * n;
  w.score_pitch = (slots + n + 3) / 4 * 4;
  w.lse = take(weights ? rows * 4 : 0);
  w.scores = take(weights ? rows * w.score_pitch * 4 : 0);
  w.total = at;
  return w;
}

static int tree_shape(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t slots, int64_t n,
                      int64_t window) {
  W8_CHECK_ARG(batch >= 0 && heads >= 1 && kv_heads >= 1 && slots >= 0 && n >= 0, "negative size");
  W8_CHECK_ARG(heads % kv_heads == 0, "heads %lld must be a multiple of kv_heads %lld", (long long)heads,
               (long long)kv_heads);
  W8_CHECK_ARG(window >= 0 && window < (1ll << 31), "window must be 0 (none) or positive, below 2^31");
  W8_CHECK_ARG(slots < (1ll << 30) && n <= 65536 && batch <= (1ll << 20) && heads <= 65536, "size beyond the limits");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512) {
    set_error("head_dim %lld is not 64, 128, 256 or 512", (long long)head_dim);
    return W8_ERR_UNSUPPORTED;
  }
  return W8_OK;
}

template <typename Kern, typename... Args>
static int launch_tree(Kern kern, dim3 grid, int threads, int smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, args...));
}

template <typename T, int D, int MT>
static int tree_main(const w8::TreeArgs& a, int64_t blocks, int device, cudaStream_t stream) {
  using C = w8::TreeCfg<D, MT>;
  static bool done[64] = {};
  if (!done[device]) {
    W8_CUDA_TRY(cudaFuncSetAttribute(w8::attn_tree_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     C::kSmem));
    done[device] = true;
  }
  return launch_tree(w8::attn_tree_kernel<T, D, MT>, dim3(static_cast<unsigned>(blocks)), w8::kTreeThreads, C::kSmem,
                     stream, a);
}

template <typename T, int D>
static int tree_go(const w8::TreeArgs& a, const TreePlan& p, int device, cudaStream_t stream) {
  W8_CHECK_ARG(p.items < (1ll << 31) / 2, "too many row tiles");
  const int64_t blocks = p.ctas;
  int st;
  if (p.tc)
    st = tree_tc(a, __is_same(T, __half), D, p.items, device, stream);
  else if constexpr (D <= 256)
    st = p.bm == 32 ? tree_main<T, D, 2>(a, blocks, device, stream) : tree_main<T, D, 1>(a, blocks, device, stream);
  else
    st = tree_main<T, D, 1>(a, blocks, device, stream);
  if (st != W8_OK) return st;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.kv_heads * a.group * a.n;
  if (p.tc ? p.splits > 1 : p.ctas > 1) {
    st = launch_tree(w8::attn_tree_combine_kernel<T, D>,
                     dim3(static_cast<unsigned>(rows), static_cast<unsigned>(D < 128 ? 1 : D / 128)), 256, 0, stream, a,
                     p.bm);
    if (st != W8_OK) return st;
  }
  if (a.scores != nullptr) {
    const int64_t blocks_w = (a.slots + a.n + 255) / 256;
    st = launch_tree(w8::attn_tree_weights_kernel,
                     dim3(static_cast<unsigned>(blocks_w), static_cast<unsigned>(a.batch * a.kv_heads)), 256, 2048,
                     stream, a);
  }
  return st;
}

// Read (and optionally clear) the sticky device status of the cache attention.
int tree_device_status(int clear, int* out) {
  int v = 0;
  W8_CUDA_TRY(cudaMemcpyFromSymbol(&v, w8::g_tree_status, sizeof(int)));
  if (clear) {
    const int zero = 0;
    W8_CUDA_TRY(cudaMemcpyToSymbol(w8::g_tree_status, &zero, sizeof(int)));
  }
  int vt = W8_OK;
  const int st = tree_tc_device_status(clear, &vt);
  if (st != W8_OK) return st;
  *out = v == W8_OK || vt == W8_ERR_DEVICE_TIMEOUT ? vt : v;
  return W8_OK;
}

}  // namespace w8host

extern "C" int64_t w8_attention_tree_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                     int64_t slots, int64_t n_new, int64_t window, int weights) {
  using namespace w8host;
  if (tree_shape(batch, heads, kv_heads, head_dim, slots, n_new, window) != W8_OK) return -1;
  int sms = 148;
  if (num_sms(&sms) != W8_OK) sms = 148;
  // The larger of the two schedules' needs: which one runs depends on the strides too.
  int64_t most = 0;
  for (const bool tma : {false, true}) {
    const TreePlan p = tree_plan(batch, kv_heads, heads / kv_heads, n_new, head_dim, slots, window, sms, tma);
    most = std::max(most, tree_ws(p, batch, kv_heads, heads / kv_heads, n_new, head_dim, slots, weights != 0).total);
  }
  return most;
}

extern "C" int w8_attention_tree(const w8_attention_tree_args* in, void* workspace, int64_t workspace_bytes,
                                 w8_stream_t stream) {
  using namespace w8host;
  W8_CHECK_ARG(in != nullptr, "null arguments");
  const w8_attention_tree_args& x = *in;
  int st = tree_shape(x.batch, x.heads, x.kv_heads, x.head_dim, x.slots, x.n_new, x.window);
  if (st != W8_OK) return st;
  W8_CHECK_ARG(x.dtype == W8_BF16 || x.dtype == W8_FP16, "dtype must be W8_BF16 or W8_FP16");
  if (x.batch == 0 || x.n_new == 0) return W8_OK;
  // (positive in the kernels' fp32 log2 units too: a masked score is -inf times it)
  const float scale_log2 = static_cast<float>(x.scale * 1.4426950408889634);
  W8_CHECK_ARG(scale_log2 > 0.f && scale_log2 < 3e38f, "scale must be positive and finite");
  W8_CHECK_ARG(x.q && x.k_new && x.v_new && x.out && x.lens, "null pointer");
  W8_CHECK_ARG(x.slots == 0 || (x.k && x.v), "null cache");
  W8_CHECK_ARG(x.tree == nullptr || x.window == 0 || x.depth != nullptr,
               "a tree with a window needs the tokens' depths");
  const bool weights = x.weights != nullptr || x.weights_out != nullptr || x.draft_weights != nullptr;
  W8_CHECK_ARG(!weights || (x.draft_weights && (x.slots == 0 || (x.weights && x.weights_out))),
               "weights, weights_out and draft_weights come together");
  const void* ptrs[6] = {x.q, x.k, x.v, x.k_new, x.v_new, x.out};
  const int64_t* strides[6] = {x.q_stride, x.k_stride, x.v_stride, x.k_new_stride, x.v_new_stride, x.out_stride};
  for (int i = 0; i < 6; ++i) {
    W8_CHECK_ALIGN(aligned(ptrs[i], 16), "q, k, v, k_new, v_new and out must be 16-byte aligned");
    for (int j = 0; j < 3; ++j)
      W8_CHECK_ALIGN(strides[i][j] % 8 == 0, "the strides of q, k, v, k_new, v_new and out must be multiples of 8");
  }
  int device = 0, sms = 0;
  st = require_sm100(&device);
  if (st != W8_OK) return st;
  st = num_sms(&sms);
  if (st != W8_OK) return st;
  const int64_t group = x.heads / x.kv_heads;
  // TMA maps take no stride of 0 (an expanded view: beams that share one prompt's cache).
  const int64_t sizes[4][3] = {{x.batch, x.kv_heads, x.slots}, {x.batch, x.kv_heads, x.slots},
                               {x.batch, x.kv_heads, x.n_new}, {x.batch, x.kv_heads, x.n_new}};
  bool tma = true;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 3; ++j)
      if (sizes[i][j] > 1 && (strides[i + 1][j] <= 0 || strides[i + 1][j] >= (1ll << 38))) tma = false;
  const TreePlan p = tree_plan(x.batch, x.kv_heads, group, x.n_new, x.head_dim, x.slots, x.window, sms, tma);
  const TreeWs w = tree_ws(p, x.batch, x.kv_heads, group, x.n_new, x.head_dim, x.slots, weights);
  W8_CHECK_ARG(w.total == 0 || (workspace != nullptr && workspace_bytes >= w.total),
               "workspace of %lld bytes needed (got %lld)", (long long)w.total, (long long)workspace_bytes);
  W8_CHECK_ALIGN(aligned(workspace, 16), "workspace must be 16-byte aligned");
  W8_CHECK_ARG(!weights || x.batch * x.kv_heads <= 65535, "batch * kv_heads beyond 65535 with weights");
  W8_CHECK_ARG(x.batch * x.heads * x.n_new < (1ll << 31), "too many query rows");
  w8::TreeArgs a = {};
  a.q = static_cast<const uint16_t*>(x.q);
  a.k = static_cast<const uint16_t*>(x.k);
  a.v = static_cast<const uint16_t*>(x.v);
  a.kn = static_cast<const uint16_t*>(x.k_new);
  a.vn = static_cast<const uint16_t*>(x.v_new);
  a.o = static_cast<uint16_t*>(x.out);
  a.lens = x.lens;
  a.tree = x.tree;
  a.depth = x.depth;
  a.q_b = x.q_stride[0], a.q_h = x.q_stride[1], a.q_t = x.q_stride[2];
  a.k_b = x.k_stride[0], a.k_h = x.k_stride[1], a.k_s = x.k_stride[2];
  a.v_b = x.v_stride[0], a.v_h = x.v_stride[1], a.v_s = x.v_stride[2];
  a.kn_b = x.k_new_stride[0], a.kn_h = x.k_new_stride[1], a.kn_t = x.k_new_stride[2];
  a.vn_b = x.v_new_stride[0], a.vn_h = x.v_new_stride[1], a.vn_t = x.v_new_stride[2];
  a.o_b = x.out_stride[0], a.o_h = x.out_stride[1], a.o_t = x.out_stride[2];
  a.tree_b = x.tree_stride[0], a.tree_i = x.tree_stride[1];
  a.depth_b = x.depth_stride;
  a.batch = static_cast<int>(x.batch);
  a.kv_heads = static_cast<int>(x.kv_heads);
  a.group = static_cast<int>(group);
  a.group_rcp = group > 1 ? static_cast<uint32_t>((1ull << 32) / static_cast<uint64_t>(group)) : 0u;
  a.n = static_cast<int>(x.n_new);
  a.slots = static_cast<int>(x.slots);
  a.window = static_cast<int>(x.window);
  a.scale_log2 = scale_log2;
  a.row_tiles = p.row_tiles;
  a.splits = p.splits;
  // Boxes of 128 query rows: the group divides 128, and no stride of 0.
  a.q_tma = group <= 128 && (group & (group - 1)) == 0;
  const int64_t q_sizes[3] = {x.batch, x.heads, x.n_new};
  for (int j = 0; j < 3; ++j)
    if (q_sizes[j] > 1 && (x.q_stride[j] <= 0 || x.q_stride[j] >= (1ll << 38))) a.q_tma = 0;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(ws + w.part_o);
  a.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
  a.info = p.tc ? nullptr : reinterpret_cast<int2*>(ws + w.info);
  if (weights) {
    a.lse = reinterpret_cast<float*>(ws + w.lse);
    a.scores = reinterpret_cast<float*>(ws + w.scores);
    a.score_pitch = w.score_pitch;
    a.w_in = x.weights;
    a.w_out = x.weights_out;
    a.w_new = x.draft_weights;
    a.wi_b = x.weights_stride[0], a.wi_h = x.weights_stride[1];
    a.wo_b = x.weights_out_stride[0], a.wo_h = x.weights_out_stride[1];
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = x.dtype == W8_BF16;
  switch (x.head_dim) {
    case 64:
      return bf ? tree_go<__nv_bfloat16, 64>(a, p, device, s) : tree_go<__half, 64>(a, p, device, s);
    case 128:
      return bf ? tree_go<__nv_bfloat16, 128>(a, p, device, s) : tree_go<__half, 128>(a, p, device, s);
    case 256:
      return bf ? tree_go<__nv_bfloat16, 256>(a, p, device, s) : tree_go<__half, 256>(a, p, device, s);
    default:
      return bf ? tree_go<__nv_bfloat16, 512>(a, p, device, s) : tree_go<__half, 512>(a, p, device, s);
  }
}
