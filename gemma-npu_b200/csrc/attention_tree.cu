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
// step of 2^-8 or 2^-11 on each weight, averaged over the keys; TreeRef has fp16's range).
//
// Decode reads every key once for few rows, so it is bound by HBM: R flops per byte for R
// rows against about 80 for the mma.sync rate over the copy rate.  A CTA owns 16 MT rows and
// a range of tiles of 64 to 256 keys (32 to 64 KB boxes, which the TMA moves at full rate),
// streamed through a ring.  Each of its 8 warps (a team of two at D = 512, half of the output
// columns each) takes 16 keys at a time for all rows, with a running maximum, sum and output of
// its own: S = Q K^T, the softmax and O += P V stay in its registers, P turning from the
// accumulator's layout into the operand's in place, and no warp waits for another until the end
// of the item, where the 8 results are joined.  (Warps that shared each tile, exchanging P and
// the maxima through shared memory with three barriers a tile, executed 6 times the
// instructions.)  32 sequences of 2048 to 8191 keys, 8 heads of 128 (671 MB) take 112 us with the
// joining of their pieces, 6.0 TB/s; of 8191 keys each 162 us, 6.6 TB/s, heads of 256 6.7 TB/s.
//
// The work is cut by what is there: all tiles of all sequences, in order, are dealt in equal
// contiguous ranges to as many CTAs as fit the GPU at once (every CTA adds up the lengths for
// itself), so ragged lengths leave no SM idle and a single long sequence fills them all.  A
// CTA writes the items that it holds whole, and partial (m, l, O) of at most two others, which
// attn_tree_combine_kernel joins.  (A cache that sequences share by expansion has no tensor map and
// is read by cp.async, once for every sequence: 40 sequences over one cache of 4000 slots, 8 heads of
// 128, take 167 us where 40 caches of their own take 106.)
#include "attention_tree.cuh"
#include "attn_mma.cuh"
#include "attn_tc.cuh"

#include <algorithm>

namespace w8 {

template <int D, int MT>
struct TreeCfg {
  static constexpr int kBM = 16 * MT;
  static constexpr int kTeam = D == 512 ? 2 : 1;            // warps that share 16 keys
  static constexpr int kGroups = kTreeWarps / kTeam;
  static constexpr int kSteps = D == 64 ? 2 : 1;            // 16-key steps of a warp in a tile
  static constexpr int kBN = kGroups * kSteps * 16;         // keys per tile: 256, 128, 128, 64
  static constexpr int kSlotBytes = kBN * D * 2;            // 32 KB (D <= 128) or 64 KB
  static constexpr int kPerSm = D == 64 && MT == 1 ? 2 : 1; // CTAs per SM (two of 32 rows would spill)
  static constexpr int kSlots = kSlotBytes > 32768 ? 3 : 6 / kPerSm;
  // Ring steps loaded ahead.  A slot freed one step ago may still be held by a slow warp, whose
  // turn to load it then waits: with small boxes two steps' grace is worth more than the fifth box.
  static constexpr int kAhead = kSlots == 6 ? 4 : 2;
  static constexpr int kPitch = D + 8;                      // fp32 row pitch of the joint outputs
  static constexpr int kOffRing = 0;
  static constexpr int kOffQ = kSlots * kSlotBytes;
  static constexpr int kOffStat = kOffQ + kBM * D * 2;      // float [2][kGroups][kBM]: maxima, sums
  static constexpr int kOffBar = kOffStat + 2 * kGroups * kBM * 4;
  static constexpr int kNumBars = 2 * kSlots;               // full, empty
  static constexpr int kSmem = kOffBar + kNumBars * 8 + 16 + 1024;
  static_assert(kPerSm * (kSmem + 1024) <= 233472, "shared memory budget exceeded");
  static_assert(kGroups * kBM * kPitch * 4 <= kOffQ, "the joint outputs fit over the ring");
};

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kTreeThreads, TreeCfg<D, MT>::kPerSm)
    attn_tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_kn, const __grid_constant__ CUtensorMap tm_vn,
                     const __grid_constant__ TreeArgs a) {
  using C = TreeCfg<D, MT>;
  constexpr int BM = C::kBM, BN = C::kBN, NS = C::kSlots, CH = D / 8;  // CH: 16-byte chunks per row
  constexpr int DW = D / C::kTeam;                                     // output columns of a warp
  constexpr bool kQRegs = MT == 1 && D <= 128;                         // Q's fragments stay in registers
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t sq = base + C::kOffQ, bar0 = base + C::kOffBar;
  float* stat = reinterpret_cast<float*>(smem + C::kOffStat);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffBar + C::kNumBars * 8);
  auto full_bar = [&](uint32_t s) { return bar0 + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar0 + 8u * (NS + s); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = a.group * a.n;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full_bar(s), a.tma ? 1 : kTreeThreads);  // arrive.expect_tx, or every thread's cp.async
      mbar_init(empty_bar(s), kTreeWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
    if (a.tma) {
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
      prefetch_tmap(&tm_kn);
      prefetch_tmap(&tm_vn);
    }
  }
  pdl_launch_dependents();
  pdl_wait();
  // ---- this CTA's range of all tiles.  A pair (sequence, row tile) has kv_heads items of
  // `nt` tiles each; pairs and their heads follow one another.
  const int pairs = a.batch * a.row_tiles;
  auto split_pair = [&](int p, int& b, int& rt) {
    b = p, rt = 0;
    if (a.row_tiles > 1) b = p / a.row_tiles, rt = p - b * a.row_tiles;
  };
  int b, rt, c = 0, len;
  TreeSpan span;
  long long pos = 0, stop = 0, item_pos = 0;  // item_pos: first tile of the current item
  TreeDeal deal = {1, 0};
  // Q rows r = i * group + g (query head c * group + g of new token i): every load is under way
  // before the first is stored, and where the first item is known without the lengths, before
  // those have come.
  constexpr int kEach = (BM * CH + kTreeThreads - 1) / kTreeThreads;
  uint4 qw[kEach];
  auto fetch_q = [&](int b, int c, int rt) {
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
      const int e = tid + x * kTreeThreads, r = rt * BM + e / CH, ch = e % CH;
      qw[x] = make_uint4(0, 0, 0, 0);
      if (e < BM * CH && r < rows) {
        int i, gq;
        tree_row(a, r, i, gq);
        qw[x] = *reinterpret_cast<const uint4*>(a.q + b * a.q_b + (static_cast<int64_t>(c) * a.group + gq) * a.q_h +
                                                i * a.q_t + ch * 8);
      }
    }
  };
  auto store_q = [&]() {
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
      const int e = tid + x * kTreeThreads, r = e / CH, ch = e % CH;
      if (e < BM * CH) st_shared_v4(sq + r * (D * 2) + ((ch ^ (r & 7)) << 4), qw[x].x, qw[x].y, qw[x].z, qw[x].w);
    }
  };
  bool q_early = false;
  if (a.direct || pairs == 1) {
    // One item (this CTA's number's), or those of one pair.
    int p = 0;
    if (a.direct) {
      p = static_cast<int>(blockIdx.x);
      if (a.kv_heads > 1) p = blockIdx.x / a.kv_heads, c = blockIdx.x - p * a.kv_heads;
    }
    split_pair(p, b, rt);
    q_early = a.direct || a.kv_heads == 1;
    if (q_early) fetch_q(b, c, rt);
    len = tree_len(a, b);
    span = tree_span<BM, BN>(a, len, rt);
    const int tiles = span.c1 - span.c0 + span.nd;
    if (a.direct) {
      stop = tiles;
    } else {
      const long long total = static_cast<long long>(tiles) * a.kv_heads;
      const uint32_t ctas = total < gridDim.x ? static_cast<uint32_t>(total) : gridDim.x;
      if (blockIdx.x >= ctas) return;
      deal.each = div_short(total, ctas);
      deal.more = total - deal.each * ctas;
      pos = deal_begin(deal, blockIdx.x);
      stop = deal_begin(deal, blockIdx.x + 1);
      c = static_cast<int>(div_short(pos, tiles));
      item_pos = static_cast<long long>(c) * tiles;
    }
    __syncthreads();  // the barriers are initialised
  } else {
    auto pair_tiles = [&](int p) {
      int pb, prt;
      split_pair(p, pb, prt);
      const TreeSpan s = tree_span<BM, BN>(a, tree_len(a, pb), prt);
      return s.c1 - s.c0 + s.nd;
    };
    long long* sched = reinterpret_cast<long long*>(smem);  // (the ring is not in use yet)
    long long sum = 0, round;
    for (int p = tid; p < pairs; p += kTreeThreads) sum += pair_tiles(p);
    long long excl = block_scan<kTreeWarps>(sum, sched, round);  // (of up to 256 pairs also each one's place)
    const long long total = round * a.kv_heads;
    const uint32_t ctas = total < gridDim.x ? static_cast<uint32_t>(total) : gridDim.x;
    if (blockIdx.x >= ctas) return;
    deal.each = div_short(total, ctas);
    deal.more = total - deal.each * ctas;
    pos = deal_begin(deal, blockIdx.x);
    stop = deal_begin(deal, blockIdx.x + 1);
    // The pair that holds `pos`: a running sum over rounds of pairs.
    long long before = 0;
    for (int p0 = 0;; p0 += kTreeThreads) {
      const int p = p0 + tid;
      long long nt = sum;
      if (pairs > kTreeThreads) {
        nt = p < pairs ? pair_tiles(p) : 0;
        excl = before + block_scan<kTreeWarps>(nt, sched, round);
      }
      if (nt > 0 && excl * a.kv_heads <= pos && pos < (excl + nt) * a.kv_heads) {
        sched[16] = p;
        sched[17] = excl * a.kv_heads;
      }
      __syncthreads();
      before += round;
      if (pos < before * a.kv_heads) break;  // (every pair has tiles, and pos < total)
      if (p0 + kTreeThreads >= pairs) return;  // only if the lengths changed under the call
    }
    split_pair(static_cast<int>(sched[16]), b, rt);
    item_pos = sched[17];
    len = tree_len(a, b);
    span = tree_span<BM, BN>(a, len, rt);
    const int tiles = span.c1 - span.c0 + span.nd;
    c = static_cast<int>(div_short(pos - item_pos, tiles));
    item_pos += static_cast<long long>(c) * tiles;
    fence_proxy_async_smem();  // the TMA writes the ring next
    __syncthreads();
  }
  int nt = span.c1 - span.c0 + span.nd;
  // The next item: the next head, or the next pair's first.
  auto advance = [&]() {
    item_pos += nt;
    if (++c == a.kv_heads) {
      c = 0;
      if (++rt == a.row_tiles) {
        rt = 0;
        ++b;
        len = tree_len(a, b);
      }
      span = tree_span<BM, BN>(a, len, rt);
      nt = span.c1 - span.c0 + span.nd;
    }
  };

  const int grp = warp / C::kTeam, part = warp % C::kTeam;  // 16-key group of a step; column part
  const int rl = lane >> 2, arow = lane & 15;
  uint32_t g = 0;  // ring steps so far (each tile's K, then V)
  bool ok = true;
  while (true) {
    const int row0 = rt * BM, bc = b * a.kv_heads + c, nc = span.c1 - span.c0;
    const int t0 = static_cast<int>(pos - item_pos);
    const int t1 = static_cast<int>(stop - item_pos < nt ? stop - item_pos : nt);
    const bool whole = t0 == 0 && t1 == nt;
    const int64_t part_row = (2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0 ? 1 : 0)) * BM;
    if (t0 == 0 && tid == 0 && !a.direct) {
      // The CTA that begins an item says where its pieces are: one in each CTA up to its last tile's.
      const int last = deal_owner(deal, item_pos + nt - 1);
      a.info[bc * a.row_tiles + rt] = make_int2(blockIdx.x, last - static_cast<int>(blockIdx.x) + 1);
    }
    // Ring step `i` of this item (tile t0 + i / 2, K or V) into its slot, once every warp has left
    // it: one thread's TMA, or (strides that no map takes) every thread's 16-byte copies into
    // the same layout, rows behind the tensor's end as zeros.
    const uint32_t g_item = g;
    auto load = [&](int i) {
      if (i >= 2 * (t1 - t0)) return;
      const int t = t0 + (i >> 1), kv = i & 1;
      const bool draft = t >= nc;
      const int key0 = (draft ? t - nc : span.c0 + t) * BN;
      const uint32_t step = g_item + i, slot = step % NS, dst = base + slot * C::kSlotBytes;
      const bool free = mbar_wait_bounded(empty_bar(slot), ((step / NS) & 1u) ^ 1u, abort_flag, &g_tree_status);
      if (!free) return;
      if (a.tma) {
        mbar_arrive_expect_tx(full_bar(slot), C::kSlotBytes);
        tma_load_5d(dst, kv ? (draft ? &tm_vn : &tm_v) : (draft ? &tm_kn : &tm_k), full_bar(slot), 0, key0, 0, c, b);
      } else {
        const uint16_t* src = kv ? (draft ? a.vn + b * a.vn_b + c * a.vn_h : a.v + b * a.v_b + c * a.v_h)
                                 : (draft ? a.kn + b * a.kn_b + c * a.kn_h : a.k + b * a.k_b + c * a.k_h);
        const int64_t pitch = kv ? (draft ? a.vn_t : a.v_s) : (draft ? a.kn_t : a.k_s);
        const int rows_here = draft ? a.n : a.slots;
#pragma unroll 2
        for (int e = tid; e < BN * CH; e += kTreeThreads) {
          const int r = e / CH, ch = e % CH;
          const bool on = key0 + r < rows_here;
          cp_async16(dst + (ch >> 3) * (BN * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4),
                     src + (on ? (key0 + r) * pitch : 0) + ch * 8, on);
        }
        cp_async_arrive(full_bar(slot));
      }
    };
    // The step kAhead ahead loads as a step begins; the warps take turns, so that waiting for the
    // others to leave the slot holds up one of them only.
    auto load_ahead = [&](int i) {
      if (!a.tma || (warp == static_cast<int>((g_item + i) % kTreeWarps) && lane == 0)) load(i + C::kAhead);
      __syncwarp();
    };
    if (!a.tma || tid == 0)
      for (int i = 0; i < C::kAhead; ++i) load(i);
    __syncwarp();

    if (!q_early) fetch_q(b, c, rt);
    store_q();
    q_early = false;
    // This thread's rows of each 16-row tile: lane / 4 and lane / 4 + 8.
    int tok[MT][2], dep[MT][2], first[MT][2];
    float m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row0 + mt * 16 + rl + 8 * h;
        int gq;
        tree_row(a, r, tok[mt][h], gq);
        if (r >= rows) tok[mt][h] = -1;
        dep[mt][h] = r < rows ? tree_depth(a, b, tok[mt][h]) : 0;
        first[mt][h] = r < rows ? tree_first(a, len, dep[mt][h]) : INT32_MAX;  // (no row: sees nothing)
        m[mt][h] = -INFINITY;
        l[mt][h] = 0.f;
      }
    float o[MT][DW / 8][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < DW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
    __syncthreads();
    uint32_t qf[kQRegs ? D / 16 : 1][4];
    if constexpr (kQRegs) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        ldsm_x4(sq + arow * (D * 2) + (((2 * kk + (lane >> 4)) ^ (arow & 7)) << 4), qf[kk]);
    }

#pragma unroll 1
    for (int t = t0; t < t1; ++t, g += 2) {
      const bool draft = t >= nc;
      const int tile0 = (draft ? t - nc : span.c0 + t) * BN, end = draft ? a.n : len;
      const uint32_t sk = base + (g % NS) * C::kSlotBytes, sv = base + ((g + 1) % NS) * C::kSlotBytes;
      load_ahead(2 * (t - t0));
      if (ok) ok = mbar_wait_bounded(full_bar(g % NS), (g / NS) & 1u, abort_flag, &g_tree_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
#pragma unroll
      for (int st = 0; st < C::kSteps; ++st) {
        const int kr = (grp * C::kSteps + st) * 16, key0 = tile0 + kr;  // this step's keys
        // ---- S = Q K^T, 16 keys
        float s[MT][2][4];
        constexpr int kChains = MT == 1 && D >= 256 ? 2 : 1;  // halves of D summed side by side
        float s2[kChains][MT][2][4];
#pragma unroll
        for (int ci = 0; ci < kChains; ++ci)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 8; ++e) s2[ci][mt][e >> 2][e & 3] = 0.f;
        const int krow = kr + (lane & 7) + ((lane >> 4) << 3);
        const uint32_t kbase = sk + krow * 128;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t kb[4];
          ldsm_x4(kbase + (kk >> 2) * (BN * 128) + ((((kk & 3) * 2 + ((lane >> 3) & 1)) ^ (krow & 7)) << 4), kb);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            if constexpr (kQRegs) {
              mma16816<T>(s2[kk % kChains][mt][0], qf[kk], kb[0], kb[1]);
              mma16816<T>(s2[kk % kChains][mt][1], qf[kk], kb[2], kb[3]);
            } else {
              uint32_t qa[4];
              const int r = mt * 16 + arow;
              ldsm_x4(sq + r * (D * 2) + (((2 * kk + (lane >> 4)) ^ (r & 7)) << 4), qa);
              mma16816<T>(s2[kk % kChains][mt][0], qa, kb[0], kb[1]);
              mma16816<T>(s2[kk % kChains][mt][1], qa, kb[2], kb[3]);
            }
          }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            s[mt][e >> 2][e & 3] = s2[0][mt][e >> 2][e & 3] + (kChains > 1 ? s2[kChains - 1][mt][e >> 2][e & 3] : 0.f);
        // ---- masks and the running softmax.  Columns of a thread: key0 + 8 n + 2 (lane % 4) + {0, 1}.
        const int col = (lane & 3) * 2;
        uint32_t keep[MT][2];  // the step's 16 keys that the row sees
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int lo = max(first[mt][h] - key0, 0), hi = min(end - key0, 16);
            keep[mt][h] = hi <= lo ? 0u : ((1u << hi) - 1u) & (0xFFFFFFFFu << lo);
          }
        if (draft) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              keep[mt][h] = tree_sees16(a, b, tok[mt][h], key0, dep[mt][h]);
        }
        float mx[MT][2];
        bool move = false;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& v = s[mt][n][2 * h + e];
                v = (keep[mt][h] >> (8 * n + col + e)) & 1u ? v * a.scale_log2 : -INFINITY;
                x = fmaxf(x, v);
              }
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            mx[mt][h] = x;
            move |= x > m[mt][h] + TreeRef<T>::kSlack;
            if (a.scores != nullptr && part == 0) {
              const int r = row0 + mt * 16 + rl + 8 * h;
              if (r < rows) {
                float* dst = a.scores + (static_cast<int64_t>(bc) * rows + r) * a.score_pitch + (draft ? a.draft_at : 0) +
                             key0 + col;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                  const int left = end - key0 - 8 * n - col;
                  if (left > 1)
                    *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(s[mt][n][2 * h], s[mt][n][2 * h + 1]);
                  else if (left > 0)
                    dst[8 * n] = s[mt][n][2 * h];
                }
              }
            }
          }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const bool mv = mx[mt][h] > m[mt][h] + TreeRef<T>::kSlack;
              const float to = mx[mt][h] - TreeRef<T>::kBelow;
              const float corr = mv ? ex2_tree(m[mt][h] - to) : 1.f;
              if (mv) m[mt][h] = to;
              l[mt][h] *= corr;
#pragma unroll
              for (int n = 0; n < DW / 8; ++n) {
                o[mt][n][2 * h] *= corr;
                o[mt][n][2 * h + 1] *= corr;
              }
            }
        }
        uint32_t pa[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float ref = m[mt][h] == -INFINITY ? 0.f : m[mt][h];
            float p[2][2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) p[n][e] = ex2_tree(s[mt][n][2 * h + e] - ref);
            l[mt][h] += (p[0][0] + p[0][1]) + (p[1][0] + p[1][1]);
            // The accumulator's layout of 16 x 16 is the A operand's.
            pa[mt][h] = pack2<T>(p[0][0], p[0][1]);
            pa[mt][2 + h] = pack2<T>(p[1][0], p[1][1]);
          }
        if (st == C::kSteps - 1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(empty_bar(g % NS));
          load_ahead(2 * (t - t0) + 1);  // (into the slot that this warp has just left too)
        }
        // ---- O += P V
        if (st == 0) {
          ok = mbar_wait_bounded(full_bar((g + 1) % NS), ((g + 1) / NS) & 1u, abort_flag, &g_tree_status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        uint32_t bad = 0;  // keys of this step whose values are not all finite (new tokens only)
        if (draft || key0 + 16 > end || key0 < span.low) {
          // Rows behind the length or before the window may hold anything and 0 * NaN is NaN: zeros.  So may a new token's
          // values where some row must not see them: cleared here, added below to the rows that do.
          for (int e = lane; e < 16 * (DW / 8); e += 32) {
            const int r = e % 16, ch = part * (DW / 8) + e / 16;
            uint4* w = reinterpret_cast<uint4*>(smem + (sv - base) + (ch >> 3) * (BN * 128) + (kr + r) * 128 +
                                                (((ch & 7) ^ ((kr + r) & 7)) << 4));
            if (key0 + r >= end || (!draft && key0 + r < span.low)) {
              *w = make_uint4(0, 0, 0, 0);
            } else if (draft) {
              uint4 x = *w;
              if (nonfinite_bits<T>(x.x) | nonfinite_bits<T>(x.y) | nonfinite_bits<T>(x.z) | nonfinite_bits<T>(x.w)) {
                uint32_t* xs = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
                for (int q = 0; q < 4; ++q) xs[q] &= ~((nonfinite_bits<T>(xs[q]) >> 15) * 0xFFFFu);
                *w = x;
                bad |= 1u << r;
              }
            }
          }
          bad = __reduce_or_sync(0xffffffffu, bad);
          fence_proxy_async_smem();  // (the TMA writes this slot again later)
          __syncwarp();
        }
        const int vrow = kr + arow;
        const uint32_t vbase = sv + vrow * 128;
#pragma unroll
        for (int n = 0; n < DW / 8; n += 2) {
          uint32_t vb[4];
          const int ch = part * (DW / 8) + n + (lane >> 4);
          ldsm_x4_t(vbase + (ch >> 3) * (BN * 128) + (((ch & 7) ^ (vrow & 7)) << 4), vb);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16816<T>(o[mt][n], pa[mt], vb[0], vb[1]);
            mma16816<T>(o[mt][n + 1], pa[mt], vb[2], vb[3]);
          }
        }
        const bool any_bad = bad != 0u;
#pragma unroll 1
        for (; bad != 0u; bad &= bad - 1u) {
          const int j = key0 + __ffs(bad) - 1;
          const uint16_t* vn = a.vn + b * a.vn_b + c * a.vn_h + j * a.vn_t + part * DW + (lane & 3) * 2;
          bool sees[MT][2];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) sees[mt][h] = tok[mt][h] >= 0 && tree_sees(a, b, tok[mt][h], j, dep[mt][h]);
#pragma unroll
          for (int n = 0; n < DW / 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint16_t v = vn[n * 8 + e];
              if (tree_nonfinite<T>(v)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                  for (int h = 0; h < 2; ++h)
                    if (sees[mt][h]) o[mt][n][2 * h + e] += tree_f32<T>(v);
              }
            }
        }
        if (any_bad) __syncwarp();  // (the next step's loads are aligned)
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_bar((g + 1) % NS));
    }

    // ---- the groups' results joined: M = max m_w, O = sum 2^(m_w - M) O_w over the ring
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 1);
        l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 2);
        if ((lane & 3) == 0 && part == 0) {
          const int r = mt * 16 + rl + 8 * h;
          stat[grp * BM + r] = m[mt][h];
          stat[(C::kGroups + grp) * BM + r] = l[mt][h];
        }
      }
    ok = __syncthreads_and(ok);  // everybody has left the ring; the statistics are there
    float* joint = reinterpret_cast<float*>(smem);  // [group][BM][pitch]
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = mt * 16 + rl + 8 * h;
        if (row0 + r >= rows) continue;
        float top = stat[r];
#pragma unroll
        for (int w = 1; w < C::kGroups; ++w) top = fmaxf(top, stat[w * BM + r]);
        const float f = m[mt][h] == -INFINITY ? 0.f : ex2_tree(m[mt][h] - top);
        float* dst = joint + (grp * BM + r) * C::kPitch + part * DW + (lane & 3) * 2;
        // (a group that saw nothing adds zeros, except what a NaN score made of it)
        const bool none = m[mt][h] == -INFINITY && l[mt][h] == 0.f;
#pragma unroll
        for (int n = 0; n < DW / 8; ++n) {
          const float s0 = m[mt][h] == -INFINITY ? 1.f : f;
          *reinterpret_cast<float2*>(dst + 8 * n) =
              none ? make_float2(0.f, 0.f) : make_float2(o[mt][n][2 * h] * s0, o[mt][n][2 * h + 1] * s0);
        }
      }
    __syncthreads();
    if (ok) {
      constexpr int Q4 = D / 4;  // float4 columns per row
      for (int e = tid; e < BM * Q4; e += kTreeThreads) {
        const int r = e / Q4, q4 = e % Q4;
        if (row0 + r >= rows) break;
        float top = stat[r];
#pragma unroll
        for (int w = 1; w < C::kGroups; ++w) top = fmaxf(top, stat[w * BM + r]);
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < C::kGroups; ++w) {
          const float mw = stat[w * BM + r];
          sum += (mw == -INFINITY ? 1.f : ex2_tree(mw - top)) * stat[(C::kGroups + w) * BM + r];
          const float4 x = *reinterpret_cast<const float4*>(joint + (w * BM + r) * C::kPitch + 4 * q4);
          v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing: zeros
          int i, gq;
          tree_row(a, row0 + r, i, gq);
          uint16_t* dst = a.o + b * a.o_b + (static_cast<int64_t>(c) * a.group + gq) * a.o_h + i * a.o_t + 4 * q4;
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
          if (a.lse != nullptr && q4 == 0)
            a.lse[static_cast<int64_t>(bc) * rows + row0 + r] = sum == 0.f ? INFINITY : top + log2f(sum);
        } else {
          *reinterpret_cast<float4*>(a.part_o + (part_row + r) * D + 4 * q4) = v;
          if (q4 == 0) a.part_ml[part_row + r] = make_float2(top, sum);
        }
      }
    }
    if (!ok) {
      // A wait gave up: let the copies in flight land before the CTA exits.
      const unsigned long long since = globaltimer();
      while (globaltimer() - since < 50000ull) {
      }
      break;
    }
    pos += t1 - t0;
    if (pos >= stop) break;
    advance();
    fence_proxy_async_smem();  // the joint outputs lay where the TMA writes next
    __syncthreads();  // the ring, Q and the statistics are free
  }
}

// Joins the pieces of one row: M = max m_s, o = sum 2^(m_s - M) O_s / sum 2^(m_s - M) l_s.
// One CTA per row and COLS columns: 4 columns a thread, the pieces over thread groups.  Few
// rows take 32 columns, so that a long sequence's many pieces are summed by more threads.
template <typename T, int D, int COLS>
__global__ void __launch_bounds__(256) attn_tree_combine_kernel(const TreeArgs a, int bm) {
  constexpr int kLanes = COLS / 4, kGroups = 256 / kLanes;
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
    // (nothing seen: 0; a maximum of -inf with another sum: NaN scores, which must show)
    const float f = ml[i].x != -INFINITY ? ex2_tree(ml[i].x - mx) : ml[i].y == 0.f ? 0.f : 1.f;
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
  const int col = blockIdx.y * COLS + ln * 4;
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

// The same for many rows of few pieces: 4 columns a thread, the pieces in turn, no barrier.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_tree_combine_rows_kernel(const TreeArgs a, int bm, int64_t all) {
  constexpr int kLanes = D / 4;
  const int rows = a.group * a.n;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = at / kLanes;
  if (row >= all) return;
  const int col = static_cast<int>(at % kLanes) * 4;
  const int bc = static_cast<int>(row / rows), r = static_cast<int>(row % rows);
  const int64_t item = static_cast<int64_t>(bc) * a.row_tiles + r / bm;
  const bool dealt = a.info != nullptr;
  const int2 info = dealt ? a.info[item] : make_int2(0, a.splits);
  if (info.y <= 1) return;  // written whole
  auto slot = [&](int s) { return dealt ? tree_slot(info, s) : item * a.splits + s; };
  float mx = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < info.y; ++s) mx = fmaxf(mx, a.part_ml[slot(s) * bm + r % bm].x);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < info.y; ++s) {
    const int64_t pr = slot(s) * bm + r % bm;
    const float2 ml = a.part_ml[pr];
    const float4 p = *reinterpret_cast<const float4*>(a.part_o + pr * D + col);
    // (nothing seen: 0, and what stands in the row is not looked at; a maximum of -inf with another
    // sum: NaN scores, which must show)
    const float f = ml.x != -INFINITY ? ex2_tree(ml.x - mx) : ml.y == 0.f ? 0.f : 1.f;
    if (f != 0.f) {
      sum += f * ml.y;
      v.x += f * p.x, v.y += f * p.y, v.z += f * p.z, v.w += f * p.w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int b = bc / a.kv_heads, c = bc % a.kv_heads;
  int i, gq;
  tree_row(a, r, i, gq);
  uint16_t* dst = a.o + b * a.o_b + (static_cast<int64_t>(c) * a.group + gq) * a.o_h + i * a.o_t + col;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
  if (a.lse != nullptr && col == 0) a.lse[row] = sum == 0.f ? INFINITY : mx + log2f(sum);
}

// Accumulated weights: slot j gets weights[j] + sum over the R rows of p_rj, p from the stored
// scores and the rows' log-sum-exp (summed in a fixed order: the same bits every time).  Four
// slots a thread, 16-byte loads of several rows in flight: bound by reading the scores.  Many
// rows are dealt to SPLIT groups of threads, joined at the end: one thread that walks 968 rows
// waits 280 us for its loads (1 cache head, 131 slots), eight 39.
template <int SPLIT>  // 1, or 8: a warp each
__global__ void __launch_bounds__(256) attn_tree_weights_kernel(const TreeArgs a) {
  constexpr int kThreads = 256 / SPLIT, kSlots = 4 * kThreads;  // of a group; slots of a CTA
  __shared__ float sm_lse[256];
  __shared__ int sm_first[256];
  __shared__ float4 sm_sum[SPLIT][SPLIT > 1 ? kThreads : 1];
  const int part = SPLIT > 1 ? threadIdx.x / kThreads : 0, at = threadIdx.x % kThreads;
  const int rows = a.group * a.n, bc = blockIdx.y, b = bc / a.kv_heads, c = bc % a.kv_heads;
  pdl_launch_dependents();
  pdl_wait();
  const int len = tree_len(a, b);
  const int begin = blockIdx.x * kSlots;
  const int j0 = begin + at * 4;  // slots [0, draft_at), then new tokens
  if (begin >= len && begin + kSlots <= a.draft_at) return;
  const bool draft = j0 >= a.draft_at;
  const int end = draft ? a.draft_at + a.n : len;
  const float* x = a.scores + static_cast<int64_t>(bc) * rows * a.score_pitch + j0;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < rows; r0 += 256) {
    // (lse, first visible slot) of up to 256 rows at a time
    __syncthreads();
    if (r0 + threadIdx.x < rows) {
      int i, gq;
      tree_row(a, r0 + threadIdx.x, i, gq);
      sm_lse[threadIdx.x] = a.lse[static_cast<int64_t>(bc) * rows + r0 + threadIdx.x];
      sm_first[threadIdx.x] = tree_first(a, len, tree_depth(a, b, i));
    }
    __syncthreads();
    if (j0 < end) {
      const int n = min(256, rows - r0);
#pragma unroll SPLIT == 1 ? 4 : 8
      for (int q = part; q < n; q += SPLIT) {
        const float4 v = *reinterpret_cast<const float4*>(x + static_cast<int64_t>(r0 + q) * a.score_pitch);
        const float e[4] = {v.x, v.y, v.z, v.w};
        // Of this thread's four, [lo, hi) were scored: no tile of the row covers slots before the
        // first that it sees, nor a causal chunk's tokens behind it.
        int lo, hi;
        if (draft) {
          int i, gq;
          tree_row(a, r0 + q, i, gq);
          lo = 0, hi = a.draft_at + (a.tree != nullptr ? a.n : i + 1) - j0;
        } else {
          lo = sm_first[q] - j0, hi = len - j0;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k >= lo && k < hi) sum[k] += ex2_tree(e[k] - sm_lse[q]);
      }
    }
  }
  if constexpr (SPLIT > 1) {
    sm_sum[part][at] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int s = 1; s < SPLIT; ++s) {
      const float4 v = sm_sum[s][at];
      sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int j = j0 + k;
    if (j >= end) break;
    if (draft)
      a.w_new[static_cast<int64_t>(bc) * a.n + j - a.draft_at] = sum[k];
    else
      a.w_out[b * a.wo_b + c * a.wo_h + j] = a.w_in[b * a.wi_b + c * a.wi_h + j] + sum[k];
  }
}

}  // namespace w8

namespace w8host {

int require_sm100(int* device);

int tree_encode_rows(CUtensorMap* map, const void* ptr, bool half, int64_t d, int64_t n, int64_t heads, int64_t batch,
                     int64_t s_b, int64_t s_h, int64_t s_n, uint32_t rows, uint32_t blocks);
int tree_tc(const w8::TreeArgs& a, bool half, int64_t d, int64_t items, int device, cudaStream_t stream);
int tree_tc_device_status(int clear, int* out);

// How a call is cut: rows per tile, row tiles, and over the keys a number of splits (tcgen05)
// or of CTAs that share all tiles (mma.sync).
struct TreePlan {
  bool tc;  // the tcgen05 schedule (attention_tree_tc.cu)
  bool direct;  // mma.sync: a CTA for each item
  int bm, row_tiles, splits, ctas;
  int64_t items;
};

// The tcgen05 schedule takes 256 rows a tile and keeps up with HBM for any number of them, so
// it is for more rows a cache head than one mma.sync tile has (`tma`: its maps can describe
// the tensors): with 16 or 32 rows, mma.sync tiles spread a sequence's keys over all SMs.  At
// D 64, which it runs as 128, two mma.sync tiles are still better (256 cache heads of 4000 keys:
// 32 rows 80 us against 241, 64 rows 150 against 237; four would take 300).
static TreePlan tree_plan(int64_t batch, int64_t kv_heads, int64_t group, int64_t n, int64_t d, int64_t slots,
                          int64_t window, int sms, bool tma) {
  TreePlan p;
  const int64_t rows = group * n;
  p.tc = tma && rows > (d == 64 ? 64 : d == 128 ? 32 : 16);
  p.bm = p.tc ? 256 : rows > 16 && d <= 128 ? 32 : 16;
  p.row_tiles = static_cast<int>((rows + p.bm - 1) / p.bm);
  p.items = batch * kv_heads * p.row_tiles;
  // Keys of one row tile: with a window, those its tokens see.
  const int64_t bn = p.tc ? 128 : d == 512 ? 64 : d == 64 ? 256 : 128;
  const int64_t tokens = std::min(n, p.bm / group + 2);
  const int64_t keys = window > 0 ? std::min(slots, window + tokens) : slots;
  const int64_t tiles = (keys + bn - 1) / bn + (n + bn - 1) / bn;
  p.splits = 1;
  if (p.tc) {
    // The number of splits with the least estimated time: waves of clusters, each 1.6 us a tile
    // and 8 us besides, then 4 us and the partials at 3 TB/s to join them.  Measured on trees of 64
    // drafts at D 256, which other head sizes share though it does not fit them as well (320 items
    // of 1000 keys at D 512: 201 us estimated, 276 measured), and with lengths near the capacity,
    // which is all that the host knows: sequences that fill little of a large cache are split into
    // more pieces than they have tiles (the tree of 60 over 4000 slots of 4096 takes 65 us, of 131072
    // 159).
    const int64_t width = d == 512 ? 2 : 1, pairs = sms / 2;
    double best = 0;
    for (int64_t s = 1; s <= std::min<int64_t>(tiles, 64); ++s) {
      const double waves = static_cast<double>((p.items * width * s + pairs - 1) / pairs);
      double us = waves * (1.6 * static_cast<double>((tiles + s - 1) / s) + 8);
      if (s > 1) us += 4 + static_cast<double>(p.items * p.bm * d) * 8 * static_cast<double>(s) / 3e6;
      if (s == 1 || us < best) best = us, p.splits = static_cast<int>(s);
    }
    p.ctas = 0;
    p.direct = false;
  } else {
    // An item per CTA, or all tiles dealt evenly: by estimated times.  A tile is about 1 us (2 us
    // of 64 KB boxes), an item's start and end 3 us, joining the pieces a launch of 4 us.  From 8
    // items an SM on ragged lengths even out by themselves.
    const double tile_us = d >= 256 || (d == 64 && p.bm == 32) ? 2.0 : 1.0;
    const double waves = static_cast<double>((p.items + sms - 1) / std::max(sms, 1));
    const double alone = waves * (static_cast<double>(tiles) * tile_us + 3);
    const double dealt = static_cast<double>(p.items) * static_cast<double>(tiles) / sms * tile_us + 3 * (waves + 1) + 4;
    p.direct = alone <= dealt || p.items >= 8 * static_cast<int64_t>(sms);
    p.ctas = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({sms * (d == 64 && p.bm == 16 ? 2 : 1), p.items * tiles, w8::kTreeMaxPieces})));  // TreeCfg::kPerSm
  }
  return p;
}

struct TreeWs {
  int64_t part_o, part_ml, info, lse, scores, total, score_pitch, draft_at;
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
  const int64_t part_rows = p.tc ? (p.splits > 1 ? p.items * p.splits * p.bm : 0) : p.direct ? 0 : 2 * static_cast<int64_t>(p.ctas) * p.bm;
  w.part_o = take(part_rows * d * 4);
  w.part_ml = take(part_rows * 8);
  w.info = take(p.tc || p.direct ? 0 : p.items * 8);
  const int64_t rows = batch * kv_heads * group * n;
  w.draft_at = (slots + 3) / 4 * 4;
  w.score_pitch = w.draft_at + (n + 3) / 4 * 4;
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
static int launch_tree(Kern kern, dim3 grid, int threads, int smem, cudaStream_t stream, const Args&... args) {
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
  constexpr bool kHalf = __is_same(T, __half);
  static bool done[64] = {};
  if (!done[device]) {
    W8_CUDA_TRY(cudaFuncSetAttribute(w8::attn_tree_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     C::kSmem));
    done[device] = true;
  }
  CUtensorMap tk = {}, tv = {}, tkn = {}, tvn = {};
  if (a.tma) {
    int st = tree_encode_rows(&tkn, a.kn, kHalf, D, a.n, a.kv_heads, a.batch, a.kn_b, a.kn_h, a.kn_t, C::kBN, D / 64);
    if (st != W8_OK) return st;
    st = tree_encode_rows(&tvn, a.vn, kHalf, D, a.n, a.kv_heads, a.batch, a.vn_b, a.vn_h, a.vn_t, C::kBN, D / 64);
    if (st != W8_OK) return st;
    tk = tkn, tv = tvn;  // an empty cache: never read
    if (a.slots > 0) {
      st = tree_encode_rows(&tk, a.k, kHalf, D, a.slots, a.kv_heads, a.batch, a.k_b, a.k_h, a.k_s, C::kBN, D / 64);
      if (st != W8_OK) return st;
      st = tree_encode_rows(&tv, a.v, kHalf, D, a.slots, a.kv_heads, a.batch, a.v_b, a.v_h, a.v_s, C::kBN, D / 64);
      if (st != W8_OK) return st;
    }
  }
  return launch_tree(w8::attn_tree_kernel<T, D, MT>, dim3(static_cast<unsigned>(blocks)), w8::kTreeThreads, C::kSmem,
                     stream, tk, tv, tkn, tvn, a);
}

// The pieces of all items joined.  Few rows: a CTA each, or for 32 columns of each, since their
// pieces may be many.
template <typename T, int D>
static int tree_join_go(const w8::TreeArgs& a, int bm, cudaStream_t stream) {
  constexpr int kWide = D < 128 ? D : 128;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.kv_heads * a.group * a.n;
  if (rows * (D / 32) <= 1024)
    return launch_tree(w8::attn_tree_combine_kernel<T, D, 32>, dim3(static_cast<unsigned>(rows), D / 32), 256, 0, stream, a,
                       bm);
  if (rows <= 512)
    return launch_tree(w8::attn_tree_combine_kernel<T, D, kWide>, dim3(static_cast<unsigned>(rows), D / kWide), 256, 0,
                       stream, a, bm);
  return launch_tree(w8::attn_tree_combine_rows_kernel<T, D>, dim3(static_cast<unsigned>((rows * (D / 4) + 255) / 256)),
                     256, 0, stream, a, bm, rows);
}

// The same for the paged cache's attention.
int tree_join(const w8::TreeArgs& a, bool half, int64_t d, int bm, cudaStream_t stream) {
  using B = __nv_bfloat16;
  switch (d) {
    case 64: return half ? tree_join_go<__half, 64>(a, bm, stream) : tree_join_go<B, 64>(a, bm, stream);
    case 128: return half ? tree_join_go<__half, 128>(a, bm, stream) : tree_join_go<B, 128>(a, bm, stream);
    case 256: return half ? tree_join_go<__half, 256>(a, bm, stream) : tree_join_go<B, 256>(a, bm, stream);
    default: return half ? tree_join_go<__half, 512>(a, bm, stream) : tree_join_go<B, 512>(a, bm, stream);
  }
}

template <typename T, int D>
static int tree_go(const w8::TreeArgs& a, const TreePlan& p, int device, cudaStream_t stream) {
  W8_CHECK_ARG(p.items < (1ll << 31) / 2, "too many row tiles");
  const int64_t blocks = p.direct ? p.items : p.ctas;
  int st;
  if (p.tc)
    st = tree_tc(a, __is_same(T, __half), D, p.items, device, stream);
  else if constexpr (D <= 128)
    st = p.bm == 32 ? tree_main<T, D, 2>(a, blocks, device, stream) : tree_main<T, D, 1>(a, blocks, device, stream);
  else
    st = tree_main<T, D, 1>(a, blocks, device, stream);
  if (st != W8_OK) return st;
  if (p.tc ? p.splits > 1 : !p.direct && p.ctas > 1) {
    st = tree_join_go<T, D>(a, p.bm, stream);
    if (st != W8_OK) return st;
  }
  if (a.scores != nullptr) {
    const bool split = a.group * a.n > 16;  // (16 rows are four rounds of loads)
    const int64_t slots = split ? 128 : 1024;
    const dim3 grid(static_cast<unsigned>((a.score_pitch + slots - 1) / slots), static_cast<unsigned>(a.batch * a.kv_heads));
    st = split ? launch_tree(w8::attn_tree_weights_kernel<8>, grid, 256, 0, stream, a)
               : launch_tree(w8::attn_tree_weights_kernel<1>, grid, 256, 0, stream, a);
  }
  return st;
}

// A call without new tokens adds nothing to the weights, which still go where they are wanted.
static int tree_no_tokens(const w8_attention_tree_args& x, cudaStream_t stream) {
  if (x.weights == x.weights_out || x.slots == 0) return W8_OK;
  W8_CHECK_ARG(x.weights && x.weights_out && x.lens, "weights, weights_out and draft_weights come together");
  W8_CHECK_ARG(x.batch * x.kv_heads <= 65535, "batch * kv_heads beyond 65535 with weights");
  int device = 0;
  const int st = require_sm100(&device);
  if (st != W8_OK) return st;
  w8::TreeArgs a = {};
  a.lens = x.lens;
  a.batch = static_cast<int>(x.batch), a.kv_heads = static_cast<int>(x.kv_heads), a.slots = static_cast<int>(x.slots);
  a.group = static_cast<int>(x.heads / x.kv_heads);
  a.draft_at = (a.slots + 3) / 4 * 4;
  a.w_in = x.weights, a.w_out = x.weights_out;
  a.wi_b = x.weights_stride[0], a.wi_h = x.weights_stride[1];
  a.wo_b = x.weights_out_stride[0], a.wo_h = x.weights_out_stride[1];
  return launch_tree(w8::attn_tree_weights_kernel<1>,
                     dim3(static_cast<unsigned>((a.draft_at + 1023) / 1024), static_cast<unsigned>(x.batch * x.kv_heads)), 256,
                     0, stream, a);
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
  if (x.batch == 0) return W8_OK;
  // In place only with the same layout: rows of one would be other rows of the other.
  W8_CHECK_ARG(x.weights == nullptr || x.weights != x.weights_out ||
                   ((x.batch == 1 || x.weights_stride[0] == x.weights_out_stride[0]) &&
                    (x.kv_heads == 1 || x.weights_stride[1] == x.weights_out_stride[1])),
               "weights_out is weights with other strides");
  if (x.n_new == 0) return tree_no_tokens(x, reinterpret_cast<cudaStream_t>(stream));
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
  W8_CHECK_ARG(x.out != x.q && x.out != x.k && x.out != x.v && x.out != x.k_new && x.out != x.v_new,
               "out must not be an input");
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
  a.tma = tma ? 1 : 0;
  a.direct = p.direct ? 1 : 0;
  a.info = p.tc ? nullptr : reinterpret_cast<int2*>(ws + w.info);
  if (weights) {
    a.lse = reinterpret_cast<float*>(ws + w.lse);
    a.scores = reinterpret_cast<float*>(ws + w.scores);
    a.score_pitch = w.score_pitch;
    a.draft_at = static_cast<int>(w.draft_at);
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
