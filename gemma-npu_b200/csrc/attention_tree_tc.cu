// Attention over a cache for many query rows (drafted trees, chunks, large groups) on the
// 5th-generation tensor cores: the contract of attention_tree.cu on the schedule of the
// prefill attention (attention_tc.cu).
//
// A cluster of two CTAs (tcgen05 cta_group::2) owns 256 of the R = G N rows of one cache
// head (128 per CTA: TMEM lanes), min(D, 256) output columns and a range of 128-key tiles:
//   S_j  = Q K_j^T     M 256 x N 128 in one of two TMEM buffers, each CTA staging 64 keys
//   P_j  = 2^(c S_j - m)   two threads a row (64 keys each): mask, maximum, sum; P_j 16-bit
//                      back into the S buffer
//   O   += P_j V_j     A = P_j from TMEM, each CTA staging half of V's columns
// m moves only when a tile's maximum exceeds it by enough (TreeRef).  Many rows per
// key make this bound by the MMAs and the softmax's exponentials, not by HBM: trees of 64
// drafts for 16 sequences, D 256, 8 heads a group, 2000 to 4000 keys take 64 us here (a tile
// some 2650 clocks of a pair, its MMAs 2048) and 672 with mma.sync.  The key axis is split over
// clusters while they would leave SMs idle, and the partial outputs joined by the combine
// kernel of attention_tree.cu.
//
// What a decode adds to prefill is ragged: the committed length ends (and the window begins)
// inside a tile, whose rows beyond may hold NaN, and so may a new token's V (0 * NaN is NaN in
// the product).  In such a tile ("careful": the first and last committed ones if they are
// partial, and tiles of new tokens that some row does not see whole) V completes on a barrier
// of its own CTA, the softmax threads clear what must not count before they hand over P, and
// non-finite values are added at the end to the rows that do see them.  Every wait is bounded,
// as in attention_tc.cu.
#include "attention_paged.cuh"
#include "attn_tc.cuh"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace w8 {

constexpr int kTtBM = 128;                 // rows per CTA; 256 per pair
constexpr int kTtBN = 128;                 // keys per tile
constexpr int kTtSoftWarps = 8;
constexpr int kTtUnpackWarps = 6;          // of a paged cache, in two teams that take its slots in turn
constexpr int kTtUnpackTeam = kTtUnpackWarps / 2;
// What the producer makes of a tile's scales, for the softmax threads: of 16 keys each the factor of a
// score in log2 units, the logarithm of V's scale in O's unit and its reciprocal; then what a change of
// the unit does to O, the unit, and bits of the 16 keys that are there.
struct TtScales {
  float to_log2[8], lg_v[8], rcp_v[8], change, unit;
  uint32_t there;
  uint32_t pad;
};
__device__ __forceinline__ const TreeArgs& tree_args(const TreeArgs& a) { return a; }
struct TtPagedArgs : PagedArgs {
  CUtensorMap k8, v8;  // the pool's
};
__device__ __forceinline__ const TreeArgs& tree_args(const PagedArgs& a) { return a.t; }
constexpr int kTtKeysPerCta = kTtBN / 2;
constexpr uint32_t kTtTmemCols = 512;
constexpr uint32_t kTtColO = 2 * kTtBN;

template <int D, bool kPaged>
struct TtCfg {
  static constexpr int kThreads = 32 * (2 + kTtSoftWarps + (kPaged ? kTtUnpackWarps : 0));
  static constexpr int kDV = D < 256 ? D : 256;           // output columns per pair
  static constexpr int kSplitD = D / kDV;                 // clusters per row block (D = 512: 2)
  static constexpr int kQBytes = kTtBM * D * 2;
  static constexpr int kKCols = D < 256 ? D : 256;        // columns of the reduction per K slot
  static constexpr int kKSlots = D / kKCols;              // slots per K tile
  static constexpr int kSlotBytes = kTtBN * kDV;          // K: 64 keys x kKCols; V: 128 keys x kDV / 2
  static constexpr int kSlots = kPaged ? (D == 512 ? 2 : D == 256 ? 3 : 8) : D == 512 ? 3 : D == 256 ? 5 : 8;
  static constexpr int kStageBytes = kSlotBytes / 2;      // a slot's values while they are 8 bits
  static constexpr int kStages = kPaged ? (D == 512 ? 2 : 4) : 0;
  static constexpr int kOffRing = kQBytes;
  static constexpr int kOffStage = kOffRing + kSlots * kSlotBytes;
  static constexpr int kOffBar = kOffStage + kStages * kStageBytes;
  // full[kSlots], empty[kSlots], own[kSlots], q_full, s_full[2], p_full[2], pv_done[2], o_ready,
  // staged[kStages], unpacked[kStages]
  static constexpr int kNumBars = 3 * kSlots + 8 + 2 * kStages;
  static constexpr int kOffXch = kOffBar + (kNumBars * 8 + 31) / 16 * 16;
  static constexpr int kOffPoison = kOffXch + 2 * kTtBM * 4;
  // The scales of the tiles from the one in the softmax to the producer's.  It writes those of tile j when
  // the staging slot of K_j's first step is free: the step kStages before has been unpacked, so the ring's
  // slot of the step kSlots before that had been left.  Steps are K_0 K_1 V_0 K_2 V_1 ..; that one is V_j-5
  // (D = 256), V_j-3 (512), or K_j-6 (S_j-6 follows P_j-8's product).
  static constexpr int kScales = kPaged ? (D < 256 ? 8 : D == 256 ? 5 : 4) : 0;
  static constexpr int kOffScale = kOffPoison + kPoisonWords * 4;
  static constexpr int kSmem = kOffScale + kScales * static_cast<int>(sizeof(TtScales)) + 1008;  // (shared memory begins on 16 bytes)
  static_assert(!kPaged || (kOffScale % 16 == 0 && sizeof(TtScales) % 16 == 0), "alignment");
  static_assert(kKCols == kDV, "K and V slots have one size");
  static_assert(kSmem <= 232448, "shared memory budget exceeded");
  static_assert(kTtBM * (kDV * 4 + 16) <= kOffBar, "the output rows fit over Q and the ring");
};

__device__ __forceinline__ float lg2_tc(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Arrive on a barrier that may lie in the peer CTA, releasing this thread's shared-memory
// writes to the cluster.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void red_or_cluster(uint32_t addr, uint32_t bits) {
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(addr), "r"(bits) : "memory");
}

// DR: columns of a head in memory.  Heads of 64 run as 128 whose upper half the boxes fill with
// zeros (S and O do not change, and only the lower half is stored): the MMAs do twice their work
// and 216 row tiles of 680 rows over 1085 keys take 194 us where mma.sync took 626.
// Over a paged 8-bit cache (kPaged; tm_k and tm_v then are the tails'): each CTA's share of a tile's
// pages comes by TMA as it is into a staging slot, and a team of three warps unpacks it to T into
// the ring's slot, which is exact; the scale of K multiplies the scores, that of
// V goes into P relative to a power of two, in which O is held (paged_unit; the first tile of 16-bit
// rows brings it to 1).  Pages are never careful: 8-bit values are finite, whatever they are.  Staging
// slots are filled ahead of the ring, whose slots the unpacking warps wait for themselves.  The
// softmax and the unpacking share the issue slots (a tile takes some 4600 clocks here where 16-bit
// rows take 2650): a short unpacking loop and no masks for pages that all rows see whole brought
// trees of 24 drafts for 16 sequences, D 256, 2000 to 4000 keys from 74 to 64 us (with mma.sync 474).
template <typename T, int D, int DR, bool kPaged, typename Args>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TtCfg<D, kPaged>::kThreads, 1)
    attn_tree_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ CUtensorMap tm_kn, const __grid_constant__ CUtensorMap tm_vn,
                        const __grid_constant__ Args args) {
  using C = TtCfg<D, kPaged>;
  const TreeArgs& a = tree_args(args);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t ring = base + C::kOffRing;
  const uint32_t bar0 = base + C::kOffBar;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffBar + C::kNumBars * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto full_bar = [&](uint32_t s) { return bar0 + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar0 + 8u * (C::kSlots + s); };
  auto own_bar = [&](uint32_t s) { return bar0 + 8u * (2 * C::kSlots + s); };
  const uint32_t q_full = bar0 + 8u * (3 * C::kSlots);
  auto s_full = [&](int b) { return q_full + 8u * (1 + b); };
  auto p_full = [&](int b) { return q_full + 8u * (3 + b); };
  auto pv_done = [&](int b) { return q_full + 8u * (5 + b); };
  const uint32_t o_ready = q_full + 8u * 7;
  auto staged_bar = [&](uint32_t s) { return q_full + 8u * (8 + s); };
  auto unpacked_bar = [&](uint32_t s) { return q_full + 8u * (8 + C::kStages + s); };
  TtScales* const scales = reinterpret_cast<TtScales*>(smem + C::kOffScale);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();  // 0 = the CTA that issues the MMAs
  const uint32_t peer = rank ^ 1u;
  const int cl = static_cast<int>(blockIdx.x >> 1);
  const int half = cl % C::kSplitD, split = cl / C::kSplitD % a.splits, item = cl / C::kSplitD / a.splits;
  const int rt = item % a.row_tiles, bc = item / a.row_tiles;
  const int b = bc / a.kv_heads, c = bc % a.kv_heads;
  const int rows = a.group * a.n;
  const int row0 = rt * (2 * kTtBM) + static_cast<int>(rank) * kTtBM;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kSlots; ++s) {
      // leader: one arrive.expect_tx + both CTAs' bytes, or (pages) the unpacking warps of both CTAs
      mbar_init(full_bar(s), kPaged ? 2 * kTtUnpackTeam : 1);
      mbar_init(empty_bar(s), 1);  // both: one MMA commit
      mbar_init(own_bar(s), 1);    // both: this CTA's bytes of a careful V tile
    }
    // leader: one arrive.expect_tx + both CTAs' bytes, or the softmax warps of both CTAs wrote Q
    mbar_init(q_full, a.q_tma ? 1 : 2 * kTtSoftWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full(i), 1);
      mbar_init(p_full(i), 2 * kTtSoftWarps);  // leader: the softmax warps of both CTAs
      mbar_init(pv_done(i), 1);
    }
    mbar_init(o_ready, 1);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(staged_bar(s), 1);
      mbar_init(unpacked_bar(s), kTtUnpackTeam);
    }
    *abort_flag = 0;
    fence_mbar_init();
    if (a.q_tma) prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    prefetch_tmap(&tm_kn);
    prefetch_tmap(&tm_vn);
    if constexpr (kPaged) {
      prefetch_tmap(&args.k8);
      prefetch_tmap(&args.v8);
    }
  }
  if (threadIdx.x < kPoisonWords) reinterpret_cast<uint32_t*>(smem + C::kOffPoison)[threadIdx.x] = 0u;
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), kTtTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barriers initialised and TMEM allocated in both CTAs
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tmem = *tmem_slot;

  // The pair's tiles: [t0, t1) of its committed, then new-token tiles; a split of an item with
  // fewer tiles than splits has none (both CTAs agree).
  const int len = tree_len(a, b);
  auto span_of = [&]() {
    if constexpr (kPaged)
      return paged_span<2 * kTtBM, kTtBN, kTtBN>(args, len, rt);
    else
      return tree_span<2 * kTtBM, kTtBN>(a, len, rt);
  };
  const auto span = span_of();
  // Tiles of pages, of committed keys (the pages' and the tail's, if paged) and all.
  int np = 0, nc, full = 0;
  if constexpr (kPaged)
    np = span.pages(), nc = np + span.tail, full = span.full;
  else
    nc = span.c1 - span.c0;
  const int nt = nc + span.nd;
  const int t0 = static_cast<int>(static_cast<int64_t>(nt) * split / a.splits);
  const int t1 = static_cast<int>(static_cast<int64_t>(nt) * (split + 1) / a.splits);
  const int ntiles = t1 - t0;
  const int64_t part_row = (static_cast<int64_t>(item) * a.splits + split) * (2 * kTtBM) + rank * kTtBM;
  auto is_draft = [&](int i) { return t0 + i >= nc; };
  auto is_page = [&](int i) { return kPaged && t0 + i < np; };
  // First key of a tile: a position, a row of the tail or a new token.
  auto key0_of = [&](int i) {
    if constexpr (kPaged) {
      const int t = t0 + i;
      if (t < np) return (t < span.ns ? t : span.c0 + t - span.ns) * kTtBN;
      return (t < nc ? t - np : t - nc) * kTtBN;
    }
    return (t0 + i >= nc ? t0 + i - nc : span.c0 + t0 + i) * kTtBN;
  };
  const int sink_left = kPaged ? a.sink - len : kNoSinks;
  // Of a causal chunk's tiles of new tokens, those that every row of the pair sees whole are as
  // plain as committed ones.
  const int tok_lo = rt * (2 * kTtBM) / a.group, tok_hi = (min((rt + 1) * (2 * kTtBM), rows) - 1) / a.group;
  auto careful = [&](int i) {
    if (is_page(i)) return false;
    const int key0 = key0_of(i);
    if (!is_draft(i)) return full + key0 + kTtBN > len || full + key0 < span.low;
    return a.tree != nullptr || a.depth != nullptr || key0 + kTtBN - 1 > tok_lo ||
           (a.window > 0 && key0 <= tok_hi - a.window);
  };
  // Ring position of V_i: K_0, then K_{i+1} and V_i in turn.
  auto v_pos = [&](int i) { return static_cast<uint32_t>(min(i + 2, ntiles) * C::kKSlots + i); };

  if (ntiles == 0) {
    if (warp >= 2) {
      const int r = (warp & 3) * 32 + lane;
      if (warp < 6 && half == 0) a.part_ml[part_row + r] = make_float2(-INFINITY, 0.f);
    }
  } else if (warp == 0) {
    if constexpr (kPaged) {
      // ---- TMA producer (both CTAs), a page a lane: the ring in the MMA order, 16-bit tiles into its
      // slots as below, pages into the staging slots once the ring's slot is free.
      uint32_t g = 0, st = 0;  // ring steps; staged ones
      bool ok = true;
      const int box_v = min(args.shift, 7), box_k = min(args.shift, 6);  // log2 of the keys of a box
      const int* table = args.table + b * args.table_b;
      // Lane j's 16 keys (of 128) of tile i: the table's entry if some row needs it, or -1; the page it
      // names; its scales.  Each is read a tile before the next needs it.
      auto entry_of = [&](int i) {
        if (i >= ntiles || !is_page(i) || lane >= kTtBN / 16) return -1;
        const int k0 = key0_of(i) + lane * 16, p0 = k0 >> args.shift << args.shift;
        // (whether a page is needed is decided for all of it within the tile)
        const int lo = max(p0, key0_of(i)), hi = min(p0 + (1 << args.shift), key0_of(i) + kTtBN);
        if (!paged_needs(args, span, lo, hi)) return -1;
        const int p = table[k0 >> args.shift];
        return p < 0 ? INT32_MAX : p;
      };
      struct Page {
        int at;
        float ks, vs;
      };
      auto page_of = [&](int entry) {
        Page p = {entry, 0.f, 0.f};
        if (entry >= args.pages) {
          atomicExch(&g_tree_status, W8_ERR_INVALID_ARG);
          p.at = -1;
        }
        if (p.at >= 0) {
          p.ks = args.ks[p.at * args.ks_p + c * args.ks_h];
          p.vs = args.vs[p.at * args.vs_p + c * args.vs_h];
        }
        return p;
      };
      auto wait_slot = [&]() {
        ok = ok && wait_phase(empty_bar(g % C::kSlots), ((g / C::kSlots) & 1u) ^ 1u, abort_flag, &g_tree_status);
        ok = __all_sync(0xffffffffu, ok);
        return ok;
      };
      auto put = [&](const CUtensorMap* m, int key0, int block0, bool own) {  // 16-bit rows
        if (!wait_slot()) return;
        const uint32_t slot = g % C::kSlots;
        if (lane == 0) {
          uint32_t bar;
          if (own) {
            mbar_arrive_expect_tx(own_bar(slot), C::kSlotBytes);
            bar = mapa_shared(own_bar(slot), rank);
            if (rank == 0) mbar_arrive_count(full_bar(slot), 2 * kTtUnpackTeam);  // the MMA thread goes by P's barrier
          } else {
            if (rank == 0) {
              mbar_arrive_expect_tx(full_bar(slot), 2 * C::kSlotBytes);
              mbar_arrive_count(full_bar(slot), 2 * kTtUnpackTeam - 1);
            }
            bar = mapa_shared(full_bar(slot), 0);
          }
          tma_load_5d_pair(ring + slot * C::kSlotBytes, m, bar, 0, key0, block0, c, b);
        }
        __syncwarp();
        ++g;
      };
      auto wait_stage = [&]() {  // (the ring's slot is the unpacking warps' to wait for)
        ok = ok && wait_phase(unpacked_bar(st % C::kStages), ((st / C::kStages) & 1u) ^ 1u, abort_flag, &g_tree_status);
        ok = __all_sync(0xffffffffu, ok);
        return ok;
      };
      // `n` boxes of 2^shift keys from key `from` of the tile and column x into the next staging slot.
      auto put_pages = [&](const CUtensorMap* m, int page, int key0, int from, int n, int shift, int bytes, int x) {
        if (!wait_stage()) return;
        const uint32_t s = st % C::kStages;
        const int mine = __shfl_sync(0xffffffffu, page, (from + (lane << shift)) / 16 & 31);
        const bool on = lane < n && mine >= 0;
        const int count = __popc(__ballot_sync(0xffffffffu, on));
        if (lane == 0) mbar_arrive_expect_tx(staged_bar(s), count * bytes);
        __syncwarp();
        if (on)
          tma_load_5d(base + C::kOffStage + s * C::kStageBytes + lane * bytes, m, staged_bar(s), x,
                      (key0 + from + (lane << shift)) & ((1 << args.shift) - 1), 0, c, mine);
        __syncwarp();
        ++g, ++st;
      };
      const int kk0 = static_cast<int>(rank) * kTtKeysPerCta;
      const int vb0 = half * (C::kDV / 64) + static_cast<int>(rank) * (C::kDV / 128);
      float unit = __uint_as_float(0x00800000u);  // of O (2^-126: nothing added yet)
      auto put_k = [&](int i, const Page& page) {
        if (is_page(i)) {
          if (!wait_stage()) return;
          // The scales first: whoever sees the tile's scores sees them.
          const float need = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(paged_unit(page.vs))));
          const float to = fmaxf(unit, need), rcp = paged_unit_rcp(to);
          const uint32_t on = __ballot_sync(0xffffffffu, page.at >= 0);
          TtScales& out = scales[i % C::kScales];
          if (lane < kTtBN / 16) {
            // (Not 0, times which a hidden key's -inf would be NaN, or whose logarithm is -inf: a page's
            // values may all be 0.  A NaN stays.)
            const float f = page.ks * a.scale_log2, x = page.vs * rcp, v = x < 0x1p-100f ? 0x1p-100f : x;
            out.to_log2[lane] = f < 1e-30f ? 1e-30f : f;
            out.lg_v[lane] = lg2_tc(v);
            out.rcp_v[lane] = 1.f / v;
          }
          if (lane == 0) out.change = unit * rcp, out.unit = to, out.there = on;
          unit = to;
          __syncwarp();
          for (int s = 0; s < C::kKSlots && ok; ++s)
            put_pages(&args.k8, page.at, key0_of(i), kk0, kTtKeysPerCta >> box_k, box_k, C::kKCols << box_k, s * C::kKCols);
        } else {
          // A slot's barrier must be at most one phase behind the one that is waited for.  Pages leave the
          // ring to the unpacking warps: once those have placed the last ones, it is.
          for (uint32_t d = 1; d <= 2 && d <= st; ++d) {
            ok = ok && wait_phase(unpacked_bar((st - d) % C::kStages), ((st - d) / C::kStages) & 1u, abort_flag, &g_tree_status);
            ok = __all_sync(0xffffffffu, ok);
          }
          for (int s = 0; s < C::kKSlots && ok; ++s)
            put(is_draft(i) ? &tm_kn : &tm_k, key0_of(i) + kk0, s * (C::kKCols / 64), false);
        }
      };
      if (a.q_tma && lane == 0) {
        if (rank == 0) mbar_arrive_expect_tx(q_full, 2 * C::kQBytes);
        tma_load_5d_pair(base, &tm_q, mapa_shared(q_full, 0), 0, c * a.group, row0 / a.group, 0, b);
      }
      __syncwarp();
      int entry = entry_of(0);
      const int entry1 = entry_of(1);
      const int entry2 = entry_of(2);
      Page page = page_of(entry), next = page_of(entry1);  // of this tile and the next
      entry = entry2;
      put_k(0, page);
      for (int i = 0; i < ntiles && ok; ++i) {
        const Page after = page_of(entry);
        entry = entry_of(i + 3);
        if (i + 1 < ntiles) put_k(i + 1, next);
        if (!ok) break;
        if (is_page(i))
          put_pages(&args.v8, page.at, key0_of(i), 0, kTtBN >> box_v, box_v, (C::kDV / 2) << box_v, vb0 * 64);
        else
          put(is_draft(i) ? &tm_vn : &tm_v, key0_of(i), vb0, careful(i));
        page = next, next = after;
      }
      // As below: copies that nobody awaits any more get time to land.
      if (!ok) {
        const unsigned long long since = globaltimer();
        while (globaltimer() - since < 50000ull) {
        }
      }
    } else if (lane == 0) {
      // ---- TMA producer (both CTAs): the ring in the MMA order; copies complete on the
      // leader's barrier, which expects both CTAs' bytes, or for a careful V on this CTA's.
      uint32_t g = 0;
      bool ok = true;
      auto put = [&](const CUtensorMap* m, int key0, int block0, bool own) {
        if (!ok) return;
        const uint32_t slot = g % C::kSlots, use = g / C::kSlots;
        ok = wait_phase(empty_bar(slot), (use & 1u) ^ 1u, abort_flag, &g_tree_status);
        if (!ok) return;
        uint32_t bar;
        if (own) {
          mbar_arrive_expect_tx(own_bar(slot), C::kSlotBytes);
          bar = mapa_shared(own_bar(slot), rank);
          if (rank == 0) mbar_arrive(full_bar(slot));  // the MMA thread goes by P's barrier
        } else {
          if (rank == 0) mbar_arrive_expect_tx(full_bar(slot), 2 * C::kSlotBytes);
          bar = mapa_shared(full_bar(slot), 0);
        }
        tma_load_5d_pair(ring + slot * C::kSlotBytes, m, bar, 0, key0, block0, c, b);
        ++g;
      };
      const int kk0 = static_cast<int>(rank) * kTtKeysPerCta;
      const int vb0 = half * (C::kDV / 64) + static_cast<int>(rank) * (C::kDV / 128);
      auto put_k = [&](int i) {
        for (int s = 0; s < C::kKSlots; ++s)
          put(is_draft(i) ? &tm_kn : &tm_k, key0_of(i) + kk0, s * (C::kKCols / 64), false);
      };
      if (a.q_tma) {
        if (rank == 0) mbar_arrive_expect_tx(q_full, 2 * C::kQBytes);
        tma_load_5d_pair(base, &tm_q, mapa_shared(q_full, 0), 0, c * a.group, row0 / a.group, 0, b);
      }
      put_k(0);
      for (int i = 0; i < ntiles && ok; ++i) {
        if (i + 1 < ntiles) put_k(i + 1);
        put(is_draft(i) ? &tm_vn : &tm_v, key0_of(i), vb0, careful(i));
      }
      // Every copy issued was awaited by the leader's MMA thread or this CTA's softmax warps
      // unless a wait gave up; then give the last copies time to land before the CTA exits.
      if (!ok) {
        const unsigned long long since = globaltimer();
        while (globaltimer() - since < 50000ull) {
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      // ---- MMA issuer (leader CTA only)
      constexpr bool kHalf = __is_same(T, __half);
      constexpr uint32_t id_s = kHalf ? idesc_fp16(2 * kTtBM, kTtBN, false) : idesc_bf16(2 * kTtBM, kTtBN, false);
      constexpr uint32_t id_o = kHalf ? idesc_fp16(2 * kTtBM, C::kDV, true) : idesc_bf16(2 * kTtBM, C::kDV, true);
      const uint32_t empty_p0 = mapa_shared(empty_bar(0), peer);
      const uint32_t s_full_p0 = mapa_shared(s_full(0), peer);
      const uint32_t pv_done_p0 = mapa_shared(pv_done(0), peer);
      const uint64_t q_desc = smem_desc_sw128(base, 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(ring, 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(ring, kTtBN * 128, 1024);
      uint32_t g = 0;
      bool ok = wait_phase(q_full, 0, abort_flag, &g_tree_status);
      auto take = [&]() {
        const uint32_t slot = g % C::kSlots, use = g / C::kSlots;
        ok = ok && wait_phase(full_bar(slot), use & 1u, abort_flag, &g_tree_status);
        return slot;
      };
      auto release = [&](uint32_t slot) {
        mma_commit_pair(empty_bar(slot));
        mma_commit_pair(empty_p0 + 8u * slot);
        ++g;
      };
      auto issue_s = [&](int i) {
        const int u = i & 1;
        for (int s = 0; s < C::kKSlots && ok; ++s) {
          const uint32_t slot = take();
          if (!ok) return;
          tc_fence_after();
          // Slot: kKCols / 64 blocks of [64 keys x 64 columns]; Q blocks hold the same columns.
#pragma unroll
          for (int h = 0; h < C::kKCols / 64; ++h)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_bf16_ss_pair(tmem + u * kTtBN, q_desc + (((s * (C::kKCols / 64) + h) * (kTtBM * 128) + kk * 32) >> 4),
                               k_desc + ((slot * C::kSlotBytes + h * (kTtKeysPerCta * 128) + kk * 32) >> 4), id_s,
                               (s | h | kk) ? 1u : 0u);
          release(slot);
        }
        if (ok) {
          mma_commit_pair(s_full(u));
          mma_commit_pair(s_full_p0 + 8u * u);
        }
      };
      issue_s(0);
      for (int i = 0; i < ntiles && ok; ++i) {
        if (i + 1 < ntiles) issue_s(i + 1);
        const int u = i & 1;
        ok = ok && wait_phase(p_full(u), (i >> 1) & 1, abort_flag, &g_tree_status);
        const uint32_t slot = take();
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < kTtBN / 16; ++s)
          mma_bf16_ts_pair(tmem + kTtColO, tmem + u * kTtBN + 8 * s,
                           v_desc + ((slot * C::kSlotBytes + s * 16 * 128) >> 4), id_o, (i | s) ? 1u : 0u);
        release(slot);
        mma_commit_pair(pv_done(u));
        mma_commit_pair(pv_done_p0 + 8u * u);
      }
      mma_commit_pair(o_ready);
      mma_commit_pair(mapa_shared(o_ready, peer));
      mbar_wait_bounded(o_ready, 0, nullptr, &g_tree_status);  // no MMA may still write TMEM when it is freed
    }
  } else if (kPaged && warp >= 2 + kTtSoftWarps) {
    if constexpr (kPaged) {
      // ---- unpacking: a staging slot's 16 bytes a thread to 32 in the ring's slot, in the MMA order.  A
      // release to the cluster drains a thread's stores first, some 1000 clocks: two teams of warps
      // take the staging slots in turn, so that one unpacks while the other waits.
      const int team = (warp - 2 - kTtSoftWarps) / kTtUnpackTeam;
      const int tid = threadIdx.x - 32 * (2 + kTtSoftWarps + team * kTtUnpackTeam);
      static_assert(C::kStages % 2 == 0, "a staging slot is one team's");
      uint32_t g = 0, st = 0;
      bool ok = true;
      auto unpack = [&](bool pages, auto columns) {  // (columns: of a row, a constant)
        if (!pages || (st & 1) != team) {
          ++g;
          st += pages;
          return;
        }
        const uint32_t slot = g % C::kSlots, s = st % C::kStages;
        // (in this order: what was put before this step, 16-bit rows among it, has waited for the ring)
        if (ok) ok = mbar_wait_bounded(staged_bar(s), (st / C::kStages) & 1u, abort_flag, &g_tree_status);
        if (ok) ok = wait_phase(empty_bar(slot), ((g / C::kSlots) & 1u) ^ 1u, abort_flag, &g_tree_status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        const uint32_t from = base + C::kOffStage + s * C::kStageBytes, to = ring + slot * C::kSlotBytes;
        // K: [64 keys x kKCols], V: [128 keys x kDV / 2], both of half a slot.
        constexpr int chunks = decltype(columns)::value / 16, keys = C::kStageBytes / 16 / chunks;
        constexpr int kStep = 32 * kTtUnpackTeam / chunks;  // a thread's chunk of every kStep-th row
        static_assert(32 * kTtUnpackTeam % chunks == 0, "a thread stays in its columns");
        const int ch = tid % chunks, r0 = tid / chunks;
        const uint32_t dst = to + (ch >> 2) * (keys * 128);
        // (Short code: several rows' loads ahead of their stores cost more, in instructions, than the waits.)
#pragma unroll 1
        for (int row = r0; row < keys; row += kStep) {
          uint32_t x[4], y[8];
          asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                       : "r"(from + (row * chunks + ch) * 16)
                       : "memory");
#pragma unroll
          for (int q = 0; q < 4; ++q) paged_unpack<T>(x[q], 0x4140u, 0x4342u, y[2 * q], y[2 * q + 1]);
          const uint32_t at = dst + row * 128 + (((2 * ch & 7) ^ (row & 7)) << 4);
          st_shared_v4(at, y[0], y[1], y[2], y[3]);
          st_shared_v4(at ^ 16u, y[4], y[5], y[6], y[7]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(unpacked_bar(s));
          mbar_arrive_cluster(mapa_shared(full_bar(slot), 0));
        }
        __syncwarp();
        ++g, ++st;
      };
      using K = std::integral_constant<int, C::kKCols>;
      using V = std::integral_constant<int, C::kDV / 2>;
      for (int s = 0; s < C::kKSlots; ++s) unpack(is_page(0), K());
      for (int i = 0; i < ntiles && ok && is_page(i); ++i) {
        if (i + 1 < ntiles)
          for (int s = 0; s < C::kKSlots; ++s) unpack(is_page(i + 1), K());
        unpack(true, V());
      }
    }
  } else {
    // ---- softmax: row r = TMEM lane r is shared by warps w and w + 4, 64 keys each.
    const int quarter = warp & 3;
    const int hv = (warp - 2) >> 2;
    const int r = quarter * 32 + lane;
    const int tid = threadIdx.x - 64;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t p_full_l0 = mapa_shared(p_full(0), 0);
    volatile float* xch = reinterpret_cast<volatile float*>(smem + C::kOffXch);
    const volatile uint32_t* poison = reinterpret_cast<const volatile uint32_t*>(smem + C::kOffPoison);
    auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); };
    auto softmax_sync = [&]() { asm volatile("bar.sync 5, %0;" ::"n"(32 * kTtSoftWarps) : "memory"); };

    // Q rows that no TMA box describes (128 rows are whole tokens only for a group that divides
    // 128), swizzled as the TMA would: 64-column blocks of [128 rows x 128 bytes].
    if (!a.q_tma) {
      // Thread: one 16-byte chunk of every (2048 / D)-th row; 8 loads in flight.
      constexpr int kStep = 32 * kTtSoftWarps / (D / 8);
      const int ch = tid % (D / 8);
#pragma unroll 1
      for (int q0 = tid / (D / 8); q0 < kTtBM; q0 += 8 * kStep) {
        uint4 w[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int qr = row0 + q0 + x * kStep;
          int i, g;
          tree_row(a, qr, i, g);
          w[x] = make_uint4(0, 0, 0, 0);
          if (qr < rows && ch < DR / 8)
            w[x] = *reinterpret_cast<const uint4*>(a.q + b * a.q_b + (static_cast<int64_t>(c) * a.group + g) * a.q_h +
                                                   i * a.q_t + ch * 8);
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int qr = q0 + x * kStep;
          st_shared_v4(base + (ch >> 3) * (kTtBM * 128) + qr * 128 + (((ch & 7) ^ (qr & 7)) << 4), w[x].x, w[x].y, w[x].z,
                       w[x].w);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(q_full, 0));
    }
    const bool drafts = t1 > nc;
    const int j_begin = drafts ? (max(t0, nc) - nc) * kTtBN : 0, j_end = drafts ? min((t1 - nc) * kTtBN, a.n) : 0;
    const int rr = row0 + r;
    int tok, head;
    tree_row(a, rr, tok, head);
    if (rr >= rows) tok = -1;
    const int dep = tok >= 0 ? tree_depth(a, b, tok) : 0;
    const int first = tok >= 0 ? tree_first(a, len, dep) : len;
    const float scale = a.scale_log2;
    float m = -INFINITY, l = 0.f;
    float unit = kPaged ? __uint_as_float(0x00800000u) : 1.f;  // of O (2^-126: nothing added yet)
    bool ok = true;
    uint32_t own_phase = 0;  // next parity of each own_bar
    // Every warp runs every iteration and meets its partner at the same pair barriers on
    // every path: after a timeout it only skips its waits and its work.
    for (int i = 0; i < ntiles; ++i) {
      const int u = i & 1, key0 = key0_of(i);
      const bool draft = is_draft(i), care = careful(i);
      if (ok) ok = mbar_wait_bounded(s_full(u), (i >> 1) & 1, abort_flag, &g_tree_status);
      if (ok && i >= 2) ok = mbar_wait_bounded(pv_done(u), ((i - 2) >> 1) & 1, abort_flag, &g_tree_status);
      ok = __all_sync(0xffffffffu, ok);
      uint32_t sv[2][32];
      float mx = -INFINITY;
      float to_log2[4] = {scale, scale, scale, scale};  // of 16 keys each
      if (ok) {
        tc_fence_after();
        tmem_ld_32x32b_x32(tmem + lane_off + u * kTtBN + 64 * hv, sv[0]);
        tmem_ld_32x32b_x32(tmem + lane_off + u * kTtBN + 64 * hv + 32, sv[1]);
        tmem_wait_ld();
        // Pages that every row sees whole need no masks (nor do rows behind the last: nobody reads theirs).
        const int k0 = key0 + 64 * hv;
        bool plain = false;
        if constexpr (kPaged) {
          if (is_page(i)) plain = k0 + 64 <= full && (tok < 0 || first <= k0) && (scales[i % C::kScales].there >> (4 * hv) & 15u) == 15u;
          plain = __all_sync(0xffffffffu, plain);
        }
        if (!plain) {
          // What the row sees, one bit per key of each 32-key half.
          uint32_t keep[2];
          if (draft) {
            if (a.tree == nullptr && a.depth == nullptr) {  // a plain chunk: closed forms
#pragma unroll
              for (int j = 0; j < 2; ++j) keep[j] = tok >= 0 ? tree_sees32(a, b, tok, k0 + 32 * j, dep, sink_left) : 0u;
            } else {
              tree_sees64_rows(a, b, tok, k0, dep, keep, sink_left);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if constexpr (kPaged) {
                // Positions from p0 on, below the full pages' end or (the tail) the length.
                const int p0 = (is_page(i) ? 0 : full) + k0 + 32 * j, hi = min((is_page(i) ? full : len) - 1 - p0, 31);
                const int lo = max(first - p0, 0), sk = tok >= 0 ? min(a.sink - p0, 32) : 0;
                uint32_t on = lo > 31 ? 0u : 0xFFFFFFFFu << lo;
                if (a.window > 0 && sk > 0) on |= 0xFFFFFFFFu >> (32 - sk);
                keep[j] = hi < 0 ? 0u : (0xFFFFFFFFu >> (31 - hi)) & on;
                if (is_page(i)) {
                  const uint32_t on16 = scales[i % C::kScales].there >> (4 * hv + 2 * j);
                  if (!(on16 & 1u)) keep[j] &= 0xFFFF0000u;
                  if (!(on16 & 2u)) keep[j] &= 0x0000FFFFu;
                }
              } else {
                const int lo = max(first - k0 - 32 * j, 0), hi = min(len - 1 - k0 - 32 * j, 31);
                keep[j] = hi < lo ? 0u : (0xFFFFFFFFu >> (31 - hi)) & (0xFFFFFFFFu << lo);
              }
            }
          }
          if (!__all_sync(0xffffffffu, (keep[0] & keep[1]) == 0xFFFFFFFFu)) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((keep[j] >> e) & 1u)) sv[j][e] = __float_as_uint(-INFINITY);
          }
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if constexpr (kPaged) {  // 16 keys have one scale; in log2 units
#pragma unroll
          for (int e = 0; e < 64; ++e) m4[e >> 4] = fmaxf(m4[e >> 4], __uint_as_float(sv[e >> 5][e & 31]));
          if (is_page(i)) {
            const float4 f = *reinterpret_cast<const float4*>(&scales[i % C::kScales].to_log2[4 * hv]);
            to_log2[0] = f.x, to_log2[1] = f.y, to_log2[2] = f.z, to_log2[3] = f.w;
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) m4[q] *= to_log2[q];
        } else {
#pragma unroll
          for (int e = 0; e < 64; ++e) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(sv[e >> 5][e & 31]));
        }
        mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        if (!kPaged && a.scores != nullptr && half == 0 && tok >= 0) {
          float* dst = a.scores + (static_cast<int64_t>(bc) * rows + rr) * a.score_pitch + (draft ? a.draft_at : 0) + k0;
          const int left = (draft ? a.n : len) - k0;
          // (16 bytes at a time: the row's two parts begin and end on multiples of 4 slots, so the last
          // store passes its end by up to 3 slots that nothing reads.)
#pragma unroll
          for (int e = 0; e < 64; e += 4)
            if (e < left)
              *reinterpret_cast<float4*>(dst + e) =
                  make_float4(__uint_as_float(sv[e >> 5][e & 31]) * scale, __uint_as_float(sv[e >> 5][(e + 1) & 31]) * scale,
                              __uint_as_float(sv[e >> 5][(e + 2) & 31]) * scale,
                              __uint_as_float(sv[e >> 5][(e + 3) & 31]) * scale);
        }
      }
      __syncwarp();
      xch[hv * kTtBM + r] = mx;
      tc_fence_before();
      pair_sync();  // both halves of S are in registers and both maxima are posted
      tc_fence_after();
      mx = fmaxf(mx, xch[(hv ^ 1) * kTtBM + r]);
      pair_sync();  // the partner's maximum is read before either posts the next one
      if (!ok) continue;
      const float mt = kPaged ? mx : mx * scale;
      const bool move = mt > m + TreeRef<T>::kSlack;
      // O's unit: not below any scale of V so far, 1 from the first 16-bit rows on (the same in all
      // threads of the pair).
      float change = unit;
      if constexpr (kPaged) {
        if (is_page(i)) change = scales[i % C::kScales].change;
      }
      const bool other = kPaged && change != 1.f;
      if (__any_sync(0xffffffffu, move) || other) {
        const float mn = move ? mt - TreeRef<T>::kBelow : m;
        float corr = move ? ex2_tc(m - mn) : 1.f;
        l *= corr;
        if constexpr (kPaged) {
          corr *= change;
          unit = is_page(i) ? scales[i % C::kScales].unit : 1.f;
        }
        if (i > 0) {
          ok = mbar_wait_bounded(pv_done((i - 1) & 1), ((i - 1) >> 1) & 1, abort_flag, &g_tree_status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) continue;
          tc_fence_after();
#pragma unroll 1
          for (int e = 0; e < C::kDV / 64; ++e) {
            uint32_t ov[32];
            const uint32_t col = kTtColO + (C::kDV / 2) * hv + e * 32;
            tmem_ld_32x32b_x32(tmem + lane_off + col, ov);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; ++x) ov[x] = __float_as_uint(__uint_as_float(ov[x]) * corr);
            tmem_st_32x32b_x32(tmem + lane_off + col, ov);
          }
        }
        m = mn;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      float l4[4] = {0.f, 0.f, 0.f, 0.f};
      if constexpr (kPaged) {
        // P in O's unit, the scale of V in the exponent: 2^(x - m + log2 v); l takes it back, 16 keys
        // at a time.
        float4 lg = make_float4(0.f, 0.f, 0.f, 0.f), rv = make_float4(1.f, 1.f, 1.f, 1.f);
        if (is_page(i)) {
          lg = *reinterpret_cast<const float4*>(&scales[i % C::kScales].lg_v[4 * hv]);
          rv = *reinterpret_cast<const float4*>(&scales[i % C::kScales].rcp_v[4 * hv]);
        }
        const float lgs[4] = {lg.x, lg.y, lg.z, lg.w}, rvs[4] = {rv.x, rv.y, rv.z, rv.w};
#pragma unroll
        for (int half16 = 0; half16 < 2; ++half16) {
          uint32_t pw[16];
#pragma unroll
          for (int q = 2 * half16; q < 2 * half16 + 2; ++q) {
            const float odd = to_log2[q] + lgs[q], ref_q = ref - lgs[q];
#pragma unroll
            for (int e = 8 * q; e < 8 * q + 8; ++e) {
              const float x0 = __uint_as_float(sv[e >> 4][(2 * e) & 31]), x1 = __uint_as_float(sv[e >> 4][(2 * e + 1) & 31]);
              const float p0 = ex2_tc(fmaf(x0, to_log2[q], -ref_q)), p1 = ex2_tc(fmaf(x1, to_log2[q], -ref_q));
              l4[q] += p0 + p1;
              pw[e & 15] = pack2<T>(p0, p1);
            }
            l4[q] *= rvs[q];
            if (odd != odd) {  // a NaN scale is for the rows that see the page (the same in the whole warp)
              l4[q] = 0.f;
#pragma unroll
              for (int e = 8 * q; e < 8 * q + 8; ++e) {
                const bool on0 = __uint_as_float(sv[e >> 4][(2 * e) & 31]) != -INFINITY;
                const bool on1 = __uint_as_float(sv[e >> 4][(2 * e + 1) & 31]) != -INFINITY;
                pw[e & 15] = pack2<T>(on0 ? odd : 0.f, on1 ? odd : 0.f);
                if (on0 || on1) l4[q] = odd;
              }
            }
          }
          tmem_st_32x32b_x16(tmem + lane_off + u * kTtBN + 32 * hv + 16 * half16, pw);
        }
      } else {
        uint32_t pw[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float p0 = ex2_tc(fmaf(__uint_as_float(sv[e >> 4][(2 * e) & 31]), scale, -ref));
          const float p1 = ex2_tc(fmaf(__uint_as_float(sv[e >> 4][(2 * e + 1) & 31]), scale, -ref));
          l4[e & 3] += p0 + p1;
          pw[e] = pack2<T>(p0, p1);
        }
        tmem_st_32x32b_x32(tmem + lane_off + u * kTtBN + 32 * hv, pw);
      }
      l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      if (care) {
        // This CTA's columns of V: rows behind the length read as zeros, and of new tokens
        // everything that is not finite.
        const uint32_t slot = v_pos(i) % C::kSlots;
        ok = mbar_wait_bounded(own_bar(slot), (own_phase >> slot) & 1u, abort_flag, &g_tree_status);
        own_phase ^= 1u << slot;
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          uint8_t* vs = smem + C::kOffRing + slot * C::kSlotBytes;
          for (int e = tid; e < C::kSlotBytes / 16; e += 32 * kTtSoftWarps) {
            const int row = (e >> 3) & (kTtBN - 1);  // blocks of [128 keys x 128 bytes]
            uint4* w = reinterpret_cast<uint4*>(vs) + e;
            if (!draft) {
              const int p = full + key0 + row;
              if (p >= len || (p < span.low && (!kPaged || p >= a.sink))) *w = make_uint4(0, 0, 0, 0);
            } else {
              uint4 x = *w;
              if (nonfinite_bits<T>(x.x) | nonfinite_bits<T>(x.y) | nonfinite_bits<T>(x.z) | nonfinite_bits<T>(x.w)) {
                uint32_t* xs = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  xs[q] &= ~((nonfinite_bits<T>(xs[q]) >> 15) * 0xFFFFu);
                *w = x;
                // Both CTAs' rows may see the token: mark it in both.  (Ordered before the epilogues
                // by the hand-over of P, the MMA that reads it and its completion.)
                const int j = key0 + row;
                const uint32_t word = base + C::kOffPoison + ((j >> 5) & (kPoisonWords - 1)) * 4;
                red_or_cluster(mapa_shared(word, 0), 1u << (j & 31));
                red_or_cluster(mapa_shared(word, 1), 1u << (j & 31));
              }
            }
          }
          fence_proxy_async_smem();
        }
        __syncwarp();  // (the wait below is aligned)
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (care)
          mbar_arrive_cluster(p_full_l0 + 8u * u);  // V's cleared rows are shared memory of this CTA
        else if (rank == 0)
          mbar_arrive(p_full(u));
        else
          mbar_arrive_tmem_handoff(p_full_l0 + 8u * u);
      }
    }
    if (ok) ok = mbar_wait_bounded(o_ready, 0, abort_flag, &g_tree_status);
    const bool good = __all_sync(0xffffffffu, ok);
    xch[hv * kTtBM + r] = l;
    softmax_sync();
    const float lt = l + xch[(hv ^ 1) * kTtBM + r];
    bool poisoned = false;  // the row sees such a token
    if (drafts && tok >= 0)
      for (int j = j_begin; j < j_end && !poisoned; j += 32) {
        const uint32_t bits = poison_of(poison, j);
        poisoned = bits != 0u && (bits & tree_sees32(a, b, tok, j, dep, sink_left)) != 0u;
      }
    __syncwarp();
    // The rows go through shared memory (Q and the ring are idle: every MMA has completed) to
    // one bulk copy each: a thread that stores its own row touches 32 rows a warp.
    const int esz = a.splits == 1 ? 2 : 4;
    const int pitch = C::kDV * esz + 16;  // an odd number of 16-byte chunks: no bank conflicts
    if (good) {
      tc_fence_after();
      const float inv = lt == 0.f ? 0.f : 1.f / lt;  // a row that sees nothing: zeros
      // (O in units of 1; a value of a row whose every P was 0 stays 0)
      auto whole = [&](uint32_t (&ov)[32]) {
        if (kPaged && unit != 1.f) {
#pragma unroll
          for (int x = 0; x < 32; ++x) ov[x] = __float_as_uint(__uint_as_float(ov[x]) * unit);
        }
      };
#pragma unroll 1
      for (int e = 0; e < C::kDV / 64; ++e) {
        uint32_t ov[32];
        const int col = (C::kDV / 2) * hv + e * 32;  // of this half
        tmem_ld_32x32b_x32(tmem + lane_off + kTtColO + col, ov);
        tmem_wait_ld();
        whole(ov);
        if (poisoned && col < DR) {
#pragma unroll 1
          for (int j0 = j_begin; j0 < j_end; j0 += 32) {
            uint32_t bits = poison_of(poison, j0);
            if (bits != 0u) bits &= tree_sees32(a, b, tok, j0, dep, sink_left);
            for (; bits != 0u; bits &= bits - 1u) {
              const uint16_t* vn = a.vn + b * a.vn_b + c * a.vn_h + (j0 + __ffs(bits) - 1) * a.vn_t + half * C::kDV + col;
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (tree_nonfinite<T>(vn[x])) ov[x] = __float_as_uint(__uint_as_float(ov[x]) + tree_f32<T>(vn[x]));
            }
          }
        }
        const uint32_t dst = base + r * pitch + col * esz;
        if (a.splits == 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
              w[x] = pack2<T>(__uint_as_float(ov[8 * j + 2 * x]) * inv, __uint_as_float(ov[8 * j + 2 * x + 1]) * inv);
            st_shared_v4(dst + 16 * j, w[0], w[1], w[2], w[3]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) st_shared_v4(dst + 16 * j, ov[4 * j], ov[4 * j + 1], ov[4 * j + 2], ov[4 * j + 3]);
        }
        __syncwarp();
      }
      fence_proxy_async_smem();
    }
    // All softmax warps meet here on every path; the rows are stored only if each has staged its own.
    uint32_t all_good;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "bar.red.and.pred p, 5, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(all_good)
        : "r"(good ? 1u : 0u), "n"(32 * kTtSoftWarps)
        : "memory");
    if (all_good) {
      if (hv == 0 && tok >= 0) {
        void* dst = a.splits == 1
                        ? static_cast<void*>(a.o + b * a.o_b + (static_cast<int64_t>(c) * a.group + head) * a.o_h + tok * a.o_t +
                                             half * C::kDV)
                        : static_cast<void*>(a.part_o + (part_row + r) * DR + half * C::kDV);
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(base + r * pitch),
                     "r"((DR < C::kDV ? DR : C::kDV) * esz)
                     : "memory");
        bulk_commit_group();
        bulk_wait_group_read<0>();  // (the grid's completion covers the writes)
      }
      if (half == 0 && hv == 0 && tok >= 0) {
        if (a.splits > 1)
          a.part_ml[part_row + r] = make_float2(m, lt);
        else if (a.lse != nullptr)
          a.lse[static_cast<int64_t>(bc) * rows + rr] = lt == 0.f ? INFINITY : m + log2f(lt);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // no CTA leaves while its peer may still touch its barriers, TMEM or copies
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, kTtTmemCols);
  }
}

}  // namespace w8

namespace w8host {

using TreeEncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static TreeEncodeFn tree_encode_fn() {
  static TreeEncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<TreeEncodeFn>(p);
  });
  return fn;
}

// A 5-D map of a cache's rows or pages.
int tree_encode(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, const cuuint64_t* dims,
                const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle, const char* what) {
  TreeEncodeFn enc = tree_encode_fn();
  if (enc == nullptr) {
    set_error("cuTensorMapEncodeTiled is not available from the driver");
    return W8_ERR_CUDA;
  }
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, type, 5, const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled (cache attention, %s) failed with CUresult %d", what, static_cast<int>(r));
    return W8_ERR_CUDA;
  }
  return W8_OK;
}

// 5-D map over rows [batch, heads, n] of d elements: (64 columns, row, 64-column block, head,
// batch).  A box {64, rows, blocks, 1, 1} lands as `blocks` 128-byte-swizzled [rows x 64]
// blocks; rows behind n and blocks behind d / 64 read as zeros.
int tree_encode_rows(CUtensorMap* map, const void* ptr, bool half, int64_t d, int64_t n, int64_t heads, int64_t batch,
                       int64_t s_b, int64_t s_h, int64_t s_n, uint32_t rows, uint32_t blocks) {
  // A dimension of one element has no stride to speak of: any valid one.
  auto bytes = [&](int64_t size, int64_t stride) { return static_cast<cuuint64_t>(size > 1 ? stride * 2 : d * 2); };
  const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(d / 64),
                              static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(batch)};
  const cuuint64_t strides[4] = {bytes(n, s_n), 128, bytes(heads, s_h), bytes(batch, s_b)};
  const cuuint32_t box[5] = {64, rows, blocks, 1, 1};
  return tree_encode(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, ptr, dims, strides,
                     box, CU_TENSOR_MAP_SWIZZLE_128B, "rows");
}

// 5-D map over q: (64 columns, head, token, 64-column block, batch).  A box {64, group,
// 128 / group, blocks, 1} lands as `blocks` swizzled blocks of 128 rows i * group + g, zeros
// behind the d / 64-th.
static int encode_q(CUtensorMap* map, const w8::TreeArgs& a, bool half, int64_t d, uint32_t blocks) {
  const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
  auto bytes = [&](int64_t size, int64_t stride) { return static_cast<cuuint64_t>(size > 1 ? stride * 2 : d * 2); };
  const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(a.n),
                              static_cast<cuuint64_t>(d / 64), static_cast<cuuint64_t>(a.batch)};
  const cuuint64_t strides[4] = {bytes(heads, a.q_h), bytes(a.n, a.q_t), 128, bytes(a.batch, a.q_b)};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(w8::kTtBM / a.group),
                             blocks, 1};
  return tree_encode(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.q, dims, strides,
                     box, CU_TENSOR_MAP_SWIZZLE_128B, "q");
}

template <typename T, int D, int DR, bool kPaged, typename Args>
static int launch_tc(const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tkn, const CUtensorMap& tvn,
                     const w8::TreeArgs& a, const Args& args, int64_t items, int device, cudaStream_t stream) {
  using C = w8::TtCfg<D, kPaged>;
  CUtensorMap tq = tkn;
  if (a.q_tma) {
    const int st = encode_q(&tq, a, __is_same(T, __half), DR, D / 64);
    if (st != W8_OK) return st;
  }
  static bool done[64] = {};
  if (!done[device]) {
    W8_CUDA_TRY(cudaFuncSetAttribute(w8::attn_tree_tc_kernel<T, D, DR, kPaged, Args>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    done[device] = true;
  }
  const int64_t blocks = 2 * items * a.splits * C::kSplitD;
  W8_CHECK_ARG(blocks < (1ll << 31), "too many row tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(C::kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(
      cudaLaunchKernelEx(&cfg, w8::attn_tree_tc_kernel<T, D, DR, kPaged, Args>, tq, tk, tv, tkn, tvn, args));
}

template <typename T, int D, int DR = D>
static int tree_tc_go(const w8::TreeArgs& a, int64_t items, int device, cudaStream_t stream) {
  using C = w8::TtCfg<D, false>;
  constexpr bool kHalf = __is_same(T, __half);
  CUtensorMap tk, tv, tkn, tvn;
  const uint32_t kb = C::kKCols / 64, vb = C::kDV / 128;
  int st = tree_encode_rows(&tkn, a.kn, kHalf, DR, a.n, a.kv_heads, a.batch, a.kn_b, a.kn_h, a.kn_t, w8::kTtKeysPerCta, kb);
  if (st != W8_OK) return st;
  st = tree_encode_rows(&tvn, a.vn, kHalf, DR, a.n, a.kv_heads, a.batch, a.vn_b, a.vn_h, a.vn_t, w8::kTtBN, vb);
  if (st != W8_OK) return st;
  tk = tkn, tv = tvn;  // an empty cache: never read
  if (a.slots > 0) {
    st = tree_encode_rows(&tk, a.k, kHalf, DR, a.slots, a.kv_heads, a.batch, a.k_b, a.k_h, a.k_s, w8::kTtKeysPerCta, kb);
    if (st != W8_OK) return st;
    st = tree_encode_rows(&tv, a.v, kHalf, DR, a.slots, a.kv_heads, a.batch, a.v_b, a.v_h, a.v_s, w8::kTtBN, vb);
    if (st != W8_OK) return st;
  }
  return launch_tc<T, D, DR, false>(tk, tv, tkn, tvn, a, a, items, device, stream);
}

// The tcgen05 schedule of w8_attention_tree (arguments checked by the caller; rows in tiles of
// 256).
int tree_tc(const w8::TreeArgs& a, bool half, int64_t d, int64_t items, int device, cudaStream_t stream) {
  if (d == 64)
    return half ? tree_tc_go<__half, 128, 64>(a, items, device, stream)
                : tree_tc_go<__nv_bfloat16, 128, 64>(a, items, device, stream);
  if (d == 128)
    return half ? tree_tc_go<__half, 128>(a, items, device, stream) : tree_tc_go<__nv_bfloat16, 128>(a, items, device, stream);
  if (d == 256)
    return half ? tree_tc_go<__half, 256>(a, items, device, stream) : tree_tc_go<__nv_bfloat16, 256>(a, items, device, stream);
  return half ? tree_tc_go<__half, 512>(a, items, device, stream) : tree_tc_go<__nv_bfloat16, 512>(a, items, device, stream);
}

// 5-D map over pages of 8-bit rows: (byte, row, 1, head, page).  A box {bytes, rows, 1, 1, 1} lands
// as rows of so many bytes, zeros behind the head's.
static int encode_pages(CUtensorMap* map, const void* ptr, int64_t d, int64_t page, int64_t heads, int64_t pages,
                        const int64_t* stride, uint32_t bytes, uint32_t rows) {
  auto of = [&](int64_t size, int64_t s) { return static_cast<cuuint64_t>(size > 1 ? s : d); };
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(page), 1, static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(pages)};
  const cuuint64_t strides[4] = {of(page, stride[2]), static_cast<cuuint64_t>(d), of(heads, stride[1]), of(pages, stride[0])};
  const cuuint32_t box[5] = {bytes, rows, 1, 1, 1};
  return tree_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE, "pages");
}

template <typename T, int D, int DR = D>
static int paged_tc_go(const w8_attention_paged_args& x, const w8::PagedArgs& pa, int64_t items, int device,
                       cudaStream_t stream) {
  using C = w8::TtCfg<D, true>;
  constexpr bool kHalf = __is_same(T, __half);
  const w8::TreeArgs& a = pa.t;
  CUtensorMap tkn, tvn, tkt, tvt;
  w8::TtPagedArgs args;
  static_cast<w8::PagedArgs&>(args) = pa;
  auto rows = [&](CUtensorMap* map, const void* p, int64_t n, const int64_t* s, bool v) {
    return tree_encode_rows(map, p, kHalf, DR, n, a.kv_heads, a.batch, s[0], s[1], s[2], v ? w8::kTtBN : w8::kTtKeysPerCta,
                            v ? C::kDV / 128 : C::kKCols / 64);
  };
  int st = rows(&tkn, x.k_new, a.n, x.k_new_stride, false);
  if (st == W8_OK) st = rows(&tvn, x.v_new, a.n, x.v_new_stride, true);
  if (st == W8_OK) st = rows(&tkt, x.k_tail, x.page, x.k_tail_stride, false);
  if (st == W8_OK) st = rows(&tvt, x.v_tail, x.page, x.v_tail_stride, true);
  args.k8 = tkn, args.v8 = tvn;  // an empty pool: never read
  const uint32_t box_k = static_cast<uint32_t>(std::min<int64_t>(x.page, w8::kTtKeysPerCta));
  const uint32_t box_v = static_cast<uint32_t>(std::min<int64_t>(x.page, w8::kTtBN));
  if (st == W8_OK && x.pages > 0)
    st = encode_pages(&args.k8, x.k, DR, x.page, x.kv_heads, x.pages, x.k_stride, C::kKCols, box_k);
  if (st == W8_OK && x.pages > 0)
    st = encode_pages(&args.v8, x.v, DR, x.page, x.kv_heads, x.pages, x.v_stride, C::kDV / 2, box_v);
  if (st != W8_OK) return st;
  return launch_tc<T, D, DR, true>(tkt, tvt, tkn, tvn, a, args, items, device, stream);
}

// The same of w8_attention_paged.
int paged_tc(const w8_attention_paged_args& x, const w8::PagedArgs& a, bool half, int64_t items, int device,
             cudaStream_t stream) {
  using B = __nv_bfloat16;
  switch (x.head_dim) {
    case 64:
      return half ? paged_tc_go<__half, 128, 64>(x, a, items, device, stream)
                  : paged_tc_go<B, 128, 64>(x, a, items, device, stream);
    case 128:
      return half ? paged_tc_go<__half, 128>(x, a, items, device, stream) : paged_tc_go<B, 128>(x, a, items, device, stream);
    case 256:
      return half ? paged_tc_go<__half, 256>(x, a, items, device, stream) : paged_tc_go<B, 256>(x, a, items, device, stream);
    default:
      return half ? paged_tc_go<__half, 512>(x, a, items, device, stream) : paged_tc_go<B, 512>(x, a, items, device, stream);
  }
}

// Read (and optionally clear) this schedule's sticky device status.
int tree_tc_device_status(int clear, int* out) {
  int v = 0;
  W8_CUDA_TRY(cudaMemcpyFromSymbol(&v, w8::g_tree_status, sizeof(int)));
  if (clear) {
    const int zero = 0;
    W8_CUDA_TRY(cudaMemcpyToSymbol(w8::g_tree_status, &zero, sizeof(int)));
  }
  *out = v;
  return W8_OK;
}

}  // namespace w8host
