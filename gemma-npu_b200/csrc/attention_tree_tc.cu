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
#include "attention_tree.cuh"
#include "attn_tc.cuh"

#include <algorithm>
#include <mutex>

namespace w8 {

constexpr int kTtBM = 128;                 // rows per CTA; 256 per pair
constexpr int kTtBN = 128;                 // keys per tile
constexpr int kTtSoftWarps = 8;
constexpr int kTtThreads = 32 * (2 + kTtSoftWarps);
constexpr int kTtKeysPerCta = kTtBN / 2;
constexpr uint32_t kTtTmemCols = 512;
constexpr uint32_t kTtColO = 2 * kTtBN;

template <int D>
struct TtCfg {
  static constexpr int kDV = D < 256 ? D : 256;           // output columns per pair
  static constexpr int kSplitD = D / kDV;                 // clusters per row block (D = 512: 2)
  static constexpr int kQBytes = kTtBM * D * 2;
  static constexpr int kKCols = D < 256 ? D : 256;        // columns of the reduction per K slot
  static constexpr int kKSlots = D / kKCols;              // slots per K tile
  static constexpr int kSlotBytes = kTtBN * kDV;          // K: 64 keys x kKCols; V: 128 keys x kDV / 2
  static constexpr int kSlots = D == 512 ? 3 : D == 256 ? 5 : 8;
  static constexpr int kOffRing = kQBytes;
  static constexpr int kOffBar = kOffRing + kSlots * kSlotBytes;
  // full[kSlots], empty[kSlots], own[kSlots], q_full, s_full[2], p_full[2], pv_done[2], o_ready
  static constexpr int kNumBars = 3 * kSlots + 8;
  static constexpr int kOffXch = kOffBar + kNumBars * 8 + 16;
  static constexpr int kOffPoison = kOffXch + 2 * kTtBM * 4;
  static constexpr int kSmem = kOffPoison + kPoisonWords * 4 + 1024;
  static_assert(kKCols == kDV, "K and V slots have one size");
  static_assert(kSmem <= 232448, "shared memory budget exceeded");
  static_assert(kTtBM * (kDV * 4 + 16) <= kOffBar, "the output rows fit over Q and the ring");
};

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
template <typename T, int D, int DR>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTtThreads, 1)
    attn_tree_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ CUtensorMap tm_kn, const __grid_constant__ CUtensorMap tm_vn,
                        const __grid_constant__ TreeArgs a) {
  using C = TtCfg<D>;
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
      mbar_init(full_bar(s), 1);   // leader: one arrive.expect_tx + both CTAs' bytes
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
    *abort_flag = 0;
    fence_mbar_init();
    if (a.q_tma) prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    prefetch_tmap(&tm_kn);
    prefetch_tmap(&tm_vn);
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
  const TreeSpan span = tree_span<2 * kTtBM, kTtBN>(a, len, rt);
  const int nc = span.c1 - span.c0, nt = nc + span.nd;
  const int t0 = static_cast<int>(static_cast<int64_t>(nt) * split / a.splits);
  const int t1 = static_cast<int>(static_cast<int64_t>(nt) * (split + 1) / a.splits);
  const int ntiles = t1 - t0;
  const int64_t part_row = (static_cast<int64_t>(item) * a.splits + split) * (2 * kTtBM) + rank * kTtBM;
  auto is_draft = [&](int i) { return t0 + i >= nc; };
  auto key0_of = [&](int i) { return (t0 + i >= nc ? t0 + i - nc : span.c0 + t0 + i) * kTtBN; };
  // Of a causal chunk's tiles of new tokens, those that every row of the pair sees whole are as
  // plain as committed ones.
  const int tok_lo = rt * (2 * kTtBM) / a.group, tok_hi = (min((rt + 1) * (2 * kTtBM), rows) - 1) / a.group;
  auto careful = [&](int i) {
    const int key0 = key0_of(i);
    if (!is_draft(i)) return key0 + kTtBN > len || key0 < span.low;
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
    if (lane == 0) {
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
      if (ok) {
        tc_fence_after();
        tmem_ld_32x32b_x32(tmem + lane_off + u * kTtBN + 64 * hv, sv[0]);
        tmem_ld_32x32b_x32(tmem + lane_off + u * kTtBN + 64 * hv + 32, sv[1]);
        tmem_wait_ld();
        // What the row sees, one bit per key of each 32-key half.
        uint32_t keep[2];
        const int k0 = key0 + 64 * hv;
        if (draft) {
          if (a.tree == nullptr && a.depth == nullptr) {  // a plain chunk: closed forms
#pragma unroll
            for (int j = 0; j < 2; ++j) keep[j] = tok >= 0 ? tree_sees32(a, b, tok, k0 + 32 * j, dep) : 0u;
          } else {
            tree_sees64_rows(a, b, tok, k0, dep, keep);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int lo = max(first - k0 - 32 * j, 0), hi = min(len - 1 - k0 - 32 * j, 31);
            keep[j] = hi < lo ? 0u : (0xFFFFFFFFu >> (31 - hi)) & (0xFFFFFFFFu << lo);
          }
        }
        if (!__all_sync(0xffffffffu, (keep[0] & keep[1]) == 0xFFFFFFFFu)) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((keep[j] >> e) & 1u)) sv[j][e] = __float_as_uint(-INFINITY);
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 64; ++e) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(sv[e >> 5][e & 31]));
        mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        if (a.scores != nullptr && half == 0 && tok >= 0) {
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
      const float mt = mx * scale;
      const bool move = mt > m + TreeRef<T>::kSlack;
      if (__any_sync(0xffffffffu, move)) {
        const float mn = move ? mt - TreeRef<T>::kBelow : m;
        const float corr = move ? ex2_tc(m - mn) : 1.f;
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
        l *= corr;
        m = mn;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      float l4[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t pw[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float p0 = ex2_tc(fmaf(__uint_as_float(sv[e >> 4][(2 * e) & 31]), scale, -ref));
        const float p1 = ex2_tc(fmaf(__uint_as_float(sv[e >> 4][(2 * e + 1) & 31]), scale, -ref));
        l4[e & 3] += p0 + p1;
        pw[e] = pack2<T>(p0, p1);
      }
      tmem_st_32x32b_x32(tmem + lane_off + u * kTtBN + 32 * hv, pw);
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
              if (key0 + row >= len || key0 + row < span.low) *w = make_uint4(0, 0, 0, 0);
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
        poisoned = bits != 0u && (bits & tree_sees32(a, b, tok, j, dep)) != 0u;
      }
    __syncwarp();
    // The rows go through shared memory (Q and the ring are idle: every MMA has completed) to
    // one bulk copy each: a thread that stores its own row touches 32 rows a warp.
    const int esz = a.splits == 1 ? 2 : 4;
    const int pitch = C::kDV * esz + 16;  // an odd number of 16-byte chunks: no bank conflicts
    if (good) {
      tc_fence_after();
      const float inv = lt == 0.f ? 0.f : 1.f / lt;  // a row that sees nothing: zeros
#pragma unroll 1
      for (int e = 0; e < C::kDV / 64; ++e) {
        uint32_t ov[32];
        const int col = (C::kDV / 2) * hv + e * 32;  // of this half
        tmem_ld_32x32b_x32(tmem + lane_off + kTtColO + col, ov);
        tmem_wait_ld();
        if (poisoned && col < DR) {
#pragma unroll 1
          for (int j0 = j_begin; j0 < j_end; j0 += 32) {
            uint32_t bits = poison_of(poison, j0);
            if (bits != 0u) bits &= tree_sees32(a, b, tok, j0, dep);
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

// 5-D map over rows [batch, heads, n] of d elements: (64 columns, row, 64-column block, head,
// batch).  A box {64, rows, blocks, 1, 1} lands as `blocks` 128-byte-swizzled [rows x 64]
// blocks; rows behind n and blocks behind d / 64 read as zeros.
int tree_encode_rows(CUtensorMap* map, const void* ptr, bool half, int64_t d, int64_t n, int64_t heads, int64_t batch,
                       int64_t s_b, int64_t s_h, int64_t s_n, uint32_t rows, uint32_t blocks) {
  TreeEncodeFn enc = tree_encode_fn();
  if (enc == nullptr) {
    set_error("cuTensorMapEncodeTiled is not available from the driver");
    return W8_ERR_CUDA;
  }
  // A dimension of one element has no stride to speak of: any valid one.
  auto bytes = [&](int64_t size, int64_t stride) { return static_cast<cuuint64_t>(size > 1 ? stride * 2 : d * 2); };
  const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(d / 64),
                              static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(batch)};
  const cuuint64_t strides[4] = {bytes(n, s_n), 128, bytes(heads, s_h), bytes(batch, s_b)};
  const cuuint32_t box[5] = {64, rows, blocks, 1, 1};
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                         const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled (cache attention) failed with CUresult %d", static_cast<int>(r));
    return W8_ERR_CUDA;
  }
  return W8_OK;
}

// 5-D map over q: (64 columns, head, token, 64-column block, batch).  A box {64, group,
// 128 / group, blocks, 1} lands as `blocks` swizzled blocks of 128 rows i * group + g, zeros
// behind the d / 64-th.
static int encode_q(CUtensorMap* map, const w8::TreeArgs& a, bool half, int64_t d, uint32_t blocks) {
  TreeEncodeFn enc = tree_encode_fn();
  if (enc == nullptr) {
    set_error("cuTensorMapEncodeTiled is not available from the driver");
    return W8_ERR_CUDA;
  }
  const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
  auto bytes = [&](int64_t size, int64_t stride) { return static_cast<cuuint64_t>(size > 1 ? stride * 2 : d * 2); };
  const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(a.n),
                              static_cast<cuuint64_t>(d / 64), static_cast<cuuint64_t>(a.batch)};
  const cuuint64_t strides[4] = {bytes(heads, a.q_h), bytes(a.n, a.q_t), 128, bytes(a.batch, a.q_b)};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(w8::kTtBM / a.group),
                             blocks, 1};
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                         const_cast<uint16_t*>(a.q), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled (cache attention, q) failed with CUresult %d", static_cast<int>(r));
    return W8_ERR_CUDA;
  }
  return W8_OK;
}

template <typename T, int D, int DR = D>
static int tree_tc_go(const w8::TreeArgs& a, int64_t items, int device, cudaStream_t stream) {
  using C = w8::TtCfg<D>;
  constexpr bool kHalf = __is_same(T, __half);
  CUtensorMap tq, tk, tv, tkn, tvn;
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
  tq = tkn;
  if (a.q_tma) {
    st = encode_q(&tq, a, kHalf, DR, D / 64);
    if (st != W8_OK) return st;
  }
  static bool done[64] = {};
  if (!done[device]) {
    W8_CUDA_TRY(cudaFuncSetAttribute(w8::attn_tree_tc_kernel<T, D, DR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     C::kSmem));
    done[device] = true;
  }
  const int64_t blocks = 2 * items * a.splits * C::kSplitD;
  W8_CHECK_ARG(blocks < (1ll << 31), "too many row tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(w8::kTtThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, w8::attn_tree_tc_kernel<T, D, DR>, tq, tk, tv, tkn, tvn, a));
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
