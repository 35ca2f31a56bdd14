// Attention of new tokens (one, a chunk or a drafted tree) over a paged 8-bit cache: the
// contract of attention_tree.cu, with the committed keys and values where a serving cache keeps
// them.  The reference attends to 16-bit keys that it concatenates (pipeline.py:133-180,
// local_attn.py:44-83).
//
// Per sequence b and cache head c, R = G N query rows share the keys
//   k_j = ks[page, c] k8_j,  v_j = vs[page, c] v8_j   (full pages, signed 8 bits)
// then the 16-bit rows of the partial page and of the new tokens:
//   x_rj = scale q_r . k_j,   p = softmax over the keys row r may see,   o_r = sum_j p_rj v_j
//
// Decode reads each key once for few rows and is bound by HBM, at half the bytes of a 16-bit
// cache, so the unpacking has to keep up with 23 values a clock and SM.  Both products run as
// fp16 mma.sync with fp32 sums, the cache as the 16-row operand and the query rows as the 8
// columns: S^T = K Q^T, O^T = V^T P^T.  (The other way round few rows would fill half of the 16
// and twice the instructions would be issued for them: 136 us where this took 91.)  ldmatrix
// brings 8-bit rows as pairs of bytes, of which a thread makes fp16 pairs without a conversion: V
// exactly (paged_unpack), K as 1152 + k8 (paged_raise, an instruction less a pair), whose 1152 times
// the sum of the row's q the scores start from with the opposite sign.  The order of the reduction
// is permuted alike on both sides, in Q when it is staged and in O's columns, which `natural` puts
// back for the 16-bit tiles and the result.  P^T is the second product's operand after movmatrix.
// Q is scaled by a power of two a row into fp16's range (largest element 2^14: what falls below
// 2^-24 is 2^-38 of that).  ks multiplies the scores; vs goes into P relative to a power of two not
// below any vs so far (paged_unit), in which unit O is held: O is rescaled when that grows or a
// row's maximum does, and P is rounded to fp16, half a step of 2^-11 on each weight (TreeRef has
// the range).
//
// The schedule is attention_tree.cu's: all tiles of all sequences dealt in equal contiguous
// ranges to the CTAs, each of 8 warps 16 or (D <= 128: 91 -> 72 us) 32 keys at a time with a running
// softmax of its own, joined at the end of an item; pieces joined by attn_tree_combine_kernel.  A ninth warp walks the page
// table ahead, a page a lane: TMA boxes of a page's rows into the ring, and its scales.  Pages
// that no row sees are not read (nor their table entries followed), so a window's old pages may
// be gone.
//
// 32 sequences of 2000 to 8191 tokens, 8 cache heads of 128, 4 query heads each: 70 us, 74% of what a
// copy moves, of which reading alone takes 62; what is left is the unpacking (some 9 instructions
// for 4 values and both products) that no longer hides behind the loads.  One sequence of one
// token is a chain (table, page, join, combine): 15 us for 3658 keys of 512.
#include "attention_paged.cuh"
#include "attn_mma.cuh"
#include "attn_tc.cuh"

#include <algorithm>

namespace w8 {

template <int D, int NT>
struct PagedCfg {
  static constexpr int kBM = 8 * NT;
  static constexpr int kWarps = 8;                         // working; a ninth loads
  static constexpr int kThreads = 32 * (kWarps + 1);
  static constexpr int kKT = D <= 128 ? 2 : 1;             // 16-key tiles of a warp's step
  static constexpr int kTeams = D == 512 ? 2 : 1;          // sets of warps that take the tiles in turn
  static constexpr int kGroups = kWarps / kTeams;          // warps of a tile
  static constexpr int kBN = kGroups * kKT * 16;           // keys of a tile of pages: 256, 256, 128, 64
  static constexpr int kBN16 = kBN / 2;                    // of a 16-bit tile, which is as large
  static constexpr int kSlotBytes = kBN * D;               // 16 KB (D = 64) or 32 KB
  // Columns of the outputs joined at a time, and the ring beside them.
  static constexpr int kJoin = NT == 2 ? 64 : D < 256 ? D : 256;
  static constexpr int kSlots = (D < 256 || NT == 2 ? 163840 : 131072) / kSlotBytes;  // 10, 5 or 4
  static constexpr int kPitch = kJoin + 4;                 // their fp32 row pitch
  static constexpr int kOffQ8 = kSlots * kSlotBytes;       // Q as fp16, scaled and permuted
  static constexpr int kOffQ16 = kOffQ8 + kBM * D * 2;     // Q as it is
  static constexpr int kOffJoin = kOffQ16 + kBM * D * 2;   // float [kWarps][kBM][kPitch]
  static constexpr int kOffStat = kOffJoin + kWarps * kBM * kPitch * 4;  // float [2][kWarps][kBM]: maxima, sums
  static constexpr int kOffRow = kOffStat + 2 * kWarps * kBM * 4;  // int4 [kBM]: token, depth, first key, Q's scale taken back
  static constexpr int kOffSum = kOffRow + kBM * 16;       // float [kBM]: -1152 times the sum of Q as fp16
  static constexpr int kOffScale = kOffSum + (kBM * 4 + 15) / 16 * 16;     // float [kSlots][kPagedMaxBoxes]
  static constexpr int kOffMask = kOffScale + kSlots * kPagedMaxBoxes * 4;  // uint32 [kSlots]: boxes that are there
  static constexpr int kOffBar = kOffMask + (kSlots * 4 + 15) / 16 * 16;
  static constexpr int kNumBars = 2 * kSlots;              // full, empty
  static constexpr int kSmem = kOffBar + kNumBars * 8 + 16 + 1024;
  static_assert(kSmem <= 232448, "shared memory budget exceeded");
  static_assert(kOffBar % 16 == 0 && kOffScale % 16 == 0 && kOffRow % 16 == 0, "alignment");
};

__device__ __forceinline__ float paged_ks(const PagedArgs& a, int page, int c) { return a.ks[page * a.ks_p + c * a.ks_h]; }
__device__ __forceinline__ float paged_vs(const PagedArgs& a, int page, int c) { return a.vs[page * a.vs_p + c * a.vs_h]; }

// 8 x 8 values of 16 bits across a warp, transposed: from a thread's (row lane / 4, columns 2 (lane % 4)
// and the next) to its (column lane / 4, rows 2 (lane % 4) and the next).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(PagedCfg<D, NT>::kThreads, 1)
    attn_paged_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ CUtensorMap tm_kt, const __grid_constant__ CUtensorMap tm_vt,
                      const __grid_constant__ CUtensorMap tm_kn, const __grid_constant__ CUtensorMap tm_vn,
                      const __grid_constant__ PagedArgs pa) {
  using C = PagedCfg<D, NT>;
  using H = __half;
  constexpr int BM = C::kBM, BN = C::kBN, BN16 = C::kBN16, NS = C::kSlots, CH = D / 8;  // CH: 16-byte chunks of a 16-bit row
  constexpr bool kQRegs = NT * D <= 128;             // Q's fragments stay in registers
  constexpr int kRowBytes = D < 128 ? D : 128;       // of a box's row in shared memory
  const TreeArgs& a = pa.t;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t sq8 = base + C::kOffQ8, sq16 = base + C::kOffQ16, bar0 = base + C::kOffBar;
  float* joint = reinterpret_cast<float*>(smem + C::kOffJoin);
  float* stat = reinterpret_cast<float*>(smem + C::kOffStat);
  int4* row_info = reinterpret_cast<int4*>(smem + C::kOffRow);
  float* row_sum = reinterpret_cast<float*>(smem + C::kOffSum);
  volatile float* scales = reinterpret_cast<volatile float*>(smem + C::kOffScale);
  volatile uint32_t* masks = reinterpret_cast<volatile uint32_t*>(smem + C::kOffMask);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffBar + C::kNumBars * 8);
  auto full_bar = [&](uint32_t s) { return bar0 + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar0 + 8u * (NS + s); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = a.group * a.n;
  const int box_shift = min(pa.shift, 31 - __clz(BN)), box = 1 << box_shift;  // keys of a box
  const int boxes = BN >> box_shift;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full_bar(s), 1);  // the producer's arrive.expect_tx
      mbar_init(empty_bar(s), C::kWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    prefetch_tmap(&tm_kt);
    prefetch_tmap(&tm_vt);
    prefetch_tmap(&tm_kn);
    prefetch_tmap(&tm_vn);
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
  PagedSpan span;
  long long pos = 0, stop = 0, item_pos = 0;  // item_pos: first tile of the current item
  TreeDeal deal = {1, 0};
  if (a.direct || pairs == 1) {
    // One item (this CTA's number's), or those of one pair.
    int p = 0;
    if (a.direct) {
      p = static_cast<int>(blockIdx.x);
      if (a.kv_heads > 1) p = blockIdx.x / a.kv_heads, c = blockIdx.x - p * a.kv_heads;
    }
    split_pair(p, b, rt);
    len = tree_len(a, b);
    span = paged_span<BM, BN, BN16>(pa, len, rt);
    const int tiles = span.tiles();
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
      return paged_span<BM, BN, BN16>(pa, tree_len(a, pb), prt).tiles();
    };
    long long* sched = reinterpret_cast<long long*>(joint);  // (not in use yet)
    long long sum = 0, round;
    for (int p = tid; p < pairs; p += C::kThreads) sum += pair_tiles(p);
    long long excl = block_scan<C::kWarps + 1>(sum, sched, round);  // (of few pairs also each one's place)
    const long long total = round * a.kv_heads;
    const uint32_t ctas = total < gridDim.x ? static_cast<uint32_t>(total) : gridDim.x;
    if (blockIdx.x >= ctas) return;
    deal.each = div_short(total, ctas);
    deal.more = total - deal.each * ctas;
    pos = deal_begin(deal, blockIdx.x);
    stop = deal_begin(deal, blockIdx.x + 1);
    // The pair that holds `pos`: a running sum over rounds of pairs.
    long long before = 0;
    for (int p0 = 0;; p0 += C::kThreads) {
      const int p = p0 + tid;
      long long nt = sum;
      if (pairs > C::kThreads) {
        nt = p < pairs ? pair_tiles(p) : 0;
        excl = before + block_scan<C::kWarps + 1>(nt, sched, round);
      }
      if (nt > 0 && excl * a.kv_heads <= pos && pos < (excl + nt) * a.kv_heads) {
        sched[32] = p;
        sched[33] = excl * a.kv_heads;
      }
      __syncthreads();
      before += round;
      if (pos < before * a.kv_heads) break;  // (every pair has tiles, and pos < total)
      if (p0 + C::kThreads >= pairs) return;  // only if the lengths changed under the call
    }
    split_pair(static_cast<int>(sched[32]), b, rt);
    item_pos = sched[33];
    len = tree_len(a, b);
    span = paged_span<BM, BN, BN16>(pa, len, rt);
    const int tiles = span.tiles();
    c = static_cast<int>(div_short(pos - item_pos, tiles));
    item_pos += static_cast<long long>(c) * tiles;
    __syncthreads();
  }
  int nt = span.tiles();
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
      span = paged_span<BM, BN, BN16>(pa, len, rt);
      nt = span.tiles();
    }
  };
  // Tile t of the item: its first key (of its kind).
  enum : int { kPages = 0, kTail = 1, kNew = 2 };
  auto kind_of = [&](int t) { return t < span.pages() ? kPages : t < span.pages() + span.tail ? kTail : kNew; };
  auto key0_of = [&](int t) {
    if (t < span.ns) return t * BN;
    if (t < span.pages()) return (span.c0 + t - span.ns) * BN;
    t -= span.pages();
    return (t < span.tail ? t : t - span.tail) * BN16;
  };

  uint32_t g = 0;  // ring steps so far (each tile's K, then V)
  bool ok = true;
  __syncwarp();
  if (warp >= C::kWarps) {
    // ---- the producer: each tile's K and V boxes into the ring as its slots are left, the table
    // entries and scales of the next tile under way meanwhile.
    while (ok) {
      const int t0 = static_cast<int>(pos - item_pos);
      const int t1 = static_cast<int>(stop - item_pos < nt ? stop - item_pos : nt);
      const int* table = pa.table + b * pa.table_b;
      // Lane j's box of tile t: the table's entry if some row needs it, or -1; the page it names; its
      // scales.  Each is asked for a tile before the next needs it.
      auto entry_of = [&](int t) {
        if (t >= t1 || kind_of(t) != kPages || lane >= boxes) return -1;
        const int k0 = key0_of(t) + (lane << box_shift);
        if (!paged_needs(pa, span, k0, k0 + box)) return -1;
        const int p = table[k0 >> pa.shift];
        return p < 0 ? INT32_MAX : p;
      };
      struct Page {
        int at;
        float ks, vs;
      };
      auto page_of = [&](int entry) {
        Page p = {entry, 0.f, 0.f};
        if (entry >= pa.pages) {
          atomicExch(&g_tree_status, W8_ERR_INVALID_ARG);
          p.at = -1;
        }
        if (p.at >= 0) p.ks = paged_ks(pa, p.at, c), p.vs = paged_vs(pa, p.at, c);
        return p;
      };
      int entry = entry_of(t0), entry1 = entry_of(t0 + 1);
      Page page = page_of(entry), next = page_of(entry1);
      entry = entry_of(t0 + 2);
      for (int t = t0; t < t1 && ok; ++t) {
        const int kind = kind_of(t), key0 = key0_of(t);
        const Page after = page_of(entry);
        entry = entry_of(t + 3);
        const uint32_t there = __ballot_sync(0xffffffffu, page.at >= 0);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++g) {
          const uint32_t slot = g % NS, dst = base + slot * C::kSlotBytes;
          ok = ok && mbar_wait_bounded(empty_bar(slot), ((g / NS) & 1u) ^ 1u, abort_flag, &g_tree_status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (kind == kPages) {
            // The copies first: the scales, which the barrier's one arrival follows, are yet to come.
            if (page.at >= 0)
              tma_load_5d(dst + lane * (box * D), kv ? &tm_v : &tm_k, full_bar(slot), 0,
                          (key0 + (lane << box_shift)) & ((1 << pa.shift) - 1), 0, c, page.at);
            if (kv == 0) continue;
            const uint32_t before = (g - 1) % NS;  // (K's slot: its arrival waits for the same loads)
            if (lane < boxes) scales[before * kPagedMaxBoxes + lane] = page.ks, scales[slot * kPagedMaxBoxes + lane] = page.vs;
            if (lane == 0) masks[before] = there;
            __syncwarp();
            if (lane == 0) {
              mbar_arrive_expect_tx(full_bar(before), __popc(there) * (box * D));
              mbar_arrive_expect_tx(full_bar(slot), __popc(there) * (box * D));
            }
          } else if (lane == 0) {
            mbar_arrive_expect_tx(full_bar(slot), C::kSlotBytes);
            const CUtensorMap* map = kind == kTail ? (kv ? &tm_vt : &tm_kt) : (kv ? &tm_vn : &tm_kn);
            tma_load_5d(dst, map, full_bar(slot), 0, key0, 0, c, b);
          }
          __syncwarp();
        }
        page = next, next = after;
      }
      pos += t1 - t0;
      if (pos >= stop) break;
      advance();
    }
    if (!ok) {
      // A wait gave up: let the copies in flight land before the CTA exits.
      const unsigned long long since = globaltimer();
      while (globaltimer() - since < 50000ull) {
      }
    }
    return;
  }
  auto rows_sync = [&]() {  // of the 8 warps without the producer
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(32 * C::kWarps) : "memory");
  };
  auto rows_sync_and = [&](bool on) {
    uint32_t all;
    __syncwarp();
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "bar.red.and.pred p, 1, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(all)
        : "r"(on ? 1u : 0u), "n"(32 * C::kWarps)
        : "memory");
    return all != 0u;
  };
  const int team = warp / C::kGroups, grp = warp % C::kGroups;  // 16-key group of a step
  const int gl = lane >> 2, tl = lane & 3;  // a thread's keys (or columns) gl, gl + 8 and rows 2 tl, 2 tl + 1
  while (true) {
    const int row0 = rt * BM, bc = b * a.kv_heads + c;
    const int t0 = static_cast<int>(pos - item_pos);
    const int t1 = static_cast<int>(stop - item_pos < nt ? stop - item_pos : nt);
    const bool whole = t0 == 0 && t1 == nt;
    const int64_t part_row = (2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0 ? 1 : 0)) * BM;
    const int sink_left = a.sink - len;
    if (t0 == 0 && tid == 0 && !a.direct) {
      // The CTA that begins an item says where its pieces are: one in each CTA up to its last tile's.
      const int last = deal_owner(deal, item_pos + nt - 1);
      a.info[bc * a.row_tiles + rt] = make_int2(blockIdx.x, last - static_cast<int>(blockIdx.x) + 1);
    }
    // Q rows r = i * group + g (query head c * group + g of new token i), a row a warp: as they
    // are, and scaled into fp16's range with 16 columns at a time in the order in which a thread's 4
    // bytes of K come: columns 4 t .. 4 t + 3 as elements 2 t, 2 t + 1, 2 t + 8, 2 t + 9.
    for (int r = warp; r < BM; r += C::kWarps) {
      float most = 0.f, sum = 0.f;
      uint4 w[(CH + 31) / 32];
      int i = -1, gq = 0, dep = 0, first = INT32_MAX;  // (no row: sees nothing)
      if (row0 + r < rows) {
        tree_row(a, row0 + r, i, gq);
        dep = tree_depth(a, b, i);
        first = tree_first(a, len, dep);
      }
#pragma unroll
      for (int x = 0; x < (CH + 31) / 32; ++x) {
        const int ch = lane + 32 * x;
        w[x] = make_uint4(0, 0, 0, 0);
        if (ch < CH && i >= 0)
          w[x] = *reinterpret_cast<const uint4*>(a.q + b * a.q_b + (static_cast<int64_t>(c) * a.group + gq) * a.q_h +
                                                 i * a.q_t + ch * 8);
        const uint32_t ws[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          most = fmaxf(most, fmaxf(fabsf(tree_f32<T>(ws[e] & 0xFFFFu)), fabsf(tree_f32<T>(ws[e] >> 16))));
        if (ch < CH) st_shared_v4(sq16 + r * (D * 2) + ((ch ^ (r & 7)) << 4), w[x].x, w[x].y, w[x].z, w[x].w);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
      // 2^(14 - exponent), at most 2^100; 1 for a row of zeros or infinities.
      const int ex = static_cast<int>(__float_as_uint(most) >> 23);
      const int up = ex == 0 || ex == 255 ? 0 : min(14 + 127 - ex, 100);
      const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
#pragma unroll
      for (int x = 0; x < (CH + 31) / 32; ++x) {
        const int ch = lane + 32 * x;
        if (ch >= CH) break;
        const uint32_t ws[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h[e] = pack2<H>(tree_f32<T>(ws[e] & 0xFFFFu) * f, tree_f32<T>(ws[e] >> 16) * f);
          sum += tree_f32<H>(h[e] & 0xFFFFu) + tree_f32<H>(h[e] >> 16);
        }
        uint8_t* row = smem + C::kOffQ8 + r * (D * 2) + 8 * (ch & 1);
        *reinterpret_cast<uint2*>(row + (((ch & ~1) ^ (r & 7)) << 4)) = make_uint2(h[0], h[2]);
        *reinterpret_cast<uint2*>(row + (((ch | 1) ^ (r & 7)) << 4)) = make_uint2(h[1], h[3]);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == 0) {
        row_info[r] = make_int4(i, dep, first, (127 - up) << 23);
        row_sum[r] = -1152.f * sum;
      }
    }
    rows_sync();
    // A row's reference: no maximum yet is kNone, which every score exceeds.
    constexpr float kNone = -3e38f;
    float m[NT][2], l[NT][2], fac[NT][2];
    float o[NT][D / 16][4];  // O transposed: columns gl and gl + 8 of 16 (or 2 gl and 2 gl + 1), rows 2 tl, 2 tl + 1
    float qsum[NT][2];
    int last_first = 0;      // the latest first key of the item's rows
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int4 info = row_info[8 * n + 2 * tl + h];
        m[n][h] = kNone, l[n][h] = 0.f;
        fac[n][h] = __int_as_float(info.w) * a.scale_log2;
        qsum[n][h] = row_sum[8 * n + 2 * tl + h];
        if (info.x >= 0) last_first = max(last_first, info.z);
      }
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][k][e] = 0.f;
    }
    last_first = __reduce_max_sync(0xffffffffu, last_first);
    // Q^T as the B operand, two steps of the reduction (32 columns) at a time.
    auto load_q = [&](uint32_t sq, int n, int k2, uint32_t (&q)[4]) {
      const int r = 8 * n + (lane & 7);
      ldsm_x4(sq + r * (D * 2) + (((4 * k2 + (lane >> 3)) ^ (r & 7)) << 4), q);
    };
    uint32_t qf[kQRegs ? NT : 1][kQRegs ? D / 32 : 1][4];
    if constexpr (kQRegs) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k2 = 0; k2 < D / 32; ++k2) load_q(sq8, n, k2, qf[n][k2]);
    }
    // Whether row 8 n + 2 tl + h sees committed positions p0 + gl and p0 + gl + 8 (below `end`), as bits 0 and 1.
    auto sees = [&](int n, int h, int p0, int end) {
      const int4 info = row_info[8 * n + 2 * tl + h];
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int p = p0 + gl + 8 * e;
        if (p < end && (p >= info.z || (p < a.sink && info.x >= 0))) bits |= 1u << e;
      }
      return bits;
    };
    // m moved where a row's maximum of the step (of this thread's keys: mx) asks for it; O and l with it,
    // O by `unit` (the change of its unit) besides.
    auto move_rows = [&](const float (&mx)[NT][2], float unit) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x = mx[n][h];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const bool mv = x > m[n][h] + TreeRef<H>::kSlack;
          const float to = x - TreeRef<H>::kBelow;
          const float corr = mv ? ex2_tree(m[n][h] - to) : 1.f;
          if (mv) m[n][h] = to;
          l[n][h] *= corr;
          const float f = corr * unit;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            o[n][k][h] *= f;
            o[n][k][2 + h] *= f;
          }
        }
    };
    float unit = __uint_as_float(0x00800000u);  // of O: the smallest, which the smallest scales have too
    bool permuted = false;                      // O holds pages' products: in `unit` and their columns' order
    // O in order and in units of 1: of each 16 columns a thread holds 2 gl and 2 gl + 1 (the even and
    // odd bytes of V's rows) and gets gl and gl + 8.
    auto natural = [&]() {
      permuted = false;
      const int s0 = ((gl >> 1) << 2) | tl, s1 = s0 + 16;
      const bool odd = gl & 1;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float v0 = o[n][k][h] * unit, v1 = o[n][k][2 + h] * unit;
            const float a0 = __shfl_sync(0xffffffffu, v0, s0), a1 = __shfl_sync(0xffffffffu, v1, s0);
            const float b0 = __shfl_sync(0xffffffffu, v0, s1), b1 = __shfl_sync(0xffffffffu, v1, s1);
            o[n][k][h] = odd ? a1 : a0;
            o[n][k][2 + h] = odd ? b1 : b0;
          }
    };

#pragma unroll 1
    for (int t = t0; t < t1; ++t, g += 2) {
      const uint32_t slot_k = g % NS, slot_v = (g + 1) % NS;
      if (ok) ok = mbar_wait_bounded(full_bar(slot_k), (g / NS) & 1u, abort_flag, &g_tree_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (C::kTeams > 1 && ((t - t0) & (C::kTeams - 1)) != team) {
        // Another team's tile (waited for all the same: a barrier's phase must not pass unseen).
        ok = mbar_wait_bounded(full_bar(slot_v), ((g + 1) / NS) & 1u, abort_flag, &g_tree_status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive(empty_bar(slot_k));
          mbar_arrive(empty_bar(slot_v));
        }
        __syncwarp();
        continue;
      }
      const int kind = kind_of(t), tile0 = key0_of(t);
      const uint32_t sk = base + slot_k * C::kSlotBytes, sv = base + slot_v * C::kSlotBytes;
      if (kind == kPages) {
        permuted = true;
        const int kr = grp * (C::kKT * 16), key0 = tile0 + kr;  // this step's keys
        // Rows of 16 bytes that a lane names for ldmatrix: 8 keys, the next 8, and the next 16 columns of
        // both.  A row's chunks are swizzled, a matter of one XOR as a row begins on 128 (64) bytes.
        uint32_t off[C::kKT];  // in the slot, of chunk lane / 16
        int bx[C::kKT];        // the 16 keys' box
#pragma unroll
        for (int kt = 0; kt < C::kKT; ++kt) {
          bx[kt] = (kr + 16 * kt) >> box_shift;
          const int lrow = ((kr + 16 * kt) & (box - 1)) + (lane & 15);
          off[kt] = bx[kt] * (box * D) + lrow * kRowBytes + (((lane >> 4) ^ (D >= 128 ? lrow & 7 : (lrow >> 1) & 3)) << 4);
        }
        auto chunks = [&](uint32_t slot, int kt, int c2) {  // chunks 2 c2 and 2 c2 + 1
          return slot + (D > 128 ? (c2 >> 2) * (box * 128) : 0) + (off[kt] ^ ((c2 & 3) << 5));
        };
        // ---- S^T = K Q^T.  The 8-bit values go in as 1024 + 128 + k8, exact in fp16, and the sums start
        // from -1152 times Q's: the products cancel to S with what fp32 sums lose at their size, about
        // 2^-23 of 1152 |sum q| against a score's 30 |q| sqrt(D): 10^-5 of it where q's elements cancel in their
        // sum, sqrt(D) times that where they are of one sign (fp16, q 4 and 30 deviations
        // off 0: outputs are off by up to 0.8 half steps at D 256 and 1.7 at 512, by 0.4 for q around 0; their
        // errors' norm grows by a third at D 256 and hardly at 512).
        float s[C::kKT][NT][4];
#pragma unroll
        for (int kt = 0; kt < C::kKT; ++kt)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[kt][n][e] = qsum[n][e & 1];
#pragma unroll
        for (int k2 = 0; k2 < D / 32; ++k2) {
          uint32_t x0[C::kKT][4], x1[C::kKT][4];
#pragma unroll
          for (int kt = 0; kt < C::kKT; ++kt) {
            uint32_t kb[4];
            ldsm_x4(chunks(sk, kt, k2), kb);
            paged_raise(kb[0], 0x4140u, 0x4342u, x0[kt][0], x0[kt][2]);
            paged_raise(kb[1], 0x4140u, 0x4342u, x0[kt][1], x0[kt][3]);
            paged_raise(kb[2], 0x4140u, 0x4342u, x1[kt][0], x1[kt][2]);
            paged_raise(kb[3], 0x4140u, 0x4342u, x1[kt][1], x1[kt][3]);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t q[4];
            if constexpr (kQRegs) {
#pragma unroll
              for (int e = 0; e < 4; ++e) q[e] = qf[n][k2][e];
            } else {
              load_q(sq8, n, k2, q);
            }
#pragma unroll
            for (int kt = 0; kt < C::kKT; ++kt) {
              mma16816<H>(s[kt][n], x0[kt], q[0], q[1]);
              mma16816<H>(s[kt][n], x1[kt], q[2], q[3]);
            }
          }
        }
        const uint32_t there = masks[slot_k];
        float ks[C::kKT];
        bool on[C::kKT], plain = true;  // plain: all rows see all keys
#pragma unroll
        for (int kt = 0; kt < C::kKT; ++kt) {
          ks[kt] = scales[slot_k * kPagedMaxBoxes + bx[kt]];
          on[kt] = (there >> bx[kt]) & 1u;
          plain = plain && on[kt];
        }
        plain = plain && key0 + 16 * C::kKT <= span.full && key0 >= last_first;
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar(slot_k));
        // ---- scores in log2 units, less m; masks
        float y[C::kKT][NT][4], most = -INFINITY;
        uint32_t hidden = 0u;  // bit (kt NT + n) 4 + e: the row does not see the key
        auto score = [&]() {
#pragma unroll
          for (int kt = 0; kt < C::kKT; ++kt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) y[kt][n][e] = fmaf(s[kt][n][e], fac[n][e & 1] * ks[kt], -m[n][e & 1]);
          if (!plain) {
#pragma unroll
            for (int kt = 0; kt < C::kKT; ++kt)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if ((hidden >> ((kt * NT + n) * 4 + e)) & 1u) y[kt][n][e] = -INFINITY;
          }
        };
        if (!plain) {
#pragma unroll
          for (int kt = 0; kt < C::kKT; ++kt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t keep = on[kt] ? sees(n, h, key0 + 16 * kt, span.full) : 0u;
                hidden |= (~keep & 1u) << ((kt * NT + n) * 4 + h) | ((~keep >> 1) & 1u) << ((kt * NT + n) * 4 + 2 + h);
              }
        }
        score();
#pragma unroll
        for (int kt = 0; kt < C::kKT; ++kt)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = fmaxf(most, y[kt][n][e]);
        ok = mbar_wait_bounded(full_bar(slot_v), ((g + 1) / NS) & 1u, abort_flag, &g_tree_status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        float vs[C::kKT], need = unit;
#pragma unroll
        for (int kt = 0; kt < C::kKT; ++kt) {
          vs[kt] = on[kt] ? scales[slot_v * kPagedMaxBoxes + bx[kt]] : 0.f;
          need = fmaxf(need, paged_unit(vs[kt]));
        }
        if (__any_sync(0xffffffffu, most > TreeRef<H>::kSlack) || need > unit) {
          float mx[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              mx[n][h] = -INFINITY;
#pragma unroll
              for (int kt = 0; kt < C::kKT; ++kt)
#pragma unroll
                for (int e = h; e < 4; e += 2)
                  if (!((hidden >> ((kt * NT + n) * 4 + e)) & 1u))
                    mx[n][h] = fmaxf(mx[n][h], s[kt][n][e] * (fac[n][h] * ks[kt]));
            }
          move_rows(mx, unit * paged_unit_rcp(need));
          unit = need;
          score();
        }
        // ---- weights, and P in O's unit
        uint32_t pw[C::kKT][NT][2];
#pragma unroll
        for (int kt = 0; kt < C::kKT; ++kt) {
          const float vr = vs[kt] * paged_unit_rcp(unit);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] = ex2_tree(y[kt][n][e]);
            l[n][0] += p[0] + p[2];
            l[n][1] += p[1] + p[3];
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] *= vr;
            if (vr != vr) {  // (a NaN scale is for the rows that see the page)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((hidden >> ((kt * NT + n) * 4 + e)) & 1u) p[e] = 0.f;
            }
            pw[kt][n][0] = transpose8x8(pack2<H>(p[0], p[1]));
            pw[kt][n][1] = transpose8x8(pack2<H>(p[2], p[3]));
          }
        }
        // ---- O^T += V^T P^T: of 16 bytes of a row of V the even columns are 8 rows of the operand, the
        // odd ones the others.
#pragma unroll
        for (int c2 = 0; c2 < D / 32; ++c2)
#pragma unroll
          for (int kt = 0; kt < C::kKT; ++kt) {
            uint32_t vb[4], x0[4], x1[4];
            ldsm_x4_t(chunks(sv, kt, c2), vb);
            paged_unpack<H>(vb[0], 0x4240u, 0x4341u, x0[0], x0[1]);
            paged_unpack<H>(vb[1], 0x4240u, 0x4341u, x0[2], x0[3]);
            paged_unpack<H>(vb[2], 0x4240u, 0x4341u, x1[0], x1[1]);
            paged_unpack<H>(vb[3], 0x4240u, 0x4341u, x1[2], x1[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma16816<H>(o[n][2 * c2], x0, pw[kt][n][0], pw[kt][n][1]);
              mma16816<H>(o[n][2 * c2 + 1], x1, pw[kt][n][0], pw[kt][n][1]);
            }
          }
      } else {
        if (permuted) natural();
        const bool fresh = kind == kNew;
        const int kr = grp * 16, key0 = tile0 + kr;  // this step's keys (rows of the tail, or new tokens)
        const int end = fresh ? a.n : len - span.full;
        const bool work = kr < BN16 && key0 < end;   // (the same for the whole warp)
        const int lrow = kr + (lane & 15);
        auto chunk = [&](int ch) { return lrow * 128 + (ch >> 3) * (BN16 * 128) + (((ch & 7) ^ (lrow & 7)) << 4); };
        uint32_t pw[NT][2];
        if (work) {
          float s[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
          for (int k2 = 0; k2 < D / 32; ++k2) {
            uint32_t x0[4], x1[4];
            ldsm_x4(sk + chunk(4 * k2 + (lane >> 4)), x0);
            ldsm_x4(sk + chunk(4 * k2 + 2 + (lane >> 4)), x1);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint32_t q[4];
              load_q(sq16, n, k2, q);
              mma16816<T>(s[n], x0, q[0], q[1]);
              mma16816<T>(s[n], x1, q[2], q[3]);
            }
          }
          float mx[NT][2], most = -INFINITY;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // (all lanes: the new tokens' depths are read by the warp)
              uint32_t keep;
              if (fresh) {
                const int4 info = row_info[8 * n + 2 * tl + h];
                const uint32_t bits = tree_sees16(a, b, info.x, key0, info.y, sink_left);
                keep = ((bits >> gl) & 1u) | ((bits >> (gl + 7)) & 2u);
              } else {
                keep = sees(n, h, span.full + key0, len);
              }
              s[n][h] = keep & 1u ? s[n][h] * a.scale_log2 : -INFINITY;
              s[n][2 + h] = keep & 2u ? s[n][2 + h] * a.scale_log2 : -INFINITY;
              mx[n][h] = fmaxf(s[n][h], s[n][2 + h]);
              most = fmaxf(most, mx[n][h] - m[n][h]);
            }
          if (__any_sync(0xffffffffu, most > TreeRef<H>::kSlack)) move_rows(mx, 1.f);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] = ex2_tree(s[n][e] - m[n][e & 1]);
            l[n][0] += p[0] + p[2];
            l[n][1] += p[1] + p[3];
            pw[n][0] = transpose8x8(pack2<T>(p[0], p[1]));
            pw[n][1] = transpose8x8(pack2<T>(p[2], p[3]));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar(slot_k));
        ok = mbar_wait_bounded(full_bar(slot_v), ((g + 1) / NS) & 1u, abort_flag, &g_tree_status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (work) {
          // Rows behind the length or before the window may hold anything and 0 * NaN is NaN: zeros.
          // So may a new token's values where some row must not see them: cleared here, added below
          // to the rows that do.
          uint32_t bad = 0;  // keys of this step whose values are not all finite (new tokens only)
          // (New rows behind the last are zeros already: the box ends there.)
          if (fresh || key0 + 16 > end || span.full + key0 < span.low) {
            const int r0 = !fresh && span.full + key0 >= span.low ? end - key0 : 0;  // rows [r0, r1) are looked at
            const int r1 = fresh ? min(end - key0, 16) : 16;
            for (int e = lane; e < (r1 - r0) * CH; e += 32) {
              const int r = r0 + e / CH, ch = e % CH, p = span.full + key0 + r;
              uint4* w = reinterpret_cast<uint4*>(smem + (sv - base) + (ch >> 3) * (BN16 * 128) + (kr + r) * 128 +
                                                  (((ch & 7) ^ ((kr + r) & 7)) << 4));
              if (!fresh) {
                if (key0 + r >= end || (p < span.low && p >= a.sink)) *w = make_uint4(0, 0, 0, 0);
              } else {
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
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            // (transposed 8 x 8 blocks: columns 0-7 and 8-15 of keys 0-7, then of keys 8-15)
            uint32_t x[4], y[4];
            ldsm_x4_t(sv + chunk(2 * k + (lane >> 4)), y);
            x[0] = y[0], x[1] = y[2], x[2] = y[1], x[3] = y[3];
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<T>(o[n][k], x, pw[n][0], pw[n][1]);
          }
          const bool any_bad = bad != 0u;
#pragma unroll 1
          for (; bad != 0u; bad &= bad - 1u) {
            const int j = key0 + __ffs(bad) - 1;
            const uint16_t* vn = a.vn + b * a.vn_b + c * a.vn_h + j * a.vn_t + gl;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int4 info = row_info[8 * n + 2 * tl + h];
                if (info.x < 0 || !tree_sees(a, b, info.x, j, info.y, sink_left)) continue;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const uint16_t v = vn[16 * k + 8 * e];
                    if (tree_nonfinite<T>(v)) o[n][k][2 * e + h] += tree_f32<T>(v);
                  }
              }
          }
          if (any_bad) __syncwarp();  // (the next step's loads are aligned)
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_bar(slot_v));
    }

    // ---- the warps' results joined: M = max m_w, O = sum 2^(m_w - M) O_w, some columns at a time
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], 4);
        l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], 8);
        l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], 16);
        if (gl == 0) {
          const int r = 8 * n + 2 * tl + h;
          stat[warp * BM + r] = m[n][h] == kNone ? -INFINITY : m[n][h];
          stat[(C::kWarps + warp) * BM + r] = l[n][h];
        }
      }
    ok = rows_sync_and(ok);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 8 * n + 2 * tl + h;
        float top = stat[r];
#pragma unroll
        for (int w = 1; w < C::kWarps; ++w) top = fmaxf(top, stat[w * BM + r]);
        // (a warp that saw nothing adds zeros, except what a NaN score made of it)
        const bool none = m[n][h] == kNone && l[n][h] == 0.f;
        fac[n][h] = none ? -1.f : m[n][h] == kNone ? 1.f : ex2_tree(m[n][h] - top);
      }
#pragma unroll
    for (int j = 0; j < D / C::kJoin; ++j) {
      if (j > 0) rows_sync();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float* dst = joint + (warp * BM + 8 * n + 2 * tl + h) * C::kPitch;
          if (permuted) {  // (pages only: columns 2 gl and 2 gl + 1, in O's unit)
            const float f = fac[n][h] * unit;
#pragma unroll
            for (int k = 0; k < C::kJoin / 16; ++k) {
              const float* v = o[n][j * (C::kJoin / 16) + k];
              *reinterpret_cast<float2*>(dst + 16 * k + 2 * gl) =
                  fac[n][h] < 0.f ? make_float2(0.f, 0.f) : make_float2(v[h] * f, v[2 + h] * f);
            }
          } else {
#pragma unroll
            for (int k = 0; k < C::kJoin / 16; ++k) {
              const float* v = o[n][j * (C::kJoin / 16) + k];
              dst[16 * k + gl] = fac[n][h] < 0.f ? 0.f : v[h] * fac[n][h];
              dst[16 * k + gl + 8] = fac[n][h] < 0.f ? 0.f : v[2 + h] * fac[n][h];
            }
          }
        }
      rows_sync();
      if (!ok) continue;
      constexpr int Q4 = C::kJoin / 4;  // float4 columns
      for (int e = tid; e < BM * Q4; e += 32 * C::kWarps) {
        const int r = e / Q4, q4 = e % Q4, col = j * C::kJoin + 4 * q4;
        if (row0 + r >= rows) break;
        float top = stat[r];
#pragma unroll
        for (int w = 1; w < C::kWarps; ++w) top = fmaxf(top, stat[w * BM + r]);
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) {
          const float mw = stat[w * BM + r];
          sum += (mw == -INFINITY ? 1.f : ex2_tree(mw - top)) * stat[(C::kWarps + w) * BM + r];
          const float4 x = *reinterpret_cast<const float4*>(joint + (w * BM + r) * C::kPitch + 4 * q4);
          v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing: zeros
          int i, gq;
          tree_row(a, row0 + r, i, gq);
          uint16_t* dst = a.o + b * a.o_b + (static_cast<int64_t>(c) * a.group + gq) * a.o_h + i * a.o_t + col;
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
        } else {
          *reinterpret_cast<float4*>(a.part_o + (part_row + r) * D + col) = v;
          if (col == 0) a.part_ml[part_row + r] = make_float2(top, sum);
        }
      }
    }
    if (!ok) break;  // (the producer waits for the copies in flight)
    pos += t1 - t0;
    if (pos >= stop) break;
    advance();
    rows_sync();  // Q, the statistics and the joint outputs are free
  }
}

}  // namespace w8

namespace w8host {

int require_sm100(int* device);

int tree_encode_rows(CUtensorMap* map, const void* ptr, bool half, int64_t d, int64_t n, int64_t heads, int64_t batch,
                     int64_t s_b, int64_t s_h, int64_t s_n, uint32_t rows, uint32_t blocks);
int tree_encode(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, const cuuint64_t* dims,
                const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle, const char* what);
int tree_join(const w8::TreeArgs& a, bool half, int64_t d, int bm, cudaStream_t stream);
int paged_tc(const w8_attention_paged_args& x, const w8::PagedArgs& a, bool half, int64_t items, int device,
             cudaStream_t stream);
int tree_tc_device_status(int clear, int* out);

// How a call is cut: rows per tile, row tiles, and over the keys a number of splits (tcgen05) or of
// CTAs that share all tiles, or an item each (mma.sync).
struct PagedPlan {
  bool tc;  // the tcgen05 schedule (attention_tree_tc.cu)
  bool direct;
  int bm, row_tiles, splits, ctas;
  int64_t items;
};

static PagedPlan paged_plan(int64_t batch, int64_t kv_heads, int64_t group, int64_t n, int64_t d, int64_t slots,
                            int64_t window, int64_t sink, int sms) {
  PagedPlan p;
  const int64_t rows = group * n;
  // Up to so many rows a cache head in tiles of 16 (D = 512: 8), more in tiles of 256 on the tensor cores'
  // schedule, whose cost hardly depends on how many of the 256 there are (40 sequences of 1000, 8 heads
  // of 128: 32 rows 90 us against 155, 48 rows 127 against 156, 64 rows 165 against 156; D = 64, 64
  // rows: 118 against 153; D = 256, 24 rows: 234 against 178; D = 512, 24 rows: 394 against 451).
  p.tc = rows > (d == 64 ? 64 : d == 128 ? 48 : d == 256 ? 16 : 24);
  p.bm = p.tc ? 256 : d == 512 || rows <= 8 ? 8 : 16;
  p.row_tiles = static_cast<int>((rows + p.bm - 1) / p.bm);
  p.items = batch * kv_heads * p.row_tiles;
  // Keys of one row tile: with a window, those its tokens see.
  const int64_t bn = p.tc ? 128 : d == 512 ? 64 : d == 256 ? 128 : 256;
  const int64_t tokens = std::min(n, p.bm / group + 2);
  const int64_t keys = window > 0 ? std::min(slots, window + tokens + sink) : slots;
  const int64_t tiles = (keys + bn - 1) / bn + 1 + ((p.tc ? 1 : 2) * n + bn - 1) / bn;
  p.splits = 1;
  p.direct = false;
  p.ctas = 0;
  if (p.tc) {
    // The number of splits with the least estimated time, as tree_plan has it.
    const int64_t width = d == 512 ? 2 : 1, pairs = sms / 2;
    double best = 0;
    for (int64_t s = 1; s <= std::min<int64_t>(tiles, 64); ++s) {
      const double waves = static_cast<double>((p.items * width * s + pairs - 1) / pairs);
      double us = waves * (1.6 * static_cast<double>((tiles + s - 1) / s) + 8);
      if (s > 1) us += 4 + static_cast<double>(p.items * p.bm * d) * 8 * static_cast<double>(s) / 3e6;
      if (s == 1 || us < best) best = us, p.splits = static_cast<int>(s);
    }
    return p;
  }
  // An item per CTA, or all tiles dealt evenly: by estimated times.  A tile is about 1 us, an item's
  // start and end 3 us, joining the pieces a launch of 4 us.  From 8 items an SM on ragged lengths
  // even out by themselves.
  const double waves = static_cast<double>((p.items + sms - 1) / std::max(sms, 1));
  const double alone = waves * (static_cast<double>(tiles) + 3);
  const double dealt = static_cast<double>(p.items) * static_cast<double>(tiles) / sms + 3 * (waves + 1) + 4;
  p.direct = alone <= dealt || p.items >= 8 * static_cast<int64_t>(sms);
  p.ctas = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({sms, p.items * tiles, w8::kTreeMaxPieces})));
  return p;
}

struct PagedWs {
  int64_t part_o, part_ml, info, total;
};
static PagedWs paged_ws(const PagedPlan& p, int64_t d) {
  PagedWs w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  const int64_t part_rows = p.tc      ? (p.splits > 1 ? p.items * p.splits * p.bm : 0)
                            : p.direct ? 0
                                       : 2 * static_cast<int64_t>(p.ctas) * p.bm;
  w.part_o = take(part_rows * d * 4);
  w.part_ml = take(part_rows * 8);
  w.info = take(p.tc || p.direct ? 0 : p.items * 8);
  w.total = at;
  return w;
}

static int paged_shape(const w8_attention_paged_args& x) {
  W8_CHECK_ARG(x.batch >= 0 && x.heads >= 1 && x.kv_heads >= 1 && x.pages >= 0 && x.table_pages >= 0 && x.n_new >= 0,
               "negative size");
  W8_CHECK_ARG(x.heads % x.kv_heads == 0, "heads %lld must be a multiple of kv_heads %lld", (long long)x.heads,
               (long long)x.kv_heads);
  W8_CHECK_ARG(x.window >= 0 && x.window < (1ll << 31), "window must be 0 (none) or positive, below 2^31");
  W8_CHECK_ARG(x.sink >= 0 && x.sink < (1ll << 30), "sink must not be negative, and below 2^30");
  W8_CHECK_ARG(x.sink == 0 || x.window > 0, "sinks go with a window");
  if (x.page != 16 && x.page != 32 && x.page != 64 && x.page != 128) {
    set_error("pages of %lld tokens are not of 16, 32, 64 or 128", (long long)x.page);
    return W8_ERR_UNSUPPORTED;
  }
  W8_CHECK_ARG(x.table_pages < (1ll << 30) / x.page && x.pages < (1ll << 31) && x.n_new <= 65536 &&
                   x.batch <= (1ll << 20) && x.heads <= 65536,
               "size beyond the limits");
  if (x.head_dim != 64 && x.head_dim != 128 && x.head_dim != 256 && x.head_dim != 512) {
    set_error("head_dim %lld is not 64, 128, 256 or 512", (long long)x.head_dim);
    return W8_ERR_UNSUPPORTED;
  }
  W8_CHECK_ARG(x.batch * x.heads * x.n_new < (1ll << 31), "too many query rows");
  return W8_OK;
}

// 5-D map over pages of 8-bit rows: (128 bytes, row, 128-byte block, head, page).  A box
// {128, rows, blocks, 1, 1} lands as `blocks` swizzled [rows x 128] blocks (of 64 for D = 64).
static int paged_encode(CUtensorMap* map, const void* ptr, int64_t d, int64_t page, int64_t heads, int64_t pages,
                        const int64_t* stride, uint32_t rows) {
  const int64_t wide = std::min<int64_t>(d, 128);
  auto bytes = [&](int64_t size, int64_t s) { return static_cast<cuuint64_t>(size > 1 ? s : d); };
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(wide), static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(d / wide),
                              static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(pages)};
  const cuuint64_t strides[4] = {bytes(page, stride[2]), static_cast<cuuint64_t>(wide), bytes(heads, stride[1]),
                                 bytes(pages, stride[0])};
  const cuuint32_t box[5] = {static_cast<cuuint32_t>(wide), rows, static_cast<cuuint32_t>(d / wide), 1, 1};
  return tree_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, ptr, dims, strides, box,
                     d == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, "pages");
}

template <typename T, int D, int NT>
static int paged_main(const w8_attention_paged_args& x, const w8::PagedArgs& pa, int64_t blocks, int device,
                      cudaStream_t stream) {
  using C = w8::PagedCfg<D, NT>;
  constexpr bool kHalf = __is_same(T, __half);
  const w8::TreeArgs& a = pa.t;
  static bool done[64] = {};
  if (!done[device]) {
    W8_CUDA_TRY(cudaFuncSetAttribute(w8::attn_paged_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     C::kSmem));
    done[device] = true;
  }
  CUtensorMap tk, tv, tkt, tvt, tkn, tvn;
  auto rows = [&](CUtensorMap* map, const void* p, int64_t n, const int64_t* s) {
    return tree_encode_rows(map, p, kHalf, D, n, a.kv_heads, a.batch, s[0], s[1], s[2], C::kBN16, D / 64);
  };
  int st = rows(&tkn, x.k_new, a.n, x.k_new_stride);
  if (st == W8_OK) st = rows(&tvn, x.v_new, a.n, x.v_new_stride);
  if (st == W8_OK) st = rows(&tkt, x.k_tail, x.page, x.k_tail_stride);
  if (st == W8_OK) st = rows(&tvt, x.v_tail, x.page, x.v_tail_stride);
  tk = tkn, tv = tvn;  // an empty pool: never read
  const uint32_t box = static_cast<uint32_t>(std::min<int64_t>(x.page, C::kBN));
  if (st == W8_OK && x.pages > 0) st = paged_encode(&tk, x.k, D, x.page, x.kv_heads, x.pages, x.k_stride, box);
  if (st == W8_OK && x.pages > 0) st = paged_encode(&tv, x.v, D, x.page, x.kv_heads, x.pages, x.v_stride, box);
  if (st != W8_OK) return st;
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
  return cuda_status(cudaLaunchKernelEx(&cfg, w8::attn_paged_kernel<T, D, NT>, tk, tv, tkt, tvt, tkn, tvn, pa));
}

template <typename T, int D>
static int paged_go(const w8_attention_paged_args& x, const w8::PagedArgs& a, const PagedPlan& p, int device,
                    cudaStream_t stream) {
  W8_CHECK_ARG(p.items < (1ll << 31) / 2, "too many row tiles");
  const int64_t blocks = p.direct ? p.items : p.ctas;
  constexpr bool kHalf = __is_same(T, __half);
  int st;
  if (p.tc) {
    st = paged_tc(x, a, kHalf, p.items, device, stream);
  } else if (p.bm == 8) {
    st = paged_main<T, D, 1>(x, a, blocks, device, stream);
  } else {
    if constexpr (D <= 256)
      st = paged_main<T, D, 2>(x, a, blocks, device, stream);
    else
      st = W8_ERR_UNSUPPORTED;  // (no plan has it)
  }
  if (st != W8_OK || (p.tc ? p.splits == 1 : p.direct || p.ctas <= 1)) return st;
  return tree_join(a.t, kHalf, D, p.bm, stream);
}

// Read (and optionally clear) the sticky device status of the paged attention.
int paged_device_status(int clear, int* out) {
  W8_CUDA_TRY(cudaMemcpyFromSymbol(out, w8::g_tree_status, sizeof(int)));
  if (clear) {
    const int zero = 0;
    W8_CUDA_TRY(cudaMemcpyToSymbol(w8::g_tree_status, &zero, sizeof(int)));
  }
  return W8_OK;
}

}  // namespace w8host

extern "C" int64_t w8_attention_paged_workspace_bytes(const w8_attention_paged_args* in) {
  using namespace w8host;
  if (in == nullptr || paged_shape(*in) != W8_OK) return -1;
  const w8_attention_paged_args& x = *in;
  int sms = 148;
  if (num_sms(&sms) != W8_OK) sms = 148;
  const PagedPlan p = paged_plan(x.batch, x.kv_heads, x.heads / x.kv_heads, x.n_new, x.head_dim, x.table_pages * x.page,
                                 x.window, x.sink, sms);
  return paged_ws(p, x.head_dim).total;
}

extern "C" int w8_attention_paged(const w8_attention_paged_args* in, void* workspace, int64_t workspace_bytes,
                                  w8_stream_t stream) {
  using namespace w8host;
  W8_CHECK_ARG(in != nullptr, "null arguments");
  const w8_attention_paged_args& x = *in;
  int st = paged_shape(x);
  if (st != W8_OK) return st;
  W8_CHECK_ARG(x.dtype == W8_BF16 || x.dtype == W8_FP16, "dtype must be W8_BF16 or W8_FP16");
  if (x.batch == 0 || x.n_new == 0) return W8_OK;
  // (positive in the kernels' fp32 log2 units too: a masked score is -inf times it)
  const float scale_log2 = static_cast<float>(x.scale * 1.4426950408889634);
  W8_CHECK_ARG(scale_log2 > 0.f && scale_log2 < 3e38f, "scale must be positive and finite");
  W8_CHECK_ARG(x.q && x.k_tail && x.v_tail && x.k_new && x.v_new && x.out && x.lens, "null pointer");
  W8_CHECK_ARG(x.pages == 0 || (x.k && x.v && x.k_scale && x.v_scale), "null pages");
  W8_CHECK_ARG(x.table_pages == 0 || x.table, "null table");
  W8_CHECK_ARG(x.tree == nullptr || x.window == 0 || x.depth != nullptr, "a tree with a window needs the tokens' depths");
  W8_CHECK_ARG(x.out != x.q && x.out != x.k && x.out != x.v && x.out != x.k_tail && x.out != x.v_tail &&
                   x.out != x.k_new && x.out != x.v_new,
               "out must not be an input");
  const void* ptrs[8] = {x.q, x.out, x.k_tail, x.v_tail, x.k_new, x.v_new, x.k, x.v};
  const int64_t* strides[8] = {x.q_stride, x.out_stride, x.k_tail_stride, x.v_tail_stride, x.k_new_stride, x.v_new_stride,
                               x.k_stride, x.v_stride};
  const int64_t KV = x.kv_heads;
  const int64_t sizes[8][3] = {{x.batch, x.heads, x.n_new}, {x.batch, x.heads, x.n_new}, {x.batch, KV, x.page},
                               {x.batch, KV, x.page},       {x.batch, KV, x.n_new},     {x.batch, KV, x.n_new},
                               {x.pages, KV, x.page},       {x.pages, KV, x.page}};
  for (int i = 0; i < 8; ++i) {
    const int64_t of = i < 6 ? 8 : 16;
    W8_CHECK_ALIGN(aligned(ptrs[i], 16), "q, pages, tails, k_new, v_new and out must be 16-byte aligned");
    for (int j = 0; j < 3; ++j) {
      if (sizes[i][j] <= 1) continue;
      W8_CHECK_ALIGN(strides[i][j] % of == 0, "the strides of q, tails, k_new, v_new and out must be multiples of 8, of pages of 16");
      W8_CHECK_ARG(i < 2 || (strides[i][j] > 0 && strides[i][j] < (1ll << 38)),
                   "the strides of pages, tails, k_new and v_new must be positive and below 2^38");
    }
  }
  int device = 0, sms = 0;
  st = require_sm100(&device);
  if (st != W8_OK) return st;
  st = num_sms(&sms);
  if (st != W8_OK) return st;
  const int64_t group = x.heads / x.kv_heads;
  const PagedPlan p = paged_plan(x.batch, KV, group, x.n_new, x.head_dim, x.table_pages * x.page, x.window, x.sink, sms);
  const PagedWs w = paged_ws(p, x.head_dim);
  W8_CHECK_ARG(w.total == 0 || (workspace != nullptr && workspace_bytes >= w.total),
               "workspace of %lld bytes needed (got %lld)", (long long)w.total, (long long)workspace_bytes);
  W8_CHECK_ALIGN(aligned(workspace, 16), "workspace must be 16-byte aligned");
  w8::PagedArgs pa = {};
  w8::TreeArgs& a = pa.t;
  a.q = static_cast<const uint16_t*>(x.q);
  a.kn = static_cast<const uint16_t*>(x.k_new);
  a.vn = static_cast<const uint16_t*>(x.v_new);
  a.o = static_cast<uint16_t*>(x.out);
  a.lens = x.lens;
  a.tree = x.tree;
  a.depth = x.depth;
  a.q_b = x.q_stride[0], a.q_h = x.q_stride[1], a.q_t = x.q_stride[2];
  a.kn_b = x.k_new_stride[0], a.kn_h = x.k_new_stride[1], a.kn_t = x.k_new_stride[2];
  a.vn_b = x.v_new_stride[0], a.vn_h = x.v_new_stride[1], a.vn_t = x.v_new_stride[2];
  a.o_b = x.out_stride[0], a.o_h = x.out_stride[1], a.o_t = x.out_stride[2];
  a.tree_b = x.tree_stride[0], a.tree_i = x.tree_stride[1];
  a.depth_b = x.depth_stride;
  a.batch = static_cast<int>(x.batch);
  a.kv_heads = static_cast<int>(KV);
  a.group = static_cast<int>(group);
  a.group_rcp = group > 1 ? static_cast<uint32_t>((1ull << 32) / static_cast<uint64_t>(group)) : 0u;
  a.n = static_cast<int>(x.n_new);
  a.slots = static_cast<int>(x.table_pages * x.page);
  a.window = static_cast<int>(x.window);
  a.sink = static_cast<int>(x.sink);
  a.scale_log2 = scale_log2;
  a.row_tiles = p.row_tiles;
  a.splits = p.splits;
  // Boxes of 128 query rows: the group divides 128, and no stride of 0.
  a.q_tma = group <= 128 && (group & (group - 1)) == 0;
  for (int j = 0; j < 3; ++j)
    if (sizes[0][j] > 1 && (x.q_stride[j] <= 0 || x.q_stride[j] >= (1ll << 38))) a.q_tma = 0;
  a.direct = p.direct ? 1 : 0;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(ws + w.part_o);
  a.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
  a.info = p.tc ? nullptr : reinterpret_cast<int2*>(ws + w.info);
  pa.table = x.table;
  pa.table_b = x.table_stride;
  pa.table_pages = static_cast<int>(x.table_pages);
  pa.pages = static_cast<int>(x.pages);
  pa.shift = x.page == 16 ? 4 : x.page == 32 ? 5 : x.page == 64 ? 6 : 7;
  pa.ks = x.k_scale, pa.vs = x.v_scale;
  pa.ks_p = x.k_scale_stride[0], pa.ks_h = x.k_scale_stride[1];
  pa.vs_p = x.v_scale_stride[0], pa.vs_h = x.v_scale_stride[1];
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = x.dtype == W8_BF16;
  switch (x.head_dim) {
    case 64:
      return bf ? paged_go<__nv_bfloat16, 64>(x, pa, p, device, s) : paged_go<__half, 64>(x, pa, p, device, s);
    case 128:
      return bf ? paged_go<__nv_bfloat16, 128>(x, pa, p, device, s) : paged_go<__half, 128>(x, pa, p, device, s);
    case 256:
      return bf ? paged_go<__nv_bfloat16, 256>(x, pa, p, device, s) : paged_go<__half, 256>(x, pa, p, device, s);
    default:
      return bf ? paged_go<__nv_bfloat16, 512>(x, pa, p, device, s) : paged_go<__half, 512>(x, pa, p, device, s);
  }
}
