// What a decode step does to its K / V caches besides attending: appending the new tokens'
// rows (a drafted tree's accepted path), evicting slots by accumulated attention weight,
// and letting beams' states follow the surviving beams.  The reference grows a
// DynamicCache by concatenation (pipeline.py:318-339) and never evicts or searches.
//
// All of it is data movement: rows of head_dim 16-bit values (any 16-byte multiple) are
// copied as 16-byte chunks, one chunk per thread, so a warp moves 512 contiguous bytes.
// Indexes come from device memory; one outside its range is skipped and recorded in the
// device status, never followed.
#include "common.cuh"

#include <algorithm>

namespace w8 {

__device__ int g_cache_status = 0;

__device__ __forceinline__ void cache_bad_index() { atomicExch(&g_cache_status, W8_ERR_INVALID_ARG); }

// ---------------------------------------------------------------- append
struct AppendArgs {
  uint8_t *k, *v;
  const uint8_t *kn, *vn;
  int64_t k_b, k_h, k_s, v_b, v_h, v_s, kn_b, kn_h, kn_t, vn_b, vn_h, vn_t;  // bytes
  const int* lens;
  const int* path;  // [B, P] or null: every new token in order
  int64_t path_b;
  float* w;
  const float* wn;  // [B, KV, N] or null: new slots start at 0
  int64_t w_b, w_h, wn_b, wn_h;
  int* pos;
  const int* seen;
  int64_t pos_b, pos_h;
  int* lens_out;
  int kv_heads, n, steps, slots, chunks;
  int shift;  // log2 of the chunks, or -1
};

constexpr int kAppendRows = 32;   // path entries per CTA
constexpr int kAppendChunks = 4;  // 16-byte chunks of a thread in flight

// One CTA: up to 32 path entries of one (sequence, cache head).  An entry counts if no entry up
// to it is negative.  The chain length, path, row is all latency, so CTAs are small and many
// enough to wait it out together (256 sequences of 8 heads, paths of 1 to 17: CTAs of 256
// threads and 16 entries 9.6 us, one CTA for all heads of a sequence 17.7, these 6.6 us,
// 2.9 TB/s).
constexpr int kAppendThreads = 128;
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const AppendArgs a) {
  __shared__ int draft[kAppendRows];
  __shared__ int ended;
  const int b = blockIdx.x / a.kv_heads, c = blockIdx.x % a.kv_heads, tid = threadIdx.x;
  const int j0 = blockIdx.y * kAppendRows, j1 = min(j0 + kAppendRows, a.steps);
  pdl_launch_dependents();
  pdl_wait();
  const int len = a.lens[b];
  int d = j0 + tid;  // this thread's entry: a draft's index, or -1
  if (a.path != nullptr) d = tid < j1 - j0 ? a.path[b * a.path_b + j0 + tid] : -1;
  int count = a.steps;  // entries before the first negative one
  if (a.path != nullptr) {
    if (tid == 0) ended = a.steps;
    __syncthreads();
    const int upto = blockIdx.y == 0 && c == 0 ? a.steps : j1;  // the first CTA counts them all
    if (d < 0 && tid < j1 - j0) atomicMin(&ended, j0 + tid);
    for (int j = tid; j < upto; j += kAppendThreads)
      if ((j < j0 || j >= j1) && a.path[b * a.path_b + j] < 0) atomicMin(&ended, j);
    __syncthreads();
    count = ended;
  }
  const bool ok = len >= 0 && len <= a.slots;
  if (!ok && tid == 0) cache_bad_index();
  if (blockIdx.y == 0 && c == 0 && tid == 0) {
    a.lens_out[b] = ok ? min(len + count, a.slots) : len;
    if (ok && len + count > a.slots) cache_bad_index();
  }
  if (!ok) return;
  const int last = min(min(j1, count), a.slots - len) - j0;  // entries of this CTA with a slot
  if (tid < kAppendRows) {
    if (tid >= last) {
      d = -1;
    } else if (d >= a.n) {
      cache_bad_index();
      d = -1;
    }
    draft[tid] = d;
    if (d >= 0) {
      const int64_t slot = len + j0 + tid;
      if (a.w != nullptr) a.w[b * a.w_b + c * a.w_h + slot] = a.wn != nullptr ? a.wn[b * a.wn_b + c * a.wn_h + d] : 0.f;
      if (a.pos != nullptr) a.pos[b * a.pos_b + c * a.pos_h + slot] = a.seen[b] + j0 + tid;
    }
  }
  __syncthreads();
  const int work = last * 2 * a.chunks;  // chunks of (entry, K or V)
  for (int e0 = tid; e0 < work; e0 += kAppendThreads * kAppendChunks) {
    uint4 x[kAppendChunks];
    uint8_t* dst[kAppendChunks];
#pragma unroll
    for (int i = 0; i < kAppendChunks; ++i) {
      dst[i] = nullptr;
      const int e = e0 + kAppendThreads * i;
      if (e >= work) continue;
      const int row = a.shift >= 0 ? e >> a.shift : e / a.chunks, ch = e - row * a.chunks, j = row >> 1, from = draft[j];
      if (from < 0) continue;
      const bool is_v = row & 1;
      const uint8_t* src = is_v ? a.vn + b * a.vn_b + c * a.vn_h + from * a.vn_t : a.kn + b * a.kn_b + c * a.kn_h + from * a.kn_t;
      x[i] = reinterpret_cast<const uint4*>(src)[ch];
      const int64_t slot = len + j0 + j;
      dst[i] = (is_v ? a.v + b * a.v_b + c * a.v_h + slot * a.v_s : a.k + b * a.k_b + c * a.k_h + slot * a.k_s) + ch * 16;
    }
#pragma unroll
    for (int i = 0; i < kAppendChunks; ++i)
      if (dst[i] != nullptr) *reinterpret_cast<uint4*>(dst[i]) = x[i];
  }
}

// ---------------------------------------------------------------- evict
struct EvictArgs {
  const float* w;
  const int* pos;
  float* w_out;
  int* pos_out;
  int64_t w_b, w_h, pos_b, pos_h, wo_b, wo_h, po_b, po_h;
  const int* lens;
  int* lens_out;
  int kv_heads, slots, budget, sink, recent;
  int* moves;  // per (sequence, head): count, then [most] destinations, then [most] sources
  int most;
  int cluster;  // CTAs of a row
};

constexpr int kEvictThreads = 512;
constexpr int kEvictCluster = 8;  // CTAs of a row at most (portable)
constexpr int kEvictLongThreads = 1024;

// Exclusive prefix sum of `v` over the block; `total` is the block's sum.
__device__ __forceinline__ int evict_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  const int before = warp > 0 ? warp_sums[warp - 1] : 0;
  total = warp_sums[31];
  __syncthreads();  // the sums may be reused
  return before + x - v;
}

// Order-preserving bits of an accumulated weight: -0 counts as 0, NaN as the lowest value.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0x007FFFFFu;  // -inf's key
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// One (sequence, cache head) of an eviction.
struct EvictRow {
  const float* w;
  const int* pos;
  float* w_out;
  int* pos_out;
  int* moves;
  int len, left;
};
__device__ __forceinline__ EvictRow evict_row(const EvictArgs& a, int row, int rank) {
  const int b = row / a.kv_heads, c = row % a.kv_heads;
  EvictRow r;
  r.w = a.w + b * a.w_b + c * a.w_h;
  r.pos = a.pos + b * a.pos_b + c * a.pos_h;
  r.w_out = a.w_out + b * a.wo_b + c * a.wo_h;
  r.pos_out = a.pos_out + b * a.po_b + c * a.po_h;
  r.moves = a.moves + static_cast<int64_t>(row) * (1 + 2 * a.most);
  r.len = a.lens[b];
  if (r.len < 0 || r.len > a.slots) {
    if (threadIdx.x == 0 && rank == 0) cache_bad_index();
    r.len = r.len < 0 ? 0 : a.slots;
  }
  r.left = min(r.len, a.budget);
  if (c == 0 && threadIdx.x == 0 && rank == 0) a.lens_out[b] = r.left;
  return r;
}

// The small state after the cut: kept slots as they are, holes from their movers, nothing
// behind.  All threads; w_out / pos_out may be w / pos (what is read is never written before).
__device__ __forceinline__ void evict_state(const EvictArgs& a, const EvictRow& r, int count, int threads) {
  const int tid = threadIdx.x;
  if (tid == 0) r.moves[0] = count;
  if (r.w_out != r.w || r.pos_out != r.pos)
#pragma unroll 8
    for (int s = tid; s < r.left; s += threads) {
      const float ws = r.w[s];
      const int ps = r.pos[s];
      r.w_out[s] = ws;
      r.pos_out[s] = ps;
    }
  __syncthreads();
#pragma unroll 8
  for (int i = tid; i < count; i += threads) {
    const int dst = r.moves[1 + i], src = r.moves[1 + a.most + i];
    r.w_out[dst] = r.w[src];
    r.pos_out[dst] = r.pos[src];
  }
  __syncthreads();
#pragma unroll 8
  for (int s = r.left + tid; s < a.slots; s += threads) {
    r.w_out[s] = 0.f;
    r.pos_out[s] = -1;
  }
}

// The last position that is not recent.
__device__ __forceinline__ int evict_recent_after(const EvictArgs& a, int last) {
  const int64_t after = static_cast<int64_t>(last) - a.recent;
  return after < INT32_MIN ? INT32_MIN : static_cast<int>(after);
}

// A slot's place in the order: protected ones (all alike, above every weight) before the others
// by weight.
__device__ __forceinline__ uint32_t evict_key(const EvictArgs& a, float w, int pos, int recent_after) {
  return pos < a.sink || pos > recent_after ? 0xFFFFFFFFu : weight_key(w);
}

// Which slots of a (sequence, cache head) stay: the `budget` largest by (protected, weight,
// lower slot).  A warp holds the keys of 32 KPT consecutive slots in registers, lane i of step
// j the slot 32 j + i; the budget-th key is found by bisection on its bits, one count over the
// block an iteration (some 15 of them: a histogram's shared-memory atomics meet in the few
// exponents that weights have, and took 16 us where this takes 8 for 3658 slots), until
// a cut has exactly `budget` keys or, among equal ones, the lowest slots fill it.  Ballots in
// slot order then pair the i-th evicted slot below the budget with the i-th kept one behind it.
template <int KPT>
__global__ void __launch_bounds__(kEvictThreads, KPT <= 32 ? 2 : 1) evict_select_kernel(const EvictArgs a) {
  constexpr int kWarps = kEvictThreads / 32;
  __shared__ int counts[2][kWarps];
  __shared__ int per_warp[3][kWarps];
  __shared__ uint32_t kept[kWarps][KPT];
  extern __shared__ uint32_t lists[];  // [most] evicted slots, [budget] sources: 16 bits each
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  const EvictRow r = evict_row(a, blockIdx.x, 0);
  // Nothing behind the last slot: written first, under the loads, unless the row is cut in place.
  auto clear = [&]() {
#pragma unroll 8
    for (int s = r.left + tid; s < a.slots; s += kEvictThreads) {
      r.w_out[s] = 0.f;
      r.pos_out[s] = -1;
    }
  };
  const bool in_place = r.w_out == r.w || r.pos_out == r.pos;
  if (!in_place) clear();
  int moved = 0;
  if (r.len > a.budget) {
    const int s0 = warp * 32 * KPT + lane;  // slot of step i: s0 + 32 i
    uint32_t key[KPT];
    int last = INT32_MIN;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const int s = s0 + 32 * i;
      key[i] = s < r.len ? __float_as_uint(r.w[s]) : 0u;
      if (s < r.len) last = max(last, r.pos[s]);
    }
    // The highest position decides what is recent (so the positions are read again, from L2: held
    // with the keys they would leave no registers for loads in flight).
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0) counts[0][warp] = last;
    __syncthreads();
    last = __reduce_max_sync(0xffffffffu, counts[0][lane % kWarps]);
    const int recent_after = evict_recent_after(a, last);
    uint32_t least = 0xFFFFFFFFu, most = 0u;  // of the keys that are not protected
#pragma unroll
    for (int i = 0; i < KPT; ++i) {  // 0 behind the length: below every slot's
      const int s = s0 + 32 * i;
      key[i] = s < r.len ? evict_key(a, __uint_as_float(key[i]), r.pos[s], recent_after) : 0u;
      if (key[i] != 0xFFFFFFFFu) most = max(most, key[i]);
      if (key[i] != 0u) least = min(least, key[i]);
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();
    if (lane == 0) counts[0][warp] = static_cast<int>(least), counts[1][warp] = static_cast<int>(most);
    __syncthreads();
    least = __reduce_min_sync(0xffffffffu, static_cast<uint32_t>(counts[0][lane % kWarps]));
    most = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(counts[1][lane % kWarps]));
    __syncthreads();
    int turn = 0;
    auto count = [&](uint32_t at) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < KPT; ++i) n += key[i] >= at ? 1 : 0;
      n = __reduce_add_sync(0xffffffffu, n);
      turn ^= 1;  // (two buffers: one barrier an iteration)
      if (lane == 0) counts[turn][warp] = n;
      __syncthreads();
      return __reduce_add_sync(0xffffffffu, lane < kWarps ? counts[turn][lane] : 0);
    };
    // Bisect: `reach` keys are >= cut, at least `budget` of them, and fewer are >= over.  The
    // protected keys (all ones) may fill the budget alone.
    uint32_t cut = least, over = 0xFFFFFFFFu;
    int reach = r.len;
    const int protect = count(0xFFFFFFFFu);
    if (protect >= a.budget)
      cut = 0xFFFFFFFFu, reach = protect;
    else
      over = most + 1;
    while (reach != a.budget && over - cut > 1) {
      const uint32_t mid = cut + (over - cut) / 2;
      const int n = count(mid);
      if (n >= a.budget)
        cut = mid, reach = n;
      else
        over = mid;
    }
    // Of the keys equal to the cut the last reach - budget in slot order go.
    __syncthreads();
    const bool ties = reach != a.budget;  // (the same for all threads)
    int room = 0;                         // equal keys that stay, counted from this warp's first
    if (ties) {
      int eq = 0;
#pragma unroll
      for (int i = 0; i < KPT; ++i) eq += __popc(__ballot_sync(0xffffffffu, key[i] == cut));
      if (lane == 0) per_warp[0][warp] = eq;
      __syncthreads();
      const int mine = lane < kWarps ? per_warp[0][lane] : 0;
      room = __reduce_add_sync(0xffffffffu, mine) - (reach - a.budget) -
             __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
    }
    const uint32_t before = (1u << lane) - 1u;
    auto low_bits = [&](int i) {  // this step's slots below the budget
      const int n = a.budget - (s0 - lane + 32 * i);
      return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
    };
    int holes = 0, movers = 0;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      bool stays = key[i] >= cut;
      if (ties) {
        const uint32_t eq = __ballot_sync(0xffffffffu, key[i] == cut);
        stays = key[i] > cut || (key[i] == cut && __popc(eq & before) < room);
        room -= __popc(eq);
      }
      const uint32_t keep = __ballot_sync(0xffffffffu, stays), low = low_bits(i);
      if (lane == 0) kept[warp][i] = keep;
      holes += __popc(~keep & low);
      movers += __popc(keep & ~low);
    }
    if (lane == 0) per_warp[1][warp] = holes, per_warp[2][warp] = movers;
    __syncthreads();
    const int wh = lane < kWarps ? per_warp[1][lane] : 0, wm = lane < kWarps ? per_warp[2][lane] : 0;
    int hole_at = __reduce_add_sync(0xffffffffu, lane < warp ? wh : 0);
    int mover_at = __reduce_add_sync(0xffffffffu, lane < warp ? wm : 0);
    moved = __reduce_add_sync(0xffffffffu, wm);
    // The evicted slots in order, in shared memory; then each mover finds its own, and each slot
    // below the budget what it will hold.
    uint16_t* hole_slots = reinterpret_cast<uint16_t*>(lists);
    uint16_t* src_slots = hole_slots + a.most;
#pragma unroll 4
    for (int i = 0; i < KPT; ++i) {
      const uint32_t low = low_bits(i), h = ~kept[warp][i] & low;
      if (low == 0u) break;
      if ((h >> lane) & 1u) hole_slots[hole_at + __popc(h & before)] = static_cast<uint16_t>(s0 + 32 * i);
      if ((low >> lane) & 1u) src_slots[s0 + 32 * i] = static_cast<uint16_t>(s0 + 32 * i);
      hole_at += __popc(h);
    }
    __syncthreads();
#pragma unroll 4
    for (int i = 0; i < KPT; ++i) {
      const uint32_t m = kept[warp][i] & ~low_bits(i);
      if ((m >> lane) & 1u) {
        const int j = mover_at + __popc(m & before), dst = hole_slots[j];
        r.moves[1 + j] = dst;
        r.moves[1 + a.most + j] = s0 + 32 * i;
        src_slots[dst] = static_cast<uint16_t>(s0 + 32 * i);
      }
      mover_at += __popc(m);
    }
    __syncthreads();
    // The small state.  (In place too: what is read from another slot lies behind the budget.)
#pragma unroll 8
    for (int s = tid; s < r.left; s += kEvictThreads) {
      const int src = src_slots[s];
      const float ws = r.w[src];
      const int ps = r.pos[src];
      r.w_out[s] = ws;
      r.pos_out[s] = ps;
    }
  } else if (r.w_out != r.w || r.pos_out != r.pos) {
#pragma unroll 8
    for (int s = tid; s < r.left; s += kEvictThreads) {
      const float ws = r.w[s];
      const int ps = r.pos[s];
      r.w_out[s] = ws;
      r.pos_out[s] = ps;
    }
  }
  if (tid == 0) r.moves[0] = moved;
  if (in_place) {
    __syncthreads();  // every slot's weight and position have been read
    clear();
  }
}

// The same for few rows or long ones: a row is held in the registers of a cluster of 2 to 8 CTAs,
// its slots in chunks of 32 KPT dealt to the CTAs in turn, a warp a chunk.  A barrier of the
// cluster costs more than a block's, so a step of the search counts the keys at three places
// between the bounds (every warp writes its counts into all CTAs' shared memory, one barrier a
// step).  Evicted slots meet their movers through the list that the moves read too, and a
// slot's weight and position are read by one thread only, so the cut may be in place.  One row
// of 16001 slots 17 us where one CTA takes 30, of 40000 27 where evict_select_long_kernel takes
// 115; 144 rows of 16001 slots, which fill the SMs by themselves, 58 and more against 56.
template <int KPT>
__global__ void __launch_bounds__(kEvictThreads, KPT <= 16 ? 2 : 1) evict_select_cluster_kernel(const EvictArgs a) {
  constexpr int kWarps = kEvictThreads / 32, kChunks = kWarps * kEvictCluster;
  constexpr bool kHeld = KPT <= 8;  // weights and positions too stay in registers
  __shared__ uint4 counts[2][kChunks];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ctas = a.cluster, rank = static_cast<int>(cluster_ctarank());
  const int chunks = kWarps * ctas, chunk = warp * ctas + rank;  // (chunks in slot order)
  pdl_launch_dependents();
  cluster_sync();  // all CTAs run: their shared memory may be written
  pdl_wait();
  const EvictRow r = evict_row(a, blockIdx.x / ctas, rank);
  if (r.len <= a.budget) {
    if (rank == 0 && tid == 0) r.moves[0] = 0;
    const int step = ctas * kEvictThreads;
    if (r.w_out != r.w || r.pos_out != r.pos) {
#pragma unroll 4
      for (int s = rank * kEvictThreads + tid; s < r.len; s += step) {
        const float ws = r.w[s];
        const int ps = r.pos[s];
        r.w_out[s] = ws;
        r.pos_out[s] = ps;
      }
    }
#pragma unroll 4
    for (int s = r.len + rank * kEvictThreads + tid; s < a.slots; s += step) {
      r.w_out[s] = 0.f;
      r.pos_out[s] = -1;
    }
    return;  // (the same for the whole cluster)
  }
  // One value of every chunk to all CTAs; `turn` alternates, so that one barrier a step is enough.
  int turn = 0;
  auto exchange = [&](uint32_t x, uint32_t y, uint32_t z) {
    turn ^= 1;
    if (lane < ctas)
      asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                       mapa_shared(smem_u32(&counts[turn][chunk]), static_cast<uint32_t>(lane))),
                   "r"(x), "r"(y), "r"(z), "r"(0u)
                   : "memory");
    cluster_sync();
  };
  const int first = chunk * 32 * KPT, s0 = first + lane;  // slot of step i: s0 + 32 i
  uint32_t key[KPT];
  float wv[kHeld ? KPT : 1];
  int pv[kHeld ? KPT : 1];
  int last = INT32_MIN;
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const int s = s0 + 32 * i;
    const float w = s < r.len ? r.w[s] : 0.f;
    const int p = s < r.len ? r.pos[s] : INT32_MIN;
    if constexpr (kHeld) wv[i] = w, pv[i] = p;
    key[i] = __float_as_uint(w);
    last = max(last, p);
  }
  // The highest position decides what is recent.
  last = __reduce_max_sync(0xffffffffu, last);
  exchange(static_cast<uint32_t>(last), 0u, 0u);
  last = INT32_MIN;
  for (int i = lane; i < chunks; i += 32) last = max(last, static_cast<int>(counts[turn][i].x));
  last = __reduce_max_sync(0xffffffffu, last);
  const int recent_after = evict_recent_after(a, last);
  uint32_t least = 0xFFFFFFFFu, most = 0u, protect = 0u;  // the bounds of the keys that are not protected
#pragma unroll
  for (int i = 0; i < KPT; ++i) {  // 0 behind the length: below every slot's
    const int s = s0 + 32 * i;
    if (s < r.len) {
      int p;
      if constexpr (kHeld)
        p = pv[i];
      else
        p = r.pos[s];
      key[i] = evict_key(a, __uint_as_float(key[i]), p, recent_after);
      if (key[i] == 0xFFFFFFFFu)
        ++protect;
      else
        most = max(most, key[i]);
      least = min(least, key[i]);
    } else {
      key[i] = 0u;
    }
  }
  exchange(__reduce_min_sync(0xffffffffu, least), __reduce_max_sync(0xffffffffu, most),
           __reduce_add_sync(0xffffffffu, protect));
  least = 0xFFFFFFFFu, most = 0u, protect = 0u;
  for (int i = lane; i < chunks; i += 32) {
    const uint4 c = counts[turn][i];
    least = min(least, c.x), most = max(most, c.y), protect += c.z;
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  const int safe = static_cast<int>(__reduce_add_sync(0xffffffffu, protect));
  // `reach` keys are >= cut, at least `budget` of them, and fewer are >= over.  The protected
  // keys (all ones) may fill the budget alone.
  uint32_t cut = least, over = most + 1;
  int reach = r.len;
  if (safe >= a.budget) cut = over = 0xFFFFFFFFu, reach = safe;
  while (reach != a.budget && over - cut > 1) {
    const uint32_t width = over - cut, q = max(width / 4, 1u);
    uint32_t at[3], n[3] = {0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 3; ++j) at[j] = cut + min((j + 1) * q, width);
    if (first < r.len) {
#pragma unroll
      for (int i = 0; i < KPT; ++i)
#pragma unroll
        for (int j = 0; j < 3; ++j) n[j] += key[i] >= at[j] ? 1u : 0u;
      const uint32_t two = __reduce_add_sync(0xffffffffu, n[0] | n[1] << 16);  // (at most 1024 each)
      n[0] = two & 0xFFFFu, n[1] = two >> 16, n[2] = __reduce_add_sync(0xffffffffu, n[2]);
    }
    exchange(n[0], n[1], n[2]);
#pragma unroll
    for (int j = 0; j < 3; ++j) n[j] = 0u;
    for (int i = lane; i < chunks; i += 32) {
      const uint4 c = counts[turn][i];
      n[0] += c.x, n[1] += c.y, n[2] += c.z;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) n[j] = __reduce_add_sync(0xffffffffu, n[j]);
    uint32_t lo = cut, hi = over;
#pragma unroll
    for (int j = 0; j < 3; ++j) {  // (counts fall: the places that `budget` keys reach come first)
      if (static_cast<int>(n[j]) >= a.budget)
        lo = at[j], reach = static_cast<int>(n[j]);
      else
        hi = min(hi, at[j]);
    }
    cut = lo, over = hi;
  }
  // Of the keys equal to the cut the last reach - budget in slot order go.
  const bool ties = reach != a.budget;  // (the same for the whole cluster)
  int room = 0;                         // equal keys that stay, counted from this chunk's first
  if (ties) {
    int eq = 0;
#pragma unroll
    for (int i = 0; i < KPT; ++i) eq += __popc(__ballot_sync(0xffffffffu, key[i] == cut));
    exchange(static_cast<uint32_t>(eq), 0u, 0u);
    for (int i = lane; i < chunks; i += 32) {
      const int c = static_cast<int>(counts[turn][i].x);
      room += i < chunk ? 0 : c;
    }
    room = __reduce_add_sync(0xffffffffu, room) - (reach - a.budget);
  }
  const uint32_t before = (1u << lane) - 1u;
  auto low_bits = [&](int i) {  // step i's slots below the budget
    const int n = a.budget - (first + 32 * i);
    return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
  };
  uint32_t kept = 0;  // lane i: step i's slots that stay
  int holes = 0, movers = 0;
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    bool stays = key[i] >= cut;
    if (ties) {
      const uint32_t eq = __ballot_sync(0xffffffffu, key[i] == cut);
      stays = key[i] > cut || (key[i] == cut && __popc(eq & before) < room);
      room -= __popc(eq);
    }
    const uint32_t keep = __ballot_sync(0xffffffffu, stays), low = low_bits(i);
    if (lane == i) kept = keep;
    holes += __popc(~keep & low);
    movers += __popc(keep & ~low);
  }
  exchange(static_cast<uint32_t>(holes), static_cast<uint32_t>(movers), 0u);
  int hole_at = 0, mover_at = 0, moved = 0;
  for (int i = lane; i < chunks; i += 32) {
    const uint4 c = counts[turn][i];
    if (i < chunk) hole_at += c.x, mover_at += c.y;
    moved += c.y;
  }
  hole_at = __reduce_add_sync(0xffffffffu, hole_at);
  mover_at = __reduce_add_sync(0xffffffffu, mover_at);
  moved = __reduce_add_sync(0xffffffffu, moved);
  if (rank == 0 && tid == 0) r.moves[0] = moved;
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const uint32_t low = low_bits(i);
    if (low == 0u) break;
    const uint32_t h = ~__shfl_sync(0xffffffffu, kept, i) & low;
    if ((h >> lane) & 1u) r.moves[1 + hole_at + __popc(h & before)] = s0 + 32 * i;
    hole_at += __popc(h);
  }
  cluster_sync();
  // The small state: each slot's thread puts what it holds where it goes.
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const int s = s0 + 32 * i;
    const uint32_t keep = __shfl_sync(0xffffffffu, kept, i), low = low_bits(i), m = keep & ~low;
    if (((keep | ~low) >> lane) & 1u && s < a.slots) {  // (a hole is its mover's to write)
      const bool stays = (keep >> lane) & 1u;
      float ws = 0.f;
      int ps = -1;
      if (stays) {
        if constexpr (kHeld)
          ws = wv[i], ps = pv[i];
        else
          ws = r.w[s], ps = r.pos[s];
      }
      if ((m >> lane) & 1u) {
        const int j = mover_at + __popc(m & before), dst = __ldcg(r.moves + 1 + j);
        r.moves[1 + a.most + j] = s;
        r.w_out[dst] = ws;
        r.pos_out[dst] = ps;
        ws = 0.f, ps = -1;
      }
      r.w_out[s] = ws;
      r.pos_out[s] = ps;
    }
    mover_at += __popc(m);
  }
}

// The same for more slots than a cluster's registers hold: a radix selection of the budget-th key over four
// passes of the row, then one in slot order.
__global__ void __launch_bounds__(kEvictLongThreads) evict_select_long_kernel(const EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int warp_sums[32];
  __shared__ int pick[2];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const EvictRow r = evict_row(a, blockIdx.x, 0);
  const float* w = r.w;
  const int* pos = r.pos;
  int* moves = r.moves;
  const int len = r.len;
  int count = 0;
  if (len > a.budget) {
    // The highest position decides what is recent.
    int last = INT32_MIN;
    for (int s = tid; s < len; s += kEvictLongThreads) last = max(last, pos[s]);
    last = __reduce_max_sync(0xffffffffu, last);
    if ((tid & 31) == 0) warp_sums[tid >> 5] = last;
    __syncthreads();
    last = __reduce_max_sync(0xffffffffu, warp_sums[tid & 31]);
    __syncthreads();
    const int recent_after = evict_recent_after(a, last);
    auto key = [&](int s) {
      return evict_key(a, w[s], pos[s], recent_after);
    };
    uint32_t prefix = 0;
    int need = a.budget;  // keys still to take among those that share the prefix
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
      for (int s = tid; s < len; s += kEvictLongThreads) {
        const uint32_t k = key(s);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid < 32) {
        // Digits from the top, 8 per lane: the first whose cumulative count reaches `need`.
        int sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += hist[255 - 8 * tid - i];
        int incl = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, d);
          if (tid >= d) incl += y;
        }
        int before = incl - sum;
        if (before < need && incl >= need) {
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {
            const int h = hist[255 - 8 * tid - i];
            if (before + h >= need) {
              pick[0] = 255 - 8 * tid - i;
              pick[1] = need - before;
              break;
            }
            before += h;
          }
        }
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(pick[0]) << shift;
      need = pick[1];
      __syncthreads();
    }
    // In slot order: keys above the cut stay, and the first `need` equal to it.
    int equals = 0, holes = 0, movers = 0;
    for (int s0 = 0; s0 < len; s0 += kEvictLongThreads) {
      const int s = s0 + tid;
      const bool in = s < len;
      const uint32_t k = in ? key(s) : 0u;
      const bool eq = in && k == prefix;
      int total;
      const int rank = equals + evict_scan(eq, warp_sums, total);
      equals += total;
      const bool keep = in && (k > prefix || (eq && rank < need));
      const bool low = s < a.budget;
      const bool hole = in && low && !keep, mover = keep && !low;
      // A chunk holds holes, movers or (once) both: one scan of both counts packed.
      int both;
      const int at = evict_scan((hole ? 1 : 0) + (mover ? 1 << 16 : 0), warp_sums, both);
      if (hole) moves[1 + holes + (at & 0xFFFF)] = s;
      if (mover) moves[1 + a.most + movers + (at >> 16)] = s;
      holes += both & 0xFFFF;
      movers += both >> 16;
    }
    count = movers;
    __syncthreads();
  }
  evict_state(a, r, count, kEvictLongThreads);
}

struct MoveArgs {
  uint8_t *k, *v;
  int64_t k_b, k_h, k_s, v_b, v_h, v_s;  // bytes
  const int* moves;
  int most, kv_heads, chunks;
  int shift;  // log2 of the chunks of a row, or -1
};

constexpr int kMoveChunks = 4;  // 16-byte chunks of a thread in flight

// The moves of one (sequence, head): destinations (below the budget) and sources (behind
// it) are disjoint, so the rows move in place in any order.  Bound by HBM and its rows' order: a
// CTA's 1024 chunks are all loaded before the first is stored (24 sequences of 8 heads of 128,
// up to 16001 slots cut to 4096: some 70 us, 4.6 TB/s of single rows of 256 bytes).
__global__ void __launch_bounds__(256) evict_move_kernel(const MoveArgs a) {
  const int row = blockIdx.y, b = row / a.kv_heads, c = row % a.kv_heads;
  pdl_launch_dependents();
  pdl_wait();
  const int* moves = a.moves + static_cast<int64_t>(row) * (1 + 2 * a.most);
  const int64_t work = static_cast<int64_t>(moves[0]) * 2 * a.chunks;
  uint8_t* k = a.k + b * a.k_b + c * a.k_h;
  uint8_t* v = a.v + b * a.v_b + c * a.v_h;
  for (int64_t e0 = static_cast<int64_t>(blockIdx.x) * (256 * kMoveChunks) + threadIdx.x; e0 < work;
       e0 += static_cast<int64_t>(gridDim.x) * (256 * kMoveChunks)) {
    uint8_t* dst[kMoveChunks];
    const uint8_t* src[kMoveChunks];
    uint4 x[kMoveChunks];
#pragma unroll
    for (int i = 0; i < kMoveChunks; ++i) {
      const int64_t e = e0 + 256 * i;
      if (e < work) {
        const int64_t m = a.shift >= 0 ? e >> a.shift : e / a.chunks;  // row: move m / 2's K or V
        const int64_t ch = (e - m * a.chunks) * 16;
        const int j = static_cast<int>(m >> 1);
        uint8_t* base = ((m & 1) ? v : k) + ch;
        const int64_t pitch = (m & 1) ? a.v_s : a.k_s;
        dst[i] = base + moves[1 + j] * pitch;
        src[i] = base + moves[1 + a.most + j] * pitch;
      }
    }
#pragma unroll
    for (int i = 0; i < kMoveChunks; ++i)
      if (e0 + 256 * i < work) x[i] = *reinterpret_cast<const uint4*>(src[i]);
#pragma unroll
    for (int i = 0; i < kMoveChunks; ++i)
      if (e0 + 256 * i < work) *reinterpret_cast<uint4*>(dst[i]) = x[i];
  }
}

// ---------------------------------------------------------------- reorder
constexpr int kReorderTensors = 64;
struct ReorderArgs {
  uint8_t* x[kReorderTensors];
  int64_t x_r, x_h, x_s;  // bytes: row (beam), head, slot
  const void* beam;       // [groups, K] int64 or int32
  const int* lens;        // [groups * K] or null
  int beam_i64, k, heads, slots, chunks;
};

// One thread owns one 16-byte column of a group's K states: it reads the column of every
// beam's parent, then writes those that moved, so the beams change places without a second
// cache and a beam that stays costs nothing.  Bound by HBM: 16 x 8 beams, 1.34 GB read and
// written in 234 us, 5.7 TB/s.
template <int KMAX>
__global__ void __launch_bounds__(256) cache_reorder_kernel(const __grid_constant__ ReorderArgs a) {
  __shared__ int src[KMAX], end[KMAX];
  __shared__ int furthest;
  const int group = blockIdx.y / a.heads, h = blockIdx.y % a.heads, tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  if (tid == 0) furthest = 0;
  __syncthreads();
  if (tid < a.k) {
    const int64_t at = static_cast<int64_t>(group) * a.k + tid;
    const int64_t p = a.beam_i64 ? static_cast<const int64_t*>(a.beam)[at] : static_cast<const int*>(a.beam)[at];
    int s = tid, n = 0;
    if (p < 0 || p >= a.k) {
      cache_bad_index();
    } else if (p != tid) {
      s = static_cast<int>(p);
      n = a.slots;
      if (a.lens != nullptr) {
        n = a.lens[static_cast<int64_t>(group) * a.k + s];
        if (n < 0 || n > a.slots) {
          cache_bad_index();
          n = 0;
        }
      }
    }
    src[tid] = s;
    end[tid] = n;  // slots to copy: 0 for a beam that stays
    atomicMax(&furthest, n);
  }
  __syncthreads();
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + tid;
  const int64_t slot = e / a.chunks;
  if (slot >= furthest) return;
  uint8_t* base = a.x[blockIdx.z] + static_cast<int64_t>(group) * a.k * a.x_r + h * a.x_h + slot * a.x_s + (e % a.chunks) * 16;
  uint4 r[KMAX];
#pragma unroll
  for (int i = 0; i < KMAX; ++i)
    if (i < a.k && slot < end[i]) r[i] = *reinterpret_cast<const uint4*>(base + src[i] * a.x_r);
#pragma unroll
  for (int i = 0; i < KMAX; ++i)
    if (i < a.k && slot < end[i]) *reinterpret_cast<uint4*>(base + i * a.x_r) = r[i];
}

}  // namespace w8

namespace w8host {

int require_sm100(int* device);

template <typename Kern, typename Args>
static int launch_cache(Kern kern, dim3 grid, int threads, cudaStream_t stream, const Args& a, int smem = 0) {
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
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, a));
}

template <int KPT>
static int launch_evict(dim3 grid, int lists, int device, cudaStream_t stream, const w8::EvictArgs& e) {
  static bool done[64] = {};
  if (!done[device]) {
    W8_CUDA_TRY(cudaFuncSetAttribute(w8::evict_select_kernel<KPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024));
    done[device] = true;
  }
  return launch_cache(w8::evict_select_kernel<KPT>, grid, w8::kEvictThreads, stream, e, lists);
}

template <int KPT>
static int launch_evict_cluster(int64_t rows, cudaStream_t stream, const w8::EvictArgs& e) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * e.cluster));
  cfg.blockDim = dim3(w8::kEvictThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(e.cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, w8::evict_select_cluster_kernel<KPT>, e));
}

// Read (and optionally clear) the sticky device status of the cache operations.
int cache_device_status(int clear, int* out) {
  int v = 0;
  W8_CUDA_TRY(cudaMemcpyFromSymbol(&v, w8::g_cache_status, sizeof(int)));
  if (clear) {
    const int zero = 0;
    W8_CUDA_TRY(cudaMemcpyToSymbol(w8::g_cache_status, &zero, sizeof(int)));
  }
  *out = v;
  return W8_OK;
}

static int cache_shape(int64_t batch, int64_t kv_heads, int64_t slots, int64_t row_bytes) {
  W8_CHECK_ARG(batch >= 0 && kv_heads >= 1 && slots >= 0 && row_bytes >= 16, "negative or empty size");
  W8_CHECK_ARG(slots < (1ll << 30) && batch * kv_heads < (1ll << 31) && batch < (1ll << 31) && kv_heads < (1ll << 31) &&
                   row_bytes <= (1 << 20),
               "size beyond the limits");
  W8_CHECK_ALIGN(row_bytes % 16 == 0, "rows of %lld bytes: must be a multiple of 16", (long long)row_bytes);
  return W8_OK;
}

// Whether two int32 arrays share memory (what one CTA writes of one, another may yet have to read
// of the other).
static bool arrays_meet(const int32_t* p, int64_t n, const int32_t* q, int64_t m) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return p != nullptr && q != nullptr && a < b + 4 * static_cast<uintptr_t>(m) && b < a + 4 * static_cast<uintptr_t>(n);
}

static int cache_rows(const char* name, const void* p, const int64_t* strides) {
  W8_CHECK_ARG(p != nullptr, "%s is null", name);
  W8_CHECK_ALIGN(aligned(p, 16), "%s must be 16-byte aligned", name);
  for (int i = 0; i < 3; ++i)
    W8_CHECK_ALIGN(strides[i] % 16 == 0, "the strides of %s must be multiples of 16 bytes", name);
  return W8_OK;
}

}  // namespace w8host

extern "C" int w8_cache_append(const w8_cache_append_args* in, w8_stream_t stream) {
  using namespace w8host;
  W8_CHECK_ARG(in != nullptr, "null arguments");
  const w8_cache_append_args& x = *in;
  int st = cache_shape(x.batch, x.kv_heads, x.slots, x.row_bytes);
  if (st != W8_OK) return st;
  W8_CHECK_ARG(x.n_new >= 0 && x.steps >= 0 && x.n_new < (1ll << 20) && x.steps <= (1 << 20), "size beyond the limits");
  W8_CHECK_ARG(x.path != nullptr || x.steps == x.n_new, "without a path every new token is appended (steps = n_new)");
  if (x.batch == 0) return W8_OK;
  W8_CHECK_ARG(x.lens && x.lens_out, "null lens");
  W8_CHECK_ARG(!arrays_meet(x.lens, x.batch, x.lens_out, x.batch), "lens_out must not be lens nor overlap it");
  W8_CHECK_ARG(!x.positions || x.seen, "positions need seen");
  W8_CHECK_ARG(!x.positions || !arrays_meet(x.seen, x.batch, x.lens_out, x.batch),
               "lens_out must not be seen nor overlap it");
  if (x.path && x.steps > 0 && arrays_meet(x.path, (x.batch - 1) * x.path_stride + x.steps, x.lens_out, x.batch))
    for (int64_t b = 0; b < x.batch; ++b)  // (it may lie between the rows)
      W8_CHECK_ARG(!arrays_meet(x.path + b * x.path_stride, x.steps, x.lens_out, x.batch), "lens_out must not overlap path");
  W8_CHECK_ARG(!x.draft_weights || x.weights, "draft_weights need weights");
  if (x.slots > 0 && x.n_new > 0) {
    if ((st = cache_rows("k", x.k, x.k_stride)) != W8_OK) return st;
    if ((st = cache_rows("v", x.v, x.v_stride)) != W8_OK) return st;
    if ((st = cache_rows("k_new", x.k_new, x.k_new_stride)) != W8_OK) return st;
    if ((st = cache_rows("v_new", x.v_new, x.v_new_stride)) != W8_OK) return st;
  }
  int device = 0;
  if ((st = require_sm100(&device)) != W8_OK) return st;
  w8::AppendArgs a = {};
  a.k = static_cast<uint8_t*>(x.k), a.v = static_cast<uint8_t*>(x.v);
  a.kn = static_cast<const uint8_t*>(x.k_new), a.vn = static_cast<const uint8_t*>(x.v_new);
  a.k_b = x.k_stride[0], a.k_h = x.k_stride[1], a.k_s = x.k_stride[2];
  a.v_b = x.v_stride[0], a.v_h = x.v_stride[1], a.v_s = x.v_stride[2];
  a.kn_b = x.k_new_stride[0], a.kn_h = x.k_new_stride[1], a.kn_t = x.k_new_stride[2];
  a.vn_b = x.v_new_stride[0], a.vn_h = x.v_new_stride[1], a.vn_t = x.v_new_stride[2];
  a.lens = x.lens, a.path = x.path, a.path_b = x.path_stride;
  a.w = x.weights, a.w_b = x.weights_stride[0], a.w_h = x.weights_stride[1];
  a.wn = x.draft_weights, a.wn_b = x.draft_weights_stride[0], a.wn_h = x.draft_weights_stride[1];
  a.pos = x.positions, a.pos_b = x.positions_stride[0], a.pos_h = x.positions_stride[1], a.seen = x.seen;
  a.lens_out = x.lens_out;
  a.kv_heads = static_cast<int>(x.kv_heads), a.n = static_cast<int>(x.n_new), a.steps = static_cast<int>(x.steps);
  a.slots = static_cast<int>(x.slots), a.chunks = static_cast<int>(x.row_bytes / 16);
  a.shift = (a.chunks & (a.chunks - 1)) == 0 ? __builtin_ctz(a.chunks) : -1;
  const int64_t parts = std::max<int64_t>(1, (x.steps + w8::kAppendRows - 1) / w8::kAppendRows);
  return launch_cache(w8::cache_append_kernel,
                      dim3(static_cast<unsigned>(x.batch * x.kv_heads), static_cast<unsigned>(parts)), w8::kAppendThreads,
                      reinterpret_cast<cudaStream_t>(stream), a);
}

extern "C" int64_t w8_cache_evict_workspace_bytes(int64_t batch, int64_t kv_heads, int64_t slots, int64_t budget) {
  if (batch < 0 || kv_heads < 1 || slots < 0 || budget < 1) return -1;
  const int64_t most = std::max<int64_t>(0, std::min(budget, slots - budget));
  return batch * kv_heads * (1 + 2 * most) * 4;
}

extern "C" int w8_cache_evict(const w8_cache_evict_args* in, void* workspace, int64_t workspace_bytes,
                              w8_stream_t stream) {
  using namespace w8host;
  W8_CHECK_ARG(in != nullptr, "null arguments");
  const w8_cache_evict_args& x = *in;
  int st = cache_shape(x.batch, x.kv_heads, x.slots, x.row_bytes);
  if (st != W8_OK) return st;
  W8_CHECK_ARG(x.budget >= 1 && x.sink >= 0 && x.recent >= 0 && x.budget < (1ll << 31) && x.sink < (1ll << 31) && x.recent < (1ll << 31),
               "budget must be positive, sink and recent not negative");
  W8_CHECK_ARG(x.sink + x.recent <= x.budget, "sink + recent (%lld) exceed the budget %lld",
               (long long)(x.sink + x.recent), (long long)x.budget);
  W8_CHECK_ARG(x.batch * x.kv_heads <= 65535, "batch * kv_heads beyond 65535");
  if (x.batch == 0) return W8_OK;
  W8_CHECK_ARG(x.lens && x.lens_out, "null lens");
  W8_CHECK_ARG(!arrays_meet(x.lens, x.batch, x.lens_out, x.batch), "lens_out must not be lens nor overlap it");
  if (x.slots > 0) {
    W8_CHECK_ARG(x.weights && x.positions && x.weights_out && x.positions_out, "null weights or positions");
    // In place only with the same layout: rows of one would be other rows of the other.
    auto same = [&](const int64_t* p, const int64_t* q) {
      return (x.batch == 1 || p[0] == q[0]) && (x.kv_heads == 1 || p[1] == q[1]);
    };
    W8_CHECK_ARG(x.weights != x.weights_out || same(x.weights_stride, x.weights_out_stride),
                 "weights_out is weights with other strides");
    W8_CHECK_ARG(x.positions != x.positions_out || same(x.positions_stride, x.positions_out_stride),
                 "positions_out is positions with other strides");
    if ((st = cache_rows("k", x.k, x.k_stride)) != W8_OK) return st;
    if ((st = cache_rows("v", x.v, x.v_stride)) != W8_OK) return st;
  }
  const int64_t need = w8_cache_evict_workspace_bytes(x.batch, x.kv_heads, x.slots, x.budget);
  W8_CHECK_ARG(workspace != nullptr && workspace_bytes >= need, "workspace of %lld bytes needed (got %lld)",
               (long long)need, (long long)workspace_bytes);
  int device = 0, sms = 0;
  if ((st = require_sm100(&device)) != W8_OK) return st;
  if ((st = num_sms(&sms)) != W8_OK) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int64_t rows = x.batch * x.kv_heads;
  const int64_t most = std::max<int64_t>(0, std::min(x.budget, x.slots - x.budget));
  w8::EvictArgs e = {};
  e.w = x.weights, e.pos = x.positions, e.w_out = x.weights_out, e.pos_out = x.positions_out;
  e.w_b = x.weights_stride[0], e.w_h = x.weights_stride[1];
  e.pos_b = x.positions_stride[0], e.pos_h = x.positions_stride[1];
  e.wo_b = x.weights_out_stride[0], e.wo_h = x.weights_out_stride[1];
  e.po_b = x.positions_out_stride[0], e.po_h = x.positions_out_stride[1];
  e.lens = x.lens, e.lens_out = x.lens_out;
  e.kv_heads = static_cast<int>(x.kv_heads), e.slots = static_cast<int>(x.slots);
  e.budget = static_cast<int>(std::min(x.budget, x.slots)), e.sink = static_cast<int>(x.sink);
  e.recent = static_cast<int>(x.recent);
  e.moves = static_cast<int*>(workspace), e.most = static_cast<int>(most);
  // Keys in registers, the fewest a thread that cover the row: up to 32768 slots of one CTA, up to
  // 131072 of a cluster, which takes rows above 8192 slots too while all their CTAs have an SM
  // of their own (the kernel's comment has both sides).
  e.cluster = 1;
  while (e.cluster < w8::kEvictCluster && (x.slots > (e.cluster == 1 ? 32768 : 16384 * e.cluster) ||
                                           (x.slots > 8192 && rows * e.cluster * 2 <= sms)))
    e.cluster *= 2;
  const int64_t per = (x.slots + w8::kEvictThreads * e.cluster - 1) / (w8::kEvictThreads * e.cluster);
  const dim3 each(static_cast<unsigned>(rows));
  const int lists = static_cast<int>(std::min<int64_t>(2 * (most + e.budget) + 4, 100 * 1024));
  if (e.cluster > 1)
    st = per <= 4    ? launch_evict_cluster<4>(rows, s, e)
         : per <= 8  ? launch_evict_cluster<8>(rows, s, e)
         : per <= 16 ? launch_evict_cluster<16>(rows, s, e)
         : per <= 32 ? launch_evict_cluster<32>(rows, s, e)
                     : launch_cache(w8::evict_select_long_kernel, each, w8::kEvictLongThreads, s, e);
  else
    st = per <= 8    ? launch_evict<8>(each, lists, device, s, e)
         : per <= 16 ? launch_evict<16>(each, lists, device, s, e)
         : per <= 32 ? launch_evict<32>(each, lists, device, s, e)
                     : launch_evict<64>(each, lists, device, s, e);
  if (st != W8_OK || most == 0) return st;
  w8::MoveArgs m = {};
  m.k = static_cast<uint8_t*>(x.k), m.v = static_cast<uint8_t*>(x.v);
  m.k_b = x.k_stride[0], m.k_h = x.k_stride[1], m.k_s = x.k_stride[2];
  m.v_b = x.v_stride[0], m.v_h = x.v_stride[1], m.v_s = x.v_stride[2];
  m.moves = e.moves, m.most = e.most, m.kv_heads = e.kv_heads, m.chunks = static_cast<int>(x.row_bytes / 16);
  m.shift = (m.chunks & (m.chunks - 1)) == 0 ? __builtin_ctz(m.chunks) : -1;
  const int64_t blocks = (most * 2 * m.chunks + 256 * w8::kMoveChunks - 1) / (256 * w8::kMoveChunks);
  const int64_t per_row = std::max<int64_t>(1, std::min(blocks, (static_cast<int64_t>(sms) * 16 + rows - 1) / rows));
  return launch_cache(w8::evict_move_kernel, dim3(static_cast<unsigned>(per_row), static_cast<unsigned>(rows)), 256, s, m);
}

extern "C" int w8_cache_reorder(void* const* tensors, int64_t count, const int64_t* strides, const void* beam,
                                int beam_i64, const int32_t* lens, int64_t groups, int64_t beams, int64_t heads,
                                int64_t slots, int64_t row_bytes, w8_stream_t stream) {
  using namespace w8host;
  int st = cache_shape(groups, heads, slots, row_bytes);
  if (st != W8_OK) return st;
  W8_CHECK_ARG(count >= 0 && beams >= 1, "negative size");
  W8_CHECK_ARG(groups * heads <= 65535, "groups * heads beyond 65535");
  if (beams > 32) {
    set_error("%lld beams: at most 32", (long long)beams);
    return W8_ERR_UNSUPPORTED;
  }
  if (count == 0 || groups == 0 || slots == 0) return W8_OK;
  W8_CHECK_ARG(tensors && strides && beam, "null pointer");
  for (int64_t i = 0; i < count; ++i)
    if ((st = cache_rows("a cache", tensors[i], strides)) != W8_OK) return st;
  int device = 0;
  if ((st = require_sm100(&device)) != W8_OK) return st;
  w8::ReorderArgs a = {};
  a.x_r = strides[0], a.x_h = strides[1], a.x_s = strides[2];
  a.beam = beam, a.beam_i64 = beam_i64, a.lens = lens;
  a.k = static_cast<int>(beams), a.heads = static_cast<int>(heads), a.slots = static_cast<int>(slots);
  a.chunks = static_cast<int>(row_bytes / 16);
  const int64_t blocks = (slots * a.chunks + 255) / 256;
  W8_CHECK_ARG(blocks < (1ll << 31), "too many slots");
  for (int64_t i = 0; i < count; i += w8::kReorderTensors) {
    const int64_t n = std::min<int64_t>(count - i, w8::kReorderTensors);
    for (int64_t j = 0; j < n; ++j) a.x[j] = static_cast<uint8_t*>(tensors[i + j]);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(groups * heads), static_cast<unsigned>(n));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (beams <= 4)
      st = launch_cache(w8::cache_reorder_kernel<4>, grid, 256, s, a);
    else if (beams <= 8)
      st = launch_cache(w8::cache_reorder_kernel<8>, grid, 256, s, a);
    else if (beams <= 16)
      st = launch_cache(w8::cache_reorder_kernel<16>, grid, 256, s, a);
    else
      st = launch_cache(w8::cache_reorder_kernel<32>, grid, 256, s, a);
    if (st != W8_OK) return st;
  }
  return W8_OK;
}
