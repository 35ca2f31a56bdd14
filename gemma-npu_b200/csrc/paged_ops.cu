// What keeps a paged 8-bit cache: giving out its pages and appending to it.  The reference grows
// a DynamicCache by concatenation (pipeline.py:318-339).
//
// How many pages a sequence needs follows from its length, which after speculative decoding only
// the device knows, so the page tables and the stack of free pages live there too.
//
// A page becomes 8 bits when its last position is appended, all of it at once and from the
// 16-bit rows themselves: one rounding a value, whatever the order in which the rows came.  Until
// then they wait in the sequence's tail, which the attention reads as it is.  Indexes come from
// device memory; one outside its range is recorded in the device status: a length's or a page's is
// skipped, a path's puts a row of zeros into the cache, which counts.
#include "common.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace w8 {

static __device__ int g_paged_status = 0;

__device__ __forceinline__ void paged_bad_index() { atomicExch(&g_paged_status, W8_ERR_INVALID_ARG); }

// ---------------------------------------------------------------- append
struct PagedAppendArgs {
  int8_t* page[2];         // K, V: [pages, KV, P] rows of D bytes
  float* scale[2];         // [pages, KV]
  uint16_t* tail[2];       // [B, KV, P] rows
  const uint16_t* fresh[2];  // [B, KV, N] rows
  int64_t page_p[2], page_h[2], page_r[2], scale_p[2], scale_h[2];
  int64_t tail_b[2], tail_h[2], tail_r[2], new_b[2], new_h[2], new_r[2];
  const int* table;
  int64_t table_b;
  const int* lens;
  const int* path;   // [B, steps] or null: the new tokens in order
  const int* count;  // [B] or null: all
  int64_t path_b;
  int* lens_out;
  int table_pages, pages, shift, kv_heads, n, steps, chunk_shift;  // 1 << chunk_shift 16-byte chunks a row
};

constexpr int kPageThreads = 1024;  // at most, with 4 16-byte chunks each, 8 for a page of 128 rows of 512 values

template <typename T>
__device__ __forceinline__ float paged_f32(uint32_t bits);
template <>
__device__ __forceinline__ float paged_f32<__nv_bfloat16>(uint32_t bits) { return __uint_as_float(bits << 16); }
template <>
__device__ __forceinline__ float paged_f32<__half>(uint32_t bits) {
  return __half2float(__ushort_as_half(static_cast<uint16_t>(bits)));
}

// The larger magnitude of each half of two pairs, a NaN above all (one instruction; the maxima of 16-bit
// integers are made of ten).
template <typename T>
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t larger2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <>
__device__ __forceinline__ uint32_t larger2<__half>(uint32_t a, uint32_t b) {
  const __half2 m = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

// round(127 x / m) to nearest even, |x| <= m.  127 x is exact in fp32 (7 more bits than x's 8 or
// 11), and so is which side of a half the quotient lies on: it differs from a half by at least
// 2^-2 over m's 8 or 11 bits where the quotient is in [64, 128), by 2^-10 over them in
// [1/4, 1), relative to it 2^-20 or more, so that the quotient rounded to fp32 never becomes
// a half that it was not.
__device__ __forceinline__ uint32_t paged_divide(float x, float m) {
  return static_cast<uint32_t>(static_cast<int>(rintf(__fdiv_rn(x * 127.f, m)))) & 0xFFu;
}
// Eight such bytes.  A product with the reciprocal (off by less than 127 2^-22) decides all but what is
// near a half; adding 1.5 2^23 leaves the integer in the sum's low bits, without a conversion
// (those and the rounding instruction have an eighth of an addition's rate: 47 us with them where
// this takes 31).
__device__ __forceinline__ uint2 paged_round8(const float (&x)[8], float m, float r, bool slow) {
  constexpr float kBig = 12582912.f;
  float far = 0.f;
  uint32_t bits[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = __fmul_rn(x[i], r), q = __fadd_rn(t, kBig);
    bits[i] = __float_as_uint(q);
    far = fmaxf(far, fabsf(__fsub_rn(t, __fsub_rn(q, kBig))));
  }
  if (far > 0.4999f || slow) {
#pragma unroll
    for (int i = 0; i < 8; ++i) bits[i] = paged_divide(x[i], m);
  }
  auto four = [&](int i) {
    return __byte_perm(__byte_perm(bits[i], bits[i + 1], 0x0040), __byte_perm(bits[i + 2], bits[i + 3], 0x0040), 0x5410);
  };
  return make_uint2(four(0), four(4));
}

// One CTA: K or V of one cache head of one sequence, and the page that is `blockIdx.y` behind the
// first partial one: filled from the tail (the first page only) and the new rows, its largest
// magnitude found and its values rounded from the registers, if the call fills it.  CTA 0 then
// writes the rows that stay in the tail, which are all new: the tail's old rows, if the page was
// filled, are read before.  Bound by the issue of its arithmetic for prompts (some 20 instructions a value of 2
// bytes read and 1 written: 4 prompts of 2500 to 4000 tokens, 8 heads of 128, take 31 us where the
// bytes alone would take 12) and by the chain length, table, row for a token (3.1 us for 8 sequences).
template <typename T, int kVecs>
__global__ void __launch_bounds__(kPageThreads) paged_append_kernel(const PagedAppendArgs a) {
  __shared__ int sm_took;
  __shared__ uint32_t sm_max[32];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int kv = blockIdx.x & 1, bc = blockIdx.x >> 1, b = bc / a.kv_heads, c = bc % a.kv_heads;
  const int page_rows = 1 << a.shift, j = blockIdx.y;
  pdl_launch_dependents();
  pdl_wait();
  const int len = a.lens[b];
  const int given = a.count != nullptr ? a.count[b] : a.steps;
  const int room = a.table_pages << a.shift;
  const bool first = j == 0 && c == 0 && kv == 0 && tid == 0;
  if (len < 0 || len > room) {
    if (first) paged_bad_index(), a.lens_out[b] = len;
    return;
  }
  int took = given;
  if (took < 0 || took > a.steps) {
    if (first) paged_bad_index();
    took = took < 0 ? 0 : a.steps;
  }
  const int* path = a.path != nullptr ? a.path + b * a.path_b : nullptr;
  if (path != nullptr) {  // entries before the first negative one
    if (tid == 0) sm_took = took;
    __syncthreads();
    int end = took;
    for (int e = tid; e < took; e += threads)
      if (path[e] < 0) {
        end = e;
        break;
      }
    if (end < took) atomicMin(&sm_took, end);
    __syncthreads();
    took = sm_took;
  }
  if (took > room - len) {
    if (first) paged_bad_index();
    took = room - len;
  }
  if (first) a.lens_out[b] = len + took;
  const int off = len & (page_rows - 1), total = off + took;  // rows from the first partial page on
  const int full = total >> a.shift;                          // pages that the call fills
  if (j > 0 && j >= full) return;
  // Row `at` of those: the tail's, or the new token's that the path names (null: out of range).
  const uint16_t* fresh = a.fresh[kv] + b * a.new_b[kv] + c * a.new_h[kv];
  uint16_t* tail = a.tail[kv] + b * a.tail_b[kv] + c * a.tail_h[kv];
  auto new_row = [&](int at) -> const uint16_t* {
    int i = at - off;
    if (path != nullptr) i = path[i];
    if (i >= a.n) {
      paged_bad_index();
      return nullptr;
    }
    return fresh + i * a.new_r[kv];
  };
  if (j < full) {
    const int entry = a.table[b * a.table_b + (len >> a.shift) + j];  // (looked at when the rows have come)
    // This thread's chunk of every (threads / chunks)-th row: addresses by steps.
    const int vecs = page_rows << a.chunk_shift, ch = tid & ((1 << a.chunk_shift) - 1), r0 = tid >> a.chunk_shift;
    const int step = threads >> a.chunk_shift, at0 = (j << a.shift) + r0;
    uint4 x[kVecs];
    uint32_t most = 0;  // the largest magnitudes, two at a time
    const uint16_t* in_tail = tail + at0 * a.tail_r[kv] + ch * 8;
    const uint16_t* in_new = fresh + (at0 - off) * a.new_r[kv] + ch * 8;
    const int64_t tail_step = step * a.tail_r[kv], new_step = step * a.new_r[kv];
#pragma unroll
    for (int i = 0; i < kVecs; ++i, in_tail += tail_step, in_new += new_step) {
      x[i] = make_uint4(0, 0, 0, 0);
      if (tid + i * threads >= vecs) continue;
      const int at = at0 + i * step;
      const uint16_t* row = in_tail;
      if (at >= off) {
        row = in_new;
        if (path != nullptr) {
          row = new_row(at);
          if (row != nullptr) row += ch * 8;
        }
      }
      if (row != nullptr) x[i] = *reinterpret_cast<const uint4*>(row);
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      most = larger2<T>(most, larger2<T>(larger2<T>(x[i].x & 0x7FFF7FFFu, x[i].y & 0x7FFF7FFFu),
                                         larger2<T>(x[i].z & 0x7FFF7FFFu, x[i].w & 0x7FFF7FFFu)));
    }
    most = __reduce_max_sync(0xffffffffu, max(most & 0xFFFFu, most >> 16));
    if ((tid & 31) == 0) sm_max[tid >> 5] = most;
    __syncthreads();  // (the tail's old rows have been read)
    for (int w = 0; w < threads / 32; ++w) most = max(most, sm_max[w]);
    constexpr uint32_t kInf = __is_same(T, __half) ? 0x7C00u : 0x7F80u;
    const bool finite = most < kInf;
    float m = paged_f32<T>(most);
    const float scale = finite ? __fdiv_rn(m, 127.f) : __uint_as_float(0x7FC00000u);
    // (values from 2^100 on are scaled by 2^-20, exactly where it matters: 127 x must not overflow)
    const float down = m > 0x1p100f ? 0x1p-20f : 1.f;
    m *= down;
    const float r = finite && m > 0.f ? 127.f / m : 0.f;
    // (magnitudes so small that 127 / m overflows are divided one by one)
    const bool slow = finite && m > 0.f && !(r < 0x1p120f);
    const int page = entry >= 0 && entry < a.pages ? entry : -1;
    if (page < 0 && tid == 0) paged_bad_index();
    if (page >= 0) {
      if (tid == 0) a.scale[kv][page * a.scale_p[kv] + c * a.scale_h[kv]] = scale;
      int8_t* dst = a.page[kv] + page * a.page_p[kv] + c * a.page_h[kv] + r0 * a.page_r[kv] + ch * 8;
      const int64_t dst_step = step * a.page_r[kv];
#pragma unroll
      for (int i = 0; i < kVecs; ++i, dst += dst_step) {
        if (tid + i * threads >= vecs) break;
        const uint32_t ws[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint2 out = make_uint2(0, 0);
        if (finite && m > 0.f) {
          float v[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = paged_f32<T>((ws[q >> 1] >> (16 * (q & 1))) & 0xFFFFu);
          if (down != 1.f) {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] *= down;
          }
          out = paged_round8(v, m, r, slow);
        }
        *reinterpret_cast<uint2*>(dst) = out;
      }
    }
  }
  if (j > 0) return;
  // What stays behind the last full page.
  const int from = full > 0 ? full << a.shift : off, rows = total - from;
  const int to = full > 0 ? 0 : off;
  for (int e = tid; e < rows << a.chunk_shift; e += threads) {
    const int r = e >> a.chunk_shift, ch = e & ((1 << a.chunk_shift) - 1);
    const uint16_t* row = new_row(from + r);
    const uint4 w = row != nullptr ? *reinterpret_cast<const uint4*>(row + ch * 8) : make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(tail + (to + r) * a.tail_r[kv] + ch * 8) = w;
  }
}

// ---------------------------------------------------------------- pages given out and taken back
struct AssignArgs {
  int* table;
  int64_t table_b;
  const int* lens;
  const uint8_t* active;
  int* free;
  int* top;
  uint8_t* ok;
  int batch, width, free_size, shift, room, window, sink;
  int wide;  // rows of the table load as 16-byte vectors
  int4* counts;  // [batch] of a large table, counted by a kernel of its own; or null
};

constexpr int kAssignThreads = 512;
constexpr int kAssignWarps = kAssignThreads / 32;
constexpr int kAssignRequests = 1024;  // of a CTA
constexpr int kAssignCluster = 8;      // CTAs at most (portable)

struct AssignRow {
  int need, dead, sinks;  // pages [0, need) but not [sinks, dead) are wanted
  bool valid, fits;
  __device__ __forceinline__ bool want(int i) const { return i < need && (i >= dead || i < sinks); }
};
__device__ __forceinline__ AssignRow assign_row(const AssignArgs& a, int b) {
  AssignRow r;
  const int64_t len = a.lens[b];
  r.valid = len >= 0 && len <= static_cast<int64_t>(a.width) << a.shift;
  const bool live = a.active == nullptr || a.active[b] != 0;
  const int64_t need = live && r.valid ? (len + a.room + (1 << a.shift) - 1) >> a.shift : 0;
  r.fits = need <= a.width;
  r.need = r.fits ? static_cast<int>(need) : a.width;
  const int64_t seen = len + 1 - a.window;  // the first position that the next token sees
  r.dead = a.window > 0 && seen > 0 ? static_cast<int>(seen >> a.shift) : 0;
  r.sinks = static_cast<int>((static_cast<int64_t>(a.sink) + (1 << a.shift) - 1) >> a.shift);
  return r;
}

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// What a warp finds in request b's table: entries that go back, missing ones, and the range [lo, hi) of
// both, in every lane.
__device__ __forceinline__ int4 assign_count(const AssignArgs& a, int b) {
  const int lane = threadIdx.x & 31;
  const AssignRow r = assign_row(a, b);
  const int* row = a.table + b * a.table_b;
  int nb = 0, nm = 0, first = a.width, last = 0;
  auto see = [&](int i, int v) {
    const bool want = r.want(i);
    const bool bk = v >= 0 && !want, ms = v < 0 && want && r.fits;
    nb += bk, nm += ms;
    if (bk || ms) first = min(first, i), last = i + 1;
  };
  if (r.valid) {
    int i = 0;
    if (a.wide) {
      const int4* row4 = reinterpret_cast<const int4*>(row);
      const int n4 = a.width >> 2;
      for (int v0 = lane; v0 < n4; v0 += 32 * 8) {
        int4 x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = v0 + 32 * u < n4 ? row4[v0 + 32 * u] : make_int4(-1, -1, -1, -1);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (v0 + 32 * u < n4) {
            const int at = 4 * (v0 + 32 * u);
            see(at, x[u].x), see(at + 1, x[u].y), see(at + 2, x[u].z), see(at + 3, x[u].w);
          }
      }
      i = n4 * 4;
    }
    for (i += lane; i < a.width; i += 32) see(i, row[i]);
  } else if (lane == 0) {
    paged_bad_index();
  }
  nb = __reduce_add_sync(0xffffffffu, nb);
  nm = __reduce_add_sync(0xffffffffu, nm);
  first = __reduce_min_sync(0xffffffffu, first);
  last = __reduce_max_sync(0xffffffffu, last);
  return make_int4(nb, nm, first, last);
}

constexpr int kCountWarps = 4;
__global__ void __launch_bounds__(32 * kCountWarps) page_count_kernel(const AssignArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x * kCountWarps + (threadIdx.x >> 5);
  if (b >= a.batch) return;
  const int4 c = assign_count(a, b);
  if ((threadIdx.x & 31) == 0) a.counts[b] = c;
}

// One cluster for the whole table, each CTA a contiguous range of requests, a warp a request.
// What goes back and what is missing is counted (of more than 16384 entries by page_count_kernel on
// all SMs: for 512 tables of 2048 a call takes 13 us where this cluster alone took 25), prefix sums (over a
// CTA's requests, then the cluster's CTAs) give every request its place in the stack, and a
// second pass, over the entries between a request's first and last change only, moves the pages:
// first all that go back, then, behind a barrier of the cluster, those that are given out.
__global__ void __launch_bounds__(kAssignThreads) page_assign_kernel(const AssignArgs a) {
  __shared__ int back[kAssignRequests], miss[kAssignRequests];        // counts, then what comes before
  __shared__ int lo[kAssignRequests], hi[kAssignRequests];            // a request's changes lie in [lo, hi)
  __shared__ unsigned long long sums[2][kAssignCluster];              // every CTA's counts (back << 32 | missing), then given
  __shared__ int scan[2][kAssignWarps];
  __shared__ int given;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t ranks;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  const int rank = static_cast<int>(cluster_ctarank());
  const int b0 = static_cast<int>(static_cast<int64_t>(a.batch) * rank / ranks);
  const int b1 = static_cast<int>(static_cast<int64_t>(a.batch) * (rank + 1) / ranks);
  const int count = b1 - b0;
  if (tid == 0) given = 0;
  pdl_launch_dependents();
  cluster_sync();  // every CTA has started: its shared memory may be written
  pdl_wait();
  const int top0 = *a.top;
  const bool bad_top = top0 < 0 || top0 > a.free_size;
  const int top = bad_top ? (top0 < 0 ? 0 : a.free_size) : top0;
  if (bad_top && rank == 0 && tid == 0) paged_bad_index();
  if (a.counts != nullptr) {
    for (int q = tid; q < count; q += kAssignThreads) {
      const int4 c = a.counts[b0 + q];
      back[q] = c.x, miss[q] = c.y, lo[q] = c.z, hi[q] = c.w;
    }
  } else {
    for (int q = warp; q < count; q += kAssignWarps) {
      const int4 c = assign_count(a, b0 + q);
      if (lane == 0) back[q] = c.x, miss[q] = c.y, lo[q] = c.z, hi[q] = c.w;
    }
  }
  __syncthreads();
  // Exclusive prefix sums over the CTA's requests (each thread a run of them).
  const int run = (count + kAssignThreads - 1) / kAssignThreads;
  const int q0 = min(tid * run, count), q1 = min(q0 + run, count);
  int sb = 0, sm = 0;
  for (int q = q0; q < q1; ++q) sb += back[q], sm += miss[q];
  int xb = sb, xm = sm;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int yb = __shfl_up_sync(0xffffffffu, xb, d), ym = __shfl_up_sync(0xffffffffu, xm, d);
    if (lane >= d) xb += yb, xm += ym;
  }
  if (lane == 31) scan[0][warp] = xb, scan[1][warp] = xm;
  __syncthreads();
  int tb = 0, tm = 0;
  xb -= sb, xm -= sm;
  for (int w = 0; w < kAssignWarps; ++w) {
    if (w < warp) xb += scan[0][w], xm += scan[1][w];
    tb += scan[0][w], tm += scan[1][w];
  }
  if (tid < static_cast<int>(ranks))
    st_cluster_u64(mapa_shared(smem_u32(&sums[0][rank]), tid),
                   static_cast<unsigned long long>(static_cast<uint32_t>(tb)) << 32 | static_cast<uint32_t>(tm));
  cluster_sync();
  int all_back = 0;
  for (int k = 0; k < static_cast<int>(ranks); ++k) {
    const int kb = static_cast<int>(sums[0][k] >> 32), km = static_cast<int>(sums[0][k] & 0xFFFFFFFFu);
    if (k < rank) xb += kb, xm += km;
    all_back += kb;
  }
  for (int q = q0; q < q1; ++q) {
    const int nb = back[q], nm = miss[q];
    back[q] = xb, miss[q] = xm;
    xb += nb, xm += nm;
    if (nb == 0 && nm == 0) hi[q] = lo[q] = 0;
  }
  __syncthreads();
  // The places of request q's pages end where the next request's begin.
  const int before_b = back[0], before_m = miss[0];
  const int end_b = before_b + tb, end_m = before_m + tm;
  auto backs = [&](int q) { return (q + 1 < count ? back[q + 1] : end_b) - back[q]; };
  auto misses = [&](int q) { return (q + 1 < count ? miss[q + 1] : end_m) - miss[q]; };
  for (int q = warp; q < count; q += kAssignWarps) {
    if (backs(q) == 0) continue;
    const AssignRow r = assign_row(a, b0 + q);
    int* row = a.table + (b0 + q) * a.table_b;
    int at = top + back[q];
    for (int i0 = lo[q]; i0 < hi[q]; i0 += 32) {
      const int i = i0 + lane, v = i < hi[q] ? row[i] : -1;
      const bool bk = v >= 0 && !r.want(i);
      const uint32_t lanes = __ballot_sync(0xffffffffu, bk);
      if (bk) {
        const int to = at + __popc(lanes & ((1u << lane) - 1u));
        if (to < a.free_size)
          a.free[to] = v;
        else
          paged_bad_index();  // (more pages than the stack was made for)
        row[i] = -1;
      }
      at += __popc(lanes);
    }
  }
  cluster_sync();
  const int have = min(static_cast<int64_t>(top) + all_back, static_cast<int64_t>(a.free_size));
  int mine = 0;
  for (int q = warp; q < count; q += kAssignWarps) {
    const AssignRow r = assign_row(a, b0 + q);
    const int nm = misses(q);
    const bool ok = r.valid && r.fits && (nm == 0 || miss[q] + nm <= have);
    if (lane == 0) a.ok[b0 + q] = ok;
    if (!ok || nm == 0) continue;
    mine += nm;
    int* row = a.table + (b0 + q) * a.table_b;
    int at = have - 1 - miss[q];
    for (int i0 = lo[q]; i0 < hi[q]; i0 += 32) {
      const int i = i0 + lane, v = i < hi[q] ? row[i] : 0;
      const bool ms = v < 0 && r.want(i);
      const uint32_t lanes = __ballot_sync(0xffffffffu, ms);
      if (ms) row[i] = a.free[at - __popc(lanes & ((1u << lane) - 1u))];
      at -= __popc(lanes);
    }
  }
  if (lane == 0 && mine > 0) atomicAdd(&given, mine);
  __syncthreads();
  if (tid == 0) st_cluster_u64(mapa_shared(smem_u32(&sums[1][rank]), 0), static_cast<unsigned long long>(given));
  cluster_sync();
  if (rank == 0 && tid == 0) {
    int left = have;
    for (int k = 0; k < static_cast<int>(ranks); ++k) left -= static_cast<int>(sums[1][k]);
    *a.top = left;
  }
}

}  // namespace w8

namespace w8host {

int require_sm100(int* device);

// Read (and optionally clear) the sticky device status of the paged cache's operations.
int paged_ops_device_status(int clear, int* out) {
  W8_CUDA_TRY(cudaMemcpyFromSymbol(out, w8::g_paged_status, sizeof(int)));
  if (clear) {
    const int zero = 0;
    W8_CUDA_TRY(cudaMemcpyToSymbol(w8::g_paged_status, &zero, sizeof(int)));
  }
  return W8_OK;
}

static int page_shift(int64_t page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }

template <typename Kern, typename Args>
static int launch_paged(Kern kern, dim3 grid, int threads, int cluster, cudaStream_t stream, const Args& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, a));
}

}  // namespace w8host

extern "C" int w8_paged_append(const w8_paged_append_args* in, w8_stream_t stream) {
  using namespace w8host;
  W8_CHECK_ARG(in != nullptr, "null arguments");
  const w8_paged_append_args& x = *in;
  W8_CHECK_ARG(x.batch >= 0 && x.kv_heads >= 1 && x.pages >= 0 && x.table_pages >= 0 && x.n_new >= 0 && x.steps >= 0,
               "negative size");
  const int shift = page_shift(x.page);
  if (shift < 0) {
    set_error("pages of %lld tokens are not of 16, 32, 64 or 128", (long long)x.page);
    return W8_ERR_UNSUPPORTED;
  }
  if (x.head_dim != 64 && x.head_dim != 128 && x.head_dim != 256 && x.head_dim != 512) {
    set_error("head_dim %lld is not 64, 128, 256 or 512", (long long)x.head_dim);
    return W8_ERR_UNSUPPORTED;
  }
  W8_CHECK_ARG(x.dtype == W8_BF16 || x.dtype == W8_FP16, "dtype must be W8_BF16 or W8_FP16");
  W8_CHECK_ARG(x.table_pages < (1ll << 30) / x.page && x.pages < (1ll << 31) && x.n_new < (1ll << 30) &&
                   x.steps < (1ll << 20) && x.batch * x.kv_heads < (1ll << 30),
               "size beyond the limits");
  W8_CHECK_ARG(x.path != nullptr || x.steps == x.n_new, "without a path the steps are the new tokens");
  if (x.batch == 0) return W8_OK;
  W8_CHECK_ARG(x.lens && x.lens_out && x.k_tail && x.v_tail && (x.n_new == 0 || (x.k_new && x.v_new)), "null pointer");
  W8_CHECK_ARG(!arrays_meet(x.lens, x.batch, x.lens_out, x.batch), "lens_out must not be lens nor overlap it");
  W8_CHECK_ARG(!arrays_meet(x.count, x.batch, x.lens_out, x.batch), "lens_out must not be count nor overlap it");
  if (x.path && x.steps > 0 && arrays_meet(x.path, (x.batch - 1) * x.path_stride + x.steps, x.lens_out, x.batch))
    for (int64_t b = 0; b < x.batch; ++b)  // (it may lie between the rows)
      W8_CHECK_ARG(!arrays_meet(x.path + b * x.path_stride, x.steps, x.lens_out, x.batch), "lens_out must not overlap path");
  W8_CHECK_ARG(x.pages == 0 || (x.k && x.v && x.k_scale && x.v_scale), "null pages");
  W8_CHECK_ARG(x.table_pages == 0 || x.table, "null table");
  if (x.table_pages > 0 && arrays_meet(x.table, (x.batch - 1) * x.table_stride + x.table_pages, x.lens_out, x.batch))
    for (int64_t b = 0; b < x.batch; ++b)  // (it may lie between the rows)
      W8_CHECK_ARG(!arrays_meet(x.table + b * x.table_stride, x.table_pages, x.lens_out, x.batch),
                   "lens_out must not overlap table");
  const void* ptrs[6] = {x.k_tail, x.v_tail, x.k_new, x.v_new, x.k, x.v};
  const int64_t* strides[6] = {x.k_tail_stride, x.v_tail_stride, x.k_new_stride, x.v_new_stride, x.k_stride, x.v_stride};
  const int64_t sizes[6][3] = {{x.batch, x.kv_heads, x.page},  {x.batch, x.kv_heads, x.page},
                               {x.batch, x.kv_heads, x.n_new}, {x.batch, x.kv_heads, x.n_new},
                               {x.pages, x.kv_heads, x.page},  {x.pages, x.kv_heads, x.page}};
  for (int i = 0; i < 6; ++i) {
    W8_CHECK_ALIGN(aligned(ptrs[i], 16), "pages, tails, k_new and v_new must be 16-byte aligned");
    for (int j = 0; j < 3; ++j)
      W8_CHECK_ALIGN(sizes[i][j] <= 1 || strides[i][j] % (i < 4 ? 8 : 16) == 0,
                     "the strides of tails, k_new and v_new must be multiples of 8, of pages of 16");
  }
  int device = 0;
  const int st = require_sm100(&device);
  if (st != W8_OK) return st;
  w8::PagedAppendArgs a = {};
  int8_t* pages[2] = {x.k, x.v};
  float* scales[2] = {x.k_scale, x.v_scale};
  void* tails[2] = {x.k_tail, x.v_tail};
  const void* fresh[2] = {x.k_new, x.v_new};
  const int64_t* ps[2] = {x.k_stride, x.v_stride};
  const int64_t* ss[2] = {x.k_scale_stride, x.v_scale_stride};
  const int64_t* ts[2] = {x.k_tail_stride, x.v_tail_stride};
  const int64_t* ns[2] = {x.k_new_stride, x.v_new_stride};
  for (int i = 0; i < 2; ++i) {
    a.page[i] = pages[i];
    a.scale[i] = scales[i];
    a.tail[i] = static_cast<uint16_t*>(tails[i]);
    a.fresh[i] = static_cast<const uint16_t*>(fresh[i]);
    a.page_p[i] = ps[i][0], a.page_h[i] = ps[i][1], a.page_r[i] = ps[i][2];
    a.scale_p[i] = ss[i][0], a.scale_h[i] = ss[i][1];
    a.tail_b[i] = ts[i][0], a.tail_h[i] = ts[i][1], a.tail_r[i] = ts[i][2];
    a.new_b[i] = ns[i][0], a.new_h[i] = ns[i][1], a.new_r[i] = ns[i][2];
  }
  a.table = x.table;
  a.table_b = x.table_stride;
  a.lens = x.lens;
  a.path = x.path;
  a.count = x.count;
  a.path_b = x.path_stride;
  a.lens_out = x.lens_out;
  a.table_pages = static_cast<int>(x.table_pages);
  a.pages = static_cast<int>(x.pages);
  a.shift = shift;
  a.kv_heads = static_cast<int>(x.kv_heads);
  a.n = static_cast<int>(x.n_new);
  a.steps = static_cast<int>(x.steps);
  a.chunk_shift = x.head_dim == 64 ? 3 : x.head_dim == 128 ? 4 : x.head_dim == 256 ? 5 : 6;
  // Pages that the call can fill (one CTA writes the tail even if none).
  const int64_t most = std::max<int64_t>(1, (x.page - 1 + x.steps) >> shift);
  W8_CHECK_ARG(most <= 65535, "too many new tokens");
  const int64_t vecs = x.page * x.head_dim / 8;
  const int threads = static_cast<int>(std::min<int64_t>(w8::kPageThreads, std::max<int64_t>(64, vecs / 4)));
  const dim3 grid(static_cast<unsigned>(2 * x.batch * x.kv_heads), static_cast<unsigned>(most));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  using B = __nv_bfloat16;
  if (vecs <= 4 * threads)
    return x.dtype == W8_BF16 ? launch_paged(w8::paged_append_kernel<B, 4>, grid, threads, 0, s, a)
                              : launch_paged(w8::paged_append_kernel<__half, 4>, grid, threads, 0, s, a);
  return x.dtype == W8_BF16 ? launch_paged(w8::paged_append_kernel<B, 8>, grid, threads, 0, s, a)
                            : launch_paged(w8::paged_append_kernel<__half, 8>, grid, threads, 0, s, a);
}

extern "C" int64_t w8_page_assign_workspace_bytes(int64_t batch, int64_t table_pages) {
  return batch > 0 && table_pages > 0 && batch * table_pages > 16384 ? batch * 16 : 0;
}

extern "C" int w8_page_assign(const w8_page_assign_args* in, void* workspace, int64_t workspace_bytes,
                              w8_stream_t stream) {
  using namespace w8host;
  W8_CHECK_ARG(in != nullptr, "null arguments");
  const w8_page_assign_args& x = *in;
  W8_CHECK_ARG(x.batch >= 0 && x.table_pages >= 0 && x.free_pages >= 0 && x.room >= 0, "negative size");
  W8_CHECK_ARG(x.window >= 0 && x.window < (1ll << 31), "window must be 0 (none) or positive, below 2^31");
  W8_CHECK_ARG(x.sink >= 0 && x.sink < (1ll << 30), "sink must not be negative, and below 2^30");
  W8_CHECK_ARG(x.sink == 0 || x.window > 0, "sinks go with a window");
  const int shift = page_shift(x.page);
  if (shift < 0) {
    set_error("pages of %lld tokens are not of 16, 32, 64 or 128", (long long)x.page);
    return W8_ERR_UNSUPPORTED;
  }
  constexpr int64_t kMost = static_cast<int64_t>(w8::kAssignRequests) * w8::kAssignCluster;
  W8_CHECK_ARG(x.batch <= kMost, "more than %lld requests", (long long)kMost);
  W8_CHECK_ARG(x.table_pages < (1ll << 30) / x.page && x.room < (1ll << 30) && x.free_pages < (1ll << 30) &&
                   x.batch * x.table_pages < (1ll << 30),
               "size beyond the limits");
  if (x.batch == 0) return W8_OK;
  W8_CHECK_ARG(x.lens && x.top && x.ok && (x.free_pages == 0 || x.free) && (x.table_pages == 0 || x.table), "null pointer");
  W8_CHECK_ARG(x.table_pages == 0 || x.batch == 1 || x.table_stride >= x.table_pages, "the rows of the table overlap");
  W8_CHECK_ARG(!arrays_meet(x.lens, x.batch, x.top, 1) && !arrays_meet(x.lens, x.batch, x.free, x.free_pages) &&
                   !arrays_meet(x.free, x.free_pages, x.top, 1),
               "lens, free and top must not overlap");
  auto on_table = [&](int64_t row, int64_t n) {
    const int32_t* at = x.table + row * x.table_stride;
    return arrays_meet(at, n, x.lens, x.batch) || arrays_meet(at, n, x.top, 1) || arrays_meet(at, n, x.free, x.free_pages);
  };
  if (x.table_pages > 0 && on_table(0, (x.batch - 1) * x.table_stride + x.table_pages))
    for (int64_t b = 0; b < x.batch; ++b)  // (they may lie between the rows)
      W8_CHECK_ARG(!on_table(b, x.table_pages), "the table must not overlap lens, free and top");
  const int64_t need = w8_page_assign_workspace_bytes(x.batch, x.table_pages);
  W8_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace of %lld bytes needed (got %lld)",
               (long long)need, (long long)workspace_bytes);
  W8_CHECK_ALIGN(aligned(workspace, 16), "workspace must be 16-byte aligned");
  int device = 0;
  const int st = require_sm100(&device);
  if (st != W8_OK) return st;
  w8::AssignArgs a = {};
  a.table = x.table;
  a.table_b = x.table_stride;
  a.lens = x.lens;
  a.active = x.active;
  a.free = x.free;
  a.top = x.top;
  a.ok = x.ok;
  a.batch = static_cast<int>(x.batch);
  a.width = static_cast<int>(x.table_pages);
  a.free_size = static_cast<int>(x.free_pages);
  a.shift = shift;
  a.room = static_cast<int>(x.room);
  a.window = static_cast<int>(x.window);
  a.sink = static_cast<int>(x.sink);
  a.wide = aligned(x.table, 16) && (x.batch == 1 || x.table_stride % 4 == 0);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (need > 0) {
    a.counts = static_cast<int4*>(workspace);
    const int blocks = static_cast<int>((x.batch + w8::kCountWarps - 1) / w8::kCountWarps);
    const int st2 = launch_paged(w8::page_count_kernel, dim3(static_cast<unsigned>(blocks)), 32 * w8::kCountWarps, 0, s, a);
    if (st2 != W8_OK) return st2;
  }
  // CTAs of the cluster: a request a warp, and as many as the requests need.
  int cluster = 1;
  while (cluster < w8::kAssignCluster && x.batch > static_cast<int64_t>(cluster) * 2 * w8::kAssignWarps) cluster *= 2;
  return launch_paged(w8::page_assign_kernel, dim3(static_cast<unsigned>(cluster)), w8::kAssignThreads, cluster, s, a);
}
