// Beam search's selection over beams and vocabulary: the many-beam counterpart of the
// greedy token (gemma_npu.py:291), over the logits of the LM head (gemma_npu.py:170-172)
// with the final softcap (pipeline.py:335-338) fused.
//
//   total(k, t) = scores[k] + y_kt - Z_k,   y = cap tanh(l / cap) (or l),  Z_k = log sum_t e^y
// and per sequence the n largest totals over all (k, t), ties to the lower beam, then the
// lower token.  Within a beam the order of totals is the order of the logits (which is kept
// where the softcap's or a total's rounding makes different logits equal), so one pass
// over the logits yields everything: each CTA streams a chunk of one beam's logits, keeping
// a running maximum and sum of e^y per thread and the maximum of every segment of 16 logits;
// after 24 tiles a value that at least n logits reach is found from the threads' maxima, and
// only the segments that reach it are read again for candidates (value, token), of which the
// n best stay.  A second kernel merges the chunks' sorted lists per beam, forms the totals in
// 64 bits and merges the beams.
//
// The bytes are the logits once, but a logit's softcap and exponential cost more issue slots
// than its bytes: 24 x 8 beams of 262144 bf16 logits, softcapped, take 47 us, the merge's 8 among
// them (100.7 MB, 2.6 TB/s of the rest), and 43 us with 29 of the 192 finished, whose logits are not
// read; the stream with a tanh of the special-function unit, or with comparisons of every logit
// against a threshold and barriers between tiles, took 76 us.  So it still does, 71 to 76 us, where
// most segments hold a logit above the cap, with caps below 0.01 or above 1000, and with rows that
// are not 16-byte aligned (an odd vocabulary), which are loaded a logit at a time.
#include "common.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace w8 {

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamVals = 16;                              // logits per thread and tile
constexpr int kBeamTile = kBeamThreads * kBeamVals;        // logits per tile
constexpr int kBeamSuper = 24;                             // tiles between two collections
constexpr int kBeamSegs = 128;                             // segments collected at once
constexpr int kBeamCap = kBeamSegs * kBeamVals;            // candidates held in shared memory
// CTAs of the chunk kernel per SM: what its registers allow without spilling the logits held.
constexpr int beam_per_sm(size_t size) { return size == 4 ? 3 : 4; }
constexpr int kBeamMaxN = 64;
constexpr int kBeamMaxBeams = 32;
constexpr int kBeamMaxChunks = 32;

struct BeamArgs {
  const void* logits;
  int64_t l_b, l_k;
  const float* scores;      // [B, K]
  const uint8_t* finished;  // [B, K] or null
  int batch, beams, vocab, n, m;  // n: continuations per sequence, m = min(n, vocab): per beam
  int pad, chunks, chunk;   // chunk: logits per chunk (a multiple of the tile)
  float cap;
  unsigned long long* keys;  // [B * K][chunks][n]: sorted (value, token) keys of each chunk
  float2* stats;             // [B * K][chunks]: running maximum (log2 units) and sum of 2^(y - max)
  float* out_scores;
  int64_t* out_beam;
  int64_t* out_token;
  int slot_order;
};

// Order-preserving 32 bits of a value (-0 as 0); a candidate is (bits, ~token) in 64 bits, so
// that larger is better and equal values favour the lower token.
__device__ __forceinline__ uint32_t beam_bits(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float beam_value(uint32_t bits) {
  return __uint_as_float((bits & 0x80000000u) ? bits & 0x7FFFFFFFu : ~bits);
}
__device__ __forceinline__ unsigned long long beam_key(float f, int token) {
  return (static_cast<unsigned long long>(beam_bits(f)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(token));
}

// 16 bytes of logits as fp32 values (4 of fp32, 8 of the 16-bit types).
__device__ __forceinline__ void beam_unpack(const uint4& w, float* v, float) {
  v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void beam_unpack(const uint4& w, float* v, __nv_bfloat16) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(x[i] << 16);
    v[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void beam_unpack(const uint4& w, float* v, __half) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
// The type's -inf, which stands for what lies behind a chunk.
__device__ __forceinline__ void beam_fill(uint32_t* w, int i, float v) { w[i] = __float_as_uint(v); }
__device__ __forceinline__ void beam_fill(uint32_t* w, int i, __nv_bfloat16 v) {
  const uint32_t u = __bfloat16_as_ushort(v);
  w[i >> 1] = (i & 1) ? (w[i >> 1] & 0xFFFFu) | u << 16 : u;
}
__device__ __forceinline__ void beam_fill(uint32_t* w, int i, __half v) {
  const uint32_t u = __half_as_ushort(v);
  w[i >> 1] = (i & 1) ? (w[i >> 1] & 0xFFFFu) | u << 16 : u;
}
template <typename T>
__device__ __forceinline__ T beam_ninf() {
  return static_cast<T>(-INFINITY);
}
// Largest and least of a thread's logits (NaN passes over to neither).
__device__ __forceinline__ void beam_range(const uint4* raw, int groups, float, float& top, float& low) {
  top = -INFINITY, low = INFINITY;
#pragma unroll
  for (int g = 0; g < groups; ++g) {
    const uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, __uint_as_float(w[i])), low = fminf(low, __uint_as_float(w[i]));
  }
}
template <typename T2>
__device__ __forceinline__ void beam_range2(const uint4* raw, int groups, float& top, float& low) {
  T2 t = *reinterpret_cast<const T2*>(&raw[0].x), m = t;
#pragma unroll
  for (int g = 0; g < groups; ++g) {
    const uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T2 x = *reinterpret_cast<const T2*>(&w[i]);
      t = __hmax2(t, x), m = __hmin2(m, x);
    }
  }
  top = fmaxf(static_cast<float>(t.x), static_cast<float>(t.y));
  low = fminf(static_cast<float>(m.x), static_cast<float>(m.y));
}
__device__ __forceinline__ void beam_range(const uint4* raw, int groups, __nv_bfloat16, float& top, float& low) {
  beam_range2<__nv_bfloat162>(raw, groups, top, low);
}
__device__ __forceinline__ void beam_range(const uint4* raw, int groups, __half, float& top, float& low) {
  beam_range2<__half2>(raw, groups, top, low);
}

__device__ __forceinline__ float ex2_beam(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Keep the n best of `count` candidates, sorted, at the front (each thread ranks its
// candidates by counting the better ones).  All threads; count <= kBeamCap.
__device__ __forceinline__ void beam_prune(unsigned long long* cand, int count, int n) {
  unsigned long long mine[kBeamCap / kBeamThreads];
  int rank[kBeamCap / kBeamThreads];
#pragma unroll
  for (int i = 0; i < kBeamCap / kBeamThreads; ++i) {
    const int at = threadIdx.x + i * kBeamThreads;
    rank[i] = kBeamCap;
    if (at < count) {
      mine[i] = cand[at];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < count; ++j) r += cand[j] > mine[i];
      rank[i] = r;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBeamCap / kBeamThreads; ++i)
    if (rank[i] < n) cand[rank[i]] = mine[i];
  __syncthreads();
}

// The softcap in log2 units, cap tanh(l / cap) log2(e), for |l| <= cap: l times a polynomial in
// l^2, the least maximum-error odd polynomial of degree 13 for tanh on [-1, 1] (fitted by
// iteratively reweighted least squares: at most 2e-8 off, 9e-8 evaluated in fp32), its
// coefficients scaled by the caller.  It runs on packed FMAs, so that a logit costs one
// operation of the special-function unit (its exponential) instead of three.
constexpr int kTanhTerms = 7;
__device__ constexpr float kTanh[kTanhTerms] = {0.9999997019767761f,  -0.33332130312919617f, 0.13319583237171173f,
                                                -0.053265832364559174f, 0.019973276183009148f, -0.005951274652034044f,
                                                0.0009637702605687082f};

// CAP: 0 no softcap, 1 one up to 1000, 2 a larger one (a kernel of its own: the branch in the stream
// cost the 24 x 8 beams 1 us of 43).
constexpr float kBeamLargeCap = 1e3f;
template <typename T, int CAP>
__global__ void __launch_bounds__(kBeamThreads, beam_per_sm(sizeof(T))) beam_chunk_kernel(const BeamArgs a) {
  __shared__ unsigned long long cand[kBeamCap];
  __shared__ float seg_max[kBeamSuper][kBeamThreads];
  __shared__ int segs[kBeamSegs];
  __shared__ int count, seg_count;
  __shared__ uint32_t wbest[kBeamWarps], wtop[kBeamWarps];
  __shared__ float2 wstat[kBeamWarps];
  constexpr int VEC = 16 / sizeof(T), GROUPS = kBeamVals / VEC;
  constexpr float kLog2e = 1.4426950408889634f;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.y, b = row / a.beams, k = row % a.beams;
  const int begin = blockIdx.x * a.chunk, end = min(begin + a.chunk, a.vocab);
  pdl_launch_dependents();
  pdl_wait();
  if (a.finished != nullptr && a.finished[row]) return;  // its continuation needs no logits
  const T* x = static_cast<const T*>(a.logits) + b * a.l_b + k * a.l_k;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  if (tid == 0) count = 0;
  float mx = -INFINITY, sum = 0.f;  // reference (log2 units) and sum of 2^(y - reference)
  unsigned long long thr = 0;       // candidates must beat this key
  const float cap_in = CAP ? 1.f / a.cap : 0.f, cap_out = CAP ? a.cap * kLog2e : 0.f;
  // (beyond 1e-2 .. 1e3 the scaled coefficients leave fp32's range: no segment is in this one)
  const float poly_to = CAP == 1 && a.cap >= 1e-2f ? a.cap : -1.f;
  uint64_t tc[kTanhTerms];
  if constexpr (CAP) {
    float f = kLog2e;
#pragma unroll
    for (int i = 0; i < kTanhTerms; ++i, f *= cap_in * cap_in) tc[i] = f2_pack(kTanh[i] * f, kTanh[i] * f);
  }
  // The softcap of any logit.  1 + tanh - 1 is off by some 2^-22 of the cap, which is nothing to a cap
  // that the logits reach; below a large one they take the polynomial, off by 2^-21 of themselves.
  auto soft = [&](float l) {
    const float t = l * cap_in;
    if constexpr (CAP == 2) {
      if (fabsf(t) <= 1.f) {
        const float u = t * t;
        float p = kTanh[kTanhTerms - 1];
#pragma unroll
        for (int q = kTanhTerms - 2; q >= 0; --q) p = fmaf(p, u, kTanh[q]);
        return l * kLog2e * p;
      }
    }
    return cap_out * (one_plus_tanh(t) - 1.f);
  };
  // The thread's segment of a tile: 16 consecutive logits.
  auto load = [&](int t0, uint4 (&raw)[GROUPS]) {
    const int at0 = t0 + tid * kBeamVals;
    if (vec && at0 + kBeamVals <= end) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) raw[g] = reinterpret_cast<const uint4*>(x + at0)[g];
    } else {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          beam_fill(w, i, at0 + g * VEC + i < end ? x[at0 + g * VEC + i] : beam_ninf<T>());
        raw[g] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  };
  int held = 0;  // candidates kept so far: `count` between two collections, the same in every thread
  uint4 next[GROUPS];
  load(begin, next);
  for (int s0 = begin; s0 < end; s0 += kBeamSuper * kBeamTile) {
    const int tiles = min(kBeamSuper, (end - s0 + kBeamTile - 1) / kBeamTile);
    float best_mine = -INFINITY;
    // ---- the stream
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int t0 = s0 + j * kBeamTile;
      uint4 raw[GROUPS];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) raw[g] = next[g];
      if (t0 + kBeamTile < end) load(t0 + kBeamTile, next);  // travels meanwhile
      float tm, low;
      beam_range(raw, GROUPS, T{}, tm, low);
      seg_max[j][tid] = tm;
      best_mine = fmaxf(best_mine, tm);
      float ym = tm * kLog2e;
      if constexpr (CAP) ym = tm == -INFINITY ? -INFINITY : soft(tm);
      if (ym > mx) {
        sum *= ex2_beam(mx - ym);
        mx = ym;
      }
      const float ref = mx == -INFINITY ? 0.f : mx;
      const uint64_t nref = f2_pack(-ref, -ref);
      uint64_t part = 0;  // two sums
      if (!CAP || (tm <= poly_to && low >= -poly_to)) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          float v[VEC];
          beam_unpack(raw[g], v, T{});
#pragma unroll
          for (int i = 0; i < VEC; i += 2) {
            const uint64_t l = f2_pack(v[i], v[i + 1]);
            uint64_t e;
            if constexpr (CAP) {
              const uint64_t u = f2_mul(l, l);
              uint64_t p = tc[kTanhTerms - 1];
#pragma unroll
              for (int q = kTanhTerms - 2; q >= 0; --q) p = f2_fma(p, u, tc[q]);
              e = f2_fma(l, p, nref);
            } else {
              e = f2_fma(l, f2_pack(kLog2e, kLog2e), nref);
            }
            float e0, e1;
            f2_unpack(e, e0, e1);
            part = f2_add(part, f2_pack(ex2_beam(e0), ex2_beam(e1)));
          }
        }
      } else {
#pragma unroll 1
        for (int g = 0; g < GROUPS; ++g) {
          float v[VEC];
          uint4 w = raw[0];
#pragma unroll
          for (int i = 1; i < GROUPS; ++i)
            if (g == i) w = raw[i];
          beam_unpack(w, v, T{});
#pragma unroll
          for (int i = 0; i < VEC; ++i) {  // (an impossible token, or one past the chunk, stays impossible)
            const float y = v[i] == -INFINITY ? -INFINITY : soft(v[i]);
            part = f2_add(part, f2_pack(ex2_beam(y - ref), 0.f));
          }
        }
      }
      float p0, p1;
      f2_unpack(part, p0, p1);
      sum += p0 + p1;
    }
    // ---- the collection.  The thread maxima are distinct logits: bisect for a value that n of
    // them reach, and not many more.
    // Bounds: the largest of all, and the least over the warps of each one's ceil(n / 8)-th
    // largest, which n reach.
    const uint32_t mine = beam_bits(best_mine);
    uint32_t left = mine, top = 0, least = 0;
    for (int i = 0; i < (a.n + kBeamWarps - 1) / kBeamWarps; ++i) {
      least = __reduce_max_sync(0xffffffffu, left);
      if (i == 0) top = least;
      const unsigned who = __ballot_sync(0xffffffffu, left == least);
      if (lane == __ffs(who) - 1) left = 0;
    }
    if (lane == 0) wbest[warp] = least, wtop[warp] = top;
    if (tid == 0) seg_count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBeamWarps; ++i) least = min(least, wbest[i]), top = max(top, wtop[i]);
    ++top;  // (no value's bits are all ones)
    while (top - least > 1) {
      const uint32_t mid = least + (top - least) / 2;
      const int reach = __syncthreads_count(mine >= mid);
      if (reach >= a.n) {
        least = mid;
        if (reach <= a.n + a.n / 4) break;
      } else {
        top = mid;
      }
    }
    // A segment's best possible key, its maximum at its first token, must beat the n-th best so
    // far and reach `least`.
    auto wanted = [&](int j) {
      const float f = seg_max[j][tid];
      return f == f && beam_bits(f) >= least && beam_key(f, s0 + j * kBeamTile + tid * kBeamVals) > thr;
    };
    if (mine >= least)
      for (int j = 0; j < tiles; ++j)
        if (wanted(j)) {
          const int p = atomicAdd(&seg_count, 1);
          if (p < kBeamSegs) segs[p] = j * kBeamThreads + tid;
        }
    __syncthreads();
    // Which branch is taken must not depend on `count`: a fast warp adds to it at once in the first.
    const int found = seg_count;
    if (found <= kBeamSegs && held + found * kBeamVals <= kBeamCap) {
      for (int e = tid; e < found * kBeamVals; e += kBeamThreads) {
        const int at = s0 + segs[e / kBeamVals] * kBeamVals + e % kBeamVals;
        if (at < end) {
          const float f = static_cast<float>(x[at]);
          const unsigned long long key = beam_key(f, at);
          if (beam_bits(f) >= least && key > thr) cand[atomicAdd(&count, 1)] = key;
        }
      }
      __syncthreads();
      const int c = count;
      beam_prune(cand, c, a.n);
      if (c >= a.n) thr = cand[a.n - 1];
      held = min(c, a.n);
      if (tid == 0) count = held;
      __syncthreads();
    } else {
      // Too many segments reach the value (ties): tile by tile in the tokens' order, pruning as
      // the room runs out; what found none tries again against the raised threshold.
      for (int j = 0; j < tiles; ++j) {
        uint32_t todo = wanted(j) ? 0xFFFFFFFFu >> (32 - kBeamVals) : 0u;
        while (__syncthreads_or(todo != 0u)) {
          uint4 raw[GROUPS];
          if (todo) load(s0 + j * kBeamTile, raw);
          if (todo) {
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
              float v[VEC];
              beam_unpack(raw[g], v, T{});
#pragma unroll
              for (int i = 0; i < VEC; ++i) {
                const uint32_t bit = 1u << (g * VEC + i);
                if (todo & bit) {
                  const int at = s0 + j * kBeamTile + tid * kBeamVals + g * VEC + i;
                  const unsigned long long key = beam_key(v[i], at);
                  if (at >= end || key <= thr) {
                    todo &= ~bit;
                  } else {
                    const int p = atomicAdd(&count, 1);
                    if (p < kBeamCap) {
                      cand[p] = key;
                      todo &= ~bit;
                    }
                  }
                }
              }
            }
          }
          __syncthreads();
          const int c = min(count, kBeamCap);
          beam_prune(cand, c, a.n);
          if (c >= a.n) thr = cand[a.n - 1];
          held = min(c, a.n);
          if (tid == 0) count = held;
          __syncthreads();
        }
      }
    }
  }
  // ---- the chunk's sorted list and its sum
  unsigned long long* out = a.keys + (static_cast<int64_t>(row) * a.chunks + blockIdx.x) * a.n;
  for (int i = tid; i < a.n; i += kBeamThreads) out[i] = i < held ? cand[i] : 0ull;  // 0: none (below every key)
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, mx, d), os = __shfl_xor_sync(0xffffffffu, sum, d);
    const float mn = fmaxf(mx, om), ref = mn == -INFINITY ? 0.f : mn;
    sum = sum * ex2_beam(mx - ref) + os * ex2_beam(om - ref);
    mx = mn;
  }
  if (lane == 0) wstat[warp] = make_float2(mx, sum);
  __syncthreads();
  if (tid == 0) {
    mx = wstat[0].x;
    for (int i = 1; i < kBeamWarps; ++i) mx = fmaxf(mx, wstat[i].x);
    const float ref = mx == -INFINITY ? 0.f : mx;
    sum = 0.f;
    for (int i = 0; i < kBeamWarps; ++i) sum += wstat[i].y * ex2_beam(wstat[i].x - ref);
    a.stats[static_cast<int64_t>(row) * a.chunks + blockIdx.x] = make_float2(mx, sum);
  }
}

constexpr int kMergeThreads = 256;
constexpr int kMergeWarps = kMergeThreads / 32;

// One CTA per sequence: each warp merges the chunk lists of its beams (lane = chunk) and
// forms their totals; then every candidate's rank among all beams' sorted lists is counted
// by binary search, and the ranks below n are the answer.
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamArgs a) {
  extern __shared__ __align__(16) uint8_t sm[];
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int m = a.m, all = a.beams * m;
  double* total = reinterpret_cast<double*>(sm);                                  // [beams][m], not increasing
  unsigned long long* list = reinterpret_cast<unsigned long long*>(total + all);  // per warp: [chunks][n]
  int* token = reinterpret_cast<int*>(list + kMergeWarps * a.chunks * a.n);       // [beams][m]
  int* rank = token + all;                                                        // [beams][m]
  int* win = rank + all;                                                          // [n]: candidate of each rank
  pdl_launch_dependents();
  pdl_wait();
  for (int k = warp; k < a.beams; k += kMergeWarps) {
    const int row = b * a.beams + k;
    const double score = static_cast<double>(a.scores[row]);
    if (a.finished != nullptr && a.finished[row]) {
      // One continuation, `pad`, at an unchanged score; the rest are impossible, in order.
      for (int i = lane; i < m; i += 32) {
        token[k * m + i] = i == 0 ? a.pad : (i - 1 < a.pad ? i - 1 : i);
        total[k * m + i] = i == 0 && isfinite(score) ? score : -INFINITY;
      }
      // (with an impossible score all are: then in the tokens' order)
      if (!isfinite(score))
        for (int i = lane; i < m; i += 32) token[k * m + i] = i;
      __syncwarp();
      continue;
    }
    float2 st = make_float2(-INFINITY, 0.f);
    if (lane < a.chunks) st = a.stats[static_cast<int64_t>(row) * a.chunks + lane];
    unsigned long long* mine = list + warp * a.chunks * a.n;
    const unsigned long long* src = a.keys + static_cast<int64_t>(row) * a.chunks * a.n;
#pragma unroll 4
    for (int i = lane; i < a.chunks * a.n; i += 32) mine[i] = src[i];
    // Z: the chunks' sums joined in 64 bits, always in the same order.
    float mx = st.x;
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    double sum = st.x == -INFINITY ? static_cast<double>(st.y) : static_cast<double>(st.y) * exp2f(st.x - mx);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const double z = 0.69314718055994530942 * (static_cast<double>(mx) + log2(sum));
    if (!isfinite(z) || !isfinite(score)) {
      for (int i = lane; i < m; i += 32) {
        token[k * m + i] = i;
        total[k * m + i] = -INFINITY;
      }
      __syncwarp();
      continue;
    }
    __syncwarp();
    int head = 0;
    unsigned long long key = lane < a.chunks ? mine[lane * a.n] : 0ull;
    for (int i = 0; i < m; ++i) {
      const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32));
      const bool top = static_cast<uint32_t>(key >> 32) == hi;
      const uint32_t lo = __reduce_max_sync(0xffffffffu, top ? static_cast<uint32_t>(key) : 0u);
      if (top && static_cast<uint32_t>(key) == lo) {  // keys are distinct: one lane (m <= vocab: never a 0 key)
        token[k * m + i] = static_cast<int>(0xFFFFFFFFu - lo);
        total[k * m + i] = static_cast<double>(beam_value(hi));
        ++head;
        key = head < a.n ? mine[lane * a.n + head] : 0ull;
      }
    }
    __syncwarp();
    for (int i = lane; i < m; i += 32) {
      const double l = total[k * m + i];
      double y = l;
      if (a.cap > 0.f) y = l == -INFINITY ? l : static_cast<double>(a.cap) * tanh(l / static_cast<double>(a.cap));
      const double t = score + (y - z);
      total[k * m + i] = isfinite(t) ? t : -INFINITY;
    }
    __syncwarp();
    if (a.cap > 0.f) {
      // tanh rounds, so where it saturates a total may exceed the one before it by a step: a
      // running minimum keeps the list in order for the searches below.
      double t0 = lane < m ? total[k * m + lane] : INFINITY, t1 = lane + 32 < m ? total[k * m + lane + 32] : INFINITY;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double u0 = __shfl_up_sync(0xffffffffu, t0, d), u1 = __shfl_up_sync(0xffffffffu, t1, d);
        if (lane >= d) t0 = fmin(t0, u0), t1 = fmin(t1, u1);
      }
      t1 = fmin(t1, __shfl_sync(0xffffffffu, t0, 31));
      if (lane < m) total[k * m + lane] = t0;
      if (lane + 32 < m) total[k * m + lane + 32] = t1;
      __syncwarp();
    }
  }
  __syncthreads();
  // A candidate's rank: its place in its own beam's list and, for each other beam, how many of
  // that list come before it (ties: the lower beam).
  for (int e = tid; e < all; e += kMergeThreads) rank[e] = e % m;
  __syncthreads();
  for (int p = tid; p < all * (a.beams - 1); p += kMergeThreads) {
    const int e = p % all, k = e / m;
    int o = p / all;
    o += o >= k;
    const double t = total[e];
    int lo = 0, hi = m;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      const double v = total[o * m + mid];
      if (v > t || (v == t && o < k)) lo = mid + 1;
      else hi = mid;
    }
    if (lo) atomicAdd(&rank[e], lo);
  }
  __syncthreads();
  for (int e = tid; e < all; e += kMergeThreads)
    if (rank[e] < a.n) win[rank[e]] = e;
  __syncthreads();
  if (!a.slot_order) {
    for (int i = tid; i < a.n; i += kMergeThreads) {
      const int e = win[i];
      const int64_t at = static_cast<int64_t>(b) * a.n + i;
      a.out_scores[at] = static_cast<float>(total[e]);
      a.out_beam[at] = e / m;
      a.out_token[at] = token[e];
    }
  } else if (warp == 0) {
    // n = beams <= 32: the best continuation of a surviving beam takes that beam's slot, the
    // others take the free slots in order, best first.
    const bool in = lane < a.n;
    const int e = in ? win[lane] : -1, parent = in ? e / m : 64 + lane;
    const unsigned same = __match_any_sync(0xffffffffu, parent);
    const bool heir = in && (__ffs(same) - 1) == lane;
    unsigned used = __reduce_or_sync(0xffffffffu, in ? 1u << parent : 0u);
    const unsigned extra = __ballot_sync(0xffffffffu, in && !heir);
    if (in) {
      int slot = parent;
      if (!heir) {
        unsigned free = ~used;
        for (int i = __popc(extra & ((1u << lane) - 1)); i > 0; --i) free &= free - 1;
        slot = __ffs(free) - 1;
      }
      const int64_t at = static_cast<int64_t>(b) * a.n + slot;
      a.out_scores[at] = static_cast<float>(total[e]);
      a.out_beam[at] = parent;
      a.out_token[at] = token[e];
    }
  }
}

}  // namespace w8

namespace w8host {

int require_sm100(int* device);

struct BeamPlan {
  int chunks, chunk;
};

// Chunks of whole tiles, at most 32 (a warp merges one list per lane): about two waves of
// CTAs, so that finished beams leave no SM idle (24 x 8 beams, 20 % finished: 3 chunks 51.4,
// 6 chunks 45.1, 11 chunks 48.6 us; one sequence of 4 beams takes all 32: 13.6 us against
// 16.8 with 11).
static BeamPlan beam_plan(int64_t rows, int64_t vocab, int sms) {
  const int64_t tiles = std::max<int64_t>(1, (vocab + w8::kBeamTile - 1) / w8::kBeamTile);
  const int64_t want = 8 * static_cast<int64_t>(sms) / std::max<int64_t>(rows, 1);
  const int64_t n = std::max<int64_t>(1, std::min<int64_t>({want, tiles, w8::kBeamMaxChunks}));
  const int64_t per = (tiles + n - 1) / n;
  BeamPlan p;
  p.chunk = static_cast<int>(per * w8::kBeamTile);
  p.chunks = static_cast<int>((tiles + per - 1) / per);
  return p;
}

static int beam_shape(int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
  W8_CHECK_ARG(batch >= 0 && beams >= 1 && vocab >= 1 && n >= 1, "empty or negative size");
  if (beams > w8::kBeamMaxBeams || n > w8::kBeamMaxN) {
    set_error("%lld beams and %lld continuations: at most %d and %d", (long long)beams, (long long)n,
              w8::kBeamMaxBeams, w8::kBeamMaxN);
    return W8_ERR_UNSUPPORTED;
  }
  W8_CHECK_ARG(vocab < (1ll << 30), "vocabulary beyond 2^30");
  W8_CHECK_ARG(n <= beams * vocab, "%lld continuations of %lld candidates", (long long)n, (long long)(beams * vocab));
  W8_CHECK_ARG(batch * beams <= 65535, "batch * beams beyond 65535");
  return W8_OK;
}

static int64_t beam_ws(int64_t rows, const BeamPlan& p, int64_t n) {
  return rows * p.chunks * (n * 8 + 8);
}

template <typename T>
static auto beam_chunk(float cap) {
  return !(cap > 0.f) ? w8::beam_chunk_kernel<T, 0>
         : cap <= w8::kBeamLargeCap ? w8::beam_chunk_kernel<T, 1> : w8::beam_chunk_kernel<T, 2>;
}

template <typename Kern>
static int launch_beam(Kern kern, dim3 grid, int threads, int smem, cudaStream_t stream, const w8::BeamArgs& a) {
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

}  // namespace w8host

extern "C" int64_t w8_beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
  using namespace w8host;
  if (beam_shape(batch, beams, vocab, n) != W8_OK) return -1;
  int sms = 148;
  if (num_sms(&sms) != W8_OK) sms = 148;
  return beam_ws(batch * beams, beam_plan(batch * beams, vocab, sms), n);
}

extern "C" int w8_beam_select(const void* logits, int dtype, int64_t stride_b, int64_t stride_k, const float* scores,
                              const uint8_t* finished, int64_t pad, float cap, int64_t batch, int64_t beams,
                              int64_t vocab, int64_t n, int slot_order, float* out_scores, int64_t* out_beam,
                              int64_t* out_token, void* workspace, int64_t workspace_bytes, w8_stream_t stream) {
  using namespace w8host;
  int st = beam_shape(batch, beams, vocab, n);
  if (st != W8_OK) return st;
  W8_CHECK_ARG(dtype == W8_BF16 || dtype == W8_FP16 || dtype == W8_FP32, "dtype must be W8_BF16, W8_FP16 or W8_FP32");
  W8_CHECK_ARG(!slot_order || n == beams, "slot order needs as many continuations as beams");
  W8_CHECK_ARG(cap <= 0.f || (cap >= 1e-30f && cap <= 1e30f), "cap must be 0 (none) or between 1e-30 and 1e30");
  W8_CHECK_ARG(pad >= 0 && pad < vocab, "pad %lld is not a token", (long long)pad);
  if (batch == 0) return W8_OK;
  W8_CHECK_ARG(logits && scores && out_scores && out_beam && out_token, "null pointer");
  W8_CHECK_ALIGN(aligned(logits, dtype == W8_FP32 ? 4 : 2), "logits must be aligned to their type");
  int device = 0, sms = 0;
  if ((st = require_sm100(&device)) != W8_OK) return st;
  if ((st = num_sms(&sms)) != W8_OK) return st;
  const int64_t rows = batch * beams;
  const BeamPlan p = beam_plan(rows, vocab, sms);
  W8_CHECK_ARG(workspace != nullptr && workspace_bytes >= beam_ws(rows, p, n), "workspace of %lld bytes needed (got %lld)",
               (long long)beam_ws(rows, p, n), (long long)workspace_bytes);
  W8_CHECK_ALIGN(aligned(workspace, 8), "workspace must be 8-byte aligned");
  w8::BeamArgs a = {};
  a.logits = logits, a.l_b = stride_b, a.l_k = stride_k;
  a.scores = scores, a.finished = finished, a.pad = static_cast<int>(pad), a.cap = cap;
  a.batch = static_cast<int>(batch), a.beams = static_cast<int>(beams), a.vocab = static_cast<int>(vocab);
  a.n = static_cast<int>(n), a.m = static_cast<int>(std::min(n, vocab));
  a.chunks = p.chunks, a.chunk = p.chunk;
  a.keys = static_cast<unsigned long long*>(workspace);
  a.stats = reinterpret_cast<float2*>(a.keys + rows * p.chunks * n);
  a.out_scores = out_scores, a.out_beam = out_beam, a.out_token = out_token, a.slot_order = slot_order;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(p.chunks), static_cast<unsigned>(rows));
  st = dtype == W8_FP32   ? launch_beam(beam_chunk<float>(cap), grid, w8::kBeamThreads, 0, s, a)
       : dtype == W8_BF16 ? launch_beam(beam_chunk<__nv_bfloat16>(cap), grid, w8::kBeamThreads, 0, s, a)
                          : launch_beam(beam_chunk<__half>(cap), grid, w8::kBeamThreads, 0, s, a);
  if (st != W8_OK) return st;
  const int64_t all = static_cast<int64_t>(a.beams) * a.m;
  const int smem = static_cast<int>(all * 16 + static_cast<int64_t>(w8::kMergeWarps) * p.chunks * n * 8 + n * 4 + 16);
  static bool done[64] = {};
  if (!done[device]) {
    // Largest: 32 beams x 64 candidates, 8 warps x 32 chunks x 64 keys.
    W8_CUDA_TRY(cudaFuncSetAttribute(w8::beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 168 * 1024));
    done[device] = true;
  }
  return launch_beam(w8::beam_merge_kernel, dim3(static_cast<unsigned>(batch)), w8::kMergeThreads, smem, s, a);
}
