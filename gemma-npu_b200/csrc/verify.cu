// Which of a sequence's drafted tokens stand, and the token after them: speculative sampling over
// a drafted tree from given random numbers, or greedily.  The reference answers greedily, one
// token a step (gemma_npu.py:291), under the final softcap (pipeline.py:335-338).
//
// With p_i = softmax(y_i / temperature), y = cap tanh(logit / cap), the target's probabilities
// after node i and q_i the draft model's (1 at the token itself where drafts were chosen, not
// sampled), node i's children c in order, w_0 = p_i:
//   c stands if  u_c q_i(t_c) < w_k(t_c);  else  w_{k+1} = max(w_k - q_i, 0) / Z,  Z its sum
// and the walk goes on at c.  Where no child stands the next token is drawn from w: the first t
// with  sum_{v <= t} w(v) > u_0 sum_v w(v).
//
// A row of the 262144-wide head is half a megabyte, and most rows of a tree are never reached, so
// one kernel walks: a cluster of CTAs a sequence, each a contiguous part of the vocabulary, reads
// a node's row only when the walk is there.  Per node a pass for the maximum and the sum in fp32
// (bound by the row's latency and bytes), then numbers that every CTA derives alike.
//
// A number that lies within the fp32 sums' error of the border where its token stands or falls is measured
// again by sums in 64 bits (one in some ten thousand; every one where a range of levels is too wide for fp32).
// What is drawn must not depend on how a sum is rounded: a boundary of the 262144 moves the token
// when it crosses u_0, and the boundaries' errors add up.  In fp32 (about 1e-8 each) one draw in
// a thousand would differ, so what is drawn from is computed in 64 bits: 2^x from a table of 32
// and a polynomial of degree 5 (P. T. P. Tang, "Table-driven implementation of the exponential
// function in IEEE floating-point arithmetic", ACM TOMS 15(2), 1989), 10 operations a value, good
// to 2^-48, and sums in double.
//
// After k rejections w is max(p - c q, 0) / Z with one c: of max(p - c q, 0) / Z less q, what is
// positive is max(p - (c + Z) q, 0).  So nothing is stored: a node's first rejection costs one pass over
// both rows, which gives Z, and by warps' chunks what the draw then needs to find its token; a further
// one takes off what the larger c drops, in 64 bits only for the values that may be (looking at all of them
// again took 24 trees 33 us longer).
//
// What bounds it: the 64-bit operations of the passes (an SM has 62 a clock) and, for short walks, the
// chain of a node (its children, a pass, two meetings of the cluster: some 5 us).  One chain of 5 drafts
// over 262144 values takes 22 to 46 us by the draw, 24 trees 135 to 169, as long as their longest walk.  A
// node's statistics do not depend on the walk: a pass over all nodes at once, on all SMs, is not built.
#include "common.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace w8 {

static __device__ int g_verify_status = 0;

// Weights of a row's logits: 2^(level - ref), the level a logit in log2 units of its probability.
struct VerifyScale {
  float most;               // 20 caps: tanh is 1 to 2^-57 from there on
  float slope, two_over_cap, cap_slope;  // for fp32
  double in, out, twice;    // log2(e) 2 / cap, cap slope (slope without a cap), 2 cap slope
  double per_cap;           // 1 / cap
};

struct VerifyArgs {
  const void *x, *d;       // target's and draft model's logits [B, N, V]; d may be null
  int64_t x_b, x_n, d_b, d_n;
  const int64_t* tokens;   // [B, N]
  const int* parent;       // [B, N] or null: i - 1
  int64_t parent_b;
  const float* u;          // [B, N]
  int* path;               // [B, N]
  int* taken;              // [B]
  int64_t* token;          // [B]
  int n, vocab, per;       // per: values of a CTA's part (a multiple of 8)
  int greedy;
  double cap, slope;       // slope: log2(e) / temperature, of y or (without a cap) the logit
  float range;             // logits of 1000 levels
  VerifyScale target, drafted;  // (here, so that they take no registers)
  float err;               // what a fp32 sum may be off by, relative to it; 1 and more: anything
};

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyCluster = 16;   // CTAs at most (8 where the GPU has no 16 free together)
constexpr int kVerifyNodes = 1024;   // of a tree at most
constexpr int kVerifyVec = 8;        // values of a thread at a time
constexpr int kVerifyChunks = 1024;  // of a CTA's part of the vocabulary at most: a warp's turns of 256 values

template <typename E>
__device__ __forceinline__ float logit_f32(E v);
template <>
__device__ __forceinline__ float logit_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float logit_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float logit_f32<__half>(__half v) { return __half2float(v); }

// 8 neighbouring values of a row as they are: loads that nothing waits for until they are looked at.
template <typename E>
struct Raw8 {
  uint4 w[sizeof(E) * kVerifyVec / 16];
  __device__ __forceinline__ void load(const E* row) {  // (16-byte aligned)
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(E)) * kVerifyVec / 16; ++i) w[i] = reinterpret_cast<const uint4*>(row)[i];
  }
  __device__ __forceinline__ void get(float (&x)[kVerifyVec]) const {
    const E* e = reinterpret_cast<const E*>(w);
#pragma unroll
    for (int i = 0; i < kVerifyVec; ++i) x[i] = logit_f32<E>(e[i]);
  }
};
// Values v .. v + 7 of a row, -inf behind `end`.
template <typename E>
__device__ __forceinline__ void load8(const E* row, int v, int end, bool on16, float (&x)[kVerifyVec]) {
  if (on16 && v + kVerifyVec <= end) {
    Raw8<E> r;
    r.load(row + v);
    r.get(x);
  } else {
#pragma unroll
    for (int i = 0; i < kVerifyVec; ++i) x[i] = v + i < end ? logit_f32<E>(row[v + i]) : -INFINITY;
  }
}

// 2^t, |t| < 1000: t = n + j / 32 + g, |g| <= 1 / 64, 2^(j / 32) from the table, 2^g a polynomial (its
// next term, (g ln 2)^6 / 720, is below 2^-48 of 1).
__device__ __forceinline__ double exp2_64(double t, const double* table) {
  const double big = t + 0x1.8p52 / 32.0;  // rounded to a multiple of 1 / 32
  const int k = __double2loint(big);
  const double g = t - (big - 0x1.8p52 / 32.0);
  double p = fma(g, 1.333355814642844e-3, 9.618129107628477e-3);  // (ln 2)^5 / 5!, (ln 2)^4 / 4!
  p = fma(g, p, 5.550410866482158e-2);
  p = fma(g, p, 2.402265069591007e-1);
  p = fma(g, p, 6.931471805599453e-1);
  const double u = table[k & 31], s = fma(u * g, p, u);
  return __hiloint2double(__double2hiint(s) + ((k >> 5) << 20), __double2loint(s));
}
// One row's probabilities: 2^(level - ref) / sum.  Without a cap ref is the largest logit's level and levels
// are differences of logits, scaled: a level by itself, rounded to fp32, would be off by 2^-24 of it, 1e-3
// at a temperature of 1e-3.  The largest logit's weight is 1 in fp32 and (to 2^-52 of ref) in 64 bits.
struct VerifyRow {
  float top, least;  // the largest logit (level, with a cap); the logit 1000 levels below it, less than which counts as 0
  double ref, out;   // its level in 64 bits; levels a logit (no cap)
  double sum;
  bool fine;  // the row has a finite largest logit and no NaN
};
// The softcap of the target's rows: none, one whose levels differ by 900 at most, or a wider one (above
// 312 temperatures), whose levels need more care (a kernel of its own: beside the common caps that care cost
// registers, and with them an SM's second CTA).
enum : int { kNoCap = 0, kCap = 1, kWideCap = 2 };
__device__ __noinline__ double tanh_64(double z) { return tanh(z); }
// In 64 bits, without branches: the values of a thread are to be under way together.
template <int kCapped>
__device__ __forceinline__ double weight_64(float x, const VerifyScale& c, const VerifyRow& row, const double* table) {
  double w;
  bool none;
  if constexpr (kCapped == kNoCap) {
    none = x < row.least;
    w = exp2_64(fma(static_cast<double>(fmaxf(x, row.least)), row.out, -row.ref), table);
  } else {
    // tanh(z) = 1 - 2 / (1 + e^2z); the reciprocal by one step of Newton's iteration from 22 bits
    const float xc = fminf(fmaxf(x, -c.most), c.most);
    const double d = 1.0 + exp2_64(static_cast<double>(xc) * c.in, table);
    float r32;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r32) : "f"(static_cast<float>(d)));
    const double r0 = static_cast<double>(r32);
    double r = fma(r0, fma(-d, r0, 1.0), r0);
    if constexpr (kCapped == kWideCap) r = fma(r, fma(-d, r, 1.0), r);
    double t = fma(-c.twice, r, c.out - row.ref);
    none = x == -INFINITY;
    if constexpr (kCapped == kWideCap) {
      // The exponential's 2^-48 moves a level by up to 2^-49 of their range: of 2^31 levels that is 4e-6 of one.
      if (c.out > 65536.0) t = fma(c.out, tanh_64(static_cast<double>(xc) * c.per_cap), -row.ref);
      none = none || t < -1000.0;
      t = fmax(t, -1000.0);
    }
    w = exp2_64(t, table);
  }
  return __hiloint2double(none ? 0 : __double2hiint(w), none ? 0 : __double2loint(w));
}
// A capped logit's level.
__device__ __forceinline__ float level_32(float x, const VerifyScale& c) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * c.two_over_cap));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return x == -INFINITY ? -INFINITY : c.cap_slope * (1.f - 2.f * r);
}
__device__ __forceinline__ float ex2_32(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A logit's level less the row's largest one's.
template <int kCapped>
__device__ __forceinline__ float below_32(float x, const VerifyScale& c, const VerifyRow& row) {
  if constexpr (kCapped != kNoCap) return level_32(x, c) - row.top;
  return (x - row.top) * c.slope;
}

// What both kernels know of their sequence: a cluster of CTAs, each with a part of the vocabulary.
struct VerifyPlace {
  int b, rank, ranks, lo, hi;
};
__device__ __forceinline__ VerifyPlace verify_place(const VerifyArgs& a) {
  VerifyPlace p;
  uint32_t ranks;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  p.ranks = static_cast<int>(ranks), p.rank = static_cast<int>(cluster_ctarank());
  p.b = blockIdx.x / p.ranks;
  p.lo = min(p.rank * a.per, a.vocab), p.hi = min(p.lo + a.per, a.vocab);
  return p;
}
__device__ __forceinline__ void st_cluster_f64(const double* at, int rank, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(at), rank)), "d"(v) : "memory");
}
// The tree as the walk needs it.  The node's next child behind `i`: parents come before children.
struct VerifyTree {
  int parents[kVerifyNodes], tokens[kVerifyNodes];  // token -1: out of range
};
__device__ __forceinline__ void verify_tree(const VerifyArgs& a, const VerifyPlace& p, VerifyTree& t) {
  for (int i = threadIdx.x; i < a.n; i += kVerifyThreads) {
    t.parents[i] = a.parent != nullptr ? a.parent[p.b * a.parent_b + i] : i - 1;
    const int64_t token = a.tokens[static_cast<int64_t>(p.b) * a.n + i];
    t.tokens[i] = token >= 0 && token < a.vocab ? static_cast<int>(token) : -1;
  }
}
__device__ __forceinline__ int child_after(const VerifyArgs& a, const VerifyPlace& p, const VerifyTree& t, int node, int i) {
  for (++i; i < a.n; ++i)
    if (t.parents[i] == node) {
      if (t.tokens[i] >= 0) break;
      if (p.rank == 0 && threadIdx.x == 0) atomicExch(&g_verify_status, W8_ERR_INVALID_ARG);  // skipped
    }
  return i;
}

constexpr int kVerifyStep = kVerifyThreads * kVerifyVec;

template <typename E>
__device__ __forceinline__ const E* verify_row(const void* p, int64_t sb, int64_t sn, int b, int i) {
  return static_cast<const E*>(p) + b * sb + i * sn;
}
template <typename E>
__device__ __forceinline__ bool verify_on16(const E* row) {
  return (reinterpret_cast<uintptr_t>(row) & 15) == 0;
}

// ---------------------------------------------------------------- greedy
// The largest logit of a node, the lowest of equal ones, is the token after it; the child with that
// token stands.
template <typename E>
__global__ void __launch_bounds__(kVerifyThreads) draft_verify_greedy_kernel(const VerifyArgs a) {
  __shared__ VerifyTree tree;
  __shared__ unsigned long long keys[kVerifyWarps];
  __shared__ unsigned long long all[2][kVerifyCluster];  // every CTA's largest, by turns
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const VerifyPlace p = verify_place(a);
  pdl_launch_dependents();
  pdl_wait();
  verify_tree(a, p, tree);
  cluster_sync();
  int cur = 0, taken = 1, turn = 0;
  int64_t next;
  while (true) {
    const E* row = verify_row<E>(a.x, a.x_b, a.x_n, p.b, cur);
    const bool on16 = verify_on16(row);
    float top = -INFINITY;
    int at = 0x7FFFFFFF;
    bool bad = false;
    auto take = [&](const float (&x)[kVerifyVec], int v) {
#pragma unroll
      for (int i = 0; i < kVerifyVec; ++i) {
        bad |= !(x[i] < INFINITY);
        if (x[i] > top) top = x[i], at = v + i;
      }
    };
    constexpr int kBatch = 4;  // loads of a thread under way
    int v = p.lo + tid * kVerifyVec;
    if (on16)
      for (; v + (kBatch - 1) * kVerifyStep + kVerifyVec <= p.hi; v += kBatch * kVerifyStep) {
        Raw8<E> r[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) r[k].load(row + v + k * kVerifyStep);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          float x[kVerifyVec];
          r[k].get(x);
          take(x, v + k * kVerifyStep);
        }
      }
#pragma unroll 1
    for (; v < p.hi; v += kVerifyStep) {
      float x[kVerifyVec];
      load8<E>(row, v, p.hi, on16, x);
      take(x, v);
    }
    // The order-preserving bits of the value, then the lower index; a NaN or an infinity above all.
    const uint32_t s = __float_as_uint(top == 0.f ? 0.f : top);
    unsigned long long key = at == 0x7FFFFFFF ? 0ull
                                              : static_cast<unsigned long long>(s & 0x80000000u ? ~s : s | 0x80000000u) << 32 |
                                                    (0xFFFFFFFFu - static_cast<uint32_t>(at));
    if (bad) key = ~0ull;
    auto largest = [&](unsigned long long k) {
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, d);
        k = other > k ? other : k;
      }
      return k;
    };
    key = largest(key);
    if (lane == 0) keys[warp] = key;
    __syncthreads();
    turn ^= 1;
    if (warp == 0) {
      key = largest(lane < kVerifyWarps ? keys[lane] : 0ull);
      if (lane < p.ranks)
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&all[turn][p.rank]), lane)), "l"(key)
                     : "memory");
    }
    cluster_sync();
    key = largest(lane < p.ranks ? all[turn][lane] : 0ull);
    next = key == 0ull || key == ~0ull ? -1 : static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
    int went = -1;
    if (next >= 0)
      for (int c = child_after(a, p, tree, cur, cur); c < a.n; c = child_after(a, p, tree, cur, c))
        if (tree.tokens[c] == next) {
          went = c;
          break;
        }
    if (went < 0) break;
    if (p.rank == 0 && tid == 0) a.path[static_cast<int64_t>(p.b) * a.n + taken] = went;
    ++taken;
    cur = went;
  }
  if (p.rank == 0) {
    int* path = a.path + static_cast<int64_t>(p.b) * a.n;
    for (int i = taken + tid; i < a.n; i += kVerifyThreads) path[i] = -1;
    if (tid == 0) path[0] = 0, a.taken[p.b] = taken, a.token[p.b] = next;
  }
}

// ---------------------------------------------------------------- sampling
// (Without draft logits two CTAs fit an SM, so that clusters may be larger: 16 chains of 6 in 35 us where one
// CTA an SM, without the spills, takes 44.)
template <typename E, int kCapped, bool kDraft>
__global__ void __launch_bounds__(kVerifyThreads, kDraft || kCapped == kWideCap ? 1 : 2) draft_verify_kernel(const VerifyArgs a) {
  __shared__ VerifyTree tree;
  __shared__ double table[32];
  __shared__ float2 tops[2][kVerifyWarps];               // (largest level, sum) of a warp's part of p and q
  __shared__ float2 all_tops[2][2][kVerifyCluster];      // of a CTA's, by turns
  __shared__ double wide[4][kVerifyWarps];               // a warp's sums
  __shared__ double shared[2][4][kVerifyCluster];        // a CTA's, by turns
  __shared__ double chunk_p[kVerifyChunks], chunk_q[kDraft ? kVerifyChunks : 1];  // of a warp's parts of the last pass
  __shared__ int gone[kDraft ? 1 : kVerifyNodes];        // without draft logits: tokens whose weight is taken
  __shared__ uint8_t queue[kDraft ? kVerifyWarps : 1][256];  // of a warp's 256 values those that a rejection may drop
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const VerifyPlace at = verify_place(a);
  const int b = at.b, rank = at.rank, ranks = at.ranks, lo = at.lo, hi = at.hi;
  if (tid < 32) table[tid] = exp2(tid / 32.0);
  const VerifyScale &target = a.target, &drafted = a.drafted;
  // Chunks of `turns` times 256 values, a warp each.
  const int turns = max(1, (a.per + 256 * kVerifyChunks - 1) / (256 * kVerifyChunks));
  const int chunks = hi > lo ? (hi - lo + 256 * turns - 1) / (256 * turns) : 0;
  pdl_launch_dependents();
  pdl_wait();
  verify_tree(a, at, tree);
  const float* u = a.u + static_cast<int64_t>(b) * a.n;
  const double u0 = static_cast<double>(u[0]);
  cluster_sync();

  // Sums over a warp's first lanes, in every lane (the same order in every warp and CTA).
  auto warp_sum = [&](double v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
  };
  auto warp_max = [&](float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
  };
  int turn = 0, top_turn = 0;
  // The CTA's sums, then every CTA's to every CTA, at shared[turn].
  auto exchange_sums = [&](double (&v)[4]) {
    constexpr int n = kDraft ? 4 : 3;  // (without q the last is 0)
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = warp_sum(v[i]);
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < n; ++i) wide[i][warp] = v[i];
    }
    __syncthreads();
    turn ^= 1;
    if (warp < n) {
      const double s = warp_sum(lane < kVerifyWarps ? wide[warp][lane] : 0.0);
      if (lane < ranks) st_cluster_f64(&shared[turn][warp][rank], lane, s);
    }
    cluster_sync();
  };
  auto shared_sum = [&](int i) { return warp_sum(lane < ranks ? shared[turn][i][lane] : 0.0); };

  // The largest levels and the sums of a target row and (if asked for, which the compiler is to know: one
  // loop for both cases took 1 us a node more) a draft row in fp32.
  auto stats = [&](const E* xr, const E* dr, auto both, VerifyRow& p, VerifyRow& q) {
    constexpr bool two = decltype(both)::value;
    const bool wx = verify_on16(xr), wd = verify_on16(dr);
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};  // of levels (a capped row) or logits
    bool bad[2] = {false, false};
    auto slope = [&](int r) { return kCapped != kNoCap && r == 0 ? 1.f : drafted.slope; };
    auto add = [&](const float (&y)[kVerifyVec], int r) {
      float most = y[0];
#pragma unroll
      for (int i = 1; i < kVerifyVec; ++i) most = fmaxf(most, y[i]);
      // (without a branch: the sum is rescaled by 1 where the maximum stays)
      const float to = fmaxf(top[r], most), ref = to == -INFINITY ? 0.f : to;
      float s = sum[r] * ex2_32((top[r] - ref) * slope(r));
#pragma unroll
      for (int i = 0; i < kVerifyVec; ++i) s += ex2_32((y[i] - ref) * slope(r));
      sum[r] = s;
      top[r] = to;
    };
    auto take = [&](const float (&x)[kVerifyVec], int r) {
      float y[kVerifyVec];
#pragma unroll
      for (int i = 0; i < kVerifyVec; ++i) {
        bad[r] |= !(x[i] < INFINITY);
        y[i] = kCapped != kNoCap && r == 0 ? level_32(x[i], target) : x[i];
      }
      add(y, r);
    };
    constexpr int kBatch = 2;  // loads of a thread and row under way
    int v = lo + tid * kVerifyVec;
    if (wx && (!two || wd))
      for (; v + (kBatch - 1) * kVerifyStep + kVerifyVec <= hi; v += kBatch * kVerifyStep) {
        Raw8<E> rx[kBatch], ry[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) rx[k].load(xr + v + k * kVerifyStep);
        if constexpr (two) {
#pragma unroll
          for (int k = 0; k < kBatch; ++k) ry[k].load(dr + v + k * kVerifyStep);
        }
        float x[kVerifyVec];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          rx[k].get(x);
          take(x, 0);
        }
        if constexpr (two) {
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            ry[k].get(x);
            take(x, 1);
          }
        }
      }
#pragma unroll 1
    for (; v < hi; v += kVerifyStep) {
      float x[kVerifyVec];
      load8<E>(xr, v, hi, wx, x);
      take(x, 0);
      if constexpr (two) {
        load8<E>(dr, v, hi, wd, x);
        take(x, 1);
      }
    }
    // A warp's, the CTA's, then the cluster's: sums relative to the largest level so far.
    auto join = [&](float2 t, float slope) {
      const float to = warp_max(t.x);
      float s = t.x == -INFINITY ? t.y : t.y * ex2_32((t.x - to) * slope);  // (a NaN stays)
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      return make_float2(to, s);
    };
    constexpr int kRows = two ? 2 : 1;
    float2 t[2];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      t[r] = join(make_float2(top[r], bad[r] ? __uint_as_float(0x7FC00000u) : sum[r]), slope(r));
      if (lane == 0) tops[r][warp] = t[r];
    }
    __syncthreads();
    top_turn ^= 1;
    if (warp < kRows) {
      const float2 c = join(lane < kVerifyWarps ? tops[warp][lane] : make_float2(-INFINITY, 0.f), slope(warp));
      if (lane < ranks)
        st_cluster_f64(reinterpret_cast<const double*>(&all_tops[top_turn][warp][rank]), lane,
                       __hiloint2double(__float_as_int(c.y), __float_as_int(c.x)));
    }
    cluster_sync();
    auto row = [&](int r, const VerifyScale& scale) {
      const float2 c = join(lane < ranks ? all_tops[top_turn][r][lane] : make_float2(-INFINITY, 0.f), slope(r));
      VerifyRow out;
      out.top = c.x;
      out.sum = static_cast<double>(c.y);
      out.fine = c.y > 0.f && c.y < INFINITY && c.x > -INFINITY && c.x < INFINITY;
      out.ref = out.top, out.out = 0.0, out.least = out.top;
      if (kCapped == kNoCap || r != 0) {
        // (From 2^40 levels on the next lower fp32 number is 2^16 below: the largest logit's weight is 1,
        // every other one's 0.)
        const float levels = fabsf(out.top) * scale.slope;
        if (levels < 0x1p40f) {
          out.ref = static_cast<double>(out.top) * scale.out, out.out = scale.out;
          out.least = __fsub_ru(out.top, a.range);
          if (levels > 0x1p28f)  // (ref is rounded to 2^-53 of it)
            out.sum *= fma(fma(static_cast<double>(out.top), out.out, -out.ref), 0.6931471805599453, 1.0);
        } else {
          out.ref = 0.0;
        }
      }
      return out;
    };
    p = row(0, target);
    if constexpr (two) q = row(1, drafted);
  };

  int cur = 0, taken = 1;
  int64_t next = -1;
  bool written = false;
  while (true) {
    int went = -1;
    const E* xr = verify_row<E>(a.x, a.x_b, a.x_n, b, cur);
    const E* dr = kDraft ? verify_row<E>(a.d, a.d_b, a.d_n, b, cur) : xr;
    int c = child_after(a, at, tree, cur, cur);
    // What decides the first child comes with the row.
    const int c0 = c;
    float x0 = 0.f, d0 = 0.f, u_c0 = 0.f;
    if (c0 < a.n) {
      x0 = logit_f32<E>(xr[tree.tokens[c0]]);
      if (kDraft) d0 = logit_f32<E>(dr[tree.tokens[c0]]);
      u_c0 = u[c0];
    }
    VerifyRow p, q = {0.f, 0.f, 0.0, 0.0, 1.0, true};
    if (kDraft && c < a.n)
      stats(xr, dr, std::bool_constant<kDraft>(), p, q);
    else
      stats(xr, dr, std::false_type(), p, q);
    if (!p.fine) break;
    // After rejections w is max(p - c q, 0) / left: c = 0 and left = 1 at first, and of that less q what
    // is positive is max(p - (c + left) q, 0).  Without draft logits the rejected tokens' weights are taken
    // away and left is the others' sum, which may be off by `slack`.
    double c_q = 0.0, left = kDraft ? 1.0 : p.sum;
    double slack = kDraft ? 0.0 : a.err < 1.f ? a.err * p.sum : INFINITY;
    int rejected = 0;
    bool sharp = false;   // the sums are in 64 bits (with draft logits)
    bool summed = false;  // shared[turn][2, 3] and the chunks have the last pass's parts of p and q
    const bool wx = verify_on16(xr), wd = kDraft && verify_on16(dr);
    auto p_of = [&](float x) { return weight_64<kCapped>(x, target, p, table); };
    auto q_of = [&](float x) { return weight_64<kNoCap>(x, drafted, q, table); };
    auto taken_away = [&](int v) {  // (without draft logits)
      bool was = false;
      for (int i = 0; i < rejected; ++i) was |= gone[i] == v;
      return was;
    };
    // A pass in 64 bits over the CTA's part, a chunk of a warp at a time: sums of p and q, and of those
    // with p > rq / rp q (two) or not taken away, which are also the chunk's.
    auto pass = [&](auto both, double (&sums)[4], double rp, double rq) {
      constexpr bool two = decltype(both)::value;
      // (the next turn's values are under way while this one's weights are computed)
      Raw8<E> rx, ry;
      auto fetch = [&](int v) {
        if (wx && v + kVerifyVec <= hi) rx.load(xr + v);
        if (two && wd && v + kVerifyVec <= hi) ry.load(dr + v);
      };
      auto first_of = [&](int k) { return lo + k * turns * 256 + lane * kVerifyVec; };
      if (warp < chunks) fetch(first_of(warp));
#pragma unroll 1
      for (int k = warp; k < chunks; k += kVerifyWarps) {
        double part[2] = {0.0, 0.0};
#pragma unroll 1
        for (int j = 0; j < turns; ++j) {
          const int v = first_of(k) + j * 256;
          float x[kVerifyVec], y[kVerifyVec];
          if (wx && v + kVerifyVec <= hi)
            rx.get(x);
          else
            load8<E>(xr, v, hi, false, x);
          if constexpr (two) {
            if (wd && v + kVerifyVec <= hi)
              ry.get(y);
            else
              load8<E>(dr, v, hi, false, y);
          }
          fetch(j + 1 < turns ? v + 256 : first_of(k + kVerifyWarps));
          double pv[kVerifyVec], qv[kVerifyVec];
#pragma unroll
          for (int i = 0; i < kVerifyVec; ++i) {
            pv[i] = p_of(x[i]);
            if constexpr (two) qv[i] = q_of(y[i]);
          }
          if constexpr (two) {
#pragma unroll
            for (int i = 0; i < kVerifyVec; ++i) {
              sums[0] += pv[i], sums[1] += qv[i];
              // (a weight that does not stay becomes 0 in its bits)
              const bool stays = __double2hiint(fma(-rq, qv[i], pv[i] * rp)) >= 0;
              part[0] += __hiloint2double(stays ? __double2hiint(pv[i]) : 0, stays ? __double2loint(pv[i]) : 0);
              part[1] += __hiloint2double(stays ? __double2hiint(qv[i]) : 0, stays ? __double2loint(qv[i]) : 0);
            }
          } else {
            if (!kDraft && rejected > 0) {
#pragma unroll
              for (int i = 0; i < kVerifyVec; ++i)
                if (taken_away(v + i)) pv[i] = 0.0;
            }
#pragma unroll
            for (int i = 0; i < kVerifyVec; ++i) part[0] += pv[i];
          }
        }
        sums[2] += part[0], sums[3] += part[1];
        part[0] = warp_sum(part[0]);
        if constexpr (two) part[1] = warp_sum(part[1]);
        if (lane == 0) {
          chunk_p[k] = part[0];
          if constexpr (kDraft) chunk_q[k] = part[1];
        }
      }
    };
    // A further rejection's pass: c has grown, so values that stayed may be dropped and none comes back.
    // fp32 tells which cannot have been (what it may be off by is 2^-18 of the levels); the others,
    // 32 at a time, are looked at in 64 bits, and those dropped taken off the chunk's and the CTA's sums.
    auto drop = [&](double (&sums)[4], double rp0, double rq0, double rp, double rq) {
      const float slack = 0x1p-18f * (kCapped != kNoCap ? fabsf(p.top) + target.cap_slope : 0.f) + 0x1p-22f;
      const float at0 = static_cast<float>(log2(rq0 / rp0)) - slack, at1 = static_cast<float>(log2(rq / rp)) + slack;
      if (tid == 0) sums[2] = shared[turn][2][rank], sums[3] = shared[turn][3][rank];
      uint8_t* mine = queue[kDraft ? warp : 0];
#pragma unroll 1
      for (int k = warp; k < chunks; k += kVerifyWarps) {
        double part[2] = {0.0, 0.0};
#pragma unroll 1
        for (int j = 0; j < turns; ++j) {
          const int v0 = lo + (k * turns + j) * 256;
          float x[kVerifyVec], y[kVerifyVec];
          load8<E>(xr, v0 + lane * kVerifyVec, hi, wx, x);
          load8<E>(dr, v0 + lane * kVerifyVec, hi, wd, y);
          int n = 0;
#pragma unroll
          for (int i = 0; i < kVerifyVec; ++i) {
            const float lp = below_32<kCapped>(x[i], target, p), lq = below_32<kNoCap>(y[i], drafted, q), d = lp - lq;
            const float off = 0x1p-18f * (fabsf(lp) + fabsf(lq));
            // (p = 0 < q was dropped before; q = 0 is never)
            const bool near = lp != -INFINITY && lq != -INFINITY && !(d > at1 + off) && !(d < at0 - off);
            const uint32_t lanes = __ballot_sync(0xffffffffu, near);
            if (near) mine[n + __popc(lanes & ((1u << lane) - 1u))] = static_cast<uint8_t>(lane * kVerifyVec + i);
            n += __popc(lanes);
          }
          __syncwarp();
#pragma unroll 1
          for (int e = lane; e < n; e += 32) {
            const int v = v0 + mine[e];
            const double pv = p_of(logit_f32<E>(xr[v])), qv = q_of(logit_f32<E>(dr[v]));
            if (__double2hiint(fma(-rq0, qv, pv * rp0)) >= 0 && __double2hiint(fma(-rq, qv, pv * rp)) < 0)
              part[0] += pv, part[1] += qv;
          }
          __syncwarp();
        }
        sums[2] -= part[0], sums[3] -= part[1];
        part[0] = warp_sum(part[0]), part[1] = warp_sum(part[1]);
        if (lane == 0) chunk_p[k] -= part[0], chunk_q[kDraft ? k : 0] -= part[1];
      }
    };
    double last_rp = 0.0, last_rq = 0.0;  // of the last pass
    if (q.fine)
      for (; c < a.n; c = child_after(a, at, tree, cur, c)) {
        const int t = tree.tokens[c];
        const double uc = static_cast<double>(c == c0 ? u_c0 : u[c]);
        double pw = p_of(c == c0 ? x0 : logit_f32<E>(xr[t]));
        if constexpr (!kDraft) {
          const bool was = taken_away(t);
          if (was) pw = 0.0;
          bool stands = uc * left < pw;
          if (pw > 0.0 && !(fabs(uc * left - pw) > uc * slack)) {
            // The number lies so near the border that the sum in 64 bits decides (of what is left: where that
            // is little, a difference of sums would not do).
            double sums[4] = {0.0, 0.0, 0.0, 0.0};
            pass(std::false_type(), sums, 0.0, 0.0);
            exchange_sums(sums);
            left = shared_sum(2), slack = 0x1p-44 * left;
            summed = left > 0.0;
            stands = uc * left < pw;
          }
          if (stands) {
            went = c;
            break;
          }
          __syncthreads();
          if (!was) {
            if (tid == 0) gone[rejected] = t;
            ++rejected;
            left -= pw;
            summed = false;
          }
          __syncthreads();
        } else {
          const double qw = q_of(c == c0 ? d0 : logit_f32<E>(dr[t]));
          // u q < max(p - c q, 0) / left, without divisions
          auto decide = [&]() { return uc * left * (qw * p.sum) < fmax(fma(-c_q, qw * p.sum, pw * q.sum), 0.0); };
          const double to_c = c_q + (rejected == 0 ? 1.0 : left);
          bool stands;
          double z = 0.0;
          if (sharp) {
            stands = decide();
          } else {
            // The first child.  It stands by more than the fp32 sums may be off by; or a pass in 64 bits, which
            // its rejection needs anyway: with the sums of p and q by themselves over the values that stay
            // positive after it, which the fp32 sums tell, one pass gives the sums over all besides.  Those
            // sums move the border p = q by some 10^-7 of it: what lies between (10^-7 of the probability,
            // where p / q is spread) is miscounted by 10^-7 of itself, which shifts no draw.  But where little
            // is left, because p and q are nearly equal, a second pass counts again.
            const double l = uc * (qw * p.sum), r = pw * q.sum;
            stands = r - l > a.err * (l + r);
            if (!stands) {
#pragma unroll 1
              for (bool again = false;; again = true) {
                double sums[4] = {0.0, 0.0, 0.0, 0.0};
                last_rp = 1.0 / p.sum, last_rq = 1.0 / q.sum;
                pass(std::true_type(), sums, last_rp, last_rq);
                exchange_sums(sums);
                if (!again) {
                  p.sum = shared_sum(0), q.sum = shared_sum(1);
                  sharp = true;
                  stands = decide();
                }
                z = shared_sum(2) / p.sum - shared_sum(3) / q.sum;
                if (again || stands || !(fabs(p.sum * last_rp - q.sum * last_rq) > 0x1p-16 * z)) break;
              }
            }
          }
          if (stands) {
            went = c;
            break;
          }
          // Rejected: what is left.
          if (rejected > 0) {
            double sums[4] = {0.0, 0.0, 0.0, 0.0};
            drop(sums, last_rp, last_rq, 1.0 / p.sum, to_c / q.sum);
            last_rp = 1.0 / p.sum, last_rq = to_c / q.sum;
            exchange_sums(sums);
            z = shared_sum(2) / p.sum - to_c * (shared_sum(3) / q.sum);
          }
          // (Nothing but rounding is left where p and q are equal: w stays.)
          summed = z > 1e-13;
          if (summed) c_q = to_c, left = z;
          ++rejected;
        }
      }
    if (went < 0) {
      // ---- the next token: the weights' sums over the CTAs, then over one CTA's chunks, then a chunk
      while (!summed) {
        // (after a residual of nothing but rounding the one before it is summed again)
        double sums[4] = {0.0, 0.0, 0.0, 0.0};
        if (kDraft && c_q > 0.0)
          pass(std::bool_constant<kDraft>(), sums, 1.0 / p.sum, c_q / q.sum);
        else
          pass(std::false_type(), sums, 0.0, 0.0);
        exchange_sums(sums);
        if (kDraft || rejected == 0 || shared_sum(2) > 0.0) break;
        rejected = 0;  // the weights taken were all there were: the target's own
      }
      const double rp = 1.0 / p.sum, rq = kDraft && c_q > 0.0 ? c_q / q.sum : 0.0;  // (a draft row may be NaN)
      auto part_of = [&](int k) { return kDraft ? fma(-rq, shared[turn][3][k], shared[turn][2][k] * rp) : shared[turn][2][k] * rp; };
      const double aim = u0 * warp_sum(lane < ranks ? fmax(part_of(lane), 0.0) : 0.0);
      // The first of `n` parts whose running sum passes the aim, or the last with any weight (-1: none).
      auto place = [&](int n, auto part, double& before) {
        int last = -1;
        double run = before, last_run = before;
        for (int k = 0; k < n; ++k) {
          const double s = part(k);
          if (s > 0.0) {
            last = k, last_run = run;
            if (run + s > aim) break;
            run += s;
          }
        }
        before = last_run;
        return last;
      };
      if (warp == 0) {
        double before = 0.0;
        const int owner = place(ranks, part_of, before);
        if (owner == rank) {
          // (the chunks' sums are there: the cluster has met since)  A lane's run of chunks, then the lane.
          const int run = (chunks + 31) / 32, k0 = min(lane * run, chunks), k1 = min(k0 + run, chunks);
          auto of = [&](int k) { return fmax(kDraft ? fma(-rq, chunk_q[kDraft ? k : 0], chunk_p[k] * rp) : chunk_p[k] * rp, 0.0); };
          double mine = 0.0;
          for (int k = k0; k < k1; ++k) mine += of(k);
          double incl = mine;
#pragma unroll
          for (int s = 1; s < 32; s <<= 1) {
            const double o = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += o;
          }
          const uint32_t some = __ballot_sync(0xffffffffu, mine > 0.0);
          uint32_t over = __ballot_sync(0xffffffffu, mine > 0.0 && before + incl > aim);
          const int l = over ? __ffs(over) - 1 : max(31 - __clz(some), 0);
          double sum_at = before + incl - mine;
          int k = place(k1 - k0, [&](int i) { return of(k0 + i); }, sum_at) + k0;
          k = max(__shfl_sync(0xffffffffu, k, l), 0);  // (a CTA with weight has such a chunk, but for rounding)
          sum_at = __shfl_sync(0xffffffffu, sum_at, l);
          // The chunk's values, 256 at a time.  What further rejections took off a chunk's sums may have left it
          // some 2^-53 of them and no value: the number then meant the next value that has weight, or
          // (it may lie at the end of the sums) the last one.
          const int begin = lo + k * turns * 256, end_own = min(begin + turns * 256, hi);
          int last = -1, token = -1, v0 = begin;
          bool own = true, back = false;
#pragma unroll 1
          while (true) {
            const int v = v0 + lane * kVerifyVec, stop = own ? hi : a.vocab;
            float x[kVerifyVec], y[kVerifyVec];
            double f[kVerifyVec], sum = 0.0;
            load8<E>(xr, v, stop, wx, x);
            if (kDraft && c_q > 0.0) load8<E>(dr, v, stop, wd, y);
            int start = 0x7FFFFFFF, end = -1;
#pragma unroll
            for (int i = 0; i < kVerifyVec; ++i) {
              f[i] = p_of(x[i]) * rp;
              if (kDraft && c_q > 0.0) f[i] = fmax(fma(-rq, q_of(y[i]), f[i]), 0.0);
              if (!kDraft && rejected > 0 && taken_away(v + i)) f[i] = 0.0;
              sum += f[i];
              if (f[i] > 0.0) start = min(start, v + i), end = v + i;
            }
            double incl = sum;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
              const double o = __shfl_up_sync(0xffffffffu, incl, s);
              if (lane >= s) incl += o;
            }
            last = max(last, __reduce_max_sync(0xffffffffu, end));
            over = __ballot_sync(0xffffffffu, own && end >= 0 && sum_at + incl > aim);
            if (over) {
              double s = sum_at + incl - sum;
              int mine_token = -1;
#pragma unroll
              for (int i = 0; i < kVerifyVec; ++i) {
                s += f[i];
                if (mine_token < 0 && f[i] > 0.0 && s > aim) mine_token = v + i;
              }
              if (mine_token < 0) mine_token = end;  // (rounding may leave the sum at the aim: the last)
              token = __shfl_sync(0xffffffffu, mine_token, __ffs(over) - 1);
              break;
            }
            sum_at += __shfl_sync(0xffffffffu, incl, 31);
            const bool more = own && v0 + 256 < end_own;
            if (!more && last >= 0) {
              token = own || back ? last : __reduce_min_sync(0xffffffffu, start);
              break;
            }
            if (back) {
              if (v0 == 0) break;
              v0 = max(v0 - 256, 0);
            } else {
              v0 = own && !more ? end_own : v0 + 256;
              own = more;
              if (!own && v0 >= a.vocab) back = true, v0 = max(begin - 256, 0);
            }
          }
          if (lane == 0) a.token[b] = token;
        } else if (owner < 0 && rank == 0 && lane == 0) {
          a.token[b] = -1;
        }
      }
      written = true;
      break;
    }
    if (rank == 0 && tid == 0) a.path[static_cast<int64_t>(b) * a.n + taken] = went;
    ++taken;
    cur = went;
    __syncthreads();  // (gone is free)
  }
  if (rank == 0) {
    int* path = a.path + static_cast<int64_t>(b) * a.n;
    for (int i = taken + tid; i < a.n; i += kVerifyThreads) path[i] = -1;
    if (tid == 0) {
      path[0] = 0;
      a.taken[b] = taken;
      if (!written) a.token[b] = next;
    }
  }
}

}  // namespace w8

namespace w8host {

int require_sm100(int* device);

// Read (and optionally clear) the sticky device status of the verification.
int verify_device_status(int clear, int* out) {
  W8_CUDA_TRY(cudaMemcpyFromSymbol(out, w8::g_verify_status, sizeof(int)));
  if (clear) {
    const int zero = 0;
    W8_CUDA_TRY(cudaMemcpyToSymbol(w8::g_verify_status, &zero, sizeof(int)));
  }
  return W8_OK;
}

template <typename Kern>
static int verify_launch(Kern kern, int (&held)[64][w8::kVerifyCluster + 1], w8::VerifyArgs a, int64_t batch, int device,
                         cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(w8::kVerifyThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // Clusters of each size that the device holds at once: its SMs come in groups, which clusters do not
  // cross (15 clusters of 8 or of 9, 22 of 6, 26 of 5).
  static std::mutex filling;
  std::unique_lock<std::mutex> lock(filling);
  if (held[device][1] == 0) {
    W8_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cfg.numAttrs = 1;
    for (int c = w8::kVerifyCluster; c >= 1; --c) {
      cfg.gridDim = dim3(static_cast<unsigned>(c), 1, 1);
      attr[0].val.clusterDim.x = static_cast<unsigned>(c);
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      held[device][c] = c == 1 ? std::max(n, 1) : n;
    }
  }
  lock.unlock();
  // CTAs of a sequence: the most with which all sequences run at once (64 bits keep an SM's pipes busy,
  // and a second wave would double the time), each with at least 2048 values.
  int cluster = 1;
  for (int c = 2; c <= w8::kVerifyCluster && c * 2048ll <= a.vocab; ++c)
    if (held[device][c] >= batch) cluster = c;
  a.per = static_cast<int>(((a.vocab + cluster - 1) / cluster + 7) / 8 * 8);
  // A thread's fp32 sum is of `values` numbers, which it scales at every eighth at most, by an exponential
  // (2^-22); the warps' and CTAs' sums, the exponentials and the roundings of their arguments (3 2^-24 of
  // each; their mean over the weights is below the logarithm of the vocabulary) are 158 2^-24 more.  A
  // capped level is off by some 2^-21 of its range.  4 / 3 of that below 1 / 4, where a quotient is
  // off by so much more.
  const double values = static_cast<double>((a.per + w8::kVerifyStep - 1) / w8::kVerifyStep * w8::kVerifyVec);
  const double err = 0x1p-24 * (2.0 * values + 160.0) + 0x1p-20 * a.cap * a.slope;
  a.err = err < 0.25 ? static_cast<float>(1.5 * err) : 1.f;
  cfg.gridDim = dim3(static_cast<unsigned>(batch * cluster), 1, 1);
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, a));
}

template <typename E, int kCapped, bool kDraft>
static int verify_sample(const w8::VerifyArgs& a, int64_t batch, int device, cudaStream_t stream) {
  static int held[64][w8::kVerifyCluster + 1] = {};
  return verify_launch(w8::draft_verify_kernel<E, kCapped, kDraft>, held, a, batch, device, stream);
}

template <typename E>
static int verify_go(const w8::VerifyArgs& a, int64_t batch, int device, cudaStream_t stream) {
  if (a.greedy) {
    static int held[64][w8::kVerifyCluster + 1] = {};
    return verify_launch(w8::draft_verify_greedy_kernel<E>, held, a, batch, device, stream);
  }
  using namespace w8;
  if (2.0 * a.cap * a.slope > 900.0)
    return a.d != nullptr ? verify_sample<E, kWideCap, true>(a, batch, device, stream)
                          : verify_sample<E, kWideCap, false>(a, batch, device, stream);
  if (a.cap > 0.0)
    return a.d != nullptr ? verify_sample<E, kCap, true>(a, batch, device, stream)
                          : verify_sample<E, kCap, false>(a, batch, device, stream);
  return a.d != nullptr ? verify_sample<E, kNoCap, true>(a, batch, device, stream)
                        : verify_sample<E, kNoCap, false>(a, batch, device, stream);
}

}  // namespace w8host

extern "C" int w8_draft_verify(const w8_draft_verify_args* in, w8_stream_t stream) {
  using namespace w8host;
  W8_CHECK_ARG(in != nullptr, "null arguments");
  const w8_draft_verify_args& x = *in;
  W8_CHECK_ARG(x.batch >= 0 && x.n_new >= 1 && x.vocab >= 1, "at least one node and one token");
  W8_CHECK_ARG(x.n_new <= w8::kVerifyNodes, "more than %d nodes", w8::kVerifyNodes);
  W8_CHECK_ARG(x.vocab < (1ll << 30) && x.batch <= (1ll << 24), "size beyond the limits");
  W8_CHECK_ARG(x.dtype == W8_BF16 || x.dtype == W8_FP16 || x.dtype == W8_FP32, "unknown dtype");
  W8_CHECK_ARG(x.temperature == 0.0 || (x.temperature >= 1e-3 && x.temperature <= 1e3),
               "temperature must be 0 (greedy) or between 1e-3 and 1e3");
  W8_CHECK_ARG(x.cap == 0.0 || (x.cap >= 1e-3 && x.cap <= 1e6), "cap must be 0 (none) or between 1e-3 and 1e6");
  if (x.batch == 0) return W8_OK;
  const bool greedy = x.temperature == 0.0;
  W8_CHECK_ARG(x.logits && x.tokens && x.path && x.taken && x.token && (greedy || x.uniform), "null pointer");
  int device = 0;
  const int st = require_sm100(&device);
  if (st != W8_OK) return st;
  w8::VerifyArgs a = {};
  a.x = x.logits, a.d = greedy ? nullptr : x.draft;
  a.x_b = x.logits_stride[0], a.x_n = x.logits_stride[1];
  a.d_b = x.draft_stride[0], a.d_n = x.draft_stride[1];
  a.tokens = x.tokens;
  a.parent = x.parent;
  a.parent_b = x.parent_stride;
  a.u = x.uniform;
  a.path = x.path, a.taken = x.taken, a.token = x.token;
  a.n = static_cast<int>(x.n_new), a.vocab = static_cast<int>(x.vocab);
  a.greedy = greedy;
  a.cap = greedy ? 0.0 : x.cap;
  a.slope = greedy ? 1.0 : 1.4426950408889634 / x.temperature;
  a.range = static_cast<float>(1000.0 / a.slope);
  a.drafted.slope = static_cast<float>(a.slope);
  a.drafted.out = a.slope;
  a.target = a.drafted;
  if (a.cap > 0.0) {
    constexpr double kLog2e = 1.4426950408889634;
    a.target.most = static_cast<float>(20.0 * a.cap);
    a.target.two_over_cap = static_cast<float>(2.0 * kLog2e / a.cap);
    a.target.cap_slope = static_cast<float>(a.cap * a.slope);
    a.target.in = 2.0 * kLog2e / a.cap;
    a.target.out = a.cap * a.slope;
    a.target.twice = 2.0 * a.target.out;
    a.target.per_cap = 1.0 / a.cap;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (x.dtype == W8_FP32) return verify_go<float>(a, x.batch, device, s);
  if (x.dtype == W8_BF16) return verify_go<__nv_bfloat16>(a, x.batch, device, s);
  return verify_go<__half>(a, x.batch, device, s);
}
