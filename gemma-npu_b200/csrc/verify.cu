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
// What is drawn must not depend on how a sum is rounded: a boundary of the 262144 moves the token
// when it crosses u_0, and the boundaries' errors add up.  In fp32 (about 1e-8 each) one draw in
// a thousand would differ, so what is drawn from is computed in 64 bits: 2^x from a table of 32
// and a polynomial of degree 5 (P. T. P. Tang, "Table-driven implementation of the exponential
// function in IEEE floating-point arithmetic", ACM TOMS 15(2), 1989), 14 operations a value, good
// to 2^-50, and sums in double.
#include "common.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace w8 {

static __device__ int g_verify_status = 0;

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
};

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyCluster = 16;   // CTAs at most (8 where the GPU has no 16 free together)
constexpr int kVerifyNodes = 1024;   // of a tree at most
constexpr int kVerifyVec = 8;        // values of a thread at a time

template <typename E>
__device__ __forceinline__ float logit_f32(E v);
template <>
__device__ __forceinline__ float logit_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float logit_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float logit_f32<__half>(__half v) { return __half2float(v); }

// Values v .. v + 7 of a row, -inf behind `end`.
template <typename E>
__device__ __forceinline__ void load8(const E* row, int v, int end, bool wide, float (&x)[kVerifyVec]) {
  if (wide && v + kVerifyVec <= end) {
    constexpr int kWords = sizeof(E) * kVerifyVec / 16;
    uint4 w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const uint4*>(row + v)[i];
    const E* e = reinterpret_cast<const E*>(w);
#pragma unroll
    for (int i = 0; i < kVerifyVec; ++i) x[i] = logit_f32<E>(e[i]);
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
// Weights of a row's logits: 2^(level - top), the level a logit in log2 units of its probability.
struct VerifyScale {
  bool capped;
  bool deep;                // a capped row's levels may differ by more than 900
  float most;               // 20 caps: tanh is 1 to 2^-57 from there on
  float slope, two_over_cap, cap_slope;  // for fp32
  double in, out, twice;    // log2(e) 2 / cap, cap slope (slope without a cap), 2 cap slope
};
// In 64 bits; `top` the row's largest level to fp32, `least` the logit whose level is 1000 below it:
// less counts as 0.  Without branches: the values of a thread are to be under way together.
__device__ __forceinline__ double weight_64(float x, const VerifyScale& c, float top, float least, const double* table) {
  double w;
  bool none;
  if (!c.capped) {
    none = x < least;
    w = exp2_64(fma(static_cast<double>(fmaxf(x, least)), c.out, -static_cast<double>(top)), table);
  } else {
    // tanh(z) = 1 - 2 / (1 + e^2z); the reciprocal by one step of Newton's iteration from 22 bits
    const float xc = fminf(fmaxf(x, -c.most), c.most);
    const double d = 1.0 + exp2_64(static_cast<double>(xc) * c.in, table);
    float r32;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r32) : "f"(static_cast<float>(d)));
    const double r0 = static_cast<double>(r32), r = fma(r0, fma(-d, r0, 1.0), r0);
    double t = fma(-c.twice, r, c.out - static_cast<double>(top));
    none = x == -INFINITY;
    if (c.deep) {
      none = none || t < -1000.0;
      t = fmax(t, -1000.0);
    }
    w = exp2_64(t, table);
  }
  return __hiloint2double(none ? 0 : __double2hiint(w), none ? 0 : __double2loint(w));
}
__device__ __forceinline__ float level_32(float x, const VerifyScale& c) {
  if (!c.capped) return x * c.slope;
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

// One row's probabilities 2^(level - top) / sum.
struct VerifyRow {
  float top, least;  // the largest level; the logit 1000 below it
  double sum;
  bool fine;  // the row has a finite largest logit and no NaN
};

template <typename E>
__global__ void __launch_bounds__(kVerifyThreads) draft_verify_kernel(const VerifyArgs a) {
  __shared__ double table[32];
  __shared__ double wide_a[kVerifyWarps], wide_b[kVerifyWarps];
  __shared__ double shared_a[2][kVerifyCluster], shared_b[2][kVerifyCluster];  // every CTA's results, by turns
  __shared__ int parents[kVerifyNodes];
  __shared__ int64_t gone[kVerifyNodes];   // without draft logits: tokens whose weight is taken
  __shared__ int found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t ranks_u;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks_u));
  const int ranks = static_cast<int>(ranks_u), rank = static_cast<int>(cluster_ctarank());
  const int b = blockIdx.x / ranks;
  const int lo = min(rank * a.per, a.vocab), hi = min(lo + a.per, a.vocab);
  if (tid < 32) table[tid] = exp2(tid / 32.0);
  pdl_launch_dependents();
  pdl_wait();
  for (int i = tid; i < a.n; i += kVerifyThreads) parents[i] = a.parent != nullptr ? a.parent[b * a.parent_b + i] : i - 1;
  const int64_t* tokens = a.tokens + static_cast<int64_t>(b) * a.n;
  const float* u = a.u != nullptr ? a.u + static_cast<int64_t>(b) * a.n : nullptr;
  cluster_sync();

  int turn = 0;
  // Every CTA's (va, vb) to every CTA, which then reads them at shared_a / shared_b[turn].
  auto exchange = [&](double va, double vb) {  // (of thread 0 .. ranks - 1)
    turn ^= 1;
    if (tid < ranks) {
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&shared_a[turn][rank]), tid)), "d"(va)
                   : "memory");
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&shared_b[turn][rank]), tid)), "d"(vb)
                   : "memory");
    }
    cluster_sync();
  };
  // Sums over the CTA, in every thread.
  auto block_sums = [&](double& va, double& vb) {
#pragma unroll
    for (int s = 16; s; s >>= 1) {
      va += __shfl_xor_sync(0xffffffffu, va, s);
      vb += __shfl_xor_sync(0xffffffffu, vb, s);
    }
    __syncthreads();
    if (lane == 0) wide_a[warp] = va, wide_b[warp] = vb;
    __syncthreads();
    va = vb = 0.0;
#pragma unroll
    for (int w = 0; w < kVerifyWarps; ++w) va += wide_a[w], vb += wide_b[w];
  };
  auto cluster_sums = [&](double& va, double& vb) {
    block_sums(va, vb);
    exchange(va, vb);
    va = vb = 0.0;
    for (int k = 0; k < ranks; ++k) va += shared_a[turn][k], vb += shared_b[turn][k];
  };
  constexpr int kStep = kVerifyThreads * kVerifyVec;
  auto row_of = [&](const void* p, int64_t sb, int64_t sn, int i) { return static_cast<const E*>(p) + b * sb + i * sn; };
  auto aligned16 = [&](const E* row) { return (reinterpret_cast<uintptr_t>(row) & 15) == 0; };

  // ---- greedy: the largest logit, the lowest of equal ones (-1: none is finite, or a NaN)
  auto best_of = [&](int node) -> int64_t {
    const E* row = row_of(a.x, a.x_b, a.x_n, node);
    const bool wide = aligned16(row);
    float top = -INFINITY;
    int at = 0x7FFFFFFF;
    bool bad = false;
#pragma unroll 2
    for (int v = lo + tid * kVerifyVec; v < hi; v += kStep) {
      float x[kVerifyVec];
      load8<E>(row, v, hi, wide, x);
#pragma unroll
      for (int i = 0; i < kVerifyVec; ++i) {
        bad |= !(x[i] < INFINITY);
        if (x[i] > top) top = x[i], at = v + i;
      }
    }
    bad = __syncthreads_or(bad);
    // (the order-preserving bits of the value, then the lower index)
    auto key_of = [&](float x, int i) {
      const uint32_t s = __float_as_uint(x == 0.f ? 0.f : x);
      return static_cast<unsigned long long>(s & 0x80000000u ? ~s : s | 0x80000000u) << 32 |
             (0xFFFFFFFFu - static_cast<uint32_t>(i));
    };
    unsigned long long key = at == 0x7FFFFFFF ? 0ull : key_of(top, at);
#pragma unroll
    for (int s = 16; s; s >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, s);
      key = other > key ? other : key;
    }
    unsigned long long* keys = reinterpret_cast<unsigned long long*>(wide_a);
    if (lane == 0) keys[warp] = key;
    __syncthreads();
    for (int w = 0; w < kVerifyWarps; ++w) key = keys[w] > key ? keys[w] : key;
    exchange(__longlong_as_double(static_cast<long long>(key)), bad ? 1.0 : 0.0);
    for (int k = 0; k < ranks; ++k) {
      const unsigned long long other = static_cast<unsigned long long>(__double_as_longlong(shared_a[turn][k]));
      key = other > key ? other : key;
      bad |= shared_b[turn][k] != 0.0;
    }
    return bad || key == 0ull ? -1 : static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
  };

  // ---- sampling: a row's maximum and sum in fp32 ...
  auto stats = [&](const E* row, const VerifyScale& scale) {
    const bool wide = aligned16(row);
    float top = -INFINITY, sum = 0.f;  // in log2 units
    bool bad = false;
#pragma unroll 2
    for (int v = lo + tid * kVerifyVec; v < hi; v += kStep) {
      float x[kVerifyVec];
      load8<E>(row, v, hi, wide, x);
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < kVerifyVec; ++i) {
        bad |= !(x[i] < INFINITY);
        x[i] = level_32(x[i], scale);
        most = fmaxf(most, x[i]);
      }
      if (most > top) sum *= ex2_32(top - most), top = most;
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int i = 0; i < kVerifyVec; ++i) sum += ex2_32(x[i] - ref);
    }
    // The CTA's, then the cluster's.
    float high = top;
#pragma unroll
    for (int s = 16; s; s >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, s));
    __syncthreads();
    if (lane == 0) wide_a[warp] = high;
    bad = __syncthreads_or(bad);
    float mine = static_cast<float>(wide_a[0]);
#pragma unroll
    for (int w = 1; w < kVerifyWarps; ++w) mine = fmaxf(mine, static_cast<float>(wide_a[w]));
    double part = top == -INFINITY ? 0.0 : static_cast<double>(sum) * ex2_32(top - mine), none = 0.0;
    block_sums(part, none);
    exchange(mine, bad ? __longlong_as_double(0x7FF8000000000000ll) : part);
    VerifyRow r;
    r.top = static_cast<float>(shared_a[turn][0]);
    for (int k = 1; k < ranks; ++k) r.top = fmaxf(r.top, static_cast<float>(shared_a[turn][k]));
    r.sum = 0.0;
    for (int k = 0; k < ranks; ++k) {
      const double s = shared_b[turn][k];  // (NaN: the row is not fine)
      if (s != 0.0) r.sum += s * ex2_32(static_cast<float>(shared_a[turn][k]) - r.top);
    }
    r.fine = r.sum > 0.0 && isfinite(r.sum) && isfinite(r.top);
    r.least = fmaxf((r.top - 1000.f) / scale.slope, -3e38f);
    return r;
  };

  VerifyScale drafted = {};
  drafted.slope = static_cast<float>(a.slope);
  drafted.out = a.slope;
  VerifyScale target = drafted;
  if (a.cap > 0.0) {
    target.capped = true;
    target.most = static_cast<float>(20.0 * a.cap);
    target.two_over_cap = static_cast<float>(2.0 * 1.4426950408889634 / a.cap);
    target.cap_slope = static_cast<float>(a.cap * a.slope);
    target.in = 2.0 * 1.4426950408889634 / a.cap;
    target.out = a.cap * a.slope;
    target.twice = 2.0 * target.out;
    target.deep = target.twice > 900.0;
  }

  int cur = 0, taken = 1;
  int64_t next = -1;
  if (rank == 0 && tid == 0) a.path[static_cast<int64_t>(b) * a.n] = 0;
  while (true) {
    // The node's next child behind `i`: parents come before children.
    auto child_after = [&](int i) {
      for (++i; i < a.n; ++i)
        if (parents[i] == cur) {
          const int64_t t = tokens[i];
          if (t >= 0 && t < a.vocab) break;
          if (rank == 0 && tid == 0) atomicExch(&g_verify_status, W8_ERR_INVALID_ARG);  // skipped
        }
      return i;
    };
    int went = -1;
    if (a.greedy) {
      next = best_of(cur);
      if (next >= 0)
        for (int c = child_after(cur); c < a.n; c = child_after(c))
          if (tokens[c] == next) {
            went = c;
            break;
          }
    } else {
      const E* xr = row_of(a.x, a.x_b, a.x_n, cur);
      const E* dr = a.d != nullptr ? row_of(a.d, a.d_b, a.d_n, cur) : nullptr;
      int c = child_after(cur);
      bool summed = false;  // the CTAs' parts of what is left stand in shared_a[turn]
      VerifyRow p = stats(xr, target), q = {0.f, 0.f, 1.0, true};
      if (dr != nullptr && c < a.n) q = stats(dr, drafted);
      if (!p.fine) break;
      // After rejections w is max(p - c q, 0) / left: c = 0 and left = 1 at first, and of that less q what
      // is positive is max(p - (c + left) q, 0).
      double c_q = 0.0, left = 1.0;
      int rejected = 0;  // without draft logits: their tokens' weights are taken, `left` stays
      bool sharp = false;  // the sums are in 64 bits
      auto p_of = [&](float x) { return weight_64(x, target, p.top, p.least, table) / p.sum; };
      auto q_of = [&](float x) { return weight_64(x, drafted, q.top, q.least, table) / q.sum; };
      if (q.fine)
        for (; c < a.n; c = child_after(c)) {
          const int64_t t = tokens[c];
          const double uc = static_cast<double>(u[c]);
          const double pt = p_of(logit_f32<E>(xr[t]));
          if (dr == nullptr) {
            bool was = false;
            for (int i = 0; i < rejected; ++i) was |= gone[i] == t;
            if (uc < (was ? 0.0 : left > 0.0 ? pt / left : pt)) {
              went = c;
              break;
            }
            __syncthreads();
            if (!was) {
              if (tid == 0) gone[rejected] = t;
              ++rejected;
              left -= pt;
            }
            __syncthreads();
            continue;
          }
          const double qt = q_of(logit_f32<E>(dr[t]));
          if (uc * qt < fmax(pt - c_q * qt, 0.0) / left) {
            went = c;
            break;
          }
          // Rejected: what is left, in 64 bits.  With the sums of p and q by themselves over the values that
          // stay positive, the first pass gives the sums over all besides: which values stay does not
          // need them so exactly (where p and q are equal to 2^-23, what is left is 2^-23 of them).
          const bool wx = aligned16(xr), wd = aligned16(dr);
          const double to_c = c_q + (rejected == 0 ? 1.0 : left);
          const double rp = 1.0 / p.sum, rq = to_c / q.sum;
          double sp = 0.0, sq = 0.0, over_p = 0.0, over_q = 0.0;
          for (int v = lo + tid * kVerifyVec; v < hi; v += kStep) {
            float x[kVerifyVec], y[kVerifyVec];
            load8<E>(xr, v, hi, wx, x);
            load8<E>(dr, v, hi, wd, y);
#pragma unroll
            for (int i = 0; i < kVerifyVec; ++i) {
              const double pv = weight_64(x[i], target, p.top, p.least, table);
              const double qv = weight_64(y[i], drafted, q.top, q.least, table);
              const bool stays = fma(pv, rp, -(qv * rq)) > 0.0;
              sp += pv, sq += qv;
              over_p += stays ? pv : 0.0;
              over_q += stays ? qv : 0.0;
            }
          }
          if (!sharp) {
            cluster_sums(sp, sq);
            p.sum = sp, q.sum = sq;
            sharp = true;
          }
          block_sums(over_p, over_q);
          exchange(over_p / p.sum - to_c * over_q / q.sum, 0.0);
          double z = 0.0;
          for (int k = 0; k < ranks; ++k) z += fmax(shared_a[turn][k], 0.0);
          ++rejected;
          if (z > 0.0) c_q = to_c, left = z;  // (nothing left: w stays)
          summed = z > 0.0;
        }
      if (went < 0) {
        // ---- the next token: the weights' sum over the CTAs, then the place in one of them
        const bool wx = aligned16(xr), wd = dr != nullptr && aligned16(dr);
        const double rp = 1.0 / p.sum, rq = c_q / q.sum;
        const bool residual = c_q > 0.0;
        auto weights = [&](int v, double (&f)[kVerifyVec]) {
          float x[kVerifyVec], y[kVerifyVec];
          load8<E>(xr, v, hi, wx, x);
          if (residual) load8<E>(dr, v, hi, wd, y);
#pragma unroll
          for (int i = 0; i < kVerifyVec; ++i) {
            f[i] = weight_64(x[i], target, p.top, p.least, table) * rp;
            if (residual) f[i] = fmax(fma(-rq, weight_64(y[i], drafted, q.top, q.least, table), f[i]), 0.0);
          }
          if (dr == nullptr)
            for (int k = 0; k < rejected; ++k)
              if (gone[k] >= v && gone[k] < v + kVerifyVec) {
#pragma unroll
                for (int i = 0; i < kVerifyVec; ++i)
                  if (gone[k] == v + i) f[i] = 0.0;
              }
        };
        double total = left;
        while (!summed) {
          double part = 0.0, none = 0.0;
          for (int v = lo + tid * kVerifyVec; v < hi; v += kStep) {
            double f[kVerifyVec];
            weights(v, f);
#pragma unroll
            for (int i = 0; i < kVerifyVec; ++i) part += f[i];
          }
          block_sums(part, none);
          exchange(part, 0.0);
          total = 0.0;
          for (int k = 0; k < ranks; ++k) total += shared_a[turn][k];
          if (total > 0.0 || rejected == 0) break;
          rejected = 0;  // the weights taken were all there were: the target's own
        }
        const double aim = static_cast<double>(u[0]) * total;
        double before = 0.0;
        int owner = -1, last = -1;
        double owner_before = 0.0, last_before = 0.0;
        for (int k = 0; k < ranks; ++k) {
          const double s = fmax(shared_a[turn][k], 0.0);
          if (s > 0.0) last = k, last_before = before;
          if (owner < 0 && before + s > aim) owner = k, owner_before = before;
          before += s;
        }
        if (owner < 0) owner = last, owner_before = last_before;
        if (owner == rank) {
          if (tid == 0) found = 0x7FFFFFFF;
          __shared__ int positive;
          if (tid == 0) positive = -1;
          double run = owner_before;
          for (int v0 = lo; v0 < hi; v0 += kStep) {
            const int v = v0 + tid * kVerifyVec;
            double f[kVerifyVec], sum = 0.0;
            int end = -1;
            if (v < hi) {
              weights(v, f);
#pragma unroll
              for (int i = 0; i < kVerifyVec; ++i) {
                sum += f[i];
                if (f[i] > 0.0) end = v + i;
              }
            }
            double incl = sum;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
              const double o = __shfl_up_sync(0xffffffffu, incl, s);
              if (lane >= s) incl += o;
            }
            __syncthreads();
            if (lane == 31) wide_a[warp] = incl;
            __syncthreads();
            double base = run, all = 0.0;
#pragma unroll
            for (int w = 0; w < kVerifyWarps; ++w) {
              if (w < warp) base += wide_a[w];
              all += wide_a[w];
            }
            if (end >= 0) atomicMax(&positive, end);
            // (the sums before a thread differ a little from those in it: the first that passes wins)
            if (v < hi && base + incl > aim) {
              double s = base + incl - sum;
#pragma unroll
              for (int i = 0; i < kVerifyVec; ++i) {
                s += f[i];
                if (f[i] > 0.0 && s > aim) {
                  atomicMin(&found, v + i);
                  break;
                }
              }
            }
            run += all;
            __syncthreads();
            if (found != 0x7FFFFFFF) break;
          }
          if (tid == 0) a.token[b] = found != 0x7FFFFFFF ? found : positive;
        } else if (owner < 0 && rank == 0 && tid == 0) {
          a.token[b] = -1;
        }
        next = -2;  // (written)
      }
    }
    if (went < 0) break;
    if (rank == 0 && tid == 0) a.path[static_cast<int64_t>(b) * a.n + taken] = went;
    ++taken;
    cur = went;
    __syncthreads();  // (gone is free)
  }
  if (rank == 0) {
    for (int i = taken + tid; i < a.n; i += kVerifyThreads) a.path[static_cast<int64_t>(b) * a.n + i] = -1;
    if (tid == 0) {
      a.taken[b] = taken;
      if (next != -2) a.token[b] = next;
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

template <typename E>
static int verify_go(w8::VerifyArgs a, int64_t batch, int device, int sms, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(w8::kVerifyThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  static int most[64] = {};  // CTAs of a cluster that the device takes
  if (most[device] == 0) {
    W8_CUDA_TRY(cudaFuncSetAttribute(w8::draft_verify_kernel<E>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cfg.gridDim = dim3(w8::kVerifyCluster, 1, 1);
    attr[0].val.clusterDim.x = w8::kVerifyCluster;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, w8::draft_verify_kernel<E>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      clusters = 0;
    }
    most[device] = clusters > 0 ? w8::kVerifyCluster : 8;
  }
  // CTAs of a sequence: as many as give each an SM to itself (64 bits keep an SM's pipes busy, and two
  // CTAs on some SMs would be what the others wait for), each with at least 2048 values.
  const int64_t fill = std::max<int64_t>(1, sms / batch), fit = std::max<int64_t>(1, a.vocab / 2048);
  const int cluster = static_cast<int>(std::min<int64_t>({most[device], fill, fit}));
  a.per = static_cast<int>(((a.vocab + cluster - 1) / cluster + 7) / 8 * 8);
  cfg.gridDim = dim3(static_cast<unsigned>(batch * cluster), 1, 1);
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, w8::draft_verify_kernel<E>, a));
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
  int device = 0, sms = 0;
  int st = require_sm100(&device);
  if (st != W8_OK) return st;
  st = num_sms(&sms);
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
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (x.dtype == W8_FP32) return verify_go<float>(a, x.batch, device, sms, s);
  if (x.dtype == W8_BF16) return verify_go<__nv_bfloat16>(a, x.batch, device, sms, s);
  return verify_go<__half>(a, x.batch, device, sms, s);
}
