// Beam search's selection over beams and vocabulary: the many-beam counterpart of the
// greedy token (gemma_npu.py:291), over the logits of the LM head (gemma_npu.py:170-172)
// with the final softcap (pipeline.py:335-338) fused.
//
//   total(k, t) = scores[k] + y_kt - Z_k,   y = cap tanh(l / cap) (or l),  Z_k = log sum_t e^y
// and per sequence the n largest totals over all (k, t), ties to the lower beam, then the
// lower token.  Within a beam the order of totals is the order of the logits, so one pass
// over the logits yields everything: each CTA streams a chunk of one beam's logits, keeping
// a running maximum and sum of e^y per thread and, in shared memory, the chunk's n best
// (value, token) keys; a second kernel merges the chunks' sorted lists per beam, forms the
// totals in 64 bits and merges the beams.
//
// Bound by reading the logits once.  A logit costs one comparison against the current
// threshold (the n-th best key so far) besides its exponential; only the few that pass it
// go to shared memory.  The first tile's threshold comes from the warps' largest thread
// maxima, later ones from pruning the candidates to n.
#include "common.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace w8 {

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamVals = 16;                              // logits per thread and tile
constexpr int kBeamTile = kBeamThreads * kBeamVals;        // logits per tile
constexpr int kBeamCap = 1024;                             // candidates held in shared memory
constexpr int kBeamPrune = 256;                            // prune after a tile that leaves more
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

template <typename T>
__device__ __forceinline__ float beam_f32(T v);
template <>
__device__ __forceinline__ float beam_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float beam_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float beam_f32<__half>(__half v) {
  return __half2float(v);
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

template <typename T>
__global__ void __launch_bounds__(kBeamThreads) beam_chunk_kernel(const BeamArgs a) {
  __shared__ unsigned long long cand[kBeamCap];
  __shared__ int count;
  __shared__ uint32_t wbest[kBeamWarps];
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
  float mx = -INFINITY, sum = 0.f;  // log2 units
  unsigned long long thr = 0;       // candidates must beat this key
  bool first = true;
  __syncthreads();
  for (int t0 = begin; t0 < end; t0 += kBeamTile) {
    float v[kBeamVals];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int at = t0 + (g * kBeamThreads + tid) * VEC;
      if (vec && at + VEC <= end) {
        const uint4 w = *reinterpret_cast<const uint4*>(x + at);
        const T* p = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[g * VEC + i] = beam_f32<T>(p[i]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[g * VEC + i] = at + i < end ? beam_f32<T>(x[at + i]) : -INFINITY;
      }
    }
    float tm = v[0];
#pragma unroll
    for (int i = 1; i < kBeamVals; ++i) tm = fmaxf(tm, v[i]);
    // ---- e^y
    float y[kBeamVals], ym;
    if (a.cap > 0.f) {
      // cap tanh(l / cap) log2(e), increasing in l
      const float in = 1.f / a.cap, out = a.cap * kLog2e;
#pragma unroll
      for (int i = 0; i < kBeamVals; ++i)  // (an impossible token, or one past the chunk, stays impossible)
        y[i] = v[i] == -INFINITY ? -INFINITY : out * (one_plus_tanh(v[i] * in) - 1.f);
      ym = y[0];
#pragma unroll
      for (int i = 1; i < kBeamVals; ++i) ym = fmaxf(ym, y[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kBeamVals; ++i) y[i] = v[i] * kLog2e;
      ym = tm * kLog2e;
    }
    const float mn = fmaxf(mx, ym), ref = mn == -INFINITY ? 0.f : mn;
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < kBeamVals; ++i) part += ex2_beam(y[i] - ref);
    sum = sum * ex2_beam(mx - ref) + part;
    mx = mn;
    // ---- candidates
    if (first) {
      // Each warp's ceil(n / 8) largest thread maxima are distinct logits: the least over the
      // warps of the last of them has at least n logits at or above it.
      uint32_t u = beam_bits(tm), best = 0;
      for (int i = 0; i < (a.n + kBeamWarps - 1) / kBeamWarps; ++i) {
        best = __reduce_max_sync(0xffffffffu, u);
        const unsigned who = __ballot_sync(0xffffffffu, u == best);
        if (lane == __ffs(who) - 1) u = 0;
      }
      if (lane == 0) wbest[warp] = best;
      __syncthreads();
      best = wbest[0];
#pragma unroll
      for (int i = 1; i < kBeamWarps; ++i) best = min(best, wbest[i]);
      thr = best > 0 ? (static_cast<unsigned long long>(best) << 32) - 1 : 0;  // all keys of `best` pass
      first = false;
    }
    uint32_t todo = 0;
    const uint32_t tb = static_cast<uint32_t>(thr >> 32);
#pragma unroll
    for (int i = 0; i < kBeamVals; ++i)
      if (beam_bits(v[i]) >= tb) todo |= 1u << i;
    while (true) {
      if (todo) {
#pragma unroll
        for (int i = 0; i < kBeamVals; ++i) {
          if (todo & (1u << i)) {
            const int at = t0 + ((i / VEC) * kBeamThreads + tid) * VEC + i % VEC;
            const unsigned long long key = beam_key(v[i], at);
            if (at >= end || key <= thr) {
              todo &= ~(1u << i);
            } else {
              const int p = atomicAdd(&count, 1);
              if (p < kBeamCap) {
                cand[p] = key;
                todo &= ~(1u << i);
              }
            }
          }
        }
      }
      __syncthreads();
      const int c = count;
      if (c <= kBeamPrune) break;
      // Prune; what found no room tries again against the raised threshold.
      const int held = min(c, kBeamCap);
      beam_prune(cand, held, a.n);
      if (held >= a.n) thr = cand[a.n - 1];
      __syncthreads();
      if (tid == 0) count = min(held, a.n);
      __syncthreads();
      if (c <= kBeamCap) break;
    }
  }
  // ---- the chunk's sorted list and its sum
  __syncthreads();
  const int c = min(count, kBeamCap);
  beam_prune(cand, c, a.n);
  unsigned long long* out = a.keys + (static_cast<int64_t>(row) * a.chunks + blockIdx.x) * a.n;
  for (int i = tid; i < a.n; i += kBeamThreads) out[i] = i < c ? cand[i] : 0ull;  // 0: none (below every key)
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
  int* win = token + all;                                                         // [n]: candidate of each rank
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
    // Z: the chunks' sums joined in 64 bits, always in the same order.
    float2 st = make_float2(-INFINITY, 0.f);
    if (lane < a.chunks) st = a.stats[static_cast<int64_t>(row) * a.chunks + lane];
    float mx = st.x;
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    double sum = st.x == -INFINITY ? static_cast<double>(st.y)
                                   : static_cast<double>(st.y) * exp2(static_cast<double>(st.x) - static_cast<double>(mx));
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
    unsigned long long* mine = list + warp * a.chunks * a.n;
    const unsigned long long* src = a.keys + static_cast<int64_t>(row) * a.chunks * a.n;
    for (int i = lane; i < a.chunks * a.n; i += 32) mine[i] = src[i];
    __syncwarp();
    int head = 0;
    unsigned long long key = lane < a.chunks ? mine[lane * a.n] : 0ull;
    for (int i = 0; i < m; ++i) {
      const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32));
      const bool top = static_cast<uint32_t>(key >> 32) == hi;
      const uint32_t lo = __reduce_max_sync(0xffffffffu, top ? static_cast<uint32_t>(key) : 0u);
      if (top && static_cast<uint32_t>(key) == lo) {  // keys are distinct: one lane (m <= vocab: never a 0 key)
        const double l = static_cast<double>(beam_value(hi));
        const double y = a.cap > 0.f && !isinf(l) ? static_cast<double>(a.cap) * tanh(l / static_cast<double>(a.cap))
                         : l > 0.0 && a.cap > 0.f  ? static_cast<double>(a.cap)
                                                   : l;
        const double t = score + (y - z);
        token[k * m + i] = static_cast<int>(0xFFFFFFFFu - lo);
        total[k * m + i] = isfinite(t) ? t : -INFINITY;
        ++head;
        key = head < a.n ? mine[lane * a.n + head] : 0ull;
      }
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
  for (int e = tid; e < all; e += kMergeThreads) {
    const int k = e / m;
    const double t = total[e];
    int rank = e % m;
    for (int o = 0; o < a.beams && rank < a.n; ++o) {
      if (o == k) continue;
      // how many of beam o's list come before (ties: the lower beam)
      int lo = 0, hi = m;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const double v = total[o * m + mid];
        if (v > t || (v == t && o < k)) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    if (rank < a.n) win[rank] = e;
  }
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

// Chunks of whole tiles, at most 32 (a warp merges one list per lane): enough CTAs for four
// per SM over all rows, or as many as there are tiles.
static BeamPlan beam_plan(int64_t rows, int64_t vocab, int sms) {
  const int64_t tiles = std::max<int64_t>(1, (vocab + w8::kBeamTile - 1) / w8::kBeamTile);
  const int64_t want = std::max<int64_t>(1, (static_cast<int64_t>(sms) * 4 + rows - 1) / std::max<int64_t>(rows, 1));
  const int64_t n = std::min<int64_t>({tiles, want, w8::kBeamMaxChunks});
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
  if (dtype == W8_FP32)
    st = launch_beam(w8::beam_chunk_kernel<float>, grid, w8::kBeamThreads, 0, s, a);
  else if (dtype == W8_BF16)
    st = launch_beam(w8::beam_chunk_kernel<__nv_bfloat16>, grid, w8::kBeamThreads, 0, s, a);
  else
    st = launch_beam(w8::beam_chunk_kernel<__half>, grid, w8::kBeamThreads, 0, s, a);
  if (st != W8_OK) return st;
  const int64_t all = static_cast<int64_t>(a.beams) * a.m;
  const int smem = static_cast<int>(all * 12 + static_cast<int64_t>(w8::kMergeWarps) * p.chunks * n * 8 + n * 4 + 16);
  static bool done[64] = {};
  if (!done[device]) {
    // Largest: 32 beams x 64 candidates, 8 warps x 32 chunks x 64 keys.
    W8_CUDA_TRY(cudaFuncSetAttribute(w8::beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    done[device] = true;
  }
  return launch_beam(w8::beam_merge_kernel, dim3(static_cast<unsigned>(batch)), w8::kMergeThreads, smem, s, a);
}
