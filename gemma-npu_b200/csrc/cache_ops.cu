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
};

constexpr int kAppendRows = 16;  // path entries per CTA

// One CTA: up to 16 path entries of one (sequence, cache head).  An entry counts if no
// entry up to it is negative.
__global__ void __launch_bounds__(256) cache_append_kernel(const AppendArgs a) {
  __shared__ int draft[kAppendRows];
  __shared__ int ended;
  const int b = blockIdx.x / a.kv_heads, c = blockIdx.x % a.kv_heads, tid = threadIdx.x;
  const int j0 = blockIdx.y * kAppendRows, j1 = min(j0 + kAppendRows, a.steps);
  pdl_launch_dependents();
  pdl_wait();
  int count = a.steps;  // entries before the first negative one
  if (a.path != nullptr) {
    if (tid == 0) ended = a.steps;
    __syncthreads();
    const int upto = blockIdx.y == 0 && c == 0 ? a.steps : j1;  // the first CTA counts them all
    for (int j = tid; j < upto; j += 256)
      if (a.path[b * a.path_b + j] < 0) atomicMin(&ended, j);
    __syncthreads();
    count = ended;
  }
  const int len = a.lens[b];
  const bool ok = len >= 0 && len <= a.slots;
  if (!ok && tid == 0) cache_bad_index();
  if (c == 0 && blockIdx.y == 0 && tid == 0) {
    a.lens_out[b] = ok ? min(len + count, a.slots) : len;
    if (ok && len + count > a.slots) cache_bad_index();
  }
  if (!ok) return;
  if (tid < j1 - j0) {
    const int j = j0 + tid;
    int d = -1;
    if (j < count && len + j < a.slots) {
      d = a.path != nullptr ? a.path[b * a.path_b + j] : j;
      if (d >= a.n) {
        cache_bad_index();
        d = -1;
      }
    }
    draft[tid] = d;
    if (d >= 0) {
      if (a.w != nullptr) a.w[b * a.w_b + c * a.w_h + len + j] = a.wn != nullptr ? a.wn[b * a.wn_b + c * a.wn_h + d] : 0.f;
      if (a.pos != nullptr) a.pos[b * a.pos_b + c * a.pos_h + len + j] = a.seen[b] + j;
    }
  }
  __syncthreads();
  const int work = (j1 - j0) * 2 * a.chunks;
  for (int e = tid; e < work; e += 256) {
    const int ch = e % a.chunks, row = e / a.chunks, j = row >> 1, d = draft[j];
    if (d < 0) continue;
    const bool is_v = row & 1;
    const uint8_t* src = is_v ? a.vn + b * a.vn_b + c * a.vn_h + d * a.vn_t : a.kn + b * a.kn_b + c * a.kn_h + d * a.kn_t;
    uint8_t* dst = is_v ? a.v + b * a.v_b + c * a.v_h + static_cast<int64_t>(len + j0 + j) * a.v_s
                        : a.k + b * a.k_b + c * a.k_h + static_cast<int64_t>(len + j0 + j) * a.k_s;
    reinterpret_cast<uint4*>(dst)[ch] = reinterpret_cast<const uint4*>(src)[ch];
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
};

constexpr int kEvictThreads = 1024;

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

// Which slots of one (sequence, cache head) stay: the `budget` largest by (protected,
// weight, lower slot), by a radix selection of the budget-th key, then one pass in slot
// order that pairs the i-th evicted slot below the budget with the i-th kept slot behind it.
__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(const EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int warp_sums[32];
  __shared__ int pick[2];
  const int row = blockIdx.x, b = row / a.kv_heads, c = row % a.kv_heads, tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const float* w = a.w + b * a.w_b + c * a.w_h;
  const int* pos = a.pos + b * a.pos_b + c * a.pos_h;
  float* w_out = a.w_out + b * a.wo_b + c * a.wo_h;
  int* pos_out = a.pos_out + b * a.po_b + c * a.po_h;
  int* moves = a.moves + static_cast<int64_t>(row) * (1 + 2 * a.most);
  int len = a.lens[b];
  if (len < 0 || len > a.slots) {
    if (tid == 0) cache_bad_index();
    len = len < 0 ? 0 : a.slots;
  }
  const int left = min(len, a.budget);
  if (c == 0 && tid == 0) a.lens_out[b] = left;
  int count = 0;
  if (len > a.budget) {
    // The highest position decides what is recent.
    int last = INT32_MIN;
    for (int s = tid; s < len; s += kEvictThreads) last = max(last, pos[s]);
    last = __reduce_max_sync(0xffffffffu, last);
    if ((tid & 31) == 0) warp_sums[tid >> 5] = last;
    __syncthreads();
    last = __reduce_max_sync(0xffffffffu, warp_sums[tid & 31]);
    __syncthreads();
    const int64_t recent_from = static_cast<int64_t>(last) - a.recent + 1;
    auto key = [&](int s) {
      const int p = pos[s];
      return p < a.sink || p >= recent_from ? 0xFFFFFFFFu : weight_key(w[s]);
    };
    uint32_t prefix = 0;
    int need = a.budget;  // keys still to take among those that share the prefix
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
      for (int s = tid; s < len; s += kEvictThreads) {
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
    for (int s0 = 0; s0 < len; s0 += kEvictThreads) {
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
  if (tid == 0) moves[0] = count;
  // The small state: kept slots as they are, holes from their movers, nothing behind.
  if (w_out != w || pos_out != pos)
    for (int s = tid; s < left; s += kEvictThreads) {
      const float ws = w[s];
      const int ps = pos[s];
      w_out[s] = ws;
      pos_out[s] = ps;
    }
  __syncthreads();
  for (int i = tid; i < count; i += kEvictThreads) {
    const int dst = moves[1 + i], src = moves[1 + a.most + i];
    w_out[dst] = w[src];
    pos_out[dst] = pos[src];
  }
  __syncthreads();
  for (int s = left + tid; s < a.slots; s += kEvictThreads) {
    w_out[s] = 0.f;
    pos_out[s] = -1;
  }
}

struct MoveArgs {
  uint8_t *k, *v;
  int64_t k_b, k_h, k_s, v_b, v_h, v_s;  // bytes
  const int* moves;
  int most, kv_heads, chunks;
};

// The moves of one (sequence, head): destinations (below the budget) and sources (behind
// it) are disjoint, so the rows move in place in any order.
__global__ void __launch_bounds__(256) evict_move_kernel(const MoveArgs a) {
  const int row = blockIdx.y, b = row / a.kv_heads, c = row % a.kv_heads;
  pdl_launch_dependents();
  pdl_wait();
  const int* moves = a.moves + static_cast<int64_t>(row) * (1 + 2 * a.most);
  const int count = moves[0];
  uint8_t* k = a.k + b * a.k_b + c * a.k_h;
  uint8_t* v = a.v + b * a.v_b + c * a.v_h;
  const int64_t work = static_cast<int64_t>(count) * 2 * a.chunks;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < work; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int ch = static_cast<int>(e % a.chunks);
    const int64_t m = e / a.chunks;
    const int i = static_cast<int>(m >> 1);
    const int64_t dst = moves[1 + i], src = moves[1 + a.most + i];
    uint8_t* base = (m & 1) ? v : k;
    const int64_t pitch = (m & 1) ? a.v_s : a.k_s;
    reinterpret_cast<uint4*>(base + dst * pitch)[ch] = reinterpret_cast<const uint4*>(base + src * pitch)[ch];
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
// cache and a beam that stays costs nothing.
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
static int launch_cache(Kern kern, dim3 grid, int threads, cudaStream_t stream, const Args& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, a));
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
  W8_CHECK_ARG(x.n_new >= 0 && x.steps >= 0 && x.n_new < (1ll << 20) && x.steps <= 16 * 65535, "size beyond the limits");
  W8_CHECK_ARG(x.path != nullptr || x.steps == x.n_new, "without a path every new token is appended (steps = n_new)");
  if (x.batch == 0) return W8_OK;
  W8_CHECK_ARG(x.lens && x.lens_out, "null lens");
  W8_CHECK_ARG(x.lens != x.lens_out, "lens_out must not be lens");
  W8_CHECK_ARG(!x.positions || x.seen, "positions need seen");
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
  const int64_t parts = std::max<int64_t>(1, (x.steps + w8::kAppendRows - 1) / w8::kAppendRows);
  return launch_cache(w8::cache_append_kernel,
                      dim3(static_cast<unsigned>(x.batch * x.kv_heads), static_cast<unsigned>(parts)), 256,
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
  W8_CHECK_ARG(x.lens != x.lens_out, "lens_out must not be lens");
  if (x.slots > 0) {
    W8_CHECK_ARG(x.weights && x.positions && x.weights_out && x.positions_out, "null weights or positions");
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
  st = launch_cache(w8::evict_select_kernel, dim3(static_cast<unsigned>(rows)), w8::kEvictThreads, s, e);
  if (st != W8_OK || most == 0) return st;
  w8::MoveArgs m = {};
  m.k = static_cast<uint8_t*>(x.k), m.v = static_cast<uint8_t*>(x.v);
  m.k_b = x.k_stride[0], m.k_h = x.k_stride[1], m.k_s = x.k_stride[2];
  m.v_b = x.v_stride[0], m.v_h = x.v_stride[1], m.v_s = x.v_stride[2];
  m.moves = e.moves, m.most = e.most, m.kv_heads = e.kv_heads, m.chunks = static_cast<int>(x.row_bytes / 16);
  const int64_t blocks = (most * 2 * m.chunks + 255) / 256;
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
