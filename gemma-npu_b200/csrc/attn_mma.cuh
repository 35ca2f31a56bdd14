// Shared by the attention kernels on warp-level tensor instructions (mma.sync): their operand
// loads, the 16-bit products, and how tiles of ragged sequences are dealt to CTAs.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace w8 {

constexpr int kTreeWarps = 8;
constexpr int kTreeThreads = 32 * kTreeWarps;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// Arrive on `bar` once every earlier cp.async of this thread has landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Quotient of a number that is seldom above 32 bits (a 64-bit division is a call of some 150
// instructions).
__device__ __forceinline__ long long div_short(long long x, uint32_t by) {
  return (x >> 32) == 0 ? static_cast<long long>(static_cast<uint32_t>(x) / by) : x / by;
}

// How `total` tiles are dealt to `ctas`: the first `more` CTAs hold one more than the others.
struct TreeDeal {
  long long each, more;
};
__device__ __forceinline__ long long deal_begin(const TreeDeal& d, long long u) {
  return u * d.each + (u < d.more ? u : d.more);
}
__device__ __forceinline__ int deal_owner(const TreeDeal& d, long long tile) {
  const long long wide = d.more * (d.each + 1);
  return static_cast<int>(tile < wide ? div_short(tile, static_cast<uint32_t>(d.each + 1))
                                      : d.more + div_short(tile - wide, static_cast<uint32_t>(d.each)));
}

// Exclusive prefix sum over a block of WARPS warps and the block's sum.
template <int WARPS>
__device__ __forceinline__ long long block_scan(long long v, long long* sm, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    if (i < warp) before += sm[i];
    total += sm[i];
  }
  __syncthreads();
  return before + x - v;
}

}  // namespace w8
