// lss_scan.cuh — sums over the rows of a batch, one CTA at a time.
#pragma once

#include "lss_common.cuh"

namespace lss {

constexpr int BL_NT = 1024;    // threads per CTA
constexpr int BL_MAXCL = 8;    // CTAs (one cluster)

// Exclusive scan of one value per thread over BL_NT threads; `total` gets the sum.
__device__ __forceinline__ int64_t bl_scan(int64_t v, int64_t* scr, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) scr[warp] = x;
  __syncthreads();
  int64_t s = scr[lane];  // BL_NT / 32 == 32 warps: one sum per lane
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  total = __shfl_sync(0xffffffffu, s, 31);
  const int64_t before = __shfl_sync(0xffffffffu, s, warp > 0 ? warp - 1 : 0);
  return (warp > 0 ? before : 0) + x - v;
}

// Blocks of 0 <= tokens <= 2^30 (a table's width): a 32-bit division.
__device__ __forceinline__ int blocks_of(int tokens, int bs) { return (int)((unsigned)(tokens + bs - 1) / (unsigned)bs); }

}  // namespace lss
