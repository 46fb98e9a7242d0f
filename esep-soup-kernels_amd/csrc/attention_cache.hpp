// What the walks over a cache (attention_cache.hip) and over pages (attention_paged.hip) share: the tiles of all
// groups laid end to end and cut into one run to a wavefront, the waits of a wavefront's own ring, the join's
// large blocks.
#pragma once

#include "attention.hpp"

namespace esep {

// The walk's geometry, found by every wavefront from the lengths: the tiles of all groups, dealt to `units`
// wavefronts, the first `extra` of them one more than `each`.
struct CachePlan {
  int total, units, each, extra;
  __device__ __forceinline__ int cut(int u) const { return u * each + (u < extra ? u : extra); }
  __device__ __forceinline__ int unit_of(int x) const {
    const int split = extra * (each + 1);
    return x < split ? x / (each + 1) : extra + (x - split) / each;
  }
};
__device__ __forceinline__ int lane_sum(int v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ CachePlan cache_plan(int tiles, int D) {
  CachePlan p;
  p.total = tiles;
  p.units = (int)cache_units(tiles, D);
  p.each = p.units > 0 ? tiles / p.units : 0;
  p.extra = tiles - p.each * p.units;
  return p;
}

// s_waitcnt vmcnt(N) and lgkmcnt(0) (the other counters at their maxima).
constexpr int wait_vm(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }
constexpr int kWaitLgkm0 = 0xC07F;

// Parts of a group from which its rows, where there are no more than CUs, are joined by blocks of 1024 threads
// instead of 256 (12 rows of 512 parts each 17 -> 5.5 us; 896 rows of 27 4.9 -> 8.7).
constexpr int64_t kCacheManyParts = 24;

}  // namespace esep
