// Where a running sum of masses reaches a goal, over the threads of a CTA: which thread says so.
// Plain C++ on a lane's numbers; the kernel and the host's checks run the same lines.
//
// A warp's lanes hold inclusive sums of their masses by a shuffle scan, whose sums are added up in
// trees that differ: one may come out a last place below that of the lane before it, and an inner
// one above the warp's whole sum. So a test of each lane's own interval can hold for two lanes, or
// for lanes of two warps. Here the warps' starts, which are added up one after the other and never
// fall, choose the warp, and the first lane whose end reaches the goal is the one.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define PS_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define PS_HOST_DEVICE inline
#endif

namespace onyx {

// End of a lane's part: the warp's start and the lane's sum, no later than the warp's end.
PS_HOST_DEVICE double ps_part_end(double warp_start, double incl, double warp_end) {
  const double end = warp_start + incl;
  return end < warp_end ? end : warp_end;
}

// `reached`: the lanes whose end is at the goal or past it.
PS_HOST_DEVICE bool ps_first_to_reach(uint32_t reached, int lane, double warp_start, double goal) {
  return warp_start < goal && (reached & (0u - reached)) == 1u << lane;
}

}  // namespace onyx
