// Inclusive sums over the 32 lanes of a warp, of masses that are not negative. The steps are
// written over a value per lane `L` with add_up(d) (each lane adds what the lane d below had)
// and max_up(d) (the larger of the two), so that the host's checks run the same lines on 32
// numbers.
// The lanes' sums are added up in trees that differ, so that one may come out a last place below
// that of the lane before it; the second loop takes that back. So no goal lies in the parts of two
// lanes. (Rounding keeps order: fl(a + b) <= fl(a + c) for b <= c, so offsets added to all of them
// do too.)
#pragma once

#ifdef __CUDACC__
#define PS_LANES __device__ __forceinline__
#else
#define PS_LANES inline
#endif

namespace onyx {

template <class L>
PS_LANES L ps_prefix_sum(L v) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) v = v.add_up(d);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) v = v.max_up(d);
  return v;
}

}  // namespace onyx
