// Which threads of a CTA say that a running sum reaches a goal, by the kernel's own lines
// (warp_prefix.cuh) and its shuffle scan written out: masses of 512 threads, 32 to a warp.
// own[i]: each thread tests its own interval instead.
#include <cstdint>

#include "../../onyx_b200/csrc/warp_prefix.cuh"

extern "C" void crossings(const double* mass, double goal, int32_t* ends_here, int32_t* own) {
  using namespace onyx;
  constexpr int kWarps = 16;
  double incl[kWarps][32], start[kWarps + 1] = {0.0};
  for (int w = 0; w < kWarps; ++w) {
    double v[32], o[32];
    for (int i = 0; i < 32; ++i) v[i] = mass[32 * w + i];
    for (int d = 1; d < 32; d <<= 1) {
      for (int i = 0; i < 32; ++i) o[i] = i >= d ? v[i] + v[i - d] : v[i];
      for (int i = 0; i < 32; ++i) v[i] = o[i];
    }
    for (int i = 0; i < 32; ++i) incl[w][i] = v[i];
    start[w + 1] = start[w] + v[31];
  }
  for (int w = 0; w < kWarps; ++w) {
    uint32_t reached = 0;
    for (int i = 0; i < 32; ++i)
      if (goal <= ps_part_end(start[w], incl[w][i], start[w + 1])) reached |= 1u << i;
    for (int i = 0; i < 32; ++i) {
      ends_here[32 * w + i] = ps_first_to_reach(reached, i, start[w], goal);
      const double before = i ? start[w] + incl[w][i - 1] : start[w];
      own[32 * w + i] = before < goal && goal <= start[w] + incl[w][i];
    }
  }
}
