// Counts, turn by turn, the copies that one warp's ring starts, with the lines that the kernel
// runs (policy_ring.cuh). out[0]: copies of chunks that are not the warp's own; out[1]: copies
// not waited for when the loop ends; out[2]: chunks of the part that were never copied, or not
// landed when they are read.
#include <cstdint>
#include <vector>

#include "../../onyx_b200/csrc/policy_ring.cuh"

extern "C" void ring_copies(int id_first, int n, int vocab, int chunk, int depth, int64_t* out) {
  using namespace onyx;
  const PsInner in = ps_inner_chunks(id_first, n, vocab, chunk);
  std::vector<int> groups;  // the chunk of every group, -1: an empty one
  out[0] = out[1] = out[2] = 0;
  for (int i = 0; i < depth - 1; ++i) groups.push_back(i < n ? i : -1);
  size_t landed = 0;
  for (int i = 0; i < n; ++i) {
    const int next = i + depth - 1;
    const bool some = ps_copies_inner(next, in) || ps_copies_edge(next, n);
    groups.push_back(some ? next : -1);
    out[0] += some && next >= n;
    landed = groups.size() - (depth - 1);  // all but the latest depth - 1
    out[2] += !((size_t)i < landed && groups[i] == i);
  }
  for (size_t i = landed; n && i < groups.size(); ++i) out[1] += groups[i] >= 0;
}
