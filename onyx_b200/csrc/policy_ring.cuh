// The copies that a warp starts while it streams its part of a row through a ring of slots.
// Plain C++ on integers: the kernel and the host's checks run the same lines. A warp copies its own
// chunks alone, so that the last turns start nothing and no copy is on its way when the loop ends:
// the lists of the later passes lie over the ring.
#pragma once

#ifdef __CUDACC__
#define PS_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define PS_HOST_DEVICE inline
#endif

namespace onyx {

// Of the chunks 0 to n - 1 of a warp's part, the first of which starts at id `id_first` (negative
// where the row starts inside it), those that lie whole inside the row: [from, to).
struct PsInner {
  int from, to;
};
PS_HOST_DEVICE PsInner ps_inner_chunks(int id_first, int n, int vocab, int chunk) {
  PsInner in;
  in.from = id_first < 0 ? 1 : 0;
  const int left = vocab - (id_first + in.from * chunk);
  in.to = in.from + (left > 0 ? left / chunk : 0);
  if (in.to > n) in.to = n;  // the chunks behind are the next warp's
  return in;
}

// Whether the ring copies chunk `next` when it comes up, as one inside the row, or else as one of
// its own at an edge of the row. (Two tests in the loop: with the answer as one value of three,
// 1,024 rows of 256,000 bfloat16 took 396 us, so 387.)
PS_HOST_DEVICE bool ps_copies_inner(int next, const PsInner& in) {
  return next >= in.from && next < in.to;
}
PS_HOST_DEVICE bool ps_copies_edge(int next, int n) { return next < n; }

}  // namespace onyx
