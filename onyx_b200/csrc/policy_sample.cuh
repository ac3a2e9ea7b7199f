// Sampling under a policy of its own for each row: temperature, top-k, top-p and min-p, with
// the random numbers given by the caller. Three operators share the row's distribution:
//   draw   one id per row;
//   probs  the filtered, renormalised probabilities of every id;
//   spec   speculative sampling of drafted tokens (rows gamma + 1 to an entry).
//
// Mathematics. For the valid ids of a row with maximum m, weight w(v) = exp((v - m) / T)
// (T = 0: the first maximum alone; any +inf: the +inf ids alone, with equal weights). Ids are
// ranked by (value falling, id rising). top-k keeps the first k; top-p keeps the shortest
// prefix of those whose mass reaches p times their mass; min-p keeps w >= min_p. All three
// keep a prefix of the ranking, so the kept set is a cut: the values above `cut`, of the ids
// equal to it the first `take` in id order, and w >= min_p. The draw is the first kept id, in
// id order, whose cumulative weight exceeds u times the kept total.
//
// Sums and weights are float64: whether a cumulative mass reaches p, or an id's interval holds
// u, decides a whole number, and float32 sums over 10^5 ids would decide it differently for
// about one row in a hundred.
//
// Shape of the work. One cluster of k CTAs per row (k = 1, 2, 4 or 8, the more the fewer the
// rows), 512 threads each, two CTAs to an SM; CTA ranks, the warps of a CTA and the 256-id
// chunks of a warp follow id order, a lane holding 8 consecutive ids (one or two 16-byte
// vectors in memory, whatever the row's alignment).
//   1  first_pass(): each warp copies its part of the row into shared memory (cp.async, all of
//      it at once where it fits, else through a ring) and finds the maximum, the maximum of
//      every 8 ids (the peaks, which stay in shared memory) and, as the policy asks, a
//      histogram of 4,096 bins and the sum of the weights. The only pass over all values.
//   2  The histograms of the CTAs are added up (each CTA a part of the bins, over distributed
//      shared memory) and every CTA scans the bins in falling order of value.
//      bfloat16 (cut_by_values): a bin is one value, its mass count times weight, and the scan
//      yields the cut. No weight is computed for an id: 8 bins share two exponentials.
//      float32, float16 (range_by_bins): bins of 1/64 in the exponent around a sample of the
//      row. They yield the few bins that hold the cut; a small top-k takes a histogram of the
//      peaks instead (range_by_peaks).
//   3  cut_from_list(), float32 and float16: the ids of those bins (a few dozen to a few
//      hundred) are listed, sorted by value and summed exactly.
//   4  The kept mass is summed by warps over lists of the vectors whose peak reaches the cut,
//      the warps' sums are scanned, and the warp whose interval holds u draws (a long list is
//      drawn by all warps of its CTA, piece by piece).
// Rows that steps 2 and 3 cannot serve (bfloat16 values of 2^7 and more, a cut among values
// next to zero, float32 maxima 40 T above the sample, lists over 1,024 ids) go through
// find_cut(): a list of the ids of the largest peaks, and where that does not reach the goal the
// histogram over ranges of order codes, each turn a 4096th of the last. No row length is bound
// to shared memory.
//
// Every CTA of a cluster computes the same totals from the same parts in the same order, so
// all take the same branches, and the result does not depend on timing. (Histograms are counts,
// whose sums do not depend on the order of the atomics; lists are sorted by value and id.)
//
// What bounds it. 256 rows of 128,256 bfloat16 (65.7 MB, 10.2 us of copying at 6,464 GB/s), one
// policy for all: instructions, and CTAs that fill 1.73 waves of the 296 that fit. The maximum
// alone takes 32 us and 153 warp instructions a chunk of 256 ids, over the whole kernel; with
// top-k 50, so with the histogram and its cut, 65 us and 341, the histogram's atomics meeting 2.8
// bank conflicts each; DRAM is 20 and 11 % busy, the issue slots 57 and 64 %. 64 rows of 151,664
// float32 (0.86 waves) take 24 us for the maximum, 37 with the sum of the weights and 69 under
// top-p 0.9, 963 instructions a chunk, 131 of them float64. One bfloat16 row of 128,256 takes
// 15.6 us under top-p 0.9: a chain of latencies, 8 us of it without any histogram. A batch under
// mixed policies waits for its slowest rows, those that keep tens of thousands of ids (256
// rows at T = 1.2, top-p 0.95: 138 us, against 75 under T = 0.8, top-p 0.9).
//
// Registers. Two CTAs of 512 threads leave 64 to a thread, and the kernels spill: bytes stored and
// reloaded a thread, of draw, probs and spec, float32 132/868, 140/620, 388/1,700; float16 224/960,
// 232/608, 332/1,596; bfloat16 16/104, 60/232, 56/148. Other widths have not been measured.
#pragma once

#include <cfloat>

#include "onyx_common.cuh"
#include "policy_ring.cuh"
#include "warp_prefix.cuh"

namespace onyx {

constexpr int kPsThreads = 512;
constexpr int kPsWarps = kPsThreads / 32;
constexpr int kPsMaxCluster = 8;
constexpr int kPsEntries = kPsMaxCluster * kPsWarps;
constexpr int kPsChunk = 256;  // ids a warp handles at a time, 8 to a lane
constexpr int kPsUnits = 256;  // pieces at most into which the drawing CTA cuts a warp's part

// The value histogram: one bin for every bf16 value with 2^-9 <= |v| < 2^7, in falling order
// of value; positive ones first. The values next to zero, |v| < 2^-9, lie between the halves.
constexpr int kPsBins = 4096;
constexpr int kPsHalf = kPsBins / 2;
constexpr uint32_t kPsLow = 0x3B00u;  // bf16 bits of 2^-9
constexpr float kPsSmall = 0x1p-9f, kPsLarge = 0x1p7f;
constexpr int kPsOwn = kPsBins / kPsThreads;  // bins a thread scans
constexpr uint32_t kPsList = 1024;            // ids sorted at most

enum PolicyOp : int { kOpDraw = 0, kOpProbs = 1, kOpSpec = 2 };

struct PolicyParams {
  const void* logits;
  int64_t group_stride;  // elements between entries (spec) or rows
  int64_t row_stride;    // elements between the rows of one entry (spec)
  int64_t vocab;
  const uint32_t* mask;  // nullptr: every id valid
  int64_t mask_group_stride, mask_row_stride;  // words
  const double* policies;  // temperature, top_k, top_p, min_p
  int64_t policy_stride;   // doubles between entries, 0: one policy for all
  const void* uniforms;
  int64_t uniform_stride;
  int32_t uniform_f64;
  int32_t per_group;  // rows per entry: 1, or gamma + 1
  int32_t sub_from, sub_count;  // spec: rows of every entry that this launch takes
  int32_t* out_idx;
  uint32_t* out_status;
  float* out_probs;
  int64_t out_stride;
  const int32_t* drafts;
  int64_t draft_stride;
  const float* draft_probs;  // nullptr: each draft has probability 1
  int64_t dp_group_stride, dp_row_stride;
  const int32_t* draft_lens;  // nullptr: gamma drafts for every entry
  int4* results;              // spec: {verdict, token, status, 0} of every row
  int32_t warp_ids;  // ids per warp, a multiple of kPsChunk
  int32_t k;         // CTAs per row
  int32_t peaks;     // the peaks are kept (else their place is empty)
  int32_t keep;      // shared memory holds all chunks of a CTA's part
  int32_t slots;     // where in dynamic shared memory the chunks' slots begin,
  int32_t lists;     // and the lists of the warps (over a ring, whose copies have landed by then)
};

enum Verdict : int { kAccepted = 0, kDecided = 1 };

struct RowPolicy {
  double temperature, top_p, min_p;
  uint32_t top_k;  // 0: off
  bool ok;
};

__device__ __forceinline__ RowPolicy load_policy(const double* p) {
  RowPolicy r;
  r.temperature = p[0];
  const double k = p[1];
  r.top_p = p[2];
  r.min_p = p[3];
  // comparisons are written so that a NaN fails them
  r.ok = r.temperature >= 0.0 && r.temperature < INFINITY && k >= 0.0 && k < INFINITY &&
         r.top_p > 0.0 && r.top_p <= 1.0 && r.min_p >= 0.0 && r.min_p <= 1.0 && k == floor(k);
  r.top_k = r.ok ? (k < 4294967295.0 ? (uint32_t)k : 0xFFFFFFFFu) : 0u;
  return r;
}

__device__ __forceinline__ double load_uniform(const PolicyParams& p, int64_t i) {
  return p.uniform_f64 ? static_cast<const double*>(p.uniforms)[i]
                       : (double)static_cast<const float*>(p.uniforms)[i];
}

__device__ __forceinline__ void ps_cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void ps_cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t ps_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
template <class T>
__device__ __forceinline__ T* ps_remote(T* p, uint32_t rank) {
  unsigned long long out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(p), "r"(rank));
  return reinterpret_cast<T*>(out);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}
__device__ __forceinline__ double warp_scan(double v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double o = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += o;
  }
  return v;
}
__device__ __forceinline__ uint32_t warp_scan(uint32_t v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// 2^(j/16), filled by every CTA when it starts.
struct PsPowers {
  double at[16];
};

struct PsBox {  // one CTA's part of a cluster-wide reduction
  double mass;
  uint32_t count, top, small;
};

struct PsCross {  // the bin in which a count or a mass is reached
  double mass;     // ahead of it
  uint32_t count;  // ahead of it
  uint32_t n;      // ids in it
  int bin;
};

struct PsScan {  // of the entries of all warps
  double total;
  double mass_before;     // kept mass before the owner's ids ...
  uint32_t ties_before;   // ... and ids at the cut before them
  uint32_t draft_before;  // ids at the cut before the draft
  int owner;  // entry whose interval of kept mass holds u times the total
};

struct PsShared {
  PsBox box[2][kPsMaxCluster];  // used alternately: one may still be read as the next is written
  double part_mass[kPsWarps];
  uint32_t part_count[kPsWarps], part_top[kPsWarps], part_small[kPsWarps];
  // one entry per warp of the cluster, in id order; the second set holds what max(p - q, 0)
  // leaves
  double entry_mass[2][kPsEntries];
  uint32_t entry_ties[kPsEntries], entry_before[kPsEntries];
  PsPowers powers;
  PsCross cross[9];
  uint32_t listed[kPsMaxCluster];  // ids that each CTA listed
  uint32_t list_fill;
  int listed_by[kPsWarps];  // vectors that each warp gathered for the passes after the cut
  PsScan scan[2];
  uint32_t ties_before[kPsWarps];
  double sums_before[kPsWarps + 1];
  uint32_t sample[2][4];
};

// Dynamic shared memory: the CTA's histogram and the cluster's; their 32 KB are used again for a
// list and its sorted form, and for the weights of the bins. Then the sums of the pieces of a
// draw, the peaks, and last the slots into which the warps copy their part of the row: all of
// its chunks where they fit (the later passes read them there), else a ring of
// ps_depth().
extern __shared__ __align__(16) unsigned char ps_dynamic[];
constexpr size_t kPsArea = kPsBins * sizeof(uint32_t);
__device__ __forceinline__ uint32_t* ps_hist() { return reinterpret_cast<uint32_t*>(ps_dynamic); }
__device__ __forceinline__ uint32_t* ps_merged() {
  return reinterpret_cast<uint32_t*>(ps_dynamic + kPsArea);
}
__device__ __forceinline__ unsigned long long* ps_list() {
  return reinterpret_cast<unsigned long long*>(ps_dynamic);
}
__device__ __forceinline__ unsigned long long* ps_sorted() {
  return reinterpret_cast<unsigned long long*>(ps_dynamic + kPsArea);
}
__device__ __forceinline__ double* ps_table() { return reinterpret_cast<double*>(ps_dynamic); }
__device__ __forceinline__ double* ps_unit_mass() {
  return reinterpret_cast<double*>(ps_dynamic + 2 * kPsArea);
}
__device__ __forceinline__ uint32_t* ps_unit_ties() {
  return reinterpret_cast<uint32_t*>(ps_dynamic + 2 * kPsArea + kPsUnits * sizeof(double));
}
// bytes ahead of the peaks
constexpr size_t kPsFixed = 2 * kPsArea + kPsUnits * (sizeof(double) + sizeof(uint32_t));
// A slot: a chunk's values, and its mask words where there is a mask.
__host__ __device__ constexpr int ps_slot(int dt, bool masked) {
  return kPsChunk * (dt == kF32 ? 4 : 2) + (masked ? 48 : 0);
}
// slots of a ring
__host__ __device__ constexpr int ps_depth(int dt) { return dt == kF32 ? 3 : 4; }

__device__ __forceinline__ void ps_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 4 bytes, or zeros
__device__ __forceinline__ void ps_copy4(uint32_t dst, const void* src, bool have) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(have ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ uint4 ps_load16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(at)
               : "memory");
  return r;
}
__device__ __forceinline__ uint32_t ps_load4(uint32_t at) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(at) : "memory");
  return r;
}
__device__ __forceinline__ void ps_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ps_await() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// waits until at most `ahead` of the latest groups are on their way (or fewer)
__device__ __forceinline__ void ps_await_all_but(int ahead) {
  if (ahead >= 8) ps_await<8>();
  else if (ahead >= 4) ps_await<4>();
  else if (ahead >= 2) ps_await<2>();
  else if (ahead == 1) ps_await<1>();
  else ps_await<0>();
}

// The part of a row that one warp owns, and how it is read. Ids are counted by positions:
// position = id + off, where `off` values lie between the 16-byte boundary at or before the
// row's start and the start. So 8 positions from a multiple of 8 are 16-byte vectors in memory
// whatever the row's alignment; those with an id outside the row are read value by value.
template <int DT>
struct RowView {
  using S = typename Elem<DT>::storage;
  static constexpr int kData = kPsChunk * (int)sizeof(S), kDepth = ps_depth(DT);
  const S* row;
  const uint32_t* mask;
  uint16_t* peaks;  // of this CTA: the peaks (see peak()) of every 8 positions, or null
  uint16_t* list;   // vectors of 8 of this part that the last gather() found,
  int listed;       // so many (without peaks: all)
  uint32_t base;    // the CTA's first position
  uint32_t begin, end;  // positions; multiples of kPsChunk, but for the row's end
  int vocab, off;
  uint32_t slots;  // of the CTA's chunks in order, if all are kept, else of the warp's ring
  int slot_bytes;
  bool kept;  // all chunks are kept

  struct Raw {  // the values at 8 positions as loaded
    uint4 a, b;
    uint32_t bits;  // which of them are valid
  };

  __device__ __forceinline__ int id_of(uint32_t pos) const { return (int)pos - off; }

  // of the 8 ids from `id` on, those inside the row
  __device__ __forceinline__ uint32_t inside(int id) const {
    uint32_t bits = 0xFFu;
    if (id < 0) bits = 0xFFu << min(-id, 8) & 0xFFu;
    const int left = vocab - id;
    if (left < 8) bits &= left > 0 ? (1u << left) - 1u : 0u;
    return bits;
  }

  __device__ __forceinline__ void load_edge(Raw& r, int id) const {
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] = 0u;
      if (id + j >= 0 && id + j < vocab) {
        if constexpr (DT == kF32) u[j] = __float_as_uint(row[id + j]);
        else u[j] = row[id + j];
      }
    }
    if constexpr (DT == kF32) {
      r.a = make_uint4(u[0], u[1], u[2], u[3]);
      r.b = make_uint4(u[4], u[5], u[6], u[7]);
    } else {
      r.a = make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
    }
  }

  // the 8 values from position `pos` on, none if they are not wanted
  __device__ __forceinline__ Raw load(uint32_t pos, bool wanted) const {
    Raw r;
    r.a = make_uint4(0u, 0u, 0u, 0u);
    if (DT == kF32) r.b = r.a;
    r.bits = 0u;
    if (!wanted) return r;
    const int id = id_of(pos);
    r.bits = inside(id);
    uint32_t lo = ~0u, hi = ~0u;
    if (kept) {
      const uint32_t at = (pos - base) >> 3, lane = at & 31u;
      const uint32_t slot = slots + (at >> 5) * (uint32_t)slot_bytes;
      r.a = ps_load16(slot + lane * 16u);
      if (DT == kF32) r.b = ps_load16(slot + 512u + lane * 16u);
      if (mask) {
        const int w = (id >> 5) - ((id - 8 * (int)lane) >> 5);
        lo = ps_load4(slot + kData + 4 * w), hi = ps_load4(slot + kData + 4 * w + 4);
      }
    } else {
      if (r.bits == 0xFFu) {
        r.a = *reinterpret_cast<const uint4*>(row + id);
        if (DT == kF32) r.b = *reinterpret_cast<const uint4*>(row + id + 4);
      }
      if (mask) {
        const int w = id >> 5, words = (vocab + 31) >> 5;
        lo = w >= 0 && w < words ? mask[w] : 0u;
        hi = (id & 31) > 24 && w + 1 < words ? mask[w + 1] : 0u;
      }
    }
    if (r.bits != 0xFFu) load_edge(r, id);
    r.bits &= __funnelshift_r(lo, hi, id & 31);
    return r;
  }

  // Starts the copy of the chunk whose first id is `id0` into `slot`.
  __device__ __forceinline__ void copy_chunk(uint32_t slot, int lane, int id0) const {
    constexpr int kVec = DT == kF32 ? 4 : 8;
    const bool inner = id0 >= 0 && id0 + kPsChunk <= vocab;
    const S* from = row + (id0 + lane * kVec);
#pragma unroll
    for (int h = 0; h < 8 / kVec; ++h) {
      const int v = lane + 32 * h, id = id0 + v * kVec;
      // float32: a lane's two vectors 512 bytes apart, so that reading them has no conflicts
      const int to = DT == kF32 ? (v & 1) * 512 + (v >> 1) * 16 : v * 16;
      if (inner || (id >= 0 && id + kVec <= vocab)) ps_copy16(slot + to, from + 32 * kVec * h);
    }
    if (mask) copy_words(slot, lane, id0);
  }
  // the mask words of the chunk
  __device__ __forceinline__ void copy_words(uint32_t slot, int lane, int id0) const {
    if (lane < 10) {
      const int w = (id0 >> 5) + lane;
      const bool have = w >= 0 && w < (vocab + 31) >> 5;
      ps_copy4(slot + kData + 4 * lane, mask + (have ? w : 0), have);
    }
  }

  __device__ __forceinline__ int chunks() const {
    return (int)((end - begin + kPsChunk - 1) / kPsChunk);
  }
  __device__ __forceinline__ uint32_t first_slot() const {
    return slots + (kept ? (begin - base) / kPsChunk * (uint32_t)slot_bytes : 0u);
  }
  // Starts all copies, or those that fill the ring but for one slot.
  __device__ __forceinline__ void start_stream(int lane) const {
    const int n = chunks(), groups = kept ? n : kDepth - 1;
    uint32_t slot = first_slot();
#pragma unroll 1
    for (int i = 0; i < groups; ++i) {
      if (i < n) copy_chunk(slot, lane, id_of(begin) + i * kPsChunk);
      ps_commit();
      slot += slot_bytes;
    }
  }

  // float32 bits of value j
  __device__ __forceinline__ static uint32_t bits_of(const Raw& r, int j) {
    const uint32_t a[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
    if constexpr (DT == kF32) {
      const uint32_t b[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
      return j < 4 ? a[j & 3] : b[j & 3];
    } else if constexpr (DT == kBF16) {
      return j & 1 ? a[j >> 1] & 0xFFFF0000u : a[j >> 1] << 16;
    } else {
      return __float_as_uint(f16_bits_to_f32(a[j >> 1] >> (16 * (j & 1)) & 0xFFFFu));
    }
  }
  __device__ __forceinline__ static float value_of(const Raw& r, int j) {
    return __uint_as_float(bits_of(r, j));
  }
  // the same for a j that is not known when compiled
  __device__ __forceinline__ static float value_at(const Raw& r, int j) {
    if constexpr (DT == kF32) {
      const uint4 h = j & 4 ? r.b : r.a;
      const uint32_t lo = j & 1 ? h.y : h.x, hi = j & 1 ? h.w : h.z;
      return __uint_as_float(j & 2 ? hi : lo);
    } else {
      const uint32_t lo = j & 2 ? r.a.y : r.a.x, hi = j & 2 ? r.a.w : r.a.z;
      const uint32_t u = (j & 4 ? hi : lo) >> (16 * (j & 1)) & 0xFFFFu;
      return DT == kBF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
    }
  }

  // f(j, whether this lane has one) for the set bits j of every lane's `set`, lowest first: as
  // many turns as the fullest lane has bits. Whole warp.
  template <class F>
  __device__ __forceinline__ static void each_set(uint32_t set, F&& f) {
    while (__any_sync(~0u, set)) {
      f(set ? __ffs(set) - 1 : 0, set != 0u);
      set &= set - 1u;
    }
  }

  // The peak of 8 values: 16 bits that rise with the largest valid one (16-bit types: their
  // own order code, float32: the upper half of it), 0 without one, 0xFFFF with a NaN. `v`:
  // masks of the valid ones; float32 also raises `top`, which a NaN turns into one.
  __device__ __forceinline__ static uint32_t peak(const Raw& r, const uint32_t (&v)[4], bool full,
                                                  float& top) {
    if constexpr (DT == kF32) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[j] = full || (r.bits >> j & 1u) ? value_of(r, j) : -INFINITY;
      const float m = max_nan_f32(max_nan_f32(max_nan_f32(x[0], x[1]), max_nan_f32(x[2], x[3])),
                                  max_nan_f32(max_nan_f32(x[4], x[5]), max_nan_f32(x[6], x[7])));
      if (r.bits == 0u) return 0u;
      top = max_nan_f32(top, m);
      return ord32(m) >> 16;
    } else {
      uint32_t a = r.a.x, b = r.a.y, d = r.a.z, e = r.a.w;
      if (!full) {
        const uint32_t none = DT == kBF16 ? 0xFF80FF80u : 0xFC00FC00u;  // -inf twice
        a = (a & v[0]) | (none & ~v[0]), b = (b & v[1]) | (none & ~v[1]);
        d = (d & v[2]) | (none & ~v[2]), e = (e & v[3]) | (none & ~v[3]);
      }
      const uint32_t x = max2(max2(a, b), max2(d, e));
      const uint32_t h = max2(x, x >> 16) & 0xFFFFu;
      return full || r.bits ? h ^ (h & 0x8000u ? 0xFFFFu : 0x8000u) : 0u;
    }
  }
  __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
    return DT == kBF16 ? max_nan_bf16x2(a, b) : max_nan_f16x2(a, b);
  }
  // order code of the largest peak of a 16-bit row
  __device__ __forceinline__ static uint32_t top_code(uint32_t peak) {
    const uint32_t h = peak ^ (peak & 0x8000u ? 0x8000u : 0xFFFFu);
    return ord32(DT == kBF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h));
  }
  // the least peak of 8 values that hold an order code of at least `code`
  __device__ __forceinline__ static uint32_t least_peak(uint32_t code) {
    uint32_t peak = code >> 16;
    if constexpr (DT == kF16) {
      const uint32_t f = (code & 0x80000000u) ? code & 0x7FFFFFFFu : ~code;
      const uint32_t h = __half_as_ushort(__float2half_rd(__uint_as_float(f)));
      peak = h ^ (h & 0x8000u ? 0xFFFFu : 0x8000u);
    }
    return DT != kF32 && peak == 0x8000u ? 0x7FFFu : peak;  // -0 counts as 0
  }

  // Lists the vectors of this part that may hold order codes of at least `code`. Whole warp.
  __device__ void gather(int lane, uint32_t code) {
    if (!peaks) {
      listed = (int)((end - begin + 7u) >> 3);
      return;
    }
    const uint32_t least = least_peak(code);
    const uint16_t* mine = peaks + ((begin - base) >> 3);
    const int stop = chunks() * 32;
    int n = 0;
#pragma unroll 1
    for (int i = 0; i < stop; i += 256) {
      const int at = i + 8 * lane;
      uint32_t set = 0;
      if (at < stop) {
        const uint4 x = *reinterpret_cast<const uint4*>(mine + at);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if ((w[j] & 0xFFFFu) >= least) set |= 1u << (2 * j);
          if (w[j] >> 16 >= least) set |= 2u << (2 * j);
        }
      }
      const uint32_t c = __popc(set), incl = warp_scan(c, lane);
      int to = n + (int)(incl - c);
      while (set) {
        list[to++] = (uint16_t)(at + __ffs(set) - 1);
        set &= set - 1u;
      }
      n += (int)__shfl_sync(~0u, incl, 31);
    }
    __syncwarp();
    listed = n;
  }
  // the entries [from, to) of the list alone
  __device__ __forceinline__ RowView slice(int from, int to) const {
    RowView part = *this;
    part.listed = to - from;
    if (peaks) part.list += from;
    else part.begin += 8u * (uint32_t)from;
    return part;
  }

  // f(position, values) over the list, a vector to a lane in rising order, the next one's loads
  // in flight; lanes past its end get no valid values. Every lane of the warp makes every call.
  template <class F>
  __device__ __forceinline__ void each(int lane, F&& f) const {
    if (listed == 0) return;
    auto at = [&](int j) {
      return begin + 8u * (j < listed ? (peaks ? (uint32_t)list[j] : (uint32_t)j) : 0u);
    };
    int j = lane;
    uint32_t pos = at(j);
    Raw r = load(pos, j < listed);
    const int turns = (listed + 31) >> 5;
#pragma unroll 1
    for (int i = 0; i < turns; ++i) {
      j += 32;
      uint32_t pos2 = pos;
      Raw more = r;
      if (i + 1 < turns) {
        pos2 = at(j);
        more = load(pos2, j < listed);
      }
      f(pos, r);
      pos = pos2;
      r = more;
    }
  }
};

// 2^(y/16) for |y| < 2^20. Table-driven in the manner of Tang (ACM TOMS 15, 1989): y = 16 e + j
// + f with |f| <= 1/2, 2^(f/16) by its Taylor polynomial of degree 6 (the next term is below
// 5e-16): within 2^-50 of 2^(y/16), and 1 for y = 0. (A weight exp(x) has the rounding of y on top,
// up to |x| 2^-51 of it: 1/T, the constant, their product and y are rounded.) The 16 entries take
// the 16 pairs of banks, so lookups of a warp do not conflict.
constexpr double kPsShift = 0x1.8p52;
__device__ __forceinline__ double exp2_parts(double t, double f, const PsPowers& powers) {
  const int n = __double2loint(t);
  // (ln 2 / 16)^k / k!
  constexpr double c1 = 0.6931471805599453 / 16.0, c2 = c1 * c1 / 2.0, c3 = c2 * c1 / 3.0;
  constexpr double c4 = c3 * c1 / 4.0, c5 = c4 * c1 / 5.0, c6 = c5 * c1 / 6.0;
  double q = fma(c6, f, c5);
  q = fma(q, f, c4);
  q = fma(q, f, c3);
  q = fma(q, f, c2);
  q = fma(q, f, c1);
  const double w = powers.at[n & 15];
  const double r = fma(w * f, q, w);
  return __hiloint2double(__double2hiint(r) + (n >> 4) * (1 << 20), __double2loint(r));
}
// 2^(y/16), 0 below 2^-1000, +inf above 2^1000
__device__ __forceinline__ double exp2_table(double y, const PsPowers& powers) {
  const double t = y + kPsShift;
  const double v = exp2_parts(t, y - (t - kPsShift), powers);
  return y > -16000.0 ? (y < 16000.0 ? v : (double)INFINITY) : 0.0;
}
// 2^((v - from) scale / 16) where that exponent lies within +-2^14
__device__ __forceinline__ double exp2_from(float v, double from, double scale,
                                            const PsPowers& powers) {
  const double x = (double)v - from, t = fma(x, scale, kPsShift);
  return exp2_parts(t, fma(x, scale, kPsShift - t), powers);
}

__device__ __forceinline__ float code_value(uint32_t code) {  // inverse of ord32
  return __uint_as_float((code & 0x80000000u) ? code & 0x7FFFFFFFu : ~code);
}

// What decides which ids of the row are kept, and their weights.
struct RowCut {
  double top, scale, inv_t, min_p;  // scale = 16 log2(e) / T
  const PsPowers* powers;
  float cut;      // ids above it are kept,
  uint32_t cut2;  // (the same in a 16-bit type, twice, once the cut stands)
  uint32_t take;  // and of those equal to it the first `take`
  bool flat;      // every kept id weighs 1 (T = 0, or +inf present)

  __device__ __forceinline__ double weight(float v) const {
    return flat ? 1.0 : exp2_table(((double)v - top) * scale, *powers);
  }
  __device__ __forceinline__ void keep(float value, uint32_t first) {
    cut = value;
    take = first;
  }
  // the lowest order code that is kept
  __device__ __forceinline__ uint32_t least() const { return ord32(cut); }

  // Weights below min_p are dropped one by one where they are summed; this raises the cut to
  // a bound below which none passes, which spares looking at them.
  __device__ __forceinline__ void bound_by_min_p() {
    if (flat || !(min_p > 0.0)) return;
    // (1e-9 for what the weights round: at a high temperature many values weigh exactly 1)
    const double low = top + (log(min_p) * (1.0 + 1e-9) - 1e-9) / inv_t - fabs(top) * 1e-9;
    const float bound = nextafterf(__double2float_rd(low), -INFINITY);
    if (bound >= cut) keep(bound, 0u);
  }
};

// A range of order codes that holds the cut.
struct PsRange {
  uint32_t hi, lo;         // inclusive
  uint32_t above, inside;  // ids above it, ids in it
};

// Weights summed so far: of the codes above `down_to`, this lane's part and the cluster's.
struct PsSummed {
  double lane, all;
  uint32_t down_to;
};

template <int DT>
struct PolicyRow {
  using View = RowView<DT>;
  using Raw = typename View::Raw;
  PsShared& sh;
  View view;
  const double* table = nullptr;  // weights of the kept bins, where the cut came from them
  PsSummed summed = {0.0, 0.0, ~0u};
  uint32_t rank, k;
  uint32_t warp_ids, row_end;  // positions of a warp, and of the row
  int warp, lane, entry;
  int parity = 0;

  __device__ PolicyRow(PsShared& s) : sh(s) {}

  // What the CTAs of the cluster stored before it can be read after it. A buffer that other
  // CTAs write or read is used again only after a publish() that lies behind its last use.
  __device__ __forceinline__ void publish() {
    if (k > 1) {
      ps_cluster_arrive();
      ps_cluster_wait();
    } else {
      __syncthreads();
    }
  }

  // cluster-wide sums, and the maximum of `top`
  __device__ PsBox reduce(double mass, uint32_t count, uint32_t top, uint32_t small) {
    mass = warp_sum(mass);
    count = __reduce_add_sync(~0u, count);
    top = __reduce_max_sync(~0u, top);
    small = __reduce_add_sync(~0u, small);
    if (lane == 0) {
      sh.part_mass[warp] = mass, sh.part_count[warp] = count;
      sh.part_top[warp] = top, sh.part_small[warp] = small;
    }
    __syncthreads();
    if (warp == 0) {
      const bool have = lane < kPsWarps;
      PsBox b = {};
      b.mass = warp_sum(have ? sh.part_mass[lane] : 0.0);
      b.count = __reduce_add_sync(~0u, have ? sh.part_count[lane] : 0u);
      b.top = __reduce_max_sync(~0u, have ? sh.part_top[lane] : 0u);
      b.small = __reduce_add_sync(~0u, have ? sh.part_small[lane] : 0u);
      if ((uint32_t)lane < k) *ps_remote(&sh.box[parity][rank], lane) = b;
    }
    publish();
    PsBox r = {};
    for (uint32_t i = 0; i < k; ++i) {
      const PsBox b = sh.box[parity][i];
      r.mass += b.mass;
      r.count += b.count;
      r.top = max(r.top, b.top);
      r.small += b.small;
    }
    parity ^= 1;
    return r;
  }

  // Exclusive scans over the CTA's threads, and the totals. The end of one thread's part is the
  // start of the next one's; first_to_reach() tells which one reaches a goal. The parts are read
  // by every thread, so a __syncthreads() has to lie between two calls.
  struct Scanned {
    uint32_t count_before, count_all;
    double mass_start;  // of the warp's first thread
    double mass_before, mass_end, mass_all;
  };
  // Whether this thread is the one to write where the sum reaches `goal`; one thread at most is.
  // Whole warp; `start` is the warp's, `reached` whether the thread's end is at the goal.
  __device__ __forceinline__ bool first_to_reach(bool reached, double start, double goal) const {
    return ps_first_to_reach(__ballot_sync(~0u, reached), lane, start, goal);
  }
  __device__ Scanned scan_parts(uint32_t count, double mass, bool masses) {
    Scanned s = {};
    const uint32_t count_incl = warp_scan(count, lane);
    const double incl = masses ? warp_scan(mass, lane) : 0.0;
    if (lane == 31) sh.part_count[warp] = count_incl, sh.part_mass[warp] = incl;
    __syncthreads();
    const uint32_t c = lane < kPsWarps ? sh.part_count[lane] : 0u;
    const uint32_t c_incl = warp_scan(c, lane);
    s.count_all = __shfl_sync(~0u, c_incl, 31);
    s.count_before = __shfl_sync(~0u, c_incl - c, warp) + count_incl - count;
    if (!masses) return s;
    if (warp == 0) {  // in order, so that the parts join
      double run = 0.0;
#pragma unroll
      for (int i = 0; i < kPsWarps; ++i) {
        const double x = sh.part_mass[i];
        if (lane == i) sh.sums_before[i] = run;
        run += x;
      }
      if (lane == 0) sh.sums_before[kPsWarps] = run;
    }
    __syncthreads();
    const double prev = __shfl_up_sync(~0u, incl, 1), mine = sh.sums_before[warp];
    s.mass_all = sh.sums_before[kPsWarps];
    s.mass_start = mine;
    s.mass_before = lane ? mine + prev : mine;
    s.mass_end = ps_part_end(mine, incl, sh.sums_before[warp + 1]);
    return s;
  }

  __device__ __forceinline__ void clear_hist() {
    for (int i = threadIdx.x; i < kPsBins / 4; i += kPsThreads)
      reinterpret_cast<uint4*>(ps_hist())[i] = make_uint4(0u, 0u, 0u, 0u);
  }

  // After a reduce(): the cluster's counts of this thread's kPsOwn bins. Every CTA adds up its
  // part of the bins and hands the sums to all. by_magnitude: bins as count_bins() lays them.
  __device__ void merge_bins(uint32_t (&n)[kPsOwn], bool by_magnitude) {
    const uint32_t* from = ps_hist();
    if (k > 1) {
      const int part = kPsBins / (int)k;
      for (int i = threadIdx.x; i < part; i += kPsThreads) {
        const int bin = (int)rank * part + i;
        uint32_t x[kPsMaxCluster];
#pragma unroll
        for (uint32_t r = 0; r < kPsMaxCluster; ++r)
          x[r] = r < k ? *ps_remote(ps_hist() + bin, r) : 0u;
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t r = 0; r < kPsMaxCluster; ++r) sum += x[r];
#pragma unroll
        for (uint32_t r = 0; r < kPsMaxCluster; ++r)
          if (r < k) *ps_remote(ps_merged() + bin, r) = sum;
      }
      publish();
      from = ps_merged();
    }
    const int mine = threadIdx.x * kPsOwn;
    const bool turned = by_magnitude && mine < kPsHalf;
    const uint32_t* at = from + (turned ? kPsHalf - kPsOwn - mine : mine);
    const uint4 x = reinterpret_cast<const uint4*>(at)[0], y = reinterpret_cast<const uint4*>(at)[1];
    const uint32_t t[kPsOwn] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int j = 0; j < kPsOwn; ++j) n[j] = turned ? t[kPsOwn - 1 - j] : t[j];
  }

  // ---- bfloat16: the cut from a histogram with a bin for every value --------------------
  __device__ __forceinline__ static uint32_t bin_bits(int bin) {  // of |v|
    return bin < kPsHalf ? kPsLow + (kPsHalf - 1 - bin) : kPsLow + (bin - kPsHalf);
  }
  __device__ __forceinline__ static float bin_value(int bin) {
    return __uint_as_float((bin_bits(bin) | (bin < kPsHalf ? 0u : 0x8000u)) << 16);
  }

  // Counts the bins of two values, the halves of `u`, where `valid` has ones; returns bit 15
  // and bit 31 set for those next to zero. In memory the bins of either sign lie by rising
  // magnitude, negative ones behind. With the sign bit set no half borrows from the other; the
  // bin is right where bits 11 to 14 come out as zeros.
  __device__ __forceinline__ static uint32_t count_values(uint32_t hist, uint32_t u,
                                                          uint32_t valid) {
    const uint32_t t = (u | 0x80008000u) - kPsLow * 0x10001u;
    const uint32_t bad = (t & 0x78007800u) | ~valid;
    const uint32_t at = ((t & 0x07FF07FFu) | ((u >> 4) & 0x08000800u)) << 2;
    // predicated, where the compiler would branch
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b32 x;\n\t"
        "and.b32 x, %2, 0xFFFF;\n\tsetp.eq.u32 p, x, 0;\n\tsetp.lt.u32 q, %2, 0x10000;\n\t"
        "@p red.shared.add.u32 [%0], 1;\n\t@q red.shared.add.u32 [%1], 1;\n\t}" ::"r"(
            hist + (at & 0xFFFFu)),
        "r"(hist + (at >> 16)), "r"(bad)
        : "memory");
    return ~t & 0x80008000u & valid;
  }

  // Sets the cut and makes the table of weights; false where the bins do not decide it. `sum`
  // has the count of the valid ids, and the count and mass of those next to zero.
  __device__ bool cut_by_values(RowCut& c, const RowPolicy& pol, const PsBox& sum) {
    uint32_t n[kPsOwn];
    merge_bins(n, true);
    if (c.flat || !(c.top < kPsLarge)) return false;
    const int mine = threadIdx.x * kPsOwn;  // this thread's bins, in falling order of value
    const bool by_mass = pol.top_p < 1.0;
    // The mass of a bin is count times weight. The values of 8 bins are equally spaced, their
    // weights a geometric series, which starts at the row's maximum in the bins that hold it
    // (those above are empty). Up to eight factors, each within 2^-50: a weight within 2^-47.
    double weight_of[kPsOwn], mass = 0.0;
    uint32_t count = 0;
#pragma unroll
    for (int j = 0; j < kPsOwn; ++j) count += n[j];
    if (by_mass) {
      const float step = __uint_as_float(bin_bits(mine) << 16 & 0x7F800000u) * 0x1p-7f;
      const double ratio = exp2_table(-(double)step * c.scale, *c.powers);
      float from = bin_value(mine);
      int at = 0;
      if ((double)from > c.top) {
#pragma unroll
        for (int j = kPsOwn - 1; j >= 0; --j)
          if (n[j]) at = j;
        from = count ? bin_value(mine + at) : -INFINITY;
      }
      double w = c.weight(from);
#pragma unroll
      for (int j = 0; j < kPsOwn; ++j) {
        weight_of[j] = j >= at ? w : 0.0;
        if (j >= at) w *= ratio;
        mass += (double)n[j] * weight_of[j];
      }
    }
    if (threadIdx.x < 2) sh.cross[threadIdx.x].bin = -1;
    const Scanned scan = scan_parts(count, mass, by_mass);
    uint32_t count_before = scan.count_before;
    double mass_start = scan.mass_start, mass_before = scan.mass_before;
    double mass_end = scan.mass_end;
    if (mine >= kPsHalf) {  // the values next to zero lie between the halves
      count_before += sum.small;
      mass_start += sum.mass, mass_before += sum.mass, mass_end += sum.mass;
    }
    const uint32_t in_bins = scan.count_all + sum.small;
    // ids at and below -2^7 lie behind the bins; they may weigh nothing next to the rest
    const bool behind_weighs = sum.count > in_bins && c.weight(-kPsLarge) > 0x1p-80;

    int cut_bin = kPsBins;
    uint32_t take = 0;
    double total = scan.mass_all + sum.mass;
    const bool by_k = pol.top_k && pol.top_k < sum.count;
    if (by_k) {
      if (pol.top_k > in_bins) return false;
      if (count_before < pol.top_k && pol.top_k <= count_before + count) {
        PsCross x = {mass_before, count_before, 0u, -1};
#pragma unroll
        for (int j = 0; j < kPsOwn; ++j)
          if (x.bin < 0) {
            if (pol.top_k <= x.count + n[j]) {
              x.bin = mine + j;
              x.n = pol.top_k - x.count;
              if (by_mass) x.mass += (double)x.n * weight_of[j];
            } else {
              x.count += n[j];
              if (by_mass) x.mass += (double)n[j] * weight_of[j];
            }
          }
        sh.cross[0] = x;
      }
      __syncthreads();
      const PsCross x = sh.cross[0];
      if (x.bin < 0) return false;  // among the values next to zero
      cut_bin = x.bin;
      take = x.n;
      total = x.mass;
    }
    if (by_mass) {
      if (!by_k && behind_weighs) return false;
      const double goal = pol.top_p * total;
      // the bins of this thread reach it, or hold the last of the k
      const bool ends = goal <= mass_end || (mine <= cut_bin && cut_bin < mine + kPsOwn);
      if (first_to_reach(ends, mass_start, goal) && count && mine <= cut_bin) {
        PsCross x = {mass_before, 0u, 0u, -1};  // the bin that reaches the goal, else the last
        double run = mass_before, weight = 0.0;
#pragma unroll
        for (int j = 0; j < kPsOwn; ++j)
          if (n[j] && mine + j <= cut_bin && run < goal) {
            x = {run, 0u, by_k && mine + j == cut_bin ? take : n[j], mine + j};
            weight = weight_of[j];
            run += (double)x.n * weight;
          }
        x.n = ties_to_reach(goal - x.mass, weight, x.n, x.mass, goal);
        sh.cross[1] = x;
      }
      __syncthreads();
      const PsCross x = sh.cross[1];
      if (x.bin < 0) return false;  // among the values next to zero
      cut_bin = x.bin;
      take = x.n;
    }
    if (cut_bin < kPsBins) c.keep(bin_value(cut_bin), take);
    // the weights of the kept bins, for the passes that follow
    __syncthreads();  // the counts have been read
    double* weights = ps_table();
#pragma unroll
    for (int j = 0; j < kPsOwn; ++j)
      if (n[j] && mine + j <= cut_bin)
        weights[mine + j] = by_mass ? weight_of[j] : c.weight(bin_value(mine + j));
    table = weights;
    __syncthreads();
    return true;
  }

  // ---- other types: the few bins that hold the cut ---------------------------------------
  // Bins of equal width, 1/64 in the exponent of the weights, from 40 above the largest of a
  // sample of the row's values to 24 below it, in falling order of value.
  struct Linear {
    float scale, shift;  // bin = round(shift - v scale) - 2^23
    bool ok;
  };
  static constexpr float kBinsPerE = 64.0f, kBinsAbove = 2560.0f, kTwo23 = 8388608.0f;

  __device__ __forceinline__ static uint32_t bin_of(const Linear& lin, float v) {
    return __float_as_uint(fmaf(v, -lin.scale, lin.shift)) - 0x4B000000u;
  }
  __device__ __forceinline__ static void count_linear(uint32_t hist, float scale, float shift,
                                                      float v, bool valid) {
    const uint32_t at = __float_as_uint(fmaf(v, -scale, shift)) - 0x4B000000u;
    const uint32_t bin = valid ? at : ~0u;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.lt.u32 p, %1, %2;\n\t@p red.shared.add.u32 [%0], 1;\n\t}" ::"r"(
            hist + (bin << 2)),
        "r"(bin), "n"(kPsBins)
        : "memory");
  }
  // Order code of the largest value whose bin is `bin` or a lower one (in value); 0 if that is
  // not found within a few steps from where it should be.
  __device__ __forceinline__ static uint32_t top_of_bin(const Linear& lin, int bin) {
    auto reaches = [&](float x) {  // not NaN; bins past either end compare by the rounded value
      return fmaf(x, -lin.scale, lin.shift) >= kTwo23 + (float)bin;
    };
    float x = (float)(((double)lin.shift - (double)kTwo23 - (double)bin + 0.5) / (double)lin.scale);
    int steps = 0;
    while (!reaches(x) && ++steps < 16) x = nextafterf(x, -INFINITY);
    while (reaches(nextafterf(x, INFINITY)) && ++steps < 16) x = nextafterf(x, INFINITY);
    return steps < 16 && x > -FLT_MAX && x < FLT_MAX ? ord32(x) : 0u;
  }

  // The bins for this row, and the value that its masses are relative to: the largest of 128
  // samples, of the valid ones if there are any.
  __device__ Linear sample_bins(float scale, double& from) {
    if (warp < 4) {
      const int id = (int)((int64_t)threadIdx.x * view.vocab >> 7);
      const float v = Elem<DT>::to_f32(view.row, id);
      const bool finite = fabsf(v) <= FLT_MAX;
      const bool valid = !view.mask || (view.mask[id >> 5] >> (id & 31) & 1u);
      const uint32_t any = __reduce_max_sync(~0u, finite ? ord32(v) : 0u);
      const uint32_t best = __reduce_max_sync(~0u, finite && valid ? ord32(v) : 0u);
      if (lane == 0) sh.sample[0][warp] = any, sh.sample[1][warp] = best;
    }
    __syncthreads();
    uint32_t any = 0, best = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) any = max(any, sh.sample[0][i]), best = max(best, sh.sample[1][i]);
    const uint32_t code = best ? best : any;
    const float middle = code ? code_value(code) : 0.0f;
    from = middle;
    const bool ok = scale < 1e30f && fabsf(middle * scale) < 1e30f;
    return {scale, fmaf(middle, scale, kTwo23 + kBinsAbove), ok};
  }

  // The range of codes that holds the cut, with top-k and top-p both also the k-th value; false
  // where the bins do not tell. `total` is the mass of all ids, if top-p needs it. `safe` holds
  // it surely, `range` in all likelihood.
  __device__ bool range_by_bins(const RowCut& c, const RowPolicy& pol, const PsBox& sum,
                                const Linear& lin, double total, PsRange& range, PsRange& safe) {
    uint32_t n[kPsOwn];
    merge_bins(n, false);
    if (c.flat || !lin.ok || bin_of(lin, (float)c.top) >= (uint32_t)kPsBins) return false;
    const int mine = threadIdx.x * kPsOwn;
    const bool by_mass = pol.top_p < 1.0, by_k = pol.top_k && pol.top_k < sum.count;
    // A bin's mass is its count times the weight of its middle, within 1/128 of it (the row's
    // maximum counts as it is): the cut lies between the bins in which that mass reaches the
    // goal less 1/120 and plus 1/120 of it (with top-k the goal itself is as far off, so twice
    // that). Many ids there mean that few of them carry the mass alone; then the errors of the
    // bins cancel: to some 5e-4 of the goal with a list of 200 by that bound, to 2e-4 where 1/320
    // still holds over 1,024. Such rows take the widest of 1/320, 1/700 and 1/1536 that makes a
    // list, and the list is checked.
    double mass = 0.0, weight_of[kPsOwn];
    uint32_t count = 0;
#pragma unroll
    for (int j = 0; j < kPsOwn; ++j) count += n[j];
    if (by_mass) {
      const double middle =
          ((double)lin.shift - (double)kTwo23 - (double)mine) / (double)lin.scale;
      const double ratio = exp2_table(-c.scale / (double)lin.scale, *c.powers);
      double w = exp2_table((middle - c.top) * c.scale, *c.powers);
#pragma unroll
      for (int j = 0; j < kPsOwn; ++j) {
        weight_of[j] = w;
        mass += (double)n[j] * w;
        w *= ratio;
      }
      const int top_bin = (int)bin_of(lin, (float)c.top) - mine;
      if (top_bin >= 0 && top_bin < kPsOwn) {
#pragma unroll
        for (int j = 0; j < kPsOwn; ++j)
          if (j == top_bin) {
            const double extra = (1.0 - weight_of[j]) / (double)n[j];
            weight_of[j] += extra;
            mass += (double)n[j] * extra;
          }
      }
    }
    if (threadIdx.x < 9) sh.cross[threadIdx.x].bin = -1;
    const Scanned scan = scan_parts(count, mass, by_mass);
    uint32_t through = 0;  // ids up to and with the last bin of the range
    int last = 0;
    if (by_k) {
      if (pol.top_k > scan.count_all) return false;
      if (scan.count_before < pol.top_k && pol.top_k <= scan.count_before + count) {
        PsCross x = {scan.mass_before, scan.count_before, 0u, -1};
#pragma unroll
        for (int j = 0; j < kPsOwn; ++j)
          if (x.bin < 0) {
            if (pol.top_k <= x.count + n[j]) {
              x.bin = mine + j;
              x.n = n[j];
              if (by_mass) x.mass += (double)(pol.top_k - x.count) * weight_of[j];
            } else {
              x.count += n[j];
              if (by_mass) x.mass += (double)n[j] * weight_of[j];
            }
          }
        sh.cross[0] = x;
      }
      __syncthreads();
      const PsCross x = sh.cross[0];
      through = x.count + x.n;
      last = x.bin;
      total = x.mass;
      if (!by_mass) range = {top_of_bin(lin, x.bin), 0u, x.count, x.n};
    }
    if (by_mass) {
      const double goal = pol.top_p * total;
      // cross[at]: the bin in which the mass reaches `mark`, ids before it and in it
      auto mark_bin = [&](int at, double mark) {
        if (first_to_reach(mark <= scan.mass_end, scan.mass_start, mark) && count) {
          PsCross x = {0.0, scan.count_before, 0u, -1};
          double run = scan.mass_before;
#pragma unroll
          for (int j = 0; j < kPsOwn; ++j)
            if (n[j] && run < mark) {
              x.count += x.n;
              x.n = n[j];
              x.bin = mine + j;
              run += (double)n[j] * weight_of[j];
            }
          sh.cross[at] = x;
        }
      };
      mark_bin(1, goal * (by_k ? 1.0 - 2.0 / 120.0 : 1.0 - 1.0 / 120.0));
      if (!by_k) {
        mark_bin(2, goal * (1.0 + 1.0 / 120.0));
        mark_bin(3, goal * (1.0 - 1.0 / 320.0));
        mark_bin(4, goal * (1.0 + 1.0 / 320.0));
        mark_bin(5, goal * (1.0 - 1.0 / 700.0));
        mark_bin(6, goal * (1.0 + 1.0 / 700.0));
        mark_bin(7, goal * (1.0 - 1.0 / 1536.0));
        mark_bin(8, goal * (1.0 + 1.0 / 1536.0));
      }
      __syncthreads();
      PsCross x = sh.cross[1];
      if (x.bin < 0) return false;
      if (!by_k) {
        PsCross y = sh.cross[2];
        if (y.bin < 0) y = {0.0, scan.count_all, 0u, kPsBins - 1};
        safe.above = x.count;
        safe.inside = y.count + y.n - x.count;
        safe.hi = top_of_bin(lin, x.bin);
        safe.lo = top_of_bin(lin, y.bin + 1) + 1u;
#pragma unroll
        for (int at = 3; at <= 7; at += 2)
          if (y.count + y.n - x.count > (at == 3 ? 192u : kPsList) && sh.cross[at].bin >= 0 &&
              sh.cross[at + 1].bin >= 0)
            x = sh.cross[at], y = sh.cross[at + 1];
        last = y.bin;
        through = y.count + y.n;
      }
      range = {top_of_bin(lin, x.bin), 0u, x.count, through - x.count};
    }
    const uint32_t below = top_of_bin(lin, last + 1);
    range.lo = below + 1u;
    if (by_k || !by_mass) safe = range;
    return range.hi && below && range.lo <= range.hi && safe.hi && safe.lo > 1u;
  }

  // ---- top-k by the peaks ----------------------------------------------------------------
  // The k-th largest peak is no larger than the k-th largest value, and few other values reach
  // it: a histogram of the peaks (an eighth of the ids, from shared memory) gives a range for
  // the list, which spares the first pass its histogram of all ids. False where that does not
  // fit a list.
  __device__ bool range_by_peaks(uint32_t rank_k, uint32_t top, uint32_t valid, PsRange& range) {
    range = {top, kOrd32NegInf, 0u, valid};
    if (valid <= kPsList) return true;
    if (!view.peaks) return false;
    // codes of one eighth of a value's range (float16) or one bfloat16 value to a bin
    constexpr int kShift = DT == kF16 ? 3 : 0;
    const uint32_t best = View::least_peak(top) >> kShift;
    const int stop = view.chunks() * 32;
    const uint16_t* mine = view.peaks + ((view.begin - view.base) >> 3);
    uint32_t* hist = ps_hist();
    for (int i = lane; i < stop; i += 32) {
      const uint32_t peak = mine[i];
      const uint32_t bin = best - min(best, peak >> kShift);
      if (peak && bin < (uint32_t)kPsBins) atomicAdd(hist + bin, 1u);
    }
    publish();
    uint32_t n[kPsOwn], count = 0;
    merge_bins(n, false);
#pragma unroll
    for (int j = 0; j < kPsOwn; ++j) count += n[j];
    if (threadIdx.x == 0) sh.cross[0].bin = -1;
    const Scanned scan = scan_parts(count, 0.0, false);
    if (scan.count_before < rank_k && rank_k <= scan.count_before + count) {
      uint32_t run = scan.count_before;
#pragma unroll
      for (int j = 0; j < kPsOwn; ++j) {
        if (run < rank_k && rank_k <= run + n[j]) {
          sh.cross[0].n = run + n[j];
          sh.cross[0].bin = (int)threadIdx.x * kPsOwn + j;
        }
        run += n[j];
      }
    }
    __syncthreads();
    const int bin = sh.cross[0].bin;
    if (bin < 0 || sh.cross[0].n > kPsList) return false;
    const uint32_t peak = (best - (uint32_t)bin) << kShift;
    if (DT == kF16) {
      const uint32_t h = peak ^ (peak & 0x8000u ? 0x8000u : 0xFFFFu);
      const float low = f16_bits_to_f32(h);
      if (low >= -65504.0f) range.lo = ord32(low);  // (else below the finite ones)
    } else {
      range.lo = peak << 16;
    }
    return true;
  }

  // Least number of ids of weight `w`, 1 to `most`, whose mass on top of `above` reaches `goal`.
  __device__ __forceinline__ static uint32_t ties_to_reach(double need, double w, uint32_t most,
                                                           double above, double goal) {
    double t = ceil(need / w);
    t = t >= 1.0 ? (t > (double)most ? (double)most : t) : 1.0;
    while (t > 1.0 && above + (t - 1.0) * w >= goal) t -= 1.0;
    while (t < (double)most && above + t * w < goal) t += 1.0;
    return (uint32_t)t;
  }

  // weight of a kept value; `bins`: the table, if there is one
  __device__ __forceinline__ static double weigh(float v, double top, double scale, bool flat,
                                                 const PsPowers& powers, const double* bins) {
    if (DT == kBF16 && bins) {
      const uint32_t bits = __float_as_uint(v);
      const uint32_t i = ((bits >> 16) & 0x7FFFu) - kPsLow;
      const uint32_t positive = (uint32_t)((int32_t)~bits >> 31);
      if (i < (uint32_t)kPsHalf) return bins[kPsHalf + (int)(i ^ positive)];
    }
    return flat ? 1.0 : exp2_table(((double)v - top) * scale, powers);
  }
  __device__ __forceinline__ double weight(const RowCut& c, float v) const {
    return weigh(v, c.top, c.scale, c.flat, *c.powers, table);
  }

  // f(j, weight) for the values j of the lane's `set` that weigh min_p at least. Whole warp.
  // Few to a lane: one after the other; else all eight side by side, which hides the latency
  // of the float64 chains.
  template <class F>
  __device__ __forceinline__ void each_weight(const RowCut& c, const Raw& r, uint32_t set,
                                              F&& f) const {
    if (__any_sync(~0u, __popc(set) > 2)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double w = weight(c, View::value_of(r, j));
        if ((set >> j & 1u) && w >= c.min_p) f(j, w);
      }
    } else {
      View::each_set(set, [&](int j, bool have) {
        const double w = weight(c, View::value_at(r, j));
        if (have && w >= c.min_p) f(j, w);
      });
    }
  }
  // the sum of those weights that are `least` at least; 0 without a call where no lane has one
  __device__ __forceinline__ double sum_of(const RowCut& c, const Raw& r, uint32_t set,
                                           double least) const {
    if (!__any_sync(~0u, set)) return 0.0;
    return sum_set(r.a.x, r.a.y, r.a.z, r.a.w, DT == kF32 ? r.b.x : 0u, DT == kF32 ? r.b.y : 0u,
                   DT == kF32 ? r.b.z : 0u, DT == kF32 ? r.b.w : 0u, set, c.top, c.scale, least,
                   c.flat, c.powers, table);
  }
  // (Scalars, for a struct that is passed by value lives in memory, and so do its copies.)
  __device__ __noinline__ static double sum_set(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3,
                                                uint32_t set, double top, double scale,
                                                double least, bool flat, const PsPowers* powers,
                                                const double* bins) {
    Raw r;
    r.a = make_uint4(a0, a1, a2, a3);
    r.b = make_uint4(b0, b1, b2, b3);
    r.bits = set;
    if (flat) return 1.0 >= least ? (double)__popc(set) : 0.0;
    double a = 0.0, b = 0.0;
    if (!__any_sync(~0u, __popc(set) > 2)) {
      View::each_set(set, [&](int j, bool have) {
        const double w = weigh(View::value_at(r, j), top, scale, false, *powers, bins);
        a += have && w >= least ? w : 0.0;
      });
      return a;
    }
    if (DT == kBF16 && bins) {
      uint32_t missed = 0;  // values without a bin
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t bits = View::bits_of(r, j);
        const uint32_t i = ((bits >> 16) & 0x7FFFu) - kPsLow;
        const uint32_t positive = (uint32_t)((int32_t)~bits >> 31);
        const bool has = i < (uint32_t)kPsHalf;
        if (!has) missed |= 1u << j;
        const double w = bins[has ? kPsHalf + (int)(i ^ positive) : 0];
        a += (set >> j & 1u) && has && w >= least ? w : 0.0;
      }
      missed &= set;
      if (__any_sync(~0u, missed))
        View::each_set(missed, [&](int j, bool have) {
          const double w = weigh(View::value_at(r, j), top, scale, false, *powers, nullptr);
          b += have && w >= least ? w : 0.0;
        });
      return a + b;
    }
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const double w = exp2_table(((double)View::value_of(r, j) - top) * scale, *powers);
      const double x = exp2_table(((double)View::value_of(r, j + 1) - top) * scale, *powers);
      a += (set >> j & 1u) && w >= least ? w : 0.0;
      b += (set >> j & 2u) && x >= least ? x : 0.0;
    }
    return a + b;
  }

  // ---- the cut from ranges of order codes -----------------------------------------------
  // mass and count of the valid ids whose order code is at least `code`
  __device__ PsBox at_least(const RowCut& c, uint32_t code) {
    double mass = 0.0;
    uint32_t count = 0;
    view.gather(lane, code);
    view.each(lane, [&](uint32_t, const Raw& r) {
      uint32_t set = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((r.bits >> j & 1u) && ord32(View::value_of(r, j)) >= code) set |= 1u << j;
      count += __popc(set);
      mass += sum_of(c, r, set, 0.0);
    });
    return reduce(mass, count, 0u, 0u);
  }

  // After a pass that summed the codes above `hi` that were not summed yet (or none): the mass
  // of all codes above `hi`.
  __device__ double sum_up(double mass, uint32_t hi, bool did) {
    const double more = reduce(mass, 0u, 0u, 0u).mass;
    if (!did) return 0.0;
    summed.lane += mass;
    summed.all += more;
    summed.down_to = hi;
    return summed.all;
  }

  // One turn of the histogram over the range: it shrinks to the bin that holds rank `rank_k`,
  // or (rank_k 0) to the bins in which the mass can reach `goal`.
  __device__ void refine(const RowCut& c, PsRange& range, uint32_t rank_k, double goal) {
    const uint32_t width = range.hi - range.lo;
    const int shift = max(0, 20 - __clz(width));  // width >> shift < 2^12
    clear_hist();
    __syncthreads();
    uint32_t* hist = ps_hist();
    double mass = 0.0;
    view.gather(lane, range.lo);
    view.each(lane, [&](uint32_t, const Raw& r) {
      uint32_t set = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t code = ord32(View::value_of(r, j));
        const bool valid = r.bits >> j & 1u;
        if (valid && code > range.hi && code <= summed.down_to) set |= 1u << j;
        if (valid && range.hi - code <= width) atomicAdd(hist + ((range.hi - code) >> shift), 1u);
      }
      if (!rank_k) mass += sum_of(c, r, set, 0.0);
    });
    const double above = sum_up(mass, range.hi, !rank_k);
    uint32_t n[kPsOwn], count = 0;
    merge_bins(n, false);
    const uint32_t mine = threadIdx.x * kPsOwn;
    double mass_high = 0.0, mass_low = 0.0, high[kPsOwn], low[kPsOwn];
#pragma unroll
    for (int j = 0; j < kPsOwn; ++j) {
      count += n[j];
      high[j] = low[j] = 0.0;
      if (!rank_k && n[j]) {
        const uint32_t first = range.hi - ((mine + j) << shift);
        const uint32_t span = min((1u << shift) - 1u, first - range.lo);
        high[j] = c.weight(code_value(first));
        low[j] = span ? c.weight(code_value(first - span)) : high[j];
        mass_high += (double)n[j] * high[j];
        mass_low += (double)n[j] * low[j];
      }
    }
    if (threadIdx.x < 2) sh.cross[threadIdx.x].bin = -1;
    const Scanned scan = scan_parts(count, mass_high, !rank_k);
    const uint32_t before = range.above + scan.count_before;
    PsCross first = {}, last = {};
    if (rank_k) {
      if (before < rank_k && rank_k <= before + count) {
        PsCross x = {0.0, before, 0u, -1};
#pragma unroll
        for (int j = 0; j < kPsOwn; ++j)
          if (x.bin < 0) {
            if (rank_k <= x.count + n[j]) x.bin = (int)mine + j, x.n = n[j];
            else x.count += n[j];
          }
        sh.cross[0] = x;
      }
      __syncthreads();
      first = last = sh.cross[0];
      last.count += last.n;
    } else {
      __syncthreads();
      const Scanned scan2 = scan_parts(0u, mass_low, true);
      const double hb = above + scan.mass_before, high_end = above + scan.mass_end;
      const double lb = above + scan2.mass_before, low_end = above + scan2.mass_end;
      const double high_start = above + scan.mass_start, low_start = above + scan2.mass_start;
      const double least = goal * (1.0 - 1e-12), most = goal * (1.0 + 1e-12);
      if (first_to_reach(least <= high_end, high_start, least) && count) {
        PsCross x = {0.0, before, 0u, -1};
        double run = hb;
        uint32_t run_count = before;
#pragma unroll
        for (int j = 0; j < kPsOwn; ++j)
          if (n[j] && run < least) {
            x = {0.0, run_count, n[j], (int)mine + j};
            run += (double)n[j] * high[j];
            run_count += n[j];
          }
        sh.cross[0] = x;
      }
      if (first_to_reach(most <= low_end, low_start, most) && count) {
        PsCross x = {0.0, before, 0u, -1};
        double run = lb;
#pragma unroll
        for (int j = 0; j < kPsOwn; ++j)
          if (n[j] && run < most) {
            run += (double)n[j] * low[j];
            x.count += n[j];
            x.bin = (int)mine + j;
          }
        sh.cross[1] = x;
      }
      __syncthreads();
      first = sh.cross[0];
      last = sh.cross[1];
      if (first.bin < 0) first = {0.0, range.above, 0u, 0};
      if (last.bin < 0) last = {0.0, range.above + range.inside, 0u, (int)(width >> shift)};
    }
    const uint32_t hi = range.hi - ((uint32_t)first.bin << shift);
    const uint32_t end = range.hi - ((uint32_t)last.bin << shift);
    const uint32_t span = min((1u << shift) - 1u, end - range.lo);
    range = {hi, end - span, first.count, last.count - first.count};
  }

  // Halves the range by the exact mass above its middle.
  __device__ void bisect(const RowCut& c, PsRange& range, double goal) {
    const uint32_t mid = range.lo + (range.hi - range.lo + 1u) / 2u;
    const PsBox b = at_least(c, mid);
    if (b.mass >= goal) {
      range = {range.hi, mid, range.above, b.count - range.above};
    } else {
      range = {mid - 1u, range.lo, b.count, range.above + range.inside - b.count};
    }
  }

  // Lists the ids of the range, sorted by value falling, and sets the cut:
  // at rank `rank_k` (0: no bound), and with by_mass where the mass reaches top_p of `total`
  // (with rank_k: of the mass of those ranks).
  // False where they are more than kPsList, or the goal lies above the range or below it.
  __device__ bool cut_from_list(RowCut& c, const PsRange& range, uint32_t rank_k, bool by_mass,
                                double top_p, double total) {
    if (threadIdx.x == 0) sh.list_fill = 0u;
    __syncthreads();
    unsigned long long* list = ps_list();
    double mass = 0.0;
    view.gather(lane, range.lo);
    view.each(lane, [&](uint32_t pos, const Raw& r) {
      const uint32_t id = (uint32_t)view.id_of(pos);
      uint32_t set = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t code = ord32(View::value_of(r, j));
        const bool valid = r.bits >> j & 1u;
        if (valid && code > range.hi && code <= summed.down_to) set |= 1u << j;
        if (valid && code >= range.lo && code <= range.hi) {
          const uint32_t at = atomicAdd(&sh.list_fill, 1u);
          // ascending keys: value falling, id rising
          if (at < kPsList) list[at] = (unsigned long long)~code << 32 | (id + j);
        }
      }
      if (by_mass) mass += sum_of(c, r, set, 0.0);
    });
    __syncthreads();
    if ((uint32_t)threadIdx.x < k)
      *ps_remote(&sh.listed[rank], threadIdx.x) = sh.list_fill;
    const double above = sum_up(mass, range.hi, by_mass);
    unsigned long long* sorted = ps_sorted();
    uint32_t n = 0;
    for (uint32_t r = 0; r < k; ++r) {  // a warp or two to each CTA's list
      const uint32_t all = sh.listed[r], m = min(all, kPsList), warps = kPsWarps / k;
      if ((uint32_t)warp / warps == r) {
        const unsigned long long* from = k > 1 ? ps_remote(list, r) : list;
        for (uint32_t i = threadIdx.x % (32u * warps); i < m; i += 32u * warps)
          if (n + i < kPsList) sorted[n + i] = from[i];
      }
      n = min(n + all, kPsList + 1u);
    }
    const bool fits = n <= kPsList;
    n = min(n, kPsList);
    uint32_t size = 2;
    while (size < n) size <<= 1;
    for (uint32_t i = n + threadIdx.x; i < size; i += kPsThreads) sorted[i] = ~0ull;
    __syncthreads();
    if (n <= 256u) {
      // each key's place is the count of the smaller ones, by up to 32 threads to a key: one
      // pass over the keys, where the sort below has up to 36 steps that wait for one another
      const uint32_t group = min(32u, kPsThreads / max(size, 16u)), part = threadIdx.x % group;
      const uint32_t i = threadIdx.x / group;
      const unsigned long long key = i < n ? sorted[i] : 0ull;
      uint32_t place = 0;
      for (uint32_t j = part; j < n; j += group) place += sorted[j] < key;
      for (uint32_t d = group / 2; d; d /= 2) place += __shfl_xor_sync(~0u, place, d);
      sorted += kPsList;
      if (i < n && part == 0) sorted[place] = key;
      size = 0;  // nothing left to sort
    }
    // bitonic sort; a warp's 64 keys need no more than the warp
    for (uint32_t run = 2; run <= size; run <<= 1)
      for (uint32_t d = run >> 1; d; d >>= 1) {
        const uint32_t t = threadIdx.x;
        if (t < size / 2) {
          const uint32_t i = 2u * t - (t & (d - 1u));
          const unsigned long long a = sorted[i], b = sorted[i + d];
          if ((a > b) == ((i & run) == 0u)) sorted[i] = b, sorted[i + d] = a;
        }
        if (d > 32u || (d == 1u && run >= 64u)) __syncthreads();
        else __syncwarp();
      }
    __syncthreads();
    // two keys to a thread
    const uint32_t at = 2u * threadIdx.x;
    const uint32_t have = rank_k ? min(n, rank_k - range.above) : n;
    uint32_t pos = have - 1u;
    bool holds = fits && have > 0u;
    if (by_mass) {
      const double w0 = at < have ? c.weight(code_value(~(uint32_t)(sorted[at] >> 32))) : 0.0;
      const double w1 =
          at + 1u < have ? c.weight(code_value(~(uint32_t)(sorted[at + 1u] >> 32))) : 0.0;
      const Scanned scan = scan_parts(0u, w0 + w1, true);
      const double end = scan.mass_end, before = scan.mass_before;
      if (rank_k) total = above + scan.mass_all;
      const double goal = top_p * total;
      holds = holds && above < goal && (rank_k || above + scan.mass_all >= goal);
      uint32_t mine = have - 1u;
      if (at < have && above + before + w0 >= goal) mine = at;
      else if (at + 1u < have && above + end >= goal) mine = at + 1u;
      mine = __reduce_min_sync(~0u, mine);
      if (lane == 0) sh.part_top[warp] = mine;
      __syncthreads();
      for (int i = 0; i < kPsWarps; ++i) pos = min(pos, sh.part_top[i]);
    }
    const uint32_t code = ~(uint32_t)(sorted[holds ? pos : 0u] >> 32);
    uint32_t same = 0;
    if (holds && at <= pos) same += ~(uint32_t)(sorted[at] >> 32) == code;
    if (holds && at + 1u <= pos) same += ~(uint32_t)(sorted[at + 1u] >> 32) == code;
    same = __reduce_add_sync(~0u, same);
    if (lane == 0) sh.part_small[warp] = same;
    __syncthreads();
    uint32_t take = 0;
    for (int i = 0; i < kPsWarps; ++i) take += sh.part_small[i];
    if (holds) c.keep(code_value(code), take);
    publish();
    return holds;
  }

  // The cut, starting from nothing but the row's maximum `top`, or from `found`, a range out of
  // the bins. `total` is the mass of all ids, or negative where it is not known.
  __device__ __forceinline__ void find_cut(RowCut& c, const RowPolicy& pol, uint32_t top,
                                           uint32_t valid, double total, const PsRange* found) {
    if (!(pol.temperature > 0.0)) {
      c.keep(code_value(top), 1u);
      return;
    }
    c.keep(c.flat ? FLT_MAX : -INFINITY, 0u);
    const bool by_mass = pol.top_p < 1.0;
    PsRange range = {top, c.flat ? top : kOrd32NegInf, 0u, valid};
    if (c.flat) range.inside = valid = at_least(c, top).count;  // the +inf ids
    const bool by_k = pol.top_k && pol.top_k < valid;
    if (!by_k && !by_mass) return;
    if (!by_k && total < 0.0) {
      // ids that weigh less than 2^-100 leave a sum of up to 2^30 of them as it is
      const float least = __double2float_rd(c.top - 69.4 / c.inv_t);
      total = at_least(c, c.flat ? range.lo : max(range.lo, ord32(least))).mass;
    }
    // Without a range from the bins the row is most often a peaked one (logits far above 40 T):
    // a list of the ids of its largest peaks reaches the goal at once. (64 rows of 151,664
    // float32 at a standard deviation of 37 T, top-p 0.9: 697 us by the search below, 76 so;
    // of 128,256 bfloat16 with values of 128 and more: 535 and 56.)
    if (!found && !c.flat && (by_k ? DT == kBF16 && pol.top_k <= kPsList / 2 : true)) {
      clear_hist();
      __syncthreads();
      PsRange best;
      if (range_by_peaks(by_k ? pol.top_k : 128u, top, valid, best) &&
          cut_from_list(c, best, by_k ? pol.top_k : 0u, by_mass, pol.top_p, total))
        return;
      summed = {0.0, 0.0, ~0u};
    }
    if (by_k) {
      if (found && !by_mass) range = *found;
      while (range.inside > kPsList && range.hi != range.lo) refine(c, range, pol.top_k, 0.0);
      if (range.hi == range.lo) c.keep(code_value(range.hi), pol.top_k - range.above);
      else cut_from_list(c, range, pol.top_k, false, 1.0, 0.0);
      if (!by_mass) return;
      const PsBox b = at_least(c, ord32(c.cut) + 1u);
      const double w = c.weight(c.cut);
      total = b.mass + (double)c.take * w;
      const double goal = pol.top_p * total;
      if (b.mass < goal) {
        c.take = ties_to_reach(goal - b.mass, w, c.take, b.mass, goal);
        return;
      }
      range = {top, ord32(c.cut) + 1u, 0u, b.count};
    }
    const double goal = pol.top_p * total;
    const PsRange all = range;
    for (bool guess = found && !by_k;; guess = false) {
      range = guess ? *found : all;
      while (range.inside > kPsList && range.hi != range.lo) {
        const uint32_t width = range.hi - range.lo;
        refine(c, range, 0u, goal);
        if (range.hi - range.lo > width / 4u) bisect(c, range, goal);
      }
      if (range.hi == range.lo) {
        const double above = at_least(c, range.hi + 1u).mass;
        const double w = c.weight(code_value(range.hi));
        if (!guess || (above < goal && above + (double)range.inside * w >= goal)) {
          c.keep(code_value(range.hi), ties_to_reach(goal - above, w, range.inside, above, goal));
          return;
        }
      } else if (cut_from_list(c, range, 0u, true, pol.top_p, total)) {
        return;
      }
      if (!guess) return;  // rounding put the goal past every id: all that was kept stays
      summed = {0.0, 0.0, ~0u};
    }
  }

  // The same out of line, on copies that are made field by field: nothing of the caller's has
  // to live in memory for it (where every asynchronous copy would have it read again).
  struct Outcome {
    float cut;
    uint32_t take;
    int parity;
    PsSummed summed;
  };
  __device__ __noinline__ static void find_cut_on(PolicyRow* row, RowCut* c, const RowPolicy* pol,
                                                  uint32_t top, uint32_t valid, double total,
                                                  const PsRange* range) {
    row->find_cut(*c, *pol, top, valid, total, range);
  }
  __device__ __forceinline__ Outcome find_cut_apart(const RowCut& c, const RowPolicy& pol,
                                                    uint32_t top, uint32_t valid, double total,
                                                    bool have, const PsRange& range) const {
    PolicyRow r(sh);
    r.view.row = view.row, r.view.mask = view.mask;
    r.view.peaks = view.peaks, r.view.list = view.list, r.view.listed = view.listed;
    r.view.base = view.base, r.view.begin = view.begin, r.view.end = view.end;
    r.view.vocab = view.vocab, r.view.off = view.off;
    r.view.slots = view.slots, r.view.slot_bytes = view.slot_bytes;
    r.view.kept = view.kept;
    r.rank = rank, r.k = k, r.warp_ids = warp_ids, r.row_end = row_end;
    r.warp = warp, r.lane = lane, r.entry = entry, r.parity = parity;
    RowCut x;
    x.top = c.top, x.scale = c.scale, x.inv_t = c.inv_t, x.min_p = c.min_p;
    x.powers = c.powers, x.cut = c.cut, x.cut2 = c.cut2, x.take = c.take, x.flat = c.flat;
    RowPolicy y;
    y.temperature = pol.temperature, y.top_p = pol.top_p, y.min_p = pol.min_p;
    y.top_k = pol.top_k, y.ok = pol.ok;
    PsRange z;
    z.hi = range.hi, z.lo = range.lo, z.above = range.above, z.inside = range.inside;
    find_cut_on(&r, &x, &y, top, valid, total, have ? &z : nullptr);
    Outcome o;
    o.cut = x.cut, o.take = x.take, o.parity = r.parity;
    o.summed.lane = r.summed.lane, o.summed.all = r.summed.all;
    o.summed.down_to = r.summed.down_to;
    return o;
  }

  // ---- the kept mass and the draw -------------------------------------------------------
  // Publishes this warp's entry to the cluster; the first warp of every CTA scans them all, a
  // lane holding up to kPer in id order. `w_tie` is the weight of an id at the cut, `mass` that
  // above it; set 1 leaves the ties as set 0 published them.
  static constexpr int kPer = kPsEntries / 32;
  __device__ PsScan scan_entries(int set, double mass, uint32_t ties, uint32_t before,
                                 uint32_t take, double w_tie, double u) {
    if ((uint32_t)lane < k) {
      PsShared* r = ps_remote(&sh, lane);
      r->entry_mass[set][entry] = mass;
      if (set == 0) {
        r->entry_ties[entry] = ties;
        r->entry_before[entry] = before;
      }
    }
    publish();
    if (warp == 0) {
      const int n = (int)k * kPsWarps, per = (n + 31) / 32, first = lane * per;
      uint32_t t[kPer], tie_sum = 0, draft = 0;
      double m[kPer], sum = 0.0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const bool have = i < per && first + i < n;
        t[i] = have ? sh.entry_ties[first + i] : 0u;
        m[i] = have ? sh.entry_mass[set][first + i] : 0.0;
        draft += have ? sh.entry_before[first + i] : 0u;
        tie_sum += t[i];
      }
      const uint32_t tie_start = warp_scan(tie_sum, lane) - tie_sum;
      uint32_t run = tie_start;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t kept = run < take ? min(t[i], take - run) : 0u;
        if (kept) m[i] += (double)kept * w_tie;
        const int own = first + i - (int)rank * kPsWarps;  // a warp of this CTA
        if (set == 0 && i < per && own >= 0 && own < kPsWarps) sh.ties_before[own] = run;
        run += t[i];
        sum += m[i];
      }
      const double incl = warp_scan(sum, lane);
      double acc = __shfl_up_sync(~0u, incl, 1);
      if (lane == 0) acc = 0.0;
      const double total = __shfl_sync(~0u, incl, 31);
      draft = __reduce_add_sync(~0u, draft);
      const double goal = u * total;
      // the first entry that passes the goal; the last with mass, if rounding leaves none
      int hit = kPsEntries, last = -1;
      double hit_mass = 0.0, last_mass = 0.0;
      uint32_t hit_ties = 0, last_ties = 0;
      run = tie_start;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (m[i] > 0.0) {
          last = first + i, last_mass = acc, last_ties = run;
          if (hit == kPsEntries && acc + m[i] > goal) hit = last, hit_mass = acc, hit_ties = run;
        }
        acc += m[i];
        run += t[i];
      }
      const int winner = __reduce_min_sync(~0u, hit);
      const int final = __reduce_max_sync(~0u, last);
      if (lane == 0) sh.scan[set].total = total, sh.scan[set].draft_before = draft;
      if (winner < kPsEntries ? hit == winner : final >= 0 ? last == final : lane == 0) {
        const bool passed = winner < kPsEntries;
        sh.scan[set].owner = passed ? hit : max(last, 0);
        sh.scan[set].mass_before = passed ? hit_mass : last_mass;
        sh.scan[set].ties_before = passed ? hit_ties : last_ties;
      }
    }
    __syncthreads();
    return sh.scan[set];
  }

  // sets of the lane's 8 values: above the cut, equal to it
  __device__ __forceinline__ static void split(const RowCut& c, const Raw& r, uint32_t& above,
                                               uint32_t& tie) {
    above = tie = 0u;
    if constexpr (DT == kF32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = View::value_of(r, j);
        if (v > c.cut) above |= 1u << j;
        if (v == c.cut) tie |= 1u << j;
      }
    } else {
      // two values at a time; no value lies between the cut and the cut rounded down
      const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t at = 0x00020001u << (2 * i);
        above |= greater2(w[i], c.cut2) & at;
        tie |= equal2(w[i], c.cut2) & at;
      }
      above = (above | above >> 16) & 0xFFu;
      tie = (tie | tie >> 16) & 0xFFu;
    }
    above &= r.bits;
    tie &= r.bits;
  }
  __device__ __forceinline__ static uint32_t greater2(uint32_t a, uint32_t b) {
    uint32_t m;
    if constexpr (DT == kBF16) asm("set.gt.u32.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    else asm("set.gt.u32.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    return m;
  }
  __device__ __forceinline__ static uint32_t equal2(uint32_t a, uint32_t b) {
    uint32_t m;
    if constexpr (DT == kBF16) asm("set.eq.u32.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    else asm("set.eq.u32.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    return m;
  }
  // the cut in the row's own type, rounded down, twice
  __device__ __forceinline__ static uint32_t twice(float cut) {
    if constexpr (DT == kBF16) {
      return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rd(cut)) * 0x10001u;
    } else if constexpr (DT == kF16) {
      return (uint32_t)__half_as_ushort(__float2half_rd(cut)) * 0x10001u;
    } else {
      return 0u;
    }
  }

  // f(id, raw values, set of the kept ones) over the vectors of `part` that may hold some;
  // `ties_before`: ids at the cut before it. A kept id may still weigh less than min_p.
  template <class F>
  __device__ __forceinline__ void each_kept(const View& part, const RowCut& c,
                                            uint32_t ties_before, F&& f) {
    uint32_t run = ties_before;
    part.each(lane, [&](uint32_t pos, const Raw& r) {
      uint32_t set, tie;
      split(c, r, set, tie);
      if (c.take && __any_sync(~0u, tie)) {
        const uint32_t n = __popc(tie);
        const uint32_t incl = warp_scan(n, lane);
        uint32_t at = run + incl - n;
        run += __shfl_sync(~0u, incl, 31);
        while (tie && at < c.take) {
          set |= tie & (0u - tie);
          tie &= tie - 1u;
          ++at;
        }
      }
      if (__any_sync(~0u, set)) f(view.id_of(pos), r, set);
    });
  }

  // The first id of `part`, in id order, at which the weights summed from `run` on exceed
  // `goal` (the last with a weight, if rounding leaves none). Whole warp; all lanes return it.
  template <class W>
  __device__ int walk(const View& part, const RowCut& c, uint32_t ties_before, double run,
                      double goal, W&& weigh) {
    int found = -1, final = -1;
    each_kept(part, c, ties_before, [&](int id, const Raw& r, uint32_t set) {
      if (found >= 0) return;  // uniform over the warp
      double sum = 0.0;
      int mine = -1;
      each_weight(c, r, set, [&](int j, double w) {
        w = weigh(id + j, w);
        sum += w;
        if (w > 0.0) mine = id + j;
      });
      const double incl = warp_scan(sum, lane);
      const uint32_t over = __ballot_sync(~0u, sum > 0.0 && run + incl > goal);
      if (over) {
        const int src = __ffs(over) - 1;
        const double prev = __shfl_up_sync(~0u, incl, 1);
        double acc = run + (lane ? prev : 0.0);
        int at = -1;
        each_weight(c, r, set, [&](int j, double w) {
          w = weigh(id + j, w);
          acc += w;
          if (at < 0 && w > 0.0 && acc > goal) at = id + j;
        });
        found = __shfl_sync(~0u, at < 0 ? mine : at, src);
        return;
      }
      final = max(final, mine);
      run += __shfl_sync(~0u, incl, 31);
    });
    return found >= 0 ? found : __reduce_max_sync(~0u, final);
  }

  // The draw, in the CTA that has the owner. A short list its owner walks alone. A long one is
  // cut into pieces, whose sums the warps take in turn; the warp that summed the piece that
  // holds the goal walks that. Returns the id in the walking warp, -1 in the others.
  // weigh(id, kept weight) is the weight to use.
  template <class W>
  __device__ int draw(const RowCut& c, const PsScan& s, double goal, W&& weigh) {
    const int own = s.owner % kPsWarps, all = sh.listed_by[own];
    View list = view;
    const uint64_t begin = (uint64_t)s.owner * warp_ids;
    list.begin = (uint32_t)min(begin, (uint64_t)row_end);
    list.end = (uint32_t)min(begin + warp_ids, (uint64_t)row_end);
    list.list += (own - warp) * (int)(warp_ids >> 3);
    list.listed = all;
    if (all <= 64) {
      if (warp != own) return -1;
      return walk(list, c, s.ties_before, s.mass_before, goal, weigh);
    }
    int wide = 32;
    while ((all + wide - 1) / wide > kPsUnits) wide *= 2;
    const int n = (all + wide - 1) / wide;
    auto piece = [&](int i) { return list.slice(i * wide, min(all, (i + 1) * wide)); };
    double* masses = ps_unit_mass();
    uint32_t* ties = ps_unit_ties();
    if (c.take) {
      for (int i = warp; i < n; i += kPsWarps) {
        uint32_t t = 0;
        piece(i).each(lane, [&](uint32_t, const Raw& r) {
          uint32_t set, tie;
          split(c, r, set, tie);
          t += __popc(tie);
        });
        t = __reduce_add_sync(~0u, t);
        if (lane == 0) ties[i] = t;
      }
      __syncthreads();
    }
    auto ties_at = [&](int i) {
      uint32_t t = 0;
      if (c.take)
        for (int j = lane; j < i; j += 32) t += ties[j];
      return s.ties_before + __reduce_add_sync(~0u, t);
    };
    for (int i = warp; i < n; i += kPsWarps) {
      double m = 0.0;
      each_kept(piece(i), c, ties_at(i), [&](int id, const Raw& r, uint32_t set) {
        each_weight(c, r, set, [&](int j, double w) { m += weigh(id + j, w); });
      });
      m = warp_sum(m);
      if (lane == 0) masses[i] = m;
    }
    __syncthreads();
    // the piece that holds the goal, and the mass before it
    int hit = -1, last = 0;
    double run = s.mass_before, hit_run = run, last_run = run;
    for (int i = 0; i < n && hit < 0; i += 32) {
      const double m = i + lane < n ? masses[i + lane] : 0.0;
      const double incl = warp_scan(m, lane);
      const double prev = __shfl_up_sync(~0u, incl, 1);
      const double before = run + (lane ? prev : 0.0);
      const uint32_t over = __ballot_sync(~0u, m > 0.0 && run + incl > goal);
      const uint32_t some = __ballot_sync(~0u, m > 0.0);
      if (over) {
        hit = i + __ffs(over) - 1;
        hit_run = __shfl_sync(~0u, before, __ffs(over) - 1);
      } else if (some) {
        last = i + 31 - __clz(some);
        last_run = __shfl_sync(~0u, before, 31 - __clz(some));
      }
      run += __shfl_sync(~0u, incl, 31);
    }
    if (hit < 0) hit = last, hit_run = last_run;  // what rounding leaves
    if (hit % kPsWarps != warp) return -1;
    return walk(piece(hit), c, ties_at(hit), hit_run, goal, weigh);
  }
};

// What the pass that reads the row from HBM finds in a lane's values.
struct PsFirst {
  uint32_t peak;  // of 16-bit types: the largest peak
  float top;      // float32: the largest value, a NaN with a NaN
  uint32_t count, small;  // valid ids; bfloat16: those next to zero
  double mass;    // MASS: of all ids relative to `from`; bfloat16 with small_mass: of those
                  // next to zero relative to 0
};

// The least value whose weight the first pass adds up, relative to `from`: 2^-937.5 at least,
// which exp2_from() can form. Rounded up, for next to a `from` of 10^10 T the float below the
// bound lies past that range; and finite, so that a value of -inf counts at no temperature.
__device__ __forceinline__ float mass_floor(double from, double scale) {
  return fmaxf(__double2float_ru(from - 15000.0 / scale), -FLT_MAX);
}

// The pass behind the copies of start_stream(): peaks, and with BINS the histogram, with MASS
// the weights. One loop for each of the four, on scalars of its own, and the chunks at the edges
// of a row apart from it: as one lambda called from a method of the view, 256 rows of 128,256
// bfloat16 took 34 us for the maximum alone with one CTA a row, and 23 so.
template <int DT, bool BINS, bool MASS>
__device__ __forceinline__ PsFirst first_pass(const RowView<DT>& view, int lane,
                                              const typename PolicyRow<DT>::Linear& bins,
                                              double from, double scale, bool small_mass,
                                              const PsPowers& powers) {
  using View = RowView<DT>;
  using Row = PolicyRow<DT>;
  using S = typename Elem<DT>::storage;
  constexpr int kVec = DT == kF32 ? 4 : 8, kDepth = View::kDepth;
  const uint32_t* const mask = view.mask;
  const int n = view.chunks();
  const uint32_t bytes = (uint32_t)view.slot_bytes;
  const bool kept = view.kept;
  // chunks inside the row; the others are copied and read with care
  const int id_first = view.id_of(view.begin);
  const PsInner inner = ps_inner_chunks(id_first, n, view.vocab, kPsChunk);
  const uint32_t start = view.slots;
  const uint32_t stop = kept ? 0xFFFFFFFFu : start + kDepth * bytes;
  uint32_t slot = view.first_slot(), fill = stop - bytes;
  const S* src = view.row + (id_first + (kDepth - 1) * kPsChunk + lane * kVec);
  const int ahead = kept ? n : kDepth - 1;  // copies started when a chunk is read
  const int half = kept ? n / 2 : -1;
  uint32_t peak_at = (uint32_t)__cvta_generic_to_shared(ps_unit_ties()), peak_step = 0u;
  if (view.peaks) {  // (else all go to a place that is not read before it is written again)
    peak_at = (uint32_t)__cvta_generic_to_shared(view.peaks) +
              2u * (((view.begin - view.base) >> 3) + (uint32_t)lane);
    peak_step = 64u;
  }
  const uint32_t hist = (uint32_t)__cvta_generic_to_shared(ps_hist());
  const float scale_b = bins.scale, shift_b = bins.shift;
  const float floor_value = mass_floor(from, scale);
  PsFirst out = {0u, -INFINITY, 0u, 0u, 0.0};
  double mass2 = 0.0;
  if (kept) ps_await_all_but(n - half);

#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    if (!kept) {
      const int next = i + ahead;
      if (ps_copies_inner(next, inner)) {
        ps_copy16(fill + (DT == kF32 ? (lane & 1) * 512 + (lane >> 1) * 16 : lane * 16), src);
        if (DT == kF32)
          ps_copy16(fill + (lane & 1) * 512 + (lane >> 1) * 16 + 256, src + 32 * kVec);
        if (mask) view.copy_words(fill, lane, id_first + next * kPsChunk);
      } else if (ps_copies_edge(next, n)) {
        view.copy_chunk(fill, lane, id_first + next * kPsChunk);
      }
      src += kPsChunk;
      fill += bytes;
      if (fill == stop) fill = start;
      ps_commit();
      ps_await<kDepth - 1>();
    } else if (i == half) {
      ps_await<0>();
    }
    if (DT == kF32 || mask) __syncwarp();  // else a lane reads what it copied itself
    typename View::Raw r;
    r.a = ps_load16(slot + lane * 16);
    if (DT == kF32) r.b = ps_load16(slot + 512 + lane * 16);
    r.bits = 0xFFu;
    bool full = !mask;
    if (i < inner.from || i >= inner.to) {
      const int id = id_first + i * kPsChunk + 8 * lane;
      r.bits = view.inside(id);
      if (r.bits != 0xFFu) view.load_edge(r, id);
      full = false;
    }
    if (mask) {
      const int id0 = id_first + i * kPsChunk, id = id0 + 8 * lane, w = (id >> 5) - (id0 >> 5);
      const uint32_t word = slot + View::kData + 4 * w;
      r.bits &= __funnelshift_r(ps_load4(word), ps_load4(word + 4), id & 31);
    }
    if (DT == kF32 || mask) __syncwarp();  // the slot has been read
    slot += bytes;
    if (slot == stop) slot = start;

    uint32_t v[4] = {~0u, ~0u, ~0u, ~0u};  // masks of the valid ones, 16 bits each
    if (DT != kF32 && !full) expand8_16(r.bits, v[0], v[1], v[2], v[3]);
    const uint32_t peak = View::peak(r, v, full, out.top);
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(peak_at), "h"((uint16_t)peak) : "memory");
    peak_at += peak_step;
    out.peak = max(out.peak, peak);
    if (MASS) {
      if (full) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float x = View::value_of(r, j), y = View::value_of(r, j + 1);
          const double a = exp2_from(fmaxf(x, floor_value), from, scale, powers);
          const double b = exp2_from(fmaxf(y, floor_value), from, scale, powers);
          out.mass += x >= floor_value ? a : 0.0;
          mass2 += y >= floor_value ? b : 0.0;
        }
      } else {
        View::each_set(r.bits, [&](int j, bool have) {
          const float x = View::value_at(r, j);
          const double a = exp2_from(fmaxf(x, floor_value), from, scale, powers);
          if (have && x >= floor_value) out.mass += a;
        });
      }
    }
    out.count += __popc(r.bits);
    if (BINS) {
      if constexpr (DT == kBF16) {
        const uint32_t near =
            Row::count_values(hist, r.a.x, v[0]) | Row::count_values(hist, r.a.y, v[1]) |
            Row::count_values(hist, r.a.z, v[2]) | Row::count_values(hist, r.a.w, v[3]);
        if (__any_sync(~0u, near)) {
          uint32_t set = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (fabsf(View::value_of(r, j)) < kPsSmall) set |= 1u << j;
          set &= r.bits;
          out.small += __popc(set);
          if (small_mass)
            View::each_set(set, [&](int j, bool have) {
              const double w = exp2_table((double)View::value_at(r, j) * scale, powers);
              if (have) out.mass += w;
            });
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          Row::count_linear(hist, scale_b, shift_b, View::value_of(r, j),
                            full || (r.bits >> j & 1u));
      }
    }
  }
  if (!kept) ps_await<0>();  // the last groups are empty; what follows writes over the ring
  out.mass += mass2;
  return out;
}

// zeros for the ids [begin, end) of a row of probabilities, by the threads of a CTA
__device__ __forceinline__ void clear_probs(float* row, uint32_t begin, uint32_t end) {
  const uint32_t lead = (uint32_t)(-(int)(reinterpret_cast<uintptr_t>(row + begin) >> 2)) & 3u;
  const uint32_t body = min(end, begin + lead), vecs = (end - body) / 4u;
  if (threadIdx.x < body - begin) row[begin + threadIdx.x] = 0.0f;
  float4* v = reinterpret_cast<float4*>(row + body);
  for (uint32_t i = threadIdx.x; i < vecs; i += kPsThreads)
    v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const uint32_t tail = body + 4u * vecs;
  if (threadIdx.x < end - tail) row[tail + threadIdx.x] = 0.0f;
}

template <int DT, int OP>
__global__ void __launch_bounds__(kPsThreads, 2) policy_kernel(const PolicyParams p) {
  using Row = PolicyRow<DT>;
  using View = RowView<DT>;
  __shared__ PsShared sh;
  const uint32_t k = (uint32_t)p.k;
  // the barrier's first phase: every CTA of the cluster runs before its memory is written
  if (k > 1) ps_cluster_arrive();
  asm volatile("griddepcontrol.launch_dependents;" :::);

  int64_t item = (int64_t)(blockIdx.x / k), group = item;
  int sub = 0;
  if (OP == kOpSpec) {
    group = item / p.sub_count;
    sub = p.sub_from + (int)(item - group * p.sub_count);
    item = group * p.per_group + sub;
  }

  Row row(sh);
  row.rank = k > 1 ? ps_rank() : 0u;
  row.k = k;
  row.warp = threadIdx.x >> 5;
  row.lane = threadIdx.x & 31;
  row.entry = (int)row.rank * kPsWarps + row.warp;
  View& view = row.view;
  using S = typename Elem<DT>::storage;
  view.row = static_cast<const S*>(p.logits) + group * p.group_stride + sub * p.row_stride;
  view.mask = p.mask ? p.mask + group * p.mask_group_stride + sub * p.mask_row_stride : nullptr;
  view.vocab = (int)p.vocab;
  view.off = (int)((reinterpret_cast<uintptr_t>(view.row) & 15u) / sizeof(S));
  row.warp_ids = (uint32_t)p.warp_ids;
  row.row_end = (uint32_t)p.vocab + (uint32_t)view.off;
  const uint64_t begin = (uint64_t)row.entry * row.warp_ids;
  view.base = row.rank * kPsWarps * row.warp_ids;
  view.begin = (uint32_t)min(begin, (uint64_t)row.row_end);
  view.end = (uint32_t)min(begin + row.warp_ids, (uint64_t)row.row_end);
  view.peaks = p.peaks ? reinterpret_cast<uint16_t*>(ps_dynamic + kPsFixed) : nullptr;
  view.list = reinterpret_cast<uint16_t*>(ps_dynamic + p.lists) + row.warp * (row.warp_ids >> 3);
  view.listed = 0;
  view.kept = p.keep != 0;
  view.slot_bytes = ps_slot(DT, view.mask != nullptr);
  view.slots = (uint32_t)__cvta_generic_to_shared(ps_dynamic) + (uint32_t)p.slots +
               (view.kept ? 0u : (uint32_t)(row.warp * View::kDepth * view.slot_bytes));
  row.clear_hist();
  if (threadIdx.x < 16) sh.powers.at[threadIdx.x] = exp2((double)threadIdx.x / 16.0);
  __syncthreads();

  // what came before on the stream has written the inputs
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (OP == kOpSpec && p.sub_from > 0) {
    // an earlier launch may have decided the entry (rows past its drafts wrote nothing)
    const int last = p.draft_lens ? p.draft_lens[group] : p.per_group - 1;
    const int rows = last < p.sub_from ? last + 1 : p.sub_from;
    bool decided = false;
    for (int i = 0; i < rows; ++i)
      decided |= p.results[group * p.per_group + i].x == kDecided;
    if (decided) {
      if (k > 1) ps_cluster_wait();
      return;
    }
  }
  view.start_stream(row.lane);  // the copies run while the policy is read

  const RowPolicy pol = load_policy(p.policies + group * p.policy_stride);
  bool ok = pol.ok;
  double u = 0.0, u_accept = 0.0;
  int len = 0;
  if (OP == kOpDraw) u = load_uniform(p, group * p.uniform_stride);
  if (OP == kOpSpec) {
    len = p.draft_lens ? p.draft_lens[group] : p.per_group - 1;
    u = load_uniform(p, group * p.uniform_stride + p.per_group - 1);
    if (sub < len && sub < p.per_group - 1)
      u_accept = load_uniform(p, group * p.uniform_stride + sub);
    ok = ok && len >= 0 && len < p.per_group && u_accept >= 0.0 && u_accept < 1.0;
  }
  if (OP != kOpProbs) ok = ok && u >= 0.0 && u < 1.0;
  if (OP == kOpProbs) {
    const uint64_t first = (uint64_t)row.rank * kPsWarps * row.warp_ids;
    clear_probs(p.out_probs + group * p.out_stride, (uint32_t)min(first, (uint64_t)p.vocab),
                (uint32_t)min(first + kPsWarps * row.warp_ids, (uint64_t)p.vocab));
  }
  if (k > 1) ps_cluster_wait();

  const bool first = row.rank == 0 && threadIdx.x == 0;
  uint32_t status = ok ? 0u : kStatusBadPolicy;
  if (OP == kOpSpec && ok && sub > len) {  // a row past the entry's drafts
    ps_await<0>();
    return;
  }

  RowCut c = {};
  c.inv_t = fmin(1.0 / pol.temperature, 1e300);  // 0 times it stays 0
  c.scale = c.inv_t * (16.0 * 1.4426950408889634);
  c.min_p = pol.min_p;
  c.powers = &sh.powers;
  c.cut = -INFINITY;
  if (ok) {
    const bool by_mass = pol.top_p < 1.0;
    const bool cuts = pol.temperature > 0.0 && (pol.top_k || by_mass);
    // A small top-k goes by the peaks, not the bins. (One float32 row of 32,000: 19.2 -> 17.5 us.
    // Not bfloat16, whose bins need no list: 256 rows of 128,256, top-k 50, took 85 us by the
    // peaks, 65 by the bins.)
    const bool by_peaks = DT != kBF16 && cuts && pol.top_k && pol.top_k <= kPsList / 2;
    const bool bins = cuts && !by_peaks;
    // The mass of all ids is summed where top-p needs it and the bins do not give it, and where
    // nothing is cut. The maximum is not known yet: it is summed relative to one of the row's
    // values (the weights of equal values come out as 1).
    const bool plain = pol.temperature > 0.0 && !cuts && !(pol.min_p > 0.0);
    const bool mass_of_all = plain || (DT != kBF16 && bins && by_mass && !pol.top_k);
    typename Row::Linear lin = {};
    double from = 0.0;
    if (DT != kBF16) {
      lin = row.sample_bins((float)(c.inv_t * Row::kBinsPerE), from);
    } else if (plain) {
      const float x = Elem<DT>::to_f32(view.row, 0);
      if (fabsf(x) < 512.0f) from = x;
    }
    PsFirst f;
    if (bins && mass_of_all) {
      if constexpr (DT != kBF16)
        f = first_pass<DT, true, true>(view, row.lane, lin, from, c.scale, false, sh.powers);
    } else if (bins) {
      f = first_pass<DT, true, false>(view, row.lane, lin, from, c.scale, by_mass, sh.powers);
    } else if (mass_of_all) {
      f = first_pass<DT, false, true>(view, row.lane, lin, from, c.scale, false, sh.powers);
    } else {
      f = first_pass<DT, false, false>(view, row.lane, lin, from, c.scale, false, sh.powers);
    }
    // order code of the maximum, 0 without a valid id
    uint32_t top = f.peak == 0u ? 0u : DT == kF32 ? ord32(f.top) : View::top_code(f.peak);
    PsBox sum = row.reduce(f.mass, f.count, top, f.small);
    top = sum.top;
    if (top == 0u) status = kStatusEmptyMask;
    if (top == kOrd32NaN) status = kStatusNanInSupport;
    if (top == kOrd32NegInf) status = kStatusAllNegInf;
    if (!status) {
      c.top = code_value(top);
      c.flat = !(pol.temperature > 0.0) || c.top == INFINITY;
      // The masses relative to the maximum, where they did not leave the range of doubles. Where
      // `from` lies above it (a masked id), the floor below `from` must leave out nothing that
      // counts: 2000 above the floor, it leaves out weights below 2^-125.
      const double shift = (from - c.top) * c.scale;
      const bool in_range = shift > -14400.0 && shift < (mass_of_all ? 13000.0 : 14400.0);
      const double factor = in_range ? exp2_table(shift, sh.powers) : 0.0;
      sum.mass = sum.mass > 0.0 ? sum.mass * factor : 0.0;
      // (not if the temperature is so low that the pass could not tell `from` from its floor)
      const bool measured =
          mass_of_all && in_range && (double)mass_floor(from, c.scale) < from - 1e-30;
      // What top-p measures by. Relative to the maximum equal values weigh exactly 1, and a mass
      // that equals its goal (270 of 300 equal ids at 0.9) has reached it; the sums relative to
      // `from` round each weight, by some 2^-51 of it, and the factor keeps that so.
      const double total = measured ? sum.mass * (1.0 - 0x1p-48) : -1.0;
      if (!cuts) {
        if (pol.temperature > 0.0) c.cut = c.flat ? FLT_MAX : -INFINITY;
        else c.keep(code_value(top), 1u);
        // The warps' parts of it serve the draw where every weight that they hold is one relative
        // to the maximum too (not below 2^-1000, which counts as 0 there), and where none that
        // lies below the floor can be drawn.
        const bool drawable = shift > -990.0 && (OP == kOpProbs || u >= 0x1p-64);
        if (plain && measured && !c.flat && drawable) row.summed = {f.mass * factor, sum.mass, 0u};
      } else {
        PsRange range = {}, safe = {};
        bool found = false, near = false;
        if (by_peaks) {
          if constexpr (DT != kBF16)
            found = !c.flat && row.range_by_peaks(pol.top_k, top, sum.count, range);
        } else if (in_range && (measured || !mass_of_all)) {
          if constexpr (DT == kBF16) found = row.cut_by_values(c, pol, sum);
          else found = row.range_by_bins(c, pol, sum, lin, total, range, safe);
        }
        if (DT != kBF16 && found && (by_peaks || range.inside <= kPsList)) {
          __syncthreads();  // what the scans left in shared memory has been read
          const bool by_k = by_peaks || (pol.top_k && pol.top_k < sum.count);
          found = row.cut_from_list(c, range, by_k ? pol.top_k : 0u, by_mass, pol.top_p, total);
          if (!found) {  // the range lay too low, or was too long for a list
            row.summed = {0.0, 0.0, ~0u};
            near = !by_peaks && !by_k;
            range = safe;
          }
        } else if (DT != kBF16 || !found) {
          near = found;
          found = false;
        }
        if (!found) {
          __syncthreads();  // (as above)
          const auto o =
              row.find_cut_apart(c, pol, top, sum.count, total, near, range);
          c.keep(o.cut, o.take);
          row.parity = o.parity;
          row.summed = o.summed;
        }
      }
      c.bound_by_min_p();
      c.cut2 = Row::twice(c.cut);
    }
  }

  if (status) {
    if (first) {
      if (OP == kOpDraw) p.out_idx[item] = -1;
      if (OP == kOpSpec) p.results[item] = make_int4(kDecided, -1, (int)status, 0);
      else p.out_status[item] = status;
    }
    ps_await<0>();  // a row that was not looked at: its copies have to land all the same
    return;
  }

  // the kept mass and the ties at the cut, by warps; for a drafted row also the ties before it
  int draft = -1;
  if (OP == kOpSpec && sub < len) {
    draft = p.drafts[group * p.draft_stride + sub];
    if (draft < 0 || draft >= view.vocab) draft = -1;
  }
  // what finding the cut has summed already, if min_p takes nothing from it
  const bool summed = !(c.min_p > 0.0);
  const uint32_t down_to = summed ? row.summed.down_to : ~0u;
  double mass = summed ? row.summed.lane : 0.0;
  uint32_t ties = 0, before = 0;
  // An id at the cut weighs what the passes below take it for: a weight out of the table differs
  // from the formula's in the last places, and min_p may lie between them.
  const double w_tie = c.take ? row.weight(c, c.cut) : 0.0;
  if (w_tie < c.min_p) c.take = 0u;
  if (c.cut == -INFINITY) view.peaks = nullptr;  // nothing is cut: every vector
  view.gather(row.lane, c.least());
  if (row.lane == 0) sh.listed_by[row.warp] = view.listed;
  if (down_to != 0u) view.each(row.lane, [&](uint32_t pos, const auto& r) {
    uint32_t set, tie;
    Row::split(c, r, set, tie);
    ties += __popc(tie);
    if (OP == kOpSpec) {
      const int ahead = draft - view.id_of(pos);
      if (ahead > 0) before += __popc(ahead < 8 ? tie & ((1u << ahead) - 1u) : tie);
    }
    if (down_to != ~0u) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ord32(View::value_of(r, j)) > down_to) set &= ~(1u << j);
    }
    mass += row.sum_of(c, r, set, c.min_p);
  });
  mass = warp_sum(mass);
  ties = __reduce_add_sync(~0u, ties);
  before = __reduce_add_sync(~0u, before);
  auto scan = row.scan_entries(0, mass, ties, before, c.take, w_tie, u);
  const double inv = 1.0 / scan.total;

  if (OP == kOpProbs) {
    float* out = p.out_probs + group * p.out_stride;
    row.each_kept(view, c, sh.ties_before[row.warp], [&](int id, const auto& r, uint32_t set) {
      row.each_weight(c, r, set, [&](int j, double w) { out[id + j] = (float)(w * inv); });
    });
    if (first) p.out_status[item] = 0u;
    return;
  }

  bool residual = false;
  const float* q = nullptr;
  if (OP == kOpSpec && sub < len) {
    double p_d = 0.0, q_d = 1.0;
    if (p.draft_probs) q = p.draft_probs + group * p.dp_group_stride + sub * p.dp_row_stride;
    if (draft >= 0) {
      if (q) q_d = fmax((double)q[draft], 0.0);
      const bool valid = !view.mask || (view.mask[draft >> 5] >> (draft & 31) & 1u);
      const float v = Elem<DT>::to_f32(view.row, draft);
      if (valid && (v > c.cut || (v == c.cut && scan.draft_before < c.take))) {
        const double w = row.weight(c, v);
        if (w >= c.min_p) p_d = w / scan.total;
      }
    }
    if (draft >= 0 && u_accept * q_d < p_d) {
      if (first) p.results[item] = make_int4(kAccepted, -1, 0, 0);
      return;
    }
    residual = true;
  }

  // what remains of p where the draft's probability is taken off
  auto rest = [&](int id, double w) {
    if (!residual) return w;
    const double q_id = q ? fmax((double)q[id], 0.0) : id == draft ? 1.0 : 0.0;
    return fmax(w * inv - q_id, 0.0);
  };
  if (OP == kOpSpec && residual) {
    double sum = 0.0;
    row.each_kept(view, c, sh.ties_before[row.warp], [&](int id, const auto& r, uint32_t set) {
      row.each_weight(c, r, set, [&](int j, double w) { sum += rest(id + j, w); });
    });
    sum = warp_sum(sum);
    const auto left = row.scan_entries(1, sum, 0u, 0u, 0u, 0.0, u);
    residual = left.total > 0.0;  // else the draft covers p everywhere: draw from p itself
    if (residual) scan = left;
  }
  if (scan.owner / kPsWarps != (int)row.rank) return;
  const int id = row.draw(c, scan, u * scan.total, rest);
  if (id >= 0 && row.lane == 0) {
    if (OP == kOpDraw) {
      p.out_idx[item] = id;
      p.out_status[item] = 0u;
    } else {
      p.results[item] = make_int4(kDecided, id, 0, 0);
    }
  }
}

// Joins the rows of every entry: the first row that decides ends it.
__global__ void spec_join_kernel(const int4* results, int64_t batch, int per_group,
                                 const int32_t* draft_lens, int32_t* accept_len,
                                 int32_t* token, uint32_t* status) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= batch) return;
  const int4* r = results + b * per_group;
  int len = draft_lens ? draft_lens[b] : per_group - 1;
  len = len < 0 || len >= per_group ? 0 : len;
  int i = 0;
  int4 x = r[0];
  while (x.x == kAccepted && i < len) x = r[++i];
  accept_len[b] = i;
  token[b] = x.y;
  status[b] = (uint32_t)x.z;
}

}  // namespace onyx
