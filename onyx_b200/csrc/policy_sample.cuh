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
// keep a prefix of the ranking, so the kept set is given by a cut (an order code), the number
// of ids equal to it that are kept in id order (`take`) and the bound w >= min_p. The draw is
// the first kept id, in id order, whose cumulative weight exceeds u times the kept total.
//
// Sums and weights are float64: whether a cumulative mass reaches p, or an id's interval holds
// u, decides a whole number, and float32 sums over 10^5 ids would decide it differently for
// about one row in a hundred.
//
// Shape of the work. One cluster of k CTAs per row (k = 1, 2, 4 or 8, the more the fewer the
// rows); CTA ranks, the warps of a CTA and the 256-id chunks of a warp follow id order, a lane
// holding 8 consecutive ids. A row is streamed from HBM by the first pass and from L2 by the
// later ones, so no row length is bound to shared memory. Cluster-wide sums: every CTA stores
// its part into every CTA's box (distributed shared memory), one cluster barrier publishes
// them, and all CTAs combine the boxes in rank order, so all hold identical totals and take
// the same branches.
#pragma once

#include <cfloat>

#include "onyx_common.cuh"

namespace onyx {

constexpr int kPsThreads = 512;
constexpr int kPsWarps = kPsThreads / 32;
constexpr int kPsMaxCluster = 8;
constexpr int kPsEntries = kPsMaxCluster * kPsWarps;
constexpr int kPsChunk = 256;  // ids a warp handles at a time, 8 to a lane
constexpr int kPsAhead = 4;    // chunks whose loads the streaming pass has in flight

// The value histogram: one bin for every bf16 value with 2^-7 <= |v| < 2^9, in falling order
// of value; positive ones first.
constexpr int kPsBins = 4096;
constexpr int kPsHalf = kPsBins / 2;
constexpr uint32_t kPsLow = 0x3C00u;  // bf16 bits of 2^-7
constexpr int kPsOwn = kPsBins / kPsThreads;  // bins a thread scans

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
  int32_t peaks;     // where in dynamic shared memory the peaks of every 8 ids lie (0: nowhere)
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
  uint32_t count, top;
  uint32_t large, low;
};

struct PsCross {  // the bin in which a count or a mass is reached
  double mass;    // ahead of it
  uint32_t count;  // ahead of it
  uint32_t n;      // ids of it that are kept
  int bin;
};

struct PsShared {
  PsBox box[2][kPsMaxCluster];  // used alternately: one may still be read as the next is written
  double part_mass[kPsWarps];
  uint32_t part_count[kPsWarps], part_top[kPsWarps];
  // one entry per warp of the cluster, in id order; the second set holds what max(p - q, 0)
  // leaves
  double entry_mass[2][kPsEntries];
  uint32_t entry_ties[kPsEntries], entry_before[kPsEntries];
  PsPowers powers;
  uint32_t part_large[kPsWarps], part_low[kPsWarps];
  PsCross cross[2];  // of top-k, of top-p
};

// dynamic shared memory: the histogram, the weights of its bins, the peaks of this CTA's ids
extern __shared__ __align__(16) unsigned char ps_dynamic[];
__device__ __forceinline__ uint32_t* ps_hist() { return reinterpret_cast<uint32_t*>(ps_dynamic); }
// weights of the bins: over the histogram where no other CTA reads it, else behind it
__device__ __forceinline__ double* ps_table(int k) {
  return reinterpret_cast<double*>(ps_dynamic + (k > 1 ? kPsBins * sizeof(uint32_t) : 0));
}

// The part of a row that one warp owns, and how it is read.
template <int DT>
struct RowView {
  using S = typename Elem<DT>::storage;
  const S* row;
  const uint8_t* mask;  // bit t & 7 of byte t >> 3
  uint16_t* peaks;      // of this warp: order code >> 16 of the maximum of every 8 ids, or null
  uint32_t begin, end, vocab;
  bool vec;  // 16-byte loads: the row starts on a 16-byte boundary

  struct Raw {  // 8 consecutive ids as loaded
    uint4 a, b;
    uint32_t bits;
  };

  __device__ __forceinline__ Raw load(uint32_t id) const {
    Raw r;
    r.a = make_uint4(0u, 0u, 0u, 0u);
    if (DT == kF32) r.b = r.a;
    r.bits = 0u;
    if (id >= end) return r;
    const uint32_t left = vocab - id;
    r.bits = mask ? mask[id >> 3] : 0xFFu;
    if (left < 8u) r.bits &= (1u << left) - 1u;
    if (vec && left >= 8u) {
      r.a = *reinterpret_cast<const uint4*>(row + id);
      if (DT == kF32) r.b = *reinterpret_cast<const uint4*>(row + id + 4);
    } else {
      uint32_t u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[j] = 0u;
        if ((uint32_t)j < left) {
          if constexpr (DT == kF32) u[j] = __float_as_uint(row[id + j]);
          else u[j] = row[id + j];
        }
      }
      if constexpr (DT == kF32) {
        r.a = make_uint4(u[0], u[1], u[2], u[3]);
        r.b = make_uint4(u[4], u[5], u[6], u[7]);
      } else {
        r.a = make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16,
                         u[6] | u[7] << 16);
      }
    }
    return r;
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

  // order code of the largest valid value, 0 without one; NaN above all
  __device__ __forceinline__ static uint32_t peak_of(const Raw& r) {
    if (!r.bits) return 0u;
    float m;
    if constexpr (DT == kF32) {
      m = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        m = max_nan_f32(m, r.bits >> j & 1u ? value_of(r, j) : -INFINITY);
    } else {
      const uint32_t none = DT == kBF16 ? 0xFF80FF80u : 0xFC00FC00u;  // -inf twice
      uint32_t m01, m23, m45, m67;
      expand8_16(r.bits, m01, m23, m45, m67);
      const uint32_t a = (r.a.x & m01) | (none & ~m01), b = (r.a.y & m23) | (none & ~m23);
      const uint32_t d = (r.a.z & m45) | (none & ~m45), e = (r.a.w & m67) | (none & ~m67);
      if constexpr (DT == kBF16) {
        const uint32_t x = max_nan_bf16x2(max_nan_bf16x2(a, b), max_nan_bf16x2(d, e));
        m = max_nan_f32(bf16_bits_to_f32(x & 0xFFFFu), bf16_bits_to_f32(x >> 16));
      } else {
        const uint32_t x = max_nan_f16x2(max_nan_f16x2(a, b), max_nan_f16x2(d, e));
        m = max_nan_f32(f16_bits_to_f32(x & 0xFFFFu), f16_bits_to_f32(x >> 16));
      }
    }
    return ord32(m);
  }

  // f(id of the lane's first value, its raw values): the pass that reads the row from HBM.
  // Every lane of the warp makes every call.
  template <class F>
  __device__ __forceinline__ void stream(int lane, F&& f) const {
    uint32_t at = begin;
    for (; at < end; at += kPsAhead * kPsChunk) {
      Raw r[kPsAhead];
#pragma unroll
      for (int i = 0; i < kPsAhead; ++i) r[i] = load(at + i * kPsChunk + 8u * lane);
#pragma unroll
      for (int i = 0; i < kPsAhead; ++i)
        if (at + i * kPsChunk < end) f(at + i * kPsChunk + 8u * lane, r[i]);
    }
  }

  // f(id, raw values) over the chunks that may hold order codes of at least `code`; lanes whose
  // 8 ids hold none get no valid ids. Every lane of the warp makes every call.
  template <class F>
  __device__ __forceinline__ void each(int lane, uint32_t code, F&& f) const {
    for (uint32_t at = begin; at < end; at += kPsChunk) {
      const uint32_t id = at + 8u * lane;
      const bool need = !peaks || peaks[(id - begin) >> 3] >= (code >> 16);
      if (!__any_sync(~0u, need)) continue;
      f(id, load(need ? id : end));
    }
  }
};

// 2^y for y <= 0 (below -1000: 0). Table-driven in the manner of Tang (ACM TOMS 15, 1989):
// y = e + j/16 + f with |f| <= 1/32, 2^f by its Taylor polynomial of degree 6 (the next term
// is below 5e-16 there), so about 1e-15 of the value. 12 float64 operations; the 16 entries
// take the 16 pairs of banks, so lookups of a warp do not conflict.
__device__ __forceinline__ double exp2_neg(double y, const PsPowers& powers) {
  if (!(y > -1000.0)) return 0.0;
  const double shift = 0x1.8p48;  // its last place is 1/16
  const double t = y + shift;
  const int n = __double2loint(t);
  const double f = y - (t - shift);
  const double f2 = f * f;
  // ln 2^k / k!
  const double a = fma(0.2402265069591007, f, 0.6931471805599453);
  const double b = fma(0.009618129107628477, f, 0.05550410866482158);
  const double d = fma(0.00015403530393381608, f, 0.0013333558146428443);
  const double q = fma(fma(d, f2, b), f2, a) * f;
  const double w = powers.at[n & 15];
  const double r = fma(w, q, w);
  return __hiloint2double(__double2hiint(r) + (n >> 4) * (1 << 20), __double2loint(r));
}

// What decides which ids of the row are kept, and their weights.
struct RowCut {
  double top, scale, inv_t, min_p;  // scale = log2(e) / T
  const PsPowers* powers;
  uint32_t cut, take;  // ids above `cut`, and the first `take` ids equal to it
  bool flat;           // every kept id weighs 1 (T = 0, or +inf present)

  __device__ __forceinline__ double weight(float v) const {
    return flat ? 1.0 : exp2_neg(((double)v - top) * scale, *powers);
  }
  // the lowest order code that is kept
  __device__ __forceinline__ uint32_t least() const { return take ? cut : cut + 1u; }

  // Weights below min_p are dropped one by one where they are summed; this raises the cut to
  // a bound below which none passes, which spares looking at them.
  __device__ __forceinline__ void bound_by_min_p() {
    if (flat || !(min_p > 0.0)) return;
    const double low = top + log(min_p) / inv_t * (1.0 + 1e-9) - fabs(top) * 1e-9;
    const uint32_t code = ord32(__double2float_rd(low)) - 1u;
    if (code >= cut) {
      cut = code;
      take = 0u;
    }
    if (take && weight(__uint_as_float(cut & 0x80000000u ? cut & 0x7FFFFFFFu : ~cut)) < min_p)
      take = 0u;
  }
};

template <int DT>
struct PolicyRow {
  using View = RowView<DT>;
  using Raw = typename View::Raw;
  PsShared& sh;
  RowView<DT> view;
  double* table = nullptr;  // weights of the kept bins, where the cut came from them
  uint32_t rank, k;
  int warp, lane, entry;
  int parity = 0;

  __device__ PolicyRow(PsShared& s) : sh(s) {}

  __device__ __forceinline__ void publish() {
    if (k > 1) {
      ps_cluster_arrive();
      ps_cluster_wait();
    } else {
      __syncthreads();
    }
  }

  // cluster-wide sums of the counts and of `mass`, and maximum of `top`
  __device__ PsBox reduce(double mass, uint32_t count, uint32_t top, uint32_t large, uint32_t low) {
    mass = warp_sum(mass);
    count = __reduce_add_sync(~0u, count);
    top = __reduce_max_sync(~0u, top);
    large = __reduce_add_sync(~0u, large);
    low = __reduce_add_sync(~0u, low);
    if (lane == 0) {
      sh.part_mass[warp] = mass, sh.part_count[warp] = count, sh.part_top[warp] = top;
      sh.part_large[warp] = large, sh.part_low[warp] = low;
    }
    __syncthreads();
    if (warp == 0) {
      PsBox b = {};
      for (int i = 0; i < kPsWarps; ++i) {
        b.mass += sh.part_mass[i];
        b.count += sh.part_count[i];
        b.top = max(b.top, sh.part_top[i]);
        b.large += sh.part_large[i];
        b.low += sh.part_low[i];
      }
      if ((uint32_t)lane < k) *ps_remote(&sh.box[parity][rank], lane) = b;
    }
    publish();
    PsBox r = {};
    for (uint32_t i = 0; i < k; ++i) {
      const PsBox b = sh.box[parity][i];
      r.mass += b.mass;
      r.count += b.count;
      r.top = max(r.top, b.top);
      r.large += b.large;
      r.low += b.low;
    }
    parity ^= 1;
    return r;
  }

  // mass and count of the valid ids whose order code is at least `code`
  __device__ PsBox at_least(const RowCut& c, uint32_t code) {
    double mass = 0.0;
    uint32_t count = 0;
    view.each(lane, code, [&](uint32_t, const Raw& r) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((r.bits >> j & 1u) && ord32(View::value_of(r, j)) >= code) {
          mass += c.weight(View::value_of(r, j));
          ++count;
        }
    });
    return reduce(mass, count, 0u, 0u, 0u);
  }

  // fills c.cut and c.take from the policy; `top` is the row's largest order code
  __device__ void find_cut(RowCut& c, const RowPolicy& pol, uint32_t top) {
    const uint32_t base = c.flat ? top - 1u : 0u;  // +inf present: those ids alone
    c.cut = base;
    c.take = 0;
    PsBox above = {0.0, 0u, 0u};  // of the ids above the cut
    bool by_k = false;
    if (!(pol.temperature > 0.0)) {
      c.cut = top;
      c.take = 1;
      return;
    }
    if (pol.top_k && pol.top_k < view.vocab) {
      uint32_t lo = base, hi = top + 1u;
      while (hi - lo > 1u) {
        const uint32_t mid = lo + (hi - lo) / 2u;
        const PsBox b = at_least(c, mid);
        if (b.count >= pol.top_k) {
          lo = mid;
        } else {
          hi = mid;
          above = b;
        }
      }
      if (lo > base) {
        by_k = true;
        c.cut = lo;
        c.take = pol.top_k - above.count;
      }
    }
    if (pol.top_p < 1.0) {
      const double w_cut = by_k ? c.weight(code_value(c.cut)) : 0.0;
      const double total = by_k ? above.mass + (double)c.take * w_cut : at_least(c, base + 1u).mass;
      const double goal = pol.top_p * total;
      uint32_t lo = c.cut, hi = top + 1u;
      PsBox over = {0.0, 0u, 0u}, level = {0.0, 0u, 0u};
      bool have = false;
      while (hi - lo > 1u) {
        const uint32_t mid = lo + (hi - lo) / 2u;
        const PsBox b = at_least(c, mid);
        if (b.mass >= goal) {
          lo = mid;
          level = b;
          have = true;
        } else {
          hi = mid;
          over = b;
        }
      }
      const uint32_t most = have ? level.count - over.count : c.take;
      if (by_k || have) {
        const double w = c.weight(code_value(lo));
        double t = ceil((goal - over.mass) / w);
        t = t < 1.0 ? 1.0 : t > (double)most ? (double)most : t;
        while (t > 1.0 && over.mass + (t - 1.0) * w >= goal) t -= 1.0;
        while (t < (double)most && over.mass + t * w < goal) t += 1.0;
        c.cut = lo;
        c.take = (uint32_t)t;
      }
    }
  }

  // ---- the cut from the value histogram (bf16: a bin is one value) ----------------------
  __device__ static float bin_value(int bin) {
    const uint32_t bits = bin < kPsHalf ? kPsLow + (kPsHalf - 1 - bin)
                                        : 0x8000u | (kPsLow + (bin - kPsHalf));
    return __uint_as_float(bits << 16);
  }

  // counts a value's bin; false for the values that have none
  __device__ __forceinline__ static bool count_bin(uint32_t* hist, uint32_t f32_bits) {
    const uint32_t i = ((f32_bits >> 16) & 0x7FFFu) - kPsLow;
    if (i >= (uint32_t)kPsHalf) return false;
    const uint32_t positive = (uint32_t)((int32_t)~f32_bits >> 31);
    atomicAdd(hist + kPsHalf + (int)(i ^ positive), 1u);
    return true;
  }

  // Sets c.cut and c.take from the counts of every value; `sum` holds what lies outside the
  // bins: `count` and `mass` of |v| < 2^-7, `large` of v >= 2^9, `low` of v <= -2^9. False
  // where the bins do not decide the cut. Every CTA adds up the bins of all CTAs and finds the
  // same cut for itself. `tab` gets the weights of the kept bins; with one CTA it may lie over
  // the histogram.
  __device__ bool find_cut_by_values(RowCut& c, const RowPolicy& pol, const PsBox& sum, double* tab) {
    if (c.flat || sum.large) return false;
    const int mine = threadIdx.x * kPsOwn;  // this thread's bins, in falling order of value
    uint32_t n[kPsOwn] = {};
    for (uint32_t r = 0; r < k; ++r) {
      const uint4* h =
          reinterpret_cast<const uint4*>((k > 1 ? ps_remote(ps_hist(), r) : ps_hist()) + mine);
#pragma unroll
      for (int i = 0; i < kPsOwn / 4; ++i) {
        const uint4 x = h[i];
        n[4 * i] += x.x, n[4 * i + 1] += x.y, n[4 * i + 2] += x.z, n[4 * i + 3] += x.w;
      }
    }
    double w[kPsOwn], mass = 0.0;
    uint32_t count = 0;
    const bool by_mass = pol.top_p < 1.0;
#pragma unroll
    for (int j = 0; j < kPsOwn; ++j) {
      w[j] = by_mass && n[j] ? c.weight(bin_value(mine + j)) : 0.0;
      mass += (double)n[j] * w[j];
      count += n[j];
    }
    if (threadIdx.x < 2) sh.cross[threadIdx.x].bin = -1;
    double mass_before = 0.0, mass_end = 0.0;
    if (by_mass) {
      mass_end = block_scan(mass, sh.part_mass);
      mass_before = __shfl_up_sync(~0u, mass_end, 1);
      if (lane == 0) mass_before = warp ? sh.part_mass[warp - 1] : 0.0;
    }
    uint32_t count_before = block_scan(count, sh.part_count) - count;
    if (mine >= kPsHalf) {  // the values next to zero lie between the halves
      mass_before += sum.mass;
      mass_end += sum.mass;
      count_before += sum.count;
    }
    const uint32_t in_bins = sh.part_count[kPsWarps - 1] + sum.count;
    const double all_mass = by_mass ? sh.part_mass[kPsWarps - 1] + sum.mass : 0.0;
    // the values below -2^9 lie behind the bins; they may weigh nothing next to the rest
    const bool low = sum.low && (c.top + 512.0) * c.inv_t < 60.0;

    int cut_bin = kPsBins;
    uint32_t take = 0;
    double above = 0.0;
    if (pol.top_k && pol.top_k < in_bins + sum.low) {
      if (pol.top_k > in_bins) return false;
      if (count_before < pol.top_k && pol.top_k <= count_before + count) {
        PsCross x = {mass_before, count_before, 0u, -1};
#pragma unroll
        for (int j = 0; j < kPsOwn; ++j)
          if (x.bin < 0) {
            if (pol.top_k <= x.count + n[j]) {
              x.bin = mine + j;
            } else {
              x.count += n[j];
              x.mass += (double)n[j] * w[j];
            }
          }
        sh.cross[0] = x;
      }
      __syncthreads();
      if (sh.cross[0].bin < 0) return false;  // among the values next to zero
      cut_bin = sh.cross[0].bin;
      take = pol.top_k - sh.cross[0].count;
      above = sh.cross[0].mass;
    }
    if (by_mass) {
      const bool by_k = cut_bin < kPsBins;
      if (!by_k && low) return false;
      const double total = by_k ? above + (double)take * c.weight(bin_value(cut_bin)) : all_mass;
      const double goal = pol.top_p * total;
      if (count && mine <= cut_bin && mass_before < goal &&
          (goal <= mass_end || cut_bin < mine + kPsOwn)) {
        PsCross x = {mass_before, 0u, 0u, -1};  // the bin that reaches the goal, else the last
        double run = mass_before, weight = 0.0;
#pragma unroll
        for (int j = 0; j < kPsOwn; ++j)
          if (n[j] && mine + j <= cut_bin && run < goal) {
            x = {run, 0u, mine + j == cut_bin ? take : n[j], mine + j};
            weight = w[j];
            run += (double)x.n * w[j];
          }
        double t = ceil((goal - x.mass) / weight);
        t = t < 1.0 ? 1.0 : t > (double)x.n ? (double)x.n : t;
        while (t > 1.0 && x.mass + (t - 1.0) * weight >= goal) t -= 1.0;
        while (t < (double)x.n && x.mass + t * weight < goal) t += 1.0;
        x.n = (uint32_t)t;
        sh.cross[1] = x;
      }
      __syncthreads();
      if (sh.cross[1].bin < 0) return false;  // among the values next to zero
      cut_bin = sh.cross[1].bin;
      take = sh.cross[1].n;
    }
    c.cut = cut_bin < kPsBins ? ord32(bin_value(cut_bin)) : 0u;
    c.take = cut_bin < kPsBins ? take : 0u;
    // the weights of the kept bins, for the passes that follow
    table = tab;
#pragma unroll
    for (int j = 0; j < kPsOwn; ++j)
      if (n[j] && mine + j <= cut_bin)
        table[mine + j] = by_mass ? w[j] : c.weight(bin_value(mine + j));
    __syncthreads();
    return true;
  }

  // inclusive scan over the CTA; part[w] becomes the sum up to and with warp w
  template <class T>
  __device__ T block_scan(T v, T* part) {
    T incl = warp_scan(v, lane);
    if (lane == 31) part[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      const T x = lane < kPsWarps ? part[lane] : T(0);
      const T y = warp_scan(x, lane);
      if (lane < kPsWarps) part[lane] = y;
    }
    __syncthreads();
    return warp ? part[warp - 1] + incl : incl;
  }

  __device__ static float code_value(uint32_t code) {
    return __uint_as_float((code & 0x80000000u) ? code & 0x7FFFFFFFu : ~code);
  }

  struct Scan {  // of the entries of all warps, as this warp sees them
    double total, mass_before;  // kept mass; of it, before this warp
    uint32_t ties_before, draft_before;
  };

  // Kept mass of the entries that lane `lane` holds: `per` of them, in id order.
  static constexpr int kPer = kPsEntries / 32;
  struct Held {
    double mass[kPer];
    int first, n;
  };
  __device__ __forceinline__ Held held(int set, uint32_t take, double w_tie, uint32_t* ties_run,
                                       uint32_t* ties_at) {
    Held h;
    const int n = (int)k * kPsWarps, per = (n + 31) / 32;
    h.first = lane * per;
    h.n = max(0, min(per, n - h.first));
    uint32_t t[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      t[i] = i < h.n ? sh.entry_ties[h.first + i] : 0u;
      h.mass[i] = i < h.n ? sh.entry_mass[set][h.first + i] : 0.0;
      sum += t[i];
    }
    uint32_t run = warp_scan(sum, lane) - sum;
    *ties_run = run;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      ties_at[i] = run;
      const uint32_t kept = run < take ? min(t[i], take - run) : 0u;
      if (kept) h.mass[i] += (double)kept * w_tie;
      run += t[i];
    }
    return h;
  }

  // Publishes this warp's entry to the cluster and scans all of them; every warp does so for
  // itself. `w_tie` is the weight of an id at the cut, `mass` that above it.
  __device__ Scan scan_entries(int set, double mass, uint32_t ties, uint32_t before,
                               uint32_t take, double w_tie) {
    if ((uint32_t)lane < k) {
      PsShared* r = ps_remote(&sh, lane);
      r->entry_mass[set][entry] = mass;
      if (set == 0) {
        r->entry_ties[entry] = ties;
        r->entry_before[entry] = before;
      }
    }
    publish();
    uint32_t run, at[kPer];
    const Held h = held(set, take, w_tie, &run, at);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += h.mass[i];
    const double incl = warp_scan(sum, lane);
    double acc = __shfl_up_sync(~0u, incl, 1);
    if (lane == 0) acc = 0.0;
    Scan s;
    s.total = __shfl_sync(~0u, incl, 31);
    const int per = ((int)k * kPsWarps + 31) / 32, src = entry / per;
    double mine = 0.0;
    uint32_t mine_ties = 0;
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (h.first + i == entry) mine = acc, mine_ties = at[i];
      if (i < h.n) b += sh.entry_before[h.first + i];
      acc += h.mass[i];
    }
    s.mass_before = __shfl_sync(~0u, mine, src);
    s.ties_before = __shfl_sync(~0u, mine_ties, src);
    s.draft_before = __reduce_add_sync(~0u, b);
    return s;
  }

  // the entry whose interval of kept mass holds `goal` (the last with mass, if rounding leaves
  // none)
  __device__ int find_owner(int set, uint32_t take, double w_tie, double goal) {
    uint32_t run, at[kPer];
    const Held h = held(set, take, w_tie, &run, at);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += h.mass[i];
    const double incl = warp_scan(sum, lane);
    double acc = __shfl_up_sync(~0u, incl, 1);
    if (lane == 0) acc = 0.0;
    int first = kPsEntries, last = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (h.mass[i] > 0.0) {
        last = h.first + i;
        if (acc + h.mass[i] > goal) first = min(first, h.first + i);
        acc += h.mass[i];
      }
    first = __reduce_min_sync(~0u, first);
    last = __reduce_max_sync(~0u, last);
    return first < kPsEntries ? first : last;
  }

  // weight of a kept value
  __device__ __forceinline__ double weight(const RowCut& c, uint32_t f32_bits) const {
    if (DT == kBF16 && table) {
      const uint32_t i = ((f32_bits >> 16) & 0x7FFFu) - kPsLow;
      const uint32_t positive = (uint32_t)((int32_t)~f32_bits >> 31);
      if (i < (uint32_t)kPsHalf) return table[kPsHalf + (int)(i ^ positive)];
    }
    return c.weight(__uint_as_float(f32_bits));
  }

  // f(id, weights of the lane's 8 ids: 0 where not kept) over this warp's ids;
  // `ties_before`: ids at the cut before this warp
  template <class F>
  __device__ __forceinline__ void each_kept(const RowCut& c, uint32_t ties_before, F&& f) {
    uint32_t run = ties_before;
    view.each(lane, c.least(), [&](uint32_t id, const Raw& r) {
      double w[8];
      uint32_t tie = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t code = ord32(View::value_of(r, j));
        const bool valid = r.bits >> j & 1u;
        w[j] = 0.0;
        if (valid && code == c.cut) tie |= 1u << j;
        if (valid && code > c.cut) {
          const double x = weight(c, View::bits_of(r, j));
          if (x >= c.min_p) w[j] = x;
        }
      }
      if (c.take && __any_sync(~0u, tie)) {
        const uint32_t n = __popc(tie);
        const uint32_t incl = warp_scan(n, lane);
        uint32_t at = run + incl - n;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (tie >> j & 1u) {
            if (at < c.take) w[j] = weight(c, View::bits_of(r, j));
            ++at;
          }
        run += __shfl_sync(~0u, incl, 31);
      }
      f(id, w);
    });
  }

  // first id, in id order, whose cumulative weight exceeds `goal`; `start` is the mass before
  // this warp; weigh(id, w[8]) may replace the kept weights. Whole warp; all lanes return it.
  template <class W>
  __device__ int pick(const RowCut& c, uint32_t ties_before, double start, double goal,
                      W&& weigh) {
    int found = -1, last = -1;
    double run = start;
    each_kept(c, ties_before, [&](uint32_t id, double* w) {
      if (found >= 0) return;  // uniform over the warp
      weigh(id, w);
      double s = 0.0;
      int mine = -1;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s += w[j];
        if (w[j] > 0.0) mine = (int)id + j;
      }
      if (!__any_sync(~0u, mine >= 0)) return;
      const double incl = warp_scan(s, lane);
      const uint32_t over = __ballot_sync(~0u, s > 0.0 && run + incl > goal);
      if (over) {
        const int src = __ffs(over) - 1;
        const double prev = __shfl_up_sync(~0u, incl, 1);
        double acc = run + (lane ? prev : 0.0);
        int at = -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          acc += w[j];
          if (at < 0 && w[j] > 0.0 && acc > goal) at = (int)id + j;
        }
        found = __shfl_sync(~0u, at < 0 ? mine : at, src);
        return;
      }
      last = max(last, mine);
      run += __shfl_sync(~0u, incl, 31);
    });
    if (found < 0) found = __reduce_max_sync(~0u, last);
    return found;
  }
};

// zeros for a lane's 8 ids
__device__ __forceinline__ void clear_probs(float* out, uint32_t id, uint32_t end) {
  if (id + 8u <= end && (reinterpret_cast<uintptr_t>(out) & 15u) == 0) {
    reinterpret_cast<float4*>(out + id)[0] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    reinterpret_cast<float4*>(out + id)[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (id + j < end) out[id + j] = 0.0f;
  }
}

template <int DT, int OP>
__global__ void __launch_bounds__(kPsThreads, 2) policy_kernel(const PolicyParams p) {
  __shared__ PsShared sh;
  const uint32_t k = (uint32_t)p.k;
  // the barrier's first phase: every CTA of the cluster runs before its boxes are written
  if (k > 1) ps_cluster_arrive();
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int64_t item = (int64_t)(blockIdx.x / k);
  const int64_t group = OP == kOpSpec ? item / p.per_group : item;
  const int sub = OP == kOpSpec ? (int)(item - group * p.per_group) : 0;

  PolicyRow<DT> row(sh);
  row.rank = k > 1 ? ps_rank() : 0u;
  row.k = k;
  row.warp = threadIdx.x >> 5;
  row.lane = threadIdx.x & 31;
  row.entry = (int)row.rank * kPsWarps + row.warp;
  using S = typename Elem<DT>::storage;
  row.view.row = static_cast<const S*>(p.logits) + group * p.group_stride + sub * p.row_stride;
  row.view.mask = reinterpret_cast<const uint8_t*>(
      p.mask ? p.mask + group * p.mask_group_stride + sub * p.mask_row_stride : nullptr);
  row.view.vocab = (uint32_t)p.vocab;
  const uint64_t begin = (uint64_t)row.entry * (uint32_t)p.warp_ids;
  row.view.begin = (uint32_t)min(begin, (uint64_t)p.vocab);
  row.view.end = (uint32_t)min(begin + (uint32_t)p.warp_ids, (uint64_t)p.vocab);
  row.view.vec = (reinterpret_cast<uintptr_t>(row.view.row) & 15u) == 0;
  row.view.peaks = p.peaks ? reinterpret_cast<uint16_t*>(ps_dynamic + p.peaks) + row.warp * (p.warp_ids >> 3) : nullptr;

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
  if (k > 1) ps_cluster_wait();

  const bool first = row.rank == 0 && threadIdx.x == 0;
  uint32_t status = ok ? 0u : kStatusBadPolicy;
  if (OP == kOpSpec && ok && sub > len) return;  // a row past the entry's drafts

  RowCut c = {};
  c.inv_t = fmin(1.0 / pol.temperature, 1e300);  // 0 times it stays 0
  c.scale = c.inv_t * 1.4426950408889634;
  c.powers = &sh.powers;
  if (threadIdx.x < 16) sh.powers.at[threadIdx.x] = exp2((double)threadIdx.x / 16.0);
  c.min_p = pol.min_p;
  if (ok) {
    // one pass over the row: its maximum, the peaks, and for bf16 the count of every value
    const bool values = DT == kBF16 && pol.temperature > 0.0 && (pol.top_k || pol.top_p < 1.0);
    uint32_t* hist = ps_hist();
    if (values) {
      for (int i = threadIdx.x; i < kPsBins / 4; i += kPsThreads)
        reinterpret_cast<uint4*>(hist)[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
    }
    uint32_t top = 0, small = 0, large = 0, low = 0;
    double small_mass = 0.0;  // relative to a value of 0
    row.view.stream(row.lane, [&](uint32_t id, const auto& r) {
      using View = RowView<DT>;
      const uint32_t peak = View::peak_of(r);
      if (row.view.peaks) row.view.peaks[(id - row.view.begin) >> 3] = (uint16_t)(peak >> 16);
      top = max(top, peak);
      if (OP == kOpProbs) clear_probs(p.out_probs + group * p.out_stride, id, row.view.end);
      if (DT == kBF16 && values) {
        uint32_t odd = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (r.bits >> j & 1u)
            if (!PolicyRow<DT>::count_bin(hist, View::bits_of(r, j))) odd |= 1u << j;
        if (odd) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (odd >> j & 1u) {
              const float v = View::value_of(r, j);
              if (fabsf(v) < 1.0f) {
                ++small;
                small_mass += exp((double)v * c.inv_t);
              } else if (v > 0.0f) {
                ++large;
              } else {
                ++low;
              }
            }
        }
      }
    });
    PsBox sum = row.reduce(small_mass, small, top, large, low);
    top = sum.top;
    if (top == 0u) status = kStatusEmptyMask;
    if (top == kOrd32NaN) status = kStatusNanInSupport;
    if (top == kOrd32NegInf) status = kStatusAllNegInf;
    if (!status) {
      const float best = PolicyRow<DT>::code_value(top);
      c.flat = !(pol.temperature > 0.0) || best == INFINITY;
      c.top = best;
      sum.mass = sum.count ? sum.mass * exp(-c.top * c.inv_t) : 0.0;
      // a small mass that left the range of doubles on the way
      const bool lost = !(sum.mass >= 0.0 && sum.mass < INFINITY);
      if (!(values && !lost && row.find_cut_by_values(c, pol, sum, ps_table(p.k)))) {
        __syncthreads();  // the scans' results have been read
        row.find_cut(c, pol, top);
      }
      c.bound_by_min_p();
    }
  }

  if (status) {
    if (OP == kOpProbs) {
      if (!ok)  // the other rows were cleared as they were read
        for (uint32_t i = row.view.begin + row.lane; i < row.view.end; i += 32u)
          p.out_probs[group * p.out_stride + i] = 0.0f;
      if (first) p.out_status[item] = status;
    } else if (first) {
      if (OP == kOpDraw) {
        p.out_idx[item] = -1;
        p.out_status[item] = status;
      } else {
        p.results[item] = make_int4(kDecided, -1, (int)status, 0);
      }
    }
    return;
  }

  // the kept mass and the ties at the cut, by warps; for a drafted row also the ties before it
  uint32_t draft = 0;
  bool drafted = false;
  if (OP == kOpSpec && sub < len) {
    const int32_t d = p.drafts[group * p.draft_stride + sub];
    drafted = d >= 0 && d < (int64_t)p.vocab;
    draft = drafted ? (uint32_t)d : 0u;
  }
  double mass = 0.0;
  uint32_t ties = 0, before = 0;
  row.view.each(row.lane, c.least(), [&](uint32_t id, const auto& r) {
    using View = RowView<DT>;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!(r.bits >> j & 1u)) continue;
      const uint32_t code = ord32(View::value_of(r, j));
      if (code == c.cut) {
        ++ties;
        if (OP == kOpSpec && id + j < draft) ++before;
      } else if (code > c.cut) {
        const double w = row.weight(c, View::bits_of(r, j));
        if (w >= c.min_p) mass += w;
      }
    }
  });
  mass = warp_sum(mass);
  ties = __reduce_add_sync(~0u, ties);
  before = __reduce_add_sync(~0u, before);
  const double w_tie = c.take ? c.weight(PolicyRow<DT>::code_value(c.cut)) : 0.0;
  auto scan = row.scan_entries(0, mass, ties, before, c.take, w_tie);
  const double total = scan.total;

  if (OP == kOpProbs) {
    float* out = p.out_probs + group * p.out_stride;
    const double inv = 1.0 / total;
    row.each_kept(c, scan.ties_before, [&](uint32_t id, double* w) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (w[j] > 0.0) out[id + j] = (float)(w[j] * inv);
    });
    if (first) p.out_status[item] = 0u;
    return;
  }

  bool residual = false;
  const float* q = nullptr;
  if (OP == kOpSpec && sub < len) {
    double p_d = 0.0, q_d = drafted ? 1.0 : 0.0;
    if (p.draft_probs) q = p.draft_probs + group * p.dp_group_stride + sub * p.dp_row_stride;
    if (drafted) {
      if (q) q_d = fmax((double)q[draft], 0.0);
      const bool valid = !row.view.mask || (row.view.mask[draft >> 3] >> (draft & 7u) & 1u);
      const float v = Elem<DT>::to_f32(row.view.row, draft);
      const uint32_t code = ord32(v);
      if (valid && (code > c.cut || (code == c.cut && scan.draft_before < c.take))) {
        const double w = c.weight(v);
        if (w >= c.min_p) p_d = w / total;
      }
    }
    if (drafted && u_accept * q_d < p_d) {
      if (first) p.results[item] = make_int4(kAccepted, -1, 0, 0);
      return;
    }
    residual = true;
  }

  // what remains of p where the draft's probability is taken off
  const double inv = 1.0 / total;
  auto rest = [&](uint32_t id, double* w) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (w[j] > 0.0) {
        const double qj = q ? fmax((double)q[id + j], 0.0)
                            : (drafted && id + j == draft ? 1.0 : 0.0);
        w[j] = fmax(w[j] * inv - qj, 0.0);
      }
  };
  if (OP == kOpSpec && residual) {
    double sum = 0.0;
    row.each_kept(c, scan.ties_before, [&](uint32_t id, double* w) {
      rest(id, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += w[j];
    });
    sum = warp_sum(sum);
    const auto left = row.scan_entries(1, sum, ties, 0u, 0u, 0.0);
    residual = left.total > 0.0;  // else the draft covers p everywhere: draw from p itself
    if (residual) scan.total = left.total, scan.mass_before = left.mass_before;
  }
  const double goal = u * scan.total;
  const int owner = residual ? row.find_owner(1, 0u, 0.0, goal)
                             : row.find_owner(0, c.take, w_tie, goal);
  if (owner == row.entry) {
    const int id = OP == kOpSpec && residual
                       ? row.pick(c, scan.ties_before, scan.mass_before, goal, rest)
                       : row.pick(c, scan.ties_before, scan.mass_before, goal,
                                  [](uint32_t, double*) {});
    if (row.lane == 0) {
      if (OP == kOpDraw) {
        p.out_idx[item] = id;
        p.out_status[item] = 0u;
      } else {
        p.results[item] = make_int4(kDecided, id, 0, 0);
      }
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
