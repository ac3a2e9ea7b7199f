// C entry points of sampling under per-row policies (include/onyx_b200.h): argument checks,
// the choice of the cluster size, launches.
#include "host_common.h"
#include "policy_sample.cuh"

#include "../../include/onyx_b200.h"

#include <algorithm>
#include <atomic>

namespace onyx {

// Streaming multiprocessors of the current device, asked once per device; 0 on an error.
static int device_sms(cudaError_t* err) {
  static std::atomic<int> known[64];
  int dev = 0;
  *err = cudaGetDevice(&dev);
  if (*err != cudaSuccess) return 0;
  if (dev >= 0 && dev < 64) {
    const int n = known[dev].load(std::memory_order_relaxed);
    if (n) return n;
  }
  int sms = 0;
  *err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (*err != cudaSuccess) return 0;
  if (dev >= 0 && dev < 64) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

// How a launch lays out its rows: CTAs per row, positions per warp, dynamic shared memory.
struct PolicyPlan {
  int k;
  int32_t warp_ids, peaks, keep, slots, lists;
  size_t smem;
};

// Shared memory spent on peaks at most; longer parts of rows do without.
constexpr size_t kPsMostPeaks = 64 * 1024;
// Dynamic shared memory with which two CTAs fit an SM (228 KB, 1 KB of it for each CTA, and the
// static part).
constexpr size_t kPsTwoFit = 228 * 1024 / 2 - 1024 - sizeof(PsShared) - 512;

static PolicyPlan plan_with(int k, int64_t vocab, int dtype, bool masked) {
  PolicyPlan pl = {};
  pl.k = k;
  const int64_t per = (int64_t)k * kPsWarps * kPsChunk;
  pl.warp_ids = (int32_t)((vocab + 7 + per - 1) / per * kPsChunk);  // up to 7 ids of offset
  pl.smem = kPsFixed;
  const size_t peaks = (size_t)pl.warp_ids / 8 * kPsWarps * sizeof(uint16_t);
  pl.peaks = peaks <= kPsMostPeaks;
  if (pl.peaks) pl.smem += peaks;
  const size_t lists = pl.peaks ? peaks : 0;
  const size_t slot = (size_t)ps_slot(dtype, masked);
  const size_t all = (size_t)pl.warp_ids / kPsChunk * kPsWarps * slot;
  pl.keep = pl.peaks && pl.smem + lists + all <= kPsTwoFit;
  pl.lists = (int32_t)pl.smem;
  pl.slots = (int32_t)(pl.smem + (pl.keep ? lists : 0));
  const size_t ring = std::max((size_t)kPsWarps * ps_depth(dtype) * slot, lists);
  pl.smem += pl.keep ? lists + all : ring;
  return pl;
}

// CTAs per row: a power of two, as many as the SMs hold two of, at least 2,048 ids each (one
// row of 32,000: 23 us with 4, 22 with 8); two at least for long rows, for a batch waits for
// its slowest rows, those whose kept ids are many (256 rows of 128,256 under mixed policies: 94
// us with 1, 85 with 2; 64 x 8 float16 rows: 273 and 185); and as many as it takes to have two
// CTAs on an SM.
static PolicyPlan make_plan(int64_t rows, int64_t vocab, int dtype, bool masked, int sms) {
  int k = vocab > 65536 ? 2 : 1;
  while (k < kPsMaxCluster && rows * k * 2 <= 2ll * sms && vocab >= 2ll * k * 2048) k *= 2;
  PolicyPlan pl = plan_with(k, vocab, dtype, masked);
  while (k < kPsMaxCluster && pl.smem > kPsTwoFit) {
    k *= 2;
    pl = plan_with(k, vocab, dtype, masked);
  }
  return pl;
}

template <int OP>
static const void* policy_fn(int dtype) {
  return dtype == kBF16 ? (const void*)policy_kernel<kBF16, OP>
         : dtype == kF16 ? (const void*)policy_kernel<kF16, OP>
                         : (const void*)policy_kernel<kF32, OP>;
}

// Lets kernel number `which` use the dynamic shared memory it may ask for, once per device.
static cudaError_t allow_shared(const void* fn, int which) {
  static std::atomic<uint16_t> done[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && (done[dev].load(std::memory_order_acquire) >> which & 1)) return e;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)(kPsFixed + 2 * kPsMostPeaks + kPsWarps * ps_depth(kF32) * ps_slot(kF32, true)));
  if (e == cudaSuccess && dev >= 0 && dev < 64)
    done[dev].fetch_or((uint16_t)(1u << which), std::memory_order_release);
  return e;
}

template <int OP>
static int launch_policy(int dtype, PolicyParams& p, int64_t rows, cudaStream_t stream) {
  cudaError_t e;
  const int sms = device_sms(&e);
  if (!sms) return finish_launch(e);
  const PolicyPlan pl = make_plan(rows, p.vocab, dtype, p.mask != nullptr, sms);
  p.k = pl.k;
  p.warp_ids = pl.warp_ids;
  p.peaks = pl.peaks;
  p.keep = pl.keep;
  p.slots = pl.slots;
  p.lists = pl.lists;
  if (rows * p.k > 0x7FFFFFFFll) return ONYX_ERR_INVALID_ARGUMENT;
  const void* fn = policy_fn<OP>(dtype);
  e = allow_shared(fn, OP * 3 + (dtype == kBF16 ? 0 : dtype == kF16 ? 1 : 2));
  if (e != cudaSuccess) return finish_launch(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * p.k), 1, 1);
  cfg.blockDim = dim3(kPsThreads, 1, 1);
  cfg.dynamicSmemBytes = pl.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.k > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)p.k;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  void* args[] = {&p};
  return finish_launch(cudaLaunchKernelExC(&cfg, fn, args));
}

static bool policy_dtype(int dt) { return dt == kF32 || dt == kF16 || dt == kBF16; }

constexpr int64_t kPsMostVocab = 1ll << 30;  // positions are counted in 32 bits

// The checks that the three entry points share; `rows` entries of the policies.
static int policy_checks(const void* logits, int dtype, int64_t rows, int64_t vocab,
                         const double* policies, int64_t policy_stride) {
  if (!policy_dtype(dtype)) return ONYX_ERR_UNSUPPORTED_DTYPE;
  if (rows < 0 || rows > 0x7FFFFFFFll || vocab <= 0 || vocab > kPsMostVocab)
    return ONYX_ERR_INVALID_ARGUMENT;
  if (rows > 0 && (!logits || !policies)) return ONYX_ERR_INVALID_ARGUMENT;
  if (policy_stride != 0 && policy_stride < 4) return ONYX_ERR_INVALID_ARGUMENT;
  return ONYX_OK;
}

static bool uniform_dtype(int dt) { return dt == kF32 || dt == kF64; }

}  // namespace onyx

using namespace onyx;

extern "C" {

int onyx_policy_sample(const void* logits, int dtype, int64_t rows, int64_t vocab,
                       int64_t row_stride, const uint32_t* mask, int64_t mask_stride,
                       const double* policies, int64_t policy_stride, const void* uniforms,
                       int uniform_dtype_code, int64_t uniform_stride, int32_t* out_idx,
                       uint32_t* out_status, void* stream) {
  const int rc = policy_checks(logits, dtype, rows, vocab, policies, policy_stride);
  if (rc != ONYX_OK) return rc;
  if (!uniform_dtype(uniform_dtype_code)) return ONYX_ERR_UNSUPPORTED_DTYPE;
  if (rows == 0) return ONYX_OK;
  if (!uniforms || !out_idx || !out_status) return ONYX_ERR_INVALID_ARGUMENT;
  if (rows > 1 && (row_stride < vocab || (mask && mask_stride < (vocab + 31) / 32) ||
                   uniform_stride < 1))
    return ONYX_ERR_INVALID_ARGUMENT;
  PolicyParams p = {};
  p.logits = logits;
  p.group_stride = row_stride;
  p.vocab = vocab;
  p.mask = mask;
  p.mask_group_stride = mask_stride;
  p.policies = policies;
  p.policy_stride = policy_stride;
  p.uniforms = uniforms;
  p.uniform_stride = uniform_stride;
  p.uniform_f64 = uniform_dtype_code == kF64;
  p.per_group = 1;
  p.out_idx = out_idx;
  p.out_status = out_status;
  return launch_policy<kOpDraw>(dtype, p, rows, (cudaStream_t)stream);
}

int onyx_policy_probs(const void* logits, int dtype, int64_t rows, int64_t vocab,
                      int64_t row_stride, const uint32_t* mask, int64_t mask_stride,
                      const double* policies, int64_t policy_stride, float* out,
                      int64_t out_stride, uint32_t* out_status, void* stream) {
  const int rc = policy_checks(logits, dtype, rows, vocab, policies, policy_stride);
  if (rc != ONYX_OK) return rc;
  if (rows == 0) return ONYX_OK;
  if (!out || !out_status) return ONYX_ERR_INVALID_ARGUMENT;
  if (rows > 1 && (row_stride < vocab || (mask && mask_stride < (vocab + 31) / 32) ||
                   out_stride < vocab))
    return ONYX_ERR_INVALID_ARGUMENT;
  PolicyParams p = {};
  p.logits = logits;
  p.group_stride = row_stride;
  p.vocab = vocab;
  p.mask = mask;
  p.mask_group_stride = mask_stride;
  p.policies = policies;
  p.policy_stride = policy_stride;
  p.per_group = 1;
  p.out_probs = out;
  p.out_stride = out_stride;
  p.out_status = out_status;
  return launch_policy<kOpProbs>(dtype, p, rows, (cudaStream_t)stream);
}

int onyx_policy_layout(int64_t rows, int64_t vocab, int dtype, int masked, int sms,
                       int32_t* layout) {
  if (!policy_dtype(dtype)) return ONYX_ERR_UNSUPPORTED_DTYPE;
  if (rows < 1 || rows > 0x7FFFFFFFll || vocab < 1 || vocab > kPsMostVocab || sms < 1 || !layout)
    return ONYX_ERR_INVALID_ARGUMENT;
  const PolicyPlan pl = make_plan(rows, vocab, dtype, masked != 0, sms);
  layout[0] = pl.k;
  layout[1] = pl.warp_ids;
  layout[2] = pl.peaks;
  layout[3] = pl.keep;
  layout[4] = (int32_t)pl.smem;
  return ONYX_OK;
}

size_t onyx_spec_sample_workspace_size(int64_t batch, int64_t gamma) {
  if (batch <= 0 || gamma < 1 || gamma > 255) return 0;
  return (size_t)batch * (size_t)(gamma + 1) * sizeof(int4);
}

int onyx_spec_sample(const void* logits, int dtype, int64_t batch, int64_t gamma, int64_t vocab,
                     int64_t batch_stride, int64_t row_stride, const uint32_t* masks,
                     int64_t mask_batch_stride, int64_t mask_row_stride, const int32_t* drafts,
                     int64_t draft_stride, const float* draft_probs, int64_t dp_batch_stride,
                     int64_t dp_row_stride, const int32_t* draft_lens, const double* policies,
                     int64_t policy_stride, const void* uniforms, int uniform_dtype_code,
                     int64_t uniform_stride, int32_t* accept_len, int32_t* token,
                     uint32_t* out_status, void* workspace, size_t workspace_bytes,
                     void* stream) {
  const int rc = policy_checks(logits, dtype, batch, vocab, policies, policy_stride);
  if (rc != ONYX_OK) return rc;
  if (!uniform_dtype(uniform_dtype_code)) return ONYX_ERR_UNSUPPORTED_DTYPE;
  if (gamma < 1 || gamma > 255 || batch > 0x7FFFFFFFll / 256) return ONYX_ERR_INVALID_ARGUMENT;
  if (batch == 0) return ONYX_OK;
  if (!drafts || !uniforms || !accept_len || !token || !out_status)
    return ONYX_ERR_INVALID_ARGUMENT;
  const int64_t words = (vocab + 31) / 32;
  if (row_stride < vocab || (masks && mask_row_stride < words) ||
      (draft_probs && gamma > 1 && dp_row_stride < vocab))
    return ONYX_ERR_INVALID_ARGUMENT;
  if (batch > 1 &&
      (batch_stride < 0 || (masks && mask_batch_stride < 0) || draft_stride < gamma ||
       (draft_probs && dp_batch_stride < 0) || uniform_stride < gamma + 1))
    return ONYX_ERR_INVALID_ARGUMENT;
  if (!workspace || ((uintptr_t)workspace & 15u) ||
      workspace_bytes < onyx_spec_sample_workspace_size(batch, gamma))
    return ONYX_ERR_WORKSPACE;
  PolicyParams p = {};
  p.logits = logits;
  p.group_stride = batch_stride;
  p.row_stride = row_stride;
  p.vocab = vocab;
  p.mask = masks;
  p.mask_group_stride = mask_batch_stride;
  p.mask_row_stride = mask_row_stride;
  p.policies = policies;
  p.policy_stride = policy_stride;
  p.uniforms = uniforms;
  p.uniform_stride = uniform_stride;
  p.uniform_f64 = uniform_dtype_code == kF64;
  p.per_group = (int32_t)gamma + 1;
  p.drafts = drafts;
  p.draft_stride = draft_stride;
  p.draft_probs = draft_probs;
  p.dp_group_stride = dp_batch_stride;
  p.dp_row_stride = dp_row_stride;
  p.draft_lens = draft_lens;
  p.results = static_cast<int4*>(workspace);
  // As many rows of every entry to a launch as the SMs take in two waves (two CTAs each, two to
  // a row): the rows behind a refusal need not be read, and the next launch sees it. (64 x 8
  // float16 rows: 165 us in one launch, 155 so. In launches of one wave the same, but 32 x 5
  // bfloat16 rows 108 us instead of 90.)
  cudaError_t e;
  const int sms = device_sms(&e);
  if (!sms) return finish_launch(e);
  const int64_t together = std::max<int64_t>(1, 2ll * sms / batch);
  for (int64_t from = 0; from <= gamma; from += together) {
    p.sub_from = (int32_t)from;
    p.sub_count = (int32_t)std::min<int64_t>(together, gamma + 1 - from);
    const int rc2 =
        launch_policy<kOpSpec>(dtype, p, batch * p.sub_count, (cudaStream_t)stream);
    if (rc2 != ONYX_OK) return rc2;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((batch + 127) / 128), 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return finish_launch(cudaLaunchKernelEx(&cfg, spec_join_kernel, (const int4*)p.results, batch,
                                          (int)gamma + 1, draft_lens, accept_len, token,
                                          out_status));
}

}  // extern "C"
