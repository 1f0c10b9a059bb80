// pck_process_logits: penalties for repeated tokens, biases and grammar masks on a batch of logits,
// written as the binary32 logits that the sampler and the membership check take.
//
// Bound by memory: the logits are read once and written once. A CTA takes a slice of a row's vocabulary
// and asks for all of it, in registers, before it looks at the history. What the history holds of the
// slice is counted in shared memory, a word for each token (integer atomics: the counts do not depend on
// their order). Up to eight CTAs of a row form a cluster that reads the history once, each its share, and
// counts into one another's shared memory: without it every slice would read the whole history, half
// as much again as the logits for 64 rows of 128,256 with 3,000 tokens each. A second word for each
// token holds the last bias that names it. What decides the time beside the bytes is the chain of
// dependent reads (lengths, ids, counts), so each is asked for as early as it can be. Each step is a
// separate binary32 operation, so the result is the formula's wherever it is evaluated.
#include <cooperative_groups.h>

#include "serving_common.cuh"

namespace pck {
namespace {

namespace cg = cooperative_groups;

constexpr int kLogitsThreads = 512;
constexpr int kLogitsWarps = kLogitsThreads / kWarp;
constexpr uint32_t kInPrompt = 0x80000000u;

struct LogitsArgs {
  const void* logits;
  int64_t row_stride;
  int64_t vocab;
  const int64_t* tokens;
  int64_t token_stride;
  int64_t max_tokens;
  const int32_t* prompt_lengths;
  const int32_t* lengths;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const int32_t* bias_starts;
  const int64_t* bias_ids;
  const float* bias_values;
  int64_t biases;
  const int32_t* mask;
  int64_t mask_stride;
  float* out;
  int64_t out_stride;
  int32_t clusters;  // of a row
};

// kPer: tokens of a thread; token j of thread t is j * kLogitsThreads + t of the slice, so a warp meets
// one word of the mask.
template <typename T, int kPer>
__global__ void __launch_bounds__(kLogitsThreads, 3) logits_kernel(const __grid_constant__ LogitsArgs a) {
  constexpr int kSlice = kPer * kLogitsThreads;
  extern __shared__ uint32_t counts[];     // how often the token was put out; kInPrompt: in the prompt
  uint32_t* const bias = counts + kSlice;  // 1 + the last of the row's biases that names the token
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const int64_t row = blockIdx.x / ctas / a.clusters;
  const int64_t first = static_cast<int64_t>(blockIdx.x / ctas % a.clusters) * ctas * kSlice;  // of the cluster
  const int64_t base = first + static_cast<int64_t>(cta) * kSlice;
  const int size = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(kSlice), a.vocab - base)));
  wait_for_producers();
  allow_dependents();
  int64_t length = 0, prompt = 0, bias0 = 0, bias1 = 0;
  if (a.tokens) {
    length = min(static_cast<int64_t>(a.lengths[row]), a.max_tokens);
    if (a.prompt_lengths) prompt = a.prompt_lengths[row];
  }
  if (a.bias_starts) {
    bias0 = max(static_cast<int64_t>(a.bias_starts[row]), int64_t{0});
    bias1 = min(static_cast<int64_t>(a.bias_starts[row + 1]), a.biases);
  }
  const T* in = static_cast<const T*>(a.logits) + row * a.row_stride + base;
  T raw[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (j * kLogitsThreads + tid < size) raw[j] = in[j * kLogitsThreads + tid];
  }
  uint32_t words = 0xffffffffu;  // lane j: the mask of the warp's j-th 32 tokens
  if (a.mask && lane < kPer && (lane * kLogitsWarps + warp) * kWarp < size) {
    words = static_cast<uint32_t>(a.mask[row * a.mask_stride + base / 32 + lane * kLogitsWarps + warp]);
  }
  const float rep = a.repetition ? a.repetition[row] : 1.0f;
  const float freq = a.frequency ? a.frequency[row] : 0.0f;
  const float pres = a.presence ? a.presence[row] : 0.0f;
  const bool marked = a.tokens || a.bias_starts;
  if (marked) {
#pragma unroll
    for (int j = 0; j < 2 * kPer / 4; ++j) {
      reinterpret_cast<uint4*>(counts)[j * kLogitsThreads + tid] = make_uint4(0, 0, 0, 0);
    }
    cluster.barrier_arrive();
    const int64_t* t = a.tokens + row * a.token_stride;
    constexpr int kAhead = 4;
    const int64_t step = static_cast<int64_t>(ctas) * kLogitsThreads;
    const int64_t start = static_cast<int64_t>(cta) * kLogitsThreads + tid;
    int64_t id[kAhead];
    auto load = [&](int64_t i) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) id[u] = i + u * step < length ? t[i + u * step] : -1;
    };
    load(start);
    int64_t bias_id = bias0 + tid < bias1 ? a.bias_ids[bias0 + tid] : -1;
    cluster.barrier_wait();  // every CTA's words are zero
    for (int64_t i = start; i < length; i += kAhead * step) {
      if (i > start) load(i);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t at = id[u] - first;
        if (id[u] < 0 || at < 0 || at >= static_cast<int64_t>(ctas) * kSlice) continue;  // (past the vocabulary: no one reads it)
        uint32_t* count = cluster.map_shared_rank(counts, static_cast<int>(at / kSlice)) + at % kSlice;
        if (i + u * step < prompt) {
          atomicOr(count, kInPrompt);
        } else {
          atomicAdd(count, 1u);
        }
      }
    }
    for (int64_t i = bias0 + tid; i < bias1; i += kLogitsThreads) {
      if (i > bias0 + tid) bias_id = a.bias_ids[i];
      const int64_t at = bias_id - base;
      if (bias_id >= 0 && at >= 0 && at < size) atomicMax(&bias[at], static_cast<uint32_t>(i - bias0 + 1));
    }
    cluster.sync();
  }
  float* out = a.out + row * a.out_stride + base;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = j * kLogitsThreads + tid;
    const uint32_t word = __shfl_sync(kFullMask, words, j);
    if (i >= size) continue;
    float l = to_float(raw[j]);
    if (marked) {
      const uint32_t c = counts[i], entry = bias[i];
      if (c) {
        l = l > 0.0f ? l / rep : l * rep;
        const uint32_t said = c & ~kInPrompt;
        if (said) l = l - freq * static_cast<float>(said) - pres;
      }
      if (entry) l += a.bias_values[bias0 + entry - 1];
    }
    out[i] = word >> lane & 1u ? l : -INFINITY;
  }
}

template <typename T, int kPer>
cudaError_t launch_slices(LogitsArgs a, int64_t rows, cudaStream_t stream) {
  const int64_t slices = (a.vocab + kPer * kLogitsThreads - 1) / (kPer * kLogitsThreads);
  // The fewest clusters of up to eight, all of the same size.
  a.clusters = static_cast<int32_t>((slices + 7) / 8);
  const int64_t ctas = (slices + a.clusters - 1) / a.clusters;
  const int64_t blocks = rows * a.clusters * ctas;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  constexpr int kSmem = 2 * kPer * kLogitsThreads * 4;
  static bool configured[64] = {};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t err =
        cudaFuncSetAttribute(logits_kernel<T, kPer>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (err != cudaSuccess) return err;
    configured[dev] = true;
  }
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(blocks));
  config.blockDim = dim3(kLogitsThreads);
  config.dynamicSmemBytes = kSmem;
  config.stream = stream;
  config.attrs = attr;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, logits_kernel<T, kPer>, a);
}

// The longest slices that still give every SM two CTAs: 8192, 4096 or 1024 tokens.
template <typename T>
cudaError_t launch_logits(const LogitsArgs& a, int64_t rows, cudaStream_t stream) {
  if (rows * a.vocab >= int64_t{2 * 148} * 16 * kLogitsThreads) return launch_slices<T, 16>(a, rows, stream);
  if (rows * a.vocab >= int64_t{2 * 148} * 8 * kLogitsThreads) return launch_slices<T, 8>(a, rows, stream);
  return launch_slices<T, 2>(a, rows, stream);
}

}  // namespace
}  // namespace pck

extern "C" int pck_process_logits(const pck_logits_desc* desc, void* stream) {
  using namespace pck;
  if (!desc) return report_error(PCK_ERR_ARGUMENT, "logits: NULL descriptor");
  const auto& [logits, dtype, rows, vocab, row_stride, tokens, token_stride, max_tokens, prompt_lengths, lengths, repetition, frequency, presence, bias_starts, bias_ids, bias_values, biases, mask, mask_stride, out, out_stride] = *desc;
  if (dtype != PCK_LOGITS_F32 && dtype != PCK_LOGITS_BF16 && dtype != PCK_LOGITS_F16) {
    return report_error(PCK_ERR_ARGUMENT, "logits: unknown dtype");
  }
  if (rows < 0 || vocab < 1 || vocab > 0x7fffffffLL || row_stride < vocab || out_stride < vocab) {
    return report_error(PCK_ERR_ARGUMENT, "logits: need rows >= 0, vocab in [1, 2^31) and strides of whole rows");
  }
  if (tokens && (!lengths || max_tokens < 0 || token_stride < max_tokens)) {
    return report_error(PCK_ERR_ARGUMENT, "logits: a history needs lengths and a stride of whole rows");
  }
  if (!tokens && (repetition || frequency || presence)) return report_error(PCK_ERR_ARGUMENT, "logits: penalties need a history");
  if (bias_starts && (biases < 0 || biases > 0x7fffffffLL || (biases > 0 && (!bias_ids || !bias_values)))) {
    return report_error(PCK_ERR_ARGUMENT, "logits: biases need ids and values");
  }
  if (mask && mask_stride < (vocab + 31) / 32) return report_error(PCK_ERR_ARGUMENT, "logits: a mask row has ceil(vocab / 32) words");
  if (rows == 0) return PCK_OK;
  if (!logits || !out) return report_error(PCK_ERR_ARGUMENT, "logits: NULL logits or out");
  LogitsArgs a{logits, row_stride, vocab, tokens, token_stride, max_tokens, prompt_lengths, lengths, repetition, frequency,
               presence, bias_starts, bias_ids, bias_values, biases, mask, mask_stride, out, out_stride, 0};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == PCK_LOGITS_F32    ? launch_logits<float>(a, rows, s)
                          : dtype == PCK_LOGITS_BF16 ? launch_logits<__nv_bfloat16>(a, rows, s)
                                                     : launch_logits<__half>(a, rows, s);
  return err == cudaSuccess ? PCK_OK : report_cuda("logits kernel", err);
}
