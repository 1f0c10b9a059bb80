// pck_process_logits: penalties for repeated tokens, biases and grammar masks on a batch of logits,
// written as the binary32 logits that the sampler and the membership check take.
//
// A CTA takes a slice of the vocabulary of one row. It reads the row's whole history and counts the
// tokens of its slice in shared memory (integer atomics: the counts do not depend on their order),
// notes for each token the last bias that names it, and then passes once over the slice. Each step
// is a separate binary32 operation, so the result is the formula's wherever it is evaluated.
// Bound by memory: the logits are read once and written once.
#include "serving_common.cuh"

namespace pck {
namespace {

constexpr int kLogitsThreads = 256;
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
  int32_t slice;   // tokens of a CTA's slice, a multiple of 32
  int32_t slices;
};

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) logits_kernel(const LogitsArgs a) {
  extern __shared__ uint32_t shared[];
  uint32_t* counts = shared;             // how often the token was put out; kInPrompt: in the prompt
  uint32_t* bias = shared + a.slice;     // 1 + the last bias entry that names the token
  const int64_t row = blockIdx.x / a.slices;
  const int64_t base = static_cast<int64_t>(blockIdx.x % a.slices) * a.slice;
  const int size = static_cast<int>(min(static_cast<int64_t>(a.slice), a.vocab - base));
  for (int i = threadIdx.x; i < size; i += kLogitsThreads) counts[i] = bias[i] = 0;
  __syncthreads();
  if (a.tokens) {
    const int64_t* t = a.tokens + row * a.token_stride;
    const int64_t length = min(max(static_cast<int64_t>(a.lengths[row]), int64_t{0}), a.max_tokens);
    const int64_t prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    for (int64_t i = threadIdx.x; i < length; i += kLogitsThreads) {
      const int64_t id = t[i] - base;
      if (id < 0 || id >= size) continue;
      if (i < prompt) {
        atomicOr(&counts[id], kInPrompt);
      } else {
        atomicAdd(&counts[id], 1u);
      }
    }
  }
  int64_t bias0 = 0, bias1 = 0;
  if (a.bias_starts) {
    bias0 = max(static_cast<int64_t>(a.bias_starts[row]), int64_t{0});
    bias1 = min(static_cast<int64_t>(a.bias_starts[row + 1]), a.biases);
    for (int64_t i = bias0 + threadIdx.x; i < bias1; i += kLogitsThreads) {
      const int64_t id = a.bias_ids[i] - base;
      if (id >= 0 && id < size) atomicMax(&bias[id], static_cast<uint32_t>(i - bias0 + 1));
    }
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[row] : 1.0f;
  const float freq = a.frequency ? a.frequency[row] : 0.0f;
  const float pres = a.presence ? a.presence[row] : 0.0f;
  const T* in = static_cast<const T*>(a.logits) + row * a.row_stride + base;
  float* out = a.out + row * a.out_stride + base;
  const int32_t* mask = a.mask ? a.mask + row * a.mask_stride + base / 32 : nullptr;
  for (int i = threadIdx.x; i < size; i += kLogitsThreads) {
    float l = to_float(in[i]);
    const uint32_t c = counts[i];
    if (c) {
      l = l > 0.0f ? l / rep : l * rep;
      const uint32_t said = c & ~kInPrompt;
      if (said) l = l - freq * static_cast<float>(said) - pres;
    }
    if (bias[i]) l += a.bias_values[bias0 + bias[i] - 1];
    if (mask && !(static_cast<uint32_t>(mask[i / 32]) >> (i % 32) & 1u)) l = -INFINITY;
    out[i] = l;
  }
}

template <typename T>
cudaError_t launch_logits(LogitsArgs a, int64_t rows, cudaStream_t stream) {
  a.slice = 4096;
  a.slices = static_cast<int32_t>((a.vocab + a.slice - 1) / a.slice);
  const int64_t blocks = rows * a.slices;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  logits_kernel<T><<<static_cast<unsigned>(blocks), kLogitsThreads, 2 * sizeof(uint32_t) * a.slice, stream>>>(a);
  return cudaGetLastError();
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
               presence, bias_starts, bias_ids, bias_values, biases, mask, mask_stride, out, out_stride, 0, 0};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == PCK_LOGITS_F32    ? launch_logits<float>(a, rows, s)
                          : dtype == PCK_LOGITS_BF16 ? launch_logits<__nv_bfloat16>(a, rows, s)
                                                     : launch_logits<__half>(a, rows, s);
  return err == cudaSuccess ? PCK_OK : report_cuda("logits kernel", err);
}
