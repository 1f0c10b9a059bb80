// pck_process_logits: penalties for repeated tokens, biases and grammar masks on a batch of logits,
// written as the binary32 logits that the sampler and the membership check take.
//
// The floor is memory: the logits are read once and written once (64 rows of 128,256, binary32, histories to
// 9,000 tokens: 25 us against 10.5). Of the marks' CTAs 296 run at once, for their shared memory, so the second
// turn of 512 counts after the pass. Two kernels, since few
// tokens of a row are in its history or its biases and what they need is a chain of dependent reads:
//   - the pass writes every logit, or -inf by the mask, at the memory's rate, and looks at nothing else;
//   - the marks, a programmatic dependent that may count beside the pass's end: a CTA takes 16,384 tokens of
//     a row's vocabulary, reads the row's history, and keeps a word of counts for each of its tokens in
//     shared memory (integer atomics: their order does not matter) and a list of those that it met. Then
//     it waits for the pass and computes the listed tokens' logits; biases are added after that, the last
//     entry of a token found by the largest entry number in the token's word.
//   (One kernel that did both held its registers and its memory requests through that chain: 31 us for 64
//   rows of 128,256, where the bytes take 10. A hash table of a row's tokens, a CTA a row, took as long:
//   text repeats its words, and their counts wait for one another.)
// In place the marks come first and the pass, which then only writes the mask's -inf, second. Each step is
// a separate binary32 operation, so the result is the formula's wherever it is evaluated.
#include "serving_common.cuh"

namespace pck {
namespace {

constexpr int kPassThreads = 256;
constexpr int kPassPer = 16;                          // tokens of a thread
constexpr int kPassChunk = kPassThreads * kPassPer;   // tokens of a CTA's step
constexpr int kPassCtas = 32;                         // of an SM at most; then a CTA takes several steps
constexpr int kMarkThreads = 512;
constexpr int kMarkSlice = 16384;                     // tokens of a marking CTA
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
  int64_t rows;
  int32_t in_place;
};

// Every logit as binary32, or -inf where the mask says so (in place: only those).
template <typename T>
__global__ void __launch_bounds__(kPassThreads) pass_kernel(const __grid_constant__ LogitsArgs a) {
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  wait_for_producers();
  allow_dependents();
  const int64_t chunks = (a.vocab + kPassChunk - 1) / kPassChunk;
  for (int64_t c = blockIdx.x; c < chunks * a.rows; c += gridDim.x) {
    const int64_t row = c / chunks, base = c % chunks * kPassChunk;
    const int size = static_cast<int>(min(static_cast<int64_t>(kPassChunk), a.vocab - base));
    // Token j of thread t is j * kPassThreads + t, so a warp meets one word of the mask, which lane j holds.
    const T* in = static_cast<const T*>(a.logits) + row * a.row_stride + base;
    T raw[kPassPer];
    if (!a.in_place) {
#pragma unroll
      for (int j = 0; j < kPassPer; ++j) {
        if (j * kPassThreads + tid < size) raw[j] = in[j * kPassThreads + tid];
      }
    }
    uint32_t words = 0xffffffffu;
    const int first = (lane * (kPassThreads / kWarp) + warp) * kWarp;
    if (a.mask && lane < kPassPer && first < size) {
      words = static_cast<uint32_t>(a.mask[row * a.mask_stride + (base + first) / 32]);
    }
    float* out = a.out + row * a.out_stride + base;
#pragma unroll
    for (int j = 0; j < kPassPer; ++j) {
      const int i = j * kPassThreads + tid;
      const bool shown = __shfl_sync(kFullMask, words, j) >> lane & 1u;
      if (i < size && !(a.in_place && shown)) out[i] = shown ? to_float(raw[j]) : -INFINITY;
    }
  }
}

// The logits of the tokens in a row's history or biases.
template <typename T>
__global__ void __launch_bounds__(kMarkThreads) mark_kernel(const __grid_constant__ LogitsArgs a) {
  extern __shared__ __align__(16) uint32_t counts[];  // times put out, kInPrompt
  uint16_t* const listed = reinterpret_cast<uint16_t*>(counts + kMarkSlice);  // tokens with a count
  __shared__ uint32_t met;
  const int tid = threadIdx.x;
  const int64_t slices = (a.vocab + kMarkSlice - 1) / kMarkSlice;
  const int64_t row = blockIdx.x / slices, base = blockIdx.x % slices * kMarkSlice;
  const int64_t size = min(static_cast<int64_t>(kMarkSlice), a.vocab - base);
  if (a.in_place) wait_for_producers();  // else this call's pass comes before, and it has waited
  allow_dependents();
  int64_t length = 0, prompt = 0, bias0 = 0, bias1 = 0;
  float rep = 1.0f, freq = 0.0f, pres = 0.0f;
  if (a.tokens) {
    length = min(static_cast<int64_t>(a.lengths[row]), a.max_tokens);
    if (a.prompt_lengths) prompt = a.prompt_lengths[row];
    if (a.repetition) rep = a.repetition[row];
    if (a.frequency) freq = a.frequency[row];
    if (a.presence) pres = a.presence[row];
  }
  if (a.bias_starts) {
    bias0 = max(static_cast<int64_t>(a.bias_starts[row]), int64_t{0});
    bias1 = min(static_cast<int64_t>(a.bias_starts[row + 1]), a.biases);
  }
  if (a.tokens) {
#pragma unroll
    for (int j = 0; j < kMarkSlice / 4 / kMarkThreads; ++j) {
      reinterpret_cast<uint4*>(counts)[j * kMarkThreads + tid] = make_uint4(0, 0, 0, 0);
    }
  }
  if (tid == 0) met = 0;
  constexpr int kAhead = 8;
  const int64_t* const tokens = a.tokens + row * a.token_stride;
  int64_t id[kAhead];
  auto load = [&](int64_t i) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) id[u] = i + u * kMarkThreads < length ? tokens[i + u * kMarkThreads] : -1;
  };
  load(tid);
  int64_t bias_id = bias0 + tid < bias1 ? a.bias_ids[bias0 + tid] : -1;
  __syncthreads();
  for (int64_t i = tid; i < length; i += kAhead * kMarkThreads) {
    if (i > tid) load(i);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t at = id[u] - base;
      if (id[u] < 0 || at < 0 || at >= size) continue;
      const uint32_t before = i + u * kMarkThreads < prompt ? atomicOr(&counts[at], kInPrompt) : atomicAdd(&counts[at], 1u);
      if (before == 0) listed[atomicAdd(&met, 1u)] = static_cast<uint16_t>(at);
    }
  }
  __syncthreads();
  if (!a.in_place) wait_for_producers();  // the pass has written its logits
  const T* in = static_cast<const T*>(a.logits) + row * a.row_stride + base;
  float* out = a.out + row * a.out_stride + base;
  auto hidden = [&](int at) {
    return a.mask && !(static_cast<uint32_t>(a.mask[row * a.mask_stride + (base + at) / 32]) >> (at % 32) & 1u);
  };
  const int count = static_cast<int>(met);
  for (int k = tid; k < count; k += kMarkThreads) {
    const int at = listed[k];
    float l = to_float(in[at]);
    if (hidden(at)) continue;
    l = l > 0.0f ? l / rep : l * rep;
    const uint32_t said = counts[at] & ~kInPrompt;
    if (said) l = l - freq * static_cast<float>(said) - pres;
    out[at] = l;
  }
  if (bias0 >= bias1) return;
  // Biases: the last entry that names a token counts.
  auto each = [&](auto&& f) {
    for (int64_t i = bias0 + tid; i < bias1; i += kMarkThreads) {
      const int64_t b = i == bias0 + tid ? bias_id : a.bias_ids[i];
      if (b >= base && b - base < size) f(i, static_cast<int>(b - base));
    }
  };
  __syncthreads();
  each([&](int64_t, int at) { counts[at] = 0; });
  __syncthreads();
  each([&](int64_t i, int at) { atomicMax(&counts[at], static_cast<uint32_t>(i - bias0 + 1)); });
  __syncthreads();
  each([&](int64_t i, int at) {
    if (counts[at] == static_cast<uint32_t>(i - bias0 + 1) && !hidden(at)) out[at] += a.bias_values[i];
  });
}

template <typename T>
cudaError_t launch_logits(const LogitsArgs& a, cudaStream_t stream) {
  constexpr int kSmem = kMarkSlice * 6;
  static bool configured[64] = {};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t err = cudaFuncSetAttribute(mark_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (err != cudaSuccess) return err;
    configured[dev] = true;
  }
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  auto pass = [&] {
    if (a.in_place && !a.mask) return cudaSuccess;
    const int64_t chunks = (a.vocab + kPassChunk - 1) / kPassChunk * a.rows;
    config.gridDim = dim3(static_cast<unsigned>(chunks < 148 * kPassCtas ? chunks : 148 * kPassCtas));
    config.blockDim = dim3(kPassThreads);
    config.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&config, pass_kernel<T>, a);
  };
  auto marks = [&] {
    if (!a.tokens && !a.bias_starts) return cudaSuccess;
    config.blockDim = dim3(kMarkThreads);
    const int64_t blocks = (a.vocab + kMarkSlice - 1) / kMarkSlice * a.rows;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    config.gridDim = dim3(static_cast<unsigned>(blocks));
    config.dynamicSmemBytes = kSmem;
    return cudaLaunchKernelEx(&config, mark_kernel<T>, a);
  };
  const cudaError_t err = a.in_place ? marks() : pass();
  return err != cudaSuccess ? err : a.in_place ? pass() : marks();
}

}  // namespace
}  // namespace pck

extern "C" int pck_process_logits(const pck_logits_desc* desc, void* stream) {
  using namespace pck;
  if (!desc) return report_error(PCK_ERR_ARGUMENT, "logits: NULL descriptor");
  const auto& [logits, dtype, rows, vocab, row_stride, tokens, token_stride, max_tokens, prompt_lengths, lengths,
               repetition, frequency, presence, bias_starts, bias_ids, bias_values, biases, mask, mask_stride, out,
               out_stride] = *desc;
  if (dtype != PCK_LOGITS_F32 && dtype != PCK_LOGITS_BF16 && dtype != PCK_LOGITS_F16) {
    return report_error(PCK_ERR_ARGUMENT, "logits: unknown dtype");
  }
  if (rows < 0 || rows > 0x7fffffffLL || vocab < 1 || vocab > 0x7fffffffLL || !rows_apart(row_stride, vocab) || out_stride < vocab) {
    return report_error(PCK_ERR_ARGUMENT, "logits: need rows >= 0, vocab in [1, 2^31) and strides of whole rows");
  }
  if (tokens && (!lengths || max_tokens < 0 || !rows_apart(token_stride, max_tokens))) {
    return report_error(PCK_ERR_ARGUMENT, "logits: a history needs lengths and a stride of whole rows");
  }
  if (!tokens && (repetition || frequency || presence)) return report_error(PCK_ERR_ARGUMENT, "logits: penalties need a history");
  if (bias_starts && (biases < 0 || biases > 0x7fffffffLL || (biases > 0 && (!bias_ids || !bias_values)))) {
    return report_error(PCK_ERR_ARGUMENT, "logits: biases need ids and values");
  }
  if (mask && !rows_apart(mask_stride, (vocab + 31) / 32)) return report_error(PCK_ERR_ARGUMENT, "logits: a mask of whole rows has ceil(vocab / 32) words");
  if (rows == 0) return PCK_OK;
  if (!logits || !out) return report_error(PCK_ERR_ARGUMENT, "logits: NULL logits or out");
  const int32_t in_place = out == logits && out_stride == row_stride && dtype == PCK_LOGITS_F32;
  const LogitsArgs a{logits, row_stride, vocab, tokens, token_stride, max_tokens, prompt_lengths, lengths, repetition, frequency,
                     presence, bias_starts, bias_ids, bias_values, biases, mask, mask_stride, out, out_stride, rows, in_place};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == PCK_LOGITS_F32    ? launch_logits<float>(a, s)
                          : dtype == PCK_LOGITS_BF16 ? launch_logits<__nv_bfloat16>(a, s)
                                                     : launch_logits<__half>(a, s);
  return err == cudaSuccess ? PCK_OK : report_cuda("logits kernel", err);
}
