// pck_lora_add: out = y + s_a B_a (A_a x) for rows that each name their adapter a.
//
// One CTA per row: a warp per rank takes the product of A's row with x, then a thread per output
// takes B's row with the rank-long intermediate, which stays in binary32.
#include "serving_common.cuh"

namespace pck {
namespace {

constexpr int kLoraMaxRank = 256;
constexpr int kLoraThreads = 256;

struct LoraArgs {
  const void* x;
  int64_t x_stride;
  const float* y;
  int64_t y_stride;
  const void* A;
  const void* B;
  const int32_t* adapters;
  const float* scales;
  const int32_t* ranks;
  float* out;
  int64_t out_stride;
  int64_t n, m;
  int32_t count, rank;
};

template <typename T>
__global__ void __launch_bounds__(kLoraThreads) lora_kernel(const LoraArgs a) {
  __shared__ float h[kLoraMaxRank];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
  int adapter = a.adapters[row];
  if (adapter >= a.count) {
    if (threadIdx.x == 0) report(kDevIndex);
    adapter = -1;
  }
  int rank = 0;
  if (adapter >= 0) {
    rank = a.ranks ? min(max(a.ranks[adapter], 0), a.rank) : a.rank;
    const float scale = a.scales ? a.scales[adapter] : 1.0f;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    for (int r = warp; r < rank; r += kLoraThreads / kWarp) {
      const T* w = static_cast<const T*>(a.A) + (static_cast<int64_t>(adapter) * a.rank + r) * a.n;
      float sum = 0.0f;
      for (int64_t j = lane; j < a.n; j += kWarp) sum = fmaf(to_float(w[j]), to_float(x[j]), sum);
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
      if (lane == 0) h[r] = sum * scale;
    }
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < a.m; i += kLoraThreads) {
    const T* w = static_cast<const T*>(a.B) + (static_cast<int64_t>(max(adapter, 0)) * a.m + i) * a.rank;
    float sum = 0.0f;
    for (int r = 0; r < rank; ++r) sum = fmaf(to_float(w[r]), h[r], sum);
    a.out[row * a.out_stride + i] = a.y[row * a.y_stride + i] + sum;
  }
}

}  // namespace

PCK_STATUS_READER(lora_status)

}  // namespace pck

extern "C" int pck_lora_add(const void* x, int dtype, int64_t tokens, int64_t n, int64_t x_stride, const float* y,
                            int64_t m, int64_t y_stride, const void* A, const void* B, int64_t count, int64_t rank,
                            const int32_t* adapters, const float* scales, const int32_t* ranks, float* out,
                            int64_t out_stride, void* stream) {
  using namespace pck;
  if (dtype != PCK_LOGITS_BF16 && dtype != PCK_LOGITS_F16) return report_error(PCK_ERR_ARGUMENT, "adapters: x must be bfloat16 or float16");
  if (tokens < 0 || tokens > 0x7fffffffLL || n < 1 || m < 0 || x_stride < n || y_stride < m || out_stride < m) {
    return report_error(PCK_ERR_ARGUMENT, "adapters: need tokens >= 0, n >= 1, m >= 0 and strides of whole rows");
  }
  if (count < 0 || count > 0x7fffffffLL) return report_error(PCK_ERR_ARGUMENT, "adapters: bad number of adapters");
  if (rank < 1 || rank > kLoraMaxRank) return report_error(PCK_ERR_ARGUMENT, "adapters: rank must be in [1, 256]");
  if (tokens == 0 || m == 0) return PCK_OK;
  if (!x || !y || !adapters || !out || (count > 0 && (!A || !B))) {
    return report_error(PCK_ERR_ARGUMENT, "adapters: NULL x, y, A, B, adapters or out");
  }
  LoraArgs a{x, x_stride, y, y_stride, A, B, adapters, scales, ranks, out, out_stride, n, m,
             static_cast<int32_t>(count), static_cast<int32_t>(rank)};
  const unsigned grid = static_cast<unsigned>(tokens);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PCK_LOGITS_BF16) {
    lora_kernel<__nv_bfloat16><<<grid, kLoraThreads, 0, s>>>(a);
  } else {
    lora_kernel<__half><<<grid, kLoraThreads, 0, s>>>(a);
  }
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? PCK_OK : report_cuda("adapter kernel", err);
}
