// pck_kv4_append: quantises keys and values to 4 bits and writes them to their slots of a cache.
//
// Per token, head and group of 64 channels: scale = bf16((max - min) / 15), zero = bf16(min), code =
// clamp(rint((x - zero) / scale), 0, 15), in binary32 with separate products and sums, so the codes
// are the same wherever the same formula is evaluated. The division by 15 is a product with the
// binary32 nearest 1/15 and the division by the scale one with its rounded reciprocal.
//
// One warp per (token, head, keys or values): a lane holds two neighbouring channels of each group,
// which is one byte of codes. Bound by memory: the inputs are read once, the codes written once.
#include "kv4_layout.cuh"
#include "serving_common.cuh"

namespace pck {
namespace {

struct AppendArgs {
  uint8_t* cache;
  const void* x[2];      // keys, values
  int64_t token_stride[2];
  int64_t head_stride[2];
  void* values[2];       // the values the codes stand for, or NULL
  const int64_t* slots;
  int64_t tokens;
  int64_t total_slots;
  int32_t heads;
  int32_t page_tiles;
};

template <typename T, int kDim>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x % kWarp;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x / kWarp) + threadIdx.x / kWarp;
  if (item >= a.tokens * a.heads * 2) return;
  const int side = static_cast<int>(item % 2);
  const int head = static_cast<int>(item / 2 % a.heads);
  const int64_t token = item / 2 / a.heads;
  int64_t slot = a.slots[token];
  if (slot >= a.total_slots) {
    if (lane == 0) report(kDevIndex);
    slot = -1;
  }
  uint8_t* tile = nullptr;
  const int at = static_cast<int>(slot % kKv4Tile);
  if (slot >= 0) {
    const int64_t page_tokens = static_cast<int64_t>(a.page_tiles) * kKv4Tile;
    const int64_t page = slot / page_tokens, in_page = slot % page_tokens;
    tile = a.cache + ((page * a.heads + head) * a.page_tiles + in_page / kKv4Tile) * kv4_tile_bytes(kDim);
  }
  const T* x = static_cast<const T*>(a.x[side]) + token * a.token_stride[side] + head * a.head_stride[side];
  T* values = static_cast<T*>(a.values[side]);
#pragma unroll
  for (int g = 0; g < kv4_groups(kDim); ++g) {
    const int c = g * kKv4Group + 2 * lane;
    const float v0 = to_float(x[c]), v1 = to_float(x[c + 1]);
    bool nan = v0 != v0 || v1 != v1;
    float low = fminf(v0, v1), high = fmaxf(v0, v1);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      low = fminf(low, __shfl_xor_sync(kFullMask, low, o));
      high = fmaxf(high, __shfl_xor_sync(kFullMask, high, o));
    }
    nan = __any_sync(kFullMask, nan);
    __nv_bfloat16 scale_b = __float2bfloat16_rn((high - low) * (1.0f / 15.0f));
    __nv_bfloat16 zero_b = __float2bfloat16_rn(low);
    float scale = __bfloat162float(scale_b), zero = __bfloat162float(zero_b);
    if (nan || !isfinite(scale) || !isfinite(zero)) {  // nothing finite stands for such a group
      scale = zero = __int_as_float(0x7fc00000);
      scale_b = zero_b = __ushort_as_bfloat16(0x7fc0);
    }
    const float inv = scale >= 0x1p-126f ? 1.0f / scale : 0.0f;
    const float q0 = fminf(fmaxf(rintf((v0 - zero) * inv), 0.0f), 15.0f);  // NaN gives 0
    const float q1 = fminf(fmaxf(rintf((v1 - zero) * inv), 0.0f), 15.0f);
    if (tile) {
      const uint8_t byte = static_cast<uint8_t>(static_cast<int>(q0) | static_cast<int>(q1) << 4);
      tile[side ? kv4_value_byte(kDim, at, c) : kv4_key_byte(kDim, at, c)] = byte;
      if (lane == 0) {
        const uint32_t pair = __bfloat16_as_ushort(scale_b) | static_cast<uint32_t>(__bfloat16_as_ushort(zero_b)) << 16;
        *reinterpret_cast<uint32_t*>(tile + (side ? kv4_value_scale(kDim, at, g) : kv4_key_scale(kDim, at, g))) = pair;
      }
    }
    if (values) {
      T* to = values + (token * a.heads + head) * kDim + c;
      to[0] = from_float<T>(q0 * scale + zero);
      to[1] = from_float<T>(q1 * scale + zero);
    }
  }
}

template <typename T>
cudaError_t launch_append(const AppendArgs& a, int dim, cudaStream_t stream) {
  constexpr int kWarps = 8;
  const int64_t blocks = (a.tokens * a.heads * 2 + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(blocks);
  if (dim == 64) append_kernel<T, 64><<<grid, kWarps * kWarp, 0, stream>>>(a);
  if (dim == 128) append_kernel<T, 128><<<grid, kWarps * kWarp, 0, stream>>>(a);
  if (dim == 256) append_kernel<T, 256><<<grid, kWarps * kWarp, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

PCK_STATUS_READER(append_status)

}  // namespace pck

extern "C" int pck_kv4_append(const pck_kv4_append_desc* desc, void* stream) {
  using namespace pck;
  if (!desc) return report_error(PCK_ERR_ARGUMENT, "append: NULL descriptor");
  const auto& [cache, pages, kv_heads, page_tiles, dim, k, v, dtype, tokens, k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots, k_values, v_values] = *desc;
  if (dim != 64 && dim != 128 && dim != 256) return report_error(PCK_ERR_ARGUMENT, "append: dim must be 64, 128 or 256");
  if (pages < 0 || kv_heads < 1 || kv_heads > 0x7fffffff || page_tiles < 1 || page_tiles > 0x7fffffff || tokens < 0) {
    return report_error(PCK_ERR_ARGUMENT, "append: need pages >= 0, kv_heads >= 1, page_tiles >= 1 and tokens >= 0");
  }
  if (dtype != PCK_LOGITS_F32 && dtype != PCK_LOGITS_BF16 && dtype != PCK_LOGITS_F16) {
    return report_error(PCK_ERR_ARGUMENT, "append: unknown dtype");
  }
  if (tokens == 0) return PCK_OK;
  if ((pages > 0 && !cache) || !k || !v || !slots) return report_error(PCK_ERR_ARGUMENT, "append: NULL cache, k, v or slots");
  if (!k_values != !v_values) return report_error(PCK_ERR_ARGUMENT, "append: k_values and v_values go together");
  if (!aligned_to(cache, 16)) return report_error(PCK_ERR_ARGUMENT, "append: the cache must be 16-byte aligned");
  AppendArgs a{};
  a.cache = static_cast<uint8_t*>(cache);
  a.x[0] = k;
  a.x[1] = v;
  a.token_stride[0] = k_token_stride;
  a.token_stride[1] = v_token_stride;
  a.head_stride[0] = k_head_stride;
  a.head_stride[1] = v_head_stride;
  a.values[0] = k_values;
  a.values[1] = v_values;
  a.slots = slots;
  a.tokens = tokens;
  a.total_slots = pages * page_tiles * kKv4Tile;
  a.heads = static_cast<int32_t>(kv_heads);
  a.page_tiles = static_cast<int32_t>(page_tiles);
  const int d = static_cast<int>(dim);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == PCK_LOGITS_F32    ? launch_append<float>(a, d, s)
                          : dtype == PCK_LOGITS_BF16 ? launch_append<__nv_bfloat16>(a, d, s)
                                                     : launch_append<__half>(a, d, s);
  return err == cudaSuccess ? PCK_OK : report_cuda("append kernel", err);
}
