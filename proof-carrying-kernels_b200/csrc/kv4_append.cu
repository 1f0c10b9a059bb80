// pck_kv4_append: quantises keys and values to 4 bits and writes them to their slots of a cache.
//
// Per token, head and group of 64 channels: scale = bf16((max - min) / 15), zero = bf16(min), code =
// clamp(rint((x - zero) / scale), 0, 15), in binary32 with separate products and sums, so the codes
// are the same wherever the same formula is evaluated. The division by 15 is a product with the
// binary32 nearest 1/15 and the division by the scale one with its rounded reciprocal.
//
// A warp takes 8 tokens of one head's keys or values, a lane a quarter of each group's channels of one
// token, so that a lane's key codes are one 16-byte piece of the tile. Value codes of two neighbouring
// tokens share 32-bit words: where the next token's slot is the next one, the two lanes exchange halves
// and write 16 bytes each; single 16-bit pieces remain for decode steps and the ends of prompts. The
// floor is memory: the inputs are read once, the codes written once, in whole 32-byte sectors. 16,381 tokens of
// 8 heads of 128, bfloat16, values returned: 32 us, 4.7 TB/s, with 67% of the issue slots taken (640 instructions a
// warp); 16 tokens: 2.8 us, one launch's latency.
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
  int32_t vector;  // rows of k and v are 16-byte aligned
};

// Smaller and larger of two, NaN if either is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 16 channels of a row, as they lie.
template <typename T>
struct Raw16 {
  uint4 w[sizeof(T)];
  __device__ __forceinline__ void load(const T* from, bool vector) {
    if (vector) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(from) + i);
    } else {
      alignas(16) T e[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = from[i];
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) w[i] = reinterpret_cast<const uint4*>(e)[i];
    }
  }
  __device__ __forceinline__ float at(int i) const { return to_float(reinterpret_cast<const T*>(w)[i]); }
};

template <typename T, int kDim>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int kPlanes = kDim > 128 ? kDim / 128 : 1, kWidth = kv4_plane_groups(kDim);
  const int lane = threadIdx.x % kWarp, row = lane / 4, quarter = lane % 4;
  const int plane = static_cast<int>(blockIdx.y) % kPlanes, side = static_cast<int>(blockIdx.y) / kPlanes % 2;
  const int head = static_cast<int>(blockIdx.y) / kPlanes / 2;
  const int64_t token = (static_cast<int64_t>(blockIdx.x) * (blockDim.x / kWarp) + threadIdx.x / kWarp) * 8 + row;
  wait_for_producers();
  allow_dependents();
  const bool there = token < a.tokens;
  int64_t slot = there ? a.slots[token] : -1;
  // The inputs are on their way before anything waits for the slot.
  const T* x = static_cast<const T*>(a.x[side]) + token * a.token_stride[side] + head * a.head_stride[side];
  Raw16<T> raw[kWidth];
#pragma unroll
  for (int g = 0; g < kWidth; ++g) {
    if (there) {
      raw[g].load(x + (plane * kWidth + g) * kKv4Group + 16 * quarter, a.vector);
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) raw[g].w[i] = make_uint4(0, 0, 0, 0);
    }
  }
  if (slot >= a.total_slots) {
    if (quarter == 0) report(kDevIndex);
    slot = -1;
  }
  // The lane that holds the other token of this one's pair of slots, if it is in this warp.
  const int other = slot % 2 == 0 ? lane + 4 : lane - 4;
  const int64_t other_slot = __shfl_sync(kFullMask, slot, other & 31);
  const bool paired = slot >= 0 && other >= 0 && other < kWarp && other_slot == (slot ^ 1);
  const int at = static_cast<int>(slot % kKv4Tile);
  uint8_t* tile = nullptr;
  if (slot >= 0) {
    // (A 64-bit division takes several times a 32-bit one; caches of 2^32 slots are rare.)
    const int64_t index = slot / kKv4Tile;
    const int64_t page = a.total_slots < int64_t{1} << 32
                             ? static_cast<uint32_t>(index) / static_cast<uint32_t>(a.page_tiles) : index / a.page_tiles;
    tile = a.cache + ((page * a.heads + head) * a.page_tiles + (index - page * a.page_tiles)) * kv4_tile_bytes(kDim);
  }
  float v[kWidth][16];
#pragma unroll
  for (int g = 0; g < kWidth; ++g) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[g][i] = raw[g].at(i);
  }
  uint32_t codes[kWidth][2], pairs[kWidth];
#pragma unroll
  for (int g = 0; g < kWidth; ++g) {
    float low = v[g][0], high = v[g][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) {
      low = min_nan(low, v[g][i]);
      high = max_nan(high, v[g][i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      low = min_nan(low, __shfl_xor_sync(kFullMask, low, o));
      high = max_nan(high, __shfl_xor_sync(kFullMask, high, o));
    }
    const __nv_bfloat16 scale_b = __float2bfloat16_rn((high - low) * (1.0f / 15.0f)), zero_b = __float2bfloat16_rn(low);
    float scale = __bfloat162float(scale_b), zero = __bfloat162float(zero_b);
    pairs[g] = __bfloat16_as_ushort(scale_b) | static_cast<uint32_t>(__bfloat16_as_ushort(zero_b)) << 16;
    if (!isfinite(scale) || !isfinite(zero)) {  // nothing finite stands for such a group
      scale = zero = __int_as_float(0x7fc00000);
      pairs[g] = 0x7fc07fc0u;
    }
    const float inv = scale >= 0x1p-126f ? 1.0f / scale : 0.0f;
    // rint of a number in [0, 15] by a sum with 1.5 2^23, which leaves it in the low bits (the codes are
    // added up with the rest of that number's bits, taken off at once below). q * scale is exact, so the
    // value's one rounding is that of the sum.
    codes[g][0] = codes[g][1] = 0u - 0x4b400000u * 0x11111111u;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float y = fminf(fmaxf((v[g][i] - zero) * inv, 0.0f), 15.0f) + 12582912.0f;  // NaN gives 0
      codes[g][i / 8] += __float_as_uint(y) << (4 * (i % 8));
      v[g][i] = fmaf(y - 12582912.0f, scale, zero);
    }
  }
  // The exchange: the token of the even slot writes the pair's first 8 channels of its quarter, the
  // other the second.
  const int mine = slot & 1;
  uint32_t theirs[kWidth];
#pragma unroll
  for (int g = 0; g < kWidth; ++g) theirs[g] = __shfl_sync(kFullMask, mine ? codes[g][0] : codes[g][1], other & 31);
  if (tile) {
    uint8_t* const plane_at = tile + plane * 512 * kWidth;
    if (side == 0) {
      uint8_t* to = plane_at + at * 32 * kWidth + quarter * 8 * kWidth;
      if constexpr (kWidth == 2) {
        *reinterpret_cast<uint4*>(to) = make_uint4(codes[0][0], codes[0][1], codes[1][0], codes[1][1]);
      } else {
        *reinterpret_cast<uint2*>(to) = make_uint2(codes[0][0], codes[0][1]);
      }
    } else {
      uint8_t* to = plane_at + 9 * kDim + at / 8 * 256 * kWidth + at % 8 / 2 * 8 * kWidth;
      if (paired) {
        uint32_t w[2 * kWidth];
#pragma unroll
        for (int g = 0; g < kWidth; ++g) {
          const uint32_t own = mine ? codes[g][1] : codes[g][0];
          const uint32_t even = mine ? theirs[g] : own, odd = mine ? own : theirs[g];
          w[2 * g] = __byte_perm(even, odd, 0x5410);
          w[2 * g + 1] = __byte_perm(even, odd, 0x7632);
        }
        to += (2 * quarter + mine) * 32 * kWidth;
        if constexpr (kWidth == 2) {
          *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
          *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
        }
      } else {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
#pragma unroll
          for (int g = 0; g < kWidth; ++g) {
            uint16_t* piece = reinterpret_cast<uint16_t*>(to + (2 * quarter + o) * 32 * kWidth + g * 8) + mine;
            piece[0] = static_cast<uint16_t>(codes[g][o]);
            piece[2] = static_cast<uint16_t>(codes[g][o] >> 16);
          }
        }
      }
    }
    if (quarter == 0) {
      uint32_t* to = reinterpret_cast<uint32_t*>(tile + (side ? kv4_value_scale(kDim, at, 0) : kv4_key_scale(kDim, at, 0)));
#pragma unroll
      for (int g = 0; g < kWidth; ++g) to[plane * kWidth + g] = pairs[g];
    }
  }
  T* values = static_cast<T*>(a.values[side]);
  if (values && there) {
#pragma unroll
    for (int g = 0; g < kWidth; ++g) {
      T* to = values + (token * a.heads + head) * kDim + (plane * kWidth + g) * kKv4Group + 16 * quarter;
      alignas(16) T e[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = from_float<T>(v[g][i]);
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(e)[i];
    }
  }
}

template <typename T, int kDim>
cudaError_t launch_dim(const AppendArgs& a, cudaStream_t stream) {
  constexpr int kPlanes = kDim > 128 ? kDim / 128 : 1;
  const int64_t warps = (a.tokens + 7) / 8, sides = static_cast<int64_t>(a.heads) * 2 * kPlanes;
  // Few tokens: a warp a CTA, on as many SMs as there are.
  const int per = warps * sides >= 2048 ? 8 : 1;
  const int64_t blocks = (warps + per - 1) / per;
  if (blocks > 0x7fffffffLL || sides > 0xffff) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(sides));
  config.blockDim = dim3(static_cast<unsigned>(per * kWarp));
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, append_kernel<T, kDim>, a);
}

template <typename T>
cudaError_t launch_append(AppendArgs a, int64_t dim, cudaStream_t stream) {
  const int64_t e = 16 / sizeof(T);
  a.vector = aligned_to(a.x[0], 16) && aligned_to(a.x[1], 16) && a.token_stride[0] % e == 0 && a.head_stride[0] % e == 0 &&
             a.token_stride[1] % e == 0 && a.head_stride[1] % e == 0;
  return dim == 64 ? launch_dim<T, 64>(a, stream) : dim == 128 ? launch_dim<T, 128>(a, stream) : launch_dim<T, 256>(a, stream);
}

}  // namespace

PCK_STATUS_READER(append_status)

}  // namespace pck

extern "C" int pck_kv4_append(const pck_kv4_append_desc* desc, void* stream) {
  using namespace pck;
  if (!desc) return report_error(PCK_ERR_ARGUMENT, "append: NULL descriptor");
  const auto& [cache, pages, kv_heads, page_tiles, dim, k, v, dtype, tokens, k_token_stride, k_head_stride,
               v_token_stride, v_head_stride, slots, k_values, v_values] = *desc;
  if (dim != 64 && dim != 128 && dim != 256) {
    return report_error(PCK_ERR_ARGUMENT, "append: dim must be 64, 128 or 256");
  }
  if (pages < 0 || kv_heads < 1 || kv_heads > 0x3fff || page_tiles < 1 || page_tiles > 0x7fffffff || tokens < 0) {
    return report_error(PCK_ERR_ARGUMENT, "append: need pages >= 0, kv_heads in [1, 16383], page_tiles >= 1 and tokens >= 0");
  }
  if (pages > (int64_t{1} << 62) / (kv_heads * kv4_tile_bytes(static_cast<int>(dim))) / page_tiles) {
    return report_error(PCK_ERR_UNSUPPORTED, "append: a cache holds at most 2^62 bytes");
  }
  if (dtype != PCK_LOGITS_F32 && dtype != PCK_LOGITS_BF16 && dtype != PCK_LOGITS_F16) {
    return report_error(PCK_ERR_ARGUMENT, "append: unknown dtype");
  }
  if (tokens == 0) return PCK_OK;
  if ((pages > 0 && !cache) || !k || !v || !slots) return report_error(PCK_ERR_ARGUMENT, "append: NULL cache, k, v or slots");
  if (!k_values != !v_values) return report_error(PCK_ERR_ARGUMENT, "append: k_values and v_values go together");
  if (!aligned_to(cache, 16) || !aligned_to(k_values, 16) || !aligned_to(v_values, 16)) {
    return report_error(PCK_ERR_ARGUMENT, "append: the cache and the values must be 16-byte aligned");
  }
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
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == PCK_LOGITS_F32    ? launch_append<float>(a, dim, s)
                          : dtype == PCK_LOGITS_BF16 ? launch_append<__nv_bfloat16>(a, dim, s)
                                                     : launch_append<__half>(a, dim, s);
  return err == cudaSuccess ? PCK_OK : report_cuda("append kernel", err);
}
