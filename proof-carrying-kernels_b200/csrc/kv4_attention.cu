// pck_kv4_attention: softmax(scale * q k^T) v over the keys and values of a 4-bit cache.
//
// One CTA per (request, key/value head, query token); its threads share the head's group of query
// rows, one row after another: a chunk of keys, a thread each, for the scores; then a thread for
// each channel over the chunk's values. Running maximum and sum in binary32.
#include "kv4_layout.cuh"
#include "serving_common.cuh"

namespace pck {
namespace {

struct AttentionArgs {
  const void* q;
  int64_t q_batch_stride, q_token_stride, q_head_stride;
  const uint8_t* cache;
  int64_t pages;
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* lengths;
  void* out;
  float scale;
  int64_t window;
  int64_t max_tokens;  // page table columns * page tokens
  int32_t queries, heads, kv_heads, page_tiles;
};

constexpr int kChunk = 128;

__device__ __forceinline__ float decode(uint8_t byte, int c, uint32_t pair) {
  const float code = static_cast<float>((byte >> (c % 2 * 4)) & 15);
  return code * bf16_lo(pair) + bf16_hi(pair);
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kChunk) attention_kernel(const AttentionArgs a) {
  __shared__ float q[kDim];
  __shared__ float p[kChunk];
  __shared__ const uint8_t* tiles[kChunk / kKv4Tile];
  __shared__ float red[kChunk / kWarp];
  const int64_t item = blockIdx.x;
  const int t = static_cast<int>(item % a.queries);
  const int kvh = static_cast<int>(item / a.queries % a.kv_heads);
  const int64_t b = item / a.queries / a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  int64_t length = a.lengths[b];
  length = length < 0 ? 0 : length > a.max_tokens ? a.max_tokens : length;
  const int64_t last = length - a.queries + t;  // this row's own position
  int64_t first = a.window > 0 && last + 1 > a.window ? last + 1 - a.window : 0;
  constexpr int kPer = (kDim + kChunk - 1) / kChunk;
  for (int r = 0; r < group; ++r) {
    const int head = kvh * group + r;
    __syncthreads();
    for (int c = tid; c < kDim; c += kChunk) {
      q[c] = to_float(static_cast<const T*>(a.q)[b * a.q_batch_stride + t * a.q_token_stride + head * a.q_head_stride + c]);
    }
    float top = -INFINITY, sum = 0.0f, acc[kPer] = {};
    for (int64_t j0 = first / kChunk * kChunk; j0 <= last; j0 += kChunk) {
      __syncthreads();
      if (tid < kChunk / kKv4Tile) {
        const int64_t tile = j0 / kKv4Tile + tid;
        const uint8_t* at = nullptr;
        if (tile * kKv4Tile <= last) {
          const int64_t page = a.page_table[b * a.table_stride + tile / a.page_tiles];
          if (page >= 0 && page < a.pages) {
            at = a.cache + ((page * a.kv_heads + kvh) * a.page_tiles + tile % a.page_tiles) * kv4_tile_bytes(kDim);
          } else {
            report(kDevIndex);
          }
        }
        tiles[tid] = at;
      }
      __syncthreads();
      const uint8_t* tile = tiles[tid / kKv4Tile];
      const int at = tid % kKv4Tile;
      float s = -INFINITY;
      if (tile && j0 + tid >= first && j0 + tid <= last) {
        s = 0.0f;
        for (int c = 0; c < kDim; ++c) {
          const uint32_t pair = *reinterpret_cast<const uint32_t*>(tile + kv4_key_scale(kDim, at, c / kKv4Group));
          s = fmaf(q[c], decode(tile[kv4_key_byte(kDim, at, c & ~1)], c, pair), s);
        }
        s *= a.scale;
      }
      float m = s;
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
      if (lane == 0) red[warp] = m;
      __syncthreads();
      m = top;
      for (int w = 0; w < kChunk / kWarp; ++w) m = fmaxf(m, red[w]);
      const float keep = top == m ? 1.0f : expf(top - m);
      top = m;
      p[tid] = s == -INFINITY ? 0.0f : expf(s - top);
      __syncthreads();
      sum *= keep;
      for (int j = 0; j < kChunk; ++j) sum += p[j];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = tid + i * kChunk;
        acc[i] *= keep;
        for (int j = 0; j < kChunk; ++j) {
          if (c < kDim && p[j] != 0.0f) {
            const uint8_t* from = tiles[j / kKv4Tile];
            const int k = j % kKv4Tile;
            const uint32_t pair = *reinterpret_cast<const uint32_t*>(from + kv4_value_scale(kDim, k, c / kKv4Group));
            acc[i] = fmaf(p[j], decode(from[kv4_value_byte(kDim, k, c & ~1)], c, pair), acc[i]);
          }
        }
      }
    }
    T* out = static_cast<T*>(a.out) + ((b * a.queries + t) * a.heads + head) * kDim;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = tid + i * kChunk;
      if (c < kDim) out[c] = from_float<T>(sum == 0.0f ? 0.0f : acc[i] / sum);
    }
  }
}

template <typename T>
cudaError_t launch_attention(const AttentionArgs& a, int64_t batch, int dim, cudaStream_t stream) {
  const int64_t blocks = batch * a.kv_heads * a.queries;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(blocks);
  if (dim == 64) attention_kernel<T, 64><<<grid, kChunk, 0, stream>>>(a);
  if (dim == 128) attention_kernel<T, 128><<<grid, kChunk, 0, stream>>>(a);
  if (dim == 256) attention_kernel<T, 256><<<grid, kChunk, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

PCK_STATUS_READER(attention_status)

}  // namespace pck

extern "C" int64_t pck_kv4_attention_scratch(int64_t batch, int64_t queries, int64_t heads, int64_t kv_heads, int64_t dim,
                                             int64_t max_tokens) {
  if (batch < 0 || queries < 1 || kv_heads < 1 || heads < kv_heads || dim < 1 || max_tokens < 0) return -1;
  return 0;
}

extern "C" int pck_kv4_attention(const void* q, int dtype, int64_t batch, int64_t queries, int64_t heads, int64_t dim,
                                 int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride, const void* cache,
                                 int64_t pages, int64_t kv_heads, int64_t page_tiles, const int32_t* page_table,
                                 int64_t table_stride, int64_t table_pages, const int32_t* lengths, double scale,
                                 int64_t window, void* out, void* scratch, int64_t scratch_bytes, void* stream) {
  using namespace pck;
  (void)scratch;
  (void)scratch_bytes;
  if (dim != 64 && dim != 128 && dim != 256) return report_error(PCK_ERR_ARGUMENT, "attention: dim must be 64, 128 or 256");
  if (dtype != PCK_LOGITS_BF16 && dtype != PCK_LOGITS_F16) return report_error(PCK_ERR_ARGUMENT, "attention: q must be bfloat16 or float16");
  if (batch < 0 || queries < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0 || heads > 0xffff ||
      queries > 0xffff) {
    return report_error(PCK_ERR_ARGUMENT, "attention: need batch >= 0, queries >= 1 and heads a multiple of kv_heads");
  }
  if (pages < 0 || page_tiles < 1 || page_tiles > 0x7fffff || table_pages < 0 || table_stride < table_pages) {
    return report_error(PCK_ERR_ARGUMENT, "attention: need pages >= 0, page_tiles >= 1 and a page table of whole rows");
  }
  if (window < 0) return report_error(PCK_ERR_ARGUMENT, "attention: window must be 0 (none) or positive");
  if (!(scale > 0.0) || !(scale < 1e30)) return report_error(PCK_ERR_ARGUMENT, "attention: scale must be positive and finite");
  if (batch == 0) return PCK_OK;
  if (!q || !lengths || !out || (table_pages > 0 && !page_table) || (pages > 0 && !cache)) {
    return report_error(PCK_ERR_ARGUMENT, "attention: NULL q, cache, page_table, lengths or out");
  }
  if (!aligned_to(cache, 16)) return report_error(PCK_ERR_ARGUMENT, "attention: the cache must be 16-byte aligned");
  AttentionArgs a{};
  a.q = q;
  a.q_batch_stride = q_batch_stride;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.cache = static_cast<const uint8_t*>(cache);
  a.pages = pages;
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.lengths = lengths;
  a.out = out;
  a.scale = static_cast<float>(scale);
  a.window = window;
  a.max_tokens = table_pages * page_tiles * kKv4Tile;
  a.queries = static_cast<int32_t>(queries);
  a.heads = static_cast<int32_t>(heads);
  a.kv_heads = static_cast<int32_t>(kv_heads);
  a.page_tiles = static_cast<int32_t>(page_tiles);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == PCK_LOGITS_BF16 ? launch_attention<__nv_bfloat16>(a, batch, static_cast<int>(dim), s)
                                                   : launch_attention<__half>(a, batch, static_cast<int>(dim), s);
  return err == cudaSuccess ? PCK_OK : report_cuda("attention kernel", err);
}
