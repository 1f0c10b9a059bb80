// pck_kv4_attention: softmax(scale * q k^T) v over the keys and values of a 4-bit cache.
//
// The floor is memory: a decode step reads every code once for a few query rows, so the cache should come
// in at the HBM's rate and the work per code has to stay small. What that led to:
//   - The query rows that share a key/value head (its group of heads, and the query tokens of a
//     request) are the columns of one matrix product, 8 at a time: a tile of 16 tokens is read and
//     unpacked once for up to 32 of them. Both products have the codes on the left (keys: tokens x
//     channels, values: channels x tokens), which fills mma.sync's 16 rows even for a single query
//     row, and a lane then meets the scales of only two tokens. tcgen05 would want the unpacked codes
//     written to shared memory first, which alone would exceed its bandwidth at two codes a byte.
//   - Codes are unpacked to binary16 with a mask and an or, two codes an instruction: the four bits
//     become mantissa bits of 1024 + n or 1024 + 16 n, from which one more instruction makes n (keys)
//     or n - 8 (values, whose sums then cancel less), exactly. Leaving the 1024 in the keys' products and
//     taking it off their sums saved 3% with 8 rows (two requests of 262,143 tokens 137 and 141 us) but
//     lost 3% with 16 (148 and 142) and 7 bits of the scores: 1e-5 of an ordinary score where a binary32
//     dot product, and this one, err by 1e-7. Queries become binary16 times a power of two of their
//     row, which loses nothing. Scales never touch the codes: with k = code * s + z,
//       q.k = sum over groups of s (q.code) + z sum(q),
//     and for the values the weight p s of a token and group goes into the matrix product instead
//     of p; sum of p z is added at the end.
//   - Scores and sums are binary32. The weights p s are rounded to binary16 (11 bits, below the
//     rounding of a bfloat16 output), each row's and group's times a power of two that follows the
//     largest p s met so far: that one lies in 2 to 2^15, so what the smallest lose is at most 2^-26
//     of it. The size of a scale whose token has no weight is of no account.
//   - The running maximum is raised only when a score passes it by 2^8 (weights then stay within
//     2^8, and that of a row's first maximum, which is mostly its last, is 1, so that its p s is exact),
//     so the accumulators are rarely rescaled and the common tile needs no exchange between lanes for
//     it. Raising it lowers all p s met so far: the power of two takes the whole powers of that.
//   - Work is cut by the lengths, on the device. With few (request, head, row block) items a CTA takes
//     an equal piece of one of them; with many, the tiles of all items form one line that is cut into
//     equal parts, a CTA each, so one long request among short ones takes no longer than the rest. A
//     part of an item leaves its sums in scratch memory and a second kernel (a programmatic dependent)
//     joins them. A CTA's four warps take pairs of tiles in turn, each through its own ring of bulk
//     copies.
// Measured with 32 query heads over 8 of dim 128, bfloat16: two requests of 262,143 tokens 142 us (604 MB at
// 4.3 TB/s), 64 requests of 300 to 16,384 tokens 116 us, one of 1,027 tokens 12 us. Long requests in pages of 64
// tokens are bound by instructions: 335 a tile, 130 cycles of an SM, and as long when every tile comes from L2.
// That explains 65 us of the 64 ragged requests'; segments that begin and end in a CTA are the likely rest.
#include <algorithm>

#include "kv4_layout.cuh"
#include "kv4_ring.h"
#include "serving_common.cuh"

namespace pck {
namespace {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * kWarp;
// What beginning and ending an item costs a CTA (its queries, the first copies' latency, the join of
// its warps), in tiles: items count as that much longer when the line is cut, or the parts that hold
// many short items would end last.
constexpr int kItemCost = 8;
constexpr int kMinPiece = 8;  // tiles of a piece of an item, at least: two for each warp
constexpr int kMinPart = 16;  // length of a part, at least
constexpr float kRaise = 8.0f;      // log2 by which a score may pass the running maximum
constexpr int kUnitBias = 127;      // of a power of two's exponent field
constexpr int kUnitMost = 245;      // field of a row's largest unit, 2^118: times a weight it stays finite
constexpr int kJoinRows = 4;     // rows of a joining CTA, four warps each
constexpr int kJoinThreads = kJoinRows * 4 * kWarp;

struct AttentionArgs {
  const void* q;
  int64_t q_batch_stride, q_token_stride, q_head_stride;
  const uint8_t* cache;
  int64_t pages;
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* lengths;
  void* out;
  float* sums;        // (2 * parts, rows, dim) unnormalised outputs of split items
  float2* top_total;  // (2 * parts, rows): maximum (log2), sum of weights
  int2* split;        // (batch, kv_heads, row_blocks): the first part of an item, and how many it has
  float scale_log2;
  int64_t batch;
  int32_t window;
  int32_t max_tokens;  // page table columns * page tokens
  int32_t queries, heads, kv_heads, page_tiles;
  int32_t group;       // heads of a key/value head
  int32_t row_blocks;  // blocks of rows of a (request, key/value head)
  int32_t parts;       // most parts of the line of tiles
  int32_t q_vector;    // q rows are 16-byte aligned
};

struct Range {
  int first;  // first tile
  int tiles;
};

// Tiles that any query of request b sees.
__device__ __forceinline__ Range request_tiles(const AttentionArgs& a, int64_t b) {
  const int length = min(a.lengths[b], a.max_tokens);
  if (length <= 0) return {0, 0};
  int first = 0;
  if (a.window > 0) first = max(0, max(0, length - a.queries) + 1 - a.window) / kKv4Tile;
  return {first, (length - 1) / kKv4Tile - first + 1};
}

// An item's length on the line.
__device__ __forceinline__ int item_length(int tiles) { return tiles > 0 ? tiles + kItemCost : 0; }

// A 64-bit division takes several times a 32-bit one, and a CTA waits for these before its first copy.
__device__ __forceinline__ int64_t divide(int64_t x, int64_t by) {
  if (x < int64_t{1} << 32 && by < int64_t{1} << 32) return static_cast<uint32_t>(x) / static_cast<uint32_t>(by);
  return x / by;
}

// The line is cut into `parts` parts of `length` or length + 1 places, the longer ones first.
struct Cut {
  int64_t parts, length, longer;
  __device__ __forceinline__ int64_t begin(int64_t c) const { return c * length + min(c, longer); }
  __device__ __forceinline__ int64_t holds(int64_t x) const {
    const int64_t end = longer * (length + 1);
    return x < end ? divide(x, length + 1) : longer + divide(x - end, length);
  }
};

__device__ __forceinline__ Cut cut_line(const AttentionArgs& a, int64_t total) {
  const int64_t parts = max(int64_t{1}, min(static_cast<int64_t>(a.parts), divide(total, kMinPart)));
  const int64_t length = divide(total, parts);
  return {parts, length, total - length * parts};
}

// 2^x to 2^-22 of itself, 0 below 2^-126: a weight is rounded to 2^-11 of itself after it.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}

// Transposes an 8 x 8 matrix of 16-bit elements held two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t half2_bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }

// 2^n, zero below binary32's normal range; n <= 127.
__device__ __forceinline__ float power(int n) {
  return n >= 1 - kUnitBias ? __uint_as_float(static_cast<uint32_t>(n + kUnitBias) << 23) : 0.0f;
}

// The exponent field of one of two positive bfloat16 numbers, and another for it (with a mantissa of 0).
__device__ __forceinline__ int unit_field(uint32_t units, int e) { return static_cast<int>(units >> (16 * e + 7) & 255u); }
__device__ __forceinline__ void set_unit_field(uint32_t& units, int e, int field) {
  units = (units & 0xffff0000u >> 16 * e) | static_cast<uint32_t>(field) << (16 * e + 7);
}

// (w & mask) | bits in one instruction: both constants come in registers.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
}

// A constant that the compiler keeps in a register instead of building it at each use.
__device__ __forceinline__ uint32_t kept(uint32_t v) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

struct Masks {
  uint32_t low, high, bits;
};

// Four pairs of codes of a 32-bit word, nibbles (i, i + 4), in the mantissas of binary16 numbers:
// 1024 + n in the even pairs and 1024 + 16 n in the odd ones.
__device__ __forceinline__ void unpack_raw(uint32_t w, const Masks& k, uint32_t (&out)[4]) {
  out[0] = and_or(w, k.low, k.bits);
  out[1] = and_or(w, k.high, k.bits);
  w >>= 8;
  out[2] = and_or(w, k.low, k.bits);
  out[3] = and_or(w, k.high, k.bits);
}

// The same as n - kLess, exactly.
template <int kLess>
__device__ __forceinline__ void unpack(uint32_t w, const Masks& k, uint32_t (&out)[4]) {
  const __half2 low = __floats2half2_rn(1024.0f + kLess, 1024.0f + kLess);
  const __half2 part = __floats2half2_rn(0.0625f, 0.0625f), high = __floats2half2_rn(-64.0f - kLess, -64.0f - kLess);
  unpack_raw(w, k, out);
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    out[i] = half2_bits(__hsub2(*reinterpret_cast<__half2*>(&out[i]), low));
    out[i + 1] = half2_bits(__hfma2(*reinterpret_cast<__half2*>(&out[i + 1]), part, high));
  }
}

// Two elements of T as binary32.
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t v) {
  if constexpr (std::is_same_v<T, __half>) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  } else {
    return make_float2(bf16_lo(v), bf16_hi(v));
  }
}

template <int kWords>
__device__ __forceinline__ void load_words(uint32_t (&w)[kWords], const uint8_t* p) {
  if constexpr (kWords == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (kWords == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  }
}

// CTAs on an SM, by the registers that the rows' products take. Three of 8 rows at dim 128 have room for
// what four spill (us with two, three and four: a batch of 64 ragged requests 142, 116 and 122, two requests of
// 196,605 tokens 125, 110 and 112, of 16,383 tokens 24, 22 and 25).
constexpr int attention_ctas(int rows, int dim) {
  if (dim == 64) return rows <= 16 ? 4 : 2;
  if (dim == 128) return rows <= 16 ? 3 : 2;
  return 2;
}

template <typename T, int kDim, int kRows>
struct Shape {
  static constexpr int kGroups = kDim / kKv4Group;
  static constexpr int kPlanes = kGroups > 2 ? kGroups / 2 : 1;
  static constexpr int kWidth = kGroups > 1 ? 2 : 1;  // groups of a plane
  static constexpr int kCols = kRows / 8;             // column blocks of the products: 8 query rows each
  static constexpr int kTileBytes = kv4_tile_bytes(kDim);
  static constexpr int kCtas = attention_ctas(kRows, kDim);
  // Tiles that a warp takes at once: two share the checks of a step, where the registers allow it.
  static constexpr int kStage = kRows == 8 || kRows * kDim <= 16 * 64 ? 2 : 1;
  static constexpr int kStageBytes = kStage * kTileBytes;
  // Copies in flight for the HBM's latency: the SM's shared memory, less what the CTAs take beside it.
  static constexpr int kMost = (216 << 10) / (kCtas * kAttnWarps * kStageBytes);
  static constexpr int kSlots = kMost < 16 ? kMost : 16;
  static constexpr int kRing = kAttnWarps * kSlots * kStageBytes;
  static_assert(kRing >= kAttnWarps * kRows * kDim * 4, "the warps' sums overlay the rings");
};

// A CTA's place on the line of items.
struct Line {
  int64_t at, end;  // what is left of its part
  int64_t base;     // where request b begins
  int64_t b;
  Cut cut;
};

// The tiles of one item in a CTA's part.
struct Segment {
  int64_t b;
  int64_t item;         // of all requests
  int64_t last;         // the item's last place on the line
  int32_t pieces;       // equal pieces of the item, a CTA each; 0: parts of the line
  int32_t kvh, row0;    // key/value head, first row of the row block
  int32_t length;       // the request's
  int32_t count;        // tiles; 0: no segment is left
  int32_t lo, hi;       // those of them that some row of the block sees
  int32_t pos0, pos1;   // positions of the block's first and last query token
  bool whole, first;    // all tiles of the item; the item's first tile
};

// Tiles [offset, offset + count) of an item of request b.
template <int kRows>
__device__ __forceinline__ void set_segment(const AttentionArgs& a, Segment& s, int64_t b, Range range, int64_t item,
                                            int offset, int count) {
  s.b = b;
  s.item = b * a.kv_heads * a.row_blocks + item;
  s.count = count;
  s.whole = count == range.tiles;
  s.first = offset == 0;
  s.length = min(a.lengths[b], a.max_tokens);
  s.kvh = static_cast<int>(item);
  s.row0 = 0;
  if (a.row_blocks > 1) {
    s.kvh = static_cast<int>(divide(item, a.row_blocks));
    s.row0 = (static_cast<int>(item) - s.kvh * a.row_blocks) * kRows;
  }
  s.pos0 = s.pos1 = s.length - 1;
  if (a.queries > 1) {
    s.pos0 = s.length - a.queries + s.row0 / a.group;
    s.pos1 = s.length - a.queries + (min(s.row0 + kRows, a.queries * a.group) - 1) / a.group;
  }
  s.lo = range.first + offset;
  s.hi = s.lo + count;
  if (a.window > 0) s.lo = max(s.lo, max(0, s.pos0 + 1 - a.window) / kKv4Tile);
  s.hi = s.pos1 < 0 ? s.lo : min(s.hi, s.pos1 / kKv4Tile + 1);
}

// The next segment of a part of the line (count 0: none is left).
template <int kRows>
__device__ __forceinline__ void next_segment(const AttentionArgs& a, Line& line, Segment& s) {
  const int64_t items = static_cast<int64_t>(a.kv_heads) * a.row_blocks;
  int64_t at = line.at, b = line.b, base = line.base;
  s.count = 0;
  while (at < line.end && s.count == 0) {
    const Range range = request_tiles(a, b);
    const int size = item_length(range.tiles);
    if (at >= base + size * items) {
      base += size * items;
      ++b;
      continue;
    }
    const int64_t item = divide(at - base, size);
    const int start = static_cast<int>(at - base - item * size);
    const int stop = static_cast<int>(min(static_cast<int64_t>(size), start + (line.end - at)));
    at += stop - start;
    // Its tiles come after its cost.
    const int offset = max(0, start - kItemCost), count = max(0, stop - kItemCost) - offset;
    if (count == 0) continue;
    set_segment<kRows>(a, s, b, range, item, offset, count);
    s.last = base + (item + 1) * size - 1;
  }
  line.at = at;
  line.b = b;
  line.base = base;
}

// Four channels of a row: sums over the sum of weights (zeros for a row that saw nothing).
template <typename T>
__device__ __forceinline__ void store_row(T* to, float4 o, float l) {
  const float v[4] = {o.x, o.y, o.z, o.w};
  uint16_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T x = from_float<T>(l == 0.0f ? 0.0f : v[i] / l);
    u[i] = *reinterpret_cast<const uint16_t*>(&x);
  }
  *reinterpret_cast<uint2*>(to) =
      make_uint2(u[0] | static_cast<uint32_t>(u[1]) << 16, u[2] | static_cast<uint32_t>(u[3]) << 16);
}

template <typename T, int kDim, int kRows>
__global__ void __launch_bounds__(kAttnThreads, Shape<T, kDim, kRows>::kCtas)
    attention_kernel(const __grid_constant__ AttentionArgs a) {
  using S = Shape<T, kDim, kRows>;
  constexpr int kG = S::kGroups, kN = S::kCols, kStage = S::kStage;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kAttnWarps][S::kSlots];
  __shared__ float2 state[kAttnWarps][kRows];
  __shared__ Line line;
  __shared__ Segment segment;

  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const int row8 = lane / 4, quarter = lane % 4;
  if (lane == 0) {
    for (int s = 0; s < S::kSlots; ++s) mbar_init(&full[warp][s], kStage);
    fence_barrier_init();
  }
  __syncwarp();
  wait_for_producers();
  allow_dependents();

  T* const out = static_cast<T*>(a.out);
  const int64_t items = static_cast<int64_t>(a.kv_heads) * a.row_blocks;  // of a request
  if (warp == 0) {
    // What this CTA takes, of the items in the order (request, head, row block). Few items: one of the
    // equal pieces of one item. Many: its part of the line.
    const int mine = lane < a.batch ? request_tiles(a, lane).tiles : 0;
    int64_t total = item_length(mine), tiles = mine, filled = mine > 0;
    for (int64_t i = lane + kWarp; i < a.batch; i += kWarp) {
      const int n = request_tiles(a, i).tiles;
      total += item_length(n);
      tiles += n;
      filled += n > 0;
    }
    for (int o = 16; o && a.batch > 1; o >>= 1) {
      total += __shfl_xor_sync(kFullMask, total, o);
      tiles += __shfl_xor_sync(kFullMask, tiles, o);
      filled += __shfl_xor_sync(kFullMask, filled, o);
    }
    tiles = __shfl_sync(kFullMask, tiles, 0);
    filled = __shfl_sync(kFullMask, filled, 0) * items;
    const bool pieces = 2 * filled <= a.parts;
    // Tiles of a piece, at most: with this many the pieces are no more than the CTAs.
    const int64_t even = pieces ? divide(tiles * items, a.parts - filled) + 1 : 1;
    const int piece = static_cast<int>(max(int64_t{kMinPiece}, even));
    auto places = [&](int n) -> int64_t { return pieces ? (n + piece - 1) / piece : item_length(n); };
    int64_t begin = blockIdx.x, end = begin + 1;
    if (!pieces) {
      const Cut cut = cut_line(a, __shfl_sync(kFullMask, total, 0) * items);
      begin = blockIdx.x < cut.parts ? cut.begin(blockIdx.x) : 0;
      end = blockIdx.x < cut.parts ? cut.begin(blockIdx.x + 1) : 0;
      if (lane == 0) line.cut = cut;
    }
    // The request in which it begins, and where that begins.
    int64_t b = 0, base = 0;
    bool any = false;
    for (; begin < end && b < a.batch; b += kWarp) {
      int64_t n = places(b == 0 ? mine : b + lane < a.batch ? request_tiles(a, b + lane).tiles : 0) * items;
      int64_t before = n;
      for (int o = 1; o < kWarp && o < a.batch; o <<= 1) {
        const int64_t v = __shfl_up_sync(kFullMask, before, o);
        if (lane >= o) before += v;
      }
      const unsigned here = __ballot_sync(kFullMask, begin < base + before);
      any = here != 0;
      if (any) {
        const int l = __ffs(here) - 1;
        b += l;
        base += __shfl_sync(kFullMask, before - n, l);
        break;
      }
      base += __shfl_sync(kFullMask, before, kWarp - 1);
    }
    if (lane == 0) {
      line.at = begin;
      line.end = any ? end : begin;
      line.base = base;
      line.b = b;
      if (pieces) {
        line.at = line.end;
        segment.count = 0;
        if (any) {
          const Range range = request_tiles(a, b);
          const int n = static_cast<int>(places(range.tiles));
          const int item = static_cast<int>(begin - base) / n, i = static_cast<int>(begin - base) - item * n;
          const int size = range.tiles / n, longer = range.tiles - size * n;
          set_segment<kRows>(a, segment, b, range, item, i * size + min(i, longer), size + (i < longer));
          segment.pieces = n;
        }
      } else {
        segment.pieces = 0;
        next_segment<kRows>(a, line, segment);
      }
    }
  } else {
    // Requests that hold nothing give zeros.
    const int64_t row_size = static_cast<int64_t>(a.queries) * a.heads * kDim;
    for (int64_t b = blockIdx.x; b < a.batch; b += gridDim.x) {
      if (request_tiles(a, b).tiles == 0) {
        constexpr int kRest = kAttnThreads - kWarp;
        for (int64_t i = tid - kWarp; i < row_size; i += kRest) out[b * row_size + i] = from_float<T>(0.0f);
        for (int64_t i = tid - kWarp; a.parts > 1 && i < items; i += kRest) a.split[b * items + i] = make_int2(0, 0);
      }
    }
  }

  const uint64_t policy = policy_evict_first();
  const Masks masks{kept(0x000f000fu), kept(0x00f000f0u), kept(0x64006400u)};
  uint8_t* const ring = smem + warp * S::kSlots * S::kStageBytes;
  uint32_t phase = 0;  // parity bit of each slot
  bool dead = false;   // a wait gave up: this warp takes no more tiles
  while (true) {
    __syncthreads();
    if (segment.count == 0) return;
    const int64_t b = segment.b;
    const int kvh = segment.kvh, row0 = segment.row0, length = segment.length;
    const int lo = segment.lo, hi = segment.hi;
    const int rows = a.queries * a.group;
    // The warp's stages: kStage tiles each, every kAttnWarps-th.
    const int stages = max(0, hi - lo + kStage - 1) / kStage;
    const int warp_stages = dead ? 0 : (max(0, stages - warp) + kAttnWarps - 1) / kAttnWarps;

    // Where the tiles lie in the cache: those of 16 stages are looked up at once, a lane each, one
    // batch ahead of their use; -1 without a page or past the end.
    const int32_t* table = a.page_table + b * a.table_stride;
    auto look_up = [&](int k) -> int32_t {
      const int tile = lo + kStage * (warp + (k + lane / kStage) * kAttnWarps) + lane % kStage;
      if (tile >= hi) return -1;
      const int32_t page = table[tile / a.page_tiles];
      if (page < 0 || page >= a.pages) {
        report(kDevIndex);
        return -1;
      }
      return (page * a.kv_heads + kvh) * a.page_tiles + tile % a.page_tiles;
    };
    constexpr int kBatch = kWarp / kStage;
    int32_t places = look_up(0), places_next = look_up(kBatch);
    uint32_t absent = __ballot_sync(kFullMask, places < 0);
    uint32_t missing = 0;  // kStage bits a slot: tiles that it does not hold
    constexpr uint32_t kNone = (1u << kStage) - 1;
    // A tile's copy is issued by the lane that looked it up.
    auto copy = [&](int slot) {
      uint64_t* bar = &full[warp][slot];
      if (places < 0) {
        mbar_arrive(bar);
      } else {
        mbar_arrive_expect_tx(bar, S::kTileBytes);
        bulk_load(ring + slot * S::kStageBytes + lane % kStage * S::kTileBytes,
                  a.cache + static_cast<int64_t>(places) * S::kTileBytes, S::kTileBytes, bar, policy);
      }
    };
    auto issue = [&](int k, int slot) {
      const int at = k % kBatch;
      if (at == 0) {
        places = places_next;
        absent = __ballot_sync(kFullMask, places < 0);
        places_next = look_up(k + kBatch);
      }
      missing = (missing & ~(kNone << slot * kStage)) | (absent >> at * kStage & kNone) << slot * kStage;
      if (lane / kStage == at) copy(slot);
    };
    static_assert(S::kSlots <= kBatch, "the first copies come from one batch of places");
    missing = absent;  // slot s holds the tiles of lanes kStage s and on
    if (lane / kStage < min(S::kSlots, warp_stages)) copy(lane / kStage);

    // q as the right operand: this lane's row lane / 4 of each block, its channels in the order of
    // the codes: for each 8 channels the pairs (0, 4), (1, 5), (2, 6), (3, 7).
    uint32_t qf[kN][kG * 4][2];
    // What the products' columns belong to: rows 2 quarter and the next of each block.
    float qsum[kN][kG][2];
    float factor[kN][2];  // of a score: the softmax's scale (log2) over the row's power of two
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int r = row0 + 8 * n + row8;
      const int t = r / a.group;
      const T* qr = static_cast<const T*>(a.q) + b * a.q_batch_stride + t * a.q_token_stride +
                    static_cast<int64_t>(kvh * a.group + r % a.group) * a.q_head_stride;
      alignas(16) uint32_t x[kG][8];
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        if (r < rows) {
          const T* from = qr + g * kKv4Group + 16 * quarter;
          if (a.q_vector) {
            *reinterpret_cast<uint4*>(x[g]) = *reinterpret_cast<const uint4*>(from);
            *reinterpret_cast<uint4*>(x[g] + 4) = *reinterpret_cast<const uint4*>(from + 8);
          } else {
            const uint16_t* u = reinterpret_cast<const uint16_t*>(from);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[g][i] = u[2 * i] | static_cast<uint32_t>(u[2 * i + 1]) << 16;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[g][i] = 0;
        }
      }
      // The row as binary16, its largest element between 2^15 and 2^16 by a power of two (rows of zeros,
      // infinities or NaN as they are): binary16 queries lose nothing, bfloat16 ones nothing of elements
      // down to 2^-32 of the largest. (Products with keys beyond 2^100 would overflow.)
      uint32_t packed = 0;
#pragma unroll
      for (int g = 0; g < kG; ++g) {
#pragma unroll
        for (int i = 0; i < 8; ++i) packed = __vmaxu2(packed, x[g][i] & 0x7fff7fffu);
      }
      packed = __vmaxu2(packed, __shfl_xor_sync(kFullMask, packed, 1));
      packed = __vmaxu2(packed, __shfl_xor_sync(kFullMask, packed, 2));
      const uint32_t largest = __float_as_uint(unpack_pair<T>(max(packed & 0xffffu, packed >> 16)).x);
      uint32_t field = largest >> 23;
      field = field == 0 || field == 255 ? 142 : max(field, 16u);
      float scale = __uint_as_float((269u - field) << 23);
      float back = a.scale_log2 * __uint_as_float((field - 15u) << 23);
      if (back < 0x1p-126f) {  // below binary32's normal numbers: scores of 0 (a factor of 0 would make NaN of -inf)
        scale = 0.0f;
        back = 1.0f;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        factor[n][e] = __shfl_sync(kFullMask, back, (2 * quarter + e) * 4);
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float2 v = unpack_pair<T>(x[g][i]);
          const __half2 h = __floats2half2_rn(v.x * scale, v.y * scale);
          x[g][i] = half2_bits(h);
          v = __half22float2(h);
          sum += v.x + v.y;
        }
        sum += __shfl_xor_sync(kFullMask, sum, 1);
        sum += __shfl_xor_sync(kFullMask, sum, 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) qsum[n][g][e] = __shfl_sync(kFullMask, sum, (2 * quarter + e) * 4);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t* y = x[g] + 4 * w;
          uint32_t(*f)[2] = &qf[n][g * 4 + 2 * w];
          f[0][0] = __byte_perm(y[0], y[2], 0x5410);
          f[0][1] = __byte_perm(y[0], y[2], 0x7632);
          f[1][0] = __byte_perm(y[1], y[3], 0x5410);
          f[1][1] = __byte_perm(y[1], y[3], 0x7632);
        }
      }
    }

    if (segment.first && a.parts > 1 && tid == kAttnThreads - 1) {
      // Parts from this one to the one with the item's last place.
      const int n = segment.pieces ? segment.pieces
                    : segment.whole ? 1 : static_cast<int>(line.cut.holds(segment.last) - blockIdx.x + 1);
      a.split[segment.item] = make_int2(blockIdx.x, n);
    }

    // Products with the values: element e of [n][g][m] is channel 8 (lane / 4) + 2 m + e / 2 of group
    // g for row 2 quarter + e % 2 of block n.
    float acc[kN][kG][4][4];
    float total_w[kN][2], zeros[kN][kG][2];
    // The running maximum (log2; 0 while there is none) and the score that raises it (-inf while there
    // is none).
    float top[kN][2], limit[kN][2];
    // The power of two by which a row's weights of the values are multiplied, as bfloat16 for two rows, and
    // the largest of them.
    uint32_t unit[kN][kG];
    float unit_most[kG];
#pragma unroll
    for (int g = 0; g < kG; ++g) unit_most[g] = power(kUnitMost - kUnitBias);
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        limit[n][e] = -INFINITY;
        total_w[n][e] = top[n][e] = 0.0f;
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        zeros[n][g][0] = zeros[n][g][1] = 0.0f;
        unit[n][g] = kUnitMost << 23 | kUnitMost << 7;
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[n][g][m][0] = acc[n][g][m][1] = acc[n][g][m][2] = acc[n][g][m][3] = 0.0f;
      }
    }

    bool first = true;  // no stage yet
    // One stage. This lane's tokens are row8 + 8 j. kMasked: some row does not see some of them, or
    // a tile is missing.
    constexpr int kJ = 2 * kStage;
    auto stage_step = [&](const uint8_t* stage, int token0, uint32_t gone, auto masked_tag) {
      constexpr bool kMasked = decltype(masked_tag)::value;
      const bool fresh = first;
      first = false;
      float s[kN][kJ][2];  // element [j][e]: token row8 + 8 j, row 2 quarter + e
      bool off[kN][kJ][2];
#pragma unroll
      for (int u = 0; u < kStage; ++u) {
        const uint8_t* tile = stage + u * S::kTileBytes;
        uint32_t pairs[2][kG];
#pragma unroll
        for (int j = 0; j < 2; ++j) load_words(pairs[j], tile + kv4_key_scale(kDim, 8 * j, 0) + row8 * 4 * kG);
#pragma unroll
        for (int p = 0; p < S::kPlanes; ++p) {
          uint32_t w[2][2 * S::kWidth];
#pragma unroll
          for (int j = 0; j < 2; ++j) load_words(w[j], tile + p * 512 * S::kWidth + (j * kWarp + lane) * 8 * S::kWidth);
#pragma unroll
          for (int i = 0; i < S::kWidth; ++i) {
            const int g = p * S::kWidth + i;
            float part[kN][4];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t k0[4], k1[4];
              unpack<0>(w[0][2 * i + c], masks, k0);
              unpack<0>(w[1][2 * i + c], masks, k1);
#pragma unroll
              for (int n = 0; n < kN; ++n) {
                if (c == 0) part[n][0] = part[n][1] = part[n][2] = part[n][3] = 0.0f;
                mma(part[n], k0[0], k1[0], k0[1], k1[1], qf[n][g * 4 + 2 * c]);
                mma(part[n], k0[2], k1[2], k0[3], k1[3], qf[n][g * 4 + 2 * c + 1]);
              }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float scale = bf16_lo(pairs[j][g]);
              const float zero = bf16_hi(pairs[j][g]);
#pragma unroll
              for (int n = 0; n < kN; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float& to = s[n][2 * u + j][e];
                  const float x = part[n][2 * j + e];
                  to = g == 0 ? scale * x : fmaf(scale, x, to);
                  to = fmaf(zero, qsum[n][g][e], to);
                }
              }
            }
          }
        }
      }
      // Raise the maximum where a score passes it by more than 2^kRaise.
      bool pass = false;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = -INFINITY;
#pragma unroll
          for (int j = 0; j < kJ; ++j) {
            if constexpr (kMasked) {
              const int token = token0 + row8 + 8 * j, r = row0 + 8 * n + 2 * quarter + e;
              const int at = r < rows ? length - a.queries + r / a.group : -1;
              off[n][j][e] = token > at || (a.window > 0 && token <= at - a.window) || (gone >> j / 2 & 1u);
              if (off[n][j][e]) s[n][j][e] = -INFINITY;
            }
            m = fmaxf(m, s[n][j][e]);
          }
          pass = pass || m > limit[n][e];
        }
      }
      if (__any_sync(kFullMask, pass)) {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = s[n][0][e];
#pragma unroll
            for (int j = 1; j < kJ; ++j) m = fmaxf(m, s[n][j][e]);
            const float old = limit[n][e] == -INFINITY ? -INFINITY : top[n][e];
            m = fmaxf(old, m * factor[n][e]);
            m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 4));
            m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 8));
            m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 16));
            top[n][e] = m == -INFINITY ? 0.0f : m;
            limit[n][e] = (m + kRaise) / factor[n][e];
            if (fresh) continue;  // the sums are zeros
            // How far it rises, and by how many whole powers (more than any product has bits is as good as all).
            const float rise = old == m ? 0.0f : m - old;
            const int by = min(__float2int_rd(rise), 512);
            const float keep = exp2_fast(-rise);
            total_w[n][e] *= keep;
#pragma unroll
            for (int g = 0; g < kG; ++g) {
              zeros[n][g][e] *= keep;
              const int field = unit_field(unit[n][g], e), next = min(field + by, kUnitMost);
              set_unit_field(unit[n][g], e, next);
              unit_most[g] = fmaxf(unit_most[g], power(next - kUnitBias));
              const float rest = exp2_fast(by - rise) * power(next - field - by);  // (1 to 1/2, if the unit can grow so far)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                acc[n][g][i][e] *= rest;
                acc[n][g][i][e + 2] *= rest;
              }
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int j = 0; j < kJ; ++j) {
            s[n][j][e] = exp2_fast(fmaf(s[n][j][e], factor[n][e], -top[n][e]));
            total_w[n][e] += s[n][j][e];
          }
        }
      }
      // The values, a group at a time: its scales go into the weights.
      uint32_t pairs[kJ][kG];
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        load_words(pairs[j], stage + j / 2 * S::kTileBytes + kv4_value_scale(kDim, 8 * (j % 2), 0) + row8 * 4 * kG);
        if constexpr (kMasked) {
          if (token0 + row8 + 8 * j >= length || (gone >> j / 2 & 1u)) {  // nothing was written there
#pragma unroll
            for (int g = 0; g < kG; ++g) pairs[j][g] = 0;
          }
        }
      }
      // Weights are up to 2^8: where a scale is up to 2^7 in the largest unit, no product leaves binary16.
      bool outgrown = false;
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        uint32_t largest = 0;
#pragma unroll
        for (int j = 0; j < kJ; ++j) largest = max(largest, pairs[j][g] << 16);
        outgrown = outgrown || !(__uint_as_float(largest) * unit_most[g] <= 128.0f);  // (or a NaN)
      }
      if (__any_sync(kFullMask, outgrown)) {
        // The units that the stage's products have really outgrown: one whose largest is 2^4 or more in it
        // has it at 2 to 4 after that.
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          int most = 0;
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            // Exponent fields of the two rows' largest products, times 2^-10, so that no weight of up to 2^8
            // overflows them.
            float largest[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
              const float scale = bf16_lo(pairs[j][g]) * power(-10);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                if (!kMasked || !off[n][j][e]) largest[e] = fmaxf(largest[e], s[n][j][e] * scale);
              }
            }
            uint32_t sizes = __byte_perm(__float_as_uint(largest[0]), __float_as_uint(largest[1]), 0x7632);
            sizes = __vmaxu2(sizes, __shfl_xor_sync(kFullMask, sizes, 4));
            sizes = __vmaxu2(sizes, __shfl_xor_sync(kFullMask, sizes, 8));
            sizes = __vmaxu2(sizes, __shfl_xor_sync(kFullMask, sizes, 16));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int size = unit_field(sizes, e) - kUnitBias + 10, field = unit_field(unit[n][g], e);
              const int next = size + field - kUnitBias >= 4 ? max(1 - size + kUnitBias, 1) : field;
              set_unit_field(unit[n][g], e, next);
              most = max(most, next);
              const float ratio = power(next - field);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                acc[n][g][i][e] *= ratio;
                acc[n][g][i][e + 2] *= ratio;
              }
            }
          }
          unit_most[g] = power(most - kUnitBias);
        }
      }
#pragma unroll
      for (int u = 0; u < kStage; ++u) {
        const uint8_t* tile = stage + u * S::kTileBytes;
#pragma unroll
        for (int p = 0; p < S::kPlanes; ++p) {
          uint32_t w[2][2 * S::kWidth];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            load_words(w[j], tile + 9 * kDim + p * 512 * S::kWidth + (j * kWarp + lane) * 8 * S::kWidth);
          }
#pragma unroll
          for (int i = 0; i < S::kWidth; ++i) {
            const int g = p * S::kWidth + i;
            uint32_t wf[kN][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t pair = pairs[2 * u + j][g];
              const float scale = bf16_lo(pair), zero = fmaf(8.0f, scale, bf16_hi(pair));
#pragma unroll
              for (int n = 0; n < kN; ++n) {
                float product[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const float weight = s[n][2 * u + j][e];
                  product[e] = weight * (e ? bf16_hi(unit[n][g]) : bf16_lo(unit[n][g])) * scale;
                  if constexpr (kMasked) {  // a NaN scale must not reach rows that do not see its token
                    if (off[n][2 * u + j][e]) {
                      product[e] = 0.0f;
                      continue;
                    }
                  }
                  zeros[n][g][e] = fmaf(weight, zero, zeros[n][g][e]);
                }
                wf[n][j] = transpose8(half2_bits(__floats2half2_rn(product[0], product[1])));
              }
            }
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              uint32_t v0[4], v1[4];
              unpack<8>(w[0][2 * i + d], masks, v0);
              unpack<8>(w[1][2 * i + d], masks, v1);
#pragma unroll
              for (int n = 0; n < kN; ++n) {
                mma(acc[n][g][2 * d], v0[0], v0[1], v1[0], v1[1], wf[n]);
                mma(acc[n][g][2 * d + 1], v0[2], v0[3], v1[2], v1[3], wf[n]);
              }
            }
          }
        }
      }
    };

    auto wait = [&](int slot) {
      const bool landed = __all_sync(kFullMask, mbar_wait(&full[warp][slot], phase >> slot & 1u));
      phase ^= 1u << slot;
      return landed;
    };
    auto use = [&](int k, int slot) {
      const uint32_t gone = missing >> slot * kStage & kNone;
      if (gone != kNone) {
        const uint8_t* stage = ring + slot * S::kStageBytes;
        const int token0 = (lo + kStage * (warp + k * kAttnWarps)) * kKv4Tile;
        if (gone == 0 && token0 + kStage * kKv4Tile - 1 <= segment.pos0 &&
            (a.window <= 0 || token0 > segment.pos1 - a.window)) {
          stage_step(stage, token0, 0, std::false_type{});
        } else {
          stage_step(stage, token0, gone, std::true_type{});
        }
      }
      __syncwarp();
    };
    dead |= !take_stages<S::kSlots>(warp_stages, wait, use, issue);

    // Join the warps: their sums in shared memory (over the rings, which are empty now), then a
    // thread for each element.
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * n + 2 * quarter + e;
        float l = total_w[n][e];
        for (int o = 4; o < kWarp; o <<= 1) l += __shfl_xor_sync(kFullMask, l, o);
        if (row8 == 0) state[warp][r] = make_float2(limit[n][e] == -INFINITY ? -INFINITY : top[n][e], l);
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          float z = zeros[n][g][e];
          for (int o = 4; o < kWarp; o <<= 1) z += __shfl_xor_sync(kFullMask, z, o);
          const float u = power(kUnitBias - unit_field(unit[n][g], e));
          float4* to = reinterpret_cast<float4*>(sums + (warp * kRows + r) * kDim + g * kKv4Group + 8 * row8);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float(*x)[4] = &acc[n][g][2 * i];
            to[i] = make_float4(fmaf(x[0][e], u, z), fmaf(x[0][e + 2], u, z), fmaf(x[1][e], u, z), fmaf(x[1][e + 2], u, z));
          }
        }
      }
    }
    __syncthreads();
    const int64_t slot_id = 2 * static_cast<int64_t>(blockIdx.x) + (segment.first ? 1 : 0);
    const int kept = min(kRows, rows - row0);
    for (int i = 4 * tid; i < kept * kDim; i += 4 * kAttnThreads) {
      const int r = i / kDim, c = i % kDim;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) m = fmaxf(m, state[w][r].x);
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float f = state[w][r].x == -INFINITY ? 0.0f : exp2_fast(state[w][r].x - m);
        const float4 v = *reinterpret_cast<const float4*>(sums + (w * kRows + r) * kDim + c);
        o = make_float4(fmaf(f, v.x, o.x), fmaf(f, v.y, o.y), fmaf(f, v.z, o.z), fmaf(f, v.w, o.w));
        l = fmaf(f, state[w][r].y, l);
      }
      if (segment.whole) {
        const int t = (row0 + r) / a.group, head = kvh * a.group + (row0 + r) % a.group;
        store_row(out + ((b * a.queries + t) * a.heads + head) * kDim + c, o, l);
      } else {
        *reinterpret_cast<float4*>(a.sums + (slot_id * kRows + r) * kDim + c) = o;
        if (c == 0) a.top_total[slot_id * kRows + r] = make_float2(m, l);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next bulk copies land here
    if (segment.pieces) return;
    __syncthreads();
    if (tid == 0) next_segment<kRows>(a, line, segment);
  }
}

// Joins the parts of split items: a CTA for each four rows of an item, four warps a row.
template <typename T, int kDim, int kRows>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ AttentionArgs a) {
  constexpr int kVectors = kDim / 128 > 1 ? 2 : 1;  // float4 of a lane (dim 64: half the lanes)
  __shared__ float4 sums[kJoinRows][4][kDim / 4];
  __shared__ float2 red[kJoinRows][4];
  const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp, w = warp % 4;
  const int chunks = (min(kRows, a.queries * a.group) + kJoinRows - 1) / kJoinRows;
  const int64_t item = blockIdx.x / chunks;
  const int in_block = static_cast<int>(blockIdx.x % chunks) * kJoinRows + warp / 4;
  const int row = static_cast<int>(item % a.row_blocks) * kRows + in_block;
  const bool mine = in_block < kRows && row < a.queries * a.group;
  wait_for_producers();
  const int2 split = a.split[item];
  const int n = split.y;
  if (n <= 1) return;  // nothing to join
  // The part that holds the item's beginning has it in its second slot, the others in their first.
  auto slot_of = [&](int i) { return (2 * (static_cast<int64_t>(split.x) + i) + (i == 0 ? 1 : 0)) * kRows + in_block; };
  const bool holds = mine && lane * 4 < kDim;
  // A warp's share of the parts, four loads at a time, by its own running maximum.
  float m = -INFINITY, l = 0.0f;
  float4 o[kVectors] = {};
  for (int i0 = w; mine && i0 < n; i0 += 16) {
    float2 tops[4];
    float4 v[4][kVectors];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + 4 * u;
      tops[u] = i < n ? a.top_total[slot_of(i)] : make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int k = 0; k < kVectors; ++k) {
        v[u][k] = i < n && holds ? reinterpret_cast<const float4*>(a.sums + slot_of(i) * kDim)[lane + k * kWarp]
                                 : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    }
    float next = m;
#pragma unroll
    for (int u = 0; u < 4; ++u) next = fmaxf(next, tops[u].x);
    const float keep = m == -INFINITY ? 0.0f : exp2_fast(m - next);
    m = next;
    l *= keep;
#pragma unroll
    for (int k = 0; k < kVectors; ++k) o[k] = make_float4(o[k].x * keep, o[k].y * keep, o[k].z * keep, o[k].w * keep);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float f = tops[u].x == -INFINITY ? 0.0f : exp2_fast(tops[u].x - m);
      l = fmaf(f, tops[u].y, l);
#pragma unroll
      for (int k = 0; k < kVectors; ++k) {
        o[k] = make_float4(fmaf(f, v[u][k].x, o[k].x), fmaf(f, v[u][k].y, o[k].y), fmaf(f, v[u][k].z, o[k].z),
                           fmaf(f, v[u][k].w, o[k].w));
      }
    }
  }
  if (lane == 0) red[warp / 4][w] = make_float2(m, l);
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    if (holds) sums[warp / 4][w][lane + k * kWarp] = o[k];
  }
  __syncthreads();
  if (w != 0 || !holds) return;
  m = -INFINITY;
  l = 0.0f;
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaxf(m, red[warp / 4][i].x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = red[warp / 4][i];
    f[i] = v.x == -INFINITY ? 0.0f : exp2_fast(v.x - m);
    l = fmaf(f[i], v.y, l);
  }
  const int64_t b = item / a.row_blocks / a.kv_heads;
  const int kvh = static_cast<int>(item / a.row_blocks % a.kv_heads);
  T* out = static_cast<T*>(a.out) + ((b * a.queries + row / a.group) * a.heads + kvh * a.group + row % a.group) * kDim;
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = sums[warp / 4][i][lane + k * kWarp];
      v = make_float4(fmaf(f[i], x.x, v.x), fmaf(f[i], x.y, v.y), fmaf(f[i], x.z, v.z), fmaf(f[i], x.w, v.w));
    }
    store_row(out + 4 * (lane + k * kWarp), v, l);
  }
}

// Rows of a block: as many as the item has, up to what the registers hold beside the products.
int block_rows(int64_t rows, int64_t dim) {
  if (rows <= 8) return 8;
  if (rows <= 16 || dim == 256) return 16;
  return dim == 128 ? 24 : 32;
}

int sm_count() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!cache[dev]) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1) v = 148;
    cache[dev] = v;
  }
  return cache[dev];
}

// Most parts of a call: the CTAs that run at once, and no more than the longest lengths can fill.
int64_t most_parts(int64_t batch, int64_t queries, int64_t group, int64_t kv_heads, int64_t dim, int64_t max_tokens) {
  const int rows = block_rows(queries * group, dim);
  const int64_t ctas = static_cast<int64_t>(sm_count()) * attention_ctas(rows, static_cast<int>(dim));
  const int64_t blocks = (queries * group + rows - 1) / rows;
  const int64_t tiles = (max_tokens + kKv4Tile - 1) / kKv4Tile;
  const int64_t items = batch * kv_heads * blocks;
  if (tiles == 0) return 1;
  return std::min(ctas, items >= ctas ? ctas : std::max<int64_t>(items * ((tiles + kMinPiece - 1) / kMinPiece), 1));
}

// Bytes of scratch of a call: sums, maxima and totals of two partial items a part, and the split items.
int64_t scratch_size(int64_t parts, int rows, int64_t dim, int64_t items) {
  return parts == 1 ? 0 : 2 * parts * rows * (dim * 4 + 8) + items * 8;
}

template <typename T, int kDim, int kRows>
cudaError_t launch(const AttentionArgs& a, cudaStream_t stream) {
  using S = Shape<T, kDim, kRows>;
  static bool configured[64] = {};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t err = cudaFuncSetAttribute(attention_kernel<T, kDim, kRows>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, S::kRing);
    if (err != cudaSuccess) return err;
    configured[dev] = true;
  }
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(a.parts));
  config.blockDim = dim3(kAttnThreads);
  config.dynamicSmemBytes = S::kRing;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  cudaError_t err = cudaLaunchKernelEx(&config, attention_kernel<T, kDim, kRows>, a);
  if (err != cudaSuccess || a.parts == 1) return err;  // one part: nothing is split
  const int chunks = (std::min(kRows, a.queries * a.group) + kJoinRows - 1) / kJoinRows;
  const int64_t joins = a.batch * a.kv_heads * a.row_blocks * chunks;
  if (joins > 0x7fffffffLL) return cudaErrorInvalidValue;
  config.gridDim = dim3(static_cast<unsigned>(joins));
  config.blockDim = dim3(kJoinThreads);
  config.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&config, join_kernel<T, kDim, kRows>, a);
}

template <typename T>
cudaError_t launch_any(const AttentionArgs& a, int64_t dim, int rows, cudaStream_t s) {
  if (dim == 64) return rows == 8 ? launch<T, 64, 8>(a, s) : rows == 16 ? launch<T, 64, 16>(a, s) : launch<T, 64, 32>(a, s);
  if (dim == 128) {
    return rows == 8 ? launch<T, 128, 8>(a, s) : rows == 16 ? launch<T, 128, 16>(a, s) : launch<T, 128, 24>(a, s);
  }
  return rows == 8 ? launch<T, 256, 8>(a, s) : launch<T, 256, 16>(a, s);
}

}  // namespace

PCK_STATUS_READER(attention_status)

}  // namespace pck

extern "C" int64_t pck_kv4_attention_scratch(int64_t batch, int64_t queries, int64_t heads, int64_t kv_heads, int64_t dim,
                                             int64_t max_tokens) {
  if (batch < 0 || queries < 1 || kv_heads < 1 || heads < kv_heads || dim < 1 || max_tokens < 0) return -1;
  const int64_t parts = pck::most_parts(batch, queries, heads / kv_heads, kv_heads, dim, max_tokens);
  const int rows = pck::block_rows(queries * (heads / kv_heads), dim);
  const int64_t blocks = (queries * (heads / kv_heads) + rows - 1) / rows;
  return pck::scratch_size(parts, rows, dim, batch * kv_heads * blocks);
}

extern "C" int pck_kv4_attention(const pck_kv4_attention_desc* desc, void* stream) {
  using namespace pck;
  if (!desc) return report_error(PCK_ERR_ARGUMENT, "attention: NULL descriptor");
  const auto& [q, dtype, batch, queries, heads, dim, q_batch_stride, q_token_stride, q_head_stride, cache, pages,
               kv_heads, page_tiles, page_table, table_stride, table_pages, lengths, scale, window, out, scratch,
               scratch_bytes] = *desc;
  if (dim != 64 && dim != 128 && dim != 256) {
    return report_error(PCK_ERR_ARGUMENT, "attention: dim must be 64, 128 or 256");
  }
  if (dtype != PCK_LOGITS_BF16 && dtype != PCK_LOGITS_F16) {
    return report_error(PCK_ERR_ARGUMENT, "attention: q must be bfloat16 or float16");
  }
  if (batch < 0 || queries < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0 || heads > 0xffff ||
      queries > 0x7fff) {
    return report_error(PCK_ERR_ARGUMENT, "attention: need batch >= 0, queries in [1, 32767] and heads a multiple of kv_heads");
  }
  if (pages < 0 || pages > 0x7fffffff || page_tiles < 1 || page_tiles > 0x7fffff || table_pages < 0 || table_pages > 0x7fffffff ||
      !rows_apart(table_stride, table_pages)) {
    return report_error(PCK_ERR_ARGUMENT, "attention: need pages >= 0, page_tiles >= 1 and a page table of whole rows");
  }
  if (window < 0) return report_error(PCK_ERR_ARGUMENT, "attention: window must be 0 (none) or positive");
  if (!(scale > 0.0) || !(scale < 1e30)) return report_error(PCK_ERR_ARGUMENT, "attention: scale must be positive and finite");
  if (batch == 0) return PCK_OK;
  if (!q || !lengths || !out || (table_pages > 0 && !page_table) || (pages > 0 && !cache)) {
    return report_error(PCK_ERR_ARGUMENT, "attention: NULL q, cache, page_table, lengths or out");
  }
  if (!aligned_to(cache, 16) || !aligned_to(out, 8)) {
    return report_error(PCK_ERR_ARGUMENT, "attention: the cache must be 16-byte aligned, out 8-byte aligned");
  }
  if (pages * kv_heads > (int64_t{1} << 31) / page_tiles) {
    return report_error(PCK_ERR_UNSUPPORTED, "attention: a cache holds at most 2^31 tiles");
  }
  const int64_t max_tokens = table_pages * page_tiles * kKv4Tile;
  if (max_tokens > 1 << 30) return report_error(PCK_ERR_UNSUPPORTED, "attention: a request holds at most 2^30 tokens");
  const int64_t group = heads / kv_heads;
  const int rows = block_rows(queries * group, dim);
  AttentionArgs a{};
  a.parts = static_cast<int32_t>(most_parts(batch, queries, group, kv_heads, dim, max_tokens));
  a.row_blocks = static_cast<int32_t>((queries * group + rows - 1) / rows);
  if (a.parts > 1) {
    if (!scratch || !aligned_to(scratch, 16) || scratch_bytes < scratch_size(a.parts, rows, dim, batch * kv_heads * a.row_blocks)) {
      return report_error(PCK_ERR_ARGUMENT, "attention: needs pck_kv4_attention_scratch() bytes of aligned scratch");
    }
    const int64_t slots = 2LL * a.parts * rows;
    a.sums = static_cast<float*>(scratch);
    a.top_total = reinterpret_cast<float2*>(a.sums + slots * dim);
    a.split = reinterpret_cast<int2*>(a.top_total + slots);
  }
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
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.window = window < max_tokens ? static_cast<int32_t>(window) : 0;
  a.max_tokens = static_cast<int32_t>(max_tokens);
  a.batch = batch;
  a.queries = static_cast<int32_t>(queries);
  a.heads = static_cast<int32_t>(heads);
  a.kv_heads = static_cast<int32_t>(kv_heads);
  a.page_tiles = static_cast<int32_t>(page_tiles);
  a.group = static_cast<int32_t>(group);
  a.q_vector = aligned_to(q, 16) && q_batch_stride % 8 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == PCK_LOGITS_BF16 ? launch_any<__nv_bfloat16>(a, dim, rows, s)
                                                   : launch_any<__half>(a, dim, rows, s);
  return err == cudaSuccess ? PCK_OK : report_cuda("attention kernel", err);
}
