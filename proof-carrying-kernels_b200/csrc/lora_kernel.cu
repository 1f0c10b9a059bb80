// pck_lora_add: out = y + s_a B_a (A_a x) for rows that each name their adapter a.
//
// Rows come in any order and are taken by their adapters, an item being some rows of one adapter:
//   - decode batches, where nearly every row has its own: up to 16 rows of one adapter, gathered from 256
//     rows, so an adapter's weights are read once for all of them;
//   - prompts, whose rows share one: the rows of one adapter in a tile of 64.
// A cluster of CTAs takes an item:
//   1. h = A x for the item's rows: the CTAs and their warps split the columns n, and each product
//      (mma.sync, binary32 sums) takes x and A straight from memory in 16-byte loads, since nothing in
//      a warp reads them twice;
//   2. the warps' and then the CTAs' partial sums are added in a fixed order, through shared and
//      distributed shared memory: h stays in binary32;
//   3. out = y + s B h: the CTAs and warps split the outputs m. h enters the products as three bfloat16
//      terms whose sum is h, or as two binary16 ones of h times a power of two of its row, the second
//      times 2^12 beside it: 23 of its 24 bits for elements down to 2^-29 of the row's largest one, and of
//      smaller ones what is above 2^-51 of that. (The sums go by 2^12 around the second term's products,
//      which costs no bit.)
// The floor is the adapters' bytes for decode batches and x, y and out for prompts. Few rows are bound by the
// latency of the two dependent passes (one row of rank 16, 4096 x 4096: 7.1 us), which is why a row is spread
// over a cluster. Prompts run their passes one after the other (4,099 rows, 14336 to 4096: 80 us against
// a floor of 39; A x 28 us, x alone at 4.1 TB/s, and the outputs 30 us, y and out at 4.5 TB/s).
#include <cooperative_groups.h>

#include <type_traits>

#include "serving_common.cuh"

namespace pck {
namespace {

namespace cg = cooperative_groups;

constexpr int kLoraMaxRank = 256;
constexpr int kLoraMaxCtas = 8;  // of a cluster
constexpr int kLoraWarps = 8;
constexpr int kLoraThreads = kLoraWarps * kWarp;

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
  int64_t n, m, tokens;
  int32_t count, rank;
  int32_t rank0;      // first rank of this launch, which takes up to `taken` of them
  int32_t taken;
  int32_t n_vector;   // rows of x and A are 16-byte aligned
  int32_t rank_vector;  // ranks that the rows of B are aligned to: 8, 4 or 0
};

template <typename T>
__device__ __forceinline__ void lora_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// The first of the terms that an element becomes: cut off in bfloat16, whose rounding would make an
// infinity of the largest binary32 numbers (the terms after it hold the rest all the same).
template <typename T>
__device__ __forceinline__ T first_term(float v) {
  if constexpr (std::is_same_v<T, __half>) {
    return __float2half_rn(v);
  } else {
    return __float2bfloat16_rz(v);
  }
}

// Elements [at, at + kN) of a row of 16-bit elements, zeros from `end` on. A row holds `held` >= end
// elements, a multiple of kN where `vector` is set; all loads are issued before any is waited for.
template <int kN>
__device__ __forceinline__ void load_row(uint32_t (&v)[kN / 2], const uint16_t* row, int64_t at, int64_t end, int64_t held,
                                         bool vector) {
  if (vector) {
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) v[i] = 0;
    if (at < held) {
      if constexpr (kN == 8) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(row + at));
        v[0] = x.x;
        v[1] = x.y;
        v[2] = x.z;
        v[3] = x.w;
      } else {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(row + at));
        v[0] = x.x;
        v[1] = x.y;
      }
    }
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const int64_t e = at + 2 * i;
      v[i] = e + 1 < end ? v[i] : e < end ? v[i] & 0xffffu : 0u;
    }
    return;
  }
  uint32_t x[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) x[i] = at + i < end ? __ldg(row + at + i) : 0;
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) v[i] = x[2 * i] | x[2 * i + 1] << 16;
}

// kSub: 16-row blocks of a tile; kNT: blocks of 8 ranks.
template <int kSub, int kNT>
struct LoraShape {
  static constexpr int kM = 16 * kSub;
  static constexpr int kR = 8 * kNT;                   // ranks, padded
  static constexpr int kStride = kR + (kR > 16 ? 4 : 0);  // of the terms' rows, for 8-byte reads at all banks
  static constexpr int kSplit = kLoraWarps / kSub;     // warps that share a block's columns
  static constexpr int kBlock = kNT < 16 ? kNT : 16;   // rank blocks whose loads are in flight together
  static constexpr int kSteps = kNT <= 2 ? 3 : kNT <= 4 ? 2 : 1;  // 32-column steps in flight together
  static constexpr int kPart = kSplit * kM * kR * 4;
  static constexpr int kTerms = 3 * kM * kStride * 2;
  static constexpr int kWork = kPart > kTerms ? kPart : kTerms;  // the terms overlay the warps' sums
  static constexpr int kSums = kWork + 2 * kM * kR * 4;
  // Tiles of several blocks: stages of 64 columns of the rows and of A, before the sums take their place.
  static constexpr int kStageBytes = (kM + kR) * 128;
  static constexpr int kStages = kNT <= 4 ? 7 : kNT <= 8 ? 6 : 4;
  static constexpr int kSmem = kSub > 1 && kStages * kStageBytes > kSums ? kStages * kStageBytes : kSums;
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// A x of a tile of several 16-row blocks, over the whole pairs of steps of [k0, k1): 64 columns of the rows
// and of A in a ring of asynchronous copies, which all the warps that share them read (a row's 16-byte
// pieces are exchanged by the row's parity, so a read meets no bank twice). Returns the step it got to.
template <typename T, int kSub, int kNT>
__device__ __forceinline__ int64_t staged_steps(const LoraArgs& a, uint8_t* smem, const uint32_t (&rows)[2], int64_t row0,
                                                int adapter, int rank, int64_t k0, int64_t k1, bool active,
                                                float (&acc)[kNT][4]) {
  using S = LoraShape<kSub, kNT>;
  if (!a.n_vector) return k0;
  const int64_t stages = (min(k1, a.n / 32) - k0) / 2;
  if (stages <= 0) return k0;
  const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
  const int row8 = lane / 4, quarter = lane % 4, sub = warp % kSub, share = warp / kSub;
  const int other = rows[0] ? __ffs(rows[0]) - 1 : 31 + __ffs(rows[1]);
  const uint16_t* const Aa = static_cast<const uint16_t*>(a.A) + (static_cast<int64_t>(adapter) * a.rank + a.rank0) * a.n;
  // The pieces that this thread copies: row i / 8, piece i % 8 of 128 bytes.
  constexpr int kPieces = (S::kM + S::kR) * 8;
  constexpr int kMine = (kPieces + kLoraThreads - 1) / kLoraThreads;
  const int used = (S::kM + rank) * 8;  // (what lies in the ranks past the adapter's is not used)
  const uint16_t* from[kMine];
  uint32_t to[kMine];
#pragma unroll
  for (int p = 0; p < kMine; ++p) {
    const int i = p * kLoraThreads + threadIdx.x, r = i / 8, c = i % 8;
    to[p] = smem_addr(smem) + r * 128 + (c ^ (r % 2 * 4)) * 16;
    if (r < S::kM) {
      const int x = (r < 32 ? rows[0] >> r : rows[1] >> (r - 32)) & 1u ? r : other;
      from[p] = static_cast<const uint16_t*>(a.x) + (row0 + x) * a.x_stride + 32 * k0 + 8 * c;
    } else {
      from[p] = Aa + min(r - S::kM, rank - 1) * a.n + 32 * k0 + 8 * c;
    }
  }
  auto copy = [&](int64_t stage) {
    if (stage < stages) {
#pragma unroll
      for (int p = 0; p < kMine; ++p) {
        if (p * kLoraThreads + static_cast<int>(threadIdx.x) < used) {
          copy16(to[p] + static_cast<uint32_t>(stage % S::kStages) * S::kStageBytes, from[p] + 64 * stage);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int s = 0; s < S::kStages - 1; ++s) copy(s);
  for (int64_t stage = 0; stage < stages; ++stage) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
    __syncthreads();  // this stage is there for every warp, and the one before it is read
    copy(stage + S::kStages - 1);
    if (active) {
      const uint8_t* at = smem + stage % S::kStages * S::kStageBytes;
      auto piece = [&](int r) {
        return *reinterpret_cast<const uint4*>(at + r * 128 + ((4 * share + quarter) ^ (r % 2 * 4)) * 16);
      };
      const uint4 x0 = piece(16 * sub + row8), x1 = piece(16 * sub + row8 + 8);
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        if (8 * j < rank) {
          const uint4 w = piece(S::kM + 8 * j + row8);
          lora_mma<T>(acc[j], x0.x, x1.x, x0.y, x1.y, w.x, w.y);
          lora_mma<T>(acc[j], x0.z, x1.z, x0.w, x1.w, w.z, w.w);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  return k0 + 2 * stages;
}

// kWhole: rows of y and out are 16-byte aligned.
template <typename T, int kSub, int kNT, bool kWhole>
__global__ void __launch_bounds__(kLoraThreads, kNT <= 8 ? 2 : 1) lora_kernel(const __grid_constant__ LoraArgs a) {
  using S = LoraShape<kSub, kNT>;
  constexpr int kTerms = std::is_same_v<T, __half> ? 2 : 3;
  constexpr float kTermUnit = std::is_same_v<T, __half> ? 4096.0f : 1.0f;  // of the second term
  extern __shared__ __align__(16) uint8_t smem[];
  float* const part = reinterpret_cast<float*>(smem);              // [split][row][rank]
  uint16_t* const terms = reinterpret_cast<uint16_t*>(smem);       // [term][row][stride]
  float* const sums = reinterpret_cast<float*>(smem + S::kWork);   // [row][rank] of this CTA
  float* const whole = sums + S::kM * S::kR;                       // and of the cluster
  __shared__ float unit[S::kM];  // what a row of terms is multiplied by
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
  const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
  const int row8 = lane / 4, quarter = lane % 4;
  const int sub = warp % kSub, share = warp / kSub;
  constexpr int kSpan = kSub == 1 ? kLoraThreads : S::kM;  // rows that a cluster's items come from
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / ctas) * kSpan;
  __shared__ int members[16];  // of an item of a decode batch: its rows
  wait_for_producers();
  allow_dependents();

  // A row's adapter: -1 for none, -2 past the last row.
  auto owner_of = [&](int r) {
    int owner = row0 + r < a.tokens ? max(a.adapters[row0 + r], -1) : -2;
    if (owner >= a.count) {
      if (cta == 0 && blockIdx.y == 0) report(kDevIndex);
      owner = -1;
    }
    return owner;
  };
  int owner[2] = {-2, -2};
  if constexpr (kSub > 1) {  // lane i has row i and row 32 + i of the tile
    owner[0] = owner_of(lane);
    owner[1] = owner_of(32 + lane);
  }
  for (int item = blockIdx.y;; item += gridDim.y) {
    // The item's adapter and its rows, as bits.
    uint32_t rows[2] = {0, 0};
    int adapter = -1;
    if constexpr (kSub == 1) {
      // Groups of 16 rows of one adapter (rows without one are another), numbered by their first rows.
      __shared__ __align__(16) int owners[kLoraThreads];
      __shared__ int firsts[kLoraWarps];
      __shared__ int found[2];
      const int tid = threadIdx.x;
      owners[tid] = owner_of(tid);
      if (tid == 0) found[0] = -2;
      __syncthreads();
      const int own = owners[tid];
      int before = 0;  // rows of the same adapter before this one
      const int upto = own == -2 ? 0 : (warp + 1) * kWarp;
      for (int k = 0; k < upto; k += 4) {
        const int4 v = *reinterpret_cast<const int4*>(owners + k);
        before += (v.x == own && k < tid) + (v.y == own && k + 1 < tid);
        before += (v.z == own && k + 2 < tid) + (v.w == own && k + 3 < tid);
      }
      const bool first = own >= -1 && before % 16 == 0;
      const unsigned ballot = __ballot_sync(kFullMask, first);
      if (lane == 0) firsts[warp] = __popc(ballot);
      __syncthreads();
      int number = __popc(ballot & ((1u << lane) - 1));
      for (int w = 0; w < warp; ++w) number += firsts[w];
      if (first && number == item) {
        found[0] = own;
        found[1] = before;
      }
      __syncthreads();
      if (found[0] == -2) return;  // there are fewer groups
      adapter = found[0];
      const int place = before - found[1];
      const bool member = own == adapter && place >= 0 && place < 16;
      if (member) members[place] = tid;
      rows[0] = (1u << __syncthreads_count(member)) - 1;
    } else {
      uint32_t left[2] = {__ballot_sync(kFullMask, owner[0] >= 0), __ballot_sync(kFullMask, owner[1] >= 0)};
      for (int i = 0; left[0] | left[1]; ++i) {
        const int first = left[0] ? __shfl_sync(kFullMask, owner[0], __ffs(left[0]) - 1)
                                  : __shfl_sync(kFullMask, owner[1], __ffs(left[1]) - 1);
        const uint32_t in0 = __ballot_sync(kFullMask, owner[0] == first);
        const uint32_t in1 = __ballot_sync(kFullMask, owner[1] == first);
        if (i == item) {
          adapter = first;
          rows[0] = in0;
          rows[1] = in1;
          break;
        }
        left[0] &= ~in0;
        left[1] &= ~in1;
      }
      if (adapter < 0 && item > 0) return;
    }
    // Rows without an adapter: a group of their own, or with the tile's first item.
    uint32_t plain[2] = {0, 0};
    if constexpr (kSub == 1) {
      if (adapter < 0) {
        plain[0] = rows[0];
        rows[0] = 0;
      }
    } else if (item == 0) {
      plain[0] = __ballot_sync(kFullMask, owner[0] == -1);
      plain[1] = __ballot_sync(kFullMask, owner[1] == -1);
    }
    int rank = adapter < 0 ? 0 : a.ranks ? min(max(a.ranks[adapter], 0), a.rank) : a.rank;
    rank = min(max(rank - a.rank0, 0), a.taken);
    if (a.rank0 > 0) {  // a later launch on the same rows: out already has what these add to
      if (rank == 0) {
        if (kSub == 1) return;
        continue;
      }
      plain[0] = plain[1] = 0;
    }
    const float scale = adapter >= 0 && a.scales ? a.scales[adapter] : 1.0f;
    // This warp's 16 rows of the item.
    const uint32_t active = (sub < 2 ? rows[0] >> 16 * sub : rows[1] >> 16 * (sub - 2)) & 0xffffu;
    const uint32_t copied = (sub < 2 ? plain[0] >> 16 * sub : plain[1] >> 16 * (sub - 2)) & 0xffffu;
    // Where row r of the block lies.
    auto row_of = [&](int r) { return row0 + (kSub == 1 ? members[r] : 16 * sub + r); };
    const int64_t m_blocks = (a.m + 31) / 32;
    const int64_t m0 = m_blocks * cta / ctas, m1 = m_blocks * (cta + 1) / ctas;
    const uint16_t* const Ba = static_cast<const uint16_t*>(a.B) + static_cast<int64_t>(max(adapter, 0)) * a.m * a.rank + a.rank0;
    if (kSub == 1 && rank > 0) {  // B is not needed before h: have it on its way
      const char* from = reinterpret_cast<const char*>(Ba + 32 * m0 * a.rank);
      const int64_t bytes = (min(32 * m1, a.m) - 32 * m0) * a.rank * 2;
      for (int64_t i = threadIdx.x * 128; i < bytes; i += kLoraThreads * 128) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(from + i));
      }
    }

    if (rank > 0) {
      // 1. This warp's share of A x.
      float acc[kNT][4];
#pragma unroll
      for (int j = 0; j < kNT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
      const int64_t steps = (a.n + 31) / 32;
      const int64_t k0 = steps * cta / ctas, k1 = steps * (cta + 1) / ctas;
      int64_t k = k0 + share * S::kSteps;
      if constexpr (kSub > 1) {
        k = staged_steps<T, kSub, kNT>(a, smem, rows, row0, adapter, rank, k0, k1, active != 0, acc) + share * S::kSteps;
      }
      if (active) {
        // Rows of the tile that are not the item's, and ranks past the adapter's, take another's elements:
        // what comes of them is not used.
        const int other = __ffs(active) - 1;
        const uint16_t* x[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = active >> (row8 + 8 * h) & 1u ? row8 + 8 * h : other;
          x[h] = static_cast<const uint16_t*>(a.x) + row_of(r) * a.x_stride;
        }
        const uint16_t* const Aa = static_cast<const uint16_t*>(a.A) + (static_cast<int64_t>(adapter) * a.rank + a.rank0) * a.n;
        auto product = [&](int j, const uint32_t (&x0)[4], const uint32_t (&x1)[4], const uint32_t (&w)[4]) {
          lora_mma<T>(acc[j], x0[0], x1[0], x0[1], x1[1], w[0], w[1]);
          lora_mma<T>(acc[j], x0[2], x1[2], x0[3], x1[3], w[2], w[3]);
        };
        // Whole steps by 16-byte loads, kSteps of them in flight together.
        const int64_t full = a.n_vector && kSub == 1 ? min(k1, a.n / 32) : k0;
        for (; k + S::kSteps <= full; k += S::kSplit * S::kSteps) {
          uint4 xv[S::kSteps][2];
#pragma unroll
          for (int u = 0; u < S::kSteps; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              xv[u][h] = __ldg(reinterpret_cast<const uint4*>(x[h] + 32 * (k + u) + 8 * quarter));
            }
          }
#pragma unroll
          for (int j0 = 0; j0 < kNT; j0 += S::kBlock) {
            if (8 * j0 < rank) {
              uint4 wv[S::kSteps][S::kBlock];
#pragma unroll
              for (int j = 0; j < S::kBlock; ++j) {
                const uint16_t* from = Aa + min(8 * (j0 + j) + row8, rank - 1) * a.n + 32 * k + 8 * quarter;
#pragma unroll
                for (int u = 0; u < S::kSteps; ++u) wv[u][j] = __ldg(reinterpret_cast<const uint4*>(from + 32 * u));
              }
#pragma unroll
              for (int u = 0; u < S::kSteps; ++u) {
                const uint32_t x0[4] = {xv[u][0].x, xv[u][0].y, xv[u][0].z, xv[u][0].w};
                const uint32_t x1[4] = {xv[u][1].x, xv[u][1].y, xv[u][1].z, xv[u][1].w};
#pragma unroll
                for (int j = 0; j < S::kBlock; ++j) {
                  product(j0 + j, x0, x1, {wv[u][j].x, wv[u][j].y, wv[u][j].z, wv[u][j].w});
                }
              }
            }
          }
        }
        // What is left, a step at a time with every element's place looked at: the last columns, or rows
        // without alignment.
        for (; k < k1; k += S::kSplit * S::kSteps) {
          for (int u = 0; u < S::kSteps && k + u < k1; ++u) {
            uint32_t xv[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) load_row<8>(xv[h], x[h], 32 * (k + u) + 8 * quarter, a.n, a.n, a.n_vector);
#pragma unroll
            for (int j = 0; j < kNT; ++j) {
              if (8 * j < rank) {
                uint32_t wv[4];
                load_row<8>(wv, Aa + min(8 * j + row8, rank - 1) * a.n, 32 * (k + u) + 8 * quarter, a.n, a.n, a.n_vector);
                product(j, xv[0], xv[1], wv);
              }
            }
          }
        }
      }
      // 2. The warps' sums, then the cluster's, in the order of their ranks.
      float* const mine = part + (share * S::kM + 16 * sub) * S::kR + 2 * quarter;
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        *reinterpret_cast<float2*>(mine + row8 * S::kR + 8 * j) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(mine + (row8 + 8) * S::kR + 8 * j) = make_float2(acc[j][2], acc[j][3]);
      }
      __syncthreads();
      for (int i = threadIdx.x; i < S::kM * S::kR / 4; i += kLoraThreads) {
        float4 v = reinterpret_cast<const float4*>(part)[i];
#pragma unroll
        for (int s = 1; s < S::kSplit; ++s) {
          const float4 x = reinterpret_cast<const float4*>(part)[s * S::kM * S::kR / 4 + i];
          v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
        }
        reinterpret_cast<float4*>(sums)[i] = v;
      }
      cluster.sync();
      for (int i = threadIdx.x; i < S::kM * S::kR / 4; i += kLoraThreads) {
        float4 v[kLoraMaxCtas];
#pragma unroll
        for (int q = 0; q < kLoraMaxCtas; ++q) {
          v[q] = q < ctas ? *cluster.map_shared_rank(reinterpret_cast<const float4*>(sums) + i, q)
                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int q = 1; q < kLoraMaxCtas; ++q) {
          v[0] = make_float4(v[0].x + v[q].x, v[0].y + v[q].y, v[0].z + v[q].z, v[0].w + v[q].w);
        }
        reinterpret_cast<float4*>(whole)[i] = v[0];
      }
      if (ctas > 1) cluster.barrier_arrive();  // this CTA has read its peers' sums
      __syncthreads();
      for (int r = warp; r < S::kM; r += kLoraWarps) {  // a warp a row
        constexpr int kPer = (S::kR + kWarp - 1) / kWarp;
        float h[kPer];
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int c = i * kWarp + lane;
          h[i] = c < rank ? whole[r * S::kR + c] * scale : 0.0f;
          if (isfinite(h[i])) largest = fmaxf(largest, fabsf(h[i]));
        }
        float down = 1.0f;
        if constexpr (std::is_same_v<T, __half>) {  // the row's largest finite one between 2^14 and 2^15
          for (int o = 16; o; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(kFullMask, largest, o));
          uint32_t field = __float_as_uint(largest) >> 23;
          field = field == 0 ? 127 : max(field, 15u);
          down = __uint_as_float((268u - field) << 23);
          if (lane == 0) unit[r] = __uint_as_float((field - 14u) << 23);
        } else {
          if (lane == 0) unit[r] = 1.0f;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int c = i * kWarp + lane;
          if (c >= S::kR) continue;
          float v = h[i] * down;
#pragma unroll
          for (int t = 0; t < kTerms; ++t) {
            const T x = t == 0 ? first_term<T>(v) : from_float<T>(v);
            terms[(t * S::kM + r) * S::kStride + c] = *reinterpret_cast<const uint16_t*>(&x);
            v = isfinite(v) ? (v - to_float(x)) * kTermUnit : 0.0f;
          }
        }
      }
      __syncthreads();
    }

    // 3. The outputs, 32 columns at a time: block j of a product has the columns 8 t + 2 j + e, so a lane
    // ends with 8 neighbouring ones of its rows. Where rows are not 16-byte aligned (!kWhole) it has the
    // columns 4 (2 j + e) + t, so that a load or store of single elements meets neighbouring ones in a quad
    // (2,000 rows of rank 32, 4096 to 4097: 94 us with a lane's columns neighbouring and their y loaded last,
    // 54 so; a choice in one kernel instead of two cost the aligned rows 40 to 45 us at 4096 to 4096).
    const int first = kWhole ? 8 * quarter : quarter;
    // Up to 64 ranks of B for a block. A lane takes neighbouring ranks of its column (16 of 64, 8 of 32, 4
    // of 16), so that a warp's load asks for whole lines of memory: as many 32-byte pieces leave most of
    // the SM's requests in flight empty.
    constexpr int kK = S::kR < 64 ? S::kR / 16 : 4;
    constexpr int kLoad = kK == 1 ? 4 : 8;  // ranks of a load
    const int held = a.rank - a.rank0;      // of a row of B from here on
    auto load_b = [&](int64_t b, int from, uint32_t (&w)[4][2 * kK]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // (Columns past the last take the last one's elements: they are not stored. Ranks past the stored
        // ones take others, which clear_b sets to zero: nothing here waits for a load.)
        const int column = kWhole ? 8 * (row8 / 2) + 2 * j + row8 % 2 : 4 * (2 * j + row8 % 2) + row8 / 2;
        const uint16_t* row = Ba + min(32 * b + column, a.m - 1) * a.rank;
        const int r = from + 4 * kK * quarter;
#pragma unroll
        for (int u = 0; u < 4 * kK / kLoad; ++u) {
          uint32_t* to = &w[j][kLoad / 2 * u];
          if (kLoad == 8 && a.rank_vector == 8) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + min(r + 8 * u, held - 8)));
            to[0] = v.x;
            to[1] = v.y;
            to[kLoad / 2 - 2] = v.z;
            to[kLoad / 2 - 1] = v.w;
          } else if (a.rank_vector) {
#pragma unroll
            for (int h = 0; h < kLoad / 4; ++h) {
              const uint2 v = __ldg(reinterpret_cast<const uint2*>(row + min(r + kLoad * u + 4 * h, held - 4)));
              to[2 * h] = v.x;
              to[2 * h + 1] = v.y;
            }
          } else {
            load_row<kLoad>(*reinterpret_cast<uint32_t(*)[kLoad / 2]>(to), row, r + kLoad * u, rank, rank, false);
          }
        }
      }
    };
    auto clear_b = [&](int from, uint32_t (&w)[4][2 * kK]) {
      if (rank >= from + 16 * kK) return;
      const int keep = rank - from - 4 * kK * quarter;  // of this lane's ranks
#pragma unroll
      for (int i = 0; i < 2 * kK; ++i) {
        const uint32_t mask = 2 * i + 1 < keep ? 0xffffffffu : 2 * i < keep ? 0xffffu : 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j][i] &= mask;
      }
    };
    // y of this lane's rows and columns; the next block's is on its way during a product.
    auto load_y = [&](int64_t b, float4 (&y)[2][2]) {
      const int64_t c0 = 32 * b + first;
      if (!kWhole || c0 + 8 <= a.m) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if ((active | copied) >> (row8 + 8 * h) & 1u) {
            const float* from = a.y + row_of(row8 + 8 * h) * a.y_stride + c0;
            if constexpr (kWhole) {
              y[h][0] = reinterpret_cast<const float4*>(from)[0];
              y[h][1] = reinterpret_cast<const float4*>(from)[1];
            } else {
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = c0 + 4 * i < a.m ? from[4 * i] : 0.0f;
              y[h][0] = make_float4(v[0], v[1], v[2], v[3]);
              y[h][1] = make_float4(v[4], v[5], v[6], v[7]);
            }
          }
        }
      }
    };
    uint32_t w[4][2 * kK];
    float4 yv[2][2], next[2][2];
    constexpr bool kAhead = kNT <= 4;  // (the registers of more ranks leave no room for it)
    if (kAhead && m0 + share < m1 && (active | copied)) load_y(m0 + share, yv);
    for (int64_t b = m0 + share; b < m1 && (active | copied); b += S::kSplit) {
      const int64_t c0 = 32 * b + first;
      const bool vector = kWhole && c0 + 8 <= a.m;
      if (active) load_b(b, 0, w);
      if (!kAhead) load_y(b, yv);
      if (kAhead && b + S::kSplit < m1) load_y(b + S::kSplit, next);
      float acc[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
      for (int k0 = 0; k0 < rank && active; k0 += 16 * kK) {
        if (k0 > 0) load_b(b, k0, w);
        clear_b(k0, w);
        auto times = [&](float by) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] *= by;
          }
        };
        if (kTermUnit != 1.0f && k0 > 0) times(kTermUnit);
#pragma unroll
        for (int t = kTerms - 1; t >= 0; --t) {
#pragma unroll
          for (int k = 0; k < kK; ++k) {
            const uint16_t* from = terms + (t * S::kM + 16 * sub + row8) * S::kStride + k0 + 4 * kK * quarter + 4 * k;
            const uint2 x0 = *reinterpret_cast<const uint2*>(from);
            const uint2 x1 = *reinterpret_cast<const uint2*>(from + 8 * S::kStride);
#pragma unroll
            for (int j = 0; j < 4; ++j) lora_mma<T>(acc[j], x0.x, x1.x, x0.y, x1.y, w[j][2 * k], w[j][2 * k + 1]);
          }
          if (kTermUnit != 1.0f && t == 1) times(1.0f / kTermUnit);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row8 + 8 * h;
        const bool on = active >> r & 1u;
        if (!on && !(copied >> r & 1u)) continue;
        const bool adds = on && rank > 0;  // the other rows are y, bit for bit
        const float by = adds ? unit[16 * sub + r] : 0.0f;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = acc[i / 2][2 * h + i % 2] * by;
        auto sum = [&](float y, int i) { return adds ? y + v[i] : y; };
        float* out = a.out + row_of(r) * a.out_stride + c0;
        if (vector) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float4 from = yv[h][i];
            reinterpret_cast<float4*>(out)[i] =
                make_float4(sum(from.x, 4 * i), sum(from.y, 4 * i + 1), sum(from.z, 4 * i + 2), sum(from.w, 4 * i + 3));
          }
        } else if constexpr (!kWhole) {
          const float y[8] = {yv[h][0].x, yv[h][0].y, yv[h][0].z, yv[h][0].w,
                              yv[h][1].x, yv[h][1].y, yv[h][1].z, yv[h][1].w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (c0 + 4 * i < a.m) out[4 * i] = sum(y[i], i);
          }
        } else {
          const float* y = a.y + row_of(r) * a.y_stride + c0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (c0 + i < a.m) out[i] = sum(y[i], i);
          }
        }
      }
#pragma unroll
      for (int h = 0; kAhead && h < 2; ++h) {
        yv[h][0] = next[h][0];
        yv[h][1] = next[h][1];
      }
    }
    if (rank > 0) {
      if (ctas > 1) cluster.barrier_wait();  // the peers have read this CTA's sums
      __syncthreads();
    }
    if (kSub == 1) return;  // (the grid has a place for every group)
  }
}

template <typename T, int kSub, int kNT, bool kWhole>
cudaError_t launch_lora(const LoraArgs& a, int tiles, int items, int ctas, cudaStream_t stream) {
  using S = LoraShape<kSub, kNT>;
  static bool configured[64] = {};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t err =
        cudaFuncSetAttribute(lora_kernel<T, kSub, kNT, kWhole>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
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
  config.gridDim = dim3(static_cast<unsigned>(tiles) * ctas, static_cast<unsigned>(items));
  config.blockDim = dim3(kLoraThreads);
  config.dynamicSmemBytes = S::kSmem;
  config.stream = stream;
  config.attrs = attr;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, lora_kernel<T, kSub, kNT, kWhole>, a);
}

template <typename T, int kSub, bool kWhole>
cudaError_t launch_rank(const LoraArgs& a, int tiles, int items, int ctas, cudaStream_t s) {
  if (a.taken <= 16) return launch_lora<T, kSub, 2, kWhole>(a, tiles, items, ctas, s);
  if (a.taken <= 32) return launch_lora<T, kSub, 4, kWhole>(a, tiles, items, ctas, s);
  if constexpr (kSub == 1) {
    if (a.taken > 128) return launch_lora<T, kSub, 32, kWhole>(a, tiles, items, ctas, s);
    if (a.taken > 64) return launch_lora<T, kSub, 16, kWhole>(a, tiles, items, ctas, s);
  }
  return launch_lora<T, kSub, 8, kWhole>(a, tiles, items, ctas, s);
}

// Up to 256 rows are taken as a decode batch: as many places for groups as there are rows, a cluster each.
// Clusters of eight CTAs shorten the two passes while there are SMs for them, four take fewer turns after
// that (4096 x 4096, 48 adapters of rank 64, us with eight and with four: 1 row 10.7 and 14.6, 32 rows 15.8
// and 15.5, 64 rows 18.2 and 19.4, 128 rows 29.5 and 21.8; of rank 16: 7.3 and 10.6, 8.7 and 10.5, 10.6
// and 12.1, 17.7 and 13.5).
// (256 rows of one adapter of rank 16, 16 groups: 17 us.)
// More are taken as prompts: two items of a tile at a time, and as many CTAs an item as run at once. That is
// made for runs of one adapter; rows that mix adapters take a tile's items in turn (rows of 48 adapters of
// rank 16: 256 in 21 us, 257 in 291; 257 of one adapter 17). 64 ranks a launch, the later ones adding to
// out: the sums of 64 rows and more ranks leave an SM one CTA and its registers no room for loads in flight
// (2,000 rows of rank 100: 145 us so, 125 us in two launches).
template <typename T, bool kWhole>
cudaError_t launch_tokens(LoraArgs a, cudaStream_t s) {
  if (a.tokens <= kLoraThreads) {
    return launch_rank<T, 1, kWhole>(a, 1, static_cast<int>(a.tokens), a.tokens <= 64 ? 8 : 4, s);
  }
  const int tiles = static_cast<int>((a.tokens + 63) / 64);
  int ctas = kLoraMaxCtas;
  while (ctas > 1 && tiles * ctas > 148 * 2) ctas /= 2;
  for (const int all = a.rank; a.rank0 < all; a.rank0 += 64) {
    a.taken = all - a.rank0 < 64 ? all - a.rank0 : 64;
    if (const cudaError_t err = launch_rank<T, 4, kWhole>(a, tiles, 2, ctas, s); err != cudaSuccess) return err;
    a.y = a.out;
    a.y_stride = a.out_stride;
  }
  return cudaSuccess;
}

}  // namespace

PCK_STATUS_READER(lora_status)

}  // namespace pck

extern "C" int pck_lora_add(const pck_lora_desc* desc, void* stream) {
  using namespace pck;
  if (!desc) return report_error(PCK_ERR_ARGUMENT, "adapters: NULL descriptor");
  const auto& [x, dtype, tokens, n, x_stride, y, m, y_stride, A, B, count, rank, adapters, scales, ranks, out,
               out_stride] = *desc;
  if (dtype != PCK_LOGITS_BF16 && dtype != PCK_LOGITS_F16) {
    return report_error(PCK_ERR_ARGUMENT, "adapters: x must be bfloat16 or float16");
  }
  if (tokens < 0 || tokens > 1 << 30 || n < 1 || m < 0 || !rows_apart(x_stride, n) || !rows_apart(y_stride, m) ||
      out_stride < m) {
    return report_error(PCK_ERR_ARGUMENT, "adapters: need tokens >= 0, n >= 1, m >= 0 and strides of whole rows");
  }
  if (count < 0 || count > 0x7fffffffLL) return report_error(PCK_ERR_ARGUMENT, "adapters: bad number of adapters");
  if (rank < 1 || rank > kLoraMaxRank) return report_error(PCK_ERR_ARGUMENT, "adapters: rank must be in [1, 256]");
  if (tokens == 0 || m == 0) return PCK_OK;
  if (!x || !y || !adapters || !out || (count > 0 && (!A || !B))) {
    return report_error(PCK_ERR_ARGUMENT, "adapters: NULL x, y, A, B, adapters or out");
  }
  LoraArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.y = y;
  a.y_stride = y_stride;
  a.A = A;
  a.B = B;
  a.adapters = adapters;
  a.scales = scales;
  a.ranks = ranks;
  a.out = out;
  a.out_stride = out_stride;
  a.n = n;
  a.m = m;
  a.tokens = tokens;
  a.count = static_cast<int32_t>(count);
  a.rank = a.taken = static_cast<int32_t>(rank);
  a.n_vector = aligned_to(x, 16) && aligned_to(A, 16) && x_stride % 8 == 0 && n % 8 == 0;
  a.rank_vector = aligned_to(B, 16) && rank % 8 == 0 ? 8 : aligned_to(B, 8) && rank % 4 == 0 ? 4 : 0;
  const bool whole = aligned_to(y, 16) && aligned_to(out, 16) && y_stride % 4 == 0 && out_stride % 4 == 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err =
      dtype == PCK_LOGITS_BF16
          ? (whole ? launch_tokens<__nv_bfloat16, true>(a, s) : launch_tokens<__nv_bfloat16, false>(a, s))
          : (whole ? launch_tokens<__half, true>(a, s) : launch_tokens<__half, false>(a, s));
  return err == cudaSuccess ? PCK_OK : report_cuda("adapter kernel", err);
}
