// The 4-bit key/value cache: where a code and its scale lie (documented in include/pck_b200.h).
//
// A cache is (pages, kv_heads, page_tiles, 18 * dim) bytes. A tile holds 16 consecutive tokens of
// one head: 8 * dim bytes of key codes, dim bytes of key scales, then the same of the values. It is
// one contiguous piece whatever the page size, so a tile is one bulk copy. Channels go in groups of
// 64 that share a (scale, zero) pair of bfloat16 per token; x = code * scale + zero.
//
// The order of the codes inside a tile is the order in which the matrix instructions of the
// attention take them, so a lane reads its operands with 16-byte loads that meet no bank twice:
//   - keys: lane (token, quarter) takes the 16 channels of its quarter in each group;
//   - values: lane (channel / 8, token / 2) takes two tokens' codes of the same four channels as
//     the two halves of a 32-bit word, so a shift and a mask give a pair along the token axis.
// Groups are paired in planes of 128 channels (one plane of 64 for dim 64).
#pragma once

#include <cstdint>

namespace pck {

constexpr int kKv4Tile = 16;   // tokens of a tile
constexpr int kKv4Group = 64;  // channels that share a scale and a zero

__host__ __device__ constexpr int kv4_groups(int dim) { return dim / kKv4Group; }
__host__ __device__ constexpr int kv4_plane_groups(int dim) { return dim > kKv4Group ? 2 : 1; }
__host__ __device__ constexpr int kv4_tile_bytes(int dim) { return 18 * dim; }

// Offsets in a tile of the byte that holds channels c and c + 1 (c even; c in the low bits).
__host__ __device__ constexpr int kv4_key_byte(int dim, int token, int c) {
  const int w = kv4_plane_groups(dim);
  const int plane = c / (kKv4Group * w), group = c / kKv4Group % w, i = c % kKv4Group;
  return plane * 512 * w + token * 32 * w + i / 16 * 8 * w + group * 8 + i % 16 / 2;
}

__host__ __device__ constexpr int kv4_value_byte(int dim, int token, int c) {
  const int w = kv4_plane_groups(dim);
  const int plane = c / (kKv4Group * w), group = c / kKv4Group % w, i = c % kKv4Group;
  return 9 * dim + plane * 512 * w + token / 8 * 256 * w + i / 8 * 32 * w + token % 8 / 2 * 8 * w + group * 8 +
         i % 8 / 4 * 4 + token % 2 * 2 + i % 4 / 2;
}

// Offsets of a token's (scale, zero) pair of a group.
__host__ __device__ constexpr int kv4_key_scale(int dim, int token, int group) {
  return 8 * dim + (token * kv4_groups(dim) + group) * 4;
}

__host__ __device__ constexpr int kv4_value_scale(int dim, int token, int group) {
  return 17 * dim + (token * kv4_groups(dim) + group) * 4;
}

}  // namespace pck
