// The 4-bit attention cache in memory, and the group transform, shared by the
// kernels that write, read and attend over it.
//
// Pages of P tokens (a power of two, 32 to 256) of every kv head: P / 32 tiles
// of one head's 32 tokens, 36 D bytes each, so a tile that a wave attends over
// is one run of memory: 16 D bytes of key codes, 16 D of value codes, 2 D of
// key scales, 2 D of value scales. The head dimension D is split in groups of
// 32 values; a group x is held as y = H x / 8 (H the Sylvester matrix of
// order 32, so one large channel spreads over its group), a scale
// s = f16(bf16(max|y| / 7)) and codes c = clamp(rint(y / s), -7, 7) + 8, and
// stands for H ((c - 8) s) / 4. Both factors are powers of two: with five
// levels of sums in a fixed order the transform rounds the same everywhere. s
// has eight significant bits and c - 8 three, so (c - 8) s is exact in f16 and
// the matrix cores see the very values that the codes stand for. At 9344,
// the largest scale, 7 s is still finite. A group with an infinity or a NaN
// holds a NaN scale: all its values are NaN when read.
//
// The order inside a tile follows the 16 x 16 x 32 matrix instructions:
//   key codes    dword [token][j][group], j = 0..3: dims 32 group + 8 j .. + 7.
//                A lane of row `token` and quarter j reads its operands of all
//                groups as one load. Nibble u holds dim 2 u (u < 4) or
//                2 (u - 4) + 1: masking a dword shifted by 4 u leaves dims 2 u
//                and 2 u + 1 in the two halves.
//   value codes  dword [octet][r][token & 7], octet = token / 8: dims 8 r ..
//                8 r + 7 in nibble order. A lane reads eight tokens of one
//                dword column, the token axis of its operands, as 32 bytes.
//   key scales   f16 [token][group]
//   value scales f16 [octet][group][token & 7]
// A token's dwords and scales are its own: appending writes no byte of
// another token.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace exl3 {

constexpr int CACHE_TILE = 32;      // tokens of a tile, and values of a group
constexpr int CACHE_MAX_REQUESTS = 4096;

struct CacheShape {
  int64_t pages;
  int kv_heads, head_dim;
  int tile_shift;                   // log2 of the tiles of a page
};

__host__ __device__ inline int64_t cache_tile_bytes(int d) { return 36 * (int64_t)d; }

// Byte offset of a tile.
__device__ __forceinline__ int64_t cache_tile_at(const CacheShape& c, int64_t page, int head,
                                                 int tile) {
  return ((((page * c.kv_heads + head) << c.tile_shift) + tile)) * cache_tile_bytes(c.head_dim);
}

// One butterfly level across lanes of a quad: the lane whose bit is clear
// keeps the sum, the other the difference. Bits 1 and 2 of the lane number
// are quad permutations.
template <int BIT>
__device__ __forceinline__ float quad_other(float v) {
  static_assert(BIT == 1 || BIT == 2, "a lane of the quad");
  constexpr int PERM = BIT == 1 ? 0xB1 : 0x4E;  // 1,0,3,2 and 2,3,0,1
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), PERM,
                                                               0xF, 0xF, true));
}
template <int BIT>
__device__ __forceinline__ float quad_butterfly(float v, int lane) {
  const float o = quad_other<BIT>(v);
  return lane & BIT ? o - v : v + o;
}

// Levels 1, 2 and 4 of eight consecutive values of a lane.
__device__ __forceinline__ void butterfly8(float (&v)[8]) {
#pragma unroll
  for (int h = 1; h < 8; h *= 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!(i & h)) {
        const float a = v[i], b = v[i + h];
        v[i] = a + b;
        v[i + h] = a - b;
      }
    }
  }
}

// H v for the group that a quad of lanes holds, eight consecutive values each.
__device__ __forceinline__ void quad_transform(float (&v)[8], int lane) {
  butterfly8(v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = quad_butterfly<1>(v[i], lane);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = quad_butterfly<2>(v[i], lane);
}

}  // namespace exl3
