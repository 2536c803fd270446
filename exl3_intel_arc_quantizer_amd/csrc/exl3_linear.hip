// MI355X (gfx950) kernels of products with trellis weights as they are stored:
//
//   linear_turn_kernel    rows of x scaled, transformed and split in float16 parts,
//                         in the order of the matrix instructions' operands
//   linear_rows_kernel    tiles decoded in registers and multiplied, up to 16 rows
//   linear_blocks_kernel  up to 64 rows, 128 of bfloat16
//   linear_wide_kernel    more
//   linear_join_kernel    sums of the shares, transformed and scaled
//
// Weights of (in, out) are tiles W of 16 x 16 codebook values, scales su and sv
// and the orthonormal Sylvester matrix H of order 128, block by block:
//   y = ((x su) H W) H sv.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "../../include/exl3_layer.h"
#include "exl3_cache_layout.h"
#include "exl3_codebook.h"
#include "exl3_errors.h"

using exl3::check_launch;
using exl3::set_error;

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int HAD = 128;
constexpr float ROOT = 0.08838834764831845f;  // 1 / sqrt(128)

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF16>
__device__ __forceinline__ float widen(uint32_t w) {
  if constexpr (BF16) return __builtin_bit_cast(float, w << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)w);
}
template <bool BF16>
__device__ __forceinline__ uint32_t narrow(float v) {
  if constexpr (BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
  return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}

// Two values as float16 parts and what these leave. That is taken from the parts as
// they are stored: where a value is a product the compiler otherwise forms its part
// again, rounded once (v_fma_mixlo_f16), while the stored one is that of the rounded
// product. One value in 8192 lies where they differ, by a whole place of the part.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& parts, uint32_t& rest) {
  parts = pair_of(a, b);
  asm("" : "+v"(parts));
  const f16x2 h = __builtin_bit_cast(f16x2, parts);
  rest = pair_of(a - (float)h[0], b - (float)h[1]);
}

// Scales of a layer: float32, or float16 as they are stored.
struct Scales {
  const void* data;
  int half;
  __device__ __forceinline__ float at(int64_t i) const {
    return half ? (float)static_cast<const _Float16*>(data)[i] : static_cast<const float*>(data)[i];
  }
};

// ------------------------------------------------------------ rows

// The order of a step of 32 input channels: quarter q of a wave's lanes holds
// channels 2 q, 2 q + 1, 2 q + 8, 2 q + 9 of both tiles of 16, which are four
// states next to each other in each tile, a lane's own operand of the decoded
// weights. So z, the transformed rows, lies as [block of rows][step][set][q]
// [16 columns][8]. A set is 16 columns: of up to 8 rows there is one, float16
// parts in columns 0..7 and what they leave in 8..15; else one or (with that
// rest) two for 16 rows.
struct TurnArgs {
  const uint16_t* x;
  int64_t stride;
  const void* su;
  u32x4* z;
  float* scale;                    // [rows]: what z is multiplied by
  int half, k, sets, block_rows;   // of a block of rows
  int rest;                        // where the rest lies behind a value, 0 for none
};

// Channels 2 q, 2 q + 1 of the 16 halves of tiles of a block of 128, times su.
template <bool BF16>
__device__ __forceinline__ void load_unit(const TurnArgs& a, const uint16_t* x, int at, float (&v)[32]) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = *reinterpret_cast<const uint32_t*>(x + at + 8 * i);
  if (a.half) {
    uint32_t s[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.su) + at + 8 * i);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      v[2 * i] = widen<BF16>(w[i] & 0xffffu) * widen<false>(s[i] & 0xffffu);
      v[2 * i + 1] = widen<BF16>(w[i] >> 16) * widen<false>(s[i] >> 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const f32x2 s = *reinterpret_cast<const f32x2*>(static_cast<const float*>(a.su) + at + 8 * i);
      v[2 * i] = widen<BF16>(w[i] & 0xffffu) * s[0];
      v[2 * i + 1] = widen<BF16>(w[i] >> 16) * s[1];
    }
  }
}

// The largest magnitude as bits: NaN above infinity above all numbers.
__device__ __forceinline__ uint32_t top_of(const float (&v)[32]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
  return top;
}

// A row is held as 2^p (hi + lo), both float16, with p from the bound
// |z| <= sqrt(128) max |x su|: 22 bits of a value, and places down to 2^-39 of
// the row's largest one, so the products are as exact as float32 makes them. More
// than 64 bfloat16 rows are held as hi alone, 11 bits, for time: a second part doubles
// the matrix work, which bounds them (2055 rows of 4096 by 12288 258 us so, 491 of two
// parts; the products of 37 rows take half as long as their decoding). What is left
// out is an eighth of the output's own rounding to 8 bits, of both signs like it:
// errors grow by under one per cent. So the 65th row changes what the others of its
// call count with. Float16 outputs, rounded to 11 bits, keep both parts.
// A workgroup takes a row, a quad of lanes a block of 128: two levels across its
// lanes, five within one. A row with an infinity or a NaN is all NaN. Sixteen rows
// share each 256 bytes of z, so the chip's dies, which get workgroups in turn, take
// runs of rows: what they write meets in one cache (the whole product with 4096 rows
// of 4096 by 4096: row by row over the dies 170 us, so 159).
template <bool BF16>
__global__ void __launch_bounds__(1024) linear_turn_kernel(TurnArgs a) {
  __shared__ uint32_t tops[16];
  const int die = blockIdx.x & 7, all = gridDim.x, row = die * (all / 8) + min(die, all % 8) + (int)(blockIdx.x >> 3);
  const int tid = threadIdx.x, q = tid & 3, units = a.k / HAD, step = blockDim.x / 4;
  const uint16_t* x = a.x + row * a.stride;
  float v[32];
  uint32_t top = 0;
  int held = tid >> 2;
  for (int unit = tid >> 2; unit < units; unit += step) {
    load_unit<BF16>(a, x, HAD * unit + 2 * q, v);
    top = max(top, top_of(v));
    held = unit;
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
  for (int i = 0; i < (int)blockDim.x / 64; ++i) top = max(top, tops[i]);
  // The row's values are under 2^11, those of z under 2^15.
  const bool finite = top < 0x7f800000u;
  const int power = max((int)(top >> 23), 1) - 126 - 11;
  if (tid == 0) a.scale[row] = finite ? ldexpf(1.0f, power) : __builtin_nanf("");
  const int block = row / a.block_rows, in_block = row - block * a.block_rows;
  u32x4* out = a.z + (int64_t)block * (a.k / 32) * a.sets * 64 + q * 16 + (in_block & 15) +
               (a.rest == 64 ? 128 : 64) * (in_block >> 4);
  // From the last unit on, which is still held.
  for (int unit = held; unit >= 0 && unit < units; unit -= step) {
    if (unit != held) load_unit<BF16>(a, x, HAD * unit + 2 * q, v);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = ldexpf(v[i], -power);
#pragma unroll
    for (int h = 1; h < 32; h *= 2)
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (!(i & h)) {
          const float y = v[i], w = v[i + h];
          v[i] = y + w, v[i + h] = y - w;
        }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = ROOT * exl3::quad_butterfly<2>(exl3::quad_butterfly<1>(v[i], tid), tid);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u32x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t parts, rest;
        split_pair(v[8 * s + 2 * e], v[8 * s + 2 * e + 1], parts, rest);
        hi[e] = parts, lo[e] = rest;
      }
      u32x4* z = out + (int64_t)(4 * unit + s) * a.sets * 64;
      z[0] = hi;
      if (a.rest) z[a.rest] = lo;
    }
  }
}

// ------------------------------------------------------------ product

struct LinearArgs {
  const uint32_t* words;
  const u32x4* z;
  float* partials;                 // [split][rows][n]
  const float* scale;              // of the rows; null where they are done
  const uint16_t* x;               // the rows themselves, of up to FEW
  int64_t stride;
  const void* su;
  int half_su;
  Scales sv;
  uint16_t* out;
  int rows, k, n, bits, splits;
};

// One butterfly level between lanes 16 or 32 apart, for two registers at once:
// the first swap brings the halves of a pair together, the second puts sums
// and differences back in their lanes.
template <int APART>
__device__ __forceinline__ void lane_butterfly(float& x, float& y) {
  auto swap = [](float& a, float& b) {
    const uint32_t u = __builtin_bit_cast(uint32_t, a), v = __builtin_bit_cast(uint32_t, b);
    const auto r = APART == 16 ? __builtin_amdgcn_permlane16_swap(u, v, false, false)
                               : __builtin_amdgcn_permlane32_swap(u, v, false, false);
    const uint32_t r0 = r[0], r1 = r[1];
    a = __builtin_bit_cast(float, r0), b = __builtin_bit_cast(float, r1);
  };
  swap(x, y);
  const float sum = x + y, difference = x - y;
  x = sum, y = difference;
  swap(x, y);
}

// The values of two states (exl3_codebook.h): the sum of a hash's bytes, scaled,
// or the sum of its halves.
template <int CB>
__device__ __forceinline__ uint32_t values_of(uint32_t s0, uint32_t s1) {
  const uint32_t x0 = hash_state(CB, s0), x1 = hash_state(CB, s1);  // (32-bit products run at full rate)
  if constexpr (CB == 2) {
    const uint32_t sums = __builtin_amdgcn_sad_hi_u8(x1, 0u, __builtin_amdgcn_sad_u8(x0, 0u, 0x64006400u));
    const f16 scale = f16_bits(0x1EEEu), shift = f16_bits(0xC931u);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, sums), f16x2{scale, scale},
                                                                  f16x2{shift, shift}));
  }
  const uint32_t y0 = (x0 & 0x8FFF8FFFu) ^ 0x3B603B60u, y1 = (x1 & 0x8FFF8FFFu) ^ 0x3B603B60u;
  const uint32_t lows = __builtin_amdgcn_perm(y1, y0, 0x05040100u), highs = __builtin_amdgcn_perm(y1, y0, 0x07060302u);
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, lows) + __builtin_bit_cast(f16x2, highs));
}

// A lane's four states of a tile: column n = lane % 16, quarter q = lane / 16
// of the rows, states 4 u .. 4 u + 3 with u = 8 (n % 8) + 2 q + n / 8. They are
// the 16 bits that end 3 K, 2 K, K and 0 bits before bit 4 K (u + 1) of the
// ring: up to K = 5 inside one 32-bit window, beyond in two (WIDE).
struct Window {
  uint32_t at0, at1, shift;        // bytes of its dwords in the tile, and bits past the window
};
__device__ __forceinline__ Window window_of(int end, int bits) {
  Window w;
  const int last = (end - 1) >> 5;
  w.at1 = 4 * last, w.at0 = 4 * (last ? last - 1 : 8 * bits - 1);
  w.shift = 31 - ((end - 1) & 31);
  return w;
}

// The tiles of a step (32 input channels) that a lane decodes, loaded ahead.
template <bool WIDE, int CT>
struct Words {
  uint32_t w[CT][2][WIDE ? 4 : 2];
};

// Two of the four values of a lane's states of a tile (the first, or of H = 1 the
// last), so that decoding can be spread over other work.
template <bool WIDE, int CB, int H>
__device__ __forceinline__ uint32_t half_of(const uint32_t (&w)[WIDE ? 4 : 2], const Window& late, const Window& early, uint32_t bits) {
  if constexpr (WIDE) {
    const uint32_t v = H ? __builtin_amdgcn_alignbit(w[0], w[1], late.shift) : __builtin_amdgcn_alignbit(w[2], w[3], early.shift);
    return values_of<CB>(__builtin_amdgcn_ubfe(v, bits, 16), v & 0xffffu);
  }
  const uint32_t v = __builtin_amdgcn_alignbit(w[0], w[1], late.shift);
  if constexpr (H) return values_of<CB>(__builtin_amdgcn_ubfe(v, bits, 16), v & 0xffffu);
  return values_of<CB>(__builtin_amdgcn_ubfe(v, 3 * bits, 16), __builtin_amdgcn_ubfe(v, 2 * bits, 16));
}

// The four values of a lane's states, of both tiles of a step: its operand.
template <bool WIDE, int CB>
__device__ __forceinline__ u32x4 operand_of(const uint32_t (&w)[2][WIDE ? 4 : 2], const Window& late, const Window& early, uint32_t bits) {
  u32x4 f;
#pragma unroll
  for (int t = 0; t < 2; ++t)
    f[2 * t] = half_of<WIDE, CB, 0>(w[t], late, early, bits), f[2 * t + 1] = half_of<WIDE, CB, 1>(w[t], late, early, bits);
  return f;
}

// Sixteen bytes a lane from memory, `lane_at` bytes past `from`, to shared memory,
// to byte `to` (of the wave's first lane) and on from there. Written out, as the
// compiler would wait for all of these before it reads any shared memory; the waits
// are the caller's (counts of vmcnt, which the compiler's own waits beside them only
// make stricter).
//
// m0, which the text writes, is named as clobbered; the compiler warns that it would
// not keep a reserved register's value across such a statement, which is meant.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_shared(const void* from, uint32_t lane_at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(lane_at), "s"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t shared_byte(const void* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p);
}

// The value of the lane whose number differs in bit X, of rows of 16 lanes.
template <int X>
__device__ __forceinline__ float row_other(float v) {
  if constexpr (X < 4) return exl3::quad_other<X>(v);
  int w = __builtin_bit_cast(int, v);
  if constexpr (X == 4) {                                // 7 - i, then back within quads
    w = __builtin_amdgcn_update_dpp(0, w, 0x141, 0xF, 0xF, true);
    w = __builtin_amdgcn_update_dpp(0, w, 0x1B, 0xF, 0xF, true);
  } else {
    w = __builtin_amdgcn_update_dpp(0, w, 0x128, 0xF, 0xF, true);
  }
  return __builtin_bit_cast(float, w);
}
template <int X>
__device__ __forceinline__ float row_butterfly(float v, int lane) {
  const float o = row_other<X>(v);
  return lane & X ? o - v : v + o;
}

// Up to 16 rows: a wave takes 32 columns and a share of the blocks of 128 input
// channels; a workgroup's eight waves add up in shared memory. Words come through
// shared memory, each wave's own, a block ahead (2 KB at 4 bits), as a lane's dwords
// lie 16 bytes from its neighbour's, and the vector cache then takes four of them at a
// time. One row of 4096 by 4096, 8.4 MB of words, takes 8.9 us in a graph, the join
// with it (in a profiler's trace, each with its own start and end, 6.6 to 6.8 and 3.6):
// launches and the first loads bound it, a wave having one block. Larger weights are
// bound by the instructions of decoding, whatever their bits: 8192 by 28672 at 2, 4 and
// 8 bits (59, 117 and 235 MB) 45, 47 and 51 us, 4096 by 131072 at 4 (268 MB) 87.
//
// FUSED (up to FEW rows): the wave transforms its blocks of the rows itself, two
// channels a lane, with a power of two of their own, which saves a launch; each of
// the n / 32 waves of a block does so, 60 instructions a row where decoding a block
// of 32 columns takes 300. Parts of a row lie in columns r and r + 4 of 8 (each twice
// in 16). Else the rows are read as linear_turn_kernel left them: SETS 1, up to 8
// rows, or 2.
constexpr int FEW = 4;
template <int K, int CB, bool BF16, int SETS, bool FUSED>
__global__ void __launch_bounds__(512) linear_rows_kernel(LinearArgs a) {
  constexpr int CT = 2, WAVES = 8, SEGMENT = CT * 32 * K, WORDS = 8 * SEGMENT, LOADS = (WORDS + 1023) / 1024;
  constexpr int OWN = 2 * WORDS > CT * 1024 ? 2 * WORDS : CT * 1024;  // bytes of a wave: two blocks' words, or its sums
  constexpr bool WIDE = K > 5;
  __shared__ u32x4 held[WAVES * OWN / 16];
  __shared__ u32x4 turned[FUSED ? WAVES * 128 : 1];      // [wave][step][q][column 8]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int column0 = blockIdx.x * CT, split = blockIdx.y;
  const int blocks = a.k / HAD, parts = a.splits * WAVES, part = split * WAVES + wave;
  const int begin = (int)((int64_t)blocks * part / parts), end = (int)((int64_t)blocks * (part + 1) / parts);
  const int n = lane & 15, q = lane >> 4, u = 8 * (n & 7) + 2 * q + (n >> 3);
  const Window late = window_of(4 * K * (u + 1), K), early = window_of(4 * K * u + 2 * K, K);

  const int64_t row_bytes = (int64_t)(a.n / 16) * 32 * K;
  const char* next_words = reinterpret_cast<const char*>(a.words) + 8 * begin * row_bytes + (int64_t)column0 * 32 * K;
  char* own = reinterpret_cast<char*>(held) + wave * OWN;
  const uint32_t own_byte = shared_byte(own);
  uint32_t word_at[LOADS];                               // (row_bytes is at most 2^28)
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int at = 1024 * i + 16 * lane;
    word_at[i] = (uint32_t)(at / SEGMENT * row_bytes + at % SEGMENT);
  }
  auto send = [&](int to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (1024 * i + 16 * lane < WORDS) to_shared(next_words, word_at[i], __builtin_amdgcn_readfirstlane(own_byte + to * WORDS + 1024 * i));
    next_words += 8 * row_bytes;
  };
  // A block's rows: two channels a lane (FUSED), or operands.
  uint32_t xs[FUSED ? FEW : 1];
  f32x2 su;
  u32x4 b[FUSED ? 1 : 4 * SETS];
  auto load = [&](int block) __attribute__((always_inline)) {
    if constexpr (FUSED) {
      const int64_t at = (int64_t)block * HAD + 2 * lane;
      if (a.half_su) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.su) + at);
        su = f32x2{widen<false>(w & 0xffffu), widen<false>(w >> 16)};
      } else {
        su = *reinterpret_cast<const f32x2*>(static_cast<const float*>(a.su) + at);
      }
#pragma unroll
      for (int r = 0; r < FEW; ++r)
        if (r < a.rows) xs[r] = *reinterpret_cast<const uint32_t*>(a.x + r * a.stride + at);
    } else {
      const u32x4* z = a.z + (int64_t)block * (4 * SETS * 64) + lane;
#pragma unroll
      for (int i = 0; i < 4 * SETS; ++i) b[i] = z[i * 64];
    }
  };
  f32x4 total[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) total[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (begin < end) {
    load(begin);
    send(0);
  }
  for (int block = begin; block < end; ++block) {
    const int now = (block - begin) & 1;
    float scale = 0.0f;                                  // of this lane's column
    u32x4* z = turned + wave * 128;
    if constexpr (FUSED) {
      // The dword of a lane's two channels in a column's operand.
      uint32_t* to = reinterpret_cast<uint32_t*>(z + ((lane >> 4) * 4 + (lane & 3)) * 8) + (lane >> 2 & 3);
#pragma unroll
      for (int r = 0; r < FEW; ++r) {
        if (r >= a.rows) break;
        float x = widen<BF16>(xs[r] & 0xffffu) * su[0], y = widen<BF16>(xs[r] >> 16) * su[1];
        // The largest magnitude as bits: NaN above infinity above all numbers.
        uint32_t top = max(__builtin_bit_cast(uint32_t, x) & 0x7fffffffu, __builtin_bit_cast(uint32_t, y) & 0x7fffffffu);
        auto other = [&](float v) { top = max(top, __builtin_bit_cast(uint32_t, v)); };
        other(row_other<1>(__builtin_bit_cast(float, top)));
        other(row_other<2>(__builtin_bit_cast(float, top)));
        other(row_other<4>(__builtin_bit_cast(float, top)));
        other(row_other<8>(__builtin_bit_cast(float, top)));
        top = max(max((uint32_t)__builtin_amdgcn_readlane((int)top, 0), (uint32_t)__builtin_amdgcn_readlane((int)top, 16)),
                  max((uint32_t)__builtin_amdgcn_readlane((int)top, 32), (uint32_t)__builtin_amdgcn_readlane((int)top, 48)));
        // As in linear_turn_kernel: values under 2^11, those of z under 2^15.
        const int power = max((int)(top >> 23), 1) - 126 - 11;
        const float own_scale = top < 0x7f800000u ? ldexpf(1.0f, power) : __builtin_nanf("");
        if ((n & 3) == r) scale = own_scale;
        x = ldexpf(x, -power), y = ldexpf(y, -power);
        const float sum = x + y, difference = x - y;
        x = row_butterfly<8>(row_butterfly<4>(row_butterfly<2>(row_butterfly<1>(sum, lane), lane), lane), lane);
        y = row_butterfly<8>(row_butterfly<4>(row_butterfly<2>(row_butterfly<1>(difference, lane), lane), lane), lane);
        lane_butterfly<16>(x, y);
        lane_butterfly<32>(x, y);
        x *= ROOT, y *= ROOT;
        split_pair(x, y, to[4 * r], to[4 * (r + 4)]);
      }
    }
    // The block's words (and what was loaded before them).
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    u32x4 rows[4 * SETS];
#pragma unroll
    for (int i = 0; i < 4 * SETS; ++i) rows[i] = FUSED ? z[(i * 4 + q) * 8 + (n & 7)] : b[i];
    if (block + 1 < end) {
      load(block + 1);
      send(now ^ 1);
    }
    f32x4 acc[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const char* from = own + now * WORDS;
#pragma unroll
    for (int step = 0; step < 4; ++step)
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        uint32_t w[2][WIDE ? 4 : 2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int place = (2 * step + t) * SEGMENT + c * 32 * K;
          auto word = [&](uint32_t at) { return *reinterpret_cast<const uint32_t*>(from + at + place); };
          w[t][0] = word(late.at0), w[t][1] = word(late.at1);
          if constexpr (WIDE) w[t][2] = word(early.at0), w[t][3] = word(early.at1);
        }
        const u32x4 f = operand_of<WIDE, CB>(w, late, early, K);
#pragma unroll
        for (int s = 0; s < SETS; ++s) acc[c] = mfma(f, rows[step * SETS + s], acc[c]);
      }
#pragma unroll
    for (int c = 0; c < CT; ++c) total[c] += FUSED ? acc[c] * scale : acc[c];
  }
  // A wave's words are read; its sums take their place.
  f32x4* sums = reinterpret_cast<f32x4*>(own);
#pragma unroll
  for (int c = 0; c < CT; ++c) sums[c * 64 + lane] = total[c];
  __syncthreads();
  constexpr int PARTS = FUSED ? 4 : 8;                   // columns between a row's parts
  for (int i = tid; i < CT * 64; i += 64 * WAVES) {
    const int c = i >> 6, l = i & 63, row = l & 15;
    if (row >= a.rows) continue;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const f32x4* of = reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(held) + w * OWN) + c * 64;
      v += of[l];
      if (SETS == 1) v += of[l + PARTS];
    }
    *reinterpret_cast<f32x4*>(a.partials + ((int64_t)split * a.rows + row) * a.n + 16 * (column0 + c) + 4 * (l >> 4)) = v;
  }
}

// Up to 64 rows, or 128 of one part: a workgroup takes all of them, 16 MT, and, eight
// waves, 256 columns, of a share of the input channels. Rows come through shared
// memory for all waves; each wave decodes its own columns, one step ahead of the
// products, and its words come through shared memory as above. 64 rows of 4096 by
// 4096, 21 us: 5 to turn the rows, 12 here, 4 to join 16 shares (four waves of twice
// the columns and 32 shares, which two waves a SIMD hide less of: 30). Latency and the
// vector instructions of decoding bound it: 20 rows of 12288 by 4096 take 27 us, 64
// 33.
//
// In step s rows s + DEPTH + 1 and words s + DEPTH + 2 are sent for, in as many
// instructions each step (past the end the last ones again, which nobody uses), so
// that a step begins when all but those of the last DEPTH steps are there.
template <int K, int CB, int MT, int PARTS>
__global__ void __launch_bounds__(512, 2) linear_blocks_kernel(LinearArgs a) {
  constexpr int CT = 2, SETS = MT * PARTS, DEPTH = 4, AHEAD = 4, HALVES = 4 * CT;
  constexpr int ROWS = SETS * 64, ROW_SLOTS = DEPTH + 2;                     // vectors of a step's rows
  constexpr int SEGMENT = CT * 32 * K, WORDS = 2 * SEGMENT, WORD_SLOTS = DEPTH + 2;  // bytes of a wave's words
  static_assert(SETS <= 8 && WORDS <= 1024, "a step's rows, and a wave's words, are one load of a wave each");
  __shared__ u32x4 rows_held[ROW_SLOTS * ROWS];
  __shared__ u32x4 words_held[8 * WORD_SLOTS * WORDS / 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups are dealt to the chip's eight dies in turn: each die takes a run
  // of them, which share a block of rows in its cache.
  const int all = gridDim.x, die = blockIdx.x & 7;
  const int unit = die * (all / 8) + min(die, all % 8) + (int)(blockIdx.x >> 3);
  const int split = unit % a.splits, group = unit / a.splits;
  const int column0 = (group * 8 + wave) * CT;
  const bool there = column0 < a.n / 16;                 // (waves past the columns read the first ones)
  const int all_steps = a.k / 32;
  const int begin = (int)((int64_t)all_steps * split / a.splits), steps = (int)((int64_t)all_steps * (split + 1) / a.splits) - begin;

  const int64_t row_bytes = (int64_t)(a.n / 16) * 32 * K;
  const char* next_words = reinterpret_cast<const char*>(a.words) + 2 * begin * row_bytes + (int64_t)(there ? column0 : 0) * 32 * K;
  const char* next_rows = reinterpret_cast<const char*>(a.z + (int64_t)begin * ROWS);
  u32x4* own_words = words_held + wave * (WORD_SLOTS * WORDS / 16);
  const uint32_t word_at = (uint32_t)(16 * lane / SEGMENT * row_bytes + 16 * lane % SEGMENT);  // (row_bytes is at most 2^28)
  int rows_sent = 0, words_sent = 0;                     // steps sent for, and places of the next
  const uint32_t rows0 = shared_byte(rows_held + wave * 64), words0 = shared_byte(own_words);
  uint32_t rows_to = rows0, words_to = words0;
  // (A wave past the rows' sets sends for its words twice, so that all count alike.)
  auto send_rows = [&]() __attribute__((always_inline)) {
    if (wave < SETS)
      to_shared(next_rows, 16 * tid, rows_to);
    else if (16 * lane < WORDS)
      to_shared(next_words, word_at, words_to);
    next_rows += ++rows_sent < steps ? 16 * ROWS : 0;
    rows_to = rows_to == rows0 + (ROW_SLOTS - 1) * (16 * ROWS) ? rows0 : rows_to + 16 * ROWS;
  };
  auto send_words = [&]() __attribute__((always_inline)) {
    if (16 * lane < WORDS) to_shared(next_words, word_at, words_to);
    next_words += ++words_sent < steps ? 2 * row_bytes : 0;
    words_to = words_to == words0 + (WORD_SLOTS - 1) * WORDS ? words0 : words_to + WORDS;
  };

  const int n = lane & 15, q = lane >> 4, u = 8 * (n & 7) + 2 * q + (n >> 3);
  const Window late = window_of(4 * K * (u + 1), K), early = window_of(4 * K * u + 2 * K, K);
  constexpr bool WIDE = K > 5;
  int reads = 0;                                         // slot of the words to read next
  Words<WIDE, CT> words;
  auto read_words = [&](const u32x4* from) __attribute__((always_inline)) {
    auto word = [&](uint32_t at, int place) {
      return *reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(from) + at + place);
    };
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int place = t * SEGMENT + c * 32 * K;
        words.w[c][t][0] = word(late.at0, place), words.w[c][t][1] = word(late.at1, place);
        if constexpr (WIDE) words.w[c][t][2] = word(early.at0, place), words.w[c][t][3] = word(early.at1, place);
      }
    reads = reads == WORD_SLOTS - 1 ? 0 : reads + 1;
  };

  f32x4 acc[CT][MT];
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[c][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  send_words();
#pragma unroll
  for (int i = 0; i <= DEPTH; ++i) {
    send_rows();
    send_words();
  }
  u32x4 f[2][CT];
  int slot = 0;                                          // of the rows
  auto wait = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(DEPTH * 2) : "memory");
  };
  wait();
  read_words(own_words);
#pragma unroll
  for (int c = 0; c < CT; ++c) f[0][c] = operand_of<WIDE, CB>(words.w[c], late, early, K);
  auto step = [&](u32x4 (&here)[CT], u32x4 (&next)[CT]) __attribute__((always_inline)) {
    wait();
    const u32x4* rows = rows_held + slot * ROWS + lane;
    slot = slot == ROW_SLOTS - 1 ? 0 : slot + 1;
    u32x4 b[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD && i < SETS; ++i) b[i] = rows[i * 64];
    read_words(own_words + reads * (WORDS / 16));
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      __builtin_amdgcn_sched_barrier(0);
      if (s == 1) send_rows();
      if (s == 2) send_words();
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[c][s / PARTS] = mfma(here[c], b[s % AHEAD], acc[c][s / PARTS]);
      if (s + AHEAD < SETS) b[s % AHEAD] = rows[(s + AHEAD) * 64];
      // This set's share of the next step's halves of tiles: (column tile, tile, half).
#pragma unroll
      for (int of = s * HALVES / SETS; of < (s + 1) * HALVES / SETS; ++of) {
        const int c = of >> 2, t = of >> 1 & 1;
        next[c][of & 3] = of & 1 ? half_of<WIDE, CB, 1>(words.w[c][t], late, early, K)
                                 : half_of<WIDE, CB, 0>(words.w[c][t], late, early, K);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int i = 0; i < steps; i += 2) {
    step(f[0], f[1]);
    if (i + 1 < steps) step(f[1], f[0]);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // nothing on its way into memory that others get
  if (!there) return;
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = 16 * m + (lane & 15), column = 16 * (column0 + c) + 4 * (lane >> 4);
      if (row < a.rows) *reinterpret_cast<f32x4*>(a.partials + ((int64_t)split * a.rows + row) * a.n + column) = acc[c][m];
    }
}

// Many rows: eight waves take 32 SETS rows (of two parts half as many) and 256 columns,
// so two waves share 64 columns, each with half of the rows. Each decodes half of the
// columns' operands, in a step for the next one, and hands them to the other through
// shared memory: vector instructions, four cycles each (and eight of a matrix one's
// sixteen) on a SIMD that two waves share, are then as long as the matrix ones.
// Products begin with a wave's own operands, and rows are read for the next step as
// this one's are used up, so nothing is waited for after the barrier.
//
// 4096 rows of 4096 by 4096, one round of the chip: 159 to 161 us with the rows' turning, 0.86
// PFLOP/s (a library product of 8192 a side reaches 1.21). Of a step's 1.0 us, 0.8 are
// left without decoding and reading: the rate of the matrix instructions bounds it, then
// their overlap with vector ones. 2055 rows of 4096 by 12288, 480 workgroups: 258 us.
template <int K, int CB, bool BF16, int PARTS, int SETS>
__global__ void __launch_bounds__(512, 2) linear_wide_kernel(LinearArgs a) {
  constexpr int MT = SETS / PARTS, DEPTH = 2;            // of a wave
  constexpr int ROWS = 2 * SETS * 64, ROW_SLOTS = DEPTH + 3;                 // vectors of a step's rows
  constexpr int SEGMENT = 2 * 32 * K, WORDS = 2 * SEGMENT, WORD_SLOTS = DEPTH + 2;  // bytes of a wave's words
  constexpr int CHUNK = 8 * 4 * 64;                      // vectors of the eight waves' 16 output rows
  constexpr bool WIDE = K > 5;
  __shared__ u32x4 rows_held[ROW_SLOTS * ROWS > 2 * CHUNK ? ROW_SLOTS * ROWS : 2 * CHUNK];
  __shared__ u32x4 words_held[8 * WORD_SLOTS * WORDS / 16];
  __shared__ u32x4 operands[2][4][4][64];                // [step & 1][column group][column tile]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int side = wave & 1, quarter = wave >> 1;        // half of the rows, 64 columns
  // Workgroups are dealt to the chip's eight dies in turn: each die takes a run
  // of them, which share a block of rows in its cache.
  const int groups = (a.n + 255) / 256, all = gridDim.x, die = blockIdx.x & 7;
  const int unit = die * (all / 8) + min(die, all % 8) + (int)(blockIdx.x >> 3);
  const int split = unit % a.splits, group = unit / a.splits % groups, block = unit / a.splits / groups;
  const int column0 = (group * 4 + quarter) * 4;
  const bool there = column0 < a.n / 16;                 // (waves past the columns read the first ones)
  const int all_steps = a.k / 32;
  const int begin = (int)((int64_t)all_steps * split / a.splits), steps = (int)((int64_t)all_steps * (split + 1) / a.splits) - begin;

  const int64_t row_bytes = (int64_t)(a.n / 16) * 32 * K;
  const char* next_words = reinterpret_cast<const char*>(a.words) + 2 * begin * row_bytes + (int64_t)((there ? column0 : 0) + 2 * side) * 32 * K;
  const uint32_t word_at = (uint32_t)(16 * lane / SEGMENT * row_bytes + 16 * lane % SEGMENT);  // (row_bytes is under 2^29)
  const char* next_rows = reinterpret_cast<const char*>(a.z + ((int64_t)block * all_steps + begin) * ROWS);
  u32x4* own_words = words_held + wave * (WORD_SLOTS * WORDS / 16);
  // What is sent for next, and its places in shared memory.
  int sent = 0;
  const uint32_t rows0 = shared_byte(rows_held + wave * 64), words0 = shared_byte(own_words);
  uint32_t rows_to = rows0, words_to = words0;
  // A step's rows are two of each thread, or of the second some waves have none and
  // send for their words twice, so that all count alike.
  static_assert(ROWS > 512 && ROWS <= 2 * 512 && 2 * SETS >= 12, "two of a thread; decoding takes eleven places of a step");
  auto send = [&](int part) __attribute__((always_inline)) {
    if (part == 0 || (part == 1 && wave < 2 * SETS - 8)) {
      to_shared(next_rows + part * 8192, 16 * tid, rows_to + part * 8192);
      return;
    }
    if (16 * lane < WORDS) to_shared(next_words, word_at, words_to);
    if (part == 1) return;
    const bool on = ++sent < steps;
    next_rows += on ? 16 * ROWS : 0, next_words += on ? 2 * row_bytes : 0;
    rows_to = rows_to == rows0 + (ROW_SLOTS - 1) * (16 * ROWS) ? rows0 : rows_to + 16 * ROWS;
    words_to = words_to == words0 + (WORD_SLOTS - 1) * WORDS ? words0 : words_to + WORDS;
  };
  // All but what the last DEPTH steps sent for.
  auto wait = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(DEPTH * 3) : "memory");
  };

  const int n = lane & 15, q = lane >> 4, u = 8 * (n & 7) + 2 * q + (n >> 3);
  const Window late = window_of(4 * K * (u + 1), K), early = window_of(4 * K * u + 2 * K, K);
  int read_slot = 0, slot = 0;
  Words<WIDE, 2> words;
  auto read_words = [&]() __attribute__((always_inline)) {
    const char* from = reinterpret_cast<const char*>(own_words) + read_slot * WORDS;
    auto word = [&](uint32_t at, int place) { return *reinterpret_cast<const uint32_t*>(from + at + place); };
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int place = t * SEGMENT + c * 32 * K;
        words.w[c][t][0] = word(late.at0, place), words.w[c][t][1] = word(late.at1, place);
        if constexpr (WIDE) words.w[c][t][2] = word(early.at0, place), words.w[c][t][3] = word(early.at1, place);
      }
    read_slot = read_slot == WORD_SLOTS - 1 ? 0 : read_slot + 1;
  };

  f32x4 acc[4][MT];                                      // of this wave's operands, then the other's
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[j][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < DEPTH + 2; ++i) send(0), send(1), send(2);
  wait();
  u32x4 f[2][2], b[SETS];
  read_words();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    f[0][c] = operand_of<WIDE, CB>(words.w[c], late, early, K);
    operands[0][quarter][2 * side + c][lane] = f[0][c];
  }
#pragma unroll
  for (int s = 0; s < SETS; ++s) b[s] = rows_held[(side * SETS + s) * 64 + lane];

  auto step = [&](u32x4 (&here)[2], u32x4 (&next)[2], int parity) __attribute__((always_inline)) {
    wait();
    slot = slot == ROW_SLOTS - 1 ? 0 : slot + 1;
    const u32x4* coming = rows_held + slot * ROWS + side * (SETS * 64) + lane;
    u32x4 other[2];
#pragma unroll
    for (int s = 0; s < 2 * SETS; ++s) {
      const int set = s % SETS;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        f32x4& sum = acc[s / SETS * 2 + c][set / PARTS];
        sum = mfma(s < SETS ? here[c] : other[c], b[set], sum);
      }
      if (s == 0) read_words();
      if (s == 1)
#pragma unroll
        for (int c = 0; c < 2; ++c) other[c] = operands[parity][quarter][2 * (side ^ 1) + c][lane];
      if (s >= 1 && s < 4) send(s - 1);
      if (s >= SETS) b[set] = coming[set * 64];
      // The next step's eight halves of tiles, (column tile, tile, half).
      if (s >= 3 && s < 11) {
        const int of = s - 3, c = of >> 2, t = of >> 1 & 1;
        next[c][of & 3] = of & 1 ? half_of<WIDE, CB, 1>(words.w[c][t], late, early, K) : half_of<WIDE, CB, 0>(words.w[c][t], late, early, K);
      }
      if (s == 7 || s == 11) operands[parity ^ 1][quarter][2 * side + s / 8][lane] = next[s / 8];
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int i = 0; i < steps; i += 2) {
    step(f[0], f[1], 0);
    if (i + 1 < steps) step(f[1], f[0], 1);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // nothing on its way into memory that is used again below

  const int row0 = (2 * block + side) * 16 * MT + (lane & 15);
  auto column_of = [&](int j) { return 16 * (column0 + (j < 2 ? 2 * side + j : 2 * (side ^ 1) + j - 2)) + 4 * (lane >> 4); };
  if (a.splits > 1) {
    if (!there) return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if (row0 + 16 * m < a.rows)
          *reinterpret_cast<f32x4*>(a.partials + ((int64_t)split * a.rows + row0 + 16 * m) * a.n + column_of(j)) = acc[j][m];
    return;
  }
  // The output's transform: a lane holds channels 4 (lane / 16) .. + 3 of its tiles,
  // so two levels lie in its registers, two across lanes, two across the four tiles,
  // and one across the waves of 64 columns beside each other.
  f32x4* exchange = reinterpret_cast<f32x4*>(rows_held);  // two chunks of it
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x4& v = acc[j][m];
      const float s0 = v[0] + v[1], s1 = v[0] - v[1], s2 = v[2] + v[3], s3 = v[2] - v[3];
      float y[4] = {s0 + s2, s1 + s3, s0 - s2, s1 - s3};
      lane_butterfly<16>(y[0], y[1]);
      lane_butterfly<16>(y[2], y[3]);
      lane_butterfly<32>(y[0], y[1]);
      lane_butterfly<32>(y[2], y[3]);
      v = f32x4{y[0], y[1], y[2], y[3]};
    }
    const f32x4 s0 = acc[0][m] + acc[1][m], s1 = acc[0][m] - acc[1][m], s2 = acc[2][m] + acc[3][m], s3 = acc[2][m] - acc[3][m];
    // The tiles of side 0 come first.
    const f32x4 d0 = side ? s2 - s0 : s0 - s2, d1 = side ? s3 - s1 : s1 - s3;
    acc[0][m] = side ? d0 : s0 + s2, acc[1][m] = side ? d1 : s1 + s3;
    acc[2][m] = side ? s0 + s2 : d0, acc[3][m] = side ? s1 + s3 : d1;
    // Two chunks take turns: a wave writes one after its partner has read the other.
    f32x4* held = exchange + (m & 1) * CHUNK;
    if (m == 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) held[(wave * 4 + j) * 64 + lane] = acc[j][m];
    __syncthreads();
    const int row = row0 + 16 * m;
    const bool writes = there && row < a.rows;
    const float scale = writes ? a.scale[row] * ROOT : 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int column = column_of(j);
      const f32x4 other = held[((wave ^ 2) * 4 + j) * 64 + lane];
      const f32x4 v = quarter & 1 ? other - acc[j][m] : acc[j][m] + other;
      if (writes) {
        u32x2 w;
        w[0] = narrow<BF16>(v[0] * scale * a.sv.at(column)) | narrow<BF16>(v[1] * scale * a.sv.at(column + 1)) << 16;
        w[1] = narrow<BF16>(v[2] * scale * a.sv.at(column + 2)) | narrow<BF16>(v[3] * scale * a.sv.at(column + 3)) << 16;
        *reinterpret_cast<u32x2*>(a.out + (int64_t)row * a.n + column) = w;
      }
    }
  }
}

// ------------------------------------------------------------ join

struct JoinArgs {
  const float *partials, *scale;
  Scales sv;
  uint16_t* out;
  int rows, n, splits;
};

// A wave takes a block of 128 outputs of a row, eight a lane; its four rows of
// lanes take shares in turn, as their loads wait for each other (16 shares of 64 rows
// of 4096: 4 us; sixteen lanes a block, shares one after another, 7.8).
template <bool BF16>
__global__ void __launch_bounds__(256) linear_join_kernel(JoinArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const int lane = threadIdx.x & 63, blocks = a.n / HAD;
  if (unit >= (int64_t)a.rows * blocks) return;
  const int row = (int)(unit / blocks), column = (int)(unit % blocks) * HAD + 8 * (lane & 15);
  float v[8] = {};
  for (int s = lane >> 4; s < a.splits; s += 16) {
    f32x4 x[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4* p = reinterpret_cast<const f32x4*>(a.partials + ((int64_t)min(s + 4 * i, a.splits - 1) * a.rows + row) * a.n + column);
      x[i][0] = p[0], x[i][1] = p[1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += s + 4 * i < a.splits ? x[i][e / 4][e % 4] : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] += __shfl_xor(v[e], 16);
    v[e] += __shfl_xor(v[e], 32);
  }
  exl3::quad_transform(v, lane);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = row_butterfly<8>(row_butterfly<4>(v[e], lane), lane);
  if (lane >= 16) return;
  const float scale = (a.scale ? a.scale[row] : 1.0f) * ROOT;
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = narrow<BF16>(v[2 * e] * scale * a.sv.at(column + 2 * e)) |
           narrow<BF16>(v[2 * e + 1] * scale * a.sv.at(column + 2 * e + 1)) << 16;
  *reinterpret_cast<u32x4*>(a.out + (int64_t)row * a.n + column) = w;
}

// ------------------------------------------------------------ plan

// Variants by the rows.
enum Variant { ROWS_FEW, ROWS8, ROWS16, BLOCK32, BLOCK48, BLOCK64, BLOCK128, BLOCK_WIDE };
constexpr int BLOCK_ROWS[] = {FEW, 8, 16, 32, 48, 64, 128};

// How a call is cut: the variant of the fewest rows that takes them all (two float16
// parts). Times in a graph, us, of the one chosen and of the next larger one, at 4
// bits: 1 row of 4096 by 4096 9.0 and 12.3, 4 rows 10.2 and 12.5; 8 rows of 4096 by
// 12288 17.0 and 18.5; 16 rows of 12288 by 4096 23.7 and 26.2; 32 rows of 4096 by 4096
// 16.1 and 16.5; 48 rows of 4096 by 12288 30.1 and 30.8; 64 rows of 4096 by 4096
// (float16) 20.8 and 28.7; 128 rows (bfloat16) 27.2 and 32.8. Of larger weights 2 to 4
// rows would gain by the variant of 8, whose waves do not each turn the rows: 4 rows of
// 4096 by 12288 17.7 and 16.7; 2 and 4 rows of 8192 by 28672 53 and 66, and 45.
struct Plan {
  Variant variant;
  int parts;                       // float16 parts of a value: 2, or 1 of more than 64 bfloat16 rows
  int block_rows, blocks, sets;    // rows of a block, blocks, sets of a block
  int groups, splits;              // column groups, shares of the input channels
  int64_t z_bytes, scale_bytes, partial_bytes;
};

constexpr int CUS = 256;

// Threads of linear_turn_kernel, by its rows' blocks of 128, four each.
int turn_threads(int64_t k) { return k <= 4096 ? 128 : k <= 8192 ? 256 : k <= 16384 ? 512 : 1024; }

Plan plan_of(int64_t rows, int64_t k, int64_t n, bool bf16) {
  Plan p{};
  p.variant = ROWS_FEW;
  while (p.variant < BLOCK_WIDE && rows > BLOCK_ROWS[p.variant]) p.variant = (Variant)(p.variant + 1);
  if (p.variant == BLOCK128 && !bf16) p.variant = BLOCK_WIDE;
  p.parts = p.variant >= BLOCK128 && bf16 ? 1 : 2;
  // Shares of the input channels that fill the chip: a wave of linear_rows_kernel
  // takes at least one block of 128, a workgroup of linear_blocks_kernel too; one of
  // linear_wide_kernel at least 640 channels, as the shares' sums go through memory
  // (300 rows of 4096 by 4096 in shares of 384, 640 and 1024 channels at least: 48, 44
  // and 48 us; in float16 47 each, at 1280 53). Fewer workgroups would take smaller
  // ones: 200 rows 36, 40 and 44, 130 rows 30, 34 and 40, 520 of 4096 by 1024 35, 40
  // and 46.
  const bool few = p.variant <= ROWS16;
  p.groups = (int)(few ? n / 32 : (n + 255) / 256);
  const int64_t most = std::max<int64_t>(1, few ? k / (8 * HAD) : p.variant == BLOCK_WIDE ? k / (5 * HAD) : k / HAD);
  auto cut = [&](int64_t block_rows) {
    p.block_rows = (int)block_rows, p.blocks = (int)((rows + block_rows - 1) / block_rows);
    p.splits = (int)std::min(most, std::max<int64_t>(1, (few ? 4 : 1) * CUS / ((int64_t)p.groups * p.blocks)));
  };
  if (p.variant < BLOCK_WIDE) {
    cut(BLOCK_ROWS[p.variant]);
  } else {
    // Blocks of 8, 7 or 6 sets (of two parts, 8 or 6) by the time of the last
    // workgroup: rounds of the chip, times a step, which takes as long as the products
    // of its sets and about two more, over the shares. (2055 rows of 4096 by 12288:
    // 8 sets 265 us, 7 254, 6 344; 300 rows of 4096 by 4096: 51, 47, 44; 4096 rows: 162,
    // 256, 242; two parts, 520 rows of 4096 by 12288: 8 sets 130, 6 210. The sums of more
    // shares are not counted: 200 rows of 4096 by 4096 39, 38, 41.)
    int64_t least = INT64_MAX, best = 8;
    for (int64_t sets = 8; sets >= 6; sets -= p.parts) {
      cut(32 * sets / p.parts);
      const int64_t rounds = ((int64_t)p.groups * p.blocks * p.splits + CUS - 1) / CUS;
      const int64_t cost = rounds * (sets + 2) * 1024 / p.splits;
      if (cost < least) least = cost, best = sets;
    }
    cut(32 * best / p.parts);
  }
  p.sets = p.variant == ROWS_FEW ? 0 : p.block_rows * p.parts / 16;
  p.z_bytes = k / 32 * p.sets * 1024 * p.blocks;
  p.scale_bytes = p.variant == ROWS_FEW ? 0 : (4 * rows + 15) & ~(int64_t)15;
  const bool direct = p.variant == BLOCK_WIDE && p.splits == 1;
  p.partial_bytes = direct ? 0 : 4 * (int64_t)p.splits * rows * n;
  return p;
}

template <int K, int CB, bool BF16>
void launch_product(const Plan& p, const LinearArgs& a, hipStream_t stream) {
  const dim3 grid(p.groups, p.splits);
  const unsigned all = (unsigned)(p.groups * p.splits * p.blocks);
  switch (p.variant) {
    case ROWS_FEW: linear_rows_kernel<K, CB, BF16, 1, true><<<grid, 512, 0, stream>>>(a); break;
    case ROWS8: linear_rows_kernel<K, CB, false, 1, false><<<grid, 512, 0, stream>>>(a); break;
    case ROWS16: linear_rows_kernel<K, CB, false, 2, false><<<grid, 512, 0, stream>>>(a); break;
    case BLOCK32: linear_blocks_kernel<K, CB, 2, 2><<<all, 512, 0, stream>>>(a); break;
    case BLOCK48: linear_blocks_kernel<K, CB, 3, 2><<<all, 512, 0, stream>>>(a); break;
    case BLOCK64: linear_blocks_kernel<K, CB, 4, 2><<<all, 512, 0, stream>>>(a); break;
    case BLOCK128: linear_blocks_kernel<K, CB, 8, 1><<<all, 512, 0, stream>>>(a); break;
    case BLOCK_WIDE:
      if constexpr (BF16) {
        if (p.block_rows == 224) {
          linear_wide_kernel<K, CB, true, 1, 7><<<all, 512, 0, stream>>>(a);
          break;
        }
      }
      if (p.block_rows * p.parts == 192)
        linear_wide_kernel<K, CB, BF16, BF16 ? 1 : 2, 6><<<all, 512, 0, stream>>>(a);
      else
        linear_wide_kernel<K, CB, BF16, BF16 ? 1 : 2, 8><<<all, 512, 0, stream>>>(a);
      break;
  }
}
template <int CB, bool BF16>
void launch_rate(const Plan& p, const LinearArgs& a, hipStream_t stream) {
  switch (a.bits) {
    case 1: launch_product<1, CB, BF16>(p, a, stream); break;
    case 2: launch_product<2, CB, BF16>(p, a, stream); break;
    case 3: launch_product<3, CB, BF16>(p, a, stream); break;
    case 4: launch_product<4, CB, BF16>(p, a, stream); break;
    case 5: launch_product<5, CB, BF16>(p, a, stream); break;
    case 6: launch_product<6, CB, BF16>(p, a, stream); break;
    case 7: launch_product<7, CB, BF16>(p, a, stream); break;
    default: launch_product<8, CB, BF16>(p, a, stream); break;
  }
}

template <bool BF16>
int launch_linear(const Plan& p, const TurnArgs& t, const LinearArgs& a, int cb, hipStream_t s) {
  if (p.variant != ROWS_FEW) {
    linear_turn_kernel<BF16><<<(unsigned)a.rows, turn_threads(t.k), 0, s>>>(t);
    if (check_launch("exl3_linear")) return 1;
  }
  cb == 0 ? launch_rate<0, BF16>(p, a, s) : cb == 1 ? launch_rate<1, BF16>(p, a, s) : launch_rate<2, BF16>(p, a, s);
  if (check_launch("exl3_linear")) return 1;
  if (!p.partial_bytes) return 0;
  JoinArgs j{};
  j.partials = a.partials, j.scale = a.scale, j.sv = a.sv, j.out = a.out, j.rows = a.rows, j.n = a.n, j.splits = p.splits;
  const int64_t units = (int64_t)a.rows * (a.n / HAD);
  linear_join_kernel<BF16><<<(unsigned)((units + 3) / 4), 256, 0, s>>>(j);
  return check_launch("exl3_linear");
}

}  // namespace

extern "C" {

int64_t exl3_linear_workspace(int64_t rows, int64_t k, int64_t n, int type) {
  if (rows < 0 || rows > 1 << 22 || k < HAD || n < HAD || k % HAD || n % HAD || k > 1 << 24 || n > 1 << 24) return -1;
  if (rows * turn_threads(k) > UINT32_MAX) return -1;    // a launch has fewer than 2^32 threads
  if (!rows) return 0;
  const Plan p = plan_of(rows, k, n, type == 2);
  return p.z_bytes + p.scale_bytes + p.partial_bytes;
}

int exl3_linear(const void* x, int64_t stride, int64_t rows, int type, const uint16_t* words, const void* su,
                const void* sv, int half_scales, int64_t k, int64_t n, int K, int cb, void* out, void* workspace,
                int64_t workspace_bytes, void* stream) {
  if (K < 1 || K > 8) return set_error("exl3_linear: K must be in 1..8, got %d", K);
  if (cb < 0 || cb > 2) return set_error("exl3_linear: cb must be 0, 1, or 2, got %d", cb);
  if (type < 1 || type > 2) return set_error("exl3_linear: rows are float16 or bfloat16");
  const int64_t need = exl3_linear_workspace(rows, k, n, type);
  if (need < 0) return set_error("exl3_linear: bad sizes: %lld rows of %lld by %lld", (long long)rows, (long long)k, (long long)n);
  if (!rows) return 0;
  if ((reinterpret_cast<uintptr_t>(x) & 15) || stride % 8 || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15) || (reinterpret_cast<uintptr_t>(words) & 15) ||
      (reinterpret_cast<uintptr_t>(su) & 15) || (reinterpret_cast<uintptr_t>(sv) & 15))
    return set_error("exl3_linear: all memory must be 16-byte aligned");
  if (workspace_bytes < need) return set_error("exl3_linear: workspace of %lld bytes is too small", (long long)workspace_bytes);
  const Plan p = plan_of(rows, k, n, type == 2);
  char* w = static_cast<char*>(workspace);
  TurnArgs t{};
  t.x = static_cast<const uint16_t*>(x), t.stride = stride, t.su = su, t.half = half_scales & 1;
  t.z = reinterpret_cast<u32x4*>(w), t.scale = reinterpret_cast<float*>(w + p.z_bytes);
  t.k = (int)k, t.sets = p.sets, t.block_rows = p.block_rows;
  t.rest = p.variant == ROWS8 ? 8 : p.parts == 2 ? 64 : 0;
  LinearArgs a{};
  a.words = reinterpret_cast<const uint32_t*>(words), a.z = t.z, a.scale = p.scale_bytes ? t.scale : nullptr;
  a.x = t.x, a.stride = stride, a.su = su, a.half_su = t.half, a.sv = {sv, half_scales >> 1 & 1};
  a.out = static_cast<uint16_t*>(out), a.partials = reinterpret_cast<float*>(w + p.z_bytes + p.scale_bytes);
  a.rows = (int)rows, a.k = (int)k, a.n = (int)n, a.bits = K, a.splits = p.splits;
  auto launch = type == 2 ? launch_linear<true> : launch_linear<false>;
  return launch(p, t, a, cb, (hipStream_t)stream);
}

}  // extern "C"
