// MI355X (gfx950) kernels of attention over the 4-bit cache of
// exl3_cache_layout.h:
//
//   attend_rows_kernel  a few query rows of one kv head against a share of its
//                       tiles, as partial or whole results
//   attend_join_kernel  the partial results of a row joined, empty rows zeroed
//
// Row i of a request's n new tokens sits at position p = length - n + i and
// attends positions max(0, p - window + 1) .. p:
//   out = sum_t softmax_t(scale q . k_t) v_t,
// 0 where nothing is attended. Groups are held as y = H x / 8 and stand for
// H y / 4, and H H = 32, so q . k = 2 (H q / 8) . (H k / 8): queries are
// transformed once, keys and values never, and an output row is taken back
// once.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "../../include/exl3_layer.h"
#include "exl3_cache_layout.h"
#include "exl3_errors.h"

using exl3::CACHE_MAX_REQUESTS;
using exl3::CACHE_TILE;
using exl3::CacheShape;
using exl3::check_launch;
using exl3::set_error;

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float NONE = -__builtin_inff();
constexpr int THREADS = 256, WAVES = THREADS / 64;

struct AttendArgs {
  const uint16_t* q;
  uint16_t* out;                 // (tokens, q_heads, D) contiguous
  const uint8_t* pages;
  const int32_t *tables, *starts, *lengths;
  float* partials;               // [2 grid][rows][D + 2]: values, then maximum and sum
  int64_t* shares;               // [requests + 1] prefix of the work, for the join
  int64_t q_token, q_head, tokens, window;
  CacheShape cache;
  int requests, width, q_heads, group, grid;
  int least;                     // tiles a workgroup takes at least
  float scale;
};

// What a request asks for, every figure bounded by the arrays' sizes whatever
// the device arrays hold.
struct Request {
  int first, n;                  // its rows of q
  int length;                    // positions held
  int tile0, tiles;              // tiles that some row attends
};
__device__ __forceinline__ Request request_of(const AttendArgs& a, int r) {
  const int64_t s0 = min(max((int64_t)a.starts[r], (int64_t)0), a.tokens);
  const int64_t s1 = min(max((int64_t)a.starts[r + 1], s0), a.tokens);
  const int64_t room = ((int64_t)a.width << a.cache.tile_shift) * CACHE_TILE;
  const int64_t length = min(max((int64_t)a.lengths[r], (int64_t)0), room);
  const int64_t low = max(length - (s1 - s0) - a.window + 1, (int64_t)0);
  Request q;
  q.first = (int)s0, q.n = (int)(s1 - s0), q.length = (int)length;
  q.tile0 = (int)(low / CACHE_TILE);
  q.tiles = q.n ? (int)((length + CACHE_TILE - 1) / CACHE_TILE) - q.tile0 : 0;
  return q;
}

// Tiles of work of a request: its tiles, for every kv head and block of ROWS
// query rows.
template <int ROWS>
__device__ __forceinline__ int64_t work_of(const AttendArgs& a, const Request& q) {
  const int64_t blocks = ((int64_t)q.n * a.group + ROWS - 1) / ROWS;
  return blocks * a.cache.kv_heads * q.tiles;
}

// prefix[r] = work before request r, prefix[requests] = all of it.
template <int ROWS>
__device__ __forceinline__ void sum_work(const AttendArgs& a, int64_t* prefix, int64_t* parts) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t base = 0;
  for (int r0 = 0; r0 < a.requests; r0 += THREADS) {
    const int r = r0 + tid;
    int64_t v = r < a.requests ? work_of<ROWS>(a, request_of(a, r)) : 0;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int64_t w = __shfl_up(v, o);
      if (lane >= o) v += w;
    }
    __syncthreads();
    if (lane == 63) parts[wave] = v;
    __syncthreads();
    int64_t before = base;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      if (i < wave) before += parts[i];
      base += parts[i];
    }
    if (r < a.requests) prefix[r + 1] = before + v;
  }
  if (tid == 0) prefix[0] = 0;
  __syncthreads();
}

// A value that all lanes of the wave hold, kept in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// The work is cut into equal shares, one a workgroup.
__device__ __forceinline__ int64_t share_of(const AttendArgs& a, int64_t all) {
  return max((all + a.grid - 1) / a.grid, (int64_t)a.least);
}

// Last index i of [0, n) with at[i] <= x; at[0] <= x.
template <typename T>
__device__ __forceinline__ int last_at_most(const T* at, int n, int64_t x) {
  int lo = 0;
  while (n > 1) {
    const int half = n >> 1;
    if (at[lo + half] <= x) lo += half;
    n -= half;
  }
  return lo;
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

// The value of the lane 8 further in its row of 16.
__device__ __forceinline__ float other_half(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128,
                                                               0xF, 0xF, true));
}

__device__ __forceinline__ uint32_t bits_of(f16x2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ f16x2 halves_of(uint32_t v) { return __builtin_bit_cast(f16x2, v); }

// Codes of a dword in bits 0..3 (LOW) or 4..7 of both halves, as (c - 8) s: a
// nibble at the bottom of the mantissa of 1024 (one place a unit), or four
// places up in that of 64, is the float16 1024 + c or 64 + c. All exact.
template <bool LOW>
__device__ __forceinline__ f16x2 values_of(uint32_t w, f16x2 s) {
  const f16x2 v = LOW ? halves_of((w & 0x000f000fu) | 0x64006400u) - f16x2{1032, 1032}
                      : halves_of((w & 0x00f000f0u) | 0x54005400u) - f16x2{72, 72};
  return v * s;
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// One tile's registers of a lane: row token of quarter j for the keys; dword
// columns r (and r + 16) of octet j for the values.
template <int D>
struct Tile {
  static constexpr int GROUPS = D / 32, SETS = D / 128 ? D / 128 : 1;
  uint32_t k[2][GROUPS];
  uint32_t ks[2][GROUPS / 2];    // pairs of key scales
  u32x4 v[SETS][2];
  u32x4 vs[SETS];                // the octet's value scales

  __device__ __forceinline__ void load(const uint8_t* tile, int lane) {
    const int row = lane & 15, j = lane >> 4;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int token = 8 * (row >> 2) + (row & 3) + 4 * u;
      const uint8_t* at = tile + token * (D / 2) + j * (4 * GROUPS);
      const uint8_t* scales = tile + 32 * D + token * (2 * GROUPS);
      if constexpr (GROUPS == 2) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(at);
        k[u][0] = w[0], k[u][1] = w[1];
        ks[u][0] = *reinterpret_cast<const uint32_t*>(scales);
      } else {
#pragma unroll
        for (int g = 0; g < GROUPS; g += 4) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(at + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) k[u][g + e] = w[e];
          const u32x2 s = *reinterpret_cast<const u32x2*>(scales + 2 * g);
          ks[u][g / 2] = s[0], ks[u][g / 2 + 1] = s[1];
        }
      }
    }
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const int r = (D == 64 ? row & 7 : row) + 16 * s;
      const uint8_t* at = tile + 16 * D + (j * (D / 8) + r) * 32;
      v[s][0] = reinterpret_cast<const u32x4*>(at)[0];
      v[s][1] = reinterpret_cast<const u32x4*>(at)[1];
      vs[s] = *reinterpret_cast<const u32x4*>(tile + 34 * D + (j * GROUPS + (r >> 2)) * 16);
    }
  }
};

// A workgroup's four waves take the tiles of its share in turn, each with a
// running maximum and sum of its own, and are joined in shared memory where a
// (request, head, row block) ends.
//
// Mathematics of a tile, per wave. S^T (tokens x rows) = K Q^T and O^T (dims x
// rows) += V^T P^T on 16 x 16 x 32 products, so that the first's result lies
// in the lanes as the second wants its operand: lane (n, j) holds row n's
// scores of tokens 8 j .. 8 j + 7, which are the eight of its value dwords.
// No score crosses lanes but for the maximum. A block of 8 rows fills half of
// the 16 columns; the other half takes what float16 leaves of the same rows:
// q = hi + lo and p = hi + lo in columns n and n + 8, so queries and weights
// count with 22 bits at no further product. The running maximum moves only
// where a row's tile maximum passes it by 8 (in powers of two: weights stay
// under 2^8), one vote a tile; then the rows agree across lanes on a new one.
// Sums and outputs are float32.
//
// The next tile's registers are loaded before the present one is multiplied.
template <int D, int CT, bool BF16>
__global__ void __launch_bounds__(THREADS, D == 256 && CT == 2 ? 1 : 2)
    attend_rows_kernel(AttendArgs a) {
  constexpr int ROWS = 8 * CT, GROUPS = D / 32, SETS = Tile<D>::SETS, NIB = D == 64 ? 4 : 8;
  extern __shared__ int64_t prefix[];                    // [requests + 1]
  __shared__ int64_t parts[WAVES];
  __shared__ float peak[WAVES][ROWS], total[WAVES][ROWS];
  __shared__ float held[WAVES][ROWS][D];

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  sum_work<ROWS>(a, prefix, parts);
  if (blockIdx.x == 0)
    for (int r = tid; r <= a.requests; r += THREADS) a.shares[r] = prefix[r];
  const int64_t all = uniform(prefix[a.requests]), share = share_of(a, all);
  const int64_t begin = blockIdx.x * share, end = min(begin + share, all);

  for (int64_t at = begin; at < end;) {
    // The segment (request, head, block of rows) that `at` lies in.
    const int r = __builtin_amdgcn_readfirstlane(last_at_most(prefix, a.requests + 1, at));
    const Request req = request_of(a, r);
    const int64_t before = uniform(prefix[r]), in_request = at - before;
    const int segment = (int)(in_request / req.tiles);
    const int blocks = (req.n * a.group + ROWS - 1) / ROWS;
    const int head = segment / blocks, block = segment - head * blocks;
    const int64_t seg0 = before + (int64_t)segment * req.tiles, seg1 = seg0 + req.tiles;
    const int t0 = req.tile0 + (int)(at - seg0);
    const int t1 = req.tile0 + (int)(min(end, seg1) - seg0);

    // Queries: hi in columns 0..7, lo in 8..15, scaled by a power of two so
    // that float16 holds them whatever the type's range.
    u32x4 qf[CT][GROUPS];
    float qs[CT];
    int last[CT], from[CT];                              // positions this lane's row attends
    const int rows = req.n * a.group;
    int most = -1, least_last = INT32_MAX, most_from = 0;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int row = block * ROWS + c * 8 + (n & 7);
      const bool there = row < rows;
      const int i = there ? row / a.group : 0, g = there ? row - i * a.group : 0;
      const uint16_t* src = a.q + (int64_t)(req.first + i) * a.q_token +
                            (int64_t)(head * a.group + g) * a.q_head;
      float x[GROUPS][8], top = 0.0f;
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(src + 32 * k + 8 * j);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = there ? widen<BF16>(w[e / 2] >> (16 * (e & 1)) & 0xffffu) : 0.0f;
        exl3::butterfly8(x[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float o = __shfl_xor(x[k][e], 16);
          x[k][e] = j & 1 ? o - x[k][e] : x[k][e] + o;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float o = __shfl_xor(x[k][e], 32);
          x[k][e] = 0.125f * (j & 2 ? o - x[k][e] : x[k][e] + o);
          top = fmaxf(top, fabsf(x[k][e]));
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      int power = 0;
      if (top > 0.0f && top < __builtin_inff()) frexpf(top, &power);
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f16x2 v;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float y = ldexpf(x[k][2 * e + h], -power);
            const _Float16 hi = (_Float16)y;
            v[h] = n & 8 ? (_Float16)(y - (float)hi) : hi;
          }
          qf[c][k][e] = bits_of(v);
        }
      }
      // 2 from the transforms, log2(e) for powers of two.
      qs[c] = ldexpf(a.scale * 2.0f * 1.4426950408889634f, power);
      last[c] = there ? req.length - req.n + i : -1;
      const int64_t low = there ? (int64_t)last[c] - a.window + 1 : 0;
      from[c] = (int)max(low, (int64_t)0);
    }
    // What all rows of the block attend needs no mask.
    {
      const int row0 = block * ROWS, row1 = min(row0 + ROWS, rows) - 1;
      least_last = req.length - req.n + row0 / a.group;
      most = req.length - req.n + row1 / a.group;
      most_from = (int)max((int64_t)most - a.window + 1, (int64_t)0);
    }

    float run[CT], sum[CT];
    f32x4 o[CT][SETS * NIB];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      run[c] = NONE, sum[c] = 0.0f;
#pragma unroll
      for (int m = 0; m < SETS * NIB; ++m) o[c][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int32_t* table = a.tables + (int64_t)r * a.width;
    // A tile's address, or NULL where the table names no page of the cache.
    auto tile_at = [&](int t) -> const uint8_t* {
      const int id = table[t >> a.cache.tile_shift];
      if (id < 0 || id >= a.cache.pages) return nullptr;
      return a.pages + exl3::cache_tile_at(a.cache, id, head, t & ((1 << a.cache.tile_shift) - 1));
    };

    Tile<D> next;
    const uint8_t* here = t0 + wave < t1 ? tile_at(t0 + wave) : nullptr;
    if (here) next.load(here, lane);
    for (int t = t0 + wave; t < t1; t += WAVES) {
      const Tile<D> tile = next;
      const bool present = here != nullptr;
      here = t + WAVES < t1 ? tile_at(t + WAVES) : nullptr;
      if (here) next.load(here, lane);
      if (!present) continue;

      const int pos = t * CACHE_TILE;
      const bool masked = pos < most_from || pos + CACHE_TILE - 1 > least_last;
      f32x4 s[CT][2];
#pragma unroll
      for (int c = 0; c < CT; ++c) s[c][0] = s[c][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
          const f16x2 pair = halves_of(tile.ks[u][k / 2]);
          const f16x2 scale = k & 1 ? f16x2{pair[1], pair[1]} : f16x2{pair[0], pair[0]};
          const uint32_t w = tile.k[u][k];
          u32x4 f;
          f[0] = bits_of(values_of<true>(w, scale));
          f[1] = bits_of(values_of<false>(w, scale));
          f[2] = bits_of(values_of<true>(w >> 8, scale));
          f[3] = bits_of(values_of<false>(w >> 8, scale));
#pragma unroll
          for (int c = 0; c < CT; ++c) s[c][u] = mfma(f, qf[c][k], s[c][u]);
        }
      }

      u32x4 p[CT];
      uint32_t attended[CT];                             // this row's tokens of the octet
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = s[c][e >> 2][e & 3];
          x[e] = (v + other_half(v)) * qs[c];
        }
        attended[c] = 0xffu;
        if (masked) {
          attended[c] = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at_pos = pos + 8 * j + e;
            const bool in = at_pos >= from[c] && at_pos <= last[c];
            x[e] = in ? x[e] : NONE;
            attended[c] |= (uint32_t)in << e;
          }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
        if (__any(top > run[c] + 8.0f)) {
          top = fmaxf(top, run[c]);
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float shrink = top == run[c] ? 1.0f : __builtin_amdgcn_exp2f(run[c] - top);
          run[c] = top;
          sum[c] *= shrink;
#pragma unroll
          for (int m = 0; m < SETS * NIB; ++m) o[c][m] *= shrink;
        }
        const float ref = run[c] == NONE ? 0.0f : run[c];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f16x2 v;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float w = __builtin_amdgcn_exp2f(x[2 * e + h] - ref);
            sum[c] += w;
            const _Float16 hi = (_Float16)w;
            v[h] = n & 8 ? (_Float16)(w - (float)hi) : hi;
          }
          p[c][e] = bits_of(v);
        }
      }

#pragma unroll
      for (int d = 0; d < SETS; ++d) {
        u32x4 scales = tile.vs[d];
        uint32_t poisoned = 0;                           // tokens of the octet without a finite scale
        if (masked) {
          // Positions that a row does not attend have a weight of 0, which a
          // NaN or infinity would pass through: such scales count as 0, and
          // rows that do attend the token get their NaN below.
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t h = scales[e / 2] >> (16 * (e & 1)) & 0x7fffu;
            if (h >= 0x7c00u) {
              poisoned |= 1u << e;
              scales[e / 2] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
            }
          }
        }
#pragma unroll
        for (int b = 0; b < NIB / 2; ++b) {
          // Byte b of a pair of tokens' dwords, one in each half; a dword of
          // D = 64 serves two rows, each half of its bytes.
          const uint32_t byte = b + (D == 64 ? (lane & 8) >> 2 : 0);
          const uint32_t pick = 0x0c000c04u | byte << 16 | byte;
          u32x4 lo, hi;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t first = tile.v[d][e >> 1][(2 * e) & 3], second = tile.v[d][e >> 1][(2 * e + 1) & 3];
            const uint32_t w = __builtin_amdgcn_perm(first, second, pick);
            const f16x2 scale = halves_of(scales[e]);
            lo[e] = bits_of(values_of<true>(w, scale));
            hi[e] = bits_of(values_of<false>(w, scale));
          }
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            o[c][d * NIB + 2 * b] = mfma(lo, p[c], o[c][d * NIB + 2 * b]);
            o[c][d * NIB + 2 * b + 1] = mfma(hi, p[c], o[c][d * NIB + 2 * b + 1]);
          }
        }
        if (masked && __any(poisoned != 0)) {
          u32x4 f;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            f[e] = (poisoned >> (2 * e) & 1u ? 0x3c00u : 0u) | (poisoned >> (2 * e + 1) & 1u ? 0x3c000000u : 0u);
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            u32x4 ones;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              ones[e] = (attended[c] >> (2 * e) & 1u ? 0x3c00u : 0u) | (attended[c] >> (2 * e + 1) & 1u ? 0x3c000000u : 0u);
            const f32x4 hit = mfma(f, ones, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int m = 0; m < NIB; ++m)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (hit[e] > 0.0f) o[c][d * NIB + m][e] = __builtin_nanf("");
          }
        }
      }
    }

    // The wave's result: hi and lo columns together, taken back from the
    // transformed basis (dims 8 (4 j + e) + m, so a lane of D >= 128 holds
    // whole groups; of D = 64, half a group each).
    __syncthreads();                                     // the last segment has been read
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      sum[c] += __shfl_xor(sum[c], 16);
      sum[c] += __shfl_xor(sum[c], 32);
      if (lane < 8) peak[wave][c * 8 + n] = run[c], total[wave][c * 8 + n] = sum[c];
#pragma unroll
      for (int d = 0; d < SETS; ++d) {
        f32x4* v = &o[c][d * NIB];
#pragma unroll
        for (int m = 0; m < NIB; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[m][e] += other_half(v[m][e]);
#pragma unroll
        for (int h = 1; h < NIB; h *= 2)
#pragma unroll
          for (int m = 0; m < NIB; ++m)
            if (!(m & h)) {
              const f32x4 x = v[m], y = v[m + h];
              v[m] = x + y;
              v[m + h] = x - y;
            }
#pragma unroll
        for (int m = 0; m < NIB; ++m) {
          if constexpr (D == 64) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = __shfl_xor(v[m][e], 32);
              v[m][e] = j & 2 ? w - v[m][e] : v[m][e] + w;
            }
          }
          const f32x4 x = v[m];
          const float s0 = x[0] + x[1], s1 = x[0] - x[1], s2 = x[2] + x[3], s3 = x[2] - x[3];
          v[m] = 0.25f * f32x4{s0 + s2, s1 + s3, s0 - s2, s1 - s3};
        }
        if (n < 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int dim = D == 64 ? 32 * (j & 1) + 8 * e + 4 * (j >> 1) : 128 * d + 32 * j + 8 * e;
            float* to = &held[wave][c * 8 + n][dim];
#pragma unroll
            for (int m = 0; m < NIB; m += 4)
              *reinterpret_cast<f32x4*>(to + m) = f32x4{v[m][e], v[m + 1][e], v[m + 2][e], v[m + 3][e]};
          }
        }
      }
    }
    __syncthreads();

    const bool whole = at == seg0 && seg1 <= end;
    float* part = a.partials + ((int64_t)blockIdx.x * 2 + (at == seg0)) * (ROWS * (D + 2));
    for (int i = tid; i < ROWS * (D / 4); i += THREADS) {
      const int row = i / (D / 4), d0 = 4 * (i - row * (D / 4));
      const int of = block * ROWS + row;
      if (of >= rows) break;
      float top = peak[0][row];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) top = fmaxf(top, peak[w][row]);
      f32x4 x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        // A wave without an attended tile holds zeros.
        const float weight = peak[w][row] == NONE ? 1.0f : __builtin_amdgcn_exp2f(peak[w][row] - top);
        l += total[w][row] * weight;
        x += *reinterpret_cast<const f32x4*>(&held[w][row][d0]) * weight;
      }
      if (whole) {
        const int token = req.first + of / a.group, h = head * a.group + of % a.group;
        u32x2 w;
        const float inverse = 1.0f / l;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = l == 0.0f ? 0.0f : x[e] * inverse;
        w[0] = narrow<BF16>(x[0]) | narrow<BF16>(x[1]) << 16;
        w[1] = narrow<BF16>(x[2]) | narrow<BF16>(x[3]) << 16;
        *reinterpret_cast<u32x2*>(a.out + ((int64_t)token * a.q_heads + h) * D + d0) = w;
      } else {
        *reinterpret_cast<f32x4*>(part + row * D + d0) = x;
        if (d0 == 0) part[ROWS * D + 2 * row] = top, part[ROWS * D + 2 * row + 1] = l;
      }
    }
    at = min(end, seg1);
  }
}

// One workgroup an output row (token, query head): rows whose segment more
// than one workgroup took are joined from its partials, in the order of the
// tiles; rows of no work are 0; whole ones are left.
template <int D, int CT, bool BF16>
__global__ void __launch_bounds__(64) attend_join_kernel(AttendArgs a) {
  constexpr int ROWS = 8 * CT;
  const int64_t token = blockIdx.x / a.q_heads;
  const int qh = (int)(blockIdx.x - token * a.q_heads), lane = threadIdx.x;
  uint16_t* out = a.out + ((int64_t)token * a.q_heads + qh) * D;
  constexpr int PER = D / 64;
  float x[PER], top = NONE, l = 0.0f;
#pragma unroll
  for (int e = 0; e < PER; ++e) x[e] = 0.0f;
  const int r = a.starts[0] <= token ? last_at_most(a.starts, a.requests + 1, token) : a.requests;
  int tiles = 0;
  Request req{};
  if (r < a.requests) {
    req = request_of(a, r);
    if (token >= req.first && token < req.first + req.n) tiles = req.tiles;
  }
  if (tiles > 0) {
    const int head = qh / a.group, of = (int)(token - req.first) * a.group + qh % a.group;
    const int blocks = (req.n * a.group + ROWS - 1) / ROWS;
    const int64_t share = share_of(a, a.shares[a.requests]);
    const int64_t seg0 = a.shares[r] + ((int64_t)head * blocks + of / ROWS) * tiles, seg1 = seg0 + tiles;
    const int64_t w0 = seg0 / share, w1 = (seg1 - 1) / share;
    if (w0 == w1) return;
    for (int64_t w = w0; w <= w1; ++w) {
      const float* part = a.partials + (2 * w + (w == w0)) * (ROWS * (D + 2));
      const int row = of % ROWS;
      const float peak = part[ROWS * D + 2 * row], sum = part[ROWS * D + 2 * row + 1];
      if (peak == NONE && sum == 0.0f) continue;
      const float newer = fmaxf(top, peak);
      const float keep = newer == top ? 1.0f : __builtin_amdgcn_exp2f(top - newer);
      const float add = newer == peak ? 1.0f : __builtin_amdgcn_exp2f(peak - newer);
      top = newer;
      l = l * keep + sum * add;
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] = x[e] * keep + part[row * D + PER * lane + e] * add;
    }
  }
  const float inverse = 1.0f / l;
#pragma unroll
  for (int e = 0; e < PER; ++e) out[PER * lane + e] = (uint16_t)narrow<BF16>(l == 0.0f ? 0.0f : x[e] * inverse);
}

constexpr int GRID = 1024;

struct Plan {
  int64_t partials, shares;      // bytes
};
Plan plan_of(int requests, int head_dim, int ct) {
  return {(int64_t)2 * GRID * 8 * ct * (head_dim + 2) * 4, (8 * ((int64_t)requests + 1) + 15) & ~(int64_t)15};
}

template <int D, int CT>
int launch_attend(const AttendArgs& args, bool bf16, hipStream_t stream) {
  const size_t lds = 8 * ((size_t)args.requests + 1);
  const unsigned rows = (unsigned)(args.tokens * args.q_heads);
  if (bf16) {
    attend_rows_kernel<D, CT, true><<<args.grid, THREADS, lds, stream>>>(args);
    if (check_launch("exl3_cache_attention")) return 1;
    attend_join_kernel<D, CT, true><<<rows, 64, 0, stream>>>(args);
  } else {
    attend_rows_kernel<D, CT, false><<<args.grid, THREADS, lds, stream>>>(args);
    if (check_launch("exl3_cache_attention")) return 1;
    attend_join_kernel<D, CT, false><<<rows, 64, 0, stream>>>(args);
  }
  return check_launch("exl3_cache_attention");
}

}  // namespace

extern "C" {

int64_t exl3_cache_attention_workspace(int requests, int head_dim) {
  if (requests < 1 || requests > CACHE_MAX_REQUESTS || (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return -1;
  const Plan p = plan_of(requests, head_dim, 2);
  return p.partials + p.shares;
}

int exl3_cache_attention(const void* q, int64_t q_token, int64_t q_head, void* out, int64_t tokens,
                         int q_heads, int type, const void* pages, int64_t num_pages, int page_size,
                         int kv_heads, int head_dim, const int32_t* tables, int width,
                         const int32_t* starts, const int32_t* lengths, int requests, float scale,
                         int64_t window, int64_t max_new, void* workspace, int64_t workspace_bytes,
                         void* stream) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error("exl3_cache_attention: head_dim must be 64, 128 or 256, got %d", head_dim);
  if (page_size < 32 || page_size > 256 || (page_size & (page_size - 1)))
    return set_error("exl3_cache_attention: page_size must be 32, 64, 128 or 256, got %d", page_size);
  if (num_pages < 0 || num_pages > INT32_MAX || kv_heads < 1 || q_heads < 1 || q_heads > 65535 ||
      q_heads % kv_heads)
    return set_error("exl3_cache_attention: q_heads (%d) must be a multiple of kv_heads (%d)", q_heads, kv_heads);
  if (requests < 1 || requests > CACHE_MAX_REQUESTS)
    return set_error("exl3_cache_attention: requests must be in 1..%d, got %d", CACHE_MAX_REQUESTS, requests);
  if (width < 1 || (int64_t)width * page_size > INT32_MAX)
    return set_error("exl3_cache_attention: bad table width %d", width);
  if (tokens < 0 || tokens * q_heads > INT32_MAX) return set_error("exl3_cache_attention: too many tokens");
  if (type < 1 || type > 2) return set_error("exl3_cache_attention: queries are float16 or bfloat16");
  if (window < 1) return set_error("exl3_cache_attention: window must be positive");
  if ((reinterpret_cast<uintptr_t>(q) & 15) || q_token % 8 || q_head % 8)
    return set_error("exl3_cache_attention: query rows must be 16-byte aligned");
  if (((reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 7))
    return set_error("exl3_cache_attention: pages, out and workspace must be aligned");
  if (workspace_bytes < exl3_cache_attention_workspace(requests, head_dim))
    return set_error("exl3_cache_attention: workspace of %lld bytes is too small", (long long)workspace_bytes);
  if (!tokens) return 0;
  AttendArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.out = static_cast<uint16_t*>(out);
  a.pages = static_cast<const uint8_t*>(pages);
  a.tables = tables, a.starts = starts, a.lengths = lengths;
  a.q_token = q_token, a.q_head = q_head, a.tokens = tokens;
  a.window = std::min<int64_t>(window, INT32_MAX);
  int shift = 0;
  while ((CACHE_TILE << shift) < page_size) ++shift;
  a.cache = CacheShape{num_pages, kv_heads, head_dim, shift};
  a.requests = requests, a.width = width, a.q_heads = q_heads, a.group = q_heads / kv_heads;
  a.scale = scale;
  a.grid = GRID, a.least = WAVES;
  const bool two = std::min<int64_t>(max_new, tokens) * a.group > 8;
  const Plan p = plan_of(requests, head_dim, two ? 2 : 1);
  a.shares = static_cast<int64_t*>(workspace);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.shares);
  const bool bf16 = type == 2;
  hipStream_t s = (hipStream_t)stream;
  if (head_dim == 64) return two ? launch_attend<64, 2>(a, bf16, s) : launch_attend<64, 1>(a, bf16, s);
  if (head_dim == 128) return two ? launch_attend<128, 2>(a, bf16, s) : launch_attend<128, 1>(a, bf16, s);
  return two ? launch_attend<256, 2>(a, bf16, s) : launch_attend<256, 1>(a, bf16, s);
}

}  // extern "C"
