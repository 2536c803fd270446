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
#include <type_traits>

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
  float* partials;               // [2 shares][rows][D + 2]: values, then maximum and sum
  int64_t* shares;               // [requests + 1] prefix of the work, for the join
  int64_t q_token, q_head, tokens, window;
  CacheShape cache;
  int requests, width, q_heads, group;
  int waves;                     // shares that the work is cut into
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
  q.tiles = q.n && a.cache.pages ? (int)((length + CACHE_TILE - 1) / CACHE_TILE) - q.tile0 : 0;
  return q;
}

// A segment is one kv head and block of ROWS query rows of a request. Its work
// is its tiles, and before them what beginning and ending it costs, as tiles:
// a share of many short segments would end late without.
constexpr int SEGMENT_COST = 8;
template <int ROWS>
__device__ __forceinline__ int64_t work_of(const AttendArgs& a, const Request& q) {
  const int64_t blocks = ((int64_t)q.n * a.group + ROWS - 1) / ROWS;
  return q.tiles ? blocks * a.cache.kv_heads * (q.tiles + SEGMENT_COST) : 0;
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

// The work is cut into equal shares, one a wave, of LEAST at least.
constexpr int LEAST = 2;
__device__ __forceinline__ int64_t share_of(const AttendArgs& a, int64_t all) {
  return max((all + a.waves - 1) / a.waves, (int64_t)LEAST);
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

// Constants of values_of in vector registers, so that mask and magic are one
// instruction (v_and_or_b32 reads one scalar).
struct Magic {
  uint32_t low, high;
  __device__ __forceinline__ Magic() : low(0x64006400u), high(0x54005400u) {
    asm volatile("" : "+v"(low), "+v"(high));
  }
};

// Codes of a dword in bits 0..3 (LOW) or 4..7 of both halves, as (c - 8) s: a
// nibble at the bottom of the mantissa of 1024 (one place a unit), or four
// places up in that of 64, is the float16 1024 + c or 64 + c. All exact.
template <bool LOW>
__device__ __forceinline__ uint32_t values_of(uint32_t w, f16x2 s, const Magic& magic) {
  const f16x2 v = LOW ? halves_of((w & 0x000f000fu) | magic.low) - f16x2{1032, 1032}
                      : halves_of((w & 0x00f000f0u) | magic.high) - f16x2{72, 72};
  return bits_of(v * s);
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// One butterfly level between lanes 16 or 32 apart, for two registers at once:
// the first swap brings the halves of a pair together, the second puts sums
// and differences back in their lanes.
template <int APART>
__device__ __forceinline__ void lane_butterfly(float& x, float& y) {
  static_assert(APART == 16 || APART == 32, "rows of the wave");
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
    const uint32_t row = lane & 15, j = lane >> 4;
    const uint32_t token = 8 * (row >> 2) + (row & 3), r = D == 64 ? row & 7 : row;
    const uint8_t *codes = tile + (token * (D / 2) + j * (4 * GROUPS)),
                  *scales = tile + (32 * D + token * (2 * GROUPS)),
                  *values = tile + (16 * D + (j * (D / 8) + r) * 32),
                  *value_scales = tile + (34 * D + (j * GROUPS + (r >> 2)) * 16);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (GROUPS == 2) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(codes + u * (2 * D));
        k[u][0] = w[0], k[u][1] = w[1];
        ks[u][0] = *reinterpret_cast<const uint32_t*>(scales + u * (8 * GROUPS));
      } else {
#pragma unroll
        for (int g = 0; g < GROUPS; g += 4) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(codes + u * (2 * D) + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) k[u][g + e] = w[e];
          const u32x2 s = *reinterpret_cast<const u32x2*>(scales + u * (8 * GROUPS) + 2 * g);
          ks[u][g / 2] = s[0], ks[u][g / 2 + 1] = s[1];
        }
      }
    }
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      v[s][0] = *reinterpret_cast<const u32x4*>(values + s * 512);
      v[s][1] = *reinterpret_cast<const u32x4*>(values + s * 512 + 16);
      vs[s] = *reinterpret_cast<const u32x4*>(value_scales + s * 64);
    }
  }
};

// Workgroups of a compute unit that a variant's registers allow.
constexpr int resident(int d, int ct) { return d == 64 ? (ct == 1 ? 4 : 3) : d == 128 ? (ct == 1 ? 3 : 2) : (ct == 1 ? 2 : 1); }

// Every wave takes one share of all work, an equal run of tiles that may end
// one segment and begin others: segments that it holds whole it finishes,
// others leave a partial result for attend_join_kernel. Waves wait for nobody;
// a workgroup's four only share the sums over the requests.
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
// Two tiles' registers take turns: one is loaded while the other is
// multiplied, and table entries are read a tile further ahead.
template <int D, int CT, bool BF16>
__global__ void __launch_bounds__(THREADS, resident(D, CT)) attend_rows_kernel(AttendArgs a) {
  constexpr int ROWS = 8 * CT, GROUPS = D / 32, SETS = Tile<D>::SETS, NIB = D == 64 ? 4 : 8;
  extern __shared__ int64_t prefix[];                    // [requests + 1]
  __shared__ int64_t parts[WAVES];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Magic magic;
  sum_work<ROWS>(a, prefix, parts);
  if (blockIdx.x == 0)
    for (int r = tid; r <= a.requests; r += THREADS) a.shares[r] = prefix[r];
  const int64_t all = uniform(prefix[a.requests]), share = share_of(a, all);
  const int owner = (int)blockIdx.x * WAVES + wave;
  const int64_t begin = owner * share, end = min(begin + share, all);

  for (int64_t at = begin; at < end;) {
    // Opaque here, so that addresses made of it are not kept in registers
    // across the tile loop from segment to segment.
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));
    const int n = lane & 15, j = lane >> 4;
    // The minus one of columns 8..15, which take what columns 0..7 leave.
    const float rest = n & 8 ? -1.0f : 0.0f;
    // The segment (request, head, block of rows) that `at` lies in.
    const int r = __builtin_amdgcn_readfirstlane(last_at_most(prefix, a.requests + 1, at));
    const Request req = request_of(a, r);
    const int64_t before = uniform(prefix[r]);
    const uint32_t in_request = (uint32_t)(at - before);
    const int segment = (int)(in_request / (uint32_t)(req.tiles + SEGMENT_COST));
    const int blocks = (req.n * a.group + ROWS - 1) / ROWS;
    const int head = segment / blocks, block = segment - head * blocks;
    const int64_t seg0 = before + (int64_t)segment * (req.tiles + SEGMENT_COST) + SEGMENT_COST;
    const int64_t seg1 = seg0 + req.tiles;               // its tiles in the row of all work
    const int first = (int)max(at - seg0, (int64_t)0), past = (int)(min(end, seg1) - seg0);
    at = min(end, seg1);
    if (past <= first) continue;
    const int t0 = req.tile0 + first, t1 = req.tile0 + past;

    // In the constant address space: read by the scalar unit.
    const auto* table = (const __attribute__((address_space(4))) int32_t*)(a.tables + (int64_t)r * a.width);
    // The page of a tile, -1 where the table names none of the cache.
    auto page_of = [&](int t) {
      const int id = table[min(t, t1 - 1) >> a.cache.tile_shift];
      return (uint32_t)id < (uint64_t)a.cache.pages ? id : -1;
    };
    auto tile_at = [&](int t, int page) {
      return a.pages + exl3::cache_tile_at(a.cache, max(page, 0), head, min(t, t1 - 1) & ((1 << a.cache.tile_shift) - 1));
    };
    // The first tiles are on their way while the queries are transformed.
    Tile<D> even, odd;
    int page_even = page_of(t0), page_odd = page_of(t0 + 1);
    even.load(tile_at(t0, page_even), lane);

    // Queries: hi in columns 0..7, lo in 8..15, scaled by a power of two so
    // that float16 holds them whatever the type's range.
    u32x4 qf[CT][GROUPS];
    float qs[CT], rise[CT];
    int last[CT], from[CT];                              // positions this lane's row attends
    const int rows = req.n * a.group;
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
        for (int e = 0; e < 8; e += 2) {
          lane_butterfly<16>(x[k][e], x[k][e + 1]);
          lane_butterfly<32>(x[k][e], x[k][e + 1]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[k][e]));
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      int power = 0;
      if (top > 0.0f && top < __builtin_inff()) frexpf(top, &power);
      // A negative scale turns the query over, so that larger scores are
      // larger weights in what follows.
      const float flip = a.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y0 = flip * ldexpf(x[k][2 * e], -power), y1 = flip * ldexpf(x[k][2 * e + 1], -power);
          const f16x2 hi = {(_Float16)y0, (_Float16)y1};
          qf[c][k][e] = bits_of(f16x2{(_Float16)__builtin_fmaf((float)hi[0], rest, y0),
                                      (_Float16)__builtin_fmaf((float)hi[1], rest, y1)});
        }
      }
      // An eighth from the query's transform, 2 from both; log2(e) for powers
      // of two.
      qs[c] = ldexpf(fabsf(a.scale) * 0.25f * 1.4426950408889634f, power);
      rise[c] = 8.0f / qs[c];
      last[c] = there ? req.length - req.n + i : -1;
      const int64_t low = there ? (int64_t)last[c] - a.window + 1 : 0;
      from[c] = (int)max(low, (int64_t)0);
    }
    // Positions that all rows of the block attend need no mask.
    const int row0 = block * ROWS, row1 = min(row0 + ROWS, rows) - 1;
    const int least_last = req.length - req.n + row0 / a.group;
    const int most_from = (int)max((int64_t)(req.length - req.n + row1 / a.group) - a.window + 1, (int64_t)0);

    float run[CT], sum[CT];                              // run: the maximum before the factor qs
    f32x4 o[CT][SETS * NIB];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      run[c] = NONE, sum[c] = 0.0f;
#pragma unroll
      for (int m = 0; m < SETS * NIB; ++m) o[c][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto attend = [&](const Tile<D>& tile, int t, int page) __attribute__((always_inline)) {
      if (t >= t1 || page < 0) return;
      // The branches on `masked` are real ones (the empty asm keeps them from
      // becoming selects): most tiles have nothing to mask.
      const bool masked = t * CACHE_TILE < most_from || t * CACHE_TILE + CACHE_TILE - 1 > least_last;
      const int pos = t * CACHE_TILE + 8 * j;
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
          f[0] = values_of<true>(w, scale, magic);
          f[1] = values_of<false>(w, scale, magic);
          f[2] = values_of<true>(w >> 8, scale, magic);
          f[3] = values_of<false>(w >> 8, scale, magic);
#pragma unroll
          for (int c = 0; c < CT; ++c) s[c][u] = mfma(f, qf[c][k], s[c][u]);
        }
      }

      u32x4 p[CT];
      uint32_t attended[CT] = {};                        // this row's tokens of the octet
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = s[c][e >> 2][e & 3];
          x[e] = v + other_half(v);
        }
        if (masked) {
          attended[c] = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool in = pos + e >= from[c] && pos + e <= last[c];
            x[e] = in ? x[e] : NONE;
            attended[c] |= (uint32_t)in << e;
            asm volatile("" : "+v"(x[e]));
          }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
        if (__any(top > run[c] + rise[c])) {
          top = fmaxf(top, run[c]);
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float shrink = top == run[c] ? 1.0f : __builtin_amdgcn_exp2f((run[c] - top) * qs[c]);
          run[c] = top;
          sum[c] *= shrink;
#pragma unroll
          for (int m = 0; m < SETS * NIB; ++m) o[c][m] *= shrink;
        }
        const float ref = run[c] == NONE ? 0.0f : -run[c] * qs[c];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float w[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            w[h] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * e + h], qs[c], ref));
            sum[c] += w[h];
          }
          const f16x2 hi = {(_Float16)w[0], (_Float16)w[1]};
          p[c][e] = bits_of(f16x2{(_Float16)__builtin_fmaf((float)hi[0], rest, w[0]),
                                  (_Float16)__builtin_fmaf((float)hi[1], rest, w[1])});
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
          asm volatile("" : "+v"(scales));
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
            lo[e] = values_of<true>(w, scale, magic);
            hi[e] = values_of<false>(w, scale, magic);
          }
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            o[c][d * NIB + 2 * b] = mfma(lo, p[c], o[c][d * NIB + 2 * b]);
            o[c][d * NIB + 2 * b + 1] = mfma(hi, p[c], o[c][d * NIB + 2 * b + 1]);
          }
        }
        if (masked && __any(poisoned != 0)) {
          // Ones where a token has no finite scale, times ones where a row
          // attends it.
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
    };
    for (int t = t0; t < t1; t += 2) {
      const int page_even_next = page_of(t + 2), page_odd_next = page_of(t + 3);
      odd.load(tile_at(t + 1, page_odd), lane);
      attend(even, t, page_even);
      even.load(tile_at(t + 2, page_even_next), lane);
      attend(odd, t + 1, page_odd);
      page_even = page_even_next, page_odd = page_odd_next;
    }

    // The result: hi and lo columns together, taken back from the transformed
    // basis. Lane (n, j) holds dims 8 (4 j + e) + m of row n: whole groups of
    // D >= 128, half a group of D = 64.
    const bool whole = past - first == req.tiles;
    float* part = a.partials + ((int64_t)owner * 2 + (first == 0)) * (ROWS * (D + 2));
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      sum[c] += __shfl_xor(sum[c], 16);
      sum[c] += __shfl_xor(sum[c], 32);
      const float inverse = sum[c] == 0.0f ? 0.0f : 1.0f / sum[c];
      const int row = c * 8 + n, of = block * ROWS + row;
      const bool writes = n < 8 && of < rows;
      if (writes && !whole && j == 0) {
        part[ROWS * D + 2 * row] = run[c] == NONE ? NONE : run[c] * qs[c];
        part[ROWS * D + 2 * row + 1] = sum[c];
      }
      uint16_t* out = a.out + ((int64_t)(req.first + of / a.group) * a.q_heads + head * a.group + of % a.group) * D;
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
          float y[4] = {v[m][0], v[m][1], v[m][2], v[m][3]};
          if constexpr (D == 64) {
            lane_butterfly<32>(y[0], y[1]);
            lane_butterfly<32>(y[2], y[3]);
          }
          const float s0 = y[0] + y[1], s1 = y[0] - y[1], s2 = y[2] + y[3], s3 = y[2] - y[3];
          v[m] = 0.25f * f32x4{s0 + s2, s1 + s3, s0 - s2, s1 - s3};
        }
        if (!writes) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int dim = D == 64 ? 32 * (j & 1) + 8 * e + 4 * (j >> 1) : 128 * d + 32 * j + 8 * e;
#pragma unroll
          for (int m = 0; m < NIB; m += 4) {
            const f32x4 x = {v[m][e], v[m + 1][e], v[m + 2][e], v[m + 3][e]};
            if (whole) {
              u32x2 w;
              w[0] = narrow<BF16>(x[0] * inverse) | narrow<BF16>(x[1] * inverse) << 16;
              w[1] = narrow<BF16>(x[2] * inverse) | narrow<BF16>(x[3] * inverse) << 16;
              *reinterpret_cast<u32x2*>(out + dim + m) = w;
            } else {
              *reinterpret_cast<f32x4*>(part + row * D + dim + m) = x;
            }
          }
        }
      }
    }
  }
}

// The partial results of an output row (token, query head) that more than one
// wave has taken, joined in the order of the tiles; rows of no work are 0;
// whole ones are left. The maxima are read first, 64 at once, so that the
// values are then summed by known weights and no load waits for another.
// SPREAD waves take one row's partials in turn: all four of a workgroup where
// there are few rows, each with many partials (one token of 4097 positions, 32
// rows: 5.6 us, with one wave a row 9.8), one where there are many rows (128
// tokens, 4096 rows: 13.7 us with four).
template <int D, int CT, bool BF16, int SPREAD>
__global__ void __launch_bounds__(THREADS) attend_join_kernel(AttendArgs a) {
  constexpr int ROWS = 8 * CT, PER = D / 64, STRIDE = ROWS * (D + 2);
  typedef float values __attribute__((ext_vector_type(PER)));
  __shared__ float held[WAVES][SPREAD > 1 ? D : 1], sums[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t at = (int64_t)blockIdx.x * (WAVES / SPREAD) + wave / SPREAD;
  if (at >= a.tokens * a.q_heads) return;
  const int64_t token = at / a.q_heads;
  const int qh = (int)(at - token * a.q_heads);
  uint16_t* out = a.out + at * D + PER * lane;
  auto write = [&](const float (&x)[PER], float l) {
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < PER; ++e) out[e] = (uint16_t)narrow<BF16>(x[e] * inverse);
  };
  // The request: as many starts after the first as are not past the token.
  int r = 0;
  for (int r0 = 0; r0 < a.requests; r0 += 64)
    r += __popcll(__ballot(r0 + lane < a.requests && a.starts[r0 + lane + 1] <= token));
  int tiles = 0;
  Request req{};
  if (r < a.requests) {
    req = request_of(a, r);
    if (token >= req.first && token < req.first + req.n) tiles = req.tiles;
  }
  float x[PER], l = 0.0f;
#pragma unroll
  for (int e = 0; e < PER; ++e) x[e] = 0.0f;
  if (tiles == 0) {
    if (wave % SPREAD == 0) write(x, l);
    return;
  }
  const int head = qh / a.group, of = (int)(token - req.first) * a.group + qh % a.group;
  const int blocks = (req.n * a.group + ROWS - 1) / ROWS, row = of % ROWS;
  const int64_t share = share_of(a, a.shares[a.requests]);
  const int64_t seg0 = a.shares[r] + ((int64_t)head * blocks + of / ROWS) * (tiles + SEGMENT_COST) + SEGMENT_COST;
  const int64_t seg1 = seg0 + tiles;
  const int w0 = (int)(seg0 / share), w1 = (int)((seg1 - 1) / share);
  if (w0 == w1) return;
  // The first owner's share ends in this segment (slot 1), the others' begin
  // in it (slot 0).
  auto slot = [&](int w) { return a.partials + (2 * (int64_t)w + (w == w0)) * STRIDE; };
  float top = NONE;
  for (int w = w0 + lane; w <= w1; w += 64) top = fmaxf(top, slot(w)[ROWS * D + 2 * row]);
#pragma unroll
  for (int o = 1; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
#pragma unroll 4
  for (int w = w0 + wave % SPREAD; w <= w1; w += SPREAD) {
    const float* part = slot(w);
    const float peak = part[ROWS * D + 2 * row];
    const float weight = peak == NONE ? 1.0f : __builtin_amdgcn_exp2f(peak - top);
    const values v = *reinterpret_cast<const values*>(part + row * D + PER * lane);
    l += part[ROWS * D + 2 * row + 1] * weight;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if constexpr (PER == 1) x[e] += v[0] * weight;
      else x[e] += v[e] * weight;
    }
  }
  if constexpr (SPREAD > 1) {
    static_assert(SPREAD == 1 || SPREAD == WAVES, "a row or a workgroup's rows");
#pragma unroll
    for (int e = 0; e < PER; ++e) held[wave][PER * lane + e] = x[e];
    if (lane == 0) sums[wave] = l;
    __syncthreads();
    if (wave != 0) return;
    l = (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int d = PER * lane + e;
      x[e] = (held[0][d] + held[1][d]) + (held[2][d] + held[3][d]);
    }
  }
  write(x, l);
}

constexpr int CUS = 256;

struct Plan {
  int64_t partials, shares;      // bytes
};
Plan plan_of(int requests, int head_dim, int ct) {
  return {(int64_t)2 * CUS * resident(head_dim, ct) * WAVES * 8 * ct * (head_dim + 2) * 4, (8 * ((int64_t)requests + 1) + 15) & ~(int64_t)15};
}

template <int D, int CT, bool BF16>
int launch_attend(AttendArgs args, hipStream_t stream) {
  args.waves = CUS * resident(D, CT) * WAVES;
  const size_t lds = 8 * ((size_t)args.requests + 1);
  const int64_t rows = args.tokens * args.q_heads;
  attend_rows_kernel<D, CT, BF16><<<CUS * resident(D, CT), THREADS, lds, stream>>>(args);
  if (check_launch("exl3_cache_attention")) return 1;
  if (rows <= 4 * CUS)
    attend_join_kernel<D, CT, BF16, WAVES><<<(unsigned)rows, THREADS, 0, stream>>>(args);
  else
    attend_join_kernel<D, CT, BF16, 1><<<(unsigned)((rows + WAVES - 1) / WAVES), THREADS, 0, stream>>>(args);
  return check_launch("exl3_cache_attention");
}

}  // namespace

extern "C" {

int64_t exl3_cache_attention_workspace(int requests, int head_dim) {
  if (requests < 1 || requests > CACHE_MAX_REQUESTS || (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return -1;
  const Plan one = plan_of(requests, head_dim, 1), two = plan_of(requests, head_dim, 2);
  return std::max(one.partials, two.partials) + one.shares;
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
  const bool two = std::min<int64_t>(max_new, tokens) * a.group > 8;
  const Plan p = plan_of(requests, head_dim, two ? 2 : 1);
  a.shares = static_cast<int64_t*>(workspace);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.shares);
  auto launch = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    hipStream_t s = (hipStream_t)stream;
    if (type == 2) return two ? launch_attend<D, 2, true>(a, s) : launch_attend<D, 1, true>(a, s);
    return two ? launch_attend<D, 2, false>(a, s) : launch_attend<D, 1, false>(a, s);
  };
  if (head_dim == 64) return launch(std::integral_constant<int, 64>{});
  if (head_dim == 128) return launch(std::integral_constant<int, 128>{});
  return launch(std::integral_constant<int, 256>{});
}

}  // extern "C"
