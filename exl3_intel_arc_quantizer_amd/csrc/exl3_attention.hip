// MI355X (gfx950) kernels of attention over the 4-bit cache of
// exl3_cache_layout.h:
//
//   attend_rows_kernel  a few query rows of one kv head against a share of its
//                       tiles, as partial or whole results
//   attend_tiles_kernel many query rows (chunks and prompts), tiles unpacked
//                       once for all rows of a workgroup
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
#include <cmath>
#include <limits>
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
// Weights are 2^(score - maximum + LIFT), scores in powers of two: float16 has
// all its bits down to 2^-14, so those down to 2^-21 of the largest keep them,
// and a long context's many small weights count beside a dominant one. The
// maximum is a running one that moves where a score passes it by RISE: weights
// stay within 2^11, and five more powers of two are left for the rounding of
// scores, whose last places are whole powers from 2^24 on.
constexpr float LIFT = 7.0f, RISE = 4.0f;
constexpr int THREADS = 256, WAVES = THREADS / 64;

// One launch of a kernel over the requests with `low` to `high` query rows to
// a kv head, in blocks of `rows`.
struct Class {
  int low, high, rows;
  int by_block;                  // attend_tiles_kernel: the work is a list of blocks,
  int blocks;                    // of which it has at most so many if they may be cut
  int whole;                     // every owner takes one segment, none is cut
  int owners;                    // else: shares that the work is cut into
  float* partials;               // [2 owners][rows][D + 2]: values, then maximum and sum
  int64_t* shares;               // [requests + 1] prefix of the work, for the join; by
                                 // block, of the blocks, and after it that of the blocks' work
};

struct AttendArgs {
  const uint16_t* q;
  uint16_t* out;                 // (tokens, q_heads, D) contiguous
  const uint8_t* pages;
  const int32_t *tables, *starts, *lengths;
  int64_t q_token, q_head, tokens, window;
  CacheShape cache;
  int requests, width, q_heads, group;
  float scale;
  int classes;
  Class of[2];
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

// A segment is one kv head and block of query rows of a request. Its work is
// its tiles, and before them what beginning and ending it costs, as tiles: a
// share of many short segments would end late without. (A ragged batch of 128
// requests: 107 us at 8, 115 at 4, 130 at 2, 108 at 12.)
constexpr int SEGMENT_COST = 8;
__device__ __forceinline__ int blocks_of(const AttendArgs& a, const Class& c, const Request& q) {
  return (int)(((int64_t)q.n * a.group + c.rows - 1) / c.rows);
}
__device__ __forceinline__ bool takes(const AttendArgs& a, const Class& c, const Request& q) {
  const int64_t rows = (int64_t)q.n * a.group;
  return q.tiles && rows >= c.low && rows <= c.high;
}
__device__ __forceinline__ int64_t work_of(const AttendArgs& a, const Class& c, const Request& q) {
  if (!takes(a, c, q)) return 0;
  const int64_t blocks = blocks_of(a, c, q);
  return c.by_block ? blocks : a.cache.kv_heads * blocks * (q.tiles + SEGMENT_COST);
}

// What a block of rows attends: positions from `low` on, tiles [t0, t1), and
// the last positions of its first and last row.
struct Block {
  int row0, row1, least_last, most_last, low, t0, t1;
};
__device__ __forceinline__ Block block_of(const AttendArgs& a, const Class& c, const Request& q, int block) {
  const int rows = q.n * a.group, offset = q.length - q.n;
  Block b;
  b.row0 = block * c.rows, b.row1 = min(b.row0 + c.rows, rows) - 1;
  b.least_last = offset + b.row0 / a.group, b.most_last = offset + b.row1 / a.group;
  b.low = (int)max((int64_t)b.least_last - a.window + 1, (int64_t)0);
  b.t0 = b.low / CACHE_TILE;
  b.t1 = max(b.most_last < 0 ? 0 : b.most_last / CACHE_TILE + 1, b.t0);
  return b;
}

// prefix[r] = work before request r, prefix[requests] = all of it.
template <int NTHREADS, typename T>
__device__ __forceinline__ void sum_work(const AttendArgs& a, const Class& c, T* prefix, int64_t* parts) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t base = 0;
  for (int r0 = 0; r0 < a.requests; r0 += NTHREADS) {
    const int r = r0 + tid;
    int64_t v = r < a.requests ? work_of(a, c, request_of(a, r)) : 0;
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
    for (int i = 0; i < NTHREADS / 64; ++i) {
      if (i < wave) before += parts[i];
      base += parts[i];
    }
    if (r < a.requests) prefix[r + 1] = (T)min(before + v, (int64_t)std::numeric_limits<T>::max());
  }
  if (tid == 0) prefix[0] = 0;
  __syncthreads();
}

// A value that all lanes of the wave hold, or that of one, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v, int lane = 0) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// x / d, which nearly always fits 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t d) {
  return (x | d) >> 32 ? x / d : (int64_t)((uint32_t)x / (uint32_t)d);
}

// The work is cut into equal shares, one an owner, of LEAST at least.
constexpr int LEAST = 2;
__device__ __forceinline__ int64_t share_of(const Class& c, int64_t all) {
  return max(quotient(all + c.owners - 1, c.owners), (int64_t)LEAST);
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

// A tile as a buffer: loads then take its base from scalar registers and a
// 32-bit offset, where pointers cost two registers and an addition a load. The
// buffer ends with the tile.
template <int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_resource(const uint8_t* tile) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(tile), 0, 36 * D, 0x00027000);
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

// The variants of attend_rows_kernel: CT column tiles of 8 rows, each with
// what float16 leaves of it beside it, or (WIDE) of 16 rows. Workgroups of a
// compute unit that a variant's registers allow:
constexpr int resident(int d, bool wide, int ct) {
  if (wide) return 2;
  return d == 64 ? (ct == 1 ? 4 : 3) : d == 128 ? (ct == 1 ? 3 : 2) : 2;
}

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
// count with 22 bits at no further product. WIDE blocks have all columns for
// rows. There queries keep their 22 bits by products of their own (bfloat16
// ones too, whose transform sums 32 values of 8 bits: rounded to 11, scores
// would be off by up to 2^-11 of |q| |k|, a factor of the weight that grows
// with the score and that no rounding of the output covers). Weights count with
// 11 bits, each off by up to 2^-11 of itself whatever the score. With values of
// both signs that adds 0.4 of the mean square error that a float16 output has by
// its own rounding (windowed chunks: 2.07e-4 to 2.45e-4 of the output's norm),
// and 0.01 of a bfloat16 one's; a rest of the weights would double the products
// of the values. The running maximum moves only where a row's tile maximum passes
// it by RISE, one vote a tile; then
// the rows agree across lanes on a new one. Sums and outputs are float32.
//
// Two tiles' registers take turns: one is loaded while the other is
// multiplied, and table entries are read a tile further ahead.
//
// Bound by reading the cache where there are few rows: 128 requests of up to
// 8192 positions, 8 kv heads of 128, one token: 504 MB in 107 us, 4.7 TB/s of the
// 4.9 a large copy reaches, vector instructions on 0.60 of the cycles. With 32
// rows a tile they (0.50) and the products (0.18) get as long as the reading: 157
// MB in 55 us, of which about 10 are the waves' start and end.
template <int D, bool WIDE, int CT, bool BF16>
__global__ void __launch_bounds__(THREADS, resident(D, WIDE, CT)) attend_rows_kernel(AttendArgs a, int index) {
  constexpr int PER = WIDE ? 16 : 8, ROWS = PER * CT, GROUPS = D / 32, SETS = Tile<D>::SETS, NIB = D == 64 ? 4 : 8;
  extern __shared__ int64_t prefix[];                    // [requests + 1]
  __shared__ int64_t parts[WAVES];

  const Class& cls = a.of[index];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Magic magic;
  sum_work<THREADS>(a, cls, prefix, parts);
  if (blockIdx.x == 0)
    for (int r = tid; r <= a.requests; r += THREADS) cls.shares[r] = prefix[r];
  const int64_t all = uniform(prefix[a.requests]), share = share_of(cls, all);
  const int owner = (int)blockIdx.x * WAVES + wave;
  const int64_t begin = owner * share, end = min(begin + share, all);

  for (int64_t at = begin; at < end;) {
    // Opaque here, so that addresses made of it are not kept in registers
    // across the tile loop from segment to segment.
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));
    const int n = lane & 15, j = lane >> 4;
    // The minus one of columns 8..15, which take what columns 0..7 leave.
    const float rest = !WIDE && n & 8 ? -1.0f : 0.0f;
    // The segment (request, head, block of rows) that `at` lies in, and the
    // tiles of it that are this wave's.
    const int r = __builtin_amdgcn_readfirstlane(last_at_most(prefix, a.requests + 1, at));
    const Request req = request_of(a, r);
    const int blocks = blocks_of(a, cls, req), rows = req.n * a.group;
    const int64_t before = uniform(prefix[r]);
    const int segment = (int)quotient(at - before, req.tiles + SEGMENT_COST);
    const int head = segment / blocks, block = segment - head * blocks;
    const int64_t seg0 = before + (int64_t)segment * (req.tiles + SEGMENT_COST) + SEGMENT_COST;
    const int64_t seg1 = seg0 + req.tiles;
    const int first = (int)max(at - seg0, (int64_t)0), past = (int)(min(end, seg1) - seg0);
    at = min(end, seg1);
    if (past <= first) continue;
    const bool whole = past - first == req.tiles;
    float* part = cls.partials + ((int64_t)owner * 2 + (first == 0)) * (ROWS * (D + 2));
    // What all of the block's rows attend, most_from .. least_last, needs no
    // mask.
    const Block b = block_of(a, cls, req, block);
    const int row0 = b.row0, row1 = b.row1, least_last = b.least_last;
    const int most_from = (int)max((int64_t)b.most_last - a.window + 1, (int64_t)0);
    const int t0 = max(req.tile0 + first, b.t0), t1 = min(req.tile0 + past, b.t1);
    if (t1 <= t0) {
      // Nothing to attend in this share.
      for (int i = lane; i <= row1 - row0; i += 64) {
        if (!whole) part[ROWS * D + 2 * i] = NONE, part[ROWS * D + 2 * i + 1] = 0.0f;
      }
      if (whole) {
        for (int i = lane; i < (row1 - row0 + 1) * (D / 4); i += 64) {
          const int of = row0 + i / (D / 4);
          uint16_t* out = a.out + ((int64_t)(req.first + of / a.group) * a.q_heads + head * a.group + of % a.group) * D;
          reinterpret_cast<u32x2*>(out)[i % (D / 4)] = u32x2{0u, 0u};
        }
      }
      continue;
    }

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
    // Queries, scaled by a power of two so that float16 holds them whatever
    // the type's range; hi in columns 0..7 and lo in 8..15 of narrow blocks.
    u32x4 qf[CT][GROUPS], ql[WIDE ? CT : 1][WIDE ? GROUPS : 1];
    float qs[CT], rise[CT];
    int last[CT], from[CT];                              // positions this lane's row attends
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int row = row0 + c * PER + (WIDE ? n : n & 7);
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
          if constexpr (WIDE)
            qf[c][k][e] = bits_of(hi);
          else
            qf[c][k][e] = bits_of(f16x2{(_Float16)__builtin_fmaf((float)hi[0], rest, y0),
                                        (_Float16)__builtin_fmaf((float)hi[1], rest, y1)});
          if constexpr (WIDE) ql[c][k][e] = bits_of(f16x2{(_Float16)(y0 - (float)hi[0]), (_Float16)(y1 - (float)hi[1])});
        }
      }
      // An eighth from the query's transform, 2 from both; log2(e) for powers
      // of two.
      // (At least 2^-120: a scale of 0 weighs all positions alike.)
      qs[c] = fmaxf(ldexpf(fabsf(a.scale) * 0.25f * 1.4426950408889634f, power), 0x1p-120f);
      rise[c] = RISE / qs[c];
      last[c] = there ? req.length - req.n + i : -1;
      const int64_t from64 = there ? (int64_t)last[c] - a.window + 1 : 0;
      from[c] = (int)max(from64, (int64_t)0);
    }

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
          for (int c = 0; c < CT; ++c) {
            s[c][u] = mfma(f, qf[c][k], s[c][u]);
            if constexpr (WIDE) s[c][u] = mfma(f, ql[c][k], s[c][u]);
          }
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
          x[e] = WIDE ? v : v + other_half(v);
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
        const float ref = run[c] == NONE ? 0.0f : LIFT - run[c] * qs[c];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float w[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            w[h] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * e + h], qs[c], ref));
            sum[c] += w[h];
          }
          const f16x2 hi = {(_Float16)w[0], (_Float16)w[1]};
          if constexpr (WIDE)
            p[c][e] = bits_of(hi);
          else
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
            const uint32_t one = tile.v[d][e >> 1][(2 * e) & 3], other = tile.v[d][e >> 1][(2 * e + 1) & 3];
            const uint32_t w = __builtin_amdgcn_perm(one, other, pick);
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
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      sum[c] += __shfl_xor(sum[c], 16);
      sum[c] += __shfl_xor(sum[c], 32);
      const float inverse = sum[c] == 0.0f ? 0.0f : 1.0f / sum[c];
      const int row = c * PER + n, of = row0 + row;
      const bool writes = n < PER && of < rows;
      if (writes && !whole && j == 0) {
        part[ROWS * D + 2 * row] = run[c] == NONE ? NONE : run[c] * qs[c];
        part[ROWS * D + 2 * row + 1] = sum[c];
      }
      uint16_t* out = a.out + ((int64_t)(req.first + of / a.group) * a.q_heads + head * a.group + of % a.group) * D;
#pragma unroll
      for (int d = 0; d < SETS; ++d) {
        f32x4* v = &o[c][d * NIB];
        if constexpr (!WIDE) {
#pragma unroll
          for (int m = 0; m < NIB; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[m][e] += other_half(v[m][e]);
        }
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

typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Many query rows to a kv head (chunks and prompts): a workgroup takes a block
// of 32 rows a wave, and unpacks two tiles at a time (of head dimension 256,
// one), as float16, into shared memory, where all its waves read them.
//
// Of head dimension 256 two waves share 32 rows, as one has no registers for
// their outputs beside a second wave on its SIMD: each multiplies half the dims
// of queries and keys, the parts of the scores are exchanged through shared
// memory, and each weighs its half of the values (a wave for all dims, one a
// SIMD: a prompt of 8192 tokens at 490 TFLOP/s, so 556).
//
// The same products as above at 32 x 32 x 16: S^T = K Q^T in one accumulator
// of 32 tokens x 32 rows a tile, O^T += V^T P^T in D / 32. Lane (n, h) of S^T
// holds row n's scores of positions 8 b + 4 h + x of the product's rows; keys
// lie in shared memory with bits 2 and 3 of their token exchanged, so that
// these are tokens 16 c + 8 h .. + 7, the eight that the lane's operand of P^T
// wants. Sixteen-byte vectors of a key row (of a value dim) are permuted by the
// low bits of the row (the dim), so that the sixteen lanes that read in one
// cycle read different banks. Two tiles a step, because the products of one
// tile's scores wait for each other. Two buffers and one barrier a step: while
// one is multiplied the next is unpacked, and the codes after it are on their
// way.
//
// Bound by issue: matrix instructions take 0.49 of the cycles, vector ones (the
// softmax above all) 0.42, and two waves a SIMD overlap them little. Head
// dimension 64: 0.44 and 0.64; 256: 0.34 and 0.43, of which both waves of a pair
// do all the softmax. A prompt of 8192 tokens, 32 heads over 8, 550 GFLOP of 128
// dims without the queries' rest: 0.74 to 0.77 ms, 711 to 747 TFLOP/s (with it
// 1.07 to 1.12 PFLOP/s; a library product of 8192 a side 1.21). Of 64 dims 0.45
// ms, 610, of 256 1.94 ms, 568; float16 and bfloat16 alike.
//
// As in WIDE blocks above, queries count with 22 bits, by a second product of the
// scores (the same prompt without it 0.59 ms), and weights with 11.
constexpr int tile_waves(int d) { return d == 64 ? 4 : 8; }
constexpr int tile_halves(int d) { return d == 256 ? 2 : 1; }  // waves that share 32 rows, each with a part of the dims
constexpr int tile_rows(int d) { return 32 * tile_waves(d) / tile_halves(d); }
constexpr int tile_groups(int d) { return d == 64 ? 3 : 1; }  // workgroups of a compute unit
template <int D, bool BF16>
__global__ void __launch_bounds__(64 * tile_waves(D), tile_groups(D) * tile_waves(D) / 4)
    attend_tiles_kernel(AttendArgs a, int index) {
  constexpr int NW = tile_waves(D), NT = 64 * NW, ROWS = tile_rows(D), STEPS = D / 16;
  constexpr int HALVES = tile_halves(D), GROUPS = D / 32, OWN = GROUPS / HALVES, TAKES = STEPS / HALVES;  // a wave's own

  constexpr int TT = D == 256 ? 1 : 2;                   // tiles of a step
  // Parts of a tile: a dword of key codes, and two dims (a byte) of four tokens'
  // values. A thread takes KN of them.
  constexpr int AHEAD = 2;
  constexpr int KN = 4 * D / NT;
  constexpr int SPAN = D == 64 ? 7 : 15;                 // vectors of a key row that are permuted, less one
  constexpr uint32_t TILE = 64 * D;                      // bytes of a tile's keys, and of its values
  extern __shared__ int64_t dynamic[];                   // costs, then prefix
  __shared__ int64_t parts[NW];
  __shared__ u32x4 keys[2 * TT * TILE / 16], values[2 * TT * TILE / 16];  // [buffer][tile]
  __shared__ f32x4 scores[HALVES == 2 ? NW * 4 * 64 : 1];  // [wave][vector][lane], a wave's part of them
  __shared__ int poison[2];

  const Class& cls = a.of[index];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows32 = wave / HALVES, half = wave % HALVES;
  const int n = lane & 31, h = lane >> 5;
  const Magic magic;
  int64_t* costs = dynamic;                              // [blocks + 1], if blocks may be cut
  int32_t* prefix = reinterpret_cast<int32_t*>(dynamic + (cls.whole ? 0 : cls.blocks + 1));  // [requests + 1]
  if (tid < 2) poison[tid] = -1;                         // seen by all after the barriers of the sums
  sum_work<NT>(a, cls, prefix, parts);
  const int owner = blockIdx.x, heads = a.cache.kv_heads;
  int listed = __builtin_amdgcn_readfirstlane(prefix[a.requests]);
  // (More are asked for only if the requests' rows overlap.)
  if (!cls.whole) listed = min(listed, cls.blocks);
  int64_t begin = owner, end = min(begin + 1, (int64_t)listed * heads);
  if (!cls.whole) {
    // Blocks of a prompt attend more and more tiles, within a window as many:
    // shares are cut by what each block really attends.
    int64_t sum = 0;
    for (int i0 = 0; i0 < listed; i0 += NT) {
      const int i = i0 + tid;
      int64_t v = 0;
      if (i < listed) {
        const int r = last_at_most(prefix, a.requests + 1, i);
        const Block b = block_of(a, cls, request_of(a, r), i - prefix[r]);
        v = b.t1 - b.t0 + SEGMENT_COST;
      }
#pragma unroll
      for (int o = 1; o < 64; o *= 2) {
        const int64_t w = __shfl_up(v, o);
        if (lane >= o) v += w;
      }
      __syncthreads();
      if (lane == 63) parts[wave] = v;
      __syncthreads();
      int64_t before = sum;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        if (w < wave) before += parts[w];
        sum += parts[w];
      }
      if (i < listed) costs[i + 1] = before + v;
    }
    if (tid == 0) costs[0] = 0;
    __syncthreads();
    if (owner == 0) {
      for (int r = tid; r <= a.requests; r += NT) cls.shares[r] = min(prefix[r], listed);
      for (int i = tid; i <= listed; i += NT) cls.shares[a.requests + 1 + i] = costs[i];
    }
    const int64_t all = uniform(costs[listed]) * heads, share = share_of(cls, all);
    begin = owner * share, end = min(begin + share, all);
  }
  // A thread's places in a tile (byte, half of the octet, dword column and
  // octet of a value part) and its operands' in shared memory, opaque so that
  // they stay one register each.
  uint32_t key_at = 4 * tid, key_scale_at = 32 * D + (tid / (D / 8) * GROUPS + tid % GROUPS) * 2;
  uint32_t value_at = 16 * D + tid / 4 * 16;
  uint32_t value_scale_at = 34 * D + ((tid / D * GROUPS + tid / 8 % (D / 8) / 4) * 2 + (tid / 4 & 1)) * 8;
  uint32_t key_row = half * D + n * (2 * D) + (h ^ (n & SPAN)) * 16, value_row = half * (OWN * 2048) + n * 64 + (h ^ (n >> 2 & 3)) * 16;
  asm volatile("" : "+v"(key_at), "+v"(key_scale_at), "+v"(value_at), "+v"(value_scale_at), "+v"(key_row), "+v"(value_row));
  int count = 0;                                         // steps so far; names a buffer's content

  for (int64_t at = begin; at < end;) {
    int r, head, block, first = 0, past = INT32_MAX;
    if (cls.whole) {
      // The longest blocks of a request first, heads next to each other:
      // workgroups are dealt to the chip's eight dies in turn, so that 8 kv
      // heads' keys and values lie in one die's cache each.
      r = __builtin_amdgcn_readfirstlane(last_at_most(prefix, a.requests + 1, at / heads));
      const int before = __builtin_amdgcn_readfirstlane(prefix[r]);
      const uint32_t unit = (uint32_t)(at - (int64_t)before * heads);
      block = __builtin_amdgcn_readfirstlane(prefix[r + 1]) - before - 1 - (int)(unit / (uint32_t)heads);
      head = (int)(unit % (uint32_t)heads);
      at = end;
    } else {
      const int i = __builtin_amdgcn_readfirstlane(last_at_most(costs, listed + 1, at / heads));
      const int64_t cost0 = uniform(costs[i]), cost = uniform(costs[i + 1]) - cost0;
      r = __builtin_amdgcn_readfirstlane(last_at_most(prefix, a.requests + 1, i));
      block = i - __builtin_amdgcn_readfirstlane(prefix[r]);
      head = quotient(at - cost0 * heads, cost);
      const int64_t seg0 = cost0 * heads + head * cost + SEGMENT_COST, seg1 = seg0 - SEGMENT_COST + cost;
      first = (int)max(at - seg0, (int64_t)0), past = (int)(min(end, seg1) - seg0);
      at = min(end, seg1);
      if (past <= first) continue;
    }
    const Request req = request_of(a, r);
    const Block b = block_of(a, cls, req, block);
    const int row0 = b.row0, row1 = b.row1, rows = req.n * a.group, offset = req.length - req.n;
    const int least_last = b.least_last;
    const int most_from = (int)max((int64_t)b.most_last - a.window + 1, (int64_t)0);
    const int t0 = b.t0 + first, t1 = min(b.t0 + min(past, b.t1 - b.t0), b.t1);
    const bool whole = t0 == b.t0 && t1 == b.t1;
    float* part = cls.partials + ((int64_t)owner * 2 + (first == 0)) * (ROWS * (D + 2));

    // This wave's rows and what they attend.
    const int row = 32 * rows32 + n;
    const bool there = row0 + row < rows;
    const int token = there ? (row0 + row) / a.group : 0, of_group = there ? row0 + row - token * a.group : 0;
    const int last = there ? offset + token : -1;
    const int from = there ? (int)max((int64_t)last - a.window + 1, (int64_t)0) : 0;
    const int wave0 = min(row0 + 32 * rows32, row1), wave1 = min(row0 + 32 * rows32 + 31, row1);
    const int wave_least = offset + wave0 / a.group, wave_most = offset + wave1 / a.group;
    const int wave_from = (int)max((int64_t)wave_most - a.window + 1, (int64_t)0);

    const auto* table = (const __attribute__((address_space(4))) int32_t*)(a.tables + (int64_t)r * a.width);
    // The page of a tile; -1 past the share's tiles and where the table names
    // no page of the cache: none of its positions is attended.
    auto page_of = [&](int t) {
      const int id = table[min(t, t1 - 1) >> a.cache.tile_shift];
      return t < t1 && (uint32_t)id < (uint64_t)a.cache.pages ? id : -1;
    };
    auto bytes_of = [&](int t, int page) {
      return a.pages + exl3::cache_tile_at(a.cache, max(page, 0), head, min(t, t1 - 1) & ((1 << a.cache.tile_shift) - 1));
    };
    // The codes and scales of this thread's parts of one tile.
    uint32_t kc[KN], ks[KN];
    u32x4 vc[KN];
    u32x2 vs[KN];
    auto fetch = [&](int t, int page) __attribute__((always_inline)) {
      const auto tile = tile_resource<D>(bytes_of(t, page));
#pragma unroll
      for (int u = 0; u < KN; ++u) {
        kc[u] = __builtin_amdgcn_raw_buffer_load_b32(tile, key_at + u * (4 * NT), 0, 0);
        ks[u] = __builtin_amdgcn_raw_buffer_load_b16(tile, key_scale_at + u * (NT / (D / 8) * GROUPS * 2), 0, 0);
        vc[u] = __builtin_amdgcn_raw_buffer_load_b128(tile, value_at + u * (4 * NT), 0, 0);
        vs[u] = __builtin_amdgcn_raw_buffer_load_b64(tile, value_scale_at + u * (NT / D * GROUPS * 16), 0, 0);
      }
    };
    // Unpacked to a tile of a buffer.
    auto unpack = [&](int buffer, int which) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < KN; ++u) {
        const uint32_t d = tid + u * NT, base = (TT * buffer + which) * (TILE / 16);
        const uint32_t token = d / (D / 8), inside = d % (D / 8);
        const uint32_t vector = 4 * (inside % GROUPS) + inside / GROUPS;
        // Bits 2 and 3 of the token exchanged.
        const uint32_t to = (token & 0x13) | (token & 4) << 1 | (token & 8) >> 1;
        const f16x2 scale = halves_of(ks[u] | ks[u] << 16);
        u32x4 f;
        f[0] = values_of<true>(kc[u], scale, magic);
        f[1] = values_of<false>(kc[u], scale, magic);
        f[2] = values_of<true>(kc[u] >> 8, scale, magic);
        f[3] = values_of<false>(kc[u] >> 8, scale, magic);
        keys[base + to * (D / 8) + (vector ^ (to & SPAN))] = f;
        const uint32_t byte = d & 3, four = d / 4, octet = d / D, column = d / 8 % (D / 8);
        const uint32_t pick = 0x0c000c04u | byte << 16 | byte;
        u32x2 lo, hi;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = __builtin_amdgcn_perm(vc[u][2 * e], vc[u][2 * e + 1], pick);
          const f16x2 scale = halves_of(vs[u][e]);
          lo[e] = values_of<true>(w, scale, magic);
          hi[e] = values_of<false>(w, scale, magic);
        }
        const uint32_t dim = 8 * column + 2 * byte;      // dims 4 x .. 4 x + 3 permute alike
        u32x2* pair = reinterpret_cast<u32x2*>(&values[base + dim * 4 + (octet ^ (dim >> 2 & 3))]) + (four & 1);
        pair[0] = lo, pair[8] = hi;
      }
    };
    // A weight of 0 must not meet a NaN or infinity: in steps that some row
    // does not attend whole, such scales of values count as 0, and the rows
    // that do attend their tokens are seen to after the product.
    auto partial = [&](int t, int missing) {
      return t * CACHE_TILE < most_from || (t + TT) * CACHE_TILE - 1 > least_last || missing < 0;
    };
    auto clean = [&](int buffer, int name) {
#pragma unroll
      for (int u = 0; u < KN; ++u) {
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bits = vs[u][e / 2] >> (16 * (e & 1)) & 0x7fffu;
          if (bits >= 0x7c00u) {
            bad = true;
            vs[u][e / 2] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
          }
        }
        if (bad) poison[buffer] = name;
        asm volatile("" : "+v"(vs[u]));
      }
    };

    // Pages of this step's tiles and of the next two steps'.
    int page[3 * TT];
    auto missing = [&](int i) { return TT == 1 ? page[i] : page[TT * i] | page[TT * i + TT - 1]; };  // < 0 if one is
    if (t0 < t1) {
#pragma unroll
      for (int i = 0; i < 3 * TT; ++i) page[i] = page_of(t0 + i);
      fetch(t0, page[0]);
    }
    // Queries, scaled by a power of two so that float16 holds them.
    u32x4 qf[TAKES], ql[TAKES];                          // and what float16 leaves of them
    float qs, rise;
    {
      const uint16_t* src = a.q + (int64_t)(req.first + token) * a.q_token + (int64_t)(head * a.group + of_group) * a.q_head;
      float x[STEPS][8], top = 0.0f;
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(src + 16 * k + 8 * h);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = there ? widen<BF16>(w[e / 2] >> (16 * (e & 1)) & 0xffffu) : 0.0f;
        exl3::butterfly8(x[k]);
#pragma unroll
        for (int e = 0; e < 8; e += 2) lane_butterfly<32>(x[k][e], x[k][e + 1]);
      }
#pragma unroll
      for (int k = 0; k < STEPS; k += 2)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = x[k][e], z = x[k + 1][e];
          x[k][e] = y + z, x[k + 1][e] = y - z;
          top = fmaxf(top, fmaxf(fabsf(y + z), fabsf(y - z)));
        }
      top = fmaxf(top, __shfl_xor(top, 32));
      int power = 0;
      if (top > 0.0f && top < __builtin_inff()) frexpf(top, &power);
      const float flip = a.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
      for (int k = 0; k < TAKES; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z0 = half ? x[STEPS - TAKES + k][2 * e] : x[k][2 * e];
          const float z1 = half ? x[STEPS - TAKES + k][2 * e + 1] : x[k][2 * e + 1];
          const float y0 = flip * ldexpf(z0, -power), y1 = flip * ldexpf(z1, -power);
          const f16x2 hi = {(_Float16)y0, (_Float16)y1};
          qf[k][e] = bits_of(hi);
          ql[k][e] = bits_of(f16x2{(_Float16)(y0 - (float)hi[0]), (_Float16)(y1 - (float)hi[1])});
        }
      qs = fmaxf(ldexpf(fabsf(a.scale) * 0.25f * 1.4426950408889634f, power), 0x1p-120f);
      rise = RISE / qs;
    }

    float run = NONE, sum = 0.0f;
    f32x16 o[OWN];
#pragma unroll
    for (int d = 0; d < OWN; ++d) o[d] = f32x16{};

    // This lane's vectors of a key row and a value dim: the permutation is an
    // exclusive or of address bits, so one address serves all of a buffer.
    auto key = [&](int k, uint32_t place) {
      return *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(keys) + ((key_row + place) ^ (2 * k & SPAN) << 4) + (2 * k & ~SPAN) * 16);
    };
    auto value = [&](int v, uint32_t place) {
      return *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(values) + ((value_row + place) ^ (v & 1) << 5) + (v >> 1) * 2048);
    };
    if (t0 < t1) {
      const bool dirty = partial(t0, missing(0));
#pragma unroll
      for (int u = 0; u < TT; ++u) {
        if (dirty) clean(count & 1, count);
        unpack(count & 1, u);
        fetch(t0 + u + 1, page[u + 1]);
      }
      __syncthreads();
    }
    for (int t = t0; t < t1; t += TT) {
      const int now = count & 1, then = now ^ 1, pos = t * CACHE_TILE;
      int after[TT];
#pragma unroll
      for (int u = 0; u < TT; ++u) after[u] = page_of(t + 3 * TT + u);
      // The next step's tiles are unpacked after this one's scores are
      // multiplied; of two, whose codes come one by one, the first before.
      const bool dirty = partial(t + TT, missing(1));
      if (dirty) clean(then, count + 1);
      if constexpr (TT == 2) {
        unpack(then, 0);
        fetch(t + 3, page[3]);
      }
      const uint32_t place = now * (TT * TILE);
      // Operands are read from shared memory AHEAD products before their use.
      // The barriers to the scheduler keep that: left alone it reads each right
      // before its product, to save registers, and every product waits for the
      // whole latency (a prompt of 8192 tokens, without the queries' rest: 647 us,
      // with them 582).
      f32x16 s[2] = {};                                  // of two tiles, or of queries and their rest
      u32x4 f[2][AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        f[0][k] = key(k, place);
        if constexpr (TT == 2) f[1][k] = key(k, place + TILE);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < TAKES; ++k) {
        const u32x4 w0 = f[0][k % AHEAD], w1 = f[1][k % AHEAD];
        if constexpr (TT == 2) {
          s[0] = mfma32(w0, qf[k], s[0]);
          s[1] = mfma32(w1, qf[k], s[1]);
          s[0] = mfma32(w0, ql[k], s[0]);
          s[1] = mfma32(w1, ql[k], s[1]);
        } else {
          // Two sums in turn, as the products of one wait for each other.
          s[0] = mfma32(w0, qf[k], s[0]);
          s[1] = mfma32(w0, ql[k], s[1]);
        }
        if (k + AHEAD < TAKES) {
          f[0][k % AHEAD] = key(k + AHEAD, place);
          if constexpr (TT == 2) f[1][k % AHEAD] = key(k + AHEAD, place + TILE);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if constexpr (HALVES == 2) {
        // Both halves add the same two parts, so they agree on every score.
        s[0] += s[1];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          scores[(wave * 4 + e) * 64 + lane] = f32x4{s[0][4 * e], s[0][4 * e + 1], s[0][4 * e + 2], s[0][4 * e + 3]};
        unpack(then, 0);
        fetch(t + 2, page[2]);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; ++e) s[1][e] = scores[((wave ^ 1) * 4 + (e >> 2)) * 64 + lane][e & 3];
      }
      float x[16 * TT];
#pragma unroll
      for (int e = 0; e < 16 * TT; ++e) x[e] = TT == 2 ? s[e >> 4][e & 15] : s[0][e & 15] + s[1][e & 15];
      if (pos < wave_from || pos + TT * CACHE_TILE - 1 > wave_least || missing(0) < 0) {
#pragma unroll
        for (int e = 0; e < 16 * TT; ++e) {
          const int p = pos + 16 * (e >> 3) + 8 * h + (e & 7);
          x[e] = p >= from && p <= last && page[e >> 4] >= 0 ? x[e] : NONE;
          asm volatile("" : "+v"(x[e]));
        }
      }
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 16 * TT; ++e) top = fmaxf(top, x[e]);
      if (__any(top > run + rise)) {
        top = fmaxf(top, run);
        top = fmaxf(top, __shfl_xor(top, 32));
        const float shrink = top == run ? 1.0f : __builtin_amdgcn_exp2f((run - top) * qs);
        run = top;
        sum *= shrink;
#pragma unroll
        for (int d = 0; d < OWN; ++d) o[d] *= shrink;
      }
      const float ref = run == NONE ? 0.0f : LIFT - run * qs;
      // Product v of the output: 16 tokens v / OWN, dims of group v % OWN.
      auto operand = [&](int v) { return value(2 * (v % OWN) + (v / OWN & 1), place + v / OWN / 2 * TILE); };
#pragma unroll
      for (int v = 0; v < 2 * AHEAD; ++v) f[v & 1][v / 2] = operand(v);
      __builtin_amdgcn_sched_barrier(0);
      if (TT == 2 && dirty) clean(then, count + 1);
      if constexpr (TT == 2) {
        unpack(then, 1);
        fetch(t + 4, page[4]);
      }
      u32x4 p[2 * TT];
#pragma unroll
      for (int e = 0; e < 8 * TT; ++e) {
        const f16x2 w = {(_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * e], qs, ref)),
                         (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * e + 1], qs, ref))};
        sum = __builtin_amdgcn_fdot2(w, f16x2{1, 1}, sum, false);
        p[e >> 2][e & 3] = bits_of(w);
      }
#pragma unroll
      for (int v = 0; v < 2 * TT * OWN; ++v) {
        u32x4& w = f[v & 1][v / 2 % AHEAD];
        o[v % OWN] = mfma32(w, p[v / OWN], o[v % OWN]);
        if (v + 2 * AHEAD < 2 * TT * OWN) {
          w = operand(v + 2 * AHEAD);
          if (v & 1) __builtin_amdgcn_sched_barrier(0);
        }
      }

      if (poison[now] == count) {
        // Rows that attend a token whose values of a group are NaN.
#pragma unroll 1
        for (int k = 0; k < TT * CACHE_TILE; ++k) {
          const int id = k < CACHE_TILE ? page[0] : page[TT - 1];
          if (id < 0) continue;
          const uint8_t* scales = bytes_of(t + k / CACHE_TILE, id) + 34 * D;
          const bool in = pos + k >= from && pos + k <= last;
#pragma unroll
          for (int d = 0; d < OWN; ++d) {
            const uint32_t bits = reinterpret_cast<const uint16_t*>(scales)[((k % CACHE_TILE >> 3) * GROUPS + half * OWN + d) * 8 + (k & 7)];
            if (in && (bits & 0x7fffu) >= 0x7c00u) o[d] = f32x16{} + __builtin_nanf("");
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 3 * TT; ++i) page[i] = i < 2 * TT ? page[i + TT] : after[i - 2 * TT];
      ++count;
      __syncthreads();
    }

    // Taken back from the transformed basis: a lane holds dims 32 d + 8 b +
    // 4 h + x of its row.
    sum += __shfl_xor(sum, 32);
    if (there && !whole && h == 0 && half == 0) {
      part[ROWS * D + 2 * row] = run == NONE ? NONE : run * qs;
      part[ROWS * D + 2 * row + 1] = sum;
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    // (From the row again, which is cheaper than two registers in the loop.)
    int of = row0 + row;
    asm volatile("" : "+v"(of));
    uint16_t* out = a.out + ((int64_t)(req.first + of / a.group) * a.q_heads + head * a.group + of % a.group) * D;
#pragma unroll
    for (int d = 0; d < OWN; ++d) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = o[d][e];
#pragma unroll
      for (int level = 1; level < 16; level *= 2)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!(e & level)) {
            const float y = v[e], z = v[e + level];
            v[e] = y + z, v[e + level] = y - z;
          }
#pragma unroll
      for (int e = 0; e < 16; e += 2) lane_butterfly<32>(v[e], v[e + 1]);
      if (!there) continue;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f32x4 y = 0.25f * f32x4{v[4 * b], v[4 * b + 1], v[4 * b + 2], v[4 * b + 3]};
        const int dim = 32 * (half * OWN + d) + 8 * b + 4 * h;
        if (whole) {
          u32x2 w;
          w[0] = narrow<BF16>(y[0] * inverse) | narrow<BF16>(y[1] * inverse) << 16;
          w[1] = narrow<BF16>(y[2] * inverse) | narrow<BF16>(y[3] * inverse) << 16;
          *reinterpret_cast<u32x2*>(out + dim) = w;
        } else {
          *reinterpret_cast<f32x4*>(part + row * D + dim) = y;
        }
      }
    }
  }
}

// The partial results of an output row (token, query head) that more than one
// owner has taken, joined; rows of no work are 0; whole ones are left. Its time
// is that of lookups and loads that wait for each other, so partials are taken
// BATCH at a time with a running maximum. SPREAD waves share one row's partials
// where there are few rows, each with many (384 rows of 85: 14 us with 8 waves,
// 15 with 16 or 4); otherwise a wave takes four rows at once, sixteen lanes
// each, and `run` one after another (51 MB of partials for 88000 rows of head
// dimension 256: 17 us, row by row 28). A prompt's rows are all whole: there it
// only has to see that (6 us for 8192 tokens).
template <int D, bool BF16, int SPREAD>
__global__ void __launch_bounds__(SPREAD > 1 ? 64 * SPREAD : THREADS) attend_join_kernel(AttendArgs a, int run) {
  constexpr int LANES = SPREAD > 1 ? 64 : 16, ROWS = 64 / LANES, PER = D / LANES, VEC = PER < 4 ? PER : 4;
  constexpr int BATCH = SPREAD > 1 || D < 256 ? 4 : 2;  // by the registers they take
  typedef float values __attribute__((ext_vector_type(VEC)));
  typedef uint16_t narrows __attribute__((ext_vector_type(VEC)));
  __shared__ float held[SPREAD][SPREAD > 1 ? D : 1], tops[SPREAD], sums[SPREAD];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t first = SPREAD > 1 ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * WAVES + wave) * run;
  const int64_t past = min(first + run, a.tokens * a.q_heads);
  int64_t found = -1;                                    // the token that `request` is of
  int request = 0;
  for (int64_t at = first; at < past; at += ROWS) {
    const int64_t row = min(at + lane / LANES, past - 1);
    const int64_t token = quotient(row, a.q_heads);
    int r = 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int64_t of = uniform(token, i * LANES);
      if (of != found) {
        // The request: as many starts after the first as are not past the token.
        found = of, request = 0;
        for (int r0 = 0; r0 < a.requests; r0 += 64)
          request += __popcll(__ballot(r0 + lane < a.requests && a.starts[r0 + lane + 1] <= of));
      }
      r = lane / LANES == i ? request : r;
    }
    float x[PER], top = NONE, l = 0.0f;
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] = 0.0f;
    bool writes = at + lane / LANES < past, skip = false;
    if (r < a.requests) {
      const Request req = request_of(a, r);
      if (req.tiles && token >= req.first && token < req.first + req.n) {
        // Field by field, so that the choice is not a load.
        const bool main = a.classes == 1 || takes(a, a.of[0], req);
        auto either = [&](auto Class::*field) { return main ? a.of[0].*field : a.of[1].*field; };
        Class cls;
        cls.rows = either(&Class::rows), cls.owners = either(&Class::owners);
        cls.by_block = either(&Class::by_block), cls.whole = either(&Class::whole);
        cls.shares = either(&Class::shares), cls.partials = either(&Class::partials);
        const int qh = (int)(row - token * a.q_heads), head = qh / a.group;
        const int of = (int)(token - req.first) * a.group + qh - head * a.group;
        const int block = of / cls.rows, line = of - block * cls.rows, stride = cls.rows * (D + 2);
        int64_t w0 = 0, w1 = 0;
        if (cls.whole) {
          skip = true;
        } else {
          int64_t seg0, seg1, all;
          if (cls.by_block) {
            const int64_t* costs = cls.shares + a.requests + 1;
            const int64_t listed = cls.shares[a.requests];
            const int64_t i = min(cls.shares[r] + block, listed - 1), before = costs[i], cost = costs[i + 1] - before;
            all = costs[listed] * a.cache.kv_heads;
            seg1 = before * a.cache.kv_heads + (head + 1) * cost;
            seg0 = seg1 - cost + SEGMENT_COST;
          } else {
            all = cls.shares[a.requests];
            seg0 = cls.shares[r] + ((int64_t)head * blocks_of(a, cls, req) + block) * (req.tiles + SEGMENT_COST) + SEGMENT_COST;
            seg1 = seg0 + req.tiles;
          }
          const int64_t share = share_of(cls, all);
          w0 = quotient(seg0, share);
          w1 = seg1 > seg0 ? quotient(seg1 - 1, share) : w0 - 1;
        }
        if (w0 == w1) writes = false, w1 = w0 - 1;
        const int stats = cls.rows * D + 2 * line;       // a row's maximum and sum in a slot
        for (int64_t w = w0 + wave % SPREAD; w <= w1; w += BATCH * SPREAD) {
          float peak[BATCH], sum[BATCH];
          values v[BATCH][PER / VEC];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            // The first owner's share ends in this segment (slot 1), the others'
            // begin in it (slot 0).
            const int64_t own = min(w + i * SPREAD, w1);
            const float* part = cls.partials + (2 * own + (own == w0)) * stride;
            peak[i] = part[stats], sum[i] = part[stats + 1];
#pragma unroll
            for (int e = 0; e < PER / VEC; ++e)
              v[i][e] = *reinterpret_cast<const values*>(part + line * D + VEC * (e * LANES + lane % LANES));
          }
          float newer = top;
#pragma unroll
          for (int i = 0; i < BATCH; ++i) newer = fmaxf(newer, peak[i]);
          const float keep = top == newer ? 1.0f : __builtin_amdgcn_exp2f(top - newer);
          top = newer;
          l *= keep;
#pragma unroll
          for (int e = 0; e < PER; ++e) x[e] *= keep;
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            // A share without an attended position leaves its values unwritten.
            const bool holds = w + i * SPREAD <= w1 && (peak[i] != NONE || sum[i] != 0.0f);
            const float weight = peak[i] == NONE ? 1.0f : __builtin_amdgcn_exp2f(peak[i] - newer);
            l += holds ? sum[i] * weight : 0.0f;
#pragma unroll
            for (int e = 0; e < PER; ++e) x[e] += holds ? v[i][e / VEC][e % VEC] * weight : 0.0f;
          }
        }
      }
    }
    if constexpr (SPREAD > 1) {
      // One row a workgroup, whose waves agree on what it is.
      if (!writes) return;
#pragma unroll
      for (int e = 0; e < PER; ++e) held[wave][PER * lane + e] = x[e];
      if (lane == 0) tops[wave] = top, sums[wave] = l;
      __syncthreads();
      if (wave != 0) return;
      top = NONE, l = 0.0f;
#pragma unroll
      for (int i = 0; i < SPREAD; ++i) top = fmaxf(top, tops[i]);
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < SPREAD; ++i) {
        const float weight = tops[i] == NONE ? 1.0f : __builtin_amdgcn_exp2f(tops[i] - top);
        l += sums[i] * weight;
#pragma unroll
        for (int e = 0; e < PER; ++e) x[e] += held[i][PER * lane + e] * weight;
      }
    }
    if (writes) {
      const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int e = 0; e < PER / VEC; ++e) {
        narrows w;
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = (uint16_t)narrow<BF16>(x[VEC * e + i] * inverse);
        *reinterpret_cast<narrows*>(a.out + row * D + VEC * (e * LANES + lane % LANES)) = w;
      }
    }
    // Where the last row's request is whole, so are the token's other rows: on
    // to the next token's first.
    if (__builtin_amdgcn_readlane(skip, 63)) at = (found + 1) * a.q_heads - ROWS;
  }
}

constexpr int CUS = 256;

// Variants by the query rows that one kv head has of a request (its new tokens
// times the query heads to a kv head): up to 8 and 16 rows at 22 bits, whose
// cost is the cache's bytes, then 32 to a wave, then blocks that share the work
// of unpacking a tile. Waves of 32 rows are kept for a few blocks' worth, each
// of which reads the cache again. In us, 8 kv heads, both types alike, rows of
// 32 to a wave and blocks that share the unpacking:
//                            64 requests of 2048      one of 131072 positions
//   128 dims, 64 rows            88  175                    90  171
//             128               143  179                   147  176
//             160               194  185                   174  181
//   64 dims,  64 rows            62   79                    60   73
//             96                 88   86                    78   78
// Head dimension 256 has no variants of 16 and 32 rows, for which a wave lacks
// registers: up to 32 rows go in blocks of 8, whose later ones find the tiles in
// the caches (16 rows 101 us, in a variant of 16 with spills 151; blocks of 8 and
// blocks that share the unpacking: 32 rows 168 and 258, one request 196 and 249;
// 48 rows 266 and 260, one request 276 and 253).
enum Variant { ROWS8, ROWS16, ROWS32, TILES };
Variant variant_of(int64_t rows, int head_dim) {
  if (head_dim == 256) return rows <= 32 ? ROWS8 : TILES;
  const int64_t most = head_dim == 128 ? 128 : 64;
  return rows <= 8 ? ROWS8 : rows <= 16 ? ROWS16 : rows <= most ? ROWS32 : TILES;
}
int rows_of(Variant v, int head_dim) { return v == TILES ? tile_rows(head_dim) : 8 << v; }
// Owners that fill the chip: waves of attend_rows_kernel, workgroups of
// attend_tiles_kernel.
int owners_of(Variant v, int head_dim) {
  if (v == TILES) return tile_groups(head_dim) * CUS;
  return CUS * WAVES * resident(head_dim, v == ROWS32, v == ROWS8 ? 1 : 2);
}
// Blocks that a launch which may cut them has at most: fewer than its owners
// take whole, over one kv head.
int64_t blocks_bound(Variant v, int head_dim) { return v == TILES ? 2 * owners_of(v, head_dim) : 0; }
int64_t shares_bytes(Variant v, int requests, int head_dim) {
  return (8 * ((int64_t)requests + 2 + blocks_bound(v, head_dim)) + 15) & ~(int64_t)15;
}
// At most so many segments.
int64_t segments_of(Variant v, int head_dim, int64_t tokens, int group, int requests, int kv_heads) {
  const int rows = rows_of(v, head_dim);
  return ((tokens * group + rows - 1) / rows + requests) * kv_heads;
}
// Blocks of attend_tiles_kernel are dealt whole, and leave no partials, where
// they fill the chip twice.
bool whole_of(Variant v, int head_dim, int64_t segments) {
  return v == TILES && segments >= 2 * owners_of(v, head_dim);
}
int64_t partials_bytes(Variant v, int head_dim) {
  return (int64_t)2 * owners_of(v, head_dim) * rows_of(v, head_dim) * (head_dim + 2) * 4;
}

// The launches of a call: the variant for its longest requests, and beside it,
// so that single tokens keep the variant made for them and up to 16 rows their
// precision, that of 8 rows for requests of up to `few` (where it takes as many
// alone, those: see above). Also where there is one request: how many of the
// tokens are its own, beside padding or under a bound, the GPU alone knows
// (a launch that finds none, as beside a whole prompt, takes 3 to 4 us). A single
// request keeps its bits in blocks of 16 rows.
struct Launches {
  int count, few;
  Variant of[2];
};
Launches launches_of(int64_t tokens, int group, int requests, int head_dim, int64_t max_new) {
  const Variant v = variant_of(std::min(max_new, tokens) * group, head_dim);
  return {v == ROWS8 || (v == ROWS16 && requests == 1) ? 1 : 2, head_dim == 256 ? 32 : v == ROWS16 ? 8 : 16, {v, ROWS8}};
}

template <int D, bool BF16>
int launch_variant(Variant v, const AttendArgs& args, int index, unsigned grid, hipStream_t stream) {
  const Class& c = args.of[index];
  const size_t requests = (size_t)args.requests + 1;
  const size_t lds = v != TILES ? 8 * requests : 4 * requests + (c.whole ? 0 : 8 * ((size_t)c.blocks + 1));
  if (v == ROWS8)
    attend_rows_kernel<D, false, 1, BF16><<<grid, THREADS, lds, stream>>>(args, index);
  else if (v == TILES)
    attend_tiles_kernel<D, BF16><<<grid, 64 * tile_waves(D), lds, stream>>>(args, index);
  else if constexpr (D != 256) {
    if (v == ROWS16)
      attend_rows_kernel<D, false, 2, BF16><<<grid, THREADS, lds, stream>>>(args, index);
    else
      attend_rows_kernel<D, true, 2, BF16><<<grid, THREADS, lds, stream>>>(args, index);
  }
  return check_launch("exl3_cache_attention");
}

template <int D, bool BF16>
int launch_attend(AttendArgs args, int64_t max_new, char* workspace, hipStream_t stream) {
  const Launches launches = launches_of(args.tokens, args.group, args.requests, D, max_new);
  args.classes = launches.count;
  for (int i = 0; i < args.classes; ++i) {
    Class& c = args.of[i];
    const Variant v = launches.of[i];
    c.rows = rows_of(v, D);
    c.low = args.classes == 2 && i == 0 ? launches.few + 1 : 1;
    c.high = args.classes == 2 && i == 1 ? launches.few : INT32_MAX;
    c.owners = owners_of(v, D);
    const int64_t segments = segments_of(v, D, args.tokens, args.group, args.requests, args.cache.kv_heads);
    c.by_block = v == TILES, c.blocks = (int)blocks_bound(v, D);
    c.whole = whole_of(v, D, segments);
    c.shares = reinterpret_cast<int64_t*>(workspace);
    workspace += shares_bytes(v, args.requests, D);
    c.partials = reinterpret_cast<float*>(workspace);
    if (!c.whole) workspace += partials_bytes(v, D);
    const int64_t grid = c.whole ? segments : v == TILES ? c.owners : c.owners / WAVES;
    // A launch has fewer than 2^32 threads.
    if (grid > UINT32_MAX / (64 * tile_waves(D))) return set_error("exl3_cache_attention: too many tokens and heads");
    if (launch_variant<D, BF16>(v, args, i, (unsigned)grid, stream)) return 1;
  }
  const int64_t rows = args.tokens * args.q_heads;
  if (rows <= 2 * CUS) {
    attend_join_kernel<D, BF16, 8><<<(unsigned)rows, 64 * 8, 0, stream>>>(args, 1);
  } else if (rows <= 8 * CUS) {
    attend_join_kernel<D, BF16, 4><<<(unsigned)rows, 64 * 4, 0, stream>>>(args, 1);
  } else {
    // Rows to a wave, by fours; as many as a token or more where all are whole.
    const int64_t run = std::min<int64_t>(std::max<int64_t>(args.of[0].whole ? 64 : 4, rows / (16 * CUS * WAVES) / 4 * 4), 64);
    const int64_t waves = (rows + run - 1) / run;
    attend_join_kernel<D, BF16, 1><<<(unsigned)((waves + WAVES - 1) / WAVES), THREADS, 0, stream>>>(args, (int)run);
  }
  return check_launch("exl3_cache_attention");
}

}  // namespace

extern "C" {

int64_t exl3_cache_attention_workspace(int64_t tokens, int q_heads, int kv_heads, int head_dim,
                                       int requests, int64_t max_new) {
  if (requests < 1 || requests > CACHE_MAX_REQUESTS || (head_dim != 64 && head_dim != 128 && head_dim != 256) ||
      tokens < 0 || kv_heads < 1 || q_heads < kv_heads || max_new < 0)
    return -1;
  const int group = q_heads / kv_heads;
  const Launches launches = launches_of(tokens, group, requests, head_dim, max_new);
  int64_t bytes = 0;
  for (int i = 0; i < launches.count; ++i) {
    const Variant v = launches.of[i];
    bytes += shares_bytes(v, requests, head_dim);
    if (!whole_of(v, head_dim, segments_of(v, head_dim, tokens, group, requests, kv_heads)))
      bytes += partials_bytes(v, head_dim);
  }
  return bytes;
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
  if (!std::isfinite(scale)) return set_error("exl3_cache_attention: scale must be finite");
  if ((reinterpret_cast<uintptr_t>(q) & 15) || q_token % 8 || q_head % 8)
    return set_error("exl3_cache_attention: query rows must be 16-byte aligned");
  if (((reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 7))
    return set_error("exl3_cache_attention: pages, out and workspace must be aligned");
  if (max_new < 0) return set_error("exl3_cache_attention: max_new %lld is negative", (long long)max_new);
  if (workspace_bytes < exl3_cache_attention_workspace(tokens, q_heads, kv_heads, head_dim, requests, max_new))
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
  auto launch = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    auto call = type == 2 ? launch_attend<D, true> : launch_attend<D, false>;
    return call(a, max_new, static_cast<char*>(workspace), (hipStream_t)stream);
  };
  if (head_dim == 64) return launch(std::integral_constant<int, 64>{});
  if (head_dim == 128) return launch(std::integral_constant<int, 128>{});
  return launch(std::integral_constant<int, 256>{});
}

}  // extern "C"
