// MI355X (gfx950) kernels of the token side of a 4-bit attention cache:
//
//   rotary_kernel   rotary positions of queries and keys, and the gradient
//   step_kernel     block tables, slots and positions from request lengths
//   append_kernel   keys and values to 4-bit cache entries, the keys (and
//                   queries) rotated on the way
//   read_kernel     cache entries back to keys and values
//
// The cache's layout and group transform: exl3_cache_layout.h; attention over
// it: exl3_attention.hip.
#include <hip/hip_bf16.h>
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

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------ element types

struct F32 {
  typedef float type;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  static __device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};

// The 16-bit types: `word` is the bits of one, values are rounded to nearest.
template <typename T, uint32_t (*NARROW)(float), float (*WIDEN)(uint32_t)>
struct Half {
  typedef uint16_t type;
  static __device__ __forceinline__ float load(const uint16_t* p) { return WIDEN(*p); }
  static __device__ __forceinline__ void store(uint16_t* p, float v) { *p = (uint16_t)NARROW(v); }
  static __device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = WIDEN(w[i] & 0xffffu), v[2 * i + 1] = WIDEN(w[i] >> 16);
  }
  static __device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = NARROW(v[2 * i]) | NARROW(v[2 * i + 1]) << 16;
    *reinterpret_cast<u32x4*>(p) = w;
  }
};

__device__ __forceinline__ uint32_t narrow_f16(float v) {
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ float widen_f16(uint32_t w) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)w);
}
__device__ __forceinline__ uint32_t narrow_bf16(float v) {
  return __builtin_bit_cast(uint16_t, (__bf16)v);
}
__device__ __forceinline__ float widen_bf16(uint32_t w) {
  return __builtin_bit_cast(float, w << 16);
}
typedef Half<_Float16, narrow_f16, widen_f16> F16;
typedef Half<__bf16, narrow_bf16, widen_bf16> BF16;

// A (tokens, heads, D) tensor whose last axis is contiguous.
template <typename T>
struct Rows {
  T* data;
  int64_t token, head;  // strides in elements
  __device__ __forceinline__ T* at(int64_t t, int h) const {
    return data + t * token + (int64_t)h * head;
  }
  Rows from(int64_t t) const { return {data ? data + t * token : data, token, head}; }
};

// Positions, int64 if wide, from token t on.
const void* positions_from(const void* positions, bool wide, int64_t t) {
  return positions ? static_cast<const char*>(positions) + t * (wide ? 8 : 4) : positions;
}

// A launch has fewer than 2^32 threads along an axis: more tokens than so many
// blocks of 256 take go in several.
constexpr int64_t MOST_BLOCKS = 1 << 23;
// launch(first token, tokens), by parts of MOST_BLOCKS blocks of `per_block`.
template <typename F>
int in_parts(int64_t tokens, int64_t per_block, F launch) {
  for (int64_t t = 0; t < tokens; t += MOST_BLOCKS * per_block)
    if (const int status = launch(t, std::min(tokens - t, MOST_BLOCKS * per_block))) return status;
  return 0;
}

// Cosines and sines of one block's tokens, [token][pair], in shared memory:
// every head of a token turns by the same angles. Angles and their functions
// are taken in 64 bits and rounded once: a float32 product at position 10^6
// would be off by 0.06 radians, and float32 functions of the exact fraction of
// a turn (1.2e-7) put three times as many rotated keys over the edge to the
// next code as rounding does.
__device__ __forceinline__ void turn_table(const void* positions, bool wide, const double* freq,
                                           int pairs, float magnitude, float sign, int64_t t0,
                                           int tokens, float* cosines, float* sines) {
  for (int i = threadIdx.x; i < tokens * pairs; i += blockDim.x) {
    const int t = i / pairs, p = i - t * pairs;
    const double at = wide ? (double)static_cast<const int64_t*>(positions)[t0 + t]
                           : (double)static_cast<const int32_t*>(positions)[t0 + t];
    const double turns = at * (freq[p] * 0.15915494309189535);
    double s, c;
    sincospi(2.0 * (turns - rint(turns)), &s, &c);
    cosines[i] = (float)(c * magnitude);
    sines[i] = (float)(s * magnitude) * sign;
  }
}

// Eight of a token's values at dims d0.., turned if they lie in the rotary
// part. `row` is the head's row, `cosines`/`sines` the token's table. In the
// half layout the other value of each pair is `pairs` away.
template <typename E>
__device__ __forceinline__ void turned8(const typename E::type* row, int d0, int pairs, bool half,
                                        const float* cosines, const float* sines, float (&v)[8]) {
  E::load8(row + d0, v);
  if (d0 >= 2 * pairs) return;
  if (half) {
    const bool second = d0 >= pairs;
    const int p = second ? d0 - pairs : d0;
    float w[8];
    E::load8(row + (second ? d0 - pairs : d0 + pairs), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = cosines[p + i], s = sines[p + i];
      v[i] = second ? v[i] * c + w[i] * s : v[i] * c - w[i] * s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = cosines[d0 / 2 + i], s = sines[d0 / 2 + i];
      const float a = v[2 * i], b = v[2 * i + 1];
      v[2 * i] = a * c - b * s;
      v[2 * i + 1] = b * c + a * s;
    }
  }
}

// ------------------------------------------------------------ rotary

struct RotaryArgs {
  const void* positions;
  const double* freq;
  int q_heads, heads, d, pairs, wide, half;
  float magnitude, sign;
};

// y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin of every pair, the other values
// copied. A block takes a token, makes its angles once and turns all heads of
// q and k: per pair one 64-bit product and one sincospi for all heads, so the pass is bound by reading and writing the rows (8192 tokens of
// 32 + 8 heads of 128 in bfloat16, 168 MB that the last-level cache holds:
// 26 us, 6.4 TB/s; one token 3 us, a launch).
// A thread turns both values of its pairs and writes them where it read them
// (out may be the input). VEC: rows are 16-byte aligned, pairs a multiple of
// 8 and D of 16, so a unit is 16 values in two wide loads.
template <typename E, bool VEC>
__global__ void __launch_bounds__(256)
    rotary_kernel(Rows<const typename E::type> q, Rows<const typename E::type> k,
                  Rows<typename E::type> q_out, Rows<typename E::type> k_out, RotaryArgs a) {
  extern __shared__ float table[];
  const int64_t t = blockIdx.x;
  float *c = table, *s = table + a.pairs;
  turn_table(a.positions, a.wide, a.freq, a.pairs, a.magnitude, a.sign, t, 1, c, s);
  __syncthreads();
  const int units = VEC ? a.d / 16 : (a.d + 1) / 2;
  const int all = a.heads * units;
  for (int i = threadIdx.x; i < all; i += blockDim.x) {
    const int h = i / units, u = i - h * units;
    const bool is_k = h >= a.q_heads;
    const typename E::type* in = is_k ? k.at(t, h - a.q_heads) : q.at(t, h);
    typename E::type* out = is_k ? k_out.at(t, h - a.q_heads) : q_out.at(t, h);
    if constexpr (VEC) {
      // Turned units first (8 pairs each), copied ones of 16 after them.
      const int turned = a.pairs / 8;
      float x[8], y[8];
      int dx, dy;
      if (u < turned) {
        dx = a.half ? 8 * u : 16 * u;
        dy = a.half ? 8 * u + a.pairs : 16 * u + 8;
      } else {
        dx = 16 * u;
        dy = dx + 8;
      }
      E::load8(in + dx, x);
      E::load8(in + dy, y);
      if (u < turned) {
        if (a.half) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float co = c[8 * u + e], si = s[8 * u + e], v = x[e];
            x[e] = v * co - y[e] * si;
            y[e] = y[e] * co + v * si;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float c0 = c[8 * u + e], s0 = s[8 * u + e], v = x[2 * e], w = y[2 * e];
            const float c1 = c[8 * u + 4 + e], s1 = s[8 * u + 4 + e];
            x[2 * e] = v * c0 - x[2 * e + 1] * s0;
            x[2 * e + 1] = x[2 * e + 1] * c0 + v * s0;
            y[2 * e] = w * c1 - y[2 * e + 1] * s1;
            y[2 * e + 1] = y[2 * e + 1] * c1 + w * s1;
          }
        }
      }
      E::store8(out + dx, x);
      E::store8(out + dy, y);
    } else {
      if (u < a.pairs) {
        const int i1 = a.half ? u : 2 * u, i2 = a.half ? u + a.pairs : 2 * u + 1;
        const float x = E::load(in + i1), y = E::load(in + i2);
        E::store(out + i1, x * c[u] - y * s[u]);
        E::store(out + i2, y * c[u] + x * s[u]);
      } else {
        // Copied as bits: their values do not change.
        out[2 * u] = in[2 * u];
        if (2 * u + 1 < a.d) out[2 * u + 1] = in[2 * u + 1];
      }
    }
  }
}

template <typename E>
int launch_rotary(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                  int64_t k_head, void* q_out, int64_t qo_token, int64_t qo_head, void* k_out,
                  int64_t ko_token, int64_t ko_head, const RotaryArgs& args, int64_t tokens,
                  bool vec, hipStream_t stream) {
  typedef typename E::type T;
  Rows<const T> rq{static_cast<const T*>(q), q_token, q_head}, rk{static_cast<const T*>(k), k_token, k_head};
  Rows<T> oq{static_cast<T*>(q_out), qo_token, qo_head}, ok{static_cast<T*>(k_out), ko_token, ko_head};
  const size_t lds = 2 * sizeof(float) * args.pairs;
  return in_parts(tokens, 1, [&](int64_t t, int64_t n) {
    RotaryArgs part = args;
    part.positions = positions_from(args.positions, args.wide, t);
    auto kernel = vec ? rotary_kernel<E, true> : rotary_kernel<E, false>;
    kernel<<<(unsigned)n, 256, lds, stream>>>(rq.from(t), rk.from(t), oq.from(t), ok.from(t), part);
    return check_launch("exl3_rotary");
  });
}

// ------------------------------------------------------------ step plan

struct StepArgs {
  const int32_t *cached, *fresh, *free_pages, *taken;
  int32_t* tables;
  int64_t* slots;
  int32_t *positions, *starts, *lengths, *taken_out, *status;
  int64_t max_tokens;
  int requests, width, page_shift, free_count;
};

constexpr int STEP_THREADS = 1024;

// Inclusive sum over the block; *total gets the block's sum. `parts` is
// STEP_THREADS / 64 values of shared memory.
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* parts, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int64_t w = __shfl_up(v, o);
    if (lane >= o) v += w;
  }
  __syncthreads();
  if (lane == 63) parts[wave] = v;
  __syncthreads();
  int64_t before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < STEP_THREADS / 64; ++i) {
    if (i < wave) before += parts[i];
    sum += parts[i];
  }
  *total = sum;
  return v + before;
}

// Last index i of [0, n) with at[i] <= x; at[0] <= x.
__device__ __forceinline__ int last_at_most(const int32_t* at, int n, int x) {
  int lo = 0;
  while (n > 1) {
    const int half = n >> 1;
    if (at[lo + half] <= x) lo += half;
    n -= half;
  }
  return lo;
}

// Request r holds have = ceil(cached / P) pages and takes need more for its
// new tokens, the free list's entries from taken + (needs before r) on. Every
// block sums the same prefixes over all requests (a few KB that lie in L2:
// cheaper than a launch of its own for the sums), keeps them in shared memory,
// and fills its share of the new table entries and of the tokens' slots. A
// slot in a new page takes the page from the free list itself, so no block
// reads what another writes. Bound by latency: two reads and two dependent
// look-ups deep (256 requests of a token 6 us, 1531 of up to 96 tokens 11 us).
__global__ void __launch_bounds__(STEP_THREADS) step_kernel(StepArgs a) {
  extern __shared__ int32_t prefix[];  // starts [requests + 1], needs [requests + 1]
  __shared__ int64_t parts[STEP_THREADS / 64];
  int32_t *starts = prefix, *needs = prefix + a.requests + 1;
  const int page = 1 << a.page_shift, tid = threadIdx.x;
  const int64_t room = (int64_t)a.width << a.page_shift;
  auto have_of = [&](int r) {
    return (int)min((int64_t)(((int64_t)max(a.cached[r], 0) + page - 1) >> a.page_shift), (int64_t)a.width);
  };
  int64_t tokens = 0, pages = 0;
  int outgrown = 0, missing = 0;
  for (int r0 = 0; r0 < a.requests; r0 += STEP_THREADS) {
    const int r = r0 + tid;
    int64_t fresh = 0, need = 0;
    if (r < a.requests) {
      const int64_t cached = max(a.cached[r], 0);
      fresh = max(a.fresh[r], 0);
      const int64_t length = cached + fresh;
      outgrown |= length > room;
      need = min((length + page - 1) >> a.page_shift, (int64_t)a.width) - have_of(r);
      if (blockIdx.x == 0) a.lengths[r] = (int32_t)min(length, (int64_t)INT32_MAX);
    }
    int64_t sum_tokens, sum_pages;
    const int64_t end_tokens = tokens + block_sum(fresh, parts, &sum_tokens);
    const int64_t end_pages = pages + block_sum(need, parts, &sum_pages);
    if (r < a.requests) {
      starts[r + 1] = (int32_t)min(end_tokens, (int64_t)INT32_MAX);
      needs[r + 1] = (int32_t)end_pages;
    }
    tokens += sum_tokens;
    pages += sum_pages;
  }
  if (tid == 0) starts[0] = needs[0] = 0;
  __syncthreads();
  const int64_t taken = max(a.taken[0], 0);
  if (blockIdx.x == 0) {
    for (int r = tid; r <= a.requests; r += STEP_THREADS) a.starts[r] = starts[r];
    // New tokens begin in a page that is held in part: without one (of a step
    // that ran out) they have no slot, though this step needs no page. (Looked
    // up here and asked for at the end, so that nothing waits for it.)
    for (int r = tid; r < a.requests; r += STEP_THREADS) {
      const int64_t cached = max(a.cached[r], 0);
      if (starts[r + 1] > starts[r] && (cached & (page - 1)) && cached < room)
        missing |= a.tables[(int64_t)r * a.width + (cached >> a.page_shift)] < 0;
    }
  }
  auto new_page = [&](int64_t i) { return taken + i < a.free_count ? a.free_pages[taken + i] : -1; };
  const int64_t step = (int64_t)gridDim.x * STEP_THREADS, first = (int64_t)blockIdx.x * STEP_THREADS + tid;
  for (int64_t i = first; i < pages; i += step) {
    const int r = last_at_most(needs, a.requests + 1, (int)i);
    a.tables[(int64_t)r * a.width + have_of(r) + (i - needs[r])] = new_page(i);
  }
  for (int64_t t = first; t < a.max_tokens; t += step) {
    int64_t slot = -1;
    int32_t position = 0;
    if (t < tokens) {
      const int r = last_at_most(starts, a.requests + 1, (int)t);
      const int64_t at = (int64_t)max(a.cached[r], 0) + (t - starts[r]);
      position = (int32_t)min(at, (int64_t)INT32_MAX);
      if (at < room) {
        const int p = (int)(at >> a.page_shift), have = have_of(r);
        const int32_t id = p < have ? a.tables[(int64_t)r * a.width + p] : new_page(needs[r] + p - have);
        if (id >= 0) slot = ((int64_t)id << a.page_shift) + (at & (page - 1));
      }
    }
    a.slots[t] = slot;
    a.positions[t] = position;
  }
  if (blockIdx.x == 0) {
    outgrown = __syncthreads_or(outgrown), missing = __syncthreads_or(missing);
    if (tid == 0) {
      a.taken_out[0] = (int32_t)min(taken + pages, (int64_t)max((int64_t)a.free_count, taken));
      a.status[0] = (taken + pages > a.free_count || missing ? 1 : 0) | (outgrown ? 2 : 0) |
                    (tokens > a.max_tokens ? 4 : 0);
    }
  }
}

// ------------------------------------------------------------ append and read

struct CellArgs {
  CacheShape cache;
  const int64_t* slots;
  const void* positions;
  const double* freq;
  int64_t tokens;
  int q_heads, pairs, wide, half, oct_shift;
  float magnitude;
};

// The dword of (token, 8 dims from d0) and the scale of its group, as offsets
// in the cache; `value` chooses values over keys.
struct Cell {
  int64_t code, scale;
};
__device__ __forceinline__ Cell cell_of(const CacheShape& c, int64_t slot, int head, int d0,
                                        bool value) {
  const int page_shift = c.tile_shift + 5, groups = c.head_dim / 32;
  const int64_t page = slot >> page_shift;
  const int in_page = (int)(slot & (((int64_t)1 << page_shift) - 1));
  const int64_t tile = exl3::cache_tile_at(c, page, head, in_page >> 5);
  const int t = in_page & 31, group = d0 >> 5, j = (d0 >> 3) & 3, d = c.head_dim;
  if (!value)
    return {tile + 4 * (t * (d / 8) + j * groups + group), tile + 32 * d + 2 * (t * groups + group)};
  return {tile + 16 * d + 4 * (((t >> 3) * (d / 8) + (d0 >> 3)) * 8 + (t & 7)),
          tile + 34 * d + 2 * (((t >> 3) * groups + group) * 8 + (t & 7))};
}

// Units of eight values of a block's tokens, four lanes (a quad) to a group of
// 32. With TOK = 8, the quads of eight tokens lie next to each other: one
// octet's value dwords, when their slots follow each other, are then whole
// 32-byte sectors of the cache instead of single dwords of eight (8191 tokens
// of 16 heads of 64: append 22.4 us, with TOK = 1 24.3; read 13.8 and 15.8).
// TOK = 1 spreads a few tokens over the chip (64 tokens of 32 + 16 heads of 128:
// append 4.0 us, with TOK = 8 4.9).
template <int TOK>
struct Units {
  int all, at;                   // units of the block, this thread's
  __device__ __forceinline__ explicit Units(int units)
      : all(TOK == 1 ? units : units * TOK), at(blockIdx.y * 256 + threadIdx.x) {}
  __device__ __forceinline__ bool more() const { return at < all; }
  __device__ __forceinline__ void next() { at += gridDim.y * 256; }
  __device__ __forceinline__ int token() const { return TOK == 1 ? 0 : at / 4 % TOK; }
  __device__ __forceinline__ int unit() const { return TOK == 1 ? at : at / (4 * TOK) * 4 + at % 4; }
};

// A quad of lanes takes one group of 32 values of a key or value, eight each:
// three butterfly levels in a lane, two by quad permutation, then the group's
// largest magnitude, scale and codes. Keys turn by their position on the way,
// in 32 bits, and queries beside them, so a decode step is one launch and one
// read of the projection. Bound by reading and writing the rows (8191 tokens of
// 3 x 16 heads of 64, float16, queries turned: 77 MB in 23 us, 3.3 TB/s).
template <typename E, bool TURN, int TOK>
__global__ void __launch_bounds__(256)
    append_kernel(Rows<const typename E::type> q, Rows<const typename E::type> k,
                  Rows<const typename E::type> v, Rows<typename E::type> q_out,
                  uint8_t* __restrict__ pages, CellArgs a) {
  extern __shared__ float table[];
  const int64_t t0 = (int64_t)blockIdx.x * TOK;
  const int tokens = (int)min((int64_t)TOK, a.tokens - t0);
  float *cosines = table, *sines = table + TOK * a.pairs;
  if constexpr (TURN) {
    turn_table(a.positions, a.wide, a.freq, a.pairs, a.magnitude, 1.0f, t0, tokens, cosines, sines);
    __syncthreads();
  }
  const int lane = threadIdx.x & 63, oct_shift = a.oct_shift, octs = 1 << oct_shift;
  const int64_t capacity = a.cache.pages << (a.cache.tile_shift + 5);
  // Units of a token: keys, values, then queries; a multiple of four each, so
  // a quad's lanes always work on the same group.
  const int kv = a.cache.kv_heads * octs;
  for (Units<TOK> i(2 * kv + a.q_heads * octs); i.more(); i.next()) {
    const int t = i.token(), u = i.unit();
    if (t >= tokens) continue;                           // a whole quad
    const float *c = cosines + t * a.pairs, *s = sines + t * a.pairs;
    float x[8];
    if (u >= 2 * kv) {
      if constexpr (TURN) {
        const int h = (u - 2 * kv) >> oct_shift, d0 = 8 * ((u - 2 * kv) & (octs - 1));
        turned8<E>(q.at(t0 + t, h), d0, a.pairs, a.half, c, s, x);
        E::store8(q_out.at(t0 + t, h) + d0, x);
      }
      continue;
    }
    const bool value = u >= kv;
    const int h = (value ? u - kv : u) >> oct_shift, d0 = 8 * ((value ? u - kv : u) & (octs - 1));
    if (value)
      E::load8(v.at(t0 + t, h) + d0, x);
    else if constexpr (TURN)
      turned8<E>(k.at(t0 + t, h), d0, a.pairs, a.half, c, s, x);
    else
      E::load8(k.at(t0 + t, h) + d0, x);
    exl3::quad_transform(x, lane);
    float most = 0.0f;
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] *= 0.125f;
      most = fmaxf(most, fabsf(x[e]));
      finite &= fabsf(x[e]) < __builtin_inff();  // false for NaN too
    }
    if (!finite) most = __builtin_inff();
    most = fmaxf(most, exl3::quad_other<1>(most));
    most = fmaxf(most, exl3::quad_other<2>(most));
    // Eight significant bits, so that the products with codes are exact in
    // f16; then to f16, which takes bits only below 2^-14.
    const float wanted = fminf(most * (1.0f / 7.0f), 9344.0f);
    uint32_t bits = narrow_f16(widen_bf16(narrow_bf16(wanted)));
    const float scale = widen_f16(bits);
    const float inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float r = fminf(fmaxf(rintf(x[e] * inverse), -7.0f), 7.0f);
      // Keys: even dims in nibbles 0..3, odd ones in 4..7.
      const int nibble = value ? e : (e >> 1) + 4 * (e & 1);
      word |= (uint32_t)((int)r + 8) << (4 * nibble);
    }
    if (!(most < __builtin_inff())) {
      bits = 0x7e00u;
      word = 0x88888888u;
    }
    const int64_t slot = a.slots[t0 + t];
    if (slot < 0 || slot >= capacity) continue;
    const Cell cell = cell_of(a.cache, slot, h, d0, value);
    *reinterpret_cast<uint32_t*>(pages + cell.code) = word;
    if (!(lane & 3)) *reinterpret_cast<uint16_t*>(pages + cell.scale) = (uint16_t)bits;
  }
}

// The values that entries stand for: H ((c - 8) s) / 4, a quad a group; zeros
// for slots outside the cache. Bound by writing them (43 MB in all in 14 us).
template <typename E, int TOK>
__global__ void __launch_bounds__(256)
    read_kernel(const uint8_t* __restrict__ pages, Rows<typename E::type> k, Rows<typename E::type> v,
                CellArgs a) {
  const int64_t t0 = (int64_t)blockIdx.x * TOK;
  const int tokens = (int)min((int64_t)TOK, a.tokens - t0);
  const int lane = threadIdx.x & 63, oct_shift = a.oct_shift, octs = 1 << oct_shift;
  const int64_t capacity = a.cache.pages << (a.cache.tile_shift + 5);
  const int kv = a.cache.kv_heads * octs;
  for (Units<TOK> i(2 * kv); i.more(); i.next()) {
    const int t = i.token(), u = i.unit();
    if (t >= tokens) continue;
    const bool value = u >= kv;
    const int h = (value ? u - kv : u) >> oct_shift, d0 = 8 * ((value ? u - kv : u) & (octs - 1));
    const int64_t slot = a.slots[t0 + t];
    float x[8];
    if (slot >= 0 && slot < capacity) {
      const Cell cell = cell_of(a.cache, slot, h, d0, value);
      const uint32_t word = *reinterpret_cast<const uint32_t*>(pages + cell.code);
      const float scale = widen_f16(*reinterpret_cast<const uint16_t*>(pages + cell.scale));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int nibble = value ? e : (e >> 1) + 4 * (e & 1);
        x[e] = (float)((int)((word >> (4 * nibble)) & 15u) - 8) * scale;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    }
    exl3::quad_transform(x, lane);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= 0.25f;
    E::store8((value ? v : k).at(t0 + t, h) + d0, x);
  }
}

// Tokens next to each other in a block: eight once the blocks fill the chip.
constexpr int64_t MANY_TOKENS = 2048;
// Blocks for `tokens` of `units` values, `passes` of each at most: what a thread
// does in turn waits in turn, but a block's angles are made once (8191 tokens:
// append 22.4 us with 4 passes, 23.7 with 2, 28.2 with 1; read 15.0, 13.8, 13.9).
template <int TOK>
dim3 grid_of(int64_t tokens, int64_t units, int64_t passes) {
  const int64_t all = (units * TOK + 255) / 256;
  return dim3((unsigned)((tokens + TOK - 1) / TOK), (unsigned)((all + passes - 1) / passes));
}

template <typename E>
int launch_append(const void* q, int64_t q_token, int64_t q_head, void* q_out, const void* k,
                  int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                  uint8_t* pages, const CellArgs& args, hipStream_t stream) {
  typedef typename E::type T;
  const int64_t d = args.cache.head_dim;
  Rows<const T> rq{static_cast<const T*>(q), q_token, q_head}, rk{static_cast<const T*>(k), k_token, k_head},
      rv{static_cast<const T*>(v), v_token, v_head};
  Rows<T> oq{static_cast<T*>(q_out), args.q_heads * d, d};
  auto launch = [&](auto tok) {
    constexpr int TOK = decltype(tok)::value;
    const int64_t units = (2 * (int64_t)args.cache.kv_heads + args.q_heads) * (d / 8);
    const size_t lds = 2 * sizeof(float) * TOK * args.pairs;
    auto kernel = args.pairs ? append_kernel<E, true, TOK> : append_kernel<E, false, TOK>;
    return in_parts(args.tokens, TOK, [&](int64_t t, int64_t n) {
      CellArgs part = args;
      part.slots = args.slots + t, part.positions = positions_from(args.positions, args.wide, t);
      part.tokens = n;
      kernel<<<grid_of<TOK>(n, units, TOK == 1 ? 1 : 4), 256, lds, stream>>>(
          rq.from(t), rk.from(t), rv.from(t), oq.from(t), pages, part);
      return check_launch("exl3_cache_append");
    });
  };
  if (args.tokens >= MANY_TOKENS) return launch(std::integral_constant<int, 8>{});
  return launch(std::integral_constant<int, 1>{});
}

template <typename E>
int launch_read(const uint8_t* pages, void* k, void* v, const CellArgs& args, hipStream_t stream) {
  typedef typename E::type T;
  const int64_t token = (int64_t)args.cache.kv_heads * args.cache.head_dim, head = args.cache.head_dim;
  const Rows<T> rk{static_cast<T*>(k), token, head}, rv{static_cast<T*>(v), token, head};
  const int64_t units = 2 * (int64_t)args.cache.kv_heads * (head / 8);
  auto launch = [&](auto tok, int64_t passes) {
    constexpr int TOK = decltype(tok)::value;
    return in_parts(args.tokens, TOK, [&](int64_t t, int64_t n) {
      CellArgs part = args;
      part.slots = args.slots + t, part.tokens = n;
      read_kernel<E, TOK><<<grid_of<TOK>(n, units, passes), 256, 0, stream>>>(pages, rk.from(t), rv.from(t), part);
      return check_launch("exl3_cache_read");
    });
  };
  if (args.tokens >= MANY_TOKENS) return launch(std::integral_constant<int, 8>{}, 2);
  return launch(std::integral_constant<int, 1>{}, 1);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// log2 of the units of eight values in a head.
int oct_shift_of(int head_dim) { return head_dim == 64 ? 3 : head_dim == 128 ? 4 : 5; }

// Rows that 16-byte loads may read: `per` elements make 16 bytes.
bool wide_rows(const void* p, int64_t token, int64_t head, int64_t per) {
  return !p || (aligned16(p) && token % per == 0 && head % per == 0);
}

int check_cache(const char* what, int64_t pages, int page_size, int kv_heads, int head_dim,
                CacheShape* cache) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error("%s: head_dim must be 64, 128 or 256, got %d", what, head_dim);
  if (page_size < 32 || page_size > 256 || (page_size & (page_size - 1)))
    return set_error("%s: page_size must be 32, 64, 128 or 256, got %d", what, page_size);
  if (pages < 0 || pages > INT32_MAX || kv_heads < 1 || kv_heads > 65535)
    return set_error("%s: bad cache shape", what);
  int shift = 0;
  while ((CACHE_TILE << shift) < page_size) ++shift;
  *cache = CacheShape{pages, kv_heads, head_dim, shift};
  return 0;
}

}  // namespace

extern "C" {

int exl3_rotary(const void* q, int64_t q_token, int64_t q_head, void* q_out, int64_t qo_token,
                int64_t qo_head, int q_heads, const void* k, int64_t k_token, int64_t k_head,
                void* k_out, int64_t ko_token, int64_t ko_head, int k_heads, int64_t tokens,
                int head_dim, int type, const void* positions, int wide_positions,
                const double* frequencies, int pairs, int layout, float magnitude, int inverse,
                void* stream) {
  if (tokens < 0 || tokens > INT32_MAX || q_heads < 0 || k_heads < 0 || q_heads + k_heads < 1 ||
      q_heads + k_heads > 65535)
    return set_error("exl3_rotary: bad sizes");
  if (head_dim < 1 || head_dim > 4096 || pairs < 1 || 2 * pairs > head_dim)
    return set_error("exl3_rotary: needs 1 <= 2 * pairs <= head_dim <= 4096");
  if (type < 0 || type > 2 || layout < 0 || layout > 1)
    return set_error("exl3_rotary: bad type or layout");
  if (!tokens) return 0;
  RotaryArgs args{};
  args.positions = positions, args.freq = frequencies;
  args.q_heads = q_heads, args.heads = q_heads + k_heads, args.d = head_dim, args.pairs = pairs;
  args.wide = wide_positions, args.half = layout == 0;
  args.magnitude = magnitude, args.sign = inverse ? -1.0f : 1.0f;
  const int64_t per = type == 0 ? 4 : 8;
  const bool vec = pairs % 8 == 0 && head_dim % 16 == 0 && wide_rows(q, q_token, q_head, per) &&
                   wide_rows(k, k_token, k_head, per) && wide_rows(q_out, qo_token, qo_head, per) &&
                   wide_rows(k_out, ko_token, ko_head, per);
  hipStream_t s = (hipStream_t)stream;
  auto launch = type == 0 ? launch_rotary<F32> : type == 1 ? launch_rotary<F16> : launch_rotary<BF16>;
  return launch(q, q_token, q_head, k, k_token, k_head, q_out, qo_token, qo_head, k_out, ko_token,
                ko_head, args, tokens, vec, s);
}

int exl3_plan_step(const int32_t* cached, const int32_t* fresh, int requests, int32_t* tables,
                   int width, const int32_t* free_pages, int free_count, const int32_t* taken,
                   int page_size, int64_t max_tokens, int64_t* slots, int32_t* positions,
                   int32_t* starts, int32_t* lengths, int32_t* taken_out, int32_t* status,
                   void* stream) {
  CacheShape cache;
  if (check_cache("exl3_plan_step", 0, page_size, 1, 64, &cache)) return 1;
  if (requests < 1 || requests > CACHE_MAX_REQUESTS)
    return set_error("exl3_plan_step: requests must be in 1..%d, got %d", CACHE_MAX_REQUESTS, requests);
  if (width < 1 || (int64_t)width * page_size > INT32_MAX || (int64_t)width * requests > INT32_MAX)
    return set_error("exl3_plan_step: bad table width %d", width);
  if (free_count < 0 || max_tokens < 0 || max_tokens > INT32_MAX)
    return set_error("exl3_plan_step: bad sizes");
  StepArgs a{};
  a.cached = cached, a.fresh = fresh, a.free_pages = free_pages, a.taken = taken, a.tables = tables;
  a.slots = slots, a.positions = positions, a.starts = starts, a.lengths = lengths;
  a.taken_out = taken_out, a.status = status, a.max_tokens = max_tokens, a.requests = requests;
  a.width = width, a.page_shift = cache.tile_shift + 5, a.free_count = free_count;
  const int64_t want = (max_tokens + STEP_THREADS - 1) / STEP_THREADS;
  const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min<int64_t>(want, 256));
  step_kernel<<<blocks, STEP_THREADS, 8 * (requests + 1), (hipStream_t)stream>>>(a);
  return check_launch("exl3_plan_step");
}

int exl3_cache_append(const void* q, int64_t q_token, int64_t q_head, void* q_out, int q_heads,
                      const void* k, int64_t k_token, int64_t k_head, const void* v,
                      int64_t v_token, int64_t v_head, int64_t tokens, int type,
                      const int64_t* slots, const void* positions, int wide_positions,
                      const double* frequencies, int pairs, int layout, float magnitude,
                      void* pages, int64_t num_pages, int page_size, int kv_heads, int head_dim,
                      void* stream) {
  CellArgs a{};
  if (check_cache("exl3_cache_append", num_pages, page_size, kv_heads, head_dim, &a.cache)) return 1;
  if (tokens < 0 || tokens > INT32_MAX || q_heads < 0 || q_heads > 65535 || type < 0 || type > 2 ||
      layout < 0 || layout > 1)
    return set_error("exl3_cache_append: bad sizes, type or layout");
  if (pairs < 0 || 2 * pairs > head_dim || pairs % 8)
    return set_error("exl3_cache_append: pairs must be a multiple of 8 up to head_dim / 2, got %d", pairs);
  if (!aligned16(pages) || (q_heads && !aligned16(q_out)))
    return set_error("exl3_cache_append: pages and q_out must be 16-byte aligned");
  if (q_heads && !pairs) return set_error("exl3_cache_append: queries are only taken to be turned");
  const int64_t per = type == 0 ? 4 : 8;
  if (!wide_rows(q_heads ? q : nullptr, q_token, q_head, per) || !wide_rows(k, k_token, k_head, per) ||
      !wide_rows(v, v_token, v_head, per))
    return set_error("exl3_cache_append: rows must be 16-byte aligned");
  if (!tokens) return 0;
  a.slots = slots, a.positions = positions, a.freq = frequencies, a.tokens = tokens;
  a.q_heads = q_heads, a.pairs = pairs, a.wide = wide_positions, a.half = layout == 0;
  a.magnitude = magnitude, a.oct_shift = oct_shift_of(head_dim);
  auto launch = type == 0 ? launch_append<F32> : type == 1 ? launch_append<F16> : launch_append<BF16>;
  return launch(q, q_token, q_head, q_out, k, k_token, k_head, v, v_token, v_head,
                static_cast<uint8_t*>(pages), a, (hipStream_t)stream);
}

int exl3_cache_read(const void* pages, int64_t num_pages, int page_size, int kv_heads, int head_dim,
                    const int64_t* slots, int64_t tokens, int type, void* k, void* v, void* stream) {
  CellArgs a{};
  if (check_cache("exl3_cache_read", num_pages, page_size, kv_heads, head_dim, &a.cache)) return 1;
  if (tokens < 0 || tokens > INT32_MAX || type < 0 || type > 2)
    return set_error("exl3_cache_read: bad sizes or type");
  if (!aligned16(pages) || !aligned16(k) || !aligned16(v))
    return set_error("exl3_cache_read: pages, k and v must be 16-byte aligned");
  if (!tokens) return 0;
  a.slots = slots, a.tokens = tokens;
  a.oct_shift = oct_shift_of(head_dim);
  const uint8_t* p = static_cast<const uint8_t*>(pages);
  auto launch = type == 0 ? launch_read<F32> : type == 1 ? launch_read<F16> : launch_read<BF16>;
  return launch(p, k, v, a, (hipStream_t)stream);
}

}  // extern "C"
