// MI355X (gfx950) kernels of products with trellis weights as they are stored:
//
//   linear_turn_kernel  rows of x scaled, transformed and split in two float16
//                       parts, in the order of the matrix instructions' operands
//   linear_kernel       tiles decoded in registers and multiplied
//   linear_join_kernel  sums of the shares, taken back and scaled
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
// weights. So z, the transformed rows, lies as [step][set][q][16 columns][8].
// Sets are 16 columns: of up to 8 rows one, float16 parts in columns 0..7 and
// what they leave in 8..15; else two for 16 rows.
struct TurnArgs {
  const uint16_t* x;
  int64_t stride;
  Scales su;
  u32x4* z;
  float* scale;                    // [rows]: what z is multiplied by
  int rows, k, sets;               // sets of all rows: 1, or 2 for each 16
};

// A row is held as 2^p (hi + lo), both float16, with p from the bound
// |z| <= sqrt(128) max |x su|: 22 bits of a value, and places down to 2^-39 of
// the row's largest one, so the products are as exact as float32 makes them.
// A quad of lanes takes a block of 128: two levels across its lanes, five within
// one. A row with an infinity or a NaN is all NaN.
template <bool BF16>
__global__ void __launch_bounds__(256) linear_turn_kernel(TurnArgs a) {
  __shared__ uint32_t tops[4];
  const int row = blockIdx.x, tid = threadIdx.x, q = tid & 3;
  const uint16_t* x = a.x + row * a.stride;
  uint32_t top = 0;                // of magnitudes as bits: NaN above infinity above all else
  for (int i = tid; i < a.k / 8; i += 256) {
    const u32x4 w = reinterpret_cast<const u32x4*>(x)[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = widen<BF16>(w[e / 2] >> (16 * (e & 1)) & 0xffffu) * a.su.at(8 * i + e);
      top = max(top, __builtin_bit_cast(uint32_t, v) & 0x7fffffffu);
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
  top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  // 2^11 > sqrt(128) 2^7.5 ... z stays below 2^15.
  const bool finite = top < 0x7f800000u;
  const int power = max((int)(top >> 23), 1) - 126 - 11;
  if (tid == 0) a.scale[row] = finite ? ldexpf(1.0f, power) : __builtin_nanf("");
  const int m = a.sets == 1 ? row : row & 15, set0 = a.sets == 1 ? 0 : row / 16 * 2;
  for (int unit = tid >> 2; unit < a.k / HAD; unit += 64) {
    float v[32];                   // [step 4][tile 2][half 2][2]: channels 32 step + 16 tile + 8 half + 2 q + e
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int at = HAD * unit + 8 * i + 2 * q;
      const uint32_t w = *reinterpret_cast<const uint32_t*>(x + at);
      v[2 * i] = widen<BF16>(w & 0xffffu) * a.su.at(at);
      v[2 * i + 1] = widen<BF16>(w >> 16) * a.su.at(at + 1);
    }
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
        const float y = v[8 * s + 2 * e], w = v[8 * s + 2 * e + 1];
        const _Float16 hy = (_Float16)y, hw = (_Float16)w;
        hi[e] = __builtin_bit_cast(uint32_t, f16x2{hy, hw});
        lo[e] = pair_of(y - (float)hy, w - (float)hw);
      }
      u32x4* z = a.z + ((int64_t)(4 * unit + s) * a.sets + set0) * 64 + q * 16 + m;
      z[0] = hi;
      z[a.sets == 1 ? 8 : 64] = lo;
    }
  }
}

// ------------------------------------------------------------ product

struct LinearArgs {
  const uint32_t* words;
  const u32x4* z;
  float* partials;                 // [split][rows][n]
  int rows, k, n, bits, splits, sets;
};

// The hash of a state, s M + A. A state has 16 bits: two 24-bit products, which
// run at full rate where a 32-bit one takes four times as long. (The empty asm
// keeps the compiler from making one 32-bit product of them.)
template <int CB>
__device__ __forceinline__ uint32_t hash_of(uint32_t s) {
  uint32_t high = s * (hash_mult(CB) >> 24);
  asm("" : "+v"(high));
  return (high << 24) + (s * (hash_mult(CB) & 0xffffffu) + (CB == 0 ? 64248484u : 0u));
}

// The values of two states (exl3_codebook.h): the sum of a hash's bytes, scaled,
// or the sum of its halves.
template <int CB>
__device__ __forceinline__ uint32_t values_of(uint32_t s0, uint32_t s1) {
  const uint32_t x0 = hash_of<CB>(s0), x1 = hash_of<CB>(s1);
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

template <bool WIDE, int CB, int SETS, int CT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) linear_kernel(LinearArgs a) {
  constexpr int ACCS = SETS == 1 ? 1 : SETS / 2;
  __shared__ f32x4 sums[WAVES][CT * ACCS][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, q = lane >> 4;
  const int tiles_n = a.n / 16, column0 = blockIdx.x * CT, split = blockIdx.y, block = blockIdx.z;
  const int steps = a.k / 32, parts = a.splits * WAVES, part = split * WAVES + wave;
  const int begin = (int)((int64_t)steps * part / parts), end = (int)((int64_t)steps * (part + 1) / parts);
  const int u = 8 * (n & 7) + 2 * q + (n >> 3), bits = a.bits;
  const Window late = window_of(4 * bits * (u + 1), bits), early = window_of(4 * bits * u + 2 * bits, bits);

  const int64_t row_bytes = (int64_t)tiles_n * 32 * bits;
  const char* next = reinterpret_cast<const char*>(a.words) + 2 * begin * row_bytes + (int64_t)column0 * 32 * bits;
  auto load = [&]() __attribute__((always_inline)) {
    Words<WIDE, CT> r;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const char* at = next + t * row_bytes + c * (32 * bits);
        auto word = [&](uint32_t byte) { return *reinterpret_cast<const uint32_t*>(at + byte); };
        r.w[c][t][0] = word(late.at0), r.w[c][t][1] = word(late.at1);
        if constexpr (WIDE) r.w[c][t][2] = word(early.at0), r.w[c][t][3] = word(early.at1);
      }
    next += 2 * row_bytes;
    return r;
  };
  f32x4 acc[CT][ACCS];
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int m = 0; m < ACCS; ++m) acc[c][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  auto multiply = [&](const Words<WIDE, CT>& r, int step) __attribute__((always_inline)) {
    const u32x4* z = a.z + ((int64_t)step * a.sets + block * SETS) * 64 + lane;
    u32x4 b[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) b[s] = z[s * 64];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      u32x4 f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t v = __builtin_amdgcn_alignbit(r.w[c][t][0], r.w[c][t][1], late.shift);
        const uint32_t s3 = v & 0xffffu, s2 = __builtin_amdgcn_ubfe(v, bits, 16);
        uint32_t s1, s0;
        if constexpr (WIDE) {
          const uint32_t e = __builtin_amdgcn_alignbit(r.w[c][t][2], r.w[c][t][3], early.shift);
          s1 = e & 0xffffu, s0 = __builtin_amdgcn_ubfe(e, bits, 16);
        } else {
          s1 = __builtin_amdgcn_ubfe(v, 2 * bits, 16), s0 = __builtin_amdgcn_ubfe(v, 3 * bits, 16);
        }
        f[2 * t] = values_of<CB>(s0, s1);
        f[2 * t + 1] = values_of<CB>(s2, s3);
      }
#pragma unroll
      for (int s = 0; s < SETS; ++s) acc[c][s / 2] = mfma(f, b[s], acc[c][s / 2]);
    }
  };

  if (begin < end) {
    Words<WIDE, CT> even = load(), odd = even;
    for (int step = begin; step < end; step += 2) {
      if (step + 1 < end) odd = load();
      multiply(even, step);
      if (step + 1 == end) break;
      if (step + 2 < end) even = load();
      multiply(odd, step + 1);
    }
  }
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int m = 0; m < ACCS; ++m) sums[wave][c * ACCS + m][lane] = acc[c][m];
  __syncthreads();
  for (int i = tid; i < CT * ACCS * 64; i += 64 * WAVES) {
    const int of = i >> 6, l = i & 63, c = of / ACCS, m = of % ACCS;
    if (SETS == 1 && (l & 8)) continue;
    f32x4 v = sums[0][of][l];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += sums[w][of][l];
    if constexpr (SETS == 1)
#pragma unroll
      for (int w = 0; w < WAVES; ++w) v += sums[w][of][l + 8];
    const int row = block * 16 * ACCS + 16 * m + (l & 15), column = 16 * (column0 + c) + 4 * (l >> 4);
    if (row < a.rows && column < a.n)
      *reinterpret_cast<f32x4*>(a.partials + ((int64_t)split * a.rows + row) * a.n + column) = v;
  }
}

// ------------------------------------------------------------ join

struct JoinArgs {
  const float *partials, *scale;
  Scales sv;
  uint16_t* out;
  int rows, n, splits;
};

// Sixteen lanes take a block of 128 outputs of a row, eight each.
template <bool BF16>
__global__ void __launch_bounds__(256) linear_join_kernel(JoinArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  const int lane = threadIdx.x & 63, blocks = a.n / HAD;
  const bool there = unit < (int64_t)a.rows * blocks;
  const int row = there ? (int)(unit / blocks) : 0, column = there ? (int)(unit % blocks) * HAD + 8 * (lane & 15) : 8 * (lane & 15);
  float v[8] = {};
  for (int s = 0; s < a.splits; ++s) {
    const f32x4* p = reinterpret_cast<const f32x4*>(a.partials + ((int64_t)s * a.rows + row) * a.n + column);
    const f32x4 x = p[0], y = p[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += x[e], v[4 + e] += y[e];
  }
  exl3::quad_transform(v, lane);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float o4 = __shfl_xor(v[e], 4);
    v[e] = lane & 4 ? o4 - v[e] : v[e] + o4;
    const float o8 = __shfl_xor(v[e], 8);
    v[e] = lane & 8 ? o8 - v[e] : v[e] + o8;
  }
  const float scale = a.scale[row] * ROOT;
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = narrow<BF16>(v[2 * e] * scale * a.sv.at(column + 2 * e)) |
           narrow<BF16>(v[2 * e + 1] * scale * a.sv.at(column + 2 * e + 1)) << 16;
  if (there) *reinterpret_cast<u32x4*>(a.out + (int64_t)row * a.n + column) = w;
}

// ------------------------------------------------------------ plan

// How a call is cut.
struct Plan {
  int sets, blocks;                // of columns of z in all; row blocks of a launch
  int columns, waves, groups;      // column tiles of a wave, waves, column groups
  int splits;
  int64_t z_bytes, scale_bytes, partial_bytes;
};

constexpr int CUS = 256;

Plan plan_of(int64_t rows, int64_t k, int64_t n) {
  Plan p{};
  const int sets = rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 32 ? 4 : 8;  // of a row block
  p.blocks = sets <= 2 ? 1 : (int)((rows + 8 * sets - 1) / (8 * sets));
  p.sets = sets * p.blocks;
  p.columns = sets <= 2 ? 2 : 4;
  p.waves = sets <= 2 ? 8 : 4;
  p.groups = (int)((n / 16 + p.columns - 1) / p.columns);
  const int64_t want = (int64_t)2 * CUS * 8 / p.waves;
  const int64_t most = std::max<int64_t>(1, k / 32 / (2 * p.waves));
  p.splits = (int)std::min(most, std::max<int64_t>(1, (want + (int64_t)p.groups * p.blocks - 1) / ((int64_t)p.groups * p.blocks)));
  p.z_bytes = k / 32 * p.sets * 1024;
  p.scale_bytes = (4 * rows + 15) & ~(int64_t)15;
  p.partial_bytes = 4 * (int64_t)p.splits * rows * n;
  return p;
}

template <bool WIDE, int CB>
void launch_product(const Plan& p, const LinearArgs& a, hipStream_t stream) {
  const dim3 grid(p.groups, p.splits, p.blocks);
  switch (p.sets / p.blocks) {
    case 1: linear_kernel<WIDE, CB, 1, 2, 8><<<grid, 512, 0, stream>>>(a); break;
    case 2: linear_kernel<WIDE, CB, 2, 2, 8><<<grid, 512, 0, stream>>>(a); break;
    case 4: linear_kernel<WIDE, CB, 4, 4, 4><<<grid, 256, 0, stream>>>(a); break;
    default: linear_kernel<WIDE, CB, 8, 4, 4><<<grid, 256, 0, stream>>>(a); break;
  }
}

}  // namespace

extern "C" {

int64_t exl3_linear_workspace(int64_t rows, int64_t k, int64_t n) {
  if (rows < 0 || rows > INT32_MAX || k < HAD || n < HAD || k % HAD || n % HAD || k > 1 << 24 || n > 1 << 24) return -1;
  const Plan p = plan_of(rows, k, n);
  return p.z_bytes + p.scale_bytes + p.partial_bytes;
}

int exl3_linear(const void* x, int64_t stride, int64_t rows, int type, const uint16_t* words, const void* su,
                const void* sv, int half_scales, int64_t k, int64_t n, int K, int cb, void* out, void* workspace,
                int64_t workspace_bytes, void* stream) {
  if (K < 1 || K > 8) return set_error("exl3_linear: K must be in 1..8, got %d", K);
  if (cb < 0 || cb > 2) return set_error("exl3_linear: cb must be 0, 1, or 2, got %d", cb);
  if (type < 1 || type > 2) return set_error("exl3_linear: rows are float16 or bfloat16");
  const int64_t need = exl3_linear_workspace(rows, k, n);
  if (need < 0) return set_error("exl3_linear: bad sizes: %lld rows of %lld by %lld", (long long)rows, (long long)k, (long long)n);
  if (!rows) return 0;
  if ((reinterpret_cast<uintptr_t>(x) & 15) || stride % 8 || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15) || (reinterpret_cast<uintptr_t>(words) & 3))
    return set_error("exl3_linear: rows, out and workspace must be 16-byte aligned, words 4-byte");
  if (workspace_bytes < need) return set_error("exl3_linear: workspace of %lld bytes is too small", (long long)workspace_bytes);
  const Plan p = plan_of(rows, k, n);
  hipStream_t s = (hipStream_t)stream;
  char* w = static_cast<char*>(workspace);
  TurnArgs t{};
  t.x = static_cast<const uint16_t*>(x), t.stride = stride, t.su = {su, half_scales & 1};
  t.z = reinterpret_cast<u32x4*>(w), t.scale = reinterpret_cast<float*>(w + p.z_bytes);
  t.rows = (int)rows, t.k = (int)k, t.sets = p.sets;
  if (type == 2)
    linear_turn_kernel<true><<<(unsigned)rows, 256, 0, s>>>(t);
  else
    linear_turn_kernel<false><<<(unsigned)rows, 256, 0, s>>>(t);
  if (check_launch("exl3_linear")) return 1;
  LinearArgs a{};
  a.words = reinterpret_cast<const uint32_t*>(words), a.z = t.z;
  a.partials = reinterpret_cast<float*>(w + p.z_bytes + p.scale_bytes);
  a.rows = (int)rows, a.k = (int)k, a.n = (int)n, a.bits = K, a.splits = p.splits, a.sets = p.sets;
  if (K > 5)
    cb == 0 ? launch_product<true, 0>(p, a, s) : cb == 1 ? launch_product<true, 1>(p, a, s) : launch_product<true, 2>(p, a, s);
  else
    cb == 0 ? launch_product<false, 0>(p, a, s) : cb == 1 ? launch_product<false, 1>(p, a, s) : launch_product<false, 2>(p, a, s);
  if (check_launch("exl3_linear")) return 1;
  JoinArgs j{};
  j.partials = a.partials, j.scale = t.scale, j.sv = {sv, half_scales >> 1 & 1};
  j.out = static_cast<uint16_t*>(out), j.rows = (int)rows, j.n = (int)n, j.splits = p.splits;
  const int64_t units = rows * (n / HAD);
  if (type == 2)
    linear_join_kernel<true><<<(unsigned)((units + 15) / 16), 256, 0, s>>>(j);
  else
    linear_join_kernel<false><<<(unsigned)((units + 15) / 16), 256, 0, s>>>(j);
  return check_launch("exl3_linear");
}

}  // extern "C"
