// out = act(x W^T + b) + r: a matrix product of 16-bit or 8-bit operands on the matrix
// instructions, summed in fp32, with the bias, the activation and the residual in its epilogue
// (amlike_linear_*).
//
// Layout.  A k-tile is 128 bytes of a row: 64 columns in 16 bits, 128 in 8.  Both kinds of matrix
// instruction used (16x16x32 bf16 / f16, 16x16x128 scaled e4m3) then look alike: with g = l / 16,
// lane l of a fragment holds row l % 16 and, of its k-tile, the 16-byte pieces g and g + 4 -- as
// two 16-bit instructions of one piece each, or as a single 8-bit one, whose scale operand is that
// of the columns 32 g .. 32 g + 31 (a lane's scale is not that of its own values).
// W is the instructions' first operand and x the second, so that a lane's results are 4 outputs of
// one row of x per fragment.
// The 8-bit instruction aligns the products of a few neighbouring columns to the largest of them
// and drops what lies more than 13 binary places below it (measured: 2^16 + 2^2 is 2^16, 2^16 + 2^3
// is whole), which leaves a relative error of about 1.5e-5 in a sum of normal values whatever its
// length (where a sum cancels, relative to the summands): below a hundredth of the rounding of a bf16
// (up to 2^-8) or 8-bit output (2^-4), a thirtieth of an f16 one's (2^-11), too much for an fp32 one.
// For an fp32 output the 8-bit operands are therefore widened to bf16, which holds value times scale
// exactly but for scales at the ends of their range (is_far_x), and multiplied there (kMx8Exact), at
// half the matrix rate.  A wave that met such a scale takes its sums once more, group by group
// (far_sums).
//   W:      [k-tile][row, padded to 64][128 bytes], zeros behind both ends
//   scales: [k-tile / 4][row, padded to 64][k-tile % 4][4 bytes], 2^0 behind both ends and for groups
//           of zeros  (8 bits only)
//
// This header holds the kernels and their launches; each kind of product is compiled in a file of its
// own (linear_bf16.hip ...), the choice of a form and the host side are in linear.hip.
#ifndef KALDI_AMD_CSRC_LINEAR_KERNELS_H_
#define KALDI_AMD_CSRC_LINEAR_KERNELS_H_

#include <algorithm>
#include <cmath>

#include "dense_common.h"

namespace amlike {

constexpr int kTileBytes = 128;  // of a row in a k-tile
constexpr int kChunks = 8;       // 16-byte pieces of it

struct LinearArgs {
  const uint8_t *x, *x_scales;  // [rows][k], row strides in bytes
  const uint8_t *w;
  const uint32_t *w_scales;
  const float *bias;  // [n padded to 64]
  const void *res;
  void *out;
  uint8_t *out_scales;
  int64_t ldx, ld_xs, ldr, ldo, ld_os;
  int32_t rows, k, n, n_pad, k_tiles;
  int32_t act, res_type, out_type;  // res_type -1: none
  int32_t max_blocks;               // of a launch
};

// The kernels' kinds of product: a layer's type, or 8-bit operands with bf16 products.
constexpr int kMx8Exact = 4;
__host__ __device__ constexpr bool IsMx8(int kind) { return kind == AMLIKE_MX8 || kind == kMx8Exact; }

// The forms of the tile kernel (linear_pipe_kernel's arguments) and of the kernel for few rows.
struct TileForm {
  int wn, wm, mf, stages, ks;
  bool copy;
};
constexpr TileForm kTileForms[7] = {{4, 2, 8, 2, 1, true}, {2, 2, 4, 2, 1, true}, {2, 2, 4, 2, 2, true}, {1, 4, 1, 4, 1, true},
                                    {1, 4, 1, 4, 2, true}, {1, 4, 1, 2, 1, false}, {2, 2, 4, 2, 1, false}};
struct ThinForm {
  int nt, mt;
};
constexpr ThinForm kThinForms[5] = {{1, 1}, {2, 1}, {1, 2}, {2, 2}, {2, 4}};

// Waves a SIMD holds of a form, by its registers.
constexpr int WavesPerSimd(int kind, const TileForm &f) { return !f.copy && f.mf == 1 && kind != kMx8Exact ? 4 : 2; }
// As many blocks as the device holds at once, by waves and LDS, in eights.
inline int BlocksHeld(int kind, const TileForm &f, int units) {
  const int lds = f.ks * (64 * f.wn + 16 * f.mf * f.wm) * (f.stages * kTileBytes + (IsMx8(kind) ? 32 : 0)) + 64;
  return std::max(8, (units * std::min(4 * WavesPerSimd(kind, f) / (f.wn * f.wm * f.ks), 163840 / lds)) & ~7);
}
// Which form a layer takes: of kThinForms if `thin`, else of kTileForms.  copy: 16-byte pieces of x can be copied as
// they are; far_apart: its rows lie more than 4 MB apart.
struct LinearChoice {
  bool thin;
  int form;
};
LinearChoice ChooseLinear(int kind, int out_type, int64_t rows, int k_tiles, int n_pad, bool copy, bool far_apart, int units);

// The layer in one of the kinds, on `st`: defined for each kind in its own file.
template <int KIND>
int LaunchLinear(const LinearArgs &a, hipStream_t st);

// Bytes [at, at + 16) of a row of x as columns, those at the row's end `bytes` and beyond as 0.
__device__ __forceinline__ u32x4 load_chunk(const uint8_t *row, int at, int bytes) {
  typedef u32x4 u32x4_byte __attribute__((aligned(1)));
  u32x4 q = {0, 0, 0, 0};
  if (at + 16 <= bytes) {
    q = *reinterpret_cast<const u32x4_byte *>(row + at);
  } else if (at < bytes) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (at + i < bytes) q[i >> 2] |= (uint32_t)row[at + i] << (8 * (i & 3));
  }
  return q;
}
// The four scale bytes of k-tile kt of a row of x; 2^0 behind the last group.
__device__ __forceinline__ uint32_t load_scales(const uint8_t *row, int kt, int groups) {
  uint32_t s = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) s |= (kt * 4 + i < groups ? (uint32_t)row[kt * 4 + i] : 127u) << (8 * i);
  return s;
}

#ifdef AMLIKE_LINEAR_KERNELS

template <int TYPE>
struct Frag;
template <>
struct Frag<AMLIKE_BF16> {
  typedef __bf16 vec __attribute__((ext_vector_type(8)));
};
template <>
struct Frag<AMLIKE_F16> {
  typedef _Float16 vec __attribute__((ext_vector_type(8)));
};
typedef int i32x8 __attribute__((ext_vector_type(8)));

// A 16-byte piece of e4m3 values times 2^(scale byte - 127 + lift), as two fragments of bf16.  The
// conversion takes the exponent of its scale as it stands.
__device__ __forceinline__ void widen(const u32x4 p, uint32_t scale_byte, int lift, Frag<AMLIKE_BF16>::vec out[2]) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const float s = as_float((scale_byte << 23) + ((uint32_t)lift << 23));
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)p[q], s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)p[q], s, true);
    out[q >> 1][(q & 1) * 4 + 0] = a[0];
    out[q >> 1][(q & 1) * 4 + 1] = a[1];
    out[q >> 1][(q & 1) * 4 + 2] = b[0];
    out[q >> 1][(q & 1) * 4 + 3] = b[1];
  }
}

// bf16 holds multiples of 2^-133 below 2^128, an 8-bit value is a multiple of 2^-9 up to 448 times
// 2^(byte - 127).  With x lifted by 2^3, and W lowered by as much, every value of x under the bytes 0
// (rows and groups of zeros have it) to 243 fits, and every one of W under the bytes 6 to 249.  Beyond,
// x would become infinite and W lose its last bits.
constexpr int kLift = 3;
// Whether one of four scale bytes of x is 244 or more (NaN's 255 too): its low seven bits plus 12
// reach the eighth, and that is set.
__device__ __forceinline__ bool is_far_x(uint32_t scales) {
  return (((scales & 0x7f7f7f7fu) + 0x0c0c0c0cu) & scales & 0x80808080u) != 0;
}
// Whether one of four scale bytes of W is below 6.  (Packed W has no byte over 247.)
__device__ __forceinline__ bool is_far_w(uint32_t scales) { return ((scales - 0x06060606u) & ~scales & 0x80808080u) != 0; }

// What a lane feeds the matrix instructions from pieces g and g + 4 of a row in one k-tile, and the
// word of the row's four scales.  lift: kLift for x, -kLift for W.
template <int KIND>
struct Operand {
  u32x4 p[2];
  int scale;
  __device__ __forceinline__ void set(u32x4 p0, u32x4 p1, uint32_t scales, int g, int /*lift*/) {
    p[0] = p0;
    p[1] = p1;
    scale = (int)(scales >> (8 * g));  // the instruction takes the lowest byte
  }
};
template <>
struct Operand<kMx8Exact> {
  Frag<AMLIKE_BF16>::vec v[4];
  __device__ __forceinline__ void set(u32x4 p0, u32x4 p1, uint32_t scales, int g, int lift) {
    widen(p0, scales >> (8 * (g >> 1)) & 0xff, lift, v);  // piece c holds columns of group c / 2
    widen(p1, scales >> (16 + 8 * (g >> 1)) & 0xff, lift, v + 2);
  }
};

// One k-tile of a fragment of W and one of x: c += W x^T.
template <int TYPE>
__device__ __forceinline__ f32x4v tile_product(const Operand<TYPE> &ow, const Operand<TYPE> &ox, f32x4v c) {
  if constexpr (TYPE == kMx8Exact) {
#pragma unroll
    for (int h = 0; h < 4; ++h) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ow.v[h], ox.v[h], c, 0, 0, 0);
    return c;
  } else if constexpr (TYPE == AMLIKE_MX8) {
    const u32x4 *w = ow.p, *x = ox.p;
    const i32x8 a = {(int)w[0][0], (int)w[0][1], (int)w[0][2], (int)w[0][3], (int)w[1][0], (int)w[1][1], (int)w[1][2], (int)w[1][3]};
    const i32x8 b = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], (int)x[1][0], (int)x[1][1], (int)x[1][2], (int)x[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, ow.scale, 0, ox.scale);
  } else {
    typedef typename Frag<TYPE>::vec V;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const V a = __builtin_bit_cast(V, ow.p[h]), b = __builtin_bit_cast(V, ox.p[h]);
      if constexpr (TYPE == AMLIKE_BF16) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
      else c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    return c;
  }
}

// ---- 8 bits as bf16: scales at the ends of their range ------------------------------------------------
// tile_product of widened 8-bit operands for any scales: per group of 32 columns the sum of the unscaled
// values' products, which then moves by both scales at once.  Rows of x that need it not keep the
// ordinary product's bits, so that no row depends on its neighbours; where a row of W needs it, all do.
__device__ __forceinline__ f32x4v far_product(const u32x4 w[2], uint32_t sw, const u32x4 x[2], uint32_t sx, int g, f32x4v c) {
  const bool far = __ballot(is_far_w(sw)) != 0 || is_far_x(sx);  // (results of row r16 of x are in the lanes that hold its scales)
  f32x4v ordinary;
  {
    Operand<kMx8Exact> ow, ox;
    ow.set(w[0], w[1], sw, g, -kLift);
    ox.set(x[0], x[1], sx, g, kLift);
    ordinary = tile_product<kMx8Exact>(ow, ox, c);
  }
  f32x4v sum = c;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    __builtin_amdgcn_sched_barrier(0);  // (few registers rather than speed)
    f32x4v part = {0, 0, 0, 0};
    Frag<AMLIKE_BF16>::vec vw[2], vx[2];
    widen(w[j >> 1], 127, 0, vw);
    widen(x[j >> 1], 127, 0, vx);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if ((g >> 1) != (j & 1)) vx[h] = Frag<AMLIKE_BF16>::vec{};  // the other lanes hold group j
      part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vw[h], vx[h], part, 0, 0, 0);
    }
    const int bx = (int)(sx >> (8 * j) & 0xff);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int bw = (int)((uint32_t)__shfl((int)sw, 4 * g + i) >> (8 * j) & 0xff);
      sum[i] += bx == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(part[i], bx + bw - 254);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sum[i] = far ? sum[i] : ordinary[i];
  return sum;
}

// A wave's sums once more for any scales, over the k-tiles of `each_tile` in the same order as before:
// fragment f of W holds outputs n + 16 f .., fragment e of x rows m + 16 e .. up to `last`.  The
// accumulators go round, because registers have to be named and the body is to be there once.
// Apart from the main loops on purpose: in them, it cost 20 registers and more.
template <int F, int E, typename Start, typename Tiles>
__device__ __forceinline__ void far_sums(const LinearArgs &a, int64_t m, int64_t last, int n, int r16, int g, f32x4v (&acc)[F][E],
                                         Start start, Tiles each_tile) {
  const int groups = (a.k + 31) >> 5;
#if __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(r16), "+v"(g));  // (or the addresses below are made, and kept, before the main loop)
#endif
#pragma clang loop unroll(disable)
  for (int i = 0; i < F * E; ++i) {
    const int out = min(n + i / E * 16 + r16, a.n_pad - 1);  // (behind the padded end: of no output)
    const int64_t row = min(m + i % E * 16 + r16, last);
    const uint8_t *x = a.x + row * a.ldx, *xs = a.x_scales + row * a.ld_xs;
    f32x4v c = start(i / E, g);
    each_tile([&](int kt) __attribute__((always_inline)) {
      const uint8_t *pw = a.w + ((int64_t)kt * a.n_pad + out) * kTileBytes + g * 16;
      const u32x4 qw[2] = {*reinterpret_cast<const u32x4 *>(pw), *reinterpret_cast<const u32x4 *>(pw + 64)};
      const uint32_t sw = a.w_scales[((int64_t)(kt >> 2) * a.n_pad + out) * 4 + (kt & 3)];
      const int at = kt * kTileBytes + g * 16;
      const u32x4 qx[2] = {load_chunk(x, at, a.k), load_chunk(x, at + 64, a.k)};
      c = far_product(qw, sw, qx, load_scales(xs, kt, groups), g, c);
    });
#pragma unroll
    for (int j = 0; j < F * E - 1; ++j) acc[j / E][j % E] = acc[(j + 1) / E][(j + 1) % E];
    acc[F - 1][E - 1] = c;
  }
}

// ---- epilogue ----------------------------------------------------------------------------------------

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

// Phi(-a), a >= 0: exp(-a^2/2) times erfcx(a / sqrt 2) / 2, the latter as a polynomial in
// t = 1 / (1 + p a) fitted by least squares iterated towards the smallest largest relative error
// on [0, 14] (beyond, the exponential is 0).  Degree 8 without constant: 1.5e-7 off, for fp32
// outputs; degree 5: 3.5e-5, less than a tenth of the rounding to f16 (4.9e-4).
template <bool EXACT>
__device__ __forceinline__ float normal_tail(float a) {
  const float e = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170368f);
  float t, p;
  if constexpr (EXACT) {
    t = __builtin_amdgcn_rcpf(fmaf(0.30f, a, 1.0f));
    p = 0.0356770197f;
    p = fmaf(p, t, -0.157212402f);
    p = fmaf(p, t, 0.206369481f);
    p = fmaf(p, t, -0.0536982531f);
    p = fmaf(p, t, 0.128569295f);
    p = fmaf(p, t, 0.0999111902f);
    p = fmaf(p, t, 0.120754321f);
    p = fmaf(p, t, 0.119629275f);
  } else {
    t = __builtin_amdgcn_rcpf(fmaf(0.38f, a, 1.0f));
    p = -0.0899287643f;
    p = fmaf(p, t, 0.188877211f);
    p = fmaf(p, t, 0.0919794799f);
    p = fmaf(p, t, 0.157829353f);
    p = fmaf(p, t, 0.151225193f);
  }
  return p * t * e;
}

// tanh: near 0, where 1 - 2 / (1 + exp(2x)) cancels, x times an even polynomial (fitted as above
// on [0, .65], 1.5e-7 off).
__device__ __forceinline__ float fast_tanh(float x) {
  const float a = __builtin_fabsf(x), z = x * x;
  float p = 0.0146252109f;
  p = fmaf(p, z, -0.0515180279f);
  p = fmaf(p, z, 0.132978768f);
  p = fmaf(p, z, -0.333315005f);
  p = fmaf(p, z, 0.999999846f);
  const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + fast_exp(2.0f * a));
  return a < 0.6f ? x * p : __builtin_copysignf(far, x);
}

__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-x)); }

// One value; EXACT: for an fp32 output.  (relu is a comparison: NaN stays.)
template <int ACT, bool EXACT>
__device__ __forceinline__ float activated(float x) {
  if constexpr (ACT == AMLIKE_ACT_RELU) return x < 0.0f ? 0.0f : x;
  if constexpr (ACT == AMLIKE_ACT_SIGMOID) return sigmoid(x);
  if constexpr (ACT == AMLIKE_ACT_TANH) return fast_tanh(x);
  if constexpr (ACT == AMLIKE_ACT_SILU) return x * sigmoid(x);
  if constexpr (ACT == AMLIKE_ACT_GELU) {
    const float q = normal_tail<EXACT>(__builtin_fabsf(x));
    return x * (x > 0.0f ? 1.0f - q : q);
  }
  return x;
}
// N values in place.  The reciprocal in sigmoid(x) leaves fp32's normal range at -87.4, x * sigmoid(x) only behind
// -91: there it is x exp(x), the exponential in two factors.  (Values so far out are rare: one
// comparison of the least of the N.  16384 x 1024 x 4096 mx8: 110.6 us, 113.0 with the two factors for all
// values, 106.7 with neither.)
template <int ACT, bool EXACT, int N>
__device__ __forceinline__ void activate(float *v) {
  if constexpr (ACT == AMLIKE_ACT_SILU) {
    constexpr float kFar = -80.0f;  // (1 + exp(x) is 1)
    float least = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) least = fminf(least, v[i]);
    if (__builtin_expect(__ballot(least < kFar) != 0, 0)) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float h = __builtin_amdgcn_exp2f(v[i] * 0.72134752044448170368f);
        v[i] = v[i] < kFar ? v[i] * h * h : activated<ACT, EXACT>(v[i]);
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = activated<ACT, EXACT>(v[i]);
}
// F(integral_constant-like tag) for the activation that the arguments name.
template <int ACT>
struct ActTag {
  static constexpr int value = ACT;
};
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
  if (act == AMLIKE_ACT_RELU) f(ActTag<AMLIKE_ACT_RELU>());
  else if (act == AMLIKE_ACT_SIGMOID) f(ActTag<AMLIKE_ACT_SIGMOID>());
  else if (act == AMLIKE_ACT_TANH) f(ActTag<AMLIKE_ACT_TANH>());
  else if (act == AMLIKE_ACT_SILU) f(ActTag<AMLIKE_ACT_SILU>());
  else if (act == AMLIKE_ACT_GELU) f(ActTag<AMLIKE_ACT_GELU>());
}

__device__ __forceinline__ uint32_t quad_max_bits(uint32_t u) {
  u = max(u, (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0xB1, 0xF, 0xF, true));
  return max(u, (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0x4E, 0xF, 0xF, true));
}

// Sums of eight consecutive outputs n .. n + 7 (n a multiple of 8) of row m become output; four
// neighbouring lanes hold a group of 32.  Every lane of a quad calls it, m >= rows or n >= n's end
// included.
__device__ __forceinline__ void finish8(const LinearArgs &a, int64_t m, int n, float v[8]) {
  const int cols = m < a.rows ? a.n - n : 0;
  if (cols > 0) {
    const f32x4v b0 = *reinterpret_cast<const f32x4v *>(a.bias + n), b1 = *reinterpret_cast<const f32x4v *>(a.bias + n + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] += b0[i];
      v[4 + i] += b1[i];
    }
    with_activation(a.act, [&](auto tag) __attribute__((always_inline)) {
      constexpr int kAct = decltype(tag)::value;
      if (kAct == AMLIKE_ACT_GELU && a.out_type != AMLIKE_F32) activate<kAct, false, 8>(v);
      else activate<kAct, true, 8>(v);
    });
    if (a.res_type >= 0) {
      float r[8];
      load8_any(a.res_type, a.res, m * a.ldr + n, cols, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
  }
  if (a.out_type == AMLIKE_MX8) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, i < cols ? finite_bits(v[i]) : 0u);
    const int k = mx8_exponent(quad_max_bits(top));
    if (cols > 0) {
      const u32x2 w = {mx8_pack4(v, k), mx8_pack4(v + 4, k)};
      store8_bytes(static_cast<uint8_t *>(a.out), m * a.ldo + n, cols, w);
      if ((n & 31) == 0) a.out_scales[m * a.ld_os + (n >> 5)] = (uint8_t)(k + 127);
    }
  } else if (cols > 0) {
    store8_any(a.out_type, a.out, m * a.ldo + n, cols, v);
  }
}

// A wave's 64 outputs over its four fragments of W, so dealt that a lane (r16, g) stores 16 bytes at
// a time and four lanes store 64 in a row: CH consecutive outputs per lane, 4 in fp32, 8 in 16 bits,
// 16 in 8.  Value 4 f + i of the lane (register i of fragment f) is element i of chunk ...
template <int CH>
__device__ __forceinline__ int chunk_output(int j, int g) { return j * (4 * CH) + g * CH; }  // of chunk j = value / CH
// ... so row rho of fragment f of W is output
__device__ __forceinline__ int fragment_output(int ch, int f, int rho) {
  const int per = ch >> 2;  // fragments per chunk
  return (f / per) * (4 * ch) + (rho >> 2) * ch + (f % per) * 4 + (rho & 3);
}

// The biases of a lane's 16 outputs.
template <int CH>
__device__ __forceinline__ void load_bias(const LinearArgs &a, int n, int g, f32x4v bias[4]) {
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    const int at = n + chunk_output<CH>(4 * f / CH, g) + 4 * f % CH;
    bias[f] = *reinterpret_cast<const f32x4v *>(a.bias + min(at, a.n_pad - 4));  // (behind the end: of no output)
  }
}

// CH consecutive elements of a row as CH floats, all there.
template <int CH, int TYPE>
__device__ __forceinline__ void load_chunk_of(const void *data, int64_t at, float *v) {
  if constexpr (CH == 4 && TYPE == AMLIKE_F32) {
    const u32x4 q = *reinterpret_cast<const u32x4_f *>(static_cast<const float *>(data) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = as_float(q[i]);
  } else if constexpr (CH == 4) {
    typedef u32x2 u32x2_half __attribute__((aligned(2)));
    const u32x2 q = *reinterpret_cast<const u32x2_half *>(static_cast<const uint16_t *>(data) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = q[i >> 1];
      v[i] = TYPE == AMLIKE_BF16 ? (i & 1 ? bf16_hi(w) : bf16_lo(w)) : (float)as_f16x2(w)[i & 1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < CH; i += 8) load8<TYPE>(data, at + i, 8, v + i);
  }
}

// The 16 activated sums of a lane for a row become output; n is the wave's first output.  INNER: all
// 64 exist; otherwise the elements go one by one.
template <int CH, bool INNER>
__device__ __forceinline__ void finish_row(const LinearArgs &a, int64_t row, int n, int g, float v[16]) {
  const bool live = row < a.rows;
  if (a.res_type >= 0 && live) {
    float r[16];
    if constexpr (INNER) {
      auto load = [&](auto tag) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 16 / CH; ++j)
          load_chunk_of<CH, decltype(tag)::value>(a.res, row * a.ldr + n + chunk_output<CH>(j, g), r + j * CH);
      };
      if (a.res_type == AMLIKE_F32) load(ActTag<AMLIKE_F32>());
      else if (a.res_type == AMLIKE_BF16) load(ActTag<AMLIKE_BF16>());
      else load(ActTag<AMLIKE_F16>());
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = n + chunk_output<CH>(i / CH, g) + i % CH;
        float one[8] = {0};
        if (at < a.n) load8_any(a.res_type, a.res, row * a.ldr + at, 1, one);
        r[i] = one[0];
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += r[i];
  }
  if constexpr (CH == 16) {
    const int at = n + chunk_output<16>(0, g), cols = INNER ? 16 : a.n - at;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, i < cols ? finite_bits(v[i]) : 0u);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));  // lanes l and l ^ 16 hold a group of 32
    const int k = mx8_exponent(top);
    if (live && cols > 0) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = mx8_pack4(v + 4 * i, k);
      uint8_t *p = static_cast<uint8_t *>(a.out) + row * a.ldo + at;
      if (INNER || cols >= 16) {
        typedef u32x4 u32x4_byte __attribute__((aligned(1)));
        *reinterpret_cast<u32x4_byte *>(p) = w;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < cols) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
      }
      if ((g & 1) == 0) a.out_scales[row * a.ld_os + (at >> 5)] = (uint8_t)(k + 127);
    }
  } else if (live) {
    if constexpr (INNER) {
#pragma unroll
      for (int j = 0; j < 16 / CH; ++j) {
        const int64_t to = row * a.ldo + n + chunk_output<CH>(j, g);
        const float *q = v + j * CH;
        if constexpr (CH == 4)
          *reinterpret_cast<u32x4_f *>(static_cast<float *>(a.out) + to) = u32x4{as_bits(q[0]), as_bits(q[1]), as_bits(q[2]), as_bits(q[3])};
        else if (a.out_type == AMLIKE_BF16) store8<AMLIKE_BF16>(a.out, to, 8, q);
        else store8<AMLIKE_F16>(a.out, to, 8, q);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = n + chunk_output<CH>(i / CH, g) + i % CH;
        float one[8] = {v[i]};
        if (at < a.n) store8_any(a.out_type, a.out, row * a.ldo + at, 1, one);
      }
    }
  }
}

// All of a wave's rows: fragments E, E + 1 .. of x, from row m of the output on.  (A recursion, not
// a loop: the registers have to be named, and the compiler gives up unrolling a body of this size.)
template <bool F32_ONLY, int MF, int E = 0>
__device__ __forceinline__ void finish_wave(const LinearArgs &a, int64_t m, int n, int r16, int g, const f32x4v acc[4][MF]) {
  if constexpr (E < MF) {
    const bool inner = n + 64 <= a.n;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = acc[i >> 2][E][i & 3];
    with_activation(a.act, [&](auto tag) __attribute__((always_inline)) {
      constexpr int kAct = decltype(tag)::value;
      if (kAct == AMLIKE_ACT_GELU && a.out_type != AMLIKE_F32) activate<kAct, false, 16>(v);
      else activate<kAct, true, 16>(v);
    });
    const int64_t row = m + E * 16 + r16;
    if (F32_ONLY || a.out_type == AMLIKE_F32) {
      if (inner) finish_row<4, true>(a, row, n, g, v);
      else finish_row<4, false>(a, row, n, g, v);
    } else if (a.out_type == AMLIKE_MX8) {
      if (inner) finish_row<16, true>(a, row, n, g, v);
      else finish_row<16, false>(a, row, n, g, v);
    } else {
      if (inner) finish_row<8, true>(a, row, n, g, v);
      else finish_row<8, false>(a, row, n, g, v);
    }
    finish_wave<F32_ONLY, MF, E + 1>(a, m, n, r16, g, acc);
  }
}

// ---- operands ----------------------------------------------------------------------------------------

// Where 16-byte piece c of row r of a tile lies in LDS: pieces of neighbouring rows are turned
// against each other, so that 16 lanes reading the same piece of 16 rows meet all banks.  For W the
// 16 rows may be neighbours or dealt as fragment_output has it: bits 0-3, 0 1 3 4 or 0 1 4 5 of r
// vary, and in each case bits 1-3 of the turn take all values.
__device__ __forceinline__ int turn_x(int r) { return r >> 1 & 7; }
__device__ __forceinline__ int turn_w(int r) { return (r >> 1 & 7) ^ (r >> 3 & 6); }
// The scales of four k-tiles are 16 bytes per row.  Those of row r of W lie at place scale_place(r), each
// 16 rows turned by 4 against the 16 before, for the same reason; row_at_place is its inverse.
__device__ __forceinline__ int scale_place(int r) { return (r & ~15) | ((r + (r >> 4 << 2)) & 15); }
__device__ __forceinline__ int row_at_place(int l) { return (l & ~15) | ((l - (l >> 4 << 2)) & 15); }

// ---- the pipelined tile kernel ---------------------------------------------------------------------------
// WN x WM waves, each with 64 outputs x 16 MF rows: 16-byte pieces of the k-tiles go from memory
// straight into LDS (no registers), those of later tiles while one is multiplied; blocks stay and go
// from tile to tile.
// What bounds the 256 x 256 form (8192 x 4096 x 16384): in bf16 852 us, 1.29 PFLOP/s, the library's plain
// product 808; the matrix pipe is busy for .59 of the cycles, at the clock the chip holds under
// such operands.  In mx8 545-560 us, 2.0 PFLOP/s (library, one scale for all: 438): without the copies it
// takes 461, without the matrix instructions 466, without the epilogue 501, so copies and products
// hide each other only in part: 64 KB have to come within the time of one k-tile's products, and LDS
// has no room for a third buffer.  (Tried, and no faster: waves of a SIMD reading and multiplying
// in turns, four waves of 128 x 128, touching the lines ahead.)

// Asynchronous copies of 16 bytes per lane: lane l's come from base + offset and go to LDS at
// `lds` + 16 l.  Written in assembly so that the compiler, which cannot tell the two halves of the
// buffer apart, does not make every read of LDS wait for them; they have no result register, and
// wait_copies ends them.
__device__ __forceinline__ void copy16_to_lds(const uint8_t *base, uint32_t offset, uint32_t lds) {
#if __HIP_DEVICE_COMPILE__
  // (the base is the wave's: said again where the compiler has lost sight of it)
  const uint64_t u = reinterpret_cast<uint64_t>(base);
  base = reinterpret_cast<const uint8_t *>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32 |
                                           (uint32_t)__builtin_amdgcn_readfirstlane((int)u));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
#endif
}
__device__ __forceinline__ void copy16_to_lds(const uint8_t *p, uint32_t lds) {  // any address per lane
#if __HIP_DEVICE_COMPILE__
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
#endif
}
__device__ __forceinline__ void wait_copies() {
#if __HIP_DEVICE_COMPILE__
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#endif
}
// ... until at most N of the wave's are under way.
template <int N>
__device__ __forceinline__ void wait_copies_but() {
  static_assert(N < 64, "six bits");
#if __HIP_DEVICE_COMPILE__
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
#endif
}
__device__ __forceinline__ void wait_lds() {
#if __HIP_DEVICE_COMPILE__
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#endif
}
template <typename T>
__device__ __forceinline__ uint32_t lds_address(T *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)p;
}
// Sixteen zero bytes: where pieces behind a row's end come from.
static __device__ u32x4 g_zero_piece;

// KS such groups of waves share a tile's k-tiles among them and add up at the end.  COPY: rows of x
// start and end on 16 bytes; otherwise its pieces go through registers.
template <int KIND, int WN, int WM, int MF, int STAGES, int KS, bool COPY>
__global__ __launch_bounds__(64 * WN * WM * KS, (WavesPerSimd(KIND, TileForm{WN, WM, MF, STAGES, KS, COPY}))) void linear_pipe_kernel(LinearArgs a, int m_tiles, int n_tiles) {
  constexpr int kWaves = WN * WM, BN = 64 * WN, BM = 16 * MF * WM;
  constexpr bool kMx = IsMx8(KIND);
  static_assert(COPY || STAGES == 2, "one k-tile in registers");
  constexpr int kPiecesW = BN * kChunks / (64 * kWaves), kPiecesX = BM * kChunks / (64 * kWaves);  // per wave
  static_assert((STAGES & (STAGES - 1)) == 0, "a power of two");
  __shared__ u32x4 s_tiles[KS][STAGES][(BN + BM) * kChunks];
  __shared__ u32x4 s_scales[KS][2][kMx ? BN + BM : 1];  // rows of W, then of x: the words of four k-tiles
  static_assert(KS == 1 || 4 * MF * kWaves * 64 * (KS - 1) <= KS * STAGES * (BN + BM) * kChunks, "the groups' sums fit where the tiles were");
  const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ks = all / kWaves, wave = all % kWaves;
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  // Step s of group ks: k-tile ks * steps + s, if there is one.  (8 bits: scales come for four k-tiles.)
  const int steps = kMx && KS > 1 ? ((a.k_tiles + KS - 1) / KS + 3) & ~3 : (a.k_tiles + KS - 1) / KS;
  const int wn = wave % WN, wm = wave / WN;

  // Blocks go to the 8 dies in turn; each die takes a run of tiles of its own, which its blocks go
  // through side by side, ordered in bands of 4 row tiles: the 32 tiles that a die works on share
  // 4 strips of x and 8 of W in its L2 (35554 x 2000 x 8600 bf16: 1148 us; bands of 2: 1208, of 8:
  // 1308).  Each band begins at outputs of its own, so that the dies do not all ask the memory for the
  // same lines of W at once (8192 x 4096 x 16384 mx8: 553 us against 594).
  const int total = m_tiles * n_tiles, die = blockIdx.x & 7, per = total >> 3, more = total & 7;
  const int end = die * per + min(die, more) + per + (die < more ? 1 : 0), stride = gridDim.x >> 3;
  int lin = die * per + min(die, more) + (blockIdx.x >> 3);
  if (lin >= end) return;
  const int bytes = a.k * (kMx ? 1 : 2);
  const int64_t w_step = (int64_t)a.n_pad * kTileBytes;

  // This lane's pieces of a tile: instruction i of the wave fills 8 rows of it, lane l the place l % 8
  // of row l / 8 (see turn_x, turn_w).  Bases are the wave's, in scalar registers.  A wave's rows of W
  // all lie before or all behind the padded end (they are then read from the wave's first tile's, of
  // no output); rows of x behind the last are read as the last.
  constexpr int kRowsW = kPiecesW * 8, kRowsX = kPiecesX * 8;
  static_assert(64 % kRowsW == 0 && (!kMx || (BN + BM) / 64 <= kWaves), "a wave's rows of W lie in one 64; a wave's scales are of 64 rows");
  int64_t m0;
  int n0;
  const uint8_t *bw, *bx;
  uint32_t ow[kPiecesW], ox[kPiecesX];
  // What comes through registers for a step: pieces of x, scales.  (Asked for and put into LDS in one
  // turn of the loop: carried into the next, the compiler would wait for it at once.)
  struct Held {
    u32x4 x[kPiecesX], scales;
  };
#pragma unroll
  for (int i = 0; i < kPiecesW; ++i) {
    const int r = i * 8 + (lane >> 3);
    ow[i] = r * kTileBytes + ((lane & 7) ^ turn_w(wave * kRowsW + r)) * 16;
  }
  auto last_row = [&]() __attribute__((always_inline)) { return (int)min((int64_t)BM, a.rows - m0) - 1; };
  auto place = [&]() __attribute__((always_inline)) {
    const int band = lin / (4 * n_tiles), in = lin - band * 4 * n_tiles, high = min(4, m_tiles - band * 4);
    m0 = (int64_t)(band * 4 + in % high) * BM;
    int nt = in / high + (int)((int64_t)band * n_tiles / ((m_tiles + 3) >> 2));
    if (nt >= n_tiles) nt -= n_tiles;
    n0 = nt * BN;
    const int wrow = n0 + wave * kRowsW;
    bw = a.w + (int64_t)(wrow < a.n_pad ? wrow : 0) * kTileBytes;
    bx = a.x + m0 * a.ldx;
#pragma unroll
    for (int i = 0; i < kPiecesX; ++i) {
      const int r = wave * kRowsX + i * 8 + (lane >> 3);
      ox[i] = (uint32_t)min(r, last_row()) * (uint32_t)a.ldx + (COPY ? ((lane & 7) ^ turn_x(r)) * 16 : 0);
    }
  };
  // Byte of a row at which this lane's piece i of k-tile kt lies.
  auto piece_at = [&](int i, int kt) __attribute__((always_inline)) {
    const int r = wave * kRowsX + i * 8 + (lane >> 3);
    return kt * kTileBytes + ((lane & 7) ^ turn_x(r)) * 16;
  };

  auto fetch = [&](int step, Held &held) __attribute__((always_inline)) {
    const int b = step & (STAGES - 1), kt = ks * steps + step;
    if (KS > 1 && kt >= a.k_tiles) return;
    const uint32_t lw = lds_address(&s_tiles[ks][b][wave * kPiecesW * 64]), lx = lds_address(&s_tiles[ks][b][BN * kChunks + wave * kPiecesX * 64]);
    const uint8_t *w = bw + kt * w_step, *x = bx + (COPY ? kt * kTileBytes : 0);
#pragma unroll
    for (int i = 0; i < kPiecesW; ++i) copy16_to_lds(w, ow[i], lw + i * 1024);
    const bool whole = (kt + 1) * kTileBytes <= bytes;  // not the last k-tile, or not a short one
    if constexpr (COPY) {
      if (whole) {
#pragma unroll
        for (int i = 0; i < kPiecesX; ++i) copy16_to_lds(x, ox[i], lx + i * 1024);
      } else {  // zeros behind the rows' end
#pragma unroll
        for (int i = 0; i < kPiecesX; ++i)
          copy16_to_lds(piece_at(i, kt) < bytes ? x + ox[i] : reinterpret_cast<const uint8_t *>(&g_zero_piece), lx + i * 1024);
      }
    } else {
      typedef u32x4 u32x4_byte __attribute__((aligned(1)));
      if (whole) {
#pragma unroll
        for (int i = 0; i < kPiecesX; ++i) held.x[i] = *reinterpret_cast<const u32x4_byte *>(x + ox[i] + piece_at(i, kt));
      } else {
#pragma unroll
        for (int i = 0; i < kPiecesX; ++i) held.x[i] = load_chunk(x + ox[i], piece_at(i, kt), bytes);
      }
    }
    if constexpr (kMx) {
      if ((step & 3) == 0 && wave < (BN + BM) / 64) {  // the scales of this k-tile and the next three
        const int r = wave * 64;  // the wave's first row
        const bool of_w = r < BN;
        const int64_t line = (int64_t)(kt >> 2) * a.n_pad + (n0 + r < a.n_pad ? n0 + r : 0);
        const uint8_t *base = of_w ? reinterpret_cast<const uint8_t *>(a.w_scales) + line * 16 : a.x_scales + m0 * a.ld_xs + (int64_t)kt * 4;
        const uint32_t offset = of_w ? row_at_place(lane) * 16 : (uint32_t)min(r - BN + lane, last_row()) * (uint32_t)a.ld_xs;
        if constexpr (COPY) {  // (what a row's last 16 bytes hold behind its last scale is put right on reading; being aligned, they leave no page)
          copy16_to_lds(base, offset, lds_address(&s_scales[ks][step >> 2 & 1][r]));
        } else {
          typedef u32x4 u32x4_byte __attribute__((aligned(1)));
          const int groups = (a.k + 31) >> 5;
          if (of_w || kt * 4 + 16 <= groups) {
            held.scales = *reinterpret_cast<const u32x4_byte *>(base + offset);
          } else {
            u32x4 q = {0, 0, 0, 0};
#pragma clang loop unroll(disable)
            for (int i = 0; i < 4; ++i) q = u32x4{q[1], q[2], q[3], load_scales(base - (int64_t)kt * 4 + offset, kt + i, groups)};
            held.scales = q;
          }
        }
      }
    }
  };
  // What fetch(step) brought into registers goes to LDS.
  auto put = [&](int step, const Held &held) __attribute__((always_inline)) {
    if constexpr (!COPY) {
      if (KS == 1 || ks * steps + step < a.k_tiles) {
#pragma unroll
        for (int i = 0; i < kPiecesX; ++i) s_tiles[ks][step & 1][BN * kChunks + (wave * kPiecesX + i) * 64 + lane] = held.x[i];
      }
    }
    if constexpr (kMx && !COPY)
      if ((step & 3) == 0 && wave < (BN + BM) / 64) s_scales[ks][step >> 2 & 1][wave * 64 + lane] = held.scales;
  };

  const int ch = KIND == kMx8Exact || a.out_type == AMLIKE_F32 ? 4 : a.out_type == AMLIKE_MX8 ? 16 : 8;
  int row_w[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) row_w[f] = wn * 64 + fragment_output(ch, f, r16);

  // k-tiles of a tile that start() asks for: with two buffers both, with more all but the one that the
  // first turn of the loop asks for, through registers one.
  constexpr int kAhead = !COPY ? 1 : STAGES == 2 ? 2 : STAGES - 1;
  // A tile's first k-tiles and its biases, on their way while the tile before is stored.  The memory
  // unit answers in order: when the biases are there, so are the k-tiles.
  f32x4v bias[4];
  Held first;  // step 0's
  auto start = [&]() __attribute__((always_inline)) {
    place();
    fetch(0, first);
    for (int s = 1; s < min(kAhead, steps); ++s) {
      Held none;  // (copies only: x, and scales with step 0's)
      fetch(s, none);
    }
    const int n = n0 + wn * 64;
    if (ch == 4) load_bias<4>(a, n, g, bias);
    else if (ch == 16) load_bias<16>(a, n, g, bias);
    else load_bias<8>(a, n, g, bias);
  };

  start();
  for (;;) {
    f32x4v acc[4][MF];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
#if __HIP_DEVICE_COMPILE__
      asm volatile("" : "+v"(bias[f])::"memory");  // the biases are there
#endif
#pragma unroll
      for (int e = 0; e < MF; ++e) acc[f][e] = ks == 0 ? bias[f] : f32x4v{0, 0, 0, 0};
    }
    auto operand = [&](int step, const u32x4 *tile, int row, int turn, int scale_row, int lift) __attribute__((always_inline)) {
      Operand<KIND> o;
      uint32_t sc = 0;
      if constexpr (kMx) {
        sc = reinterpret_cast<const uint32_t *>(&s_scales[ks][step >> 2 & 1][scale_row])[step & 3];
        if constexpr (COPY) {  // 2^0 behind the row's last scale
          const int groups = ((a.k + 31) >> 5) - (ks * steps + step) * 4;
          if (groups < 4) sc = (sc & ~(~0u << (8 * groups))) | (0x7f7f7f7fu << (8 * groups));
        }
      }
      o.set(tile[row * kChunks + (g ^ turn)], tile[row * kChunks + (g ^ 4 ^ turn)], sc, g, lift);
      return o;
    };
    bool far = false;  // kMx8Exact: whether far_sums is needed (this lane's part of it)
    int step = 0;
#if __HIP_DEVICE_COMPILE__
    asm volatile("" : "+s"(step));  // (one copy of the loop's body: the first steps are not to be peeled off)
#endif
    put(0, first);
#pragma clang loop unroll(disable)
    for (; step < steps; ++step) {
      // This wave's pieces for the step have to be in LDS, and its reads of the step before done.  The
      // copies of the STAGES - 2 steps behind may be under way (in order: nothing else is behind them).
      const int behind = step + STAGES - 2;  // the last of them, if it was asked for (a group's last steps may have no k-tile)
      if (step < kAhead) wait_lds();
      else if (STAGES > 2 && behind < steps && ks * steps + behind < a.k_tiles) wait_copies_but<(STAGES - 2) * (kPiecesW + kPiecesX)>();
      else wait_copies();
      __builtin_amdgcn_s_barrier();  // everybody's
      Held held;
      const bool ahead = step + STAGES - 1 >= kAhead && step + STAGES - 1 < steps;
      if (ahead) fetch(step + STAGES - 1, held);
      const int b = step & (STAGES - 1);
      if (KS == 1 || ks * steps + step < a.k_tiles) {
      const u32x4 *tw = s_tiles[ks][b], *tx = tw + BN * kChunks;
      Operand<KIND> fw[4];
#pragma unroll
      for (int f = 0; f < 4; ++f) fw[f] = operand(step, tw, row_w[f], turn_w(row_w[f]), scale_place(row_w[f]), -kLift);
#pragma unroll
      for (int e = 0; e < MF; ++e) {
        const Operand<KIND> fx = operand(step, tx, wm * 16 * MF + e * 16 + r16, turn_x(r16), BN + wm * 16 * MF + e * 16 + r16, kLift);
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[f][e] = tile_product<KIND>(fw[f], fx, acc[f][e]);
      }
      if constexpr (KIND == kMx8Exact) {
        if ((step & 3) == 0) {  // the scales of this k-tile and the next three: lane (r, q) looks at k-tile step + q of its rows
          int r = r16, q = g;
#if __HIP_DEVICE_COMPILE__
          asm volatile("" : "+v"(r), "+v"(q));  // (or the addresses below stay in registers through the k-tiles)
#endif
          const u32x4 *scales = s_scales[ks][step >> 2 & 1];
          const int there = ((a.k + 31) >> 5) - (ks * steps + step + q) * 4;  // groups that rows of x have from there on
          const uint32_t mask = there >= 4 ? ~0u : there <= 0 ? 0u : ~(~0u << (8 * there));
#pragma unroll
          for (int f = 0; f < 4; ++f) far |= is_far_w(scales[scale_place(wn * 64 + fragment_output(4, f, r))][q]);
#pragma unroll
          for (int e = 0; e < MF; ++e) far |= is_far_x(scales[BN + (wm * MF + e) * 16 + r][q] & mask);
        }
      }
      }
      if (ahead) put(step + STAGES - 1, held);  // (where nobody reads now: the barriers of this turn and the next)
    }
    const int64_t m = m0 + wm * 16 * MF;
    const int n = n0 + wn * 64;
    if constexpr (KIND == kMx8Exact) {
      if (__builtin_expect(__ballot(far) != 0, 0))
        far_sums(a, m, m0 + last_row(), n, r16, g, acc, [&](int f, int q) {
          return ks == 0 ? *reinterpret_cast<const f32x4v *>(a.bias + min(n + f * 16 + q * 4, a.n_pad - 4)) : f32x4v{0, 0, 0, 0};
        }, [&](auto tile) __attribute__((always_inline)) {
#pragma clang loop unroll(disable)
          for (int kt = ks * steps; kt < min((ks + 1) * steps, a.k_tiles); ++kt) tile(kt);
        });
    }
    if constexpr (KS > 1) {  // the first group adds the others' sums to its own, in their order
      f32x4v *part = reinterpret_cast<f32x4v *>(s_tiles);
      wait_lds();
      __builtin_amdgcn_s_barrier();
      if (ks > 0) {
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
          for (int e = 0; e < MF; ++e) part[(((ks - 1) * 4 * MF + f * MF + e) * kWaves + wave) * 64 + lane] = acc[f][e];
      }
      __syncthreads();
      if (ks == 0) {
#pragma unroll
        for (int q = 0; q < KS - 1; ++q)
#pragma unroll
          for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int e = 0; e < MF; ++e) acc[f][e] += part[((q * 4 * MF + f * MF + e) * kWaves + wave) * 64 + lane];
      }
    }
    lin += stride;
    if (lin < end) {
      wait_lds();
      __builtin_amdgcn_s_barrier();  // all buffers are free
      start();
    }
    if (KS > 1 && ks > 0) {
      if (lin >= end) break;
      continue;
    }
    int er = r16, eg = g;
#if __HIP_DEVICE_COMPILE__
    asm volatile("" : "+v"(er), "+v"(eg));  // (or the compiler keeps every address of the epilogue through the k-tiles)
#endif
    finish_wave<KIND == kMx8Exact, MF>(a, m, n, er, eg, acc);
    if (lin >= end) break;
  }
}

// ---- few rows ------------------------------------------------------------------------------------------
// 16 NT outputs x 16 MT rows per block; its eight waves share the k-tiles among them, each from
// memory straight into registers, and add up in LDS in wave order; kBatch k-tiles of each are in
// flight.  For few rows the way of W bounds it (16 x 8192 x 8192 bf16: 26.2 us and 5.1 TB/s from HBM, six layers of
// 134 MB in turn; 25.2 us with the one layer's W in the last-level cache), for small products a launch and two
// trips to memory (1 x 2048 x 2048 bf16: 6.3 us from HBM, 80 layers in turn, 4.7 from the caches, of which 2.2 are any
// launch's).  (Tried: biases and residual asked for before the k-tiles, 0; the k-tile that rows end in
// moved out of the batches, 0; eight whole lines a load instead of sixteen halves, with lanes trading
// pieces, -5 %.)
template <int KIND, int NT, int MT>
__global__ __launch_bounds__(512) void linear_thin_kernel(LinearArgs a, int m_tiles, int n_tiles) {
  constexpr int kWaves = 8, kCols = 16 * NT, kRows = 16 * MT, kBatch = MT >= 4 ? 2 : 4;
  constexpr bool kMx = IsMx8(KIND);
  typedef u32x4 u32x4_byte __attribute__((aligned(1)));
  typedef uint32_t u32_byte __attribute__((aligned(1)));
  __shared__ float s_c[kWaves][kRows][kCols + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
  // Strips of the larger operand are dealt to the XCDs (blocks b, b + 8 ..), each with all its tiles.
  const bool by_rows = m_tiles > n_tiles;
  const int inner = by_rows ? n_tiles : m_tiles, j = blockIdx.x >> 3;
  const int strip = j / inner * 8 + (blockIdx.x & 7), in = j % inner;
  if (strip >= (by_rows ? m_tiles : n_tiles)) return;
  const int n0 = (by_rows ? in : strip) * kCols;
  const int64_t m0 = (int64_t)(by_rows ? strip : in) * kRows;
  const int bytes = a.k * (kMx ? 1 : 2), all_groups = (a.k + 31) >> 5;
  const uint8_t *w = a.w + (int64_t)(n0 + r16) * kTileBytes + g * 16;
  const uint8_t *x[MT], *xs[kMx ? MT : 1];
#pragma unroll
  for (int e = 0; e < MT; ++e) {
    const int64_t row = min(m0 + e * 16 + r16, (int64_t)a.rows - 1);
    x[e] = a.x + row * a.ldx;
    if constexpr (kMx) xs[e] = a.x_scales + row * a.ld_xs;
  }
  f32x4v acc[NT][MT] = {};
  bool far = false;  // kMx8Exact: whether far_sums is needed (this lane's part of it)
  // A batch is every eighth k-tile, in 8 bits neighbours: their scales are one load per row.
  constexpr int kNext = kMx ? 1 : kWaves;
  for (int kt0 = wave * (kMx ? kBatch : 1); kt0 < a.k_tiles; kt0 += kWaves * kBatch) {
    u32x4 qw[kBatch][NT][2], qx[kBatch][MT][2];
    uint32_t sw[kBatch][NT], sx[kBatch][MT];
    if constexpr (kMx) {
      typedef uint32_t words __attribute__((ext_vector_type(kBatch)));
      typedef words words_byte __attribute__((aligned(1)));
#pragma unroll
      for (int f = 0; f < NT; ++f) {  // (whole fours of k-tiles are there)
        const words q = *reinterpret_cast<const words *>(a.w_scales + ((int64_t)(kt0 >> 2) * a.n_pad + n0 + f * 16 + r16) * 4 + (kt0 & 3));
#pragma unroll
        for (int u = 0; u < kBatch; ++u) sw[u][f] = q[u];
      }
      const bool whole = (kt0 + kBatch) * 4 <= all_groups;
#pragma unroll
      for (int e = 0; e < MT; ++e) {
        if (whole) {
          const words q = *reinterpret_cast<const words_byte *>(xs[e] + kt0 * 4);
#pragma unroll
          for (int u = 0; u < kBatch; ++u) sx[u][e] = q[u];
        } else {
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int kt = kt0 + u;
            sx[u][e] = 0;
            if ((kt + 1) * 4 <= all_groups) sx[u][e] = *reinterpret_cast<const u32_byte *>(xs[e] + kt * 4);
            else if (kt < a.k_tiles) sx[u][e] = load_scales(xs[e], kt, all_groups);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int kt = kt0 + u * kNext;
      if (kt >= a.k_tiles) continue;
      const uint8_t *p = w + (int64_t)kt * a.n_pad * kTileBytes;
#pragma unroll
      for (int f = 0; f < NT; ++f) {
        qw[u][f][0] = *reinterpret_cast<const u32x4 *>(p + f * 16 * kTileBytes);
        qw[u][f][1] = *reinterpret_cast<const u32x4 *>(p + f * 16 * kTileBytes + 64);
        if constexpr (!kMx) sw[u][f] = 0;
      }
      const int at = kt * kTileBytes + g * 16;
      if ((kt + 1) * kTileBytes <= bytes) {
#pragma unroll
        for (int e = 0; e < MT; ++e) {
          qx[u][e][0] = *reinterpret_cast<const u32x4_byte *>(x[e] + at);
          qx[u][e][1] = *reinterpret_cast<const u32x4_byte *>(x[e] + at + 64);
          if constexpr (!kMx) sx[u][e] = 0;
        }
      } else {
#pragma unroll
        for (int e = 0; e < MT; ++e) {
          qx[u][e][0] = load_chunk(x[e], at, bytes);
          qx[u][e][1] = load_chunk(x[e], at + 64, bytes);
          if constexpr (!kMx) sx[u][e] = 0;
        }
      }
    }
    if constexpr (KIND == kMx8Exact) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {  // (behind the last k-tile: W's are 2^0, those of x 0)
#pragma unroll
        for (int f = 0; f < NT; ++f) far |= is_far_w(sw[u][f]);
#pragma unroll
        for (int e = 0; e < MT; ++e) far |= is_far_x(sx[u][e]);
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (kt0 + u * kNext >= a.k_tiles) break;
      Operand<KIND> fw[NT];
#pragma unroll
      for (int f = 0; f < NT; ++f) fw[f].set(qw[u][f][0], qw[u][f][1], sw[u][f], g, -kLift);
#pragma unroll
      for (int e = 0; e < MT; ++e) {
        Operand<KIND> fx;
        fx.set(qx[u][e][0], qx[u][e][1], sx[u][e], g, kLift);
#pragma unroll
        for (int f = 0; f < NT; ++f) acc[f][e] = tile_product<KIND>(fw[f], fx, acc[f][e]);
      }
    }
  }
  if constexpr (KIND == kMx8Exact) {
    if (__builtin_expect(__ballot(far) != 0, 0))
      far_sums(a, m0, (int64_t)a.rows - 1, n0, r16, g, acc, [](int, int) { return f32x4v{0, 0, 0, 0}; },
               [&](auto tile) __attribute__((always_inline)) {
#pragma clang loop unroll(disable)
                 for (int kt0 = wave * kBatch; kt0 < a.k_tiles; kt0 += kWaves * kBatch)
#pragma clang loop unroll(disable)
                   for (int kt = kt0; kt < min(kt0 + kBatch, a.k_tiles); ++kt) tile(kt);
               });
  }
#pragma unroll
  for (int e = 0; e < MT; ++e)
#pragma unroll
    for (int f = 0; f < NT; ++f) *reinterpret_cast<f32x4v *>(&s_c[wave][e * 16 + r16][f * 16 + g * 4]) = acc[f][e];
  __syncthreads();
  constexpr int kPer = kCols / 8;  // pieces of 8 outputs in a row
  for (int p = tid; p < kRows * kPer; p += 512) {
    const int m = p / kPer, c = p % kPer * 8;
    float v[8] = {};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const f32x4v lo = *reinterpret_cast<const f32x4v *>(&s_c[i][m][c]), hi = *reinterpret_cast<const f32x4v *>(&s_c[i][m][c + 4]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] += lo[j];
        v[4 + j] += hi[j];
      }
    }
    finish8(a, m0 + m, n0 + c, v);
  }
}

// ---- launches ------------------------------------------------------------------------------------------

namespace {

// Calls `launch` on stretches of the rows, all of them but for outputs beyond max_blocks (2^22) blocks of
// `tile` elements: a grid holds less than 2^32 threads, 2^23 blocks of 512.
template <typename F>
int ByRows(LinearArgs a, int tile, F launch) {
  const int64_t most = std::max<int64_t>((int64_t)a.max_blocks * tile / a.n_pad / 256 * 256, 256);
  const int64_t rows = a.rows;
  const int rb = a.res_type < 0 ? 0 : TypeBytes(a.res_type), ob = TypeBytes(a.out_type);
  for (int64_t r = 0; r < rows; r += most) {
    a.rows = (int32_t)std::min(most, rows - r);
    if (int rc = launch(a)) return rc;
    a.x += most * a.ldx;
    if (a.x_scales) a.x_scales += most * a.ld_xs;
    if (a.res) a.res = static_cast<const char *>(a.res) + most * a.ldr * rb;
    a.out = static_cast<char *>(a.out) + most * a.ldo * ob;
    if (a.out_scales) a.out_scales += most * a.ld_os;
  }
  return AMLIKE_OK;
}

template <int KIND, int FORM>
int LaunchPipe(const LinearArgs &args, hipStream_t st) {
  return ByRows(args, 2048, [&](const LinearArgs &a) -> int {
    constexpr TileForm f = kTileForms[FORM];
    const int m_tiles = (a.rows + 16 * f.mf * f.wm - 1) / (16 * f.mf * f.wm), n_tiles = (a.n_pad + 64 * f.wn - 1) / (64 * f.wn);
    const int held = BlocksHeld(KIND, f, NumComputeUnits());
    hipLaunchKernelGGL((linear_pipe_kernel<KIND, f.wn, f.wm, f.mf, f.stages, f.ks, f.copy>), dim3((unsigned)std::min((m_tiles * n_tiles + 7) & ~7, held)),
                       dim3(64 * f.wn * f.wm * f.ks), 0, st, a, m_tiles, n_tiles);
    AMLIKE_HIP(hipGetLastError());
    return AMLIKE_OK;
  });
}

// Whether 16-byte pieces of x can be copied as they are: rows, of scales too, start on 16 bytes and
// end on one (or the last piece would bring what lies behind the row; scales are looked after).
bool Copyable(const LinearArgs &a, int kind) {
  return (reinterpret_cast<uintptr_t>(a.x) | (uintptr_t)a.ldx | (uintptr_t)a.k * (IsMx8(kind) ? 1 : 2)) % 16 == 0 &&
         (!IsMx8(kind) || (reinterpret_cast<uintptr_t>(a.x_scales) | (uintptr_t)a.ld_xs) % 16 == 0);
}

template <int KIND, int FORM>
int LaunchThin(const LinearArgs &args, hipStream_t st) {
  constexpr int NT = kThinForms[FORM].nt, MT = kThinForms[FORM].mt;
  return ByRows(args, 256 * NT * MT, [&](const LinearArgs &a) -> int {
    const int m_tiles = (a.rows + 16 * MT - 1) / (16 * MT), n_tiles = a.n_pad / (16 * NT);
    const unsigned blocks = (unsigned)((std::max(m_tiles, n_tiles) + 7) & ~7) * std::min(m_tiles, n_tiles);
    hipLaunchKernelGGL((linear_thin_kernel<KIND, NT, MT>), dim3(blocks), dim3(512), 0, st, a, m_tiles, n_tiles);
    AMLIKE_HIP(hipGetLastError());
    return AMLIKE_OK;
  });
}

}  // namespace

template <int KIND>
int LaunchLinear(const LinearArgs &a, hipStream_t st) {
  // (the tile kernel addresses a tile's rows with 32 bits)
  const bool far_apart = a.ldx > 1 << 22 || a.ld_xs > 1 << 22;
  const LinearChoice c = ChooseLinear(KIND, a.out_type, a.rows, a.k_tiles, a.n_pad, Copyable(a, KIND), far_apart, NumComputeUnits());
  if (c.thin) {
    if (c.form == 0) return LaunchThin<KIND, 0>(a, st);
    if (c.form == 1) return LaunchThin<KIND, 1>(a, st);
    if (c.form == 2) return LaunchThin<KIND, 2>(a, st);
    if (c.form == 3) return LaunchThin<KIND, 3>(a, st);
    return LaunchThin<KIND, 4>(a, st);
  }
  if (c.form == 1) return LaunchPipe<KIND, 1>(a, st);
  if (c.form == 2) return LaunchPipe<KIND, 2>(a, st);
  if (c.form == 3) return LaunchPipe<KIND, 3>(a, st);
  if (c.form == 4) return LaunchPipe<KIND, 4>(a, st);
  if (c.form == 5) return LaunchPipe<KIND, 5>(a, st);
  if (c.form == 6) return LaunchPipe<KIND, 6>(a, st);
  if constexpr (KIND != kMx8Exact) return LaunchPipe<KIND, 0>(a, st);
  return AMLIKE_EINVAL;
}

#endif  // AMLIKE_LINEAR_KERNELS
}  // namespace amlike

#endif  // KALDI_AMD_CSRC_LINEAR_KERNELS_H_
