// What the dense-layer operators (row_ops.hip, linear.hip) share: the device view of an
// amlike_matrix_t, loads and stores of eight consecutive columns in every type, the 8-bit format,
// and the host's checks of their arguments.
#ifndef KALDI_AMD_CSRC_DENSE_COMMON_H_
#define KALDI_AMD_CSRC_DENSE_COMMON_H_

#include "amlike_common.h"

namespace amlike {

static inline int TypeBytes(int type) { return type == AMLIKE_F32 ? 4 : type == AMLIKE_MX8 ? 1 : 2; }

// AMLIKE_OK or AMLIKE_EINVAL with a text: `m` describes a [rows x cols] matrix that a kernel may
// touch.  With rows == 0 only the type is looked at.
int CheckMatrix(const char *call, const char *name, const amlike_matrix_t *m, int64_t rows, int64_t cols);
// The same for a matrix that is written: its values and scales do not share bytes either.
int CheckOutput(const char *call, const amlike_matrix_t *out, int64_t rows, int64_t cols);
// Whether a byte (of values or scales) belongs to both matrices.
bool MatricesOverlap(const amlike_matrix_t *a, int64_t rows_a, int64_t cols_a, const amlike_matrix_t *b,
                     int64_t rows_b, int64_t cols_b);
// Whether they are one matrix: an element is read and written by the same thread then.
static inline bool SameMatrix(const amlike_matrix_t *a, const amlike_matrix_t *b) {
  return a->data == b->data && a->type == b->type && a->ld == b->ld && a->type != AMLIKE_MX8;
}
// The convert operator's launch, for callers that have checked their arguments.
int LaunchConvert(const amlike_matrix_t &x, int64_t rows, int64_t cols, const amlike_matrix_t &out, hipStream_t st);

#if defined(__HIPCC__)

typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
// Eight or sixteen bytes at any element boundary: the vector memory unit takes unaligned
// addresses, and aligned ones cost nothing extra in this form.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x4 u32x4_f __attribute__((aligned(4)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));

// (By value: __builtin_bit_cast of a vector's element reads element 0 whichever is named.)
__device__ __forceinline__ float as_float(uint32_t w) { return __builtin_bit_cast(float, w); }
__device__ __forceinline__ uint32_t as_bits(float v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ f16x2v as_f16x2(uint32_t w) { return __builtin_bit_cast(f16x2v, w); }
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const f32x2v v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2v));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const f32x2v v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2v));
}

// v[0..7] = elements [at, at + 8) of a row, those at `n` and beyond as 0 (n >= 8: all there).
template <int TYPE>
__device__ __forceinline__ void load8(const void *data, int64_t at, int n, float v[8]) {
  if constexpr (TYPE == AMLIKE_F32) {
    const float *p = static_cast<const float *>(data) + at;
    if (n >= 8) {
      const u32x4 a = *reinterpret_cast<const u32x4_f *>(p), b = *reinterpret_cast<const u32x4_f *>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = as_float(a[i]);
        v[4 + i] = as_float(b[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
    }
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(data) + at;
    u32x4 a;
    if (n >= 8) {
      a = *reinterpret_cast<const u32x4_any *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        a[i] = (2 * i < n ? (uint32_t)p[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)p[2 * i + 1] << 16 : 0u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == AMLIKE_BF16) {
        v[2 * i] = bf16_lo(a[i]);
        v[2 * i + 1] = bf16_hi(a[i]);
      } else {
        const f16x2v h = as_f16x2(a[i]);
        v[2 * i] = (float)h[0];
        v[2 * i + 1] = (float)h[1];
      }
    }
  }
}

// The first min(n, 8) of v to elements [at, at + 8), rounded to nearest even.
template <int TYPE>
__device__ __forceinline__ void store8(void *data, int64_t at, int n, const float v[8]) {
  if constexpr (TYPE == AMLIKE_F32) {
    float *p = static_cast<float *>(data) + at;
    if (n >= 8) {
      u32x4 a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = __builtin_bit_cast(uint32_t, v[i]);
        b[i] = __builtin_bit_cast(uint32_t, v[4 + i]);
      }
      *reinterpret_cast<u32x4_f *>(p) = a;
      *reinterpret_cast<u32x4_f *>(p + 4) = b;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = v[i];
    }
  } else {
    uint16_t *p = static_cast<uint16_t *>(data) + at;
    u32x4 a;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      a[i] = TYPE == AMLIKE_BF16 ? pack_bf16(v[2 * i], v[2 * i + 1]) : pack_f16(v[2 * i], v[2 * i + 1]);
    if (n >= 8) {
      *reinterpret_cast<u32x4_any *>(p) = a;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (uint16_t)(a[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// The type known only at run time: one scalar branch per call.
__device__ __forceinline__ void load8_any(int type, const void *data, int64_t at, int n, float v[8]) {
  if (type == AMLIKE_F32) load8<AMLIKE_F32>(data, at, n, v);
  else if (type == AMLIKE_BF16) load8<AMLIKE_BF16>(data, at, n, v);
  else load8<AMLIKE_F16>(data, at, n, v);
}
__device__ __forceinline__ void store8_any(int type, void *data, int64_t at, int n, const float v[8]) {
  if (type == AMLIKE_F32) store8<AMLIKE_F32>(data, at, n, v);
  else if (type == AMLIKE_BF16) store8<AMLIKE_BF16>(data, at, n, v);
  else store8<AMLIKE_F16>(data, at, n, v);
}

// ---- the 8-bit form ----
// The magnitude's bits of |y| where it is finite, else 0: as integers these order like the values.
__device__ __forceinline__ uint32_t finite_bits(float y) {
  const uint32_t u = __builtin_bit_cast(uint32_t, y) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}
// The smallest k in [-127, 120] with amax <= 448 * 2^k, from the bits of amax.  448 = 1.75 * 2^8:
// k is amax's exponent - 8, one more where its fraction exceeds .75 (0x600000).  Below 2^-119
// the clamp decides; a denormal amax has exponent field 0 and ends there too.
__device__ __forceinline__ int mx8_exponent(uint32_t amax_bits) {
  const int k = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return k < -127 ? -127 : k;
}
// Four values times 2^-k as four e4m3 bytes.  The scaling is exact (no value leaves the range
// above, and what falls below fp32's smallest denormal is far below e4m3's); the conversion
// rounds to nearest even.  What is not finite becomes NaN before it gets there.
__device__ __forceinline__ uint32_t mx8_pack4(const float *v, int k) {
  float t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = __builtin_amdgcn_ldexpf(v[i], -k);
    t[i] = __builtin_fabsf(t[i]) <= 448.0f ? t[i] : __builtin_nanf("");
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], w, true);
  return (uint32_t)w;
}
// The first min(n, 8) bytes of the pair to a row's bytes [at, at + 8).
__device__ __forceinline__ void store8_bytes(uint8_t *data, int64_t at, int n, u32x2 w) {
  uint8_t *p = data + at;
  if (n >= 8) {
    *reinterpret_cast<u32x2_any *>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}

#endif  // __HIPCC__
}  // namespace amlike

#endif  // KALDI_AMD_CSRC_DENSE_COMMON_H_
