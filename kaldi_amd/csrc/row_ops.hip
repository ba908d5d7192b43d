// Operators on the rows of a matrix: the root-mean-square norm with the residual's addition
// (amlike_norm_*) and the conversion between types (amlike_convert_dev), both with an output in
// 8 bits if wanted.  One kernel: a row belongs to a team of threads that keeps it in registers,
//   s = x + r;   y = s * rsqrt(mean(s^2) + eps) * w      (norm)
//   y = x                                                 (convert)
// so every input is read once and every output written once: the bound is HBM.  16 384 x 4096 bf16 with
// residual and sum into 8 bits: 85 us, 5.6 TB/s (a copy of 1 GiB reaches 4.95); 35 554 x 2000 bf16 into
// 8 bits: 46 us, 4.7 TB/s.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <new>
#include <utility>

#include "dense_common.h"

namespace amlike {

struct RowArgs {
  const void *x, *r;
  void *sum, *out;
  uint8_t *scales;
  const float *weight;
  int64_t ldx, ldr, lds, ldo, ld_scales;
  int64_t rows, blocks;
  int32_t dim, out_type, col_blocks;
  float eps, inv_dim;
};

// Eight elements as they lie in memory.
template <int TYPE>
struct Raw8 {
  u32x4 w[TYPE == AMLIKE_F32 ? 2 : 1];
};
template <int TYPE>
__device__ __forceinline__ Raw8<TYPE> load_raw8(const void *data, int64_t at, int n) {
  Raw8<TYPE> q;
  if constexpr (TYPE == AMLIKE_F32) {
    const float *p = static_cast<const float *>(data) + at;
    if (n >= 8) {
      q.w[0] = *reinterpret_cast<const u32x4_f *>(p);
      q.w[1] = *reinterpret_cast<const u32x4_f *>(p + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) q.w[i >> 2][i & 3] = i < n ? __builtin_bit_cast(uint32_t, p[i]) : 0u;
    }
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(data) + at;
    if (n >= 8) {
      q.w[0] = *reinterpret_cast<const u32x4_any *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q.w[0][i] = (2 * i < n ? (uint32_t)p[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)p[2 * i + 1] << 16 : 0u);
    }
  }
  return q;
}
template <int TYPE>
__device__ __forceinline__ float raw_at(const Raw8<TYPE> &q, int i) {
  if constexpr (TYPE == AMLIKE_F32) return as_float(q.w[i >> 2][i & 3]);
  const uint32_t w = q.w[0][i >> 1];
  if constexpr (TYPE == AMLIKE_BF16) return i & 1 ? bf16_hi(w) : bf16_lo(w);
  return (float)__builtin_bit_cast(f16x2v, w)[i & 1];
}

// The sum over a team of TPR threads, the same bits in each of them: lanes by a butterfly, waves
// through LDS in wave order.
template <int TPR>
__device__ __forceinline__ float team_sum(float a, float *s_part) {
#pragma unroll
  for (int m = 1; m < (TPR < 64 ? TPR : 64); m <<= 1) a += __shfl_xor(a, m);
  if constexpr (TPR > 64) {
    __syncthreads();  // the last use of s_part is over
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = a;
    __syncthreads();
    a = 0.0f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) a += s_part[i];
  }
  return a;
}

// Largest of four neighbouring lanes (one group of 32 columns).
__device__ __forceinline__ uint32_t quad_max(uint32_t u) {
  u = max(u, (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0xB1, 0xF, 0xF, true));
  return max(u, (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0x4E, 0xF, 0xF, true));
}

// TPR threads own a row (NORM) or a stretch of TPR * NCH * 8 columns of it; thread t holds the
// chunks t, t + TPR, ... of 8 columns, so that neighbours read neighbouring 16 bytes and four
// neighbours hold a group of 32 columns.
template <int TIN, bool NORM, int TPR, int NCH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void dense_rows_kernel(RowArgs a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, kTeams = kThreads / TPR;
  __shared__ float s_part[TPR > 64 ? TPR / 64 : 1];
  const int team = threadIdx.x / TPR, t = threadIdx.x % TPR;
  for (int64_t blk = blockIdx.x; blk < a.blocks; blk += gridDim.x) {
    int64_t rblk = blk;
    int col0 = t * 8;
    if constexpr (!NORM) {
      rblk = blk / a.col_blocks;
      col0 += (int)(blk - rblk * a.col_blocks) * (TPR * NCH * 8);
    }
    const int64_t row = rblk * kTeams + team;
    const int cols = row < a.rows ? a.dim : 0;  // a row behind the last one has no columns
    float v[NCH][8];
    {
      Raw8<TIN> qx[NCH], qr[NORM ? NCH : 1];
#pragma unroll
      for (int i = 0; i < NCH; ++i) qx[i] = load_raw8<TIN>(a.x, row * a.ldx + col0 + i * TPR * 8, cols - (col0 + i * TPR * 8));
      if (NORM && a.r) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
          qr[NORM ? i : 0] = load_raw8<TIN>(a.r, row * a.ldr + col0 + i * TPR * 8, cols - (col0 + i * TPR * 8));
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = raw_at<TIN>(qx[i], j) + raw_at<TIN>(qr[NORM ? i : 0], j);
      } else {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = raw_at<TIN>(qx[i], j);
      }
    }
    if constexpr (NORM) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
      ss = team_sum<TPR>(ss, s_part);
      float rstd;
      if (ss < __builtin_inff()) {
        rstd = __builtin_amdgcn_rsqf(fmaf(ss, a.inv_dim, a.eps));
      } else {  // the squares left fp32's range (or hold a NaN): once more at 2^-80, where eps no longer counts
        ss = 0.0f;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float z = v[i][j] * 0x1p-80f;
            ss = fmaf(z, z, ss);
          }
        ss = team_sum<TPR>(ss, s_part);
        rstd = __builtin_amdgcn_rsqf(ss * a.inv_dim) * 0x1p-80f;
      }
      if (a.sum) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          const int c = col0 + i * TPR * 8;
          if (c < cols) store8<TIN>(a.sum, row * a.lds + c, cols - c, v[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = col0 + i * TPR * 8;
        if (a.weight) {
          float w[8];
          load8<AMLIKE_F32>(a.weight, c, cols - c, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * rstd * w[j];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] *= rstd;
        }
      }
    }
    if (a.out_type == AMLIKE_MX8) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = col0 + i * TPR * 8;
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, finite_bits(v[i][j]));
        const int k = mx8_exponent(quad_max(top));
        if (c < cols) {
          const u32x2 w = {mx8_pack4(v[i], k), mx8_pack4(v[i] + 4, k)};
          store8_bytes(static_cast<uint8_t *>(a.out), row * a.ldo + c, cols - c, w);
          if ((t & 3) == 0) a.scales[row * a.ld_scales + (c >> 5)] = (uint8_t)(k + 127);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = col0 + i * TPR * 8;
        if (c < cols) store8_any(a.out_type, a.out, row * a.ldo + c, cols - c, v[i]);
      }
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------

int CheckMatrix(const char *call, const char *name, const amlike_matrix_t *m, int64_t rows, int64_t cols) {
  if (!m || m->type < AMLIKE_F32 || m->type > AMLIKE_MX8) {
    SetError("%s: %s is missing or of an unknown type", call, name);
    return AMLIKE_EINVAL;
  }
  if (rows == 0) return AMLIKE_OK;
  const bool mx8 = m->type == AMLIKE_MX8;
  if (!m->data || reinterpret_cast<uintptr_t>(m->data) % TypeBytes(m->type) || (mx8 && !m->scales)) {
    SetError("%s: %s has no data%s, or data not aligned to its type", call, name, mx8 ? " or no scales" : "");
    return AMLIKE_EINVAL;
  }
  // (2^48 elements: further than any device's memory, and products with rows stay in 64 bits)
  if (m->ld < cols || (mx8 && m->ld_scales < (cols + 31) / 32) || m->ld > ((int64_t)1 << 48) / rows ||
      (mx8 && m->ld_scales > ((int64_t)1 << 48) / rows)) {
    SetError("%s: %s has row stride %lld (scales %lld) for %lld rows of %lld columns", call, name, (long long)m->ld,
             mx8 ? (long long)m->ld_scales : 0LL, (long long)rows, (long long)cols);
    return AMLIKE_EINVAL;
  }
  return AMLIKE_OK;
}

namespace {

// Rows of bytes: the values or the scales of a matrix.  (A single row has no stride.)
struct Strip {
  uintptr_t at;
  uint64_t stride, width, rows;
};
int Strips(const amlike_matrix_t *m, int64_t rows, int64_t cols, Strip s[2]) {
  const uint64_t es = TypeBytes(m->type), n = (uint64_t)rows;
  s[0] = {reinterpret_cast<uintptr_t>(m->data), n > 1 ? (uint64_t)m->ld * es : 0, (uint64_t)cols * es, n};
  if (m->type != AMLIKE_MX8) return 1;
  s[1] = {reinterpret_cast<uintptr_t>(m->scales), n > 1 ? (uint64_t)m->ld_scales : 0, (uint64_t)(cols + 31) / 32, n};
  return 2;
}
// The sum of floor((a i + b) / m) over 0 <= i < n, by turning the count of lattice points below the line
// round as often as Euclid's algorithm has steps.
typedef unsigned __int128 Wide;
Wide FloorSum(Wide n, Wide m, Wide a, Wide b) {
  Wide sum = 0;
  for (;;) {
    sum += n * (n - 1) / 2 * (a / m) + n * (b / m);
    a %= m;
    b %= m;
    const Wide top = a * n + b;
    if (top < m) return sum;
    n = top / m;
    b = top % m;
    std::swap(m, a);
  }
}
// Whether a byte belongs to both.
bool StripsMeet(Strip a, Strip b) {
  if (b.stride == 0) std::swap(a, b);
  const uintptr_t a_end = a.at + (a.rows - 1) * a.stride + a.width, b_end = b.at + (b.rows - 1) * b.stride + b.width;
  if (a.at >= b_end || b.at >= a_end) return false;
  if (b.stride == 0) return true;  // two single rows
  // Rows of a that lie within b's stretch, if only in part.  A row meets a row of b, whichever, if one of the
  // starts b.at + j * b.stride lies in the b.width - 1 bytes before it or in itself: the floors count them.
  // (A start that is not one of b's, before the first or behind the last, only counts where the first or last does.)
  const uint64_t lo = a.at + a.width > b.at ? 0 : a.stride ? (b.at - (a.at + a.width)) / a.stride + 1 : a.rows;
  const uint64_t hi = a.stride ? std::min<uint64_t>(a.rows - 1, (b_end - 1 - a.at) / a.stride) : 0;
  if (lo > hi) return false;
  const uint64_t up = (b.at + b.width) / b.stride + 1;  // (the starts moved up by whole strides: nothing is negative)
  const Wide first = (Wide)a.at + (Wide)lo * a.stride + (Wide)up * b.stride - b.at;
  const Wide n = hi - lo + 1;
  return FloorSum(n, b.stride, a.stride, first + a.width - 1) != FloorSum(n, b.stride, a.stride, first - b.width);
}

template <int TIN, bool NORM, int TPR, int NCH>
int LaunchRows(RowArgs a, hipStream_t st) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, kTeams = kThreads / TPR;
  a.col_blocks = NORM ? 1 : (a.dim + TPR * NCH * 8 - 1) / (TPR * NCH * 8);
  a.blocks = (a.rows + kTeams - 1) / kTeams * a.col_blocks;
  // (a grid holds less than 2^32 threads; the kernel strides over what is left)
  const unsigned grid = (unsigned)std::min<int64_t>(a.blocks, (int64_t)1 << 21);
  hipLaunchKernelGGL((dense_rows_kernel<TIN, NORM, TPR, NCH>), dim3(grid), dim3(kThreads), 0, st, a);
  AMLIKE_HIP(hipGetLastError());
  return AMLIKE_OK;
}

// Teams by the row's chunks of 8 columns: as many threads as it has chunks while they are lanes of a
// wave, then two chunks a thread, then as many as a block may have.  Microseconds, bf16, norm with residual and
// sum (35 554 rows / 64 rows; the first is bounded by HBM, the second by latency):
//   128 wide, to bf16    16 lanes  7.2 / 2.64    64 lanes         14.3 / 3.03
//   1024, to 8 bits      64 x 2   39.9 / 3.39    256 threads      52.4 / 3.26
//   2000                 256 x 1  96.9 / 3.36    64 lanes x 4     98.7 / 4.54
//   4096 (16 384 rows)   256 x 2  82.7 / 3.55    1024 threads      102 / 3.89
//   8192 (8 192 rows)    1024 x 1 85.4 / 4.08    256 threads x 4  84.3 / 4.56
// Conversion of 35 554 x 2000 bf16 to 8 bits: 64 x 2 36.1, 64 x 1 39.2, 256 x 1 36.2; of 360 columns
// of fp32: 64 x 1 12.7, 256 x 1 26.7.
template <int TIN, bool NORM>
int PickTeams(const RowArgs &a, hipStream_t st) {
  const int64_t chunks = ((int64_t)a.dim + 7) / 8;
  if (chunks <= 16) return LaunchRows<TIN, NORM, 16, 1>(a, st);
  if (chunks <= 32) return LaunchRows<TIN, NORM, 32, 1>(a, st);
  if (chunks <= 64) return LaunchRows<TIN, NORM, 64, 1>(a, st);
  if (chunks <= 128 || !NORM) return LaunchRows<TIN, NORM, 64, 2>(a, st);
  if constexpr (NORM) {
    if (chunks <= 256) return LaunchRows<TIN, NORM, 256, 1>(a, st);
    if (chunks <= 512) return LaunchRows<TIN, NORM, 256, 2>(a, st);
    if (chunks <= 1024) return LaunchRows<TIN, NORM, 1024, 1>(a, st);
    if (chunks <= 2048) return LaunchRows<TIN, NORM, 1024, 2>(a, st);
    return LaunchRows<TIN, NORM, 1024, 4>(a, st);
  }
  return AMLIKE_EINVAL;
}

template <bool NORM>
int PickType(int type, const RowArgs &a, hipStream_t st) {
  if (type == AMLIKE_F32) return PickTeams<AMLIKE_F32, NORM>(a, st);
  if (type == AMLIKE_BF16) return PickTeams<AMLIKE_BF16, NORM>(a, st);
  return PickTeams<AMLIKE_F16, NORM>(a, st);
}

constexpr int kNormMaxDim = 32768;  // 1024 threads x 4 chunks x 8 columns

}  // namespace

bool MatricesOverlap(const amlike_matrix_t *a, int64_t rows_a, int64_t cols_a, const amlike_matrix_t *b,
                     int64_t rows_b, int64_t cols_b) {
  Strip sa[2], sb[2];
  const int na = Strips(a, rows_a, cols_a, sa), nb = Strips(b, rows_b, cols_b, sb);
  for (int i = 0; i < na; ++i)
    for (int j = 0; j < nb; ++j)
      if (StripsMeet(sa[i], sb[j])) return true;
  return false;
}

int CheckOutput(const char *call, const amlike_matrix_t *out, int64_t rows, int64_t cols) {
  if (int rc = CheckMatrix(call, "out", out, rows, cols)) return rc;
  Strip s[2];
  if (rows > 0 && Strips(out, rows, cols, s) == 2 && StripsMeet(s[0], s[1])) {
    SetError("%s: out's values and scales overlap", call);
    return AMLIKE_EINVAL;
  }
  return AMLIKE_OK;
}

int LaunchConvert(const amlike_matrix_t &x, int64_t rows, int64_t cols, const amlike_matrix_t &out, hipStream_t st) {
  RowArgs a = {};
  a.x = x.data;
  a.ldx = x.ld;
  a.out = out.data;
  a.ldo = out.ld;
  a.scales = static_cast<uint8_t *>(out.scales);
  a.ld_scales = out.ld_scales;
  a.rows = rows;
  a.dim = (int32_t)cols;
  a.out_type = out.type;
  return PickType<false>(x.type, a, st);
}

}  // namespace amlike

using namespace amlike;

struct amlike_norm {
  int device = 0;
  int dim = 0;
  float eps = 0;
  float *d_weight = nullptr;  // NULL: ones
  // the host-pointer call's own stream and buffers
  hipStream_t stream = nullptr;
  DeviceBuffer ws_x, ws_r, ws_out;
  std::mutex mu;
};

extern "C" {

int amlike_convert_dev(const amlike_matrix_t *x, int32_t rows, int32_t cols, const amlike_matrix_t *out,
                       void *stream) {
  const char *call = "amlike_convert";
  if (int rc = BindThread()) return rc;
  if (rows < 0 || cols <= 0 || cols > (1 << 30)) {
    SetError("%s: %d rows of %d columns", call, rows, cols);
    return AMLIKE_EINVAL;
  }
  if (int rc = CheckMatrix(call, "x", x, rows, cols)) return rc;
  if (int rc = CheckOutput(call, out, rows, cols)) return rc;
  if (x->type == AMLIKE_MX8) {
    SetError("%s: x in 8 bits is not an input", call);
    return AMLIKE_EINVAL;
  }
  if (rows == 0) return AMLIKE_OK;
  if (MatricesOverlap(x, rows, cols, out, rows, cols)) {
    SetError("%s: x and out overlap", call);
    return AMLIKE_EINVAL;
  }
  if (CurrentDevice() < 0) {
    if (int rc = amlike_init(0)) return rc;
  }
  return LaunchConvert(*x, rows, cols, *out, static_cast<hipStream_t>(stream));
}

int amlike_norm_create(const float *weight, int32_t dim, float eps, amlike_norm_t **out) {
  if (int rc = BindThread()) return rc;
  if (!out || dim <= 0 || dim > kNormMaxDim || !(eps >= 1e-30f && eps <= 1.0f)) {
    SetError("amlike_norm_create: dim %d (1 to %d) or eps %g (1e-30 to 1) out of range", dim, kNormMaxDim, (double)eps);
    return AMLIKE_EINVAL;
  }
  *out = nullptr;
  if (CurrentDevice() < 0) {
    if (int rc = amlike_init(0)) return rc;
  }
  amlike_norm *h = new (std::nothrow) amlike_norm;
  if (!h) {
    SetError("amlike_norm_create: out of host memory");
    return AMLIKE_EOOM;
  }
  h->device = CurrentDevice();
  h->dim = dim;
  h->eps = eps;
  hipError_t e = hipSuccess;
  if (weight) {
    e = hipMalloc(reinterpret_cast<void **>(&h->d_weight), (size_t)dim * sizeof(float));
    if (e == hipSuccess) e = hipMemcpy(h->d_weight, weight, (size_t)dim * sizeof(float), hipMemcpyHostToDevice);
  }
  if (e == hipSuccess) e = hipStreamCreateWithFlags(&h->stream, hipStreamNonBlocking);
  if (e != hipSuccess) {
    SetError("amlike_norm_create: %s", HipFailure(e));
    amlike_norm_destroy(h);
    return e == hipErrorOutOfMemory ? AMLIKE_EOOM : AMLIKE_EHIP;
  }
  *out = h;
  return AMLIKE_OK;
}

int amlike_norm_destroy(amlike_norm_t *h) {
  if (int rc = BindHandle(h)) return rc;
  if (!h) return AMLIKE_OK;
  (void)hipFree(h->d_weight);
  h->ws_x.Free();
  h->ws_r.Free();
  h->ws_out.Free();
  if (h->stream) (void)hipStreamDestroy(h->stream);
  delete h;
  return AMLIKE_OK;
}

int32_t amlike_norm_dim(const amlike_norm_t *h) { return h ? h->dim : 0; }
int32_t amlike_norm_device(const amlike_norm_t *h) { return h ? h->device : -1; }

int amlike_norm_apply_dev(const amlike_norm_t *h, const amlike_matrix_t *x, const amlike_matrix_t *residual,
                          int32_t rows, const amlike_matrix_t *sum, const amlike_matrix_t *out, void *stream) {
  const char *call = "amlike_norm_apply";
  if (int rc = BindHandle(h)) return rc;
  if (!h || rows < 0) {
    SetError("%s: no handle, or %d rows", call, rows);
    return AMLIKE_EINVAL;
  }
  const int dim = h->dim;
  if (int rc = CheckMatrix(call, "x", x, rows, dim)) return rc;
  if (int rc = CheckOutput(call, out, rows, dim)) return rc;
  if (residual)
    if (int rc = CheckMatrix(call, "residual", residual, rows, dim)) return rc;
  if (sum)
    if (int rc = CheckMatrix(call, "sum", sum, rows, dim)) return rc;
  if (x->type == AMLIKE_MX8 || (residual && residual->type != x->type) || (sum && sum->type != x->type)) {
    SetError("%s: x, residual and sum are of one type, which is not the 8-bit one", call);
    return AMLIKE_EINVAL;
  }
  if (rows == 0) return AMLIKE_OK;
  const amlike_matrix_t *writes[2] = {out, sum}, *reads[2] = {x, residual};
  for (const amlike_matrix_t *w : writes)
    for (const amlike_matrix_t *r : reads)
      if (w && r && !SameMatrix(w, r) && MatricesOverlap(w, rows, dim, r, rows, dim)) {
        SetError("%s: an output overlaps an input and is not the same matrix", call);
        return AMLIKE_EINVAL;
      }
  if (sum && MatricesOverlap(sum, rows, dim, out, rows, dim)) {
    SetError("%s: sum and out overlap", call);
    return AMLIKE_EINVAL;
  }
  RowArgs a = {};
  a.x = x->data;
  a.ldx = x->ld;
  if (residual) {
    a.r = residual->data;
    a.ldr = residual->ld;
  }
  if (sum) {
    a.sum = sum->data;
    a.lds = sum->ld;
  }
  a.out = out->data;
  a.ldo = out->ld;
  a.scales = static_cast<uint8_t *>(out->scales);
  a.ld_scales = out->ld_scales;
  a.weight = h->d_weight;
  a.rows = rows;
  a.dim = dim;
  a.out_type = out->type;
  a.eps = h->eps;
  a.inv_dim = (float)(1.0 / dim);
  return PickType<true>(x->type, a, static_cast<hipStream_t>(stream));
}

int amlike_norm_apply(amlike_norm_t *h, const float *x, int32_t ld, const float *residual, int32_t ldr,
                      int32_t rows, float *sum, int32_t lds, float *out, int32_t ldo) {
  if (int rc = BindHandle(h)) return rc;
  if (!h || !x || !out || rows < 0 || ld < h->dim || ldo < h->dim || (residual && ldr < h->dim) || (sum && lds < h->dim)) {
    SetError("amlike_norm_apply: invalid argument");
    return AMLIKE_EINVAL;
  }
  if (rows == 0) return AMLIKE_OK;
  std::lock_guard<std::mutex> lock(h->mu);
  const size_t row = (size_t)h->dim * sizeof(float), bytes = row * rows;
  int rc = h->ws_x.Reserve(bytes);
  if (rc == AMLIKE_OK && residual) rc = h->ws_r.Reserve(bytes);
  if (rc == AMLIKE_OK) rc = h->ws_out.Reserve(bytes);
  if (rc != AMLIKE_OK) return rc;
  AMLIKE_HIP(hipMemcpy2DAsync(h->ws_x.ptr, row, x, (size_t)ld * sizeof(float), row, rows, hipMemcpyHostToDevice, h->stream));
  if (residual)
    AMLIKE_HIP(hipMemcpy2DAsync(h->ws_r.ptr, row, residual, (size_t)ldr * sizeof(float), row, rows, hipMemcpyHostToDevice,
                                h->stream));
  const amlike_matrix_t mx = {h->ws_x.ptr, nullptr, h->dim, 0, AMLIKE_F32}, mr = {h->ws_r.ptr, nullptr, h->dim, 0, AMLIKE_F32},
                        mo = {h->ws_out.ptr, nullptr, h->dim, 0, AMLIKE_F32};
  // the sum replaces x in place
  rc = amlike_norm_apply_dev(h, &mx, residual ? &mr : nullptr, rows, sum ? &mx : nullptr, &mo, h->stream);
  if (rc != AMLIKE_OK) {
    (void)hipStreamSynchronize(h->stream);  // the copies above read the caller's arrays
    return rc;
  }
  if (sum)
    AMLIKE_HIP(hipMemcpy2DAsync(sum, (size_t)lds * sizeof(float), h->ws_x.ptr, row, row, rows, hipMemcpyDeviceToHost, h->stream));
  return CopyMatrixToHost(out, (size_t)ldo, static_cast<const float *>(h->ws_out.ptr), rows, h->dim, h->stream);
}

}  // extern "C"
