// amlike_linear_*: the host side of the matrix product with bias, activation and residual, the choice of
// a kernel's form, and the packing of the weights.  The kernels: linear_kernels.h.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <new>

#include "linear_kernels.h"

namespace amlike {

constexpr int kLinearMaxDim = 1 << 20;  // either dimension of a layer
constexpr int kMaxBlocks = 1 << 22;     // of a launch

extern template int LaunchLinear<AMLIKE_BF16>(const LinearArgs &, hipStream_t);
extern template int LaunchLinear<AMLIKE_F16>(const LinearArgs &, hipStream_t);
extern template int LaunchLinear<AMLIKE_MX8>(const LinearArgs &, hipStream_t);
extern template int LaunchLinear<kMx8Exact>(const LinearArgs &, hipStream_t);

// ---- the choice of a form ---------------------------------------------------------------------------------

// The form with the least estimated time, from the turns that the busiest compute unit has to take.
// Microseconds per k-tile and per turn, measured in bf16 at the sizes behind each line with W in the caches (less
// the 2.2 that every launch takes); only their relation matters.
//   256 x 256, 8 waves                      1.62 kt + 7    35554 x 2000 x 8600: 1118 (measured 1157)
//   128 x 128, 4 waves, alone on its unit   0.65 kt + 2    1024 x 4096 x 4096: 44 (44.5)
//              two of them                  0.95 kt + 4    4096 x 2048 x 2048: 34 (34.4)
//   128 x 128, 2 groups of 4 waves          0.55 kt + 3    1024 x 4096 x 4096: 38 (38.7)
//   64 x 64, 4 waves, alone                 0.31 kt + 1    300 x 360 x 2000: 2.9 (5.5 with the launch)
//            two of them                    0.38 kt + 2    1024 x 4096 x 4096: 53 (54)
//   64 x 64, 2 groups of 4 waves            0.27 kt + 1.5  32 x 4096 x 16384: 21 (22.4 with it)
// Rows of x that do not start and end on 16 bytes go through registers, in two forms:
//   64 x 64, four blocks a unit             0.36 kt each   1237 x 1999 x 2001 bf16: 30.0 (128 x 128: 39.5)
//            alone                          0.45 kt        64 x 2000 x 1024: 14.4 (16.0 with it)
//   128 x 128, alone / two of them   1.25 kt / 2.0 kt      2000 x 2002 x 4096 mx8: 32.0 (64 x 64: 53.1)
// The thin kernel, whatever the rows' places; the second figure where they are not on 16 bytes
// (sizes and times as above, all with the launch), and 0.5 a turn:
//   16 rows x 16 outputs                    0.12, 0.18 kt  64 x 4096 x 1024: 9.5 (64 x 64: 21.3)
//   16 rows x 32 outputs                    0.19, 0.20 kt  16 x 8192 x 8192: 24.9 (16 x 16: 31.1)
//   32 rows x 16 outputs                    0.18, 0.33 kt  128 x 4096 x 1024: 13.0 (64 x 64: 21.4)
//   32 rows x 32 outputs                    0.25, 0.37 kt  64 x 4096 x 4096: 17.5 (64 x 64: 21.7)
//   64 rows x 32 outputs                    0.35, 0.66 kt  256 x 4096 x 2048 mx8 to f32: 17.2 (20.0)
// 8-bit operands widened to 16 cost the tile kernels 1.9 times a k-tile (twice the products, and every wave
// widens what it reads) and the thin one 1.08 times: 1.75 in relation.
LinearChoice ChooseLinear(int kind, int out_type, int64_t rows, int k_tiles, int n_pad, bool copy, bool far_apart, int units) {
  const double k = k_tiles, kt = kind == kMx8Exact ? 1.75 * k : k;
  auto turns = [&](int r, int outputs) {
    return std::ceil((double)((rows + r - 1) / r * ((n_pad + outputs - 1) / outputs)) / std::max(1, units));
  };
  auto thin_cost = [&](int r, int outputs, double on_16, double off) { return turns(r, outputs) * ((copy ? on_16 : off) * k + 0.5); };
  const double thin[5] = {thin_cost(16, 16, 0.12, 0.18), thin_cost(16, 32, 0.19, 0.20), thin_cost(32, 16, 0.18, 0.33),
                          thin_cost(32, 32, 0.25, 0.37), thin_cost(64, 32, 0.35, 0.66)};
  const double t256 = turns(256, 256), t128 = turns(128, 128), t64 = turns(64, 64);
  const double tile[7] = {t256 * (1.62 * kt + 7),
                          t128 <= 1 ? 0.65 * kt + 2 : std::ceil(t128 / 2) * (0.95 * kt + 4),
                          t128 * (0.55 * kt + 3),
                          t64 <= 1 ? 0.31 * kt + 1 : std::ceil(t64 / 2) * (0.38 * kt + 2),
                          t64 * (0.27 * kt + 1.5),
                          t64 <= 1 ? 0.45 * kt : std::ceil(t64 / 4) * std::min(t64, 4.0) * 0.36 * kt,
                          t128 <= 1 ? 1.25 * kt : std::ceil(t128 / 2) * 2.0 * kt};
  // (with widened 8-bit operands the largest tile's registers do not suffice)
  const int first = !copy ? 5 : kind == kMx8Exact ? 1 : 0, last = copy ? 5 : 7;
  const int best = (int)(std::min_element(tile + first, tile + last) - tile);
  // (a group of 32 8-bit outputs stays in one block)
  int few = out_type == AMLIKE_MX8 ? 1 : 0;
  for (int i = few + 1; i < 5; ++i)
    if (thin[i] < thin[few] && (i != 2 || out_type != AMLIKE_MX8)) few = i;
  if (thin[few] < tile[best] || far_apart) return {true, few};
  return {false, best};
}

// ---- packing the weights ---------------------------------------------------------------------------------

// One 16-byte piece of the packed W per thread, from rows already in the handle's type.
__global__ __launch_bounds__(256) void linear_pack_kernel(const uint8_t *__restrict__ src, int type, int n, int k,
                                                          int n_pad, int64_t pieces, u32x4 *__restrict__ dst,
                                                          int *__restrict__ bad) {
  for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < pieces; p += (int64_t)gridDim.x * 256) {
    const int c = (int)(p & 7);
    const int64_t tr = p >> 3;
    const int kt = (int)(tr / n_pad), row = (int)(tr - (int64_t)kt * n_pad);
    const int es = type == AMLIKE_MX8 ? 1 : 2;
    u32x4 q = {0, 0, 0, 0};
    if (row < n) q = load_chunk(src + (int64_t)row * k * es, kt * kTileBytes + c * 16, k * es);
    dst[p] = q;
    bool no = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (type == AMLIKE_MX8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) no |= (q[i] >> (8 * j) & 0x7f) == 0x7f;
      } else {
        const uint32_t e = type == AMLIKE_BF16 ? 0x7f80u : 0x7c00u;
        no |= (q[i] & e) == e || (q[i] >> 16 & e) == e;
      }
    }
    if (no) ctl_or(bad, 1);
  }
}
// One word (four groups' scales) per thread.  A group of zeros has 2^0 here instead of the format's smallest
// scale: the same products, and nothing for a kernel to look at closely.
__global__ __launch_bounds__(256) void linear_pack_scales_kernel(const uint8_t *__restrict__ src, const uint8_t *__restrict__ values,
                                                                 int n, int k, int n_pad, int64_t words, uint32_t *__restrict__ dst) {
  const int groups = (k + 31) >> 5;
  for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < words; p += (int64_t)gridDim.x * 256) {
    const int64_t line = p >> 2;
    const int four = (int)(line / n_pad), row = (int)(line - (int64_t)four * n_pad);
    uint32_t s = 0x7f7f7f7fu;
    if (row < n) {
      const int kt = four * 4 + (int)(p & 3);
      s = load_scales(src + (int64_t)row * groups, kt, groups);
      for (int i = 0; i < 4; ++i) {
        if ((s >> (8 * i) & 0xff) != 0) continue;
        const int first = (kt * 4 + i) * 32;
        uint8_t any = 0;
        for (int c = first; c < min(first + 32, k); ++c) any |= values[(int64_t)row * k + c] & 0x7f;
        if (any == 0) s |= 0x7fu << (8 * i);
      }
    }
    dst[p] = s;
  }
}

}  // namespace amlike

using namespace amlike;

struct amlike_linear {
  int device = 0;
  int k = 0, n = 0, n_pad = 0, k_tiles = 0, type = 0;
  int max_blocks = kMaxBlocks;  // AMLIKE_LINEAR_MAX_BLOCKS: fewer, for tests of a call in several launches
  uint8_t *d_w = nullptr;
  uint32_t *d_scales = nullptr;
  float *d_bias = nullptr;
  // the host-pointer call's own stream and buffers
  hipStream_t stream = nullptr;
  DeviceBuffer ws_x, ws_q, ws_r, ws_out;
  std::mutex mu;
};

namespace amlike {
namespace {

int PadOutputs(int n) { return (n + 63) / 64 * 64; }
int KTiles(int k, int type) { return (int)(((int64_t)k * TypeBytes(type) + kTileBytes - 1) / kTileBytes); }
// The kind of product of a layer's type for an output's.
int KindOf(int type, int out_type) { return type == AMLIKE_MX8 && out_type == AMLIKE_F32 ? kMx8Exact : type; }

int PackWeights(amlike_linear *h, const float *weights, int64_t ld, const float *bias) {
  const size_t row = (size_t)h->k * sizeof(float);
  const int es = TypeBytes(h->type), groups = (h->k + 31) / 32;
  const int64_t pieces = (int64_t)h->k_tiles * h->n_pad * kChunks;
  DeviceBuffer src, typed, scales, flag;
  auto work = [&]() -> int {
    int rc = src.Reserve(row * h->n);
    if (rc == AMLIKE_OK) rc = typed.Reserve((size_t)h->n * h->k * es);
    if (rc == AMLIKE_OK && h->type == AMLIKE_MX8) rc = scales.Reserve((size_t)h->n * groups);
    if (rc == AMLIKE_OK) rc = flag.Reserve(sizeof(int));
    if (rc != AMLIKE_OK) return rc;
    AMLIKE_HIP(hipMalloc(reinterpret_cast<void **>(&h->d_w), (size_t)pieces * 16));
    AMLIKE_HIP(hipMalloc(reinterpret_cast<void **>(&h->d_bias), (size_t)h->n_pad * sizeof(float)));
    rc = ClearWords(static_cast<int *>(flag.ptr), 1, h->stream);
    if (rc == AMLIKE_OK) rc = ClearWords(reinterpret_cast<int *>(h->d_bias), h->n_pad, h->stream);
    if (rc != AMLIKE_OK) return rc;
    if (bias) AMLIKE_HIP(hipMemcpyAsync(h->d_bias, bias, (size_t)h->n * sizeof(float), hipMemcpyHostToDevice, h->stream));
    AMLIKE_HIP(hipMemcpy2DAsync(src.ptr, row, weights, (size_t)ld * sizeof(float), row, h->n, hipMemcpyHostToDevice, h->stream));
    const amlike_matrix_t ms = {src.ptr, nullptr, h->k, 0, AMLIKE_F32}, mt = {typed.ptr, scales.ptr, h->k, groups, h->type};
    rc = LaunchConvert(ms, h->n, h->k, mt, h->stream);
    if (rc != AMLIKE_OK) return rc;
    hipLaunchKernelGGL(linear_pack_kernel, dim3((unsigned)std::min<int64_t>((pieces + 255) / 256, 1 << 16)), dim3(256), 0,
                       h->stream, static_cast<const uint8_t *>(typed.ptr), h->type, h->n, h->k, h->n_pad, pieces,
                       reinterpret_cast<u32x4 *>(h->d_w), static_cast<int *>(flag.ptr));
    AMLIKE_HIP(hipGetLastError());
    if (h->type == AMLIKE_MX8) {
      const int64_t words = (int64_t)((h->k_tiles + 3) & ~3) * h->n_pad;
      AMLIKE_HIP(hipMalloc(reinterpret_cast<void **>(&h->d_scales), (size_t)words * 4));
      hipLaunchKernelGGL(linear_pack_scales_kernel, dim3((unsigned)std::min<int64_t>((words + 255) / 256, 1 << 16)), dim3(256), 0,
                         h->stream, static_cast<const uint8_t *>(scales.ptr), static_cast<const uint8_t *>(typed.ptr), h->n, h->k,
                         h->n_pad, words, h->d_scales);
      AMLIKE_HIP(hipGetLastError());
    }
    int bad = 0;
    AMLIKE_HIP(hipMemcpyAsync(&bad, flag.ptr, sizeof(int), hipMemcpyDeviceToHost, h->stream));
    AMLIKE_HIP(hipStreamSynchronize(h->stream));
    if (bad) {
      SetError("amlike_linear_create: a weight is not finite in the layer's type");
      return AMLIKE_ENONFINITE;
    }
    return AMLIKE_OK;
  };
  const int rc = work();
  if (rc != AMLIKE_OK) (void)hipStreamSynchronize(h->stream);
  src.Free();
  typed.Free();
  scales.Free();
  flag.Free();
  return rc;
}

}  // namespace
}  // namespace amlike

extern "C" {

int amlike_linear_create(const float *weights, int32_t ld, const float *bias, int32_t input_dim, int32_t output_dim,
                         int32_t type, amlike_linear_t **out) {
  if (int rc = BindThread()) return rc;
  if (!out || !weights || input_dim <= 0 || output_dim <= 0 || input_dim > kLinearMaxDim || output_dim > kLinearMaxDim ||
      ld < input_dim || (type != AMLIKE_BF16 && type != AMLIKE_F16 && type != AMLIKE_MX8)) {
    SetError("amlike_linear_create: invalid argument (dimensions 1 to %d, type BF16, F16 or MX8)", kLinearMaxDim);
    return AMLIKE_EINVAL;
  }
  *out = nullptr;
  if (bias)
    for (int i = 0; i < output_dim; ++i)
      if (!(bias[i] - bias[i] == 0.0f)) {
        SetError("amlike_linear_create: bias %d is not finite", i);
        return AMLIKE_ENONFINITE;
      }
  if (CurrentDevice() < 0) {
    if (int rc = amlike_init(0)) return rc;
  }
  amlike_linear *h = new (std::nothrow) amlike_linear;
  if (!h) {
    SetError("amlike_linear_create: out of host memory");
    return AMLIKE_EOOM;
  }
  h->device = CurrentDevice();
  h->k = input_dim;
  h->n = output_dim;
  h->type = type;
  h->n_pad = PadOutputs(output_dim);
  h->k_tiles = KTiles(input_dim, type);
  if (const char *e = getenv("AMLIKE_LINEAR_MAX_BLOCKS")) h->max_blocks = std::max(1, std::min(kMaxBlocks, atoi(e)));
  const hipError_t e = hipStreamCreateWithFlags(&h->stream, hipStreamNonBlocking);
  int rc = AMLIKE_OK;
  if (e != hipSuccess) {
    SetError("amlike_linear_create: %s", HipFailure(e));
    rc = AMLIKE_EHIP;
  }
  if (rc == AMLIKE_OK) rc = PackWeights(h, weights, ld, bias);
  if (rc != AMLIKE_OK) {
    amlike_linear_destroy(h);
    return rc;
  }
  *out = h;
  return AMLIKE_OK;
}

int amlike_linear_destroy(amlike_linear_t *h) {
  if (int rc = BindHandle(h)) return rc;
  if (!h) return AMLIKE_OK;
  (void)hipFree(h->d_w);
  (void)hipFree(h->d_scales);
  (void)hipFree(h->d_bias);
  h->ws_x.Free();
  h->ws_q.Free();
  h->ws_r.Free();
  h->ws_out.Free();
  if (h->stream) (void)hipStreamDestroy(h->stream);
  delete h;
  return AMLIKE_OK;
}

int32_t amlike_linear_input_dim(const amlike_linear_t *h) { return h ? h->k : 0; }
int32_t amlike_linear_output_dim(const amlike_linear_t *h) { return h ? h->n : 0; }
int32_t amlike_linear_type(const amlike_linear_t *h) { return h ? h->type : -1; }
int32_t amlike_linear_device(const amlike_linear_t *h) { return h ? h->device : -1; }

int amlike_linear_apply_dev(const amlike_linear_t *h, const amlike_matrix_t *x, int32_t rows, int32_t activation,
                            const amlike_matrix_t *residual, const amlike_matrix_t *out, void *stream) {
  const char *call = "amlike_linear_apply";
  if (int rc = BindHandle(h)) return rc;
  if (!h || rows < 0 || activation < AMLIKE_ACT_NONE || activation > AMLIKE_ACT_GELU) {
    SetError("%s: no handle, %d rows, or unknown activation %d", call, rows, activation);
    return AMLIKE_EINVAL;
  }
  if (int rc = CheckMatrix(call, "x", x, rows, h->k)) return rc;
  if (int rc = CheckOutput(call, out, rows, h->n)) return rc;
  if (residual)
    if (int rc = CheckMatrix(call, "residual", residual, rows, h->n)) return rc;
  if (x->type != h->type || (residual && residual->type == AMLIKE_MX8)) {
    SetError("%s: x has not the layer's type, or the residual is in 8 bits", call);
    return AMLIKE_EINVAL;
  }
  if (rows == 0) return AMLIKE_OK;
  if (MatricesOverlap(x, rows, h->k, out, rows, h->n) ||
      (residual && !SameMatrix(residual, out) && MatricesOverlap(residual, rows, h->n, out, rows, h->n))) {
    SetError("%s: out overlaps an input", call);
    return AMLIKE_EINVAL;
  }
  LinearArgs a = {};
  a.x = static_cast<const uint8_t *>(x->data);
  a.ldx = x->ld * TypeBytes(x->type);
  if (x->type == AMLIKE_MX8) {  // (in the other types the fields may hold anything)
    a.x_scales = static_cast<const uint8_t *>(x->scales);
    a.ld_xs = x->ld_scales;
  }
  a.w = h->d_w;
  a.w_scales = h->d_scales;
  a.bias = h->d_bias;
  a.res_type = -1;
  if (residual) {
    a.res = residual->data;
    a.ldr = residual->ld;
    a.res_type = residual->type;
  }
  a.out = out->data;
  a.ldo = out->ld;
  if (out->type == AMLIKE_MX8) {
    a.out_scales = static_cast<uint8_t *>(out->scales);
    a.ld_os = out->ld_scales;
  }
  a.out_type = out->type;
  a.rows = rows;
  a.k = h->k;
  a.n = h->n;
  a.n_pad = h->n_pad;
  a.k_tiles = h->k_tiles;
  a.act = activation;
  a.max_blocks = h->max_blocks;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int kind = KindOf(h->type, out->type);
  if (kind == AMLIKE_BF16) return LaunchLinear<AMLIKE_BF16>(a, st);
  if (kind == AMLIKE_F16) return LaunchLinear<AMLIKE_F16>(a, st);
  if (kind == kMx8Exact) return LaunchLinear<kMx8Exact>(a, st);
  return LaunchLinear<AMLIKE_MX8>(a, st);
}

const char *amlike_linear_kernel_info(int32_t type, int32_t out_type, int32_t rows, int32_t input_dim, int32_t output_dim,
                                      int32_t aligned, int32_t units) {
  static thread_local char text[128];
  text[0] = 0;
  if (type < AMLIKE_BF16 || type > AMLIKE_MX8 || out_type < AMLIKE_F32 || out_type > AMLIKE_MX8 || rows <= 0 || input_dim <= 0 ||
      output_dim <= 0 || input_dim > kLinearMaxDim || output_dim > kLinearMaxDim || units <= 0 || units > 1 << 16)
    return text;
  const int kind = KindOf(type, out_type), n_pad = PadOutputs(output_dim);
  const LinearChoice c = ChooseLinear(kind, out_type, rows, KTiles(input_dim, type), n_pad, aligned != 0, false, units);
  if (c.thin) {
    const ThinForm f = kThinForms[c.form];
    snprintf(text, sizeof(text), "linear_thin_kernel<%d,%d,%d> rows=%d outputs=%d", kind, f.nt, f.mt, 16 * f.mt, 16 * f.nt);
  } else {
    const TileForm f = kTileForms[c.form];
    const long long m = ((long long)rows + 16 * f.mf * f.wm - 1) / (16 * f.mf * f.wm), n = (n_pad + 64 * f.wn - 1) / (64 * f.wn);
    snprintf(text, sizeof(text), "linear_pipe_kernel<%d,%d,%d,%d,%d,%d,%d> rows=%d outputs=%d tiles=%lld blocks=%lld", kind, f.wn, f.wm,
             f.mf, f.stages, f.ks, f.copy ? 1 : 0, 16 * f.mf * f.wm, 64 * f.wn, m * n,
             std::min<long long>((m * n + 7) & ~7LL, BlocksHeld(kind, f, units)));
  }
  return text;
}

int amlike_linear_apply(amlike_linear_t *h, const float *x, int32_t ld, int32_t rows, int32_t activation,
                        const float *residual, int32_t ldr, float *out, int32_t ldo) {
  if (int rc = BindHandle(h)) return rc;
  if (!h || !x || !out || rows < 0 || ld < h->k || ldo < h->n || (residual && ldr < h->n)) {
    SetError("amlike_linear_apply: invalid argument");
    return AMLIKE_EINVAL;
  }
  if (rows == 0) return AMLIKE_OK;
  std::lock_guard<std::mutex> lock(h->mu);
  const size_t xrow = (size_t)h->k * sizeof(float), orow = (size_t)h->n * sizeof(float);
  const int groups = ((h->k + 31) / 32 + 15) / 16 * 16;  // (a row's scales start on 16 bytes)
  const size_t ldq = ((size_t)h->k + 15) / 16 * 16, values = ldq * TypeBytes(h->type) * rows;
  int rc = h->ws_x.Reserve(xrow * rows);
  if (rc == AMLIKE_OK) rc = h->ws_q.Reserve(values + (h->type == AMLIKE_MX8 ? (size_t)groups * rows : 0));
  if (rc == AMLIKE_OK && residual) rc = h->ws_r.Reserve(orow * rows);
  if (rc == AMLIKE_OK) rc = h->ws_out.Reserve(orow * rows);
  if (rc != AMLIKE_OK) return rc;
  AMLIKE_HIP(hipMemcpy2DAsync(h->ws_x.ptr, xrow, x, (size_t)ld * sizeof(float), xrow, rows, hipMemcpyHostToDevice, h->stream));
  if (residual)
    AMLIKE_HIP(hipMemcpy2DAsync(h->ws_r.ptr, orow, residual, (size_t)ldr * sizeof(float), orow, rows, hipMemcpyHostToDevice,
                                h->stream));
  const amlike_matrix_t mx = {h->ws_x.ptr, nullptr, h->k, 0, AMLIKE_F32},
                        mq = {h->ws_q.ptr, h->type == AMLIKE_MX8 ? static_cast<char *>(h->ws_q.ptr) + values : nullptr,
                              (int64_t)ldq, groups, h->type},
                        mr = {h->ws_r.ptr, nullptr, h->n, 0, AMLIKE_F32}, mo = {h->ws_out.ptr, nullptr, h->n, 0, AMLIKE_F32};
  rc = LaunchConvert(mx, rows, h->k, mq, h->stream);
  if (rc == AMLIKE_OK) rc = amlike_linear_apply_dev(h, &mq, rows, activation, residual ? &mr : nullptr, &mo, h->stream);
  if (rc != AMLIKE_OK) {
    (void)hipStreamSynchronize(h->stream);  // the copies above read the caller's arrays
    return rc;
  }
  return CopyMatrixToHost(out, (size_t)ldo, static_cast<const float *>(h->ws_out.ptr), rows, h->n, h->stream);
}

}  // extern "C"
