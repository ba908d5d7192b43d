// amlike_linear_*: the host side of the matrix product with bias, activation and residual, and the
// packing of its weights.  The kernels: linear_kernels.h.
#include <mutex>
#include <new>

#include "linear_kernels.h"

namespace amlike {

constexpr int kLinearMaxDim = 1 << 20;  // either dimension of a layer

extern template int LaunchLinear<AMLIKE_BF16>(const LinearArgs &, hipStream_t);
extern template int LaunchLinear<AMLIKE_F16>(const LinearArgs &, hipStream_t);
extern template int LaunchLinear<AMLIKE_MX8>(const LinearArgs &, hipStream_t);
extern template int LaunchLinear<kMx8Exact>(const LinearArgs &, hipStream_t);

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
  h->n_pad = (output_dim + 63) / 64 * 64;
  h->k_tiles = (int)(((int64_t)input_dim * TypeBytes(type) + kTileBytes - 1) / kTileBytes);
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
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (h->type == AMLIKE_BF16) return LaunchLinear<AMLIKE_BF16>(a, st);
  if (h->type == AMLIKE_F16) return LaunchLinear<AMLIKE_F16>(a, st);
  if (out->type == AMLIKE_F32) return LaunchLinear<kMx8Exact>(a, st);
  return LaunchLinear<AMLIKE_MX8>(a, st);
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
