// Layer norm, forward and backward (include/qnn.h: qnn_layer_norm_fwd, qnn_layer_norm_bwd).
//   mean = sum(x) / d, var = sum((x - mean)^2) / d, rstd = 1 / sqrt(var + eps), xh = (x - mean) rstd
//   y = xh w + b;  g = dy w;  dx = rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over rows of dy xh;  db = sum over rows of dy
#include "float_common.h"

namespace qnn {
namespace {
using namespace fl;

constexpr int NT = 256;

__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = wave_sum_f(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = sh[0];
  for (int w = 1; w < NT / 64; ++w) r += sh[w];
  return r;
}

// one block per row
template <class T, class W>
__global__ __launch_bounds__(NT) void layer_norm_fwd_kernel(const T* x, int64_t ldx, const W* w, const W* b, T* y,
                                                            float* mean, float* rstd, int64_t dim, float eps) {
  __shared__ float sh[NT / 64];
  const int64_t r = blockIdx.x;
  const T* xr = x + r * ldx;
  T* yr = y + r * dim;
  float s = 0.0f;
  for (int64_t c = threadIdx.x; c < dim; c += NT) s += (float)xr[c];
  const float mu = block_sum(s, sh) / (float)dim;
  float q = 0.0f;
  for (int64_t c = threadIdx.x; c < dim; c += NT) {
    const float d = (float)xr[c] - mu;
    q = fmaf(d, d, q);
  }
  const float rs = 1.0f / sqrtf(block_sum(q, sh) / (float)dim + eps);
  for (int64_t c = threadIdx.x; c < dim; c += NT) {
    const float xh = ((float)xr[c] - mu) * rs;
    yr[c] = (T)fmaf(xh, w ? (float)w[c] : 1.0f, b ? (float)b[c] : 0.0f);
  }
  if (threadIdx.x == 0) {
    if (mean) mean[r] = mu;
    if (rstd) rstd[r] = rs;
  }
}

template <class T, class W>
__global__ __launch_bounds__(NT) void layer_norm_dx_kernel(const T* dy, int64_t ldy, const T* x, int64_t ldx,
                                                           const W* w, const float* mean, const float* rstd, T* dx,
                                                           int64_t dim) {
  __shared__ float sh[NT / 64];
  const int64_t r = blockIdx.x;
  const float mu = mean[r], rs = rstd[r];
  float sg = 0.0f, sx = 0.0f;
  for (int64_t c = threadIdx.x; c < dim; c += NT) {
    const float g = (float)dy[r * ldy + c] * (w ? (float)w[c] : 1.0f);
    sg += g;
    sx = fmaf(g, ((float)x[r * ldx + c] - mu) * rs, sx);
  }
  sg = block_sum(sg, sh) / (float)dim;
  sx = block_sum(sx, sh) / (float)dim;
  for (int64_t c = threadIdx.x; c < dim; c += NT) {
    const float g = (float)dy[r * ldy + c] * (w ? (float)w[c] : 1.0f);
    const float xh = ((float)x[r * ldx + c] - mu) * rs;
    dx[r * dim + c] = (T)(rs * (g - sg - xh * sx));
  }
}

// one thread per column
template <class T, class W>
__global__ __launch_bounds__(NT) void layer_norm_dw_kernel(const T* dy, int64_t ldy, const T* x, int64_t ldx,
                                                           const float* mean, const float* rstd, W* dw, W* db,
                                                           int64_t rows, int64_t dim) {
  const int64_t c = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (c >= dim) return;
  float a = 0.0f, s = 0.0f;
  for (int64_t r = 0; r < rows; ++r) {
    const float g = (float)dy[r * ldy + c];
    a = fmaf(g, ((float)x[r * ldx + c] - mean[r]) * rstd[r], a);
    s += g;
  }
  if (dw) dw[c] = (W)a;
  if (db) db[c] = (W)s;
}

template <class F>
int with_types(int dtype, int wdtype, F&& f) {
  if (wdtype != dtype && wdtype != QNN_F32) return arg_error("wdtype: the rows' type or QNN_F32");
  return with_type(dtype, [&](auto t) {
    if (wdtype == QNN_F32) return f(t, 0.0f);
    return f(t, t);
  });
}

int check(int64_t rows, int64_t dim, int64_t ld) {
  QNN_REQUIRE(rows >= 0 && rows < (1LL << 31), "rows: 0 to 2^31 - 1");
  QNN_REQUIRE(dim >= 1 && dim < (1LL << 31), "dim: 1 to 2^31 - 1");
  QNN_REQUIRE(ld >= dim, "a row stride is shorter than the row");
  return QNN_OK;
}

}  // namespace
}  // namespace qnn

using namespace qnn;
using namespace qnn::fl;

extern "C" {

int qnn_layer_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, void* y, float* mean, float* rstd,
                       int64_t rows, int64_t dim, float eps, int dtype, int wdtype, qnn_stream_t stream) {
  if (int rc = check(rows, dim, ldx)) return rc;
  QNN_REQUIRE(eps >= 0.0f, "eps: not negative");
  if (rows == 0) return QNN_OK;
  QNN_REQUIRE(x && y, "null pointer");
  return with_types(dtype, wdtype, [&](auto t, auto tw) {
    using T = decltype(t);
    using W = decltype(tw);
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, W>), dim3((unsigned)rows), dim3(NT), 0, (hipStream_t)stream,
                       (const T*)x, ldx, (const W*)w, (const W*)b, (T*)y, mean, rstd, dim, eps);
    QNN_LAUNCH_CHECK("qnn_layer_norm_fwd");
    return (int)QNN_OK;
  });
}

int qnn_layer_norm_bwd_work(int64_t rows, int64_t dim, int dtype, int64_t* bytes) {
  if (int rc = check(rows, dim, dim)) return rc;
  QNN_REQUIRE(bytes, "null pointer");
  *bytes = 0;
  return QNN_OK;
}

int qnn_layer_norm_bwd(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* w, const float* mean,
                       const float* rstd, void* dx, void* dw, void* db, int64_t rows, int64_t dim, int dtype,
                       int wdtype, void* work, int64_t work_bytes, qnn_stream_t stream) {
  if (int rc = check(rows, dim, ldx)) return rc;
  if (int rc = check(rows, dim, ldy)) return rc;
  QNN_REQUIRE(rows == 0 || (dy && x && mean && rstd), "null pointer");
  return with_types(dtype, wdtype, [&](auto t, auto tw) {
    using T = decltype(t);
    using W = decltype(tw);
    hipStream_t s = (hipStream_t)stream;
    if (dx && rows > 0)
      hipLaunchKernelGGL((layer_norm_dx_kernel<T, W>), dim3((unsigned)rows), dim3(NT), 0, s, (const T*)dy, ldy,
                         (const T*)x, ldx, (const W*)w, mean, rstd, (T*)dx, dim);
    QNN_LAUNCH_CHECK("qnn_layer_norm_bwd");
    if (dw || db)
      hipLaunchKernelGGL((layer_norm_dw_kernel<T, W>), dim3((unsigned)cdiv(dim, NT)), dim3(NT), 0, s, (const T*)dy,
                         ldy, (const T*)x, ldx, mean, rstd, (W*)dw, (W*)db, rows, dim);
    QNN_LAUNCH_CHECK("qnn_layer_norm_bwd");
    return (int)QNN_OK;
  });
}

}  // extern "C"
