// Float matrix product with bias, residual and activation in its epilogue, forward and backward
// (include/qnn.h: qnn_linear_act_fwd, qnn_linear_act_bwd).
//   z = x w^T + bias + res, y = act(z);  dz = dy act'(z), dx = dz w, dw = dz^T x, db = sum of dz's rows
#include "float_common.h"

namespace qnn {
namespace {
using namespace fl;

// What is done to 8 neighbouring columns of z before they are written.
struct Epilogue {
  const void* bias;
  const void* res;
  int64_t ldr;
  void* y;
  void* slope;
  int act;
};

template <class T>
__device__ __forceinline__ void finish8(float (&z)[8], const Epilogue& e, int64_t row, int64_t col, int64_t n) {
  const int64_t left = n - col;
  if (e.bias) {
    float b[8];
    load_n<T, 8>(b, (const T*)e.bias + col, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] += b[i];
  }
  if (e.res) {
    float b[8];
    load_n<T, 8>(b, (const T*)e.res + row * e.ldr + col, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] += b[i];
  }
  if (e.act == QNN_ACT_RELU) {
    unsigned mask = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool on = !(z[i] <= 0.0f);
      mask |= (unsigned)on << i;
      z[i] = on ? z[i] : 0.0f;
    }
    if (e.slope) ((uint8_t*)e.slope)[row * ((n + 7) / 8) + col / 8] = (uint8_t)mask;
  } else if (e.act == QNN_ACT_GELU) {
    float d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) gelu_f(z[i], z[i], d[i]);
    if (e.slope) {
      if constexpr (sizeof(T) == 4) {
        store_n<float, 8>((float*)e.slope + row * n + col, d, left);
      } else {
        Vec<int16_t, 8> q;
#pragma unroll
        for (int i = 0; i < 8; ++i) q.v[i] = slope_pack(d[i]);
        store_group((int16_t*)e.slope + row * n + col, q, left);
      }
    }
  }
  store_n<T, 8>((T*)e.y + row * n + col, z, left);
}

// c[i][j] = sum over k of a(i, k) b(j, k), a and b by element strides
template <class T>
__global__ __launch_bounds__(256) void matmul_kernel(const T* a, int64_t ai, int64_t ak, const T* b, int64_t bj,
                                                     int64_t bk, int64_t m, int64_t n, int64_t k, Epilogue e) {
  constexpr int BM = 32, BN = 64, BK = 32;
  __shared__ float sa[BM][BK + 1], sb[BN][BK + 1];
  const int64_t tn = (n + BN - 1) / BN, i0 = blockIdx.x / tn * BM, j0 = blockIdx.x % tn * BN;
  const int t = threadIdx.x, ti = t / 8, tj = t % 8 * 8;
  float acc[8] = {};
  for (int64_t k0 = 0; k0 < k; k0 += BK) {
    __syncthreads();
    for (int u = t; u < BM * BK; u += 256) {
      const int i = ak == 1 ? u / BK : u % BM, kk = ak == 1 ? u % BK : u / BM;
      sa[i][kk] = i0 + i < m && k0 + kk < k ? (float)a[(i0 + i) * ai + (k0 + kk) * ak] : 0.0f;
    }
    for (int u = t; u < BN * BK; u += 256) {
      const int j = bk == 1 ? u / BK : u % BN, kk = bk == 1 ? u % BK : u / BN;
      sb[j][kk] = j0 + j < n && k0 + kk < k ? (float)b[(j0 + j) * bj + (k0 + kk) * bk] : 0.0f;
    }
    __syncthreads();
    for (int kk = 0; kk < BK; ++kk) {
      const float v = sa[ti][kk];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = fmaf(v, sb[tj + j][kk], acc[j]);
    }
  }
  if (i0 + ti < m && j0 + tj < n) finish8<T>(acc, e, i0 + ti, j0 + tj, n);
}

template <class T>
int matmul(const void* a, int64_t ai, int64_t ak, const void* b, int64_t bj, int64_t bk, int64_t m, int64_t n,
           int64_t k, const Epilogue& e, hipStream_t s) {
  hipLaunchKernelGGL((matmul_kernel<T>), dim3((unsigned)(cdiv(m, 32) * cdiv(n, 64))), dim3(256), 0, s, (const T*)a, ai,
                     ak, (const T*)b, bj, bk, m, n, k, e);
  QNN_LAUNCH_CHECK("matmul_kernel");
  return QNN_OK;
}

// dz = dy act'(z)
template <class T>
__global__ __launch_bounds__(256) void linear_dz_kernel(const T* dy, int64_t ldy, const void* slope, T* dz, int64_t m,
                                                        int64_t n, int act) {
  const int64_t chunks = (n + 255) / 256, row = blockIdx.x / chunks;
  const int64_t c = blockIdx.x % chunks * 256 + threadIdx.x;
  if (c >= n) return;
  const float g = (float)dy[row * ldy + c];
  float v;
  if (act == QNN_ACT_RELU)
    v = ((const uint8_t*)slope)[row * ((n + 7) / 8) + c / 8] >> (c & 7) & 1 ? g : 0.0f;
  else if constexpr (sizeof(T) == 4)
    v = g * ((const float*)slope)[row * n + c];
  else
    v = g * slope_unpack(((const int16_t*)slope)[row * n + c]);
  dz[row * n + c] = (T)v;
}

template <class T>
__global__ __launch_bounds__(256) void linear_db_kernel(const T* dz, int64_t ld, T* db, int64_t m, int64_t n) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  float a = 0.0f;
  for (int64_t r = 0; r < m; ++r) a += (float)dz[r * ld + c];
  db[c] = (T)a;
}

int check(int64_t m, int64_t n, int64_t k) {
  QNN_REQUIRE(m >= 0 && m < (1LL << 31), "m: 0 to 2^31 - 1");
  QNN_REQUIRE(n >= 1 && n < (1LL << 31), "n: 1 to 2^31 - 1");
  QNN_REQUIRE(k >= 1 && k < (1LL << 31), "k: 1 to 2^31 - 1");
  return QNN_OK;
}

}  // namespace
}  // namespace qnn

using namespace qnn;
using namespace qnn::fl;

extern "C" {

int qnn_linear_act_fwd_work(int64_t m, int64_t n, int64_t k, int dtype, int64_t* bytes) {
  if (int rc = check(m, n, k)) return rc;
  QNN_REQUIRE(bytes, "null pointer");
  *bytes = 0;
  return QNN_OK;
}

int qnn_linear_act_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res,
                       int64_t ldr, void* y, void* slope, int64_t m, int64_t n, int64_t k, int dtype, int act,
                       void* work, int64_t work_bytes, qnn_stream_t stream) {
  if (int rc = check(m, n, k)) return rc;
  QNN_REQUIRE(act >= QNN_ACT_NONE && act <= QNN_ACT_GELU, "act: QNN_ACT_NONE, QNN_ACT_RELU or QNN_ACT_GELU");
  QNN_REQUIRE(ldx >= k && ldw >= k && (!res || ldr >= n), "a row stride is shorter than the row");
  if (m == 0) return QNN_OK;
  QNN_REQUIRE(x && w && y, "null pointer");
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const Epilogue e = {bias, res, ldr, y, slope, act};
    return matmul<T>(x, ldx, 1, w, ldw, 1, m, n, k, e, (hipStream_t)stream);
  });
}

int qnn_linear_act_bwd_work(int64_t m, int64_t n, int64_t k, int dtype, int64_t* bytes) {
  if (int rc = check(m, n, k)) return rc;
  QNN_REQUIRE(bytes, "null pointer");
  *bytes = 0;
  return QNN_OK;
}

int qnn_linear_act_bwd(const void* dy, int64_t ldy, const void* slope, const void* x, int64_t ldx, const void* w,
                       int64_t ldw, void* dz, void* dx, void* dw, void* db, int64_t m, int64_t n, int64_t k,
                       int dtype, int act, void* work, int64_t work_bytes, qnn_stream_t stream) {
  if (int rc = check(m, n, k)) return rc;
  QNN_REQUIRE(act >= QNN_ACT_NONE && act <= QNN_ACT_GELU, "act: QNN_ACT_NONE, QNN_ACT_RELU or QNN_ACT_GELU");
  QNN_REQUIRE(ldy >= n && (!dw || ldx >= k) && (!dx || ldw >= k), "a row stride is shorter than the row");
  QNN_REQUIRE(m == 0 || (dy && (!dx || w) && (!dw || x)), "null pointer");
  QNN_REQUIRE(m == 0 || act == QNN_ACT_NONE || (slope && dz), "an activation's gradient needs slope and dz");
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipStream_t s = (hipStream_t)stream;
    const T* g = (const T*)dy;
    int64_t ldg = ldy;
    if (act != QNN_ACT_NONE && m > 0) {
      hipLaunchKernelGGL((linear_dz_kernel<T>), dim3((unsigned)(cdiv(n, 256) * m)), dim3(256), 0, s, g, ldy,
                         slope, (T*)dz, m, n, act);
      QNN_LAUNCH_CHECK("linear_dz_kernel");
      g = (const T*)dz;
      ldg = n;
    }
    const Epilogue none = {nullptr, nullptr, 0, dx, nullptr, QNN_ACT_NONE};
    if (dx && m > 0)
      if (int rc = matmul<T>(g, ldg, 1, w, 1, ldw, m, k, n, none, s)) return rc;
    Epilogue to_dw = none;
    to_dw.y = dw;
    if (dw)
      if (int rc = matmul<T>(g, 1, ldg, x, 1, ldx, n, k, m, to_dw, s)) return rc;
    if (db) {
      hipLaunchKernelGGL((linear_db_kernel<T>), dim3((unsigned)cdiv(n, 256)), dim3(256), 0, s, g, ldg, (T*)db, m, n);
      QNN_LAUNCH_CHECK("linear_db_kernel");
    }
    return (int)QNN_OK;
  });
}

}  // extern "C"
