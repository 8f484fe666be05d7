// Distillation from a teacher's top logits (include/qnn.h: qnn_topk_distill_fwd, qnn_topk_distill_bwd).
//   p = softmax(t / T) over a row's entries that are there, q = softmax(s / T) over the vocabulary
//   row_loss = T^2 sum_e p_e (log p_e - log q_{i_e});  ds_j = g T (q_j - sum over i_e == j of p_e)
// stats, four floats a row: the largest student logit, 1 / sum of e^((s - largest) / T), the largest
// teacher logit, 1 / the teacher's sum (0: the row is not counted); then the number of counted rows.
// A row whose statistics are not numbers (an index past the vocabulary, all of its logits -inf, a
// NaN) carries a NaN in the second, which makes its whole gradient NaN.
#include "float_common.h"

namespace qnn {
namespace {
using namespace fl;

constexpr int NT = 256;
constexpr int MAX_TOP = 1024;

__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = wave_sum_f(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = sh[0];
  for (int w = 1; w < NT / 64; ++w) r += sh[w];
  return r;
}

__device__ __forceinline__ float block_max(float v, float* sh) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = sh[0];
  for (int w = 1; w < NT / 64; ++w) r = fmaxf(r, sh[w]);
  return r;
}

struct Entries {
  const void* t;
  int64_t ldt;
  const void* index;
  int64_t ldi;
  int top, tdtype, index_bytes;
  __device__ float logit(int64_t r, int e) const {
    const int64_t at = r * ldt + e;
    return tdtype == QNN_F32 ? ((const float*)t)[at]
                             : tdtype == QNN_BF16 ? (float)((const bf16*)t)[at] : (float)((const f16*)t)[at];
  }
  __device__ int64_t klass(int64_t r, int e) const {
    const int64_t at = r * ldi + e;
    return index_bytes == 8 ? ((const int64_t*)index)[at] : (int64_t)((const int32_t*)index)[at];
  }
};

// one block per row
template <class T>
__global__ __launch_bounds__(NT) void distill_rows_kernel(const T* s, int64_t lds, Entries en, int64_t vocab,
                                                          float temp, float* row_loss, float* stats) {
  __shared__ float sh[NT / 64];
  const int64_t r = blockIdx.x;
  const T* sr = s + r * lds;
  const float it = 1.0f / temp;
  float m = -INFINITY;
  for (int64_t c = threadIdx.x; c < vocab; c += NT) m = fmaxf(m, (float)sr[c]);
  m = block_max(m, sh);
  float sum = 0.0f;
  for (int64_t c = threadIdx.x; c < vocab; c += NT) sum += exp_f(((float)sr[c] - m) * it);
  sum = block_sum(sum, sh);
  float tm = -INFINITY, bad = 0.0f;
  for (int e = threadIdx.x; e < en.top; e += NT) {
    const int64_t i = en.klass(r, e);
    if (i >= 0) tm = fmaxf(tm, en.logit(r, e));
    if (i >= vocab) bad = 1.0f;
  }
  tm = block_max(tm, sh);
  bad = block_max(bad, sh);
  const bool counted = tm > -INFINITY || bad > 0.0f;
  float ts = 0.0f;
  if (tm > -INFINITY)
    for (int e = threadIdx.x; e < en.top; e += NT)
      if (en.klass(r, e) >= 0) ts += exp_f((en.logit(r, e) - tm) * it);
  ts = block_sum(ts, sh);
  float l = 0.0f;
  if (tm > -INFINITY && bad == 0.0f)
    for (int e = threadIdx.x; e < en.top; e += NT) {
      const int64_t i = en.klass(r, e);
      if (i < 0) continue;
      const float u = (en.logit(r, e) - tm) * it, p = exp_f(u) / ts;
      if (p != 0.0f) l += p * ((u - logf(ts)) - (((float)sr[i] - m) * it - logf(sum)));
    }
  l = block_sum(l, sh);
  if (threadIdx.x == 0) {
    if (bad > 0.0f) l = sum = __builtin_nanf("");
    row_loss[r] = counted ? temp * temp * l : 0.0f;
    stats[4 * r] = m;
    stats[4 * r + 1] = 1.0f / sum;
    stats[4 * r + 2] = tm;
    stats[4 * r + 3] = counted ? (bad > 0.0f ? 1.0f : 1.0f / ts) : 0.0f;
  }
}

__global__ __launch_bounds__(NT) void distill_join_kernel(const float* row_loss, float* stats, float* loss,
                                                          int64_t rows, int mean) {
  __shared__ double sh[NT / 64], shn[NT / 64];
  double a = 0.0, n = 0.0;
  for (int64_t r = threadIdx.x; r < rows; r += NT) {
    a += (double)row_loss[r];
    n += stats[4 * r + 3] != 0.0f ? 1.0 : 0.0;
  }
  a = wave_sum(a);
  n = wave_sum(n);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a, shn[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < NT / 64; ++w) a += sh[w], n += shn[w];
    stats[4 * rows] = (float)n;
    if (loss) loss[0] = (float)(mean ? a / (n > 0.0 ? n : 1.0) : a);
  }
}

template <class T>
__global__ __launch_bounds__(NT) void distill_grad_kernel(const T* s, int64_t lds, Entries en, const float* stats,
                                                          const float* grad, int grad_rows, T* ds, int64_t rows,
                                                          int64_t vocab, float temp, int mean) {
  __shared__ int64_t cls[MAX_TOP];
  const int64_t r = blockIdx.x;
  const T* sr = s + r * lds;
  T* dr = ds + r * vocab;
  const float it = 1.0f / temp;
  const float m = stats[4 * r], inv = stats[4 * r + 1], tm = stats[4 * r + 2], ti = stats[4 * r + 3];
  float g = temp * (grad_rows ? grad[r] : grad[0]);
  if (mean) g /= fmaxf(stats[4 * rows], 1.0f);
  for (int e = threadIdx.x; e < en.top; e += NT) cls[e] = en.klass(r, e);
  for (int64_t c = threadIdx.x; c < vocab; c += NT)
    dr[c] = ti == 0.0f ? (T)0.0f : (T)(g * (exp_f(((float)sr[c] - m) * it) * inv));
  __syncthreads();  // the entries' classes are written again, by the first entry of each class
  if (ti == 0.0f) return;
  for (int e = threadIdx.x; e < en.top; e += NT) {
    const int64_t i = cls[e];
    if (i < 0 || i >= vocab) continue;
    bool first = true;
    for (int f = 0; f < e; ++f) first = first && cls[f] != i;
    if (!first) continue;
    float p = 0.0f;
    for (int f = e; f < en.top; ++f)
      if (cls[f] == i) p += exp_f((en.logit(r, f) - tm) * it) * ti;
    dr[i] = (T)(g * (exp_f(((float)sr[i] - m) * it) * inv - p));
  }
}

int check(const void* s, int64_t lds, const void* t, int64_t ldt, const void* index, int64_t ldi, int64_t rows,
          int64_t vocab, int64_t top, float temp, int tdtype, int index_bytes, const float* stats) {
  QNN_REQUIRE(rows >= 0 && rows < (1LL << 31), "rows: 0 to 2^31 - 1");
  QNN_REQUIRE(vocab >= 1 && vocab < (1LL << 31), "vocab: 1 to 2^31 - 1");
  QNN_REQUIRE(top >= 1 && top <= MAX_TOP, "top: 1 to 1024");
  QNN_REQUIRE(lds >= vocab && ldt >= top && ldi >= top, "a row stride is shorter than the row");
  QNN_REQUIRE(temp > 0.0f && temp < INFINITY, "temp: positive and finite");
  QNN_REQUIRE(tdtype == QNN_F32 || tdtype == QNN_BF16 || tdtype == QNN_F16, "tdtype: QNN_F32, QNN_BF16 or QNN_F16");
  QNN_REQUIRE(index_bytes == 4 || index_bytes == 8, "index_bytes: 4 or 8");
  QNN_REQUIRE(stats && (rows == 0 || (s && t && index)), "null pointer");
  return QNN_OK;
}

}  // namespace
}  // namespace qnn

using namespace qnn;
using namespace qnn::fl;

extern "C" {

int qnn_topk_distill_fwd_work(int64_t rows, int64_t vocab, int dtype, int64_t* bytes) {
  QNN_REQUIRE(rows >= 0 && vocab >= 1 && bytes, "bad shape or null pointer");
  *bytes = 0;
  return QNN_OK;
}

int qnn_topk_distill_fwd(const void* s, int64_t lds, const void* t, int64_t ldt, const void* index, int64_t ldi,
                         int64_t rows, int64_t vocab, int64_t top, float temp, int mean, int dtype, int tdtype,
                         int index_bytes, float* row_loss, float* stats, float* loss, void* work,
                         int64_t work_bytes, qnn_stream_t stream) {
  if (int rc = check(s, lds, t, ldt, index, ldi, rows, vocab, top, temp, tdtype, index_bytes, stats)) return rc;
  QNN_REQUIRE(rows == 0 || row_loss, "null pointer");
  const Entries en = {t, ldt, index, ldi, (int)top, tdtype, index_bytes};
  hipStream_t st = (hipStream_t)stream;
  const int rc = with_type(dtype, [&](auto z) {
    using T = decltype(z);
    if (rows > 0)
      hipLaunchKernelGGL((distill_rows_kernel<T>), dim3((unsigned)rows), dim3(NT), 0, st, (const T*)s, lds, en, vocab,
                         temp, row_loss, stats);
    QNN_LAUNCH_CHECK("qnn_topk_distill_fwd");
    return (int)QNN_OK;
  });
  if (rc) return rc;
  hipLaunchKernelGGL(distill_join_kernel, dim3(1), dim3(NT), 0, st, row_loss, stats, loss, rows, mean);
  QNN_LAUNCH_CHECK("qnn_topk_distill_fwd");
  return QNN_OK;
}

int qnn_topk_distill_bwd(const void* s, int64_t lds, const void* t, int64_t ldt, const void* index, int64_t ldi,
                         const float* stats, const float* grad, int grad_rows, void* ds, int64_t rows,
                         int64_t vocab, int64_t top, float temp, int mean, int dtype, int tdtype, int index_bytes,
                         qnn_stream_t stream) {
  if (int rc = check(s, lds, t, ldt, index, ldi, rows, vocab, top, temp, tdtype, index_bytes, stats)) return rc;
  if (rows == 0) return QNN_OK;
  QNN_REQUIRE(grad && ds, "null pointer");
  const Entries en = {t, ldt, index, ldi, (int)top, tdtype, index_bytes};
  return with_type(dtype, [&](auto z) {
    using T = decltype(z);
    hipLaunchKernelGGL((distill_grad_kernel<T>), dim3((unsigned)rows), dim3(NT), 0, (hipStream_t)stream, (const T*)s,
                       lds, en, stats, grad, grad_rows, (T*)ds, rows, vocab, temp, mean);
    QNN_LAUNCH_CHECK("qnn_topk_distill_bwd");
    return (int)QNN_OK;
  });
}

}  // extern "C"
