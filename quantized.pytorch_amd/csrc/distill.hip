// Distillation from a teacher's top logits (include/qnn.h: qnn_topk_distill_fwd, qnn_topk_distill_bwd).
//   p = softmax(t / T) over a row's entries that are there, q = softmax(s / T) over the vocabulary
//   row_loss = T^2 sum_e p_e (log p_e - log q_{i_e});  ds_j = g T (q_j - sum over i_e == j of p_e)
//
// Bound by HBM: forward reads the logits once (largest logit and sum of exponentials together, the sum
// rescaled when the maximum grows), backward reads them and writes their gradient.  A wave takes a row
// of up to 16 KiB, a workgroup a longer one; where there are few long rows the forward pass cuts them
// into pieces whose (maximum, sum) pairs a second launch joins.  The gradient is dense but for the
// teacher's classes: a workgroup writes its piece of the row as if there were none, and then the
// classes that lie in it again, the first entry of a class with the sum of all of them.
// 4096 x 131072 bf16, 64 entries a row: forward 221 us (4.9 TB/s), gradient 390 (5.5 TB/s).
//
// stats, four floats a row: the largest student logit, 1 / sum of e^((s - largest) / T), the largest
// teacher logit, 1 / the teacher's sum (0: the row is not counted); then the number of counted rows.
// A row whose statistics are not numbers (an index past the vocabulary, all of its logits -inf, a
// NaN, the teacher's too) carries a NaN in the second, which makes its whole gradient NaN.
#include "float_common.h"

namespace qnn {
namespace {
using namespace fl;

constexpr int NT = 256;
constexpr int MAX_TOP = 1024;
constexpr int WIDE = 512;        // lanes for a row or a piece that is longer than a wave's
constexpr int WAVE_BYTES = 16384;  // the longest row that a wave takes
constexpr int MAX_SPLITS = 64;   // pieces of a row: a lane each when they are joined
constexpr float LOG2E = 1.44269504088896341f;

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
  Entries from(int64_t r) const {  // row r on
    Entries e = *this;
    e.t = (const char*)t + r * ldt * type_bytes(tdtype);
    e.index = (const char*)index + r * ldi * index_bytes;
    return e;
  }
};

// A running (maximum, sum of e^((x - maximum) / T)); k = log2(e) / T.  While the maximum is -inf the
// sum is taken from 0 instead, so that logits of -inf add 0 and not NaN.
struct Run {
  float m, s;
};
__device__ __forceinline__ float from(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ Run joined(Run a, Run b, float k) {
  const float m = fmaxf(a.m, b.m), f = from(m);
  return {m, a.s * __builtin_amdgcn_exp2f((a.m - f) * k) + b.s * __builtin_amdgcn_exp2f((b.m - f) * k)};
}

// This lane's run over s[lo, hi): groups (lo + lane GROUP), L GROUP apart, U of them in flight.  A sum of more than
// CHAIN terms is the sum of such sums.
template <class T, int L>
__device__ __forceinline__ Run run_over(const T* s, int64_t lo, int64_t hi, int lane, float k) {
  constexpr int GR = GROUP<T>, U = 4, CHAIN = 512;
  Run all = {-INFINITY, 0.0f};
  for (int64_t end; lo < hi; lo = end) {
    end = hi - lo > (int64_t)CHAIN * L ? lo + (int64_t)CHAIN * L : hi;
    Run a = {-INFINITY, 0.0f};
    auto add = [&](const float* v, int n) {
      float m = a.m;
#pragma unroll
      for (int i = 0; i < n; ++i) m = fmaxf(m, v[i]);
      const float f = from(m);
      float t = a.s * __builtin_amdgcn_exp2f((a.m - f) * k);
#pragma unroll
      for (int i = 0; i < n; ++i) t += __builtin_amdgcn_exp2f((v[i] - f) * k);
      a = {m, t};
    };
    int64_t c = lo + lane * GR;
    for (; c + (U - 1) * L * GR + GR <= end; c += U * L * GR) {
      Vec<T, GR> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = load_group(s + c + u * L * GR, GR);
#pragma unroll
      for (int u = 0; u < U; u += 2) {
        float v[2 * GR];
#pragma unroll
        for (int i = 0; i < GR; ++i) v[i] = (float)raw[u].v[i], v[GR + i] = (float)raw[u + 1].v[i];
        add(v, 2 * GR);
      }
    }
    for (; c < end; c += L * GR) {
      const Vec<T, GR> raw = load_group(s + c, end - c);
      float v[GR];
#pragma unroll
      for (int i = 0; i < GR; ++i) v[i] = c + i < end ? (float)raw.v[i] : -INFINITY;
      add(v, GR);
    }
    all = joined(all, a, k);
  }
  return all;
}

// ---- reductions over the L lanes of a row (L 64, or a workgroup)
template <int L, class V, class Op>
__device__ __forceinline__ V over_lanes(V v, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  if constexpr (L > 64) {
    __shared__ V sh[L / 64];
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x / 64] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < L / 64; ++w) v = op(v, sh[w]);
  }
  return v;
}
template <int L>
__device__ __forceinline__ Run over_lanes_run(Run a, float k) {
  const float m = over_lanes<L>(a.m, [](float x, float y) { return fmaxf(x, y); });
  const float s = a.s * __builtin_amdgcn_exp2f((a.m - from(m)) * k);
  return {m, over_lanes<L>(s, [](float x, float y) { return x + y; })};
}

// The row's statistics and loss from its lanes' runs.
template <class T, int L>
__device__ __forceinline__ void finish_row(const T* sr, Run a, const Entries& en, int64_t r, int64_t vocab, float temp,
                                           int lane, float* row_loss, float* stats) {
  auto add = [](float x, float y) { return x + y; };
  auto most = [](float x, float y) { return fmaxf(x, y); };
  const float k = LOG2E / temp, it = 1.0f / temp;
  a = over_lanes_run<L>(a, k);
  if (a.m == -INFINITY) a.s = __builtin_nanf("");  // all of the row's logits are -inf
  float tm = -INFINITY, bad = 0.0f;
  for (int e = lane; e < en.top; e += L) {
    const int64_t i = en.klass(r, e);
    const float t = i >= 0 ? en.logit(r, e) : -INFINITY;
    tm = fmaxf(tm, t);
    if (i >= vocab || t != t) bad = 1.0f;
  }
  tm = over_lanes<L>(tm, most);
  bad = over_lanes<L>(bad, most);
  const bool some = tm > -INFINITY;
  // sum of the teacher's exponentials, and of e_e (u_e - log q_e): the loss is their quotient less log
  // of the sum, since the p_e add up to 1
  float ts = 0.0f;
  if (some)
    for (int e = lane; e < en.top; e += L)
      if (en.klass(r, e) >= 0) ts += __builtin_amdgcn_exp2f((en.logit(r, e) - tm) * k);
  ts = over_lanes<L>(ts, add);
  const float lts = logf(ts), ls = logf(a.s);
  float l = 0.0f;
  if (some && bad == 0.0f)
    for (int e = lane; e < en.top; e += L) {
      const int64_t i = en.klass(r, e);
      if (i < 0) continue;
      const float u = (en.logit(r, e) - tm) * it, p = __builtin_amdgcn_exp2f(u * LOG2E) / ts;
      if (p != 0.0f) l += p * ((u - lts) - (((float)sr[i] - a.m) * it - ls));
    }
  l = over_lanes<L>(l, add);
  if (lane == 0) {
    if (bad > 0.0f) l = a.s = __builtin_nanf("");
    const bool counted = some || bad > 0.0f;
    row_loss[r] = counted ? temp * temp * l : 0.0f;
    float4 st = {a.m, 1.0f / a.s, tm, counted ? (bad > 0.0f ? 1.0f : 1.0f / ts) : 0.0f};
    *reinterpret_cast<float4*>(stats + 4 * r) = st;
  }
}

// L lanes a row
template <class T, int L>
__global__ __launch_bounds__(L > NT ? L : NT) void distill_rows_kernel(const T* s, int64_t lds, Entries en, int64_t rows,
                                                                       int64_t vocab, float temp, float* row_loss,
                                                                       float* stats) {
  constexpr int ROWS = L > NT ? 1 : NT / L;
  const int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / L;
  if (r >= rows) return;  // a whole wave: L > 64 has a row for every workgroup
  const int lane = threadIdx.x % L;
  const Run a = run_over<T, L>(s + r * lds, 0, vocab, lane, LOG2E / temp);
  finish_row<T, L>(s + r * lds, a, en, r, vocab, temp, lane, row_loss, stats);
}

// piece (row, split) of long rows: its run into part[row][split]
template <class T>
__global__ __launch_bounds__(WIDE) void distill_part_kernel(const T* s, int64_t lds, int64_t vocab, float temp,
                                                            int splits, int64_t piece, Run* part) {
  const int64_t r = blockIdx.x / splits;
  const int64_t lo = blockIdx.x % splits * piece, hi = lo + piece < vocab ? lo + piece : vocab;
  const float k = LOG2E / temp;
  const Run a = over_lanes_run<WIDE>(run_over<T, WIDE>(s + r * lds, lo, hi, threadIdx.x, k), k);
  if (threadIdx.x == 0) part[(int64_t)blockIdx.x] = a;
}

// The rows' statistics from their pieces' runs, a wave a row.  ALL: the launch is one workgroup that has
// every row, and gives the loss too.
constexpr int ALL_ROWS = 16;
template <class T, bool ALL>
__global__ __launch_bounds__(ALL ? 64 * ALL_ROWS : NT) void distill_split_rows_kernel(
    const T* s, int64_t lds, Entries en, int64_t rows, int64_t vocab, float temp, int splits, const Run* part,
    float* row_loss, float* stats, float* loss, int mean) {
  const int64_t r = (int64_t)blockIdx.x * (NT / 64) + threadIdx.x / 64;
  if (r < rows) {
    const int lane = threadIdx.x % 64;
    const Run a = lane < splits ? part[r * splits + lane] : Run{-INFINITY, 0.0f};
    finish_row<T, 64>(s + r * lds, a, en, r, vocab, temp, lane, row_loss, stats);
  }
  if constexpr (ALL) {
    __syncthreads();
    if (threadIdx.x == 0) {
      double a = 0.0, n = 0.0;
      for (int k = 0; k < (int)rows; ++k) {
        a += (double)row_loss[k];
        n += stats[4 * k + 3] != 0.0f ? 1.0 : 0.0;
      }
      stats[4 * rows] = (float)n;
      if (loss) loss[0] = (float)(mean ? a / (n > 0.0 ? n : 1.0) : a);
    }
  }
}

// The loss from the rows' losses, one workgroup, eight of a thread's rows under way.
constexpr int JOIN = 1024;
__global__ __launch_bounds__(JOIN) void distill_join_kernel(const float* __restrict__ row_loss,
                                                            const float* __restrict__ row_stats,
                                                            float* __restrict__ count, float* __restrict__ loss,
                                                            int64_t rows, int mean) {
  __shared__ double sh[JOIN / 64], shn[JOIN / 64];
  double a = 0.0, n = 0.0;
  for (int64_t r0 = threadIdx.x; r0 < rows; r0 += 8 * JOIN) {
    float l[8], c[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t r = r0 + u * JOIN < rows ? r0 + u * JOIN : rows - 1;
      l[u] = row_loss[r];
      c[u] = row_stats[4 * r + 3];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (r0 + u * JOIN < rows) {
        a += (double)l[u];
        n += c[u] != 0.0f ? 1.0 : 0.0;
      }
  }
  a = wave_sum(a);
  n = wave_sum(n);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a, shn[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < JOIN / 64; ++w) a += sh[w], n += shn[w];
    count[0] = (float)n;
    if (loss) loss[0] = (float)(mean ? a / (n > 0.0 ? n : 1.0) : a);
  }
}

// The gradient of a row's piece [lo, lo + PIECE), L lanes.
template <class T, int L>
struct Grad {
  static constexpr int THREADS = L > NT ? L : NT, ROWS = THREADS / L;
  static constexpr int64_t PIECE = L > 64 ? (int64_t)L * 4 * GROUP<T> : WAVE_BYTES / (int)sizeof(T);
};

template <class T, int L>
__global__ __launch_bounds__((Grad<T, L>::THREADS)) void distill_grad_kernel(const T* s, int64_t lds, Entries en,
                                                                             const float* stats, const float* count,
                                                                             const float* grad, int grad_rows, T* ds,
                                                                             int64_t rows,
                                                                             int64_t vocab, int pieces, float temp,
                                                                             int mean) {
  constexpr int GR = GROUP<T>, ROWS = Grad<T, L>::ROWS;
  __shared__ int cls[ROWS][MAX_TOP];
  __shared__ float mass[ROWS][MAX_TOP];
  __shared__ int found[ROWS];
  const int sub = threadIdx.x / L, lane = threadIdx.x % L;
  const int64_t r = (int64_t)(blockIdx.x / pieces) * ROWS + sub;
  const int64_t lo = blockIdx.x % pieces * Grad<T, L>::PIECE;
  const int64_t hi = lo + Grad<T, L>::PIECE < vocab ? lo + Grad<T, L>::PIECE : vocab;
  const float k = LOG2E / temp;
  const T* sr = s + r * lds;
  T* dr = ds + r * vocab;
  float m = 0.0f, inv = 0.0f, ti = 0.0f, g = 0.0f;
  if (r < rows) {
    const float4 st = *reinterpret_cast<const float4*>(stats + 4 * r);
    m = st.x, inv = st.y, ti = st.w;
    g = temp * (grad_rows ? grad[r] : grad[0]);
    if (mean) g /= fmaxf(count[0], 1.0f);
    if (lane < 64) {  // the row's first wave picks the entries of this piece, in their order
      int n = 0;
      for (int e0 = 0; e0 < en.top; e0 += 64) {
        const int e = e0 + lane;
        const int64_t i = e < en.top && ti != 0.0f ? en.klass(r, e) : -1;
        const bool in = i >= lo && i < hi;
        const unsigned long long all = __ballot(in);
        if (in) {
          const int at = n + __popcll(all & ((1ull << lane) - 1));
          cls[sub][at] = (int)i;
          mass[sub][at] = __builtin_amdgcn_exp2f((en.logit(r, e) - st.z) * k) * ti;
        }
        n += __popcll(all);
      }
      if (lane == 0) found[sub] = n;
    }
    auto value = [&](float v) { return ti == 0.0f ? 0.0f : g * (__builtin_amdgcn_exp2f((v - m) * k) * inv); };
    constexpr int U = 4;
    int64_t c = lo + lane * GR;
    for (; c + (U - 1) * L * GR + GR <= hi; c += U * L * GR) {
      Vec<T, GR> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = load_group(sr + c + u * L * GR, GR);
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < GR; ++i) raw[u].v[i] = (T)value((float)raw[u].v[i]);
        store_group(dr + c + u * L * GR, raw[u], GR);
      }
    }
    for (; c < hi; c += L * GR) {
      Vec<T, GR> raw = load_group(sr + c, hi - c);
#pragma unroll
      for (int i = 0; i < GR; ++i) raw.v[i] = (T)value((float)raw.v[i]);
      store_group(dr + c, raw, hi - c);
    }
  }
  __syncthreads();  // the lists, and the piece as it is without the teacher
  if (r >= rows) return;
  const int n = found[sub];
  for (int e = lane; e < n; e += L) {
    const int i = cls[sub][e];
    bool first = true;
    for (int f = 0; f < e; ++f) first = first && cls[sub][f] != i;
    if (!first) continue;
    float p = mass[sub][e];
    for (int f = e + 1; f < n; ++f)
      if (cls[sub][f] == i) p += mass[sub][f];
    dr[i] = (T)(g * (__builtin_amdgcn_exp2f(((float)sr[i] - m) * k) * inv - p));
  }
}

// Pieces of a row in the forward pass: none for rows that a wave takes; else as many as fill the chip
// with four workgroups a CU, each with two rounds of loads at least.
int splits_of(int64_t rows, int64_t vocab, int dtype) {
  const int64_t size = type_bytes(dtype);
  if (rows == 0 || vocab * size <= WAVE_BYTES) return 1;
  int64_t n = cdiv(1024, rows);
  const int64_t most = cdiv(vocab * size, WIDE * 16 * 2);
  if (n > most) n = most;
  return (int)(n > MAX_SPLITS ? MAX_SPLITS : n);
}

// Rows in a launch of `blocks` workgroups of `threads` for each `each` rows: a launch has fewer than 2^32 threads.
int64_t slice_of(int64_t each, int64_t blocks, int threads) { return ((1LL << 32) - 1) / threads / blocks * each; }

int check(const void* s, int64_t lds, const void* t, int64_t ldt, const void* index, int64_t ldi, int64_t rows,
          int64_t vocab, int64_t top, float temp, int tdtype, int index_bytes, const float* stats) {
  QNN_REQUIRE(rows >= 0 && rows < (1LL << 31), "rows: 0 to 2^31 - 1");
  QNN_REQUIRE(vocab >= 1 && vocab < (1LL << 31), "vocab: 1 to 2^31 - 1");
  QNN_REQUIRE(top >= 1 && top <= MAX_TOP, "top: 1 to 1024");
  QNN_REQUIRE(lds >= vocab && ldt >= top && ldi >= top, "a row stride is shorter than the row");
  QNN_REQUIRE(temp >= 0x1p-60f && temp <= 0x1p60f, "temp: 2^-60 to 2^60");
  QNN_REQUIRE(tdtype == QNN_F32 || tdtype == QNN_BF16 || tdtype == QNN_F16, "tdtype: QNN_F32, QNN_BF16 or QNN_F16");
  QNN_REQUIRE(index_bytes == 4 || index_bytes == 8, "index_bytes: 4 or 8");
  QNN_REQUIRE(stats && (rows == 0 || (s && t && index)), "null pointer");
  QNN_REQUIRE(aligned16(stats), "stats: on a 16-byte boundary");
  return QNN_OK;
}

}  // namespace
}  // namespace qnn

using namespace qnn;
using namespace qnn::fl;

extern "C" {

int qnn_topk_distill_fwd_work(int64_t rows, int64_t vocab, int dtype, int64_t* bytes) {
  QNN_REQUIRE(rows >= 0 && vocab >= 1 && bytes, "bad shape or null pointer");
  QNN_REQUIRE(dtype == QNN_F32 || dtype == QNN_BF16 || dtype == QNN_F16, "dtype: QNN_F32, QNN_BF16 or QNN_F16");
  const int n = splits_of(rows, vocab, dtype);
  *bytes = n > 1 ? rows * n * (int64_t)sizeof(Run) : 0;
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
  const int splits = splits_of(rows, vocab, dtype);
  const bool all = splits > 1 && rows <= ALL_ROWS;
  const int rc = with_type(dtype, [&](auto z) {
    using T = decltype(z);
    if (rows == 0) return (int)QNN_OK;
    if (splits > 1) {
      QNN_REQUIRE(work && work_bytes >= rows * splits * (int64_t)sizeof(Run),
                  "work: at least what qnn_topk_distill_fwd_work says");
      // a whole number of groups, so that pieces begin where a lane's loads do
      const int64_t piece = cdiv(cdiv(vocab, splits), GROUP<T>) * GROUP<T>;
      hipLaunchKernelGGL((distill_part_kernel<T>), dim3((unsigned)(rows * splits)), dim3(WIDE), 0, st, (const T*)s, lds,
                         vocab, temp, splits, piece, (Run*)work);
      QNN_LAUNCH_CHECK("qnn_topk_distill_fwd");
      if (all)
        hipLaunchKernelGGL((distill_split_rows_kernel<T, true>), dim3(1), dim3(64 * ALL_ROWS), 0, st, (const T*)s, lds, en,
                           rows, vocab, temp, splits, (const Run*)work, row_loss, stats, loss, mean);
      else
        hipLaunchKernelGGL((distill_split_rows_kernel<T, false>), dim3((unsigned)cdiv(rows, NT / 64)), dim3(NT), 0, st,
                           (const T*)s, lds, en, rows, vocab, temp, splits, (const Run*)work, row_loss, stats, loss,
                           mean);
    } else {
      auto launch = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value, THREADS = L > NT ? L : NT, ROWS = THREADS / L;
        const int64_t slice = slice_of(ROWS, 1, THREADS);
        for (int64_t r = 0; r < rows; r += slice) {
          const int64_t n = rows - r < slice ? rows - r : slice;
          hipLaunchKernelGGL((distill_rows_kernel<T, L>), dim3((unsigned)cdiv(n, ROWS)), dim3(THREADS), 0, st,
                             (const T*)s + r * lds, lds, en.from(r), n, vocab, temp, row_loss + r, stats + 4 * r);
        }
      };
      if (vocab * (int64_t)sizeof(T) <= WAVE_BYTES) launch(std::integral_constant<int, 64>{});
      else launch(std::integral_constant<int, WIDE>{});
    }
    QNN_LAUNCH_CHECK("qnn_topk_distill_fwd");
    return (int)QNN_OK;
  });
  if (rc || all) return rc;
  hipLaunchKernelGGL(distill_join_kernel, dim3(1), dim3(JOIN), 0, st, row_loss, stats, stats + 4 * rows, loss, rows,
                     mean);
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
    auto launch = [&](auto lanes) {
      constexpr int L = decltype(lanes)::value;
      using G = Grad<T, L>;
      const int64_t pieces = cdiv(vocab, G::PIECE), slice = slice_of(G::ROWS, pieces, G::THREADS);
      for (int64_t r = 0; r < rows; r += slice) {
        const int64_t n = rows - r < slice ? rows - r : slice;
        hipLaunchKernelGGL((distill_grad_kernel<T, L>), dim3((unsigned)(cdiv(n, G::ROWS) * pieces)), dim3(G::THREADS), 0,
                           (hipStream_t)stream, (const T*)s + r * lds, lds, en.from(r), stats + 4 * r, stats + 4 * rows,
                           grad_rows ? grad + r : grad, grad_rows, (T*)ds + r * vocab, n, vocab, (int)pieces, temp, mean);
      }
    };
    if (vocab * (int64_t)sizeof(T) <= WAVE_BYTES) launch(std::integral_constant<int, 64>{});
    else launch(std::integral_constant<int, WIDE>{});
    QNN_LAUNCH_CHECK("qnn_topk_distill_bwd");
    return (int)QNN_OK;
  });
}

}  // extern "C"
