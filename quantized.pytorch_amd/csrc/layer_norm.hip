// Layer norm, forward and backward (include/qnn.h: qnn_layer_norm_fwd, qnn_layer_norm_bwd).
//   mean = sum(x) / d, var = sum((x - mean)^2) / d, rstd = 1 / sqrt(var + eps), xh = (x - mean) rstd
//   y = xh w + b;  g = dy w;  dx = rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over rows of dy xh;  db = sum over rows of dy
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx, each once.  A row
// lives in the registers of L lanes (G groups of 16 bytes a lane), so the two-step variance and the two
// means of the backward pass cost no second read.  A workgroup takes rows in strides of the grid with
// the next two on their way while it works on one; the weights stay in registers from row to row.
// 16384 x 4096 bf16: forward 47 us (5.7 TB/s), backward 85 (4.7 TB/s) and 5.
//
// Wide rows ask for more registers than there are.  Backward over 8192 columns spills 164 to 1052 bytes a lane, forward
// over 2048 groups (16384 columns of 16 bits, 8192 of fp32) 20 to 444; 4097 to 8192 columns of 16 bits leave the
// backward pass one wave a SIMD.  1000 x 8192 bf16 forward 12 us and backward 22, 1000 x
// 16384 18 and 70 (of which the bytes are 13 and 20), 1000 x 12288 fp32 26 and 112 (20 and 30), 1000 x 32768 bf16
// 97 and 358 (27 and 40).
//
// The backward pass sums dw and db on the way: a lane has the same columns in every row, so they are sums
// in its registers, joined over a workgroup's rows in LDS, written as one partial row a workgroup and
// added up by a second, small launch in a fixed order.  Where a workgroup has one row of few (up to 512), the
// partial rows are more than the data: 512 x 4096 bf16 33.6 MB beside 12.6, 12.5 us and 4.8 (the bytes: 2.6).
//
// Rows shorter than a group are a thread's each: 4.2 million x 4 bf16 24 us and 63 (the bytes: 14 and 21).
#include "float_common.h"

namespace qnn {
namespace {
using namespace fl;

// Sums over the L lanes that share a row: shuffles, then (L > 64) the waves' results through LDS,
// two slots used in turn so that one barrier a sum is enough.
template <int L, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* sh, int& turn) {
#pragma unroll
  for (int o = (L < 64 ? L : 64) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o, 64);
  if constexpr (L > 64) {
    constexpr int W = L / 64;
    float* at = sh + turn * 2 * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) at[i * W + threadIdx.x / 64] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = at[i * W];
#pragma unroll
      for (int w = 1; w < W; ++w) s += at[i * W + w];
      v[i] = s;
    }
  }
}

// L lanes a row, G groups of 16 bytes a lane, D rows ahead of the present one on their way.
template <int L_, int G_>
struct Shape {
  static constexpr int L = L_, G = G_, NT = L > 256 ? L : 256, ROWS = NT / L, D = 2;
};

// A lane's columns: group j is columns at[j] ... at[j] + GROUP - 1, of which the first skip[j] belong to
// another lane too.  The groups lie (j L + lane) GROUP from the row's start, but no further than the last
// whole one that the row holds: every load is a whole group inside the row, without a branch, and what a
// lane has twice is left out of sums and written twice with the same value.
template <class T, class S>
struct Columns {
  int at[S::G], skip[S::G];
  __device__ __forceinline__ Columns(int lane, int dim) {
#pragma unroll
    for (int j = 0; j < S::G; ++j) {
      const int c = (j * S::L + lane) * GROUP<T>;
      at[j] = c < dim - GROUP<T> ? c : dim - GROUP<T>;
      skip[j] = c - at[j];
    }
  }
  __device__ __forceinline__ bool owns(int j, int i) const { return i >= skip[j]; }
  __device__ __forceinline__ bool any(int j) const { return skip[j] < GROUP<T>; }
};

template <class T, class W, class S>
__global__ __launch_bounds__(S::NT) void layer_norm_fwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                               const W* __restrict__ w, const W* __restrict__ b,
                                                               T* __restrict__ y, float* __restrict__ mean,
                                                               float* __restrict__ rstd, int64_t rows, int dim,
                                                               float eps) {
  constexpr int L = S::L, G = S::G, GR = GROUP<T>, D = S::D;
  __shared__ float sh[4 * (L > 64 ? L / 64 : 1)];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const Columns<T, S> col(lane, dim);
  int turn = 0;
  const float inv = 1.0f / (float)dim;
  float wv[G][GR], bv[G][GR];
  Vec<T, GR> ahead[D][G];
  const int64_t first = (int64_t)blockIdx.x * S::ROWS + sub, step = (int64_t)gridDim.x * S::ROWS;
  auto fetch = [&](int64_t row, int d) {  // (past the last row: that one again, which is not used)
    const T* p = x + (row < rows ? row : rows - 1) * ldx;
#pragma unroll
    for (int j = 0; j < G; ++j) ahead[d][j] = load_group(p + col.at[j], GR);
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(first + d * step, d);
#pragma unroll
  for (int j = 0; j < G; ++j) {
#pragma unroll
    for (int i = 0; i < GR; ++i) {
      wv[j][i] = 1.0f;
      bv[j][i] = 0.0f;
    }
    if (w) load_n<W, GR>(wv[j], w + col.at[j], GR);
    if (b) load_n<W, GR>(bv[j], b + col.at[j], GR);
  }
  auto one = [&](int64_t r, int d) {
    float v[G][GR];
    float s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int i = 0; i < GR; ++i) {
        v[j][i] = (float)ahead[d][j].v[i];
        s[0] += col.owns(j, i) ? v[j][i] : 0.0f;
      }
    fetch(r + D * step, d);
    row_sums<L>(s, sh, turn);
    const float mu = s[0] * inv;
    float q[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int i = 0; i < GR; ++i) {
        v[j][i] -= mu;
        q[0] = fmaf(v[j][i], col.owns(j, i) ? v[j][i] : 0.0f, q[0]);
      }
    row_sums<L>(q, sh, turn);
    const float rs = 1.0f / sqrtf(fmaf(q[0], inv, eps));
    if (r < rows) {
#pragma unroll
      for (int j = 0; j < G; ++j) {
        Vec<T, GR> o;
#pragma unroll
        for (int i = 0; i < GR; ++i) o.v[i] = (T)fmaf(v[j][i] * rs, wv[j][i], bv[j][i]);
        if (col.any(j)) store_group(y + r * dim + col.at[j], o, GR);
      }
      if (lane == 0 && mean) mean[r] = mu;
      if (lane == 0 && rstd) rstd[r] = rs;
    }
  };
  // every lane of a workgroup takes part in every round, for the barriers in its sums
  int64_t r = first;
  for (int64_t r0 = (int64_t)blockIdx.x * S::ROWS; r0 < rows; r0 += D * step, r += D * step)
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (d == 0 || r0 + d * step < rows) one(r + d * step, d);
}

// part: [gridDim.x][2][dim], this workgroup's sums of dw and db (null: not wanted)
template <class T, class W, class S>
__global__ __launch_bounds__(S::NT) void layer_norm_bwd_kernel(const T* __restrict__ dy, int64_t ldy,
                                                               const T* __restrict__ x, int64_t ldx,
                                                               const W* __restrict__ w,
                                                               const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, T* __restrict__ dx,
                                                               float* __restrict__ part, int64_t rows, int dim) {
  constexpr int L = S::L, G = S::G, GR = GROUP<T>, D = S::D;
  __shared__ float sh[4 * (L > 64 ? L / 64 : 1)];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const Columns<T, S> col(lane, dim);
  int turn = 0;
  const float inv = 1.0f / (float)dim;
  float wv[G][GR], aw[G][GR] = {}, ab[G][GR] = {};
  Vec<T, GR> nx[D][G], ny[D][G];
  float nmu[D], nrs[D];
  const int64_t first = (int64_t)blockIdx.x * S::ROWS + sub, step = (int64_t)gridDim.x * S::ROWS;
  auto fetch = [&](int64_t row, int d) {
    const int64_t k = row < rows ? row : rows - 1;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      nx[d][j] = load_group(x + k * ldx + col.at[j], GR);
      ny[d][j] = load_group(dy + k * ldy + col.at[j], GR);
    }
    nmu[d] = mean[k];
    nrs[d] = rstd[k];
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(first + d * step, d);
#pragma unroll
  for (int j = 0; j < G; ++j) {
#pragma unroll
    for (int i = 0; i < GR; ++i) wv[j][i] = 1.0f;
    if (w) load_n<W, GR>(wv[j], w + col.at[j], GR);
  }
  auto one = [&](int64_t r, int d) {
    float h[G][GR], g[G][GR];
    float s[2] = {0.0f, 0.0f};
    const float mu = nmu[d], rs = nrs[d];
    const bool there = r < rows;
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int i = 0; i < GR; ++i) {
        h[j][i] = ((float)nx[d][j].v[i] - mu) * rs;
        const float v = there ? (float)ny[d][j].v[i] : 0.0f;
        g[j][i] = v * wv[j][i];
        aw[j][i] = fmaf(v, there ? h[j][i] : 0.0f, aw[j][i]);
        ab[j][i] += v;
        const float mine = col.owns(j, i) ? g[j][i] : 0.0f;
        s[0] += mine;
        s[1] = fmaf(mine, h[j][i], s[1]);
      }
    fetch(r + D * step, d);
    if (dx) {
      row_sums<L>(s, sh, turn);
      const float sg = s[0] * inv, sx = s[1] * inv;
      if (there) {
#pragma unroll
        for (int j = 0; j < G; ++j) {
          Vec<T, GR> o;
#pragma unroll
          for (int i = 0; i < GR; ++i) o.v[i] = (T)(rs * (g[j][i] - sg - h[j][i] * sx));
          if (col.any(j)) store_group(dx + r * dim + col.at[j], o, GR);
        }
      }
    }
  };
  int64_t r = first;
  for (int64_t r0 = (int64_t)blockIdx.x * S::ROWS; r0 < rows; r0 += D * step, r += D * step)
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (d == 0 || r0 + d * step < rows) one(r + d * step, d);
  if (!part) return;
  if constexpr (S::ROWS > 1) {  // the workgroup's rows, in their order
    __shared__ float all[S::ROWS][L * G * GR];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < G; ++j)
#pragma unroll
        for (int i = 0; i < GR; ++i)
          if (col.owns(j, i)) all[sub][col.at[j] + i] = which ? ab[j][i] : aw[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < dim; c += S::NT) {
        float s = all[0][c];
#pragma unroll
        for (int k = 1; k < S::ROWS; ++k) s += all[k][c];
        part[((int64_t)blockIdx.x * 2 + which) * dim + c] = s;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < G; ++j)
      if (col.any(j)) {
        float* p = part + (int64_t)blockIdx.x * 2 * dim + col.at[j];
        store_n<float, GR>(p, aw[j], GR);
        store_n<float, GR>(p + dim, ab[j], GR);
      }
  }
}

// A sum is at most 1024 additions deep (of rows to 2^27 columns): CHAIN of a lane's own terms one after another, the rows
// of a workgroup, JOINED partial rows, and the sums of those.
constexpr int CHAIN = 512, JOINED = 256;

// dw and db from `parts` partial rows: 64 columns a workgroup at a time, 16 threads a column
template <class W>
__global__ __launch_bounds__(1024) void layer_norm_join_kernel(const float* __restrict__ part, int parts, int dim,
                                                               W* dw, W* db) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, k = threadIdx.x >> 6;
  for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < 2 * (int64_t)dim; c0 += (int64_t)gridDim.x * 64) {
    const int64_t c = c0 + lane;  // over dw's columns, then db's
    float s = 0.0f;
    if (c < 2 * (int64_t)dim)
      for (int p0 = k; p0 < parts; p0 += 16 * JOINED) {
        const int p1 = p0 + 16 * JOINED < parts ? p0 + 16 * JOINED : parts;
        float t = 0.0f;
#pragma unroll 8
        for (int p = p0; p < p1; p += 16) t += part[(int64_t)p * 2 * dim + c];
        s += t;
      }
    sh[k][lane] = s;
    __syncthreads();
    if (k == 0 && c < 2 * (int64_t)dim) {
#pragma unroll
      for (int i = 1; i < 16; ++i) s += sh[i][lane];
      if (c < dim) {
        if (dw) dw[c] = (W)s;
      } else if (db) {
        db[c - dim] = (W)s;
      }
    }
    __syncthreads();
  }
}

// ---- rows shorter than a group: a row a thread
constexpr int NARROW = 256;

template <class T>
__device__ __forceinline__ void load_narrow(float (&v)[GROUP<T>], const T* p, int dim) {
#pragma unroll
  for (int i = 0; i < GROUP<T>; ++i) v[i] = i < dim ? (float)p[i] : 0.0f;
}

template <class T, class W>
__global__ __launch_bounds__(NARROW) void layer_norm_fwd_narrow_kernel(const T* x, int64_t ldx, const W* w, const W* b,
                                                                       T* y, float* mean, float* rstd, int64_t rows,
                                                                       int dim, float eps) {
  constexpr int GR = GROUP<T>;
  float wv[GR], bv[GR];
#pragma unroll
  for (int i = 0; i < GR; ++i) {
    wv[i] = w && i < dim ? (float)w[i] : 1.0f;
    bv[i] = b && i < dim ? (float)b[i] : 0.0f;
  }
  for (int64_t r = (int64_t)blockIdx.x * NARROW + threadIdx.x; r < rows; r += (int64_t)gridDim.x * NARROW) {
    float v[GR], s = 0.0f, q = 0.0f;
    load_narrow<T>(v, x + r * ldx, dim);
#pragma unroll
    for (int i = 0; i < GR; ++i) s += v[i];
    const float mu = s / (float)dim;
#pragma unroll
    for (int i = 0; i < GR; ++i) {
      const float d = i < dim ? v[i] - mu : 0.0f;
      q = fmaf(d, d, q);
    }
    const float rs = 1.0f / sqrtf(q / (float)dim + eps);
#pragma unroll
    for (int i = 0; i < GR; ++i)
      if (i < dim) y[r * dim + i] = (T)fmaf((v[i] - mu) * rs, wv[i], bv[i]);
    if (mean) mean[r] = mu;
    if (rstd) rstd[r] = rs;
  }
}

// dx, and this workgroup's sums of dw and db into part as in layer_norm_bwd_kernel (each null: not wanted)
template <class T, class W>
__global__ __launch_bounds__(NARROW) void layer_norm_bwd_narrow_kernel(const T* dy, int64_t ldy, const T* x,
                                                                       int64_t ldx, const W* w, const float* mean,
                                                                       const float* rstd, T* dx, float* part,
                                                                       int64_t rows, int dim) {
  constexpr int GR = GROUP<T>;
  __shared__ float sh[NARROW / 64][2][GR];
  float wv[GR], sum[2][GR] = {};
#pragma unroll
  for (int i = 0; i < GR; ++i) wv[i] = w && i < dim ? (float)w[i] : 1.0f;
  for (int64_t r = (int64_t)blockIdx.x * NARROW + threadIdx.x; r < rows; r += (int64_t)gridDim.x * NARROW) {
    float v[GR], d[GR], s = 0.0f, q = 0.0f;
    load_narrow<T>(v, x + r * ldx, dim);
    load_narrow<T>(d, dy + r * ldy, dim);
    const float mu = mean[r], rs = rstd[r];
#pragma unroll
    for (int i = 0; i < GR; ++i) {
      v[i] = i < dim ? (v[i] - mu) * rs : 0.0f;
      sum[0][i] = fmaf(d[i], v[i], sum[0][i]);
      sum[1][i] += d[i];
      d[i] *= wv[i];
      s += d[i];
      q = fmaf(d[i], v[i], q);
    }
    const float sg = s / (float)dim, sx = q / (float)dim;
    if (dx)
#pragma unroll
      for (int i = 0; i < GR; ++i)
        if (i < dim) dx[r * dim + i] = (T)(rs * (d[i] - sg - v[i] * sx));
  }
  if (!part) return;
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int i = 0; i < GR; ++i) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sum[which][i] += __shfl_xor(sum[which][i], o, 64);
      if ((threadIdx.x & 63) == 0) sh[threadIdx.x / 64][which][i] = sum[which][i];
    }
  __syncthreads();
  const int which = threadIdx.x / GR, i = threadIdx.x % GR;
  if (which < 2 && i < dim) {
    float s = sh[0][which][i];
#pragma unroll
    for (int k = 1; k < NARROW / 64; ++k) s += sh[k][which][i];
    part[((int64_t)blockIdx.x * 2 + which) * dim + i] = s;
  }
}

// ---- rows too long for registers: a workgroup a row, read again (from L2) for each step
constexpr int LONG = 1024;
// columns over which a thread adds one after another: CHAIN of its own
constexpr int64_t RUN = (int64_t)LONG * CHAIN;

template <class T, class W>
__global__ __launch_bounds__(LONG) void layer_norm_fwd_long_kernel(const T* x, int64_t ldx, const W* w, const W* b,
                                                                   T* y, float* mean, float* rstd, int64_t dim,
                                                                   float eps) {
  constexpr int GR = GROUP<T>;
  __shared__ float sh[4 * (LONG / 64)];
  const int64_t r = blockIdx.x;
  const T* xr = x + r * ldx;
  int turn = 0;
  float s[1] = {0.0f}, q[1] = {0.0f}, v[GR];
  for (int64_t c0 = 0; c0 < dim; c0 += RUN) {
    const int64_t end = c0 + RUN < dim ? c0 + RUN : dim;
    float t = 0.0f;
    for (int64_t c = c0 + threadIdx.x * GR; c < end; c += LONG * GR) {
      load_n<T, GR>(v, xr + c, dim - c);
#pragma unroll
      for (int i = 0; i < GR; ++i) t += v[i];
    }
    s[0] += t;
  }
  row_sums<LONG>(s, sh, turn);
  const float mu = s[0] / (float)dim;
  for (int64_t c0 = 0; c0 < dim; c0 += RUN) {
    const int64_t end = c0 + RUN < dim ? c0 + RUN : dim;
    float t = 0.0f;
    for (int64_t c = c0 + threadIdx.x * GR; c < end; c += LONG * GR) {
      load_n<T, GR>(v, xr + c, dim - c);
#pragma unroll
      for (int i = 0; i < GR; ++i) {
        const float d = c + i < dim ? v[i] - mu : 0.0f;
        t = fmaf(d, d, t);
      }
    }
    q[0] += t;
  }
  row_sums<LONG>(q, sh, turn);
  const float rs = 1.0f / sqrtf(q[0] / (float)dim + eps);
  for (int64_t c = threadIdx.x * GR; c < dim; c += LONG * GR) {
    float wv[GR], bv[GR];
    load_n<T, GR>(v, xr + c, dim - c);
    if (w) load_n<W, GR>(wv, w + c, dim - c);
    if (b) load_n<W, GR>(bv, b + c, dim - c);
#pragma unroll
    for (int i = 0; i < GR; ++i) v[i] = fmaf((v[i] - mu) * rs, w ? wv[i] : 1.0f, b ? bv[i] : 0.0f);
    store_n<T, GR>(y + r * dim + c, v, dim - c);
  }
  if (threadIdx.x == 0) {
    if (mean) mean[r] = mu;
    if (rstd) rstd[r] = rs;
  }
}

template <class T, class W>
__global__ __launch_bounds__(LONG) void layer_norm_dx_long_kernel(const T* dy, int64_t ldy, const T* x, int64_t ldx,
                                                                  const W* w, const float* mean, const float* rstd,
                                                                  T* dx, int64_t dim) {
  constexpr int GR = GROUP<T>;
  __shared__ float sh[4 * (LONG / 64)];
  const int64_t r = blockIdx.x;
  const float mu = mean[r], rs = rstd[r];
  int turn = 0;
  float s[2] = {0.0f, 0.0f}, v[GR], g[GR], wv[GR];
  auto load = [&](int64_t c) {
    load_n<T, GR>(v, x + r * ldx + c, dim - c);
    load_n<T, GR>(g, dy + r * ldy + c, dim - c);
    if (w) load_n<W, GR>(wv, w + c, dim - c);
#pragma unroll
    for (int i = 0; i < GR; ++i) {
      v[i] = (v[i] - mu) * rs;
      if (w) g[i] *= wv[i];
    }
  };
  for (int64_t c0 = 0; c0 < dim; c0 += RUN) {
    const int64_t end = c0 + RUN < dim ? c0 + RUN : dim;
    float t0 = 0.0f, t1 = 0.0f;
    for (int64_t c = c0 + threadIdx.x * GR; c < end; c += LONG * GR) {
      load(c);
#pragma unroll
      for (int i = 0; i < GR; ++i) {
        t0 += g[i];
        t1 = fmaf(g[i], v[i], t1);
      }
    }
    s[0] += t0;
    s[1] += t1;
  }
  row_sums<LONG>(s, sh, turn);
  const float sg = s[0] / (float)dim, sx = s[1] / (float)dim;
  for (int64_t c = threadIdx.x * GR; c < dim; c += LONG * GR) {
    load(c);
#pragma unroll
    for (int i = 0; i < GR; ++i) v[i] = rs * (g[i] - sg - v[i] * sx);
    store_n<T, GR>(dx + r * dim + c, v, dim - c);
  }
}

// part as in layer_norm_bwd_kernel: workgroup (c, p) sums rows p, p + parts, ... of its 256 groups
template <class T>
__global__ __launch_bounds__(256) void layer_norm_dw_long_kernel(const T* dy, int64_t ldy, const T* x, int64_t ldx,
                                                                 const float* mean, const float* rstd, float* part,
                                                                 int64_t rows, int64_t dim) {
  constexpr int GR = GROUP<T>;
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * GR;
  if (c >= dim) return;
  float aw[GR] = {}, ab[GR] = {}, v[GR], d[GR];
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    load_n<T, GR>(v, x + r * ldx + c, dim - c);
    load_n<T, GR>(d, dy + r * ldy + c, dim - c);
    const float mu = mean[r], rs = rstd[r];
#pragma unroll
    for (int i = 0; i < GR; ++i) {
      aw[i] = fmaf(d[i], (v[i] - mu) * rs, aw[i]);
      ab[i] += d[i];
    }
  }
  float* p = part + (int64_t)blockIdx.y * 2 * dim + c;
  store_n<float, GR>(p, aw, dim - c);
  store_n<float, GR>(p + dim, ab, dim - c);
}

template <class F>
int with_types(int dtype, int wdtype, F&& f) {
  if (wdtype != dtype && wdtype != QNN_F32) return arg_error("wdtype: the rows' type or QNN_F32");
  return with_type(dtype, [&](auto t) {
    if (wdtype == QNN_F32) return f(t, 0.0f);
    return f(t, t);
  });
}

// The shape for rows of `dim`: the fewest lanes with at most 2 groups each up to a wave, then
// workgroups of 256 (up to 4) and of 1024.  False: too long, or shorter than a group.
template <class T, class F>
bool with_shape(int64_t dim, F&& f) {
  const int64_t g = cdiv(dim, GROUP<T>);
  if (dim < GROUP<T>) return false;  // no whole group
  if (g <= 16) f(Shape<16, 1>{});
  else if (g <= 64) f(Shape<64, 1>{});
  else if (g <= 128) f(Shape<64, 2>{});
  else if (g <= 256) f(Shape<256, 1>{});
  else if (g <= 512) f(Shape<256, 2>{});
  else if (g <= 1024) f(Shape<256, 4>{});
  else if (g <= 2048) f(Shape<1024, 2>{});
  else if (g <= 4096) f(Shape<1024, 4>{});
  else return false;
  return true;
}

// Partial rows of dw and db: two workgroups of 256 a CU (where their registers let two of them in, see above), and as
// many as keep a lane's sums within CHAIN rows.
constexpr int MAX_PARTS = 512;

// workgroups of a launch over all rows, `each` of them at a time in one
unsigned row_blocks(int64_t rows, int64_t each, int64_t most) {
  const int64_t n = cdiv(rows, each);
  return (unsigned)(n < most ? n : most);
}
int64_t row_parts(int64_t rows, int64_t each, int64_t most = MAX_PARTS) {
  const int64_t chains = cdiv(rows, each * CHAIN);
  return row_blocks(rows, each, chains > most ? chains : most);
}
template <class T>
int64_t parts_of(int64_t rows, int64_t dim) {
  int64_t parts = 0;
  if (with_shape<T>(dim, [&](auto shape) { parts = row_parts(rows, decltype(shape)::ROWS); })) return parts;
  return dim < GROUP<T> ? row_parts(rows, NARROW) : row_parts(rows, 1, 64);
}

int check(int64_t rows, int64_t dim, int64_t ld) {
  QNN_REQUIRE(rows >= 0 && rows < (1LL << 31), "rows: 0 to 2^31 - 1");
  QNN_REQUIRE(dim >= 1 && dim < (1LL << 31), "dim: 1 to 2^31 - 1");
  QNN_REQUIRE(ld >= dim, "a row stride is shorter than the row");
  return QNN_OK;
}

// Rows too long for registers are a workgroup each, and a launch has fewer than 2^32 threads.
template <class T>
int check_long(int64_t rows, int64_t dim) {
  QNN_REQUIRE(cdiv(dim, GROUP<T>) <= 4096 || rows < (1LL << 32) / LONG,
              "too many rows for one call: under 2^22 of more than 4096 groups of 16 bytes");
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
    hipStream_t s = (hipStream_t)stream;
    if (int rc = check_long<T>(rows, dim)) return rc;
    const bool held = with_shape<T>(dim, [&](auto shape) {
      using S = decltype(shape);
      hipLaunchKernelGGL((layer_norm_fwd_kernel<T, W, S>), dim3(row_blocks(rows, S::ROWS, S::NT > 256 ? 512 : 1024)),
                         dim3(S::NT), 0, s, (const T*)x, ldx, (const W*)w, (const W*)b, (T*)y, mean, rstd, rows,
                         (int)dim, eps);
    });
    if (!held && dim < GROUP<T>)
      hipLaunchKernelGGL((layer_norm_fwd_narrow_kernel<T, W>), dim3(row_blocks(rows, NARROW, 2048)), dim3(NARROW), 0, s,
                         (const T*)x, ldx, (const W*)w, (const W*)b, (T*)y, mean, rstd, rows, (int)dim, eps);
    else if (!held)
      hipLaunchKernelGGL((layer_norm_fwd_long_kernel<T, W>), dim3((unsigned)rows), dim3(LONG), 0, s, (const T*)x, ldx,
                         (const W*)w, (const W*)b, (T*)y, mean, rstd, dim, eps);
    QNN_LAUNCH_CHECK("qnn_layer_norm_fwd");
    return (int)QNN_OK;
  });
}

int qnn_layer_norm_bwd_work(int64_t rows, int64_t dim, int dtype, int64_t* bytes) {
  if (int rc = check(rows, dim, dim)) return rc;
  QNN_REQUIRE(bytes, "null pointer");
  return with_type(dtype, [&](auto t) {
    *bytes = parts_of<decltype(t)>(rows, dim) * 2 * dim * (int64_t)sizeof(float);
    return (int)QNN_OK;
  });
}

int qnn_layer_norm_bwd(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* w, const float* mean,
                       const float* rstd, void* dx, void* dw, void* db, int64_t rows, int64_t dim, int dtype,
                       int wdtype, void* work, int64_t work_bytes, qnn_stream_t stream) {
  if (int rc = check(rows, dim, ldx)) return rc;
  if (int rc = check(rows, dim, ldy)) return rc;
  QNN_REQUIRE(rows == 0 || (dy && x && mean && rstd), "null pointer");
  const bool sums = dw || db;
  return with_types(dtype, wdtype, [&](auto t, auto tw) {
    using T = decltype(t);
    using W = decltype(tw);
    hipStream_t s = (hipStream_t)stream;
    const int64_t parts = parts_of<T>(rows, dim);
    QNN_REQUIRE(!sums || rows == 0 || (work && work_bytes >= parts * 2 * dim * (int64_t)sizeof(float)),
                "work: at least what qnn_layer_norm_bwd_work says");
    if (int rc = check_long<T>(rows, dim)) return rc;
    float* part = sums ? (float*)work : nullptr;
    if (rows > 0 && (dx || sums)) {
      const bool held = with_shape<T>(dim, [&](auto shape) {
        using S = decltype(shape);
        hipLaunchKernelGGL((layer_norm_bwd_kernel<T, W, S>), dim3((unsigned)parts), dim3(S::NT), 0, s, (const T*)dy,
                           ldy, (const T*)x, ldx, (const W*)w, mean, rstd, (T*)dx, part, rows, (int)dim);
      });
      if (!held && dim < GROUP<T>) {
        hipLaunchKernelGGL((layer_norm_bwd_narrow_kernel<T, W>), dim3((unsigned)parts), dim3(NARROW), 0, s,
                           (const T*)dy, ldy, (const T*)x, ldx, (const W*)w, mean, rstd, (T*)dx, part, rows, (int)dim);
      } else if (!held) {
        if (dx)
          hipLaunchKernelGGL((layer_norm_dx_long_kernel<T, W>), dim3((unsigned)rows), dim3(LONG), 0, s, (const T*)dy,
                             ldy, (const T*)x, ldx, (const W*)w, mean, rstd, (T*)dx, dim);
        if (sums)
          hipLaunchKernelGGL((layer_norm_dw_long_kernel<T>),
                             dim3((unsigned)cdiv(dim, 256 * GROUP<T>), (unsigned)parts), dim3(256), 0, s,
                             (const T*)dy, ldy, (const T*)x, ldx, mean, rstd, part, rows, dim);
      }
      QNN_LAUNCH_CHECK("qnn_layer_norm_bwd");
    }
    if (sums) {
      hipLaunchKernelGGL((layer_norm_join_kernel<W>), dim3(row_blocks(2 * dim, 64, 1 << 20)), dim3(1024), 0, s, part,
                         (int)parts, (int)dim, (W*)dw, (W*)db);
      QNN_LAUNCH_CHECK("qnn_layer_norm_bwd");
    }
    return (int)QNN_OK;
  });
}

}  // extern "C"
