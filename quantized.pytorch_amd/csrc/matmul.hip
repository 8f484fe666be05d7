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

// The bias of 8 columns.
template <class T>
__device__ __forceinline__ void bias8(float (&b)[8], const Epilogue& e, int64_t col, int64_t n) {
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = 0.0f;
  if (e.bias) load_n<T, 8>(b, (const T*)e.bias + col, n - col);
}

// WHOLE: all 8 are inside the matrix, which the compiler then need not ask in front of each access.
template <class T, bool WHOLE>
__device__ __forceinline__ void finish8(float (&z)[8], const float (&bias)[8], const Epilogue& e, int64_t row,
                                        int64_t col, int64_t n) {
  const int64_t left = WHOLE ? 8 : n - col;
  if (e.res) {
    float r[8];
    load_n<T, 8>(r, (const T*)e.res + row * e.ldr + col, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] += r[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] += bias[i];
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
    for (int i = 0; i < 8; ++i) gelu_f<sizeof(T) == 4>(z[i], z[i], d[i]);
    if (e.slope) {
      if constexpr (sizeof(T) == 4) {
        store_n<float, 8>((float*)e.slope + row * n + col, d, left);
      } else {
        Vec<int16_t, 8> q;
#pragma unroll
        for (int i = 0; i < 8; ++i) q.v[i] = slope_pack<T>(d[i]);
        store_group((int16_t*)e.slope + row * n + col, q, left);
      }
    }
  }
  store_n<T, 8>((T*)e.y + row * n + col, z, left);
}

// ---------------------------------------------------------------------------- the tiled product
// c[i][j] = sum over k of a(i, k) b(j, k).  An operand is DENSE in k ([rows][k], as x and w in the
// forward pass) or not ([k][rows], as both of dz^T x): then its rows are what is contiguous in memory.
//
// (linear_y_kernel: the forward pass; linear_grads_kernel: both products of the backward pass.)
// A workgroup of WM x WN waves computes a (16 TM WM) x (16 TN WN) tile, a wave (16 TM) x (16 TN) of it
// in 16x16 MFMAs.  k advances in stages of 64 bytes (32 elements of 16 bits, 16 of 32) through a ring
// of 4 LDS slots that direct loads fill (buffer_load ... lds, 16 bytes a lane), three stages ahead; a
// wave reads the fragments of the next stage from LDS while the MFMAs work on the present one's, so
// there is one barrier a stage and no wait for LDS in it.  A fragment is 16 bytes a lane: row lane % 16,
// the (lane / 16)-th quarter of the stage -- one 16x16x32 MFMA of 16-bit types, four 16x16x4 of fp32,
// each k in the same place on both sides.
//   DENSE tile in LDS: [rows][64 bytes], 16-byte chunks XORed by row bits 2-3, read by ds_read_b128.
//   Else: [k of the stage][rows], granules of 16 rows XORed by the bits of k in which the lanes of a
//   read differ; 16-bit types are turned around by ds_read_b64_tr_b16, fp32 read by ds_read_b32.
// The XOR is made on the side of the load's source, since a direct load fills LDS in lane order.
// Rows past the matrix and k past its end are loaded from an offset past the buffer's size, which
// fills LDS with zeros; stages past the last are such loads too, so the counts of loads in flight hold.
//
// The 16 bytes of a direct load may begin at any word.  So rows of fp32 and rows of 16-bit types of an even
// length and stride are loaded as they are, and only the elements that a group of theirs would bring from
// past the matrix or from the next row come after the loop, one at a time (Product::tail): of
// 1890 x 1470 x 11714 bf16 the forward pass takes 90 us and the backward one 138 where copies padded to whole
// groups made them 111 and 152, 22 x 1895 x 10407 fp32 backward 53 for 96.
constexpr uint32_t PAST = 0x80000000u;  // a buffer offset that is past every size below

// Waits until at most N of this wave's loads and none of its LDS reads are under way, then for the other
// waves.  By the builtin, which the compiler counts with: after an asm wait it would add its own before
// each use of a fragment, too long a one where more reads are under way than its 4-bit counter holds.
template <int N>
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

typedef __attribute__((address_space(3))) void* lds_t;
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4* lds_s4_t;

// Four 16-bit elements of one k from each of the lane's neighbours in k (its 16 lanes name 4 k of 16 rows;
// it gets row lane % 16).  `restrict`, because the compiler gives this read no alias information of its
// own, and waits for every direct load under way before it if nothing says that they are apart.
__device__ __forceinline__ s4 turned(const __attribute__((address_space(3))) s4* __restrict p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)p);
}

struct Operand {
  const void* p;
  int64_t ld;    // elements between rows of the matrix in memory
  int64_t rows;  // of the product's operand: m or n
};

// R rows of an operand in a workgroup of W waves: its loads into LDS and its fragments from there.
// SEG: of rows that begin at any 16 bytes (c chunks past a 64-byte boundary), a stage's slot holds what lies
// between two such boundaries: chunk q of the stage is in that slot or, past its end, in the next one.  A load
// of 64 bytes across a boundary takes the memory pipe twice as long: 1336 x 2072 x 3496 fp16 47 -> 37 us,
// 6680 x 1256 x 5136 bf16 128 -> 107, 5556 x 9264 x 2896 328 -> 294.
template <class T, bool DENSE, int R, int W, bool SEG = false>
struct Side {
  static constexpr int ES = (int)sizeof(T), KE = 64 / ES, BYTES = R * 64, LOADS = R / 16 / W;
  static_assert(R % (16 * W) == 0, "a wave loads whole KiB");
  static constexpr int GRAN = 16 * ES, GMASK = R / 16 < 8 ? R / 16 - 1 : 7;  // bytes, and the XOR's bits

  static __device__ __forceinline__ int past(const Operand& o, int64_t row) {
    return SEG ? (int)((uintptr_t)((const T*)o.p + row * o.ld) >> 4 & 3) : 0;
  }
  static __device__ __forceinline__ int turn(int row) { return -(row >> 2) & 3; }  // of a chunk's index, DENSE
  static __device__ __forceinline__ int spread(int k) {  // what a granule's index is XORed with, not DENSE
    if constexpr (ES == 2) return ((k & 3) | (k >> 3 & 1) << 2) & GMASK;
    else return k >> 2 & 3 & GMASK;
  }

  uint32_t off[LOADS];  // this lane's byte offsets from the tile's corner, PAST outside the rows
  int kat[LOADS];       // its k in the stage (elements)
  const char* base;
  int64_t step;

  // from row i0 and element k0 on
  __device__ __forceinline__ void begin(const Operand& o, int64_t i0, int64_t k0, int wave, int lane) {
    if constexpr (DENSE) {
      base = (const char*)o.p + (i0 * o.ld + k0) * ES - (SEG ? 64 : 0);
      step = 64;
    } else {
      base = (const char*)o.p + (k0 * o.ld + i0) * ES;
      step = KE * o.ld * ES;
    }
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int at = (wave * LOADS + j) * 1024 + lane * 16;
      if constexpr (DENSE) {
        const int row = at / 64, chunk = (at / 16 % 4 ^ turn(row)) - past(o, i0 + row);
        kat[j] = chunk * 16 / ES;
        off[j] = i0 + row < o.rows ? (uint32_t)(row * (int)o.ld * ES + chunk * 16 + (SEG ? 64 : 0)) : PAST;
      } else {
        const int k = at / (R * ES), in = at % (R * ES);
        const int col = ((in / GRAN ^ spread(k)) * GRAN + in % GRAN) / ES;
        kat[j] = k;
        off[j] = i0 + col < o.rows ? (uint32_t)((k * (int)o.ld + col) * ES) : PAST;
      }
    }
  }
  // load j of the next stage, of which `left` elements of k are there, into the slot at lds
  // (first: the one in which k begins, where SEG has chunks before it)
  __device__ __forceinline__ void load(char* lds, int j, int left, int wave, bool first) const {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass drops a kernel that names the resource type, without a word
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t)(lds + (wave * LOADS + j) * 1024), 16,
                                             kat[j] < left && !(SEG && first && kat[j] < 0) ? off[j] : PAST, 0, 0, 0);
#endif
  }
  // fragment f (rows 16 f ... of the wave's, which begin at row r0)
  static __device__ __forceinline__ int place(int r0, int lane, int c) {
    if constexpr (DENSE) {
      const int row = lane & 15;
      return (r0 + row) * 64 + ((((lane >> 4) + c) & 3) ^ turn(row)) * 16;
    } else if constexpr (ES == 2) {
      return ((lane >> 4) * 8 + (lane >> 2 & 3)) * R * ES + (lane & 3) * 8;
    } else {
      return (lane >> 4) * 4 * R * ES + (lane & 15) * 4;
    }
  }
  static __device__ __forceinline__ f4 fragment(char* lds, int at, int r0, int f, int lane) {
    if constexpr (DENSE) {
      return *reinterpret_cast<const f4*>(lds + at + f * 1024);
    } else if constexpr (ES == 2) {
      const int h = spread((lane >> 4) * 8 + (lane >> 2 & 3));
      char* p = lds + at + ((r0 / 16 + f) ^ h) * GRAN;
      union {
        s4 s[2];
        f4 v;
      } u;
      u.s[0] = turned((lds_s4_t)p);
      u.s[1] = turned((lds_s4_t)(p + 4 * R * ES));
      return u.v;
    } else {
      const int h = spread((lane >> 4) * 4);
      const char* p = lds + at + ((r0 / 16 + f) ^ h) * GRAN;
      f4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float*>(p + j * R * ES);
      return v;
    }
  }
};

// acc += the 16x16 product of two fragments; the first's rows become the lane's four neighbours
template <class T>
__device__ __forceinline__ f4 mma(f4 a, f4 b, f4 acc) {
  if constexpr (std::is_same_v<T, bf16>) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), acc, 0, 0, 0);
  } else if constexpr (std::is_same_v<T, f16>) {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
    return acc;
  }
}

// The lane's fragment of the last `count` elements of k, from element k on, straight from memory.
template <class T, bool DENSE>
__device__ __forceinline__ f4 rest(const Operand& o, int64_t row, int64_t k, int count, int lane) {
  constexpr int GR = GROUP<T>;
  Vec<T, GR> v = {};
  if (lane < 16) {  // the others' part of the stage is past the end
    row = row + lane < o.rows ? row + lane : o.rows - 1;
    const T* p = (const T*)o.p + (DENSE ? row * o.ld + k : k * o.ld + row);
#pragma unroll
    for (int e = 0; e < GR; ++e)
      if (e < count) v.v[e] = p[DENSE ? e : e * o.ld];
  }
  return __builtin_bit_cast(f4, v);
}

// One product, as a launch's workgroups take it.  Its tiles' sums go through the epilogue, or (splits > 1)
// as they are into part[split][m][ldp].
struct Product {
  Operand a, b;
  int64_t m, n, k;
  int tm, tn;        // tiles
  int splits;
  int blocks;        // tm tn splits
  int64_t span;      // elements of k in a split, a whole number of stages
  int tail, edge;    // the last elements of k that direct loads must not take, at most GROUP<T>, in all tiles and
                     // in those that reach the end of an operand's rows
  float* part;
  int64_t ldp;
  Epilogue e;
};

// Workgroup -> (split, tile row, tile column).  The card deals workgroups out to its 8 XCDs in turn; each
// XCD gets a run of neighbouring tiles, 8 tile rows at a time, so that the panels they share meet in
// its L2.
__device__ __forceinline__ void tile_of(const Product& t, int id, int& split, int& ti, int& tj) {
  const int x = id & 7, q = t.blocks >> 3, r = t.blocks & 7;
  const int lin = x * q + (x < r ? x : r) + (id >> 3);
  const int tiles = t.tm * t.tn;
  split = lin / tiles;
  const int u = lin - split * tiles, band = u / (8 * t.tn), in = u - band * 8 * t.tn;
  const int rows = t.tm - band * 8 < 8 ? t.tm - band * 8 : 8;
  tj = in / rows;
  ti = band * 8 + in - tj * rows;
}

template <int WM_, int WN_, int TM_, int TN_, int EU_>
struct Cfg {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, W = WM * WN, NT = 64 * W, EU = EU_;
  static constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN, SLOT = (BM + BN) * 64, LDS = 4 * SLOT;
};

// A wave's sums to where they go.
template <class T, class C>
__device__ __forceinline__ void emit(const Product& t, const f4 (&acc)[C::TM][C::TN], char* lds, int split, int64_t i0,
                                     int64_t j0, int ri, int rj, int wave, int lane) {
  constexpr int TM = C::TM, TN = C::TN;
  const Epilogue& e = t.e;
  // acc[i][j]: row 16 i + lane % 16, columns 16 j + lane / 16 * 4 ... + 3.  A wave turns as many rows at a
  // time around in its share of LDS as fit, so that a lane has 8 neighbouring columns, the same ones in
  // every row, and a row's are together.  Chunks of 16 bytes are XORed by the row.
  constexpr int COLS = 16 * TN, PER = COLS / 8, FIT = C::LDS / C::W / (COLS * 4) / 16;
  constexpr int TURN = FIT < TM ? FIT : TM;  // 16-row tiles at a time
  static_assert(TURN > 0 && TM % TURN == 0, "whole turns");
  char* mine = lds + wave * (C::LDS / C::W);
  const int col = lane % PER * 8;
  const int64_t gj = j0 + rj + col;
  float bias[8];
  bias8<T>(bias, e, gj, t.n);
  auto rows_out = [&](int64_t gi0, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll 2
    for (int u = 0; u < TURN * 16 * PER / 64; ++u) {
      const int row = u * (64 / PER) + lane / PER;
      float z[8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f4*>(z + 4 * h) =
            *reinterpret_cast<const f4*>(mine + row * COLS * 4 + ((col / 4 + h) ^ (row & (COLS / 4 - 1))) * 16);
      const int64_t gi = gi0 + row;
      if (!WHOLE && (gi >= t.m || gj >= t.n)) continue;
      if (t.splits > 1)
        store_n<float, 8>(t.part + (split * t.m + gi) * t.ldp + gj, z, 8);  // (ldp: whole groups of 8)
      else
        finish8<T, WHOLE>(z, bias, e, gi, gj, t.n);
    }
  };
  const bool inside = i0 + C::BM <= t.m && j0 + C::BN <= t.n;
#pragma unroll
  for (int i = 0; i < TM; i += TURN) {
#pragma unroll
    for (int k = 0; k < TURN; ++k)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = 16 * k + (lane & 15);
        *reinterpret_cast<f4*>(mine + row * COLS * 4 + ((4 * j + (lane >> 4)) ^ (row & (COLS / 4 - 1))) * 16) = acc[i + k][j];
      }
    __builtin_amdgcn_wave_barrier();
    if (inside) rows_out(i0 + ri + 16 * i, std::true_type{});
    else rows_out(i0 + ri + 16 * i, std::false_type{});
    __builtin_amdgcn_wave_barrier();
  }
}

// Workgroup `id` of the product's.
template <class T, bool AD, bool BD, class C, bool SEG>
__device__ __forceinline__ void tile(const Product& t, int id) {
  using A = Side<T, AD, C::BM, C::W, SEG && AD>;
  using B = Side<T, BD, C::BN, C::W, SEG && BD>;
  constexpr int TM = C::TM, TN = C::TN, KE = A::KE, P = A::LOADS + B::LOADS;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int split, ti, tj;
  tile_of(t, id, split, ti, tj);
  const int64_t i0 = (int64_t)ti * C::BM, j0 = (int64_t)tj * C::BN, k0 = split * t.span;
  const bool at_edge = (!AD && i0 + C::BM > t.a.rows) || (!BD && j0 + C::BN > t.b.rows);
  const int tail = t.tail ? t.tail : at_edge ? t.edge : 0;
  const int64_t whole = t.k - tail;
  int left = (int)(whole - k0 < t.span ? whole - k0 : t.span);
  const int stages = (left + KE - 1) / KE;
  const int ri = wave / C::WN * 16 * TM, rj = wave % C::WN * 16 * TN;  // this wave's corner in the tile

  A sa;
  B sb;
  sa.begin(t.a, i0, k0, wave, lane);
  sb.begin(t.b, j0, k0, wave, lane);
  auto load = [&](int slot, int j, bool first = false) {  // load j of P of the next stage
    if (j < A::LOADS) sa.load(lds + slot * C::SLOT, j, left, wave, first);
    else sb.load(lds + slot * C::SLOT + A::BYTES, j - A::LOADS, left, wave, first);
    if (j == P - 1) {
      sa.base += sa.step;
      sb.base += sb.step;
      left -= KE;
    }
  };
  // the same for all of a lane's rows, which are 16 apart
  const int ca = A::past(t.a, i0 + (lane & 15)), cb = B::past(t.b, j0 + (lane & 15));
  const int pa = A::place(ri, lane, ca), pb = B::place(rj, lane, cb);
  const bool na = (lane >> 4) + ca > 3, nb = (lane >> 4) + cb > 3;  // in the next slot
  f4 fa[2][TM], fb[2][TN], acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
  auto fetch = [&](int s, int to, int f) {  // fragment f of TN + TM of stage s
    const int here = (s & 3) * C::SLOT, next = ((s + 1) & 3) * C::SLOT;
    if (f < TN) fb[to][f] = B::fragment(lds + (SEG && BD && nb ? next : here) + A::BYTES, pb, rj, f, lane);
    else fa[to][f - TN] = A::fragment(lds + (SEG && AD && na ? next : here), pa, ri, f - TN, lane);
  };
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int j = 0; j < P; ++j) load(s, j, s == 0 && k0 == 0);
  meet<(SEG ? 2 : 3) * P>();
#pragma unroll
  for (int f = 0; f < TM + TN; ++f) fetch(0, 0, f);
  // step s: stage s is in registers, s + 1 to s + 3 in LDS or on their way
  auto step = [&](int s, auto cur) {
    constexpr int C0 = decltype(cur)::value;
    meet<(SEG ? 1 : 2) * P>();  // stage s + 1 has landed (SEG: s + 2), and stage s has left its slot
    // rows of MFMAs with the loads of stage s + 4 and the reads of stage s + 1 between them, in this
    // order: left to itself the compiler puts the reads last, where the next step waits for them
    constexpr int BUSY = TM > 2 ? TM - 2 : 1, READS = (TM + TN + BUSY - 1) / BUSY, LOADS = (P + BUSY - 1) / BUSY;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = i * LOADS; j < (i + 1) * LOADS && j < P; ++j) load(s & 3, j);
#pragma unroll
      for (int f = i * READS; f < (i + 1) * READS && f < TM + TN; ++f) fetch(s + 1, C0 ^ 1, f);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mma<T>(fb[C0][j], fa[C0][i], acc[i][j]);
      } else {  // one after another on different sums
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[C0][j][q], fa[C0][i][q], acc[i][j], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int s = 0;
  for (; s + 1 < stages; s += 2) {
    step(s, std::integral_constant<int, 0>{});
    step(s + 1, std::integral_constant<int, 1>{});
  }
  if (s < stages) step(s, std::integral_constant<int, 0>{});
  meet<0>();

  if (tail && split == t.splits - 1) {
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[0][j] = rest<T, BD>(t.b, j0 + rj + 16 * j, whole, tail, lane);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const f4 a = rest<T, AD>(t.a, i0 + ri + 16 * i, whole, tail, lane);
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mma<T>(fb[0][j], a, acc[i][j]);
    }
  }
  emit<T, C>(t, acc, lds, split, i0, j0, ri, rj, wave, lane);
}

struct __attribute__((packed, aligned(4))) Words {
  uint32_t v[4];
};

template <int N, int I = 0, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, I + 1>(f);
  }
}

// The same for 16-bit operands DENSE in k whose rows begin inside words, which direct loads do not take: 16
// bytes a lane into registers, four stages ahead, and from there to LDS.  Rows past the matrix are its last one
// again (their sums are not written); the stage that is no whole one comes first, so that all others'
// loads need no guard.  Against padded copies it saves their launch and twice the operands' bytes:
// 203 x 5003 x 1535 fp16 24.0 -> 18.6 us (with 1536 and direct loads: 11.6), 64 x 1000 x 4001 bf16
// 17.1 -> 12.2 (six or eight stages ahead are no faster than four).
template <class T, class C>
__device__ __forceinline__ void loose_tile(const Product& t, int id) {
  using A = Side<T, true, C::BM, C::W>;
  using B = Side<T, true, C::BN, C::W>;
  constexpr int TM = C::TM, TN = C::TN, KE = A::KE, GR = GROUP<T>, P = A::LOADS + B::LOADS, D = 4;
  static_assert(sizeof(T) == 2, "rows of 32 bits begin at words");
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int split, ti, tj;
  tile_of(t, id, split, ti, tj);
  const int64_t i0 = (int64_t)ti * C::BM, j0 = (int64_t)tj * C::BN, k0 = split * t.span;
  const int all = (int)(t.k - k0 < t.span ? t.k - k0 : t.span), stages = (all + KE - 1) / KE;
  const int head = all - (stages - 1) * KE;  // elements of stage 0
  const int ri = wave / C::WN * 16 * TM, rj = wave % C::WN * 16 * TN;

  const T* from[P];  // this lane's group of load j in stage 1; its byte in a slot
  int to[P], group[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const bool is_a = j < A::LOADS;
    const int at = (wave * (is_a ? A::LOADS : B::LOADS) + (is_a ? j : j - A::LOADS)) * 1024 + lane * 16;
    const int row = at / 64, chunk = at / 16 % 4 ^ A::turn(row);
    const Operand& o = is_a ? t.a : t.b;
    const int64_t r = (is_a ? i0 : j0) + row;
    from[j] = (const T*)o.p + (r < o.rows ? r : o.rows - 1) * o.ld + k0 + head + chunk * GR;
    to[j] = (is_a ? 0 : A::BYTES) + at;
    group[j] = chunk * GR;
  }
  // Loads of 16 bytes that do not begin at a word take twice as long.  So a group of 16-bit elements that
  // begins inside a word is loaded from the element before it on (there is one from stage 1 on), and its last
  // element comes from the lane with the row's next group, which has it first in its own -- for the last
  // group of a stage that is the first one's lane, with the next stage; after the last stage `tail`.
  int odd[P], next[P];  // bytes of a word before the group; the lane with the next one
  uint32_t tail[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    odd[j] = (int)((uintptr_t)from[j] & 2);
    const int chunk = group[j] / GR, flip = chunk ^ (lane & 3);
    next[j] = ((lane & ~3) | ((chunk + 1 & 3) ^ flip)) * 4;
    tail[j] = reinterpret_cast<const uint16_t*>(from[j])[all - 1 - head - group[j]];
  }
  Words held[D][P];  // stage s in held[s % D]
  auto load = [&](int s, auto slot) {  // stage s >= 1 (past the last: that one again, which is not used)
    const int64_t c = (int64_t)((s < stages ? s : stages - 1) - 1) * KE;
#pragma unroll
    for (int j = 0; j < P; ++j)
      held[decltype(slot)::value][j] = *reinterpret_cast<const Words*>((const char*)(from[j] + c) - odd[j]);
  };
  auto put = [&](int s, auto slot) {
    constexpr int S = decltype(slot)::value;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const uint32_t* v = held[S][j].v;
      const uint32_t mine = group[j] == 0 ? held[(S + 1) % D][j].v[0] : v[0];
      uint32_t last = (uint32_t)__builtin_amdgcn_ds_bpermute(next[j], (int)mine);
      last = s == stages - 1 && group[j] == 3 * GR ? tail[j] : last;
      const uint4 w = {__builtin_amdgcn_alignbyte(v[1], v[0], odd[j]), __builtin_amdgcn_alignbyte(v[2], v[1], odd[j]),
                       __builtin_amdgcn_alignbyte(v[3], v[2], odd[j]), __builtin_amdgcn_alignbyte(last, v[3], odd[j])};
      *reinterpret_cast<uint4*>(lds + (s & 3) * C::SLOT + to[j]) = w;
    }
  };
  const int pa = A::place(ri, lane, 0), pb = B::place(rj, lane, 0);
  f4 fa[2][TM], fb[2][TN], acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
  auto fetch = [&](int slot, int set) {
    char* s = lds + slot * C::SLOT;
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[set][j] = B::fragment(s + A::BYTES, pb, rj, j, lane);
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[set][i] = A::fragment(s, pa, ri, i, lane);
  };
  if (stages > 1) static_for<D - 1>([&](auto j) { load(1 + j, std::integral_constant<int, 1 + j>{}); });
#pragma unroll
  for (int j = 0; j < P; ++j)
    *reinterpret_cast<Vec<T, GR>*>(lds + to[j]) = load_group(from[j] - head, head - group[j]);
  if (stages > 1) {
    load(D, std::integral_constant<int, 0>{});
    put(1, std::integral_constant<int, 1>{});
    load(D + 1, std::integral_constant<int, 1>{});
  }
  meet<63>();
  fetch(0, 0);
  // step s: stage s is in registers for the MFMAs, s + 1 in LDS, s + 2 to s + D + 1 on their way to `held`
  auto step = [&](int s, auto slot, auto set) {
    constexpr int S = decltype(set)::value;
    meet<63>();  // every wave has read stage s from LDS and written stage s + 1
    if (stages > 1) {
      put(s + 2, slot);
      load(s + 2 + D, slot);
    }
    fetch((s + 1) & 3, S ^ 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mma<T>(fb[S][j], fa[S][i], acc[i][j]);
  };
  for (int s = 0; s < stages; s += D)
    static_for<D>([&](auto j) {
      if (s + j < stages) step(s + j, std::integral_constant<int, (j + 2) % D>{}, std::integral_constant<int, j % 2>{});
    });
  meet<0>();
  emit<T, C>(t, acc, lds, split, i0, j0, ri, rj, wave, lane);
}

template <class T, class C, bool SEG>
__global__ __launch_bounds__(C::NT, C::EU) void linear_y_kernel(Product y) {
  tile<T, true, true, C, SEG>(y, blockIdx.x);
}

template <class T, class C>
__global__ __launch_bounds__(C::NT, C::EU) void linear_y_loose_kernel(Product y) {
  loose_tile<T, C>(y, blockIdx.x);
}

// db of a few rows of dy beside the products (no activation: dz is dy), 64 columns a workgroup: one launch less
// in front of them.
struct ColumnSums {
  const void* dy;
  void* db;
  int64_t ldy, m, n;
  int blocks;  // 0: not wanted
};
template <class T, class C>
__device__ __forceinline__ void column_sums(const ColumnSums& t, int id) {
  constexpr int SUBS = C::NT / 8, U = 4;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  float(*sh)[64] = reinterpret_cast<float(*)[64]>(lds);
  const int in = threadIdx.x & 7, sub = threadIdx.x >> 3;
  const int64_t c = (int64_t)id * 64 + in * 8, left = t.n - c;
  float sum[8] = {};
  if (left > 0)
    for (int64_t r = sub; r < t.m; r += U * SUBS) {
      Vec<T, 8> g[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {  // (past the last row: that one again, which is not used)
        const int64_t k = r + u * SUBS < t.m ? r + u * SUBS : t.m - 1;
        g[u] = load_eight((const T*)t.dy + k * t.ldy + c, left);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += r + u * SUBS < t.m ? (float)g[u].v[i] : 0.0f;
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) sh[sub][in * 8 + i] = sum[i];
  __syncthreads();
  const int64_t col = (int64_t)id * 64 + threadIdx.x;
  if (threadIdx.x < 64 && col < t.n) {
    float s = 0.0f;
#pragma unroll 8
    for (int k = 0; k < SUBS; ++k) s += sh[k][threadIdx.x];
    ((T*)t.db)[col] = (T)s;
  }
}

// dx = dz w and dw = dz^T x in one launch, so that the one's last tiles and the other's first share the
// chip.  The first's workgroups are counted up to a multiple of 8, which keeps the second's on the XCDs
// that tile_of takes them to be on; a product with no workgroups is not wanted.
template <class T, class C, bool SEG>
__global__ __launch_bounds__(C::NT, C::EU) void linear_grads_kernel(Product dx, Product dw, int dw_first,
                                                                    ColumnSums db) {
  if (const int rest = (int)gridDim.x - db.blocks; (int)blockIdx.x >= rest) {
    column_sums<T, C>(db, blockIdx.x - rest);
    return;
  }
  const int lead = ((dw_first ? dw.blocks : dx.blocks) + 7) & ~7, id = blockIdx.x;
  const bool is_dw = (id < lead) == (dw_first != 0);
  const int at = id < lead ? id : id - lead;
  if (at >= (is_dw ? dw.blocks : dx.blocks)) return;
  if (is_dw) tile<T, false, false, C, false>(dw, at);
  else tile<T, true, false, C, SEG>(dx, at);
}

// The splits' sums of up to two products, in their order, through the epilogue: 8 columns a thread.
struct Joins {
  Product p[2];
  int64_t blocks[2];  // 0: not split
};
template <class T>
__global__ __launch_bounds__(256) void matmul_join_kernel(Joins j) {
  const bool second = blockIdx.x >= j.blocks[0];
  const Product& t = second ? j.p[1] : j.p[0];
  const int64_t at = (blockIdx.x - (second ? j.blocks[0] : 0)) * 256 + threadIdx.x, per = t.ldp / 8;
  const int64_t row = at / per, col = at % per * 8;
  if (row >= t.m) return;
  float z[8], v[8], bias[8];
  load_n<float, 8>(z, t.part + row * t.ldp + col, 8);
#pragma unroll 8
  for (int s = 1; s < t.splits; ++s) {
    load_n<float, 8>(v, t.part + (s * t.m + row) * t.ldp + col, 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] += v[i];
  }
  bias8<T>(bias, t.e, col, t.n);
  finish8<T, false>(z, bias, t.e, row, col, t.n);
}

// ------------------------------------------------------------------------- few rows: the weight is all
// y for up to 16 rows of x, both operands dense in k.  A workgroup has 16 outputs; its waves share
// k between them in turns of 128 bytes a row, loads going straight into the fragments, and join
// their sums in LDS in a fixed order.  Bound by the weight's way from HBM: one row of 16384 x 16384
// bf16 in 109 us (4.9 TB/s), of 4096 x 4096 in 7.2; the launch's waves have most of it in flight at once.
// Rows past either matrix are its last one again: their sums are not written, and no load needs a guard but
// those of the last turn, where k ends inside it.
template <class T, int W>
__global__ __launch_bounds__(64 * W) void few_rows_kernel(const T* x, int64_t ldx, const T* w, int64_t ldw, int m,
                                                          int64_t n, int64_t k, Epilogue e) {
  constexpr int GR = GROUP<T>, TURN = 8 * GR, U = 4;  // elements of a row a turn; turns in flight
  __shared__ f4 sums[W][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15;
  const int64_t j0 = (int64_t)blockIdx.x * 16;
  const T* wp = w + (j0 + row < n ? j0 + row : n - 1) * ldw + (lane >> 4) * GR;
  const T* xp = x + (row < m ? row : m - 1) * ldx + (lane >> 4) * GR;
  f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  auto frag = [](const Vec<T, GR>& v) {
    f4 f;
    __builtin_memcpy(&f, &v, 16);
    return f;
  };
  const int64_t whole = k / TURN;
  for (int64_t t = wave; t < whole; t += W * U) {
    f4 fw[U][2], fx[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t c = (t + u * W < whole ? t + u * W : t) * TURN;  // (past the last: the first again, not used)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        fw[u][h] = frag(load_group(wp + c + h * 4 * GR, GR));
        fx[u][h] = frag(load_group(xp + c + h * 4 * GR, GR));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u * W < whole)
#pragma unroll
        for (int h = 0; h < 2; ++h) acc = mma<T>(fw[u][h], fx[u][h], acc);
  }
  if (whole * TURN < k && wave == whole % W)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t c = whole * TURN + h * 4 * GR, left = k - c - (lane >> 4) * GR;
      acc = mma<T>(frag(load_group(wp + c, left)), frag(load_group(xp + c, left)), acc);
    }
  sums[wave][lane] = acc;
  __syncthreads();
  // thread: row t / 2, 8 columns from 8 (t % 2); lane (c / 4) 16 + row of a wave has columns c ... c + 3
  const int t = threadIdx.x;
  if (t >= 2 * m) return;
  const int r = t >> 1, c = (t & 1) * 8;
  if (j0 + c >= n) return;
  float bias[8];
  bias8<T>(bias, e, j0 + c, n);
  float z[8] = {};
  for (int v = 0; v < W; ++v) {
    const f4 lo = sums[v][(c / 4) * 16 + r], hi = sums[v][(c / 4 + 1) * 16 + r];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] += lo[i], z[4 + i] += hi[i];
  }
  finish8<T, false>(z, bias, e, r, j0 + c, n);
}

// ------------------------------------------------------------------------------ rows on boundaries
// Matrices whose rows are no whole number of 16-byte groups, with rows that are, zeros behind them: what
// the tiled product's loads take.  Up to three in one launch.  Bound by memory (15 MB of fp16 in 7 us).
struct Padding {
  int count;
  struct One {
    const void* from;
    void* to;
    int64_t ld, rows, cols, per, blocks;  // per: groups of an output row
  } one[3];
};
template <class T>
__global__ __launch_bounds__(256) void pad_rows_kernel(Padding p) {
  constexpr int GR = GROUP<T>;
  int64_t block = blockIdx.x;
  int which = 0;
  while (which + 1 < p.count && block >= p.one[which].blocks) block -= p.one[which++].blocks;
  const Padding::One& o = p.one[which];
  const int64_t at = block * 256 + threadIdx.x, row = at / o.per, c = at % o.per * GR;
  if (row >= o.rows) return;
  store_group((T*)o.to + at * GR, load_group((const T*)o.from + row * o.ld + c, o.cols - c), GR);
}

template <class T>
__global__ __launch_bounds__(256) void zero_kernel(T* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = (T)0.0f;
}

// -------------------------------------------------------------------------- dz, and the bias's gradient
// dz = dy act'(z), and this strip of rows' sums of it: 64 lanes with 8 columns each, SUBS rows at a time,
// 4 of a lane's rows on their way together.  part: [strips][n], or where one strip is all of it db itself
// (both null: not wanted).  Without an activation dz is dy and is not written.  Bound by memory: 8192 x 8192 bf16
// of GELU in 81 us (dy, slopes and dz: 5.0 TB/s).
template <class T, int SUBS, int ACT>
__global__ __launch_bounds__(64 * SUBS) void linear_dz_kernel(const T* __restrict__ dy, int64_t ldy,
                                                              const void* __restrict__ slope, T* __restrict__ dz,
                                                              float* __restrict__ part, T* __restrict__ db, int64_t m,
                                                              int64_t n, int chunks, int64_t strip) {
  constexpr int U = 4;
  using Slope = std::conditional_t<ACT == QNN_ACT_RELU, uint8_t, std::conditional_t<sizeof(T) == 4, float, int16_t>>;
  __shared__ float sh[SUBS][64][9];
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6;
  const int64_t c = ((int64_t)(blockIdx.x % chunks) * 64 + lane) * 8, left = n - c;
  const int64_t s = blockIdx.x / chunks, r1 = (s + 1) * strip < m ? (s + 1) * strip : m;
  float sum[8] = {};
  auto rows = [&](auto whole) {
    const int64_t there = decltype(whole)::value ? 8 : left;
    for (int64_t r = s * strip + sub; r < r1; r += U * SUBS) {
      Vec<T, 8> g[U];
      Vec<Slope, 8> d[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {  // (past the last row: that one again, which is not used)
        const int64_t k = r + u * SUBS < r1 ? r + u * SUBS : r1 - 1;
        g[u] = load_eight(dy + k * ldy + c, there);
        if constexpr (ACT == QNN_ACT_RELU) d[u].v[0] = ((const uint8_t*)slope)[k * ((n + 7) / 8) + c / 8];
        else if constexpr (ACT == QNN_ACT_GELU) d[u] = load_eight((const Slope*)slope + k * n + c, there);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t k = r + u * SUBS;
        if (k >= r1) break;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = (float)g[u].v[i];
          if constexpr (ACT == QNN_ACT_RELU) v[i] = d[u].v[0] >> i & 1 ? v[i] : 0.0f;
          else if constexpr (ACT == QNN_ACT_GELU && sizeof(T) == 4) v[i] *= d[u].v[i];
          else if constexpr (ACT == QNN_ACT_GELU) v[i] *= slope_unpack<T>(d[u].v[i]);
          v[i] = (float)(T)v[i];  // db is the sum of dz as it is written
          sum[i] += v[i];
        }
        if (ACT != QNN_ACT_NONE) store_n<T, 8>(dz + k * n + c, v, there);
      }
    }
  };
  if ((blockIdx.x % chunks + 1) * 512 <= n) rows(std::true_type{});  // all of the workgroup's columns are there
  else if (left > 0) rows(std::false_type{});
  if (!part && !db) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sh[sub][lane][i] = sum[i];
  __syncthreads();
  if (sub == 0 && left > 0) {
#pragma unroll
    for (int k = 1; k < SUBS; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += sh[k][lane][i];
    if (db) store_n<T, 8>(db + c, sum, left);
    else store_n<float, 8>(part + s * n + c, sum, left);
  }
}

// db from the strips' sums: 64 columns a workgroup, 4 threads a column, which add up to JOINED strips one after another
// and then those sums
constexpr int JOINED = 256;
template <class T>
__global__ __launch_bounds__(256) void linear_db_kernel(const float* part, int strips, T* db, int64_t n) {
  __shared__ float sh[4][64];
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (c < n)
    for (int p0 = sub; p0 < strips; p0 += 4 * JOINED) {
      const int p1 = p0 + 4 * JOINED < strips ? p0 + 4 * JOINED : strips;
      float t = 0.0f;
#pragma unroll 8
      for (int p = p0; p < p1; p += 4) t += part[p * n + c];
      s += t;
    }
  sh[sub][lane] = s;
  __syncthreads();
  if (sub == 0 && c < n) db[c] = (T)(sh[0][lane] + sh[1][lane] + sh[2][lane] + sh[3][lane]);
}

// ---------------------------------------------------------------------------------------- host side
// The tiles.  Measured time of one stage of k for a workgroup that has its CU's turn, and of a workgroup's
// start and end, in us (stage: 16-bit types, fp32):
//   Big    256 x 256  0.72   -    10   (8 waves, one workgroup a CU)
//   Middle 128 x 128  0.26  0.97   5   (8 waves)
//   Half   128 x 64   0.19  0.50   4
//   Small  64 x 64    0.10  0.25   4   (0.13 alone on its CU: latency)
//   Low    32 x 64     -    0.21  1.5  (2 waves; 0.29 alone; fp32, whose MFMAs take Small longer than its bytes
//                                       where few of its rows are there: 32 x 4096 x 4096 backward 60 -> 45 us)
// A larger tile does more MFMAs for each byte it loads; a smaller one fills the chip with fewer rows.
using Big = Cfg<2, 4, 8, 4, 2>;
using Middle = Cfg<2, 4, 4, 2, 2>;
using Half = Cfg<2, 2, 4, 2, 2>;
using Small = Cfg<2, 2, 2, 2, 4>;
using Low = Cfg<1, 2, 2, 2, 4>;
struct Shape {
  int bm, bn, threads;
  float stage16, stage32, ends;
  float alone;   // what one by itself on a CU takes of its stage's time (16 bits, and Low)
  // what each takes where the first operand's rows, DENSE, begin off 64-byte boundaries (16 bits): at 16 bytes, elsewhere
  float off16, off;
};
constexpr Shape SHAPES[] = {{Big::BM, Big::BN, Big::NT, 0.72f, 0.0f, 10.0f, 1.0f, 1.0f, 1.0f},
                            {Middle::BM, Middle::BN, Middle::NT, 0.26f, 0.97f, 5.0f, 1.0f, 1.15f, 1.4f},
                            {Half::BM, Half::BN, Half::NT, 0.19f, 0.50f, 4.0f, 1.0f, 1.5f, 1.6f},
                            {Small::BM, Small::BN, Small::NT, 0.105f, 0.25f, 4.0f, 1.2f, 1.5f, 1.5f},
                            {Low::BM, Low::BN, Low::NT, 0.0f, 0.21f, 1.5f, 1.4f, 1.0f, 1.0f}};

int64_t up(int64_t a, int64_t b) { return cdiv(a, b) * b; }

struct Split {
  int n;         // splits of k
  int64_t span;  // elements of k in each
  int64_t ldp, bytes;
};
struct Size {
  int64_t m, n, k;
};
struct Plan {
  int shape;  // of SHAPES, for all products of the launch
  Split split[2];
  float us;      // what it is taken to cost
  bool loose;    // forward: rows as they are (Small) and not padded
};

constexpr int MAX_SPLITS = 64;

// The tile and the splits of k of the one or two products of a launch: the least of the times above for
// the busiest of 256 CUs; splits cost a second launch (5.5 us with its host time) and their sums' way
// through memory (at 4 TB/s).  Over the sizes that were swept (m, n 64 to 8192, k 64 to 8192) what it
// picks for one product is mostly within 10 % of the best pair, 20 % where the whole takes under 20 us.
// from: the first tile to consider; dense: the first operand is DENSE in k.
Plan plan_of(const Size* size, int count, int dtype, int from = 0, bool dense = true) {
  const int64_t ke = 64 / type_bytes(dtype);
  Plan best = {};
  float least = INFINITY;
  for (int c = dtype == QNN_F32 && from == 0 ? 1 : from; c < (dtype == QNN_F32 ? 5 : 4); ++c) {
    const Shape& h = SHAPES[c];
    const float stage = dtype == QNN_F32 ? h.stage32 : h.stage16, alone = dtype == QNN_F32 && c < 4 ? 1.0f : h.alone;
    const bool on = dtype == QNN_F32 || !dense || size[0].k % 32 == 0;
    const float off = on ? 1.0f : size[0].k % 8 == 0 ? h.off16 : h.off;
    int64_t tiles[2], stages[2];
    for (int i = 0; i < count; ++i) {
      tiles[i] = cdiv(size[i].m, h.bm) * cdiv(size[i].n, h.bn);
      stages[i] = cdiv(size[i].k, ke);
    }
    // a split for each product: none, or as many as give it so many workgroups
    constexpr int WANT[] = {0, 128, 256, 512, 1024}, WANTS = 5;
    for (int x = 0; x < (count > 1 ? WANTS * WANTS : WANTS); ++x) {
      int64_t each[2], n[2];
      float work = 0.0f, longest = 0.0f, shortest = INFINITY, us = 0.0f;
      int64_t blocks = 0, grid = 0;
      bool skip = false, split = false;
      for (int i = 0; i < count; ++i) {
        const int want = WANT[i ? x / WANTS : x % WANTS];
        int64_t s = want / tiles[i];
        if (s > stages[i] / 4) s = stages[i] / 4;
        if (s > MAX_SPLITS) s = MAX_SPLITS;
        skip = skip || (want > 0 && s < 2);
        if (s < 1) s = 1;
        each[i] = cdiv(stages[i], s);
        n[i] = cdiv(stages[i], each[i]);
        blocks += tiles[i] * n[i];
        grid += up(tiles[i] * n[i], 8);
        const float time = (float)each[i] * (i == 0 ? off : 1.0f);
        work += (float)(tiles[i] * n[i]) * time;
        longest = fmaxf(longest, time);
        shortest = fminf(shortest, time);
        split = split || n[i] > 1;
        if (n[i] > 1) us += (float)(n[i] * size[i].m * size[i].n) * 2e-6f;
      }
      if (skip) continue;
      const float turns = (float)cdiv(blocks, 256);
      // in whole turns of the longest, or evenly but for the end, where the shortest ones are
      const float most = fmaxf(longest * alone, fminf(turns * longest, work / 256.0f + 0.6f * shortest));
      us += most * stage + (0.6f * turns + 0.4f) * h.ends + (split ? 5.5f : 0.0f);
      if (grid >= (1LL << 32) / h.threads) us += 1e30f;  // more threads than a launch takes: refused if no tile has fewer
      if (us < least) {
        least = us;
        best.us = us;
        best.shape = c;
        for (int i = 0; i < count; ++i) {
          const int64_t ldp = up(size[i].n, 8);
          best.split[i] = {(int)n[i], each[i] * ke, ldp, n[i] > 1 ? up(n[i] * size[i].m * ldp * 4, 256) : 0};
        }
      }
    }
  }
  return best;
}

// Whether few_rows_kernel takes the forward product: up to 16 rows of x, but 2 where the rows' groups begin
// inside words (4 x 4096 x 4097 bf16 takes it 21 us and loose_tile 18, one row 16), and one where w of 16-bit
// types is large (2 x 8192 x 8191 bf16 72 us and 33 in tiles, 8 x 8192 x 8192 28 and 23; but 9 x 4096 x 4096
// 8.8 and 10.1).  "Large" is 20 million elements, between those two weights of 17 and 67; where between them the sides
// cross was not measured.
constexpr int FEW = 16;
bool is_few(int64_t m, int64_t n, int64_t k, int dtype) {
  if (dtype == QNN_F32) return m <= FEW;
  return n * k > 20000000 ? m == 1 : m <= (k % 2 ? 2 : FEW);
}

// The forward product's plan where rows (of 16 bits) begin inside words: padded (a launch and their bytes there
// and back, 4 us and 4 TB/s) or taken as they are, whichever is the less.  What loose_tile does besides takes
// it to 1.3 of the Small tile's estimate (203 x 5003 x 1535 fp16 19.0 us, padded 24.4; 407 x 7271 x 5585 bf16
// padded 100 us, as they are 131).
Plan plan_loose(const Size& z, int dtype) {
  Plan p = plan_of(&z, 1, dtype);
  const float padded = p.us + 4.0f + (float)((z.m + z.n) * z.k) * 1e-6f;
  Plan q = plan_of(&z, 1, dtype, 3);
  if (q.us * 1.3f > padded) return p;
  q.loose = true;
  return q;
}

// The plans of dx and dw: one launch, or two where tiles of one shape would cost well more (5 x 11562 x 7871 fp32,
// whose dx has 5 rows and dw 91 million elements: 203 us for 264).
struct Grads {
  Plan plan[2];  // one launch: the same one
  bool apart;
};
Grads plan_grads(int64_t m, int64_t n, int64_t k, int dtype) {
  // 3 us of host time, asked for twice a call: the last ones are kept
  struct Kept {
    int64_t m, n, k;
    int dtype;
    Grads g;
  };
  static thread_local Kept kept[32] = {};
  Kept& slot = kept[(m * 31 + n * 7 + k + dtype) & 31];
  if (slot.m == m && slot.n == n && slot.k == k && slot.dtype == dtype) return slot.g;
  const Size z[2] = {{m, k, n}, {n, k, m}};
  Plan both = plan_of(z, 2, dtype), dx = plan_of(z, 1, dtype), dw = plan_of(z + 1, 1, dtype, 0, false);
  const bool apart = dx.us + dw.us + 4.0f < 0.85f * both.us;
  if (apart) dw.split[1] = dw.split[0];
  slot = {m, n, k, dtype, apart ? Grads{{dx, dw}, true} : Grads{{both, both}, false}};
  return slot.g;
}

int check_grid(int64_t blocks, int threads) {
  QNN_REQUIRE(blocks < (1LL << 32) / threads, "too many rows for one call: a launch has fewer than 2^32 threads");
  return QNN_OK;
}

// The plan's product i of c = a b^T; its sums' scratch is taken from room.
int product_of(Product& p, const Plan& plan, int i, const Size& z, const Operand& a, const Operand& b, int tail,
               int edge, const Epilogue& e, char*& room) {
  const Shape& h = SHAPES[plan.shape];
  const Split& s = plan.split[i];
  const int64_t tm = cdiv(z.m, h.bm), tn = cdiv(z.n, h.bn);
  if (int rc = check_grid(up(tm * tn * s.n, 8), h.threads)) return rc;  // (up: as launch_grads counts the first's)
  if (s.n > 1)
    if (int rc = check_grid(2 * cdiv(z.m * (s.ldp / 8), 256), 256)) return rc;  // join, of two such products at most
  p = {a, b, z.m, z.n, z.k, (int)tm, (int)tn, s.n, (int)(tm * tn * s.n), s.span, tail, edge, (float*)room, s.ldp, e};
  room += s.bytes;
  return QNN_OK;
}

// More than 64 KiB of LDS: said once for each kernel and device.
int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& told) {
  if (bytes <= 65536) return QNN_OK;
  int dev = 0;
  if (hipError_t er = hipGetDevice(&dev); er != hipSuccess) return hip_check(er, "hipGetDevice");
  if (dev < 64 && (told.load(std::memory_order_relaxed) >> dev & 1)) return QNN_OK;
  if (hipError_t er = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes); er != hipSuccess)
    return hip_check(er, "hipFuncSetAttribute");
  if (dev < 64) told.fetch_or(1ull << dev, std::memory_order_relaxed);
  return QNN_OK;
}

template <class T, class F>
int with_cfg(int shape, F&& f) {
  if constexpr (sizeof(T) == 2)
    if (shape == 0) return f(Big{});
  if (shape == 1) return f(Middle{});
  if constexpr (sizeof(T) == 4)
    if (shape == 4) return f(Low{});
  if (shape == 2) return f(Half{});
  return f(Small{});
}

template <class T>
int join(const Product* p, int count, hipStream_t s) {
  Joins j = {};
  for (int i = 0; i < count; ++i) {
    j.p[i] = p[i];
    if (p[i].blocks > 0 && p[i].splits > 1) j.blocks[i] = cdiv(p[i].m * (p[i].ldp / 8), 256);
  }
  const int64_t blocks = j.blocks[0] + j.blocks[1];
  if (blocks == 0) return QNN_OK;
  hipLaunchKernelGGL((matmul_join_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, j);
  QNN_LAUNCH_CHECK("matmul_join_kernel");
  return QNN_OK;
}

// Whether the rows of an operand DENSE in k are taken between 64-byte boundaries (Side's SEG).
template <class T>
bool in_segments(const Operand& o) {
  const int64_t ld = o.ld * (int64_t)sizeof(T);
  return sizeof(T) == 2 && (uintptr_t)o.p % 16 == 0 && ld % 16 == 0 && ((uintptr_t)o.p % 64 != 0 || ld % 64 != 0);
}
// (Not in Small tiles: they are where latency counts, and SEG has one stage less on its way: 1000 x 1000 x 1000
// fp16 8.0 us in segments, 6.9 without, 24 x 12568 x 7368 bf16 49 and 34.)
template <class T, class C, class F>
int with_segments(bool seg, F&& f) {
  if constexpr (sizeof(T) == 2 && !std::is_same_v<C, Small>)
    if (seg) return f(std::true_type{});
  return f(std::false_type{});
}

template <class T>
int launch_y(int shape, const Product& y, hipStream_t s) {
  const bool seg = y.tail == 0 && (in_segments<T>(y.a) || in_segments<T>(y.b));
  const int rc = with_cfg<T>(shape, [&](auto cfg) {
    using C = decltype(cfg);
    return with_segments<T, C>(seg, [&](auto in) {
      constexpr bool SEG = decltype(in)::value;
      static std::atomic<uint64_t> told{0};
      if (int rc = allow_lds((const void*)&linear_y_kernel<T, C, SEG>, C::LDS, told)) return rc;
      hipLaunchKernelGGL((linear_y_kernel<T, C, SEG>), dim3((unsigned)y.blocks), dim3(C::NT), C::LDS, s, y);
      QNN_LAUNCH_CHECK("linear_y_kernel");
      return (int)QNN_OK;
    });
  });
  return rc ? rc : join<T>(&y, 1, s);
}

// p: dx, dw (no blocks: not wanted); the one whose workgroups take longer goes first
int first_of(const Product (&p)[2]) {
  return p[1].blocks > 0 && (p[0].blocks == 0 || p[1].span > p[0].span) ? 1 : 0;
}
int64_t grid_of(const Product (&p)[2], const ColumnSums& db) {
  const int first = first_of(p);
  return up(p[first].blocks, 8) + p[1 - first].blocks + db.blocks;
}
template <class T>
int launch_grads(int shape, const Product (&p)[2], const ColumnSums& db, hipStream_t s) {
  const bool seg = p[0].blocks > 0 && p[0].tail == 0 && in_segments<T>(p[0].a);
  const int first = first_of(p);
  const unsigned blocks = (unsigned)grid_of(p, db);
  const int rc = with_cfg<T>(shape, [&](auto cfg) {
    using C = decltype(cfg);
    return with_segments<T, C>(seg, [&](auto in) {
      constexpr bool SEG = decltype(in)::value;
      static std::atomic<uint64_t> told{0};
      if (int rc = allow_lds((const void*)&linear_grads_kernel<T, C, SEG>, C::LDS, told)) return rc;
      hipLaunchKernelGGL((linear_grads_kernel<T, C, SEG>), dim3(blocks), dim3(C::NT), C::LDS, s, p[0], p[1], first, db);
      QNN_LAUNCH_CHECK("linear_grads_kernel");
      return (int)QNN_OK;
    });
  });
  return rc ? rc : join<T>(p, 2, s);
}

// Whether direct loads take the matrix's rows as they are: their groups begin at words.  A row's last group may
// then reach past the row.  In an operand DENSE in k those last elements are left to Product::tail.  Else what
// such a group brings from the next row belongs to columns past the operand's end, which are not written, and
// only the last row, after which there is nothing, is left to the tail (so a row has to hold a group).
bool at_words(const void* p, int64_t ld, int64_t cols, int dtype) {
  return dtype == QNN_F32 || cols % 8 == 0 || ((uintptr_t)p % 4 == 0 && ld % 2 == 0 && cols % 2 == 0);
}

// A matrix as the tiled product takes it: itself, or (noted in `pads`) padded into `room`, of which it
// takes what it needs.
template <class T>
void on_boundaries(const void*& p, int64_t& ld, int64_t rows, int64_t cols, char*& room, Padding& pads) {
  const int64_t per = cdiv(cols, GROUP<T>);
  pads.one[pads.count++] = {p, room, ld, rows, cols, per, cdiv(rows * per, 256)};
  p = room;
  ld = per * GROUP<T>;
  room += up(rows * ld * (int64_t)sizeof(T), 256);
}
int64_t grid_of(const Padding& pads) {
  int64_t blocks = 0;
  for (int i = 0; i < pads.count; ++i) blocks += pads.one[i].blocks;
  return blocks;
}
template <class T>
int pad(const Padding& pads, hipStream_t s) {
  const int64_t blocks = grid_of(pads);
  if (blocks == 0) return QNN_OK;
  hipLaunchKernelGGL((pad_rows_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, pads);
  QNN_LAUNCH_CHECK("pad_rows_kernel");
  return QNN_OK;
}

// The room for that, whatever the matrix's row stride.
int64_t padded_bytes(int64_t rows, int64_t cols, int dtype) {
  const int64_t size = type_bytes(dtype), group = 16 / size;
  return cols % group == 0 ? 0 : up(rows * up(cols, group) * size, 256);
}
// where it is taken as it is if its rows begin at words
int64_t loose_bytes(int64_t rows, int64_t cols, int dtype) {
  return dtype == QNN_F32 && cols >= 4 ? 0 : padded_bytes(rows, cols, dtype);
}

int64_t fwd_bytes(int64_t m, int64_t n, int64_t k, int dtype) {
  if (m == 0 || is_few(m, n, k, dtype)) return 0;
  const Size z = {m, n, k};
  const int64_t words = plan_of(&z, 1, dtype).split[0].bytes;
  if (dtype == QNN_F32 || k % 8 == 0) return words;
  const Plan p = plan_loose(z, dtype);
  const int64_t loose = (p.loose ? 0 : padded_bytes(m, k, dtype) + padded_bytes(n, k, dtype)) + p.split[0].bytes;
  return words > loose ? words : loose;
}

// Strips of rows for dz's sums: one of 16 rows at a time for a few rows, which saves the launch that adds
// the strips up; else enough workgroups of 4 to fill the chip, and as many as leave a lane 512 rows to add.
struct Strips {
  int chunks;
  int64_t n, rows;  // strips, and rows in each
};
Strips strips_of(int64_t m, int64_t n) {
  const int64_t chunks = cdiv(n, 512);
  if (m <= 256) return {(int)chunks, m > 0, m};
  const int64_t want = cdiv(1024, chunks), most = cdiv(m, 16), s = want < most ? want : most;
  const int64_t rows = cdiv(m, s) < 4 * 512 ? cdiv(m, s) : 4 * 512;
  return {(int)chunks, cdiv(m, rows), rows};
}

int64_t bwd_bytes(int64_t m, int64_t n, int64_t k, int dtype) {
  if (m == 0) return 0;
  const Grads p = plan_grads(m, n, k, dtype);
  return padded_bytes(m, n, dtype) + loose_bytes(n, k, dtype) + loose_bytes(m, k, dtype) +
         up(strips_of(m, n).n * n * 4, 256) + p.plan[0].split[0].bytes + p.plan[1].split[1].bytes;
}

constexpr int64_t LONGEST = 1LL << 21;  // of a row stride: offsets inside a tile's rows are 32 bits

int check(int64_t m, int64_t n, int64_t k, int dtype) {
  QNN_REQUIRE(m >= 0 && m < (1LL << 31), "m: 0 to 2^31 - 1");
  QNN_REQUIRE(n >= 1 && n <= LONGEST, "n: 1 to 2^21");
  QNN_REQUIRE(k >= 1 && k <= LONGEST, "k: 1 to 2^21");
  QNN_REQUIRE(dtype == QNN_F32 || dtype == QNN_BF16 || dtype == QNN_F16, "dtype: QNN_F32, QNN_BF16 or QNN_F16");
  return QNN_OK;
}

// A matrix that is read: rows of whole 16-byte groups begin on 16-byte boundaries.
int check_matrix(const void* p, int64_t ld, int64_t rows, int64_t cols, int dtype) {
  QNN_REQUIRE(p, "null pointer");
  QNN_REQUIRE(ld >= cols && ld <= LONGEST, "a row stride is shorter than the row, or over 2^21");
  const int64_t size = type_bytes(dtype);
  QNN_REQUIRE(cols * size % 16 != 0 || (aligned16(p) && (rows <= 1 || ld * size % 16 == 0)),
              "rows of whole 16-byte groups have to begin on 16-byte boundaries");
  return QNN_OK;
}

}  // namespace
}  // namespace qnn

using namespace qnn;
using namespace qnn::fl;

extern "C" {

int qnn_linear_act_fwd_work(int64_t m, int64_t n, int64_t k, int dtype, int64_t* bytes) {
  if (int rc = check(m, n, k, dtype)) return rc;
  QNN_REQUIRE(bytes, "null pointer");
  *bytes = fwd_bytes(m, n, k, dtype);
  return QNN_OK;
}

int qnn_linear_act_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res,
                       int64_t ldr, void* y, void* slope, int64_t m, int64_t n, int64_t k, int dtype, int act,
                       void* work, int64_t work_bytes, qnn_stream_t stream) {
  if (int rc = check(m, n, k, dtype)) return rc;
  QNN_REQUIRE(act >= QNN_ACT_NONE && act <= QNN_ACT_GELU, "act: QNN_ACT_NONE, QNN_ACT_RELU or QNN_ACT_GELU");
  if (m == 0) return QNN_OK;
  if (int rc = check_matrix(x, ldx, m, k, dtype)) return rc;
  if (int rc = check_matrix(w, ldw, n, k, dtype)) return rc;
  QNN_REQUIRE(y, "null pointer");
  QNN_REQUIRE(!res || ldr >= n, "a row stride is shorter than the row");
  const int64_t need = fwd_bytes(m, n, k, dtype);
  QNN_REQUIRE(need == 0 || (work && work_bytes >= need && aligned16(work)),
              "work: at least what qnn_linear_act_fwd_work says, on a 16-byte boundary");
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipStream_t s = (hipStream_t)stream;
    const Epilogue e = {bias, res, ldr, y, slope, act};
    if (is_few(m, n, k, dtype)) {
      hipLaunchKernelGGL((few_rows_kernel<T, 16>), dim3((unsigned)cdiv(n, 16)), dim3(1024), 0, s, (const T*)x, ldx,
                         (const T*)w, ldw, (int)m, n, k, e);
      QNN_LAUNCH_CHECK("few_rows_kernel");
      return (int)QNN_OK;
    }
    char* room = (char*)work;
    const void *px = x, *pw = w;
    int64_t lx = ldx, lw = ldw;
    const Size z = {m, n, k};
    const bool words = at_words(x, ldx, k, dtype) && at_words(w, ldw, k, dtype);
    const Plan plan = words ? plan_of(&z, 1, dtype) : plan_loose(z, dtype);
    Padding pads = {};
    if (!words && !plan.loose) {
      on_boundaries<T>(px, lx, m, k, room, pads);
      on_boundaries<T>(pw, lw, n, k, room, pads);
    }
    Product p;
    const int tail = words ? (int)(k % GROUP<T>) : 0;
    if (int rc = product_of(p, plan, 0, z, {px, lx, m}, {pw, lw, n}, tail, 0, e, room)) return rc;
    if (int rc = check_grid(grid_of(pads), 256)) return rc;
    if (int rc = pad<T>(pads, s)) return rc;
    if constexpr (sizeof(T) == 2)
      if (plan.loose) {
        hipLaunchKernelGGL((linear_y_loose_kernel<T, Small>), dim3((unsigned)p.blocks), dim3(Small::NT), Small::LDS, s, p);
        QNN_LAUNCH_CHECK("linear_y_loose_kernel");
        return join<T>(&p, 1, s);
      }
    return launch_y<T>(plan.shape, p, s);
  });
}

int qnn_linear_act_plan(int64_t m, int64_t n, int64_t k, int dtype, int grads, int* tile_m, int* tile_n, int* splits) {
  if (int rc = check(m, n, k, dtype)) return rc;
  QNN_REQUIRE(m > 0, "m: at least 1");
  QNN_REQUIRE(tile_m && tile_n && splits, "null pointer");
  if (!grads && is_few(m, n, k, dtype)) {
    *tile_m = *tile_n = FEW;
    splits[0] = splits[1] = 1;
    return QNN_OK;
  }
  const Size y = {m, n, k};
  const bool words = dtype == QNN_F32 || k % 2 == 0;
  Plan p[2] = {};
  if (grads) {
    const Grads both = plan_grads(m, n, k, dtype);
    p[0] = both.plan[0], p[1] = both.plan[1];
  } else {
    p[0] = words ? plan_of(&y, 1, dtype) : plan_loose(y, dtype);
  }
  *tile_m = SHAPES[p[0].shape].bm;
  *tile_n = SHAPES[p[0].shape].bn;
  splits[0] = p[0].split[0].n;
  splits[1] = grads ? p[1].split[1].n : 1;
  return QNN_OK;
}

int qnn_linear_act_bwd_work(int64_t m, int64_t n, int64_t k, int dtype, int64_t* bytes) {
  if (int rc = check(m, n, k, dtype)) return rc;
  QNN_REQUIRE(bytes, "null pointer");
  *bytes = bwd_bytes(m, n, k, dtype);
  return QNN_OK;
}

int qnn_linear_act_bwd(const void* dy, int64_t ldy, const void* slope, const void* x, int64_t ldx, const void* w,
                       int64_t ldw, void* dz, void* dx, void* dw, void* db, int64_t m, int64_t n, int64_t k,
                       int dtype, int act, void* work, int64_t work_bytes, qnn_stream_t stream) {
  if (int rc = check(m, n, k, dtype)) return rc;
  QNN_REQUIRE(act >= QNN_ACT_NONE && act <= QNN_ACT_GELU, "act: QNN_ACT_NONE, QNN_ACT_RELU or QNN_ACT_GELU");
  if (m > 0) {
    if (int rc = check_matrix(dy, ldy, m, n, dtype)) return rc;
    if (dx)
      if (int rc = check_matrix(w, ldw, n, k, dtype)) return rc;
    if (dw)
      if (int rc = check_matrix(x, ldx, m, k, dtype)) return rc;
    QNN_REQUIRE(act == QNN_ACT_NONE || (slope && dz && aligned16(dz)),
                "an activation's gradient needs slope and dz, on a 16-byte boundary");
  }
  const int64_t need = bwd_bytes(m, n, k, dtype);
  QNN_REQUIRE(need == 0 || (work && work_bytes >= need && aligned16(work)),
              "work: at least what qnn_linear_act_bwd_work says, on a 16-byte boundary");
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipStream_t s = (hipStream_t)stream;
    char* room = (char*)work;
    const void* g = dy;
    int64_t ldg = ldy;
    const Strips st = strips_of(m, n);
    float* part = db && st.n > 1 ? (float*)room : nullptr;
    room += up(st.n * n * 4, 256);
    const Grads plan = m > 0 ? plan_grads(m, n, k, dtype) : Grads{};
    const bool db_beside = db && act == QNN_ACT_NONE && st.n == 1 && (dx || dw) && !plan.apart;
    if (act != QNN_ACT_NONE) {
      g = dz;
      ldg = n;
    }
    Padding pads = {};
    Product p[2] = {};
    const ColumnSums sums = {dy, db, ldy, m, n, db_beside ? (int)cdiv(n, 64) : 0};
    if (m > 0 && (dx || dw)) {
      const Size z[2] = {{m, k, n}, {n, k, m}};
      // w and x: taken as they are; g: too, where padding it costs more than dx' product loses by it (its rows' short
      // pieces then lie across the memory's lines: 1890 x 1470 x 11715 bf16 91 us padded, 107 as it is)
      constexpr int64_t group = GROUP<T>;
      const bool ww = at_words(w, ldw, k, dtype) && k >= group, xw = at_words(x, ldx, k, dtype) && k >= group;
      const bool pads_too = (dx && !ww) || (dw && !xw);
      const float loss = dx ? plan.plan[0].us * (dtype == QNN_F32 ? 0.04f : 0.1f) : 0.0f;
      const bool gw = at_words(g, ldg, n, dtype) && n >= group &&
                      (n % group == 0 || loss < (float)(m * n) * 0.5e-6f * sizeof(T) + (pads_too ? 0.0f : 4.0f));
      if (!gw) on_boundaries<T>(g, ldg, m, n, room, pads);
      const void *px = x, *pw = w;
      int64_t lx = ldx, lw = ldw;
      if (dx && !ww) on_boundaries<T>(pw, lw, n, k, room, pads);
      if (dw && !xw) on_boundaries<T>(px, lx, m, k, room, pads);
      const int over = gw ? (int)(n % group) : 0, all = (int)((n - 1) % group + 1);
      const int dx_edge = ww && k % group ? all : 0, dw_edge = over || (xw && k % group) ? 1 : 0;
      const Epilogue to_dx = {nullptr, nullptr, 0, dx, nullptr, QNN_ACT_NONE};
      const Epilogue to_dw = {nullptr, nullptr, 0, dw, nullptr, QNN_ACT_NONE};
      if (dx)
        if (int rc = product_of(p[0], plan.plan[0], 0, z[0], {g, ldg, m}, {pw, lw, k}, over, dx_edge, to_dx, room)) return rc;
      if (dw)
        if (int rc = product_of(p[1], plan.plan[1], 1, z[1], {g, ldg, n}, {px, lx, k}, 0, dw_edge, to_dw, room)) return rc;
      if (int rc = check_grid(grid_of(pads), 256)) return rc;
      if (!plan.apart)
        if (int rc = check_grid(grid_of(p, sums), SHAPES[plan.plan[0].shape].threads)) return rc;
    }
    // all of the call's launches can be made
    if (m > 0 && (act != QNN_ACT_NONE || (db && !db_beside))) {
      auto launch_dz = [&](auto subs, auto of) {
        constexpr int SUBS = decltype(subs)::value, ACT = decltype(of)::value;
        hipLaunchKernelGGL((linear_dz_kernel<T, SUBS, ACT>), dim3((unsigned)(st.n * st.chunks)), dim3(64 * SUBS), 0, s,
                           (const T*)dy, ldy, slope, (T*)dz, part, st.n == 1 ? (T*)db : nullptr, m, n, st.chunks,
                           st.rows);
      };
      auto with_subs = [&](auto of) {
        if (st.n == 1) launch_dz(std::integral_constant<int, 16>{}, of);
        else launch_dz(std::integral_constant<int, 4>{}, of);
      };
      if (act == QNN_ACT_RELU) with_subs(std::integral_constant<int, QNN_ACT_RELU>{});
      else if (act == QNN_ACT_GELU) with_subs(std::integral_constant<int, QNN_ACT_GELU>{});
      else with_subs(std::integral_constant<int, QNN_ACT_NONE>{});
      QNN_LAUNCH_CHECK("linear_dz_kernel");
    }
    if (db && st.n != 1) {  // (no strip: zeros)
      hipLaunchKernelGGL((linear_db_kernel<T>), dim3((unsigned)cdiv(n, 64)), dim3(256), 0, s, part, (int)st.n, (T*)db,
                         n);
      QNN_LAUNCH_CHECK("linear_db_kernel");
    }
    if (!dx && !dw) return (int)QNN_OK;
    if (m == 0) {  // an empty sum
      if (dw) {
        const int64_t blocks = cdiv(n * k, 256);
        hipLaunchKernelGGL((zero_kernel<T>), dim3((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20)), dim3(256), 0, s,
                           (T*)dw, n * k);
        QNN_LAUNCH_CHECK("zero_kernel");
      }
      return (int)QNN_OK;
    }
    if (int rc = pad<T>(pads, s)) return rc;
    if (!plan.apart) return launch_grads<T>(plan.plan[0].shape, p, sums, s);
    for (int i = 0; i < 2; ++i) {
      Product one[2] = {};
      one[i] = p[i];
      if (p[i].blocks > 0)
        if (int rc = launch_grads<T>(plan.plan[i].shape, one, {}, s)) return rc;
    }
    return (int)QNN_OK;
  });
}

}  // extern "C"
