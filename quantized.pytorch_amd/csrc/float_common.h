// Shared by the float operators (matmul.hip, layer_norm.hip, distill.hip): element types,
// 16-byte groups of a row, the activations.
#pragma once
#include <math.h>

#include <type_traits>

#include "qnn_internal.h"

namespace qnn {
namespace fl {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f4 __attribute__((ext_vector_type(4)));

// Elements of a type in one 16-byte load: the group in which rows are read and written.
template <class T>
constexpr int GROUP = 16 / (int)sizeof(T);

// N elements that may begin at any element: the type's alignment is all that the compiler assumes, and
// the card's loads and stores of 16 bytes take any address.
template <class T, int N>
struct Vec {
  T v[N];
};
struct __attribute__((packed, aligned(2))) Bytes16 {
  uint32_t v[4];
};

// The group of elements at p, raw: 16 bytes in one load if all of it is there, else those at or past
// `left` as 0.
template <class T>
__device__ __forceinline__ Vec<T, GROUP<T>> load_group(const T* p, int64_t left) {
  Vec<T, GROUP<T>> o;
  if (left >= GROUP<T>) {
    const Bytes16 t = *reinterpret_cast<const Bytes16*>(p);
    __builtin_memcpy(&o, &t, 16);
  } else {
#pragma unroll
    for (int i = 0; i < GROUP<T>; ++i) o.v[i] = i < left ? p[i] : (T)0.0f;
  }
  return o;
}

// The same of 8 elements: one group of a 16-bit type, two of fp32.
template <class T>
__device__ __forceinline__ Vec<T, 8> load_eight(const T* p, int64_t left) {
  Vec<T, 8> o;
#pragma unroll
  for (int g = 0; g < 8 / GROUP<T>; ++g) {
    const Vec<T, GROUP<T>> t = load_group(p + g * GROUP<T>, left - g * GROUP<T>);
#pragma unroll
    for (int i = 0; i < GROUP<T>; ++i) o.v[g * GROUP<T> + i] = t.v[i];
  }
  return o;
}

template <class T>
__device__ __forceinline__ void store_group(T* p, const Vec<T, GROUP<T>>& o, int64_t left) {
  if (left >= GROUP<T>) {
    Bytes16 t;
    __builtin_memcpy(&t, &o, 16);
    *reinterpret_cast<Bytes16*>(p) = t;
  } else {
#pragma unroll
    for (int i = 0; i < GROUP<T>; ++i)
      if (i < left) p[i] = o.v[i];
  }
}

// N consecutive elements at p as floats, those at or past `left` as 0 (N a whole number of groups).
template <class T, int N>
__device__ __forceinline__ void load_n(float (&o)[N], const T* p, int64_t left) {
  constexpr int G = GROUP<T>;
  if (left >= N) {
#pragma unroll
    for (int g = 0; g < N / G; ++g) {
      const Vec<T, G> t = load_group(p + g * G, G);
#pragma unroll
      for (int i = 0; i < G; ++i) o[g * G + i] = (float)t.v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = i < left ? (float)p[i] : 0.0f;
  }
}

template <class T, int N>
__device__ __forceinline__ void store_n(T* p, const float (&o)[N], int64_t left) {
  constexpr int G = GROUP<T>;
  if (left >= N) {
#pragma unroll
    for (int g = 0; g < N / G; ++g) {
      Vec<T, G> t;
#pragma unroll
      for (int i = 0; i < G; ++i) t.v[i] = (T)o[g * G + i];
      store_group(p + g * G, t, G);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = (T)o[i];
  }
}

// GELU z Phi(z) and its derivative Phi(z) + z phi(z) together, from one exponential.  With a = |z|, the
// tail Phi(-a) = erfc(a / sqrt 2) / 2 = e^(-a^2 / 2) t P(t), t = 1 / (1 + c a), P fitted here to the
// scaled complement e^(u^2) erfc(u), so that the far negative side keeps its relative precision too:
//   y = max(z, 0) - a tail,  slope = d below 0 and 1 - d above, d = tail - a phi(a).
// For results of 16 bits P has degree 5 (relative error 1.1e-6 to |z| = 6.5, past which y is under 1e-9;
// fp16's rounding is 4.9e-4 of the value); for fp32 degree 9 (4.1e-8 to |z| = 20) and a^2 with its rounding error.
// The two products with a take it clamped, which gives the limits at the infinities; a NaN stays one.
template <bool FP32>
__device__ __forceinline__ void gelu_f(float z, float& y, float& slope) {
  const float s = z * z, a = __builtin_amdgcn_fmed3f(fabsf(z), 0.0f, 20.0f);
  float e, p, t;
  if constexpr (FP32) {
    const float low = fabsf(z) < 20.0f ? fmaf(z, z, -s) : 0.0f;  // (inf - inf; e is 0 in 32 bits long before)
    e = __builtin_amdgcn_exp2f(-0.72134752044448170f * s) * fmaf(-0.5f, low, 1.0f);
    t = __builtin_amdgcn_rcpf(fmaf(0.36f * 0.70710678118654752f, fabsf(z), 1.0f));
    p = 0.5f * 0.03754199f;
    p = fmaf(p, t, 0.5f * -0.14138553f);
    p = fmaf(p, t, 0.5f * 0.14222577f);
    p = fmaf(p, t, 0.5f * -0.02727648f);
    p = fmaf(p, t, 0.5f * 0.10558839f);
    p = fmaf(p, t, 0.5f * 0.12331503f);
    p = fmaf(p, t, 0.5f * 0.16381756f);
    p = fmaf(p, t, 0.5f * 0.18995832f);
    p = fmaf(p, t, 0.5f * 0.20310671f);
    p = fmaf(p, t, 0.5f * 0.20310828f);
  } else {
    e = __builtin_amdgcn_exp2f(-0.72134752044448170f * s);
    t = __builtin_amdgcn_rcpf(fmaf(0.42f * 0.70710678118654752f, fabsf(z), 1.0f));
    p = 0.5f * -0.171326101f;
    p = fmaf(p, t, 0.5f * 0.503957272f);
    p = fmaf(p, t, 0.5f * -0.116222054f);
    p = fmaf(p, t, 0.5f * 0.331291884f);
    p = fmaf(p, t, 0.5f * 0.213374555f);
    p = fmaf(p, t, 0.5f * 0.23892343f);
  }
  const float tail = p * (t * e);
  y = fmaf(-a, tail, z < 0.0f ? 0.0f : z);
  const float d = fmaf(a * -0.39894228040143268f, e, tail);
  slope = z < 0.0f ? d : 1.0f - d;
}

// The derivative d of GELU between the passes, for 16-bit types, in 16 bits.  It lies in [-0.13, 1.13] and goes to 0 with
// z (-7e-6 at -5), where its relative error has to stay small too: the gradient of z is dy d, rounded to the type.
//
// bf16: d 2^15 in fp16.  Off by 2^-11 of d, an eighth of bf16's half step (2^-8), down to 2^-29, and by 2^-40 below that.
//
// fp16, whose half step (2^-11) that would double: s = sign(d) |d|^(1/4) in fixed point of 1 / 40192 around 24096 (0: a
// NaN).  Off by 1.25e-5 in s, by 5e-5 |d|^(3/4) in d: a tenth of the half step near 1, the whole of it at 1e-4
// (z = -4.4), eight of them at z = -6, where dy d under 2^9 is subnormal in fp16 itself.  Without branches, 11 and 7
// operations: dz of 300000 x 64 94 us, where a code of two ranges, fixed point and floating, made it 130.
constexpr float SLOPE_STEPS = 40192.0f, SLOPE_ZERO = 24096.0f;
template <class T>
__device__ __forceinline__ int16_t slope_pack(float d) {
  if constexpr (std::is_same_v<T, bf16>) return __builtin_bit_cast(int16_t, (f16)(d * 32768.0f));
  const float s = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(fabsf(d)));
  return (int16_t)(uint16_t)(uint32_t)fmaf(copysignf(s, d), SLOPE_STEPS, SLOPE_ZERO + 0.5f);  // (of a NaN: 0)
}
template <class T>
__device__ __forceinline__ float slope_unpack(int16_t q) {
  if constexpr (std::is_same_v<T, bf16>) return (float)__builtin_bit_cast(f16, q) * (1.0f / 32768.0f);
  const int v = (uint16_t)q;
  const float s = ((float)v - SLOPE_ZERO) * (1.0f / SLOPE_STEPS), t = s * s;
  return v == 0 ? __builtin_nanf("") : copysignf(t * t, s);
}

template <class F>
static inline int with_type(int dtype, F&& f) {
  switch (dtype) {
    case QNN_F32: return f((float)0);
    case QNN_BF16: return f((bf16)0.0f);
    case QNN_F16: return f((f16)0.0f);
  }
  return arg_error("dtype: QNN_F32, QNN_BF16 or QNN_F16");
}

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static inline int type_bytes(int dtype) { return dtype == QNN_F32 ? 4 : 2; }

}  // namespace fl
}  // namespace qnn
