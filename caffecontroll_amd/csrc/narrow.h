// Element types of the vocabulary operators (embedding, vocabulary loss, distillation loss): fp32, and bf16 in
// memory with every sum in fp32.  16-byte vectors of either, at any element alignment (gfx950 loads and stores
// dwords at every byte address), with a scalar tail for widths that are no whole number of vectors.
#pragma once
#include "cct_common.h"

namespace cct {

typedef __bf16 bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <class T>
struct Num;
template <>
struct Num<float> {
  static constexpr int DTYPE = CCT_F32;
  static constexpr int V = 4;  // elements of a 16-byte vector
  typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
  static constexpr const char *NAME = "float";
};
template <>
struct Num<bf16> {
  static constexpr int DTYPE = CCT_BF16;
  static constexpr int V = 8;
  typedef bf16 vec __attribute__((ext_vector_type(8), aligned(2)));
  static constexpr const char *NAME = "bf16";
};

inline size_t dtype_bytes(int dtype) { return dtype == CCT_BF16 ? 2 : 4; }

// Elements [col, col + V) of a row of `width` elements as floats; those past the end read as zero.
template <class T>
__device__ __forceinline__ void load_vec(float (&f)[Num<T>::V], const T *__restrict__ row, int col, int width) {
  constexpr int V = Num<T>::V;
  if (col + V <= width) {
    const typename Num<T>::vec v = *reinterpret_cast<const typename Num<T>::vec *>(row + col);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = col + i < width ? (float)row[col + i] : 0.0f;
  }
}

// One rounding per element, to nearest even (v_cvt_pk_bf16_f32).
template <class T>
__device__ __forceinline__ void store_vec(T *__restrict__ row, const float (&f)[Num<T>::V], int col, int width) {
  constexpr int V = Num<T>::V;
  if (col + V <= width) {
    typename Num<T>::vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)f[i];
    *reinterpret_cast<typename Num<T>::vec *>(row + col) = v;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (col + i < width) row[col + i] = (T)f[i];
  }
}

// The same past the caches, for results that are large and not read again soon.
template <class T>
__device__ __forceinline__ void store_vec_stream(T *__restrict__ row, const float (&f)[Num<T>::V], int col, int width) {
  constexpr int V = Num<T>::V;
  if (col + V <= width) {
    typename Num<T>::vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)f[i];
    __builtin_nontemporal_store(v, reinterpret_cast<typename Num<T>::vec *>(row + col));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (col + i < width) row[col + i] = (T)f[i];
  }
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Running maximum and sum of a softmax: m the largest value seen so far, s the sum of 2^((v - m) * scale2) with
// scale2 = log2(e) / temperature.  The maximum is kept in the values' own units and subtracted before the scale is applied, so
// that rows at the type's lowest value do not overflow.  An empty or fully masked (-inf) part has m = -inf, s = 0 and
// joins another part without changing it; NaN values make the sum NaN.
struct SoftStat {
  float m, s;
};
__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ SoftStat join(SoftStat a, SoftStat b, float scale2) {
  const float m = fmaxf(a.m, b.m);
  // the side that holds the maximum keeps its sum (with both at -inf: 0, or NaN if there was one)
  const float fa = a.m == m ? 1.0f : exp2_fast((a.m - m) * scale2), fb = b.m == m ? 1.0f : exp2_fast((b.m - m) * scale2);
  return SoftStat{m, a.s * fa + b.s * fb};
}
__device__ __forceinline__ SoftStat shfl_xor_join(SoftStat a, int mask, float scale2) {
  return join(a, SoftStat{__shfl_xor(a.m, mask, 64), __shfl_xor(a.s, mask, 64)}, scale2);
}
// log of the sum of exp(v / T); inv_t = 1 / T
__device__ __forceinline__ float log_sum(SoftStat a, float inv_t) {
  return __builtin_fmaf(a.m, inv_t, __builtin_log2f(a.s) * kLn2);
}
// log_sum less v / T, without the rounding of log_sum
__device__ __forceinline__ float label_loss(SoftStat a, float v, float inv_t) {
  return __builtin_fmaf(a.m - v, inv_t, __builtin_log2f(a.s) * kLn2);
}

}  // namespace cct
