// activation.h — what group_norm.hip and product.hip share: the pointwise functions behind a
// norm or a product, and 16-byte vectors of the element types.
#pragma once
#include "common.h"
#include "dml.h"

namespace dml {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// v Phi(v) with Phi(v) = 1/2 erfc(-v / sqrt 2). With z = |v| / sqrt 2 and t = 1 / (1 + 0.3275911 z),
// Abramowitz & Stegun 7.1.26: erfc(z) = t (a1 + t (a2 + ... + t a5)) e^-z^2, off by at most 1.5e-7,
// so gelu by at most 7.5e-8 |v|: a 32-bit result keeps 23 bits of v.
__device__ __forceinline__ float gelu_erf(float v) {
  const float z = fabsf(v) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * z);
  const float p = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  const float tail = 0.5f * p * __builtin_amdgcn_exp2f(-1.4426950408889634f * z * z);  // Phi(-|v|)
  return v * (v < 0.f ? tail : 1.f - tail);
}

// v / (1 + e^-(a v + b v^3))
__device__ __forceinline__ float swish(float v, float a, float b) {
  const float u = v * (a + b * v * v);
  return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * u));
}

// N values through the activation `act` (DML_ACT_*, wave-uniform), in fp32. NaN stays NaN (ReLU
// included: a comparison, not fmaxf).
//   silu(v)      = v / (1 + e^-v)
//   gelu(v)      = v Phi(v)
//   gelu_tanh(v) = v/2 (1 + tanh u) = v / (1 + e^-2u),  u = sqrt(2/pi) (v + 0.044715 v^3)
// exp and 1/x are the hardware's, good to a step or two: 1e-7 relative each.
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  if (act == DML_ACT_NONE) return;
  if (act == DML_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];
  } else if (act == DML_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = gelu_erf(v[j]);
  } else {
    const float a = act == DML_ACT_SILU ? 1.f : 1.5957691216057308f;
    const float b = act == DML_ACT_SILU ? 0.f : 0.07135481627159f;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = swish(v[j], a, b);
  }
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(f16 v) { return (float)v; }

// 16 bytes of T, loaded and stored at any element alignment (the hardware splits what needs it).
template <class T>
struct Vec16 {
  static constexpr int N = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(N)));
  vec v;
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(&v, p, 16); }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, &v, 16); }
  __device__ __forceinline__ void load(const T* p, int n) {  // the first n; 0 behind them
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < n ? p[j] : (T)0.f;
  }
  __device__ __forceinline__ void store(T* p, int n) const {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) p[j] = v[j];
  }
  __device__ __forceinline__ void get(float (&f)[N]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = to_f32(v[j]);
  }
  __device__ __forceinline__ void set(const float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)f[j];
  }
};

}  // namespace dml
