// activation.h — what group_norm.hip and product.hip share: the pointwise functions behind a
// norm or a product, and 16-byte vectors of the element types.
#pragma once
#include "common.h"
#include "dml.h"
#include <cmath>
#include <type_traits>

namespace dml {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// v Phi(v) = max(v, 0) - |v| Phi(-|v|), Phi the normal distribution, with Phi(-a) = 2^P(a): P of degree 8 fits
// log2 Phi(-a) on [0, 6] (least maximum of the error times Phi(-a); P(0) = -1 exactly), and falls without bound
// behind it. gelu comes out within 1e-7 |v|, two thirds of the instructions of a rational form of erfc. The bound on a keeps
// infinity times 0 out of it.
__device__ __forceinline__ float gelu_erf(float v) {
  const float a = fminf(fabsf(v), 64.f);
  float p = -2.8349129479465773e-06f;
  p = p * a + 3.93776863347739e-05f;
  p = p * a - 1.861801720224321e-04f;
  p = p * a - 1.3693659275304526e-04f;
  p = p * a + 7.0634204894304276e-03f;
  p = p * a - 5.2496179938316345e-02f;
  p = p * a - 0.4592081904411316f;
  p = p * a - 1.1511051654815674f;
  p = p * a - 1.f;
  return 0.5f * (v + fabsf(v)) - a * __builtin_amdgcn_exp2f(p);
}

// v / (1 + 2^-(a v + b v^3))
__device__ __forceinline__ float swish(float v, float a, float b) {
  return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * (-a - b * v * v)));
}

// The activations (DML_ACT_*) as three kinds of code, each with two parameters:
//   none, relu       max(v, a), a = -infinity or 0 (by comparison: NaN stays NaN)
//   silu, gelu_tanh  v / (1 + 2^-(a v + b v^3)): a = 1 / ln 2, b the least normal number for silu (0 times infinity
//                    would be NaN; b v^2 is below a's rounding up to |v| = 10^15, where 2^-av is long 0 or infinite);
//                    gelu_tanh(v) = v/2 (1 + tanh u) = v / (1 + e^-2u), u = sqrt(2/pi) (v + 0.044715 v^3)
//   gelu             v Phi(v)
// exp and 1/x are the hardware's, good to a step or two: 1e-7 relative each.
enum { kClamp, kSwish, kErf };
struct Act {
  float a, b;
  template <int KIND>
  __device__ __forceinline__ float run(float v) const {
    return KIND == kClamp ? (v < a ? a : v) : KIND == kSwish ? swish(v, a, b) : gelu_erf(v);
  }
};
__device__ __forceinline__ Act act_parameters(int act) {
  return act <= DML_ACT_RELU ? Act{act == DML_ACT_RELU ? 0.f : -INFINITY, 0.f}
         : act == DML_ACT_GELU_TANH ? Act{2.3022081981f, 0.102943239580f} : Act{1.4426950409f, 0x1p-126f};
}
// one value, of a wave-uniform `act`
__device__ __forceinline__ float activate(float v, int act) {
  const Act p = act_parameters(act);
  return act <= DML_ACT_RELU ? p.run<kClamp>(v) : act == DML_ACT_GELU ? p.run<kErf>(v) : p.run<kSwish>(v);
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
  typedef vec __attribute__((aligned(sizeof(T)))) any;
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(&v, p, 16); }
  __device__ __forceinline__ void load_once(const T* p) { v = __builtin_nontemporal_load((const any*)p); }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, &v, 16); }
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
