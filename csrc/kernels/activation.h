// activation.h — what group_norm.hip and product.hip share: the pointwise functions behind a
// norm or a product, and loads / stores of one element of a run-time or template type.
#pragma once
#include "common.h"
#include "dml.h"

namespace dml {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// One value through the activation `act` (DML_ACT_*), in fp32. NaN stays NaN (ReLU included:
// a comparison, not fmaxf).
//   silu(v)      = v / (1 + e^-v)
//   gelu(v)      = v Phi(v) = v/2 erfc(-v / sqrt 2)
//   gelu_tanh(v) = v/2 (1 + tanh u) = v / (1 + e^-2u),  u = sqrt(2/pi) (v + 0.044715 v^3)
__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {  // wave-uniform
    case DML_ACT_RELU: return v < 0.f ? 0.f : v;
    case DML_ACT_SILU: return v / (1.f + expf(-v));
    case DML_ACT_GELU: return 0.5f * v * erfcf(v * -0.70710678118654752f);
    case DML_ACT_GELU_TANH: return v / (1.f + expf(-1.5957691216057308f * (v + 0.044715f * v * v * v)));
    default: return v;
  }
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(f16 v) { return (float)v; }

}  // namespace dml
