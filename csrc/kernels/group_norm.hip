// group_norm.hip — group norm with its affine map and an activation, channels last (gfx950).
//
//   mu[n,g]  = mean over pixels p and the channels c of group g of x[n,p,c]
//   var[n,g] = mean of (x - mu)^2
//   y[n,p,c] = act((x - mu) / sqrt(var + eps) * weight[c] + bias[c])
//
// Statistics in fp32 from centred values (a second look at the data once the mean is known:
// E[x^2] - mu^2 loses all digits where the mean is large against the spread).
#include "activation.h"

namespace dml {
namespace gn {

template <class T>
__global__ __launch_bounds__(256) void group_norm_simple(DmlGroupNormArgs a) {
  __shared__ float part[4];
  const int g = blockIdx.x % a.G, n = blockIdx.x / a.G;
  const int cg = a.C / a.G, c0 = g * cg;
  const long count = (long)a.HW * cg;
  const T* x = (const T*)a.x + n * a.xn + c0;
  T* y = (T*)a.y + n * a.yn + c0;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  auto total = [&](float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if (lane == 0) part[wid] = v;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
  };
  float s = 0.f;
  for (long i = threadIdx.x; i < count; i += 256) s += to_f32(x[(i / cg) * a.ldx + i % cg]);
  const float mu = total(s) / (float)count;
  s = 0.f;
  for (long i = threadIdx.x; i < count; i += 256) {
    const float d = to_f32(x[(i / cg) * a.ldx + i % cg]) - mu;
    s += d * d;
  }
  const float rs = 1.f / sqrtf(total(s) / (float)count + a.eps);
  for (long i = threadIdx.x; i < count; i += 256) {
    const int c = (int)(i % cg);
    float v = (to_f32(x[(i / cg) * a.ldx + c]) - mu) * rs;
    v = v * (a.weight ? a.weight[c0 + c] : 1.f) + (a.bias ? a.bias[c0 + c] : 0.f);
    y[(i / cg) * a.ldy + c] = (T)activate(v, a.act);
  }
}

template <class T>
static int launch(const DmlGroupNormArgs* a, hipStream_t s) {
  hipLaunchKernelGGL(group_norm_simple<T>, dim3((unsigned)((long)a->N * a->G)), dim3(256), 0, s, *a);
  DML_CHECK_LAUNCH();
  return 0;
}

}  // namespace gn
}  // namespace dml

extern "C" int dml_group_norm(const DmlGroupNormArgs* a, hipStream_t s) {
  if (!a || a->N < 0 || a->HW < 0 || a->C < 1 || a->G < 1 || a->C % a->G) {
    dml_set_error("dml_group_norm: need N, HW >= 0 and a channel count that the groups divide");
    return -1;
  }
  if (a->dtype < DML_BF16 || a->dtype > DML_F32 || a->act < 0 || a->act >= DML_ACT_COUNT) {
    dml_set_error("dml_group_norm: dtype or act out of range");
    return -1;
  }
  if (a->N == 0 || a->HW == 0) return 0;
  if (!a->x || !a->y || a->ldx < 0 || a->ldy < a->C || (long)a->N * a->G > 0x7fffffffl) {
    dml_set_error("dml_group_norm: null tensor, a pixel stride out of range, or over 2^31 (sample, group) pairs");
    return -1;
  }
  switch (a->dtype) {
    case DML_BF16: return dml::gn::launch<bf16>(a, s);
    case DML_F16: return dml::gn::launch<dml::f16>(a, s);
    default: return dml::gn::launch<float>(a, s);
  }
}
