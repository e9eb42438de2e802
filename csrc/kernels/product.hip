// product.hip — matrix products with a fused epilogue, over one weight or over a weight per
// group of rows (gfx950).
//
//   y[m,:] = act(x[m,:] . W_e^T + b_e) + r[m,:]       (act_last: act(x . W_e^T + b_e + r))
//
// with e the group that row m belongs to: group e owns the rows [ends[e-1], ends[e]) (one
// group of all M rows without `ends`). Products and sums in fp32, one rounding at the store.
// The ends are read on the device and clamped to an ascending sequence within [0, M], so no
// content of theirs reaches past a tensor.
#include "activation.h"
#include <climits>

namespace dml {
namespace prod {

// Where a row tile lies: group e, rows [row, row + rows) of the tensors; rows = 0: none.
struct Place {
  int e, row, rows;
};

__device__ __forceinline__ int ends_at(const DmlProductArgs& a, int e) {
  const long v = a.ends64 ? ((const long*)a.ends)[e] : (long)((const int*)a.ends)[e];
  return (int)(v < 0 ? 0 : v > a.M ? a.M : v);
}

// Row tile t of the sequence "every group's rows cut into tiles of BM, the groups in order
// (then, with a.fill, the rows behind the last group as group E)". Each wave scans the ends
// 64 at a time: a running maximum makes them ascend, a prefix sum of the groups' tile counts
// finds the group that owns tile t. The result is wave-uniform.
template <int BM>
__device__ __forceinline__ Place locate(const DmlProductArgs& a, int t) {
  if (!a.ends) return {0, t * BM, min(BM, a.M - t * BM)};
  const int lane = threadIdx.x & 63;
  int start = 0, before = 0;  // first row / first tile of this chunk's first group
  for (int base = 0; base < a.E + a.fill; base += 64) {
    const int e = base + lane;
    int end = e < a.E ? ends_at(a, e) : e == a.E && a.fill ? a.M : 0;
    end = max(end, start);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(end, o, 64);
      if (lane >= o) end = max(end, v);
    }
    int beg = __shfl_up(end, 1, 64);
    if (lane == 0) beg = start;
    const int tiles = (end - beg + BM - 1) / BM;
    int upto = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    upto += before;
    const unsigned long long past = __ballot(upto > t);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int first = __shfl(upto - tiles, l, 64), b = __shfl(beg, l, 64), n = __shfl(end, l, 64);
      const int row = b + (t - first) * BM;
      return {base + l, row, min(BM, n - row)};
    }
    start = __shfl(end, 63, 64);
    before = __shfl(upto, 63, 64);
  }
  return {0, 0, 0};
}

template <class T> struct Mfma;
template <> struct Mfma<bf16> {
  typedef bf16x8 vec;
  __device__ __forceinline__ static f32x4 run(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mfma<f16> {
  typedef f16x8 vec;
  __device__ __forceinline__ static f32x4 run(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// One output element: row `row`, column `col` of group e.
template <class T>
__device__ __forceinline__ void finish(const DmlProductArgs& a, int e, int row, int col, float v) {
  if (a.bias) v += a.bias[e * a.bias_group + col];
  float r = 0.f;
  if (a.res)
    r = a.out_f32 ? ((const float*)a.res)[row * a.ldr + col] : to_f32(((const T*)a.res)[row * a.ldr + col]);
  if (a.act_last) v += r;
  v = activate(v, a.act);
  if (!a.act_last) v += r;
  if (a.out_f32) ((float*)a.y)[row * a.ldy + col] = v;
  else ((T*)a.y)[row * a.ldy + col] = (T)v;
}

// Tiles of 64 x 64, four waves of 32 x 32, operands through LDS 32 deep; any K, strides and
// alignment (elements are loaded one by one).
template <class T>
__global__ __launch_bounds__(256) void product_simple(DmlProductArgs a) {
  typedef typename Mfma<T>::vec vec;
  constexpr int BM = 64, BN = 64, P = 40;  // LDS row pitch in elements
  __shared__ __attribute__((aligned(16))) T sx[BM * P], sw[BN * P];
  const int ntn = (a.N + BN - 1) / BN;
  const Place at = locate<BM>(a, blockIdx.x / ntn);
  if (at.rows <= 0) return;
  const int n0 = (blockIdx.x % ntn) * BN;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const bool fill = at.e >= a.E;
  const T* x = (const T*)a.x + at.row * a.ldx;
  const T* w = (const T*)a.w + (fill ? 0 : at.e) * a.w_group + n0 * a.ldw;
  f32x4 acc[2][2] = {};
  const int wm = (wid >> 1) * 32, wn = (wid & 1) * 32;
  const int r = tid >> 2, kc = (tid & 3) * 8;
  for (int k0 = 0; k0 < (fill ? 0 : a.K); k0 += 32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = k0 + kc + j;
      sx[r * P + kc + j] = r < at.rows && k < a.K ? x[r * a.ldx + k] : (T)0.f;
      sw[r * P + kc + j] = n0 + r < a.N && k < a.K ? w[r * a.ldw + k] : (T)0.f;
    }
    __syncthreads();
    vec fx[2], fw[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fx[i] = *(const vec*)(sx + (wm + i * 16 + (lane & 15)) * P + (lane >> 4) * 8);
      fw[i] = *(const vec*)(sw + (wn + i * 16 + (lane & 15)) * P + (lane >> 4) * 8);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = Mfma<T>::run(fw[i], fx[j], acc[i][j]);
    __syncthreads();
  }
  // lane: columns 4 (lane >> 4) + q of weight fragment i, row lane & 15 of row fragment j
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = wm + j * 16 + (lane & 15), col = n0 + wn + i * 16 + (lane >> 4) * 4 + q;
        if (m >= at.rows || col >= a.N) continue;
        if (fill) {
          if (a.out_f32) ((float*)a.y)[(at.row + m) * a.ldy + col] = 0.f;
          else ((T*)a.y)[(at.row + m) * a.ldy + col] = (T)0.f;
        } else {
          finish<T>(a, at.e, at.row + m, col, acc[i][j][q]);
        }
      }
}

// row tiles that a grid needs: every group may end in a tile of its own
static long row_tiles(const DmlProductArgs* a, int bm) {
  if (!a->ends) return ((long)a->M + bm - 1) / bm;
  const long used = a->E < a->M ? a->E : a->M;
  return (a->M + (used + a->fill) * (bm - 1)) / bm;
}

template <class T>
static int launch(const DmlProductArgs* a, hipStream_t s) {
  const long blocks = row_tiles(a, 64) * ((a->N + 63) / 64);
  if (blocks > INT_MAX) {
    dml_set_error("dml_product: over 2^31 tiles");
    return -1;
  }
  if (blocks == 0) return 0;
  hipLaunchKernelGGL(product_simple<T>, dim3((unsigned)blocks), dim3(256), 0, s, *a);
  DML_CHECK_LAUNCH();
  return 0;
}

}  // namespace prod
}  // namespace dml

extern "C" int dml_product(const DmlProductArgs* a, hipStream_t s) {
  if (!a || a->M < 0 || a->N < 0 || a->K < 0 || a->E < 0 || (!a->ends && a->E != 1)) {
    dml_set_error("dml_product: need M, N, K, E >= 0, and E = 1 without ends");
    return -1;
  }
  if ((a->dtype != DML_BF16 && a->dtype != DML_F16) || a->act < 0 || a->act >= DML_ACT_COUNT) {
    dml_set_error("dml_product: dtype or act out of range");
    return -1;
  }
  if (a->M == 0 || a->N == 0) return 0;
  if (!a->y || (a->K > 0 && a->E > 0 && (!a->x || !a->w)) || a->ldy < a->N || a->ldx < 0 || a->ldw < 0 ||
      a->ldr < 0) {
    dml_set_error("dml_product: null tensor or row stride out of range");
    return -1;
  }
  return a->dtype == DML_BF16 ? dml::prod::launch<bf16>(a, s) : dml::prod::launch<dml::f16>(a, s);
}
