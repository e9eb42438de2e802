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
#include "conv_shared.h"
#include <climits>

namespace dml {
namespace prod {

using convk::lds_void;
using convk::wait_vmcnt;

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
      const int row = __builtin_amdgcn_readfirstlane(b + (t - first) * BM);
      return {__builtin_amdgcn_readfirstlane(base + l), row, __builtin_amdgcn_readfirstlane(min(BM, n - row))};
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

// One output element: column `col` of row `row`, in group e.
template <class T>
__device__ __forceinline__ void finish1(const DmlProductArgs& a, int e, int64_t row, int col, float v) {
  if (a.bias) v += a.bias[e * a.bias_group + col];
  float r = 0.f;
  if (a.res)
    r = a.out_f32 ? ((const float*)a.res)[row * a.ldr + col] : to_f32(((const T*)a.res)[row * a.ldr + col]);
  v = a.act_last ? activate(v + r, a.act) : activate(v, a.act) + r;
  if (a.out_f32) ((float*)a.y)[row * a.ldy + col] = v;
  else ((T*)a.y)[row * a.ldy + col] = (T)v;
}

// Bias of the eight columns that a lane holds in each pair of its wave's column fragments.
template <class C>
struct Bias {
  float v[C::FI / 2][8];
  __device__ __forceinline__ void load(const DmlProductArgs& a, int e, int col0, int lane) {
#pragma unroll
    for (int p = 0; p < C::FI / 2; ++p) {
      const int col = col0 + p * 32 + (lane >> 4) * 8;
      const float* b = a.bias + e * a.bias_group;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[p][j] = a.bias && col + j < a.N ? b[col + j] : 0.f;
    }
  }
};

// A wave's accumulators (rows wm.., columns col0..) through the epilogue: of its 16 x 32 pieces those whose number is
// `mine` modulo `of`. A lane has eight columns of a row in a piece, and leaves them out unless all are inside. The
// residuals of its pieces are read G at a time ahead of the stores, which could be to the same memory.
template <int KIND, class C>
__device__ __forceinline__ void finish_as(const DmlProductArgs& a, const Place& at, f32x4 (&acc)[C::FI][C::FJ],
                                          const Bias<C>& bias, int wm, int col0, int lane, int mine, int of) {
  typedef typename C::T T;
  const Act act = act_parameters(a.act);
  constexpr int G = C::FJ % 4 == 0 ? 4 : C::FJ % 3 == 0 ? 3 : C::FJ % 2 == 0 ? 2 : 1;
  const int m0 = wm + (lane & 15);
#pragma unroll
  for (int p = 0; p < C::FI / 2; ++p) {
    const int64_t col = col0 + p * 32 + (lane >> 4) * 8;
    if (col + 8 > a.N) continue;
    const int64_t y0 = (at.row + m0) * a.ldy + col, r0 = (at.row + m0) * a.ldr + col;
#pragma unroll
    for (int j0 = 0; j0 < C::FJ; j0 += G) {
      float r[G][8] = {};
      if (a.res) {
#pragma unroll
        for (int j = 0; j < G; ++j)
          if ((p * C::FJ + j0 + j) % of == mine && m0 + (j0 + j) * 16 < at.rows) {
            const int64_t i = r0 + (j0 + j) * 16 * a.ldr;
            if (a.out_f32) {
              __builtin_memcpy(r[j], (const float*)a.res + i, 32);
            } else {
              Vec16<T> t;
              t.load((const T*)a.res + i);
              t.get(r[j]);
            }
          }
      }
#pragma unroll
      for (int j = 0; j < G; ++j) {
        if ((p * C::FJ + j0 + j) % of != mine || m0 + (j0 + j) * 16 >= at.rows) continue;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = acc[2 * p + q / 4][j0 + j][q % 4] + bias.v[p][q];
        if (a.act_last) {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = act.run<KIND>(v[q] + r[j][q]);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = act.run<KIND>(v[q]) + r[j][q];
        }
        const int64_t i = y0 + (j0 + j) * 16 * a.ldy;
        if (a.out_f32) {
          __builtin_memcpy((float*)a.y + i, v, 32);
        } else {
          Vec16<T> t;
          t.set(v);
          t.store((T*)a.y + i);
        }
      }
    }
  }
}

// The last N % 8 columns, which no lane of finish_as has: 16 rows at a time through `lds` (512 bytes a wave), element
// by element in the columns' order.
template <class C>
__device__ __forceinline__ void finish_last(const DmlProductArgs& a, const Place& at, f32x4 (&acc)[C::FI][C::FJ], int wm,
                                            int col0, int lane, int mine, int of, float* lds) {
  const int last = a.N & ~7;
#pragma unroll
  for (int p = 0; p < C::FI / 2; ++p) {
    const int piece = col0 + p * 32;
    if (last < piece || last >= piece + 32) continue;
#pragma unroll
    for (int j = 0; j < C::FJ; ++j) {
      if ((p * C::FJ + j) % of != mine) continue;
      if (piece + (lane >> 4) * 8 == last) {
#pragma unroll
        for (int q = 0; q < 8; ++q) lds[(lane & 15) * 8 + q] = acc[2 * p + q / 4][j][q % 4];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int i = lane; i < 128; i += 64) {
        const int m = wm + j * 16 + i / 8, col = last + i % 8;
        if (m < at.rows && col < a.N) finish1<typename C::T>(a, at.e, (int64_t)at.row + m, col, lds[i]);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

template <class C>
__device__ __forceinline__ void finish(const DmlProductArgs& a, const Place& at, f32x4 (&acc)[C::FI][C::FJ],
                                       const Bias<C>& bias, int wm, int n0, int wn, int lane, int mine, int of, char* lds,
                                       int wave) {
  if (a.act <= DML_ACT_RELU) finish_as<kClamp, C>(a, at, acc, bias, wm, n0 + wn, lane, mine, of);
  else if (a.act == DML_ACT_GELU) finish_as<kErf, C>(a, at, acc, bias, wm, n0 + wn, lane, mine, of);
  else finish_as<kSwish, C>(a, at, acc, bias, wm, n0 + wn, lane, mine, of);
  if ((a.N & 7) && n0 + C::BN > a.N) {
    __syncthreads();
    finish_last<C>(a, at, acc, wm, n0 + wn, lane, mine, of, (float*)lds + wave * 128);
  }
}

// Zeros into rows wm .. wm + rows, columns col0 .. col0 + cols of a tile.
template <class T>
__device__ __forceinline__ void zero_rows(const DmlProductArgs& a, const Place& at, int col0, int cols, int wm, int rows,
                                          int lane) {
  for (int m = wm; m < min(wm + rows, at.rows); ++m)
    for (int c = col0 + lane; c < min(col0 + cols, a.N); c += 64) {
      const int64_t i = (int64_t)(at.row + m) * a.ldy + c;
      if (a.out_f32) ((float*)a.y)[i] = 0.f;
      else ((T*)a.y)[i] = (T)0.f;
    }
}

// ---- tiles through LDS ----
//
// A workgroup of WM x WN waves computes BM rows x BN columns, D[column][row] = W X^T: the MFMA rows are output columns,
// so a lane holds runs of columns of one row. Operands go through LDS in K slices of 64 (whole 128-byte lines of a
// row; slices of 32 had the L2 serve twice the requests: 8192^3 bf16 904 us against 824), two slices in turn, copied
// there by LDS-DMA. The fragments of one half slice are read while the other's products run: a row fragment's
// register is refilled as soon as its products are issued, the column fragments alternate. So a wave waits once a
// slice, at the barrier that hands over the next one, and the slice behind that is requested right after it.
//
// 16-byte chunks lie in a tile row XORed with a key of the row, chosen so that the lanes that LDS serves together
// (0-3, 12-15, 20-23, 24-27 and so on) hit all 64 banks with both operands' row patterns: no conflicts by the counters.
//
// KG > 1: KG such sets of waves, each with LDS of its own, take the slices in turn; their sums meet in LDS at the end
// and are added in the sets' order. Where there are few tiles this is what fills the CUs (256 x 4096 x 4096: 32 us
// with one set, 20 with four).
template <class T_, int BM_, int BN_, int WM_, int WN_, int KG_, bool DMA_>
struct Tile {
  typedef T_ T;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KG = KG_, BK = 64;
  static constexpr bool DMA = DMA_;
  static constexpr int NW = WM * WN, NT = KG * NW * 64;       // waves of a set, threads
  static constexpr int TM = BM / WM, TN = BN / WN;            // rows, columns of a wave
  static constexpr int FJ = TM / 16, FI = TN / 16;            // fragments along rows, columns
  static constexpr int XI = BM / 8 / NW, WI = BN / 8 / NW;    // pieces of 8 tile rows that a wave copies per slice
  static constexpr int STAGE = (BM + BN) * 128, LDS = KG * 2 * STAGE;
  static constexpr int MINW = (LDS <= 40960 ? 4 : LDS <= 81920 ? 2 : 1) * KG * NW / 4;  // waves a SIMD that LDS leaves room for
  static_assert(KG == 1 || BM * BN * 4 <= 2 * STAGE, "a set's sums fit its LDS");
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && TN % 32 == 0 && TM % 16 == 0 && LDS <= 163840, "tile");
  __device__ __forceinline__ static int xkey(int row) { return row & 7; }
  __device__ __forceinline__ static int wkey(int row) { return (row & 3) | ((row >> 1) & 4); }
};

// Without DMA (operands that are not 16-byte aligned, or rows too far apart for its 32-bit offsets): the same copies
// through registers, loaded half a slice ahead of the barrier that frees their place.
template <class C>
__global__ __launch_bounds__(C::NT, C::MINW) void product_tile(DmlProductArgs a) {
#ifdef __HIP_DEVICE_COMPILE__  // the host needs the entry only
  typedef typename C::T T;
  typedef typename Mfma<T>::vec vec;
  __shared__ __attribute__((aligned(1024))) char all[C::LDS];
  // blocks of one XCD take neighbouring tiles, eight row tiles by all column tiles at a time
  const int ntn = (a.N + C::BN - 1) / C::BN, nb = gridDim.x;
  const int b = xcd_remap(blockIdx.x, nb), s0 = b / (8 * ntn) * 8;
  const int high = min(8, nb / ntn - s0), r = b - s0 * ntn;
  const int tn = r / high, tm = s0 + r - tn * high;
  const Place at = locate<C::BM>(a, tm);
  if (at.rows <= 0) return;
  const int n0 = tn * C::BN, cols = a.N - n0;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / C::NW, wid = wave % C::NW;
  const int wm = wid / C::WN * C::TM, wn = wid % C::WN * C::TN;
  if (at.e >= a.E) {
    if (kg == 0) zero_rows<T>(a, at, n0 + wn, C::TN, wm, C::TM, lane);
    return;
  }
  const int nk = (a.K + C::KG * C::BK - 1) / (C::KG * C::BK);  // slices of a set; those past K are zeros
  char* const smem = all + kg * 2 * C::STAGE;
  const T* const x = (const T*)a.x + at.row * a.ldx;
  const T* const w = (const T*)a.w + at.e * a.w_group + (int64_t)n0 * a.ldw;

  // A copy piece is 8 tile rows: lane l fills place l % 8 of row l / 8, so it fetches the chunk that belongs there.
  // With DMA, rows and chunks outside the operands get an offset past the descriptor's range: it writes zeros.
  const int lrow = lane >> 3, lplace = lane & 7;
  const int xrow0 = wid * C::XI * 8 + lrow, wrow0 = wid * C::WI * 8 + lrow;
  const int dx = wid * C::XI * 1024, dw = C::BM * 128 + wid * C::WI * 1024;
  constexpr unsigned kOut = 0x80000000u;
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc((void*)x, 0, 0x7ffffff0, 0x00020000);
  const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc((void*)w, 0, 0x7ffffff0, 0x00020000);
  unsigned ox[C::XI], ow[C::WI];
  uint4 hx[C::DMA ? 1 : C::XI], hw[C::DMA ? 1 : C::WI];
  if constexpr (C::DMA) {
#pragma unroll
    for (int j = 0; j < C::XI; ++j) {
      const int row = xrow0 + j * 8;
      ox[j] = row < at.rows ? (unsigned)(row * (int)(a.ldx * 2) + (lplace ^ C::xkey(row)) * 16) : kOut;
    }
#pragma unroll
    for (int j = 0; j < C::WI; ++j) {
      const int row = wrow0 + j * 8;
      ow[j] = row < cols ? (unsigned)(row * (int)(a.ldw * 2) + (lplace ^ C::wkey(row)) * 16) : kOut;
    }
  }
  auto fetch = [&](uint4& v, const T* p, int k) {  // the eight values from k of a row; 0 behind K
    if (k + 8 <= a.K) {
      __builtin_memcpy(&v, p + k, 16);
    } else {
      T t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = k + i < a.K ? p[k + i] : (T)0.f;
      __builtin_memcpy(&v, t, 16);
    }
  };
  // request slice kt: by DMA into `stage`, or into hx and hw
  auto issue = [&](int kt, int stage) {
    const int k0 = (kt * C::KG + kg) * C::BK;
    if constexpr (C::DMA) {
      if (k0 + C::BK > a.K) {  // chunks past K are out from now on
#pragma unroll
        for (int j = 0; j < C::XI; ++j)
          if (k0 + (lplace ^ C::xkey(xrow0 + j * 8)) * 8 >= a.K) ox[j] = kOut;
#pragma unroll
        for (int j = 0; j < C::WI; ++j)
          if (k0 + (lplace ^ C::wkey(wrow0 + j * 8)) * 8 >= a.K) ow[j] = kOut;
      }
#pragma unroll
      for (int j = 0; j < C::XI; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void*)(smem + dx + stage * C::STAGE + j * 1024), 16, ox[j],
                                                 k0 * 2, 0, 0);
#pragma unroll
      for (int j = 0; j < C::WI; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_void*)(smem + dw + stage * C::STAGE + j * 1024), 16, ow[j],
                                                 k0 * 2, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < C::XI; ++j) {
        const int row = xrow0 + j * 8;
        hx[j] = make_uint4(0, 0, 0, 0);
        if (row < at.rows) fetch(hx[j], x + row * a.ldx, k0 + (lplace ^ C::xkey(row)) * 8);
      }
#pragma unroll
      for (int j = 0; j < C::WI; ++j) {
        const int row = wrow0 + j * 8;
        hw[j] = make_uint4(0, 0, 0, 0);
        if (row < cols) fetch(hw[j], w + row * a.ldw, k0 + (lplace ^ C::wkey(row)) * 8);
      }
    }
  };
  auto put = [&](int stage) {  // hx and hw into their places
    if constexpr (!C::DMA) {
#pragma unroll
      for (int j = 0; j < C::XI; ++j) *(uint4*)(smem + dx + stage * C::STAGE + j * 1024 + lane * 16) = hx[j];
#pragma unroll
      for (int j = 0; j < C::WI; ++j) *(uint4*)(smem + dw + stage * C::STAGE + j * 1024 + lane * 16) = hw[j];
    }
  };

  f32x4 acc[C::FI][C::FJ];
#pragma unroll
  for (int i = 0; i < C::FI; ++i)
#pragma unroll
    for (int j = 0; j < C::FJ; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  // fragment i's row r is column 32 (i / 2) + 8 (r / 4) + 4 (i % 2) + r % 4 of the wave: lane group q then holds
  // columns 32 p + 8 q .. + 7 in fragments 2p and 2p + 1, and stores 16 bytes
  const int fr = lane & 15, fq = lane >> 4;
  const int xrow = wm + fr, wrow = wn + (fr >> 2) * 8 + (fr & 3);
  const int ax[2] = {xrow * 128 + ((fq ^ C::xkey(xrow)) << 4), xrow * 128 + (((4 + fq) ^ C::xkey(xrow)) << 4)};
  const int aw[2] = {(C::BM + wrow) * 128 + ((fq ^ C::wkey(wrow)) << 4),
                     (C::BM + wrow) * 128 + (((4 + fq) ^ C::wkey(wrow)) << 4)};
  auto read_x = [&](vec& v, int stage, int half, int j) {
    v = *(const vec*)(smem + stage * C::STAGE + ax[half] + j * 16 * 128);
  };
  auto read_w = [&](vec& v, int stage, int half, int i) {
    v = *(const vec*)(smem + stage * C::STAGE + aw[half] + ((i & 1) * 4 + (i >> 1) * 32) * 128);
  };
  vec fx[C::FJ], fa[C::FI], fb[C::FI];
  Bias<C> bias;
  // the products of one half, reading the next half's row fragments behind them
  auto run = [&](vec(&f)[C::FI], bool more, int stage, int half) {
#pragma unroll
    for (int j = 0; j < C::FJ; ++j) {
#pragma unroll
      for (int i = 0; i < C::FI; ++i) acc[i][j] = Mfma<T>::run(f[i], fx[j], acc[i][j]);
      if (more) read_x(fx[j], stage, half, j);
    }
  };
  auto first = [&](int stage) {  // the first half of a slice
#pragma unroll
    for (int i = 0; i < C::FI; ++i) read_w(fb[i], stage, 1, i);
    run(fa, true, stage, 1);
  };

  if (nk > 0) {
    issue(0, 0);
    put(0);
    issue(1, 1);
    put(1);
    if constexpr (C::DMA) wait_vmcnt<C::XI + C::WI>();
    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int i = 0; i < C::FI; ++i) read_w(fa[i], 0, 0, i);
#pragma unroll
    for (int j = 0; j < C::FJ; ++j) read_x(fx[j], 0, 0, j);
    for (int kt = 0; kt < nk - 1; ++kt) {
      const int stage = kt & 1;
      if constexpr (!C::DMA) issue(kt + 2, stage);
      first(stage);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave is done reading `stage`
      if constexpr (C::DMA) wait_vmcnt<0>();              // and slice kt + 1 is there
      __builtin_amdgcn_s_barrier();
#pragma unroll
      for (int i = 0; i < C::FI; ++i) read_w(fa[i], stage ^ 1, 0, i);
      if constexpr (C::DMA) issue(kt + 2, stage);
      else put(stage);
      run(fb, true, stage ^ 1, 0);
    }
    bias.load(a, at.e, n0 + wn, lane);  // in flight over the last slice
    first((nk - 1) & 1);
    run(fb, false, 0, 0);
    if constexpr (C::DMA) wait_vmcnt<0>();  // slices past the last are zeros that still have to land
  } else {
    bias.load(a, at.e, n0 + wn, lane);
  }
  if constexpr (C::KG == 1) {
    finish<C>(a, at, acc, bias, wm, n0, wn, lane, 0, 1, all, wave);
  } else {
    __syncthreads();
    f32x4* const sums = (f32x4*)all;  // [set][wave][fragment][lane]
    constexpr int F = C::FI * C::FJ;
#pragma unroll
    for (int i = 0; i < C::FI; ++i)
#pragma unroll
      for (int j = 0; j < C::FJ; ++j) sums[((kg * C::NW + wid) * F + i * C::FJ + j) * 64 + lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < C::FI; ++i)
#pragma unroll
      for (int j = 0; j < C::FJ; ++j)
        if (((i / 2) * C::FJ + j) % C::KG == kg) {
          acc[i][j] = sums[(wid * F + i * C::FJ + j) * 64 + lane];
#pragma unroll
          for (int g = 1; g < C::KG; ++g) acc[i][j] += sums[((g * C::NW + wid) * F + i * C::FJ + j) * 64 + lane];
        }
    finish<C>(a, at, acc, bias, wm, n0, wn, lane, kg, C::KG, all, wave);
  }
#endif
}

// ---- few rows: K split over the waves ----
//
// A workgroup of NW waves computes 16 MF rows x 16 NF columns; the waves take the K slices of 64 in turn and load their
// fragments straight from memory (any alignment): with few rows the weight is read once, in order, and nothing is
// shared but the end, where the waves' sums meet in LDS and are added in the waves' order. Bound by the weight's bytes
// (one row, 2048 x 1000) or by the latency of a few loads in a row, so a wave keeps U slices in flight.
template <class T, int MF, int NF, int NW, int U>
__global__ __launch_bounds__(NW * 64) void product_rows(DmlProductArgs a) {
#ifdef __HIP_DEVICE_COMPILE__  // the host needs the entry only
  typedef typename Mfma<T>::vec vec;
  constexpr int F = MF * NF;
  __shared__ f32x4 part[NW][F][64];
  const int ntn = (a.N + NF * 16 - 1) / (NF * 16);
  const int b = xcd_remap(blockIdx.x, gridDim.x), tm = b / ntn, n0 = (b - tm * ntn) * NF * 16;
  const Place at = locate<MF * 16>(a, tm);
  if (at.rows <= 0) return;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (at.e >= a.E) {
    if (wid == 0) zero_rows<T>(a, at, n0, NF * 16, 0, MF * 16, lane);
    return;
  }
  const int fr = lane & 15, fq = lane >> 4;
  const T* const x = (const T*)a.x + (at.row + fr) * a.ldx;
  const T* const w = (const T*)a.w + at.e * a.w_group + (n0 + fr) * a.ldw;
  // Rows that start in the middle of a dword (the lane's rows are 16 apart: all of them or none) are loaded from the
  // dword's start and shifted: 16-byte loads off the dword grid took 1.7 times as long (1 x 4001 x 2000: 15 us, 9 for
  // 4002). The value ahead of the row shares its dword with the first.
  const bool oddx = ((uintptr_t)x & 2) != 0, oddw = ((uintptr_t)w & 2) != 0;
  auto fetch = [&](vec& v, const T* p, int k, bool row, bool odd) {  // eight values from k of a row; 0 outside
    if (row && k + 8 <= a.K) {
      uint4 u;
      __builtin_memcpy(&u, p + k - (odd ? 1 : 0), 16);
      if (odd) {
        const unsigned last = *(const unsigned short*)(p + k + 7);
        u.x = __builtin_amdgcn_alignbyte(u.y, u.x, 2);
        u.y = __builtin_amdgcn_alignbyte(u.z, u.y, 2);
        u.z = __builtin_amdgcn_alignbyte(u.w, u.z, 2);
        u.w = __builtin_amdgcn_alignbyte(last, u.w, 2);
      }
      __builtin_memcpy(&v, &u, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (T)0.f;
      if (row && k < a.K) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i < a.K) v[i] = p[k + i];
      }
    }
  };
  f32x4 acc[MF][NF];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int n = 0; n < NF; ++n) acc[m][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int k0 = wid * 64; k0 < a.K; k0 += NW * 64 * U) {
    vec fx[U][2][MF], fw[U][2][NF];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + u * NW * 64 + h * 32 + fq * 8;
#pragma unroll
        for (int n = 0; n < NF; ++n) fetch(fw[u][h][n], w + n * 16 * a.ldw, k, n0 + n * 16 + fr < a.N, oddw);
#pragma unroll
        for (int m = 0; m < MF; ++m) fetch(fx[u][h][m], x + m * 16 * a.ldx, k, m * 16 + fr < at.rows, oddx);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < MF; ++m)
#pragma unroll
          for (int n = 0; n < NF; ++n) acc[m][n] = Mfma<T>::run(fw[u][h][n], fx[u][h][m], acc[m][n]);
  }
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int n = 0; n < NF; ++n) part[wid][m * NF + n][lane] = acc[m][n];
  __syncthreads();
  for (int f = wid; f < F; f += NW) {
    f32x4 v = part[0][f][lane];
#pragma unroll
    for (int i = 1; i < NW; ++i) v += part[i][f][lane];
    const int m = f / NF * 16 + fr, col = n0 + f % NF * 16 + fq * 4;
    if (m >= at.rows) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (col + q < a.N) finish1<T>(a, at.e, (int64_t)at.row + m, col + q, v[q]);
  }
#endif
}

// row tiles that a grid needs: every group may end in a tile of its own
static long row_tiles(const DmlProductArgs* a, int bm) {
  if (!a->ends) return ((long)a->M + bm - 1) / bm;
  const long used = a->E < a->M ? a->E : a->M;
  return (a->M + (used + a->fill) * (bm - 1)) / bm;
}

static long tiles_of(const DmlProductArgs* a, int bm, int bn) { return row_tiles(a, bm) * ((a->N + bn - 1) / bn); }

// a grid has under 2^32 threads
static bool launchable(long blocks, int threads) { return blocks <= (long)(UINT_MAX / threads); }

template <class C>
static int launch(const DmlProductArgs* a, hipStream_t s) {
  const long blocks = tiles_of(a, C::BM, C::BN);
  hipLaunchKernelGGL(product_tile<C>, dim3((unsigned)blocks), dim3(C::NT), 0, s, *a);
  DML_CHECK_LAUNCH();
  return 0;
}

template <class T, int F, int NW, int U>
static int launch_rows(const DmlProductArgs* a, hipStream_t s) {
  const long blocks = tiles_of(a, 16 * F, 16 * F);
  hipLaunchKernelGGL((product_rows<T, F, F, NW, U>), dim3((unsigned)blocks), dim3(NW * 64), 0, s, *a);
  DML_CHECK_LAUNCH();
  return 0;
}

// The tiled forms a product can run in, and what each costs in microseconds: `first` once, `fixed` a tile (its ends),
// and a slice of 64 (KG of them) from `low`, on a card that is otherwise idle, to `high`, with a workgroup on every CU,
// for as many workgroups as a CU holds, or `shared` times their number if that is more. Fitted to 2000 timings over 1 to
// 12000 rows, K 64 to 8192, N 32 to 7000; of 255 of those products the form chosen is 1.4 % slower than the best of all in
// the mean, 19 % at worst. Where each wins: 300 x 6144 x 346 takes 14.7 us in tiles of 32 with KG = 8 and 25.9 in tiles of
// 64 with 4 (more workgroups to load); 1024 x 512 x 2048 7.6 with KG = 1, 8.6 with 2, 11.3 with 4; 17664 x 1024 x 4096 192
// in tiles of 256, 160 of 192 x 128, 180 of 128; 16384 x 4096 x 4096 430 / 462 / 500; 6304 x 4096 x 1024 83 / 76 / 54.
struct Form {
  int bm, bn, kg, per_cu, threads;
  double first, fixed, low, high, shared;
};
constexpr Form kForms[] = {{32, 32, 8, 1, 512, 1.8, 2.3, 0.50, 0.84, 0},     {64, 64, 1, 4, 256, 2.7, 0.6, 0.21, 0.44, 0.18},
                           {64, 64, 2, 2, 512, 2.3, 1.4, 0.30, 0.69, 0},     {64, 64, 4, 1, 1024, 1.9, 2.7, 0.51, 0.99, 0},
                           {128, 128, 1, 2, 256, 2.5, 2.6, 0.41, 0.81, 0.42}, {192, 128, 1, 2, 256, 2.8, 3.6, 0.57, 1.09, 0},
                           {256, 256, 1, 1, 512, 0, 7.9, 1.09, 1.61, 0}};

static double cost(const DmlProductArgs* a, const Form& f, bool dma) {
  const long tiles = tiles_of(a, f.bm, f.bn), per = (tiles + 255) / 256, rounds = per / f.per_cu, rest = per % f.per_cu;
  const double one = f.low + (f.high - f.low) * (tiles < 256 ? tiles / 256.0 : 1.0);
  const auto slice = [&](long n) { return n == 0 ? 0.0 : n * f.shared > one ? n * f.shared : one; };
  // rows off the 128-byte lines: a slice takes two lines each, which costs the forms that the L2 bounds (5000 x 2000 x
  // 6000 bf16: 134 us in tiles of 256, 153 of 192 x 128)
  const double lines = f.bm < 256 && ((a->ldx | a->ldw) & 63) ? 1.2 : 1.0;
  const int slices = (a->K + 64 * f.kg - 1) / (64 * f.kg);
  const double t = lines * slices * (rounds * slice(f.per_cu) + slice(rest)) + per * f.fixed;
  return f.first + (dma ? t : 1.4 * t + (f.kg > 1 ? 4 : 2));  // through registers
}

template <class T>
static int dispatch(const DmlProductArgs* a, hipStream_t s) {
  // LDS-DMA moves aligned 16 bytes at 32-bit offsets from a tile's first row
  const bool dma = a->K % 8 == 0 && a->ldx % 8 == 0 && a->ldw % 8 == 0 && a->w_group % 8 == 0 &&
                   (((uintptr_t)a->x | (uintptr_t)a->w) & 15) == 0 && a->ldx < (1 << 22) && a->ldw < (1 << 22) &&
                   255 * (a->ldx > a->ldw ? a->ldx : a->ldw) + a->K < (1 << 30) - 512 && a->K < (1 << 22);
  // product_rows in 16 x 16 (16 waves: 2048 of K in flight) and 32 x 32 (8 waves, 512), by the same timings: a workgroup
  // on a CU takes 3.6 us per 2048 of K, less where there is one tile of rows, and 1.3 to 1.6 per 512 (more
  // off the dword grid: 67 x 519 x 1388 takes 6.8 us in 16 x 16, 7.9 in 32 x 32). Off the 16-byte grid the choice among
  // these and the forms through registers was 3.1 % slower than the best in the mean over 130 products, 34 % at worst
  // (591 x 152 x 598).
  const double k = a->K / 2048.0, t32 = (double)tiles_of(a, 32, 32);
  const double rows16 = 3.1 + (tiles_of(a, 16, 16) + 255) / 256 * (k < 0.45 ? 0.45 : k) * (a->M <= 16 ? 3.0 : 3.6);
  const double each32 = 1.3 + 0.3 * (t32 < 256 ? t32 / 256 : 1.0), all32 = ((long)t32 + 255) / 256 * ((a->K + 511) / 512) * each32;
  const double rows32 = dma ? 3.1 + all32 : 3.8 + 1.25 * all32;
  // the cheapest that a grid holds: products of 2^30 rows take larger tiles
  int best = -3;
  double least = 1e300;
  if (launchable(tiles_of(a, 16, 16), 16 * 64)) least = rows16, best = -1;
  if (launchable((long)t32, 8 * 64) && rows32 <= least) least = rows32, best = -2;
  for (int i = 0; i < (int)(sizeof(kForms) / sizeof(kForms[0])); ++i) {
    if (!dma && (kForms[i].bm > 128 || kForms[i].kg == 2 || kForms[i].kg == 8)) continue;  // not built through registers
    if (!launchable(tiles_of(a, kForms[i].bm, kForms[i].bn), kForms[i].threads)) continue;
    const double c = cost(a, kForms[i], dma);
    if (c < least) least = c, best = i;
  }
  switch (best) {
    case -3: dml_set_error("dml_product: over 2^32 threads"); return -1;
    case -2: return launch_rows<T, 2, 8, 1>(a, s);
    case -1: return launch_rows<T, 1, 16, 2>(a, s);
    case 0: return launch<Tile<T, 32, 32, 1, 1, 8, true>>(a, s);
    case 1: return dma ? launch<Tile<T, 64, 64, 2, 2, 1, true>>(a, s) : launch<Tile<T, 64, 64, 2, 2, 1, false>>(a, s);
    case 2: return launch<Tile<T, 64, 64, 2, 2, 2, true>>(a, s);
    case 3: return dma ? launch<Tile<T, 64, 64, 2, 2, 4, true>>(a, s) : launch<Tile<T, 64, 64, 2, 2, 4, false>>(a, s);
    case 4: return dma ? launch<Tile<T, 128, 128, 2, 2, 1, true>>(a, s) : launch<Tile<T, 128, 128, 2, 2, 1, false>>(a, s);
    case 5: return launch<Tile<T, 192, 128, 2, 2, 1, true>>(a, s);
    default: return launch<Tile<T, 256, 256, 2, 4, 1, true>>(a, s);
  }
}

}  // namespace prod
}  // namespace dml

extern "C" int dml_product(const DmlProductArgs* a, hipStream_t s) {
  if (!a || a->M < 0 || a->N < 0 || a->K < 0 || a->E < 0 || a->K > (1 << 30) || a->M > INT_MAX - 512 ||
      a->N > INT_MAX - 512 || a->E > INT_MAX - 512 || (!a->ends && a->E != 1)) {
    dml_set_error("dml_product: need M, N, K, E from 0 to 2^31 - 513, K to 2^30, and E = 1 without ends");
    return -1;
  }
  if ((a->dtype != DML_BF16 && a->dtype != DML_F16) || a->act < 0 || a->act >= DML_ACT_COUNT) {
    dml_set_error("dml_product: dtype or act out of range");
    return -1;
  }
  if (a->M == 0 || a->N == 0) return 0;
  if (!a->y || (a->K > 0 && a->E > 0 && (!a->x || !a->w)) || a->ldy < a->N || a->ldx < 0 || a->ldw < 0 ||
      a->ldr < 0 || a->w_group < 0 || a->bias_group < 0 || a->ldx > INT64_MAX / 4 / a->M || a->ldw > INT64_MAX / 4 / a->N ||
      a->ldy > INT64_MAX / 4 / a->M || a->ldr > INT64_MAX / 4 / a->M) {
    dml_set_error("dml_product: null tensor or row stride out of range");
    return -1;
  }
  return a->dtype == DML_BF16 ? dml::prod::dispatch<bf16>(a, s) : dml::prod::dispatch<dml::f16>(a, s);
}
