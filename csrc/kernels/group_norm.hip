// group_norm.hip — group norm with its affine map and an activation, channels last (gfx950).
//
//   mu[n,g]  = mean over pixels p and the channels c of group g of x[n,p,c]
//   var[n,g] = mean of (x - mu)^2
//   y[n,p,c] = act((x - mu) / sqrt(var + eps) * weight[c] + bias[c])
//
// Bound by memory: x once in, y once out. A workgroup owns a SLAB of one sample: S channels
// (whole groups) over all pixels, read in 16-byte vectors so that a pixel's piece of the slab
// is a run of S channels. A thread keeps one column of vectors, hence one set of channels,
// weights and groups, and walks the rows.
//
//  * one_pass: the slab stays in registers between its one read and its one write, up to 16
//    vectors in each of 1024 threads (256 KiB).
//  * stats + apply: slabs beyond that, or too few slabs to fill the card. Every chunk of rows
//    yields (mean, sum of squared distances from it) per group in the workspace; the second
//    kernel merges the chunks and reads x again.
//
// Statistics in fp32 from centred values (E[x^2] - mu^2 loses all digits where the mean is
// large against the spread), chunks merged by the parallel form of the same
// (M2 = sum M2_i + n_i (mu_i - mu)^2), all sums in a fixed order.
#include "activation.h"

namespace dml {
namespace gn {

constexpr int kMaxGroups = 256;  // groups of a slab

// How a slab lies over NT threads.
template <class T, int NT, bool CH>
struct Slab {
  static constexpr int V = Vec16<T>::N;
  static constexpr int PC = CH ? V : 1;  // partial sums of a thread: per channel, or one where a vector is in one group
  int S, cg, cols, gs, RT, rt, col, n;   // channels, group width, vector columns, groups, row threads; mine; valid channels
  bool on;
  __device__ __forceinline__ Slab(int S_, int cg_) : S(S_), cg(cg_) {
    cols = (S + V - 1) / V;
    gs = S / cg;
    RT = NT / cols;
    rt = threadIdx.x / cols;
    col = threadIdx.x - rt * cols;
    on = rt < RT;
    n = min(V, S - col * V);
  }
  // Sums of v over the slab's groups -> stat[0 .. gs): every thread leaves its partial sums in
  // LDS, then one wave per group adds the group's in a fixed order.
  __device__ __forceinline__ void sum(const float (&v)[PC], float* part, float* stat) const {
    if (on) {
#pragma unroll
      for (int p = 0; p < PC; ++p) part[threadIdx.x * PC + p] = v[p];
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, SW = cols * PC, gw = CH ? cg : cg / V;
    for (int g = threadIdx.x >> 6; g < gs; g += NT / 64) {
      float s = 0.f;
      for (int t = lane; t < RT * gw; t += 64) {
        const int r = t / gw;
        s += part[r * SW + g * gw + t - r * gw];
      }
#pragma unroll
      for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
      if (lane == 0) stat[g] = s;
    }
    __syncthreads();
  }
  // stat of this thread's channels (PC of them)
  __device__ __forceinline__ void mine(const float* stat, float (&f)[PC]) const {
#pragma unroll
    for (int p = 0; p < PC; ++p) f[p] = stat[min((col * V + p) / cg, gs - 1)];
  }
  __device__ __forceinline__ void load(Vec16<T>& v, const T* p) const {
    if (n == V) v.load(p);
    else v.load(p, n);
  }
  __device__ __forceinline__ void store(const Vec16<T>& v, T* p) const {
    if (n == V) v.store(p);
    else v.store(p, n);
  }
};

// weight and bias of a thread's channels; `scale` = weight / sqrt(var + eps)
template <class T, int PC>
struct Affine {
  static constexpr int V = Vec16<T>::N;
  float scale[V], shift[V], mu[PC];
  __device__ __forceinline__ void load(const DmlGroupNormArgs& a, int c, int n) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      scale[j] = a.weight && j < n ? a.weight[c + j] : 1.f;
      shift[j] = a.bias && j < n ? a.bias[c + j] : 0.f;
    }
  }
  __device__ __forceinline__ void apply(Vec16<T>& v, int act) const {
    float f[V];
    v.get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = (f[j] - mu[PC == 1 ? 0 : j]) * scale[j] + shift[j];
    activate(f, act);
    v.set(f);
  }
};

// Rows [row0, row0 + rows) of the slab in registers; mean and M2 of its groups -> stat[0..gs), stat[kMaxGroups + ...)
template <class T, int NT, int R, bool CH>
__device__ __forceinline__ void read_and_sum(const Slab<T, NT, CH>& s, const T* x, int64_t ldx, int rows, float count,
                                             Vec16<T> (&v)[R], float (&mu)[Slab<T, NT, CH>::PC], float* part,
                                             float* stat) {
  constexpr int V = Vec16<T>::N, PC = Slab<T, NT, CH>::PC;
  float acc[PC] = {};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = s.rt + i * s.RT;
    if (s.on && r < rows) s.load(v[i], x + (int64_t)r * ldx);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (s.on && s.rt + i * s.RT < rows) {
      float f[V];
      v[i].get(f);
#pragma unroll
      for (int j = 0; j < V; ++j) acc[PC == 1 ? 0 : j] += f[j];
    }
  }
  s.sum(acc, part, stat);
  s.mine(stat, mu);
#pragma unroll
  for (int p = 0; p < PC; ++p) {
    mu[p] /= count;
    acc[p] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (s.on && s.rt + i * s.RT < rows) {
      float f[V];
      v[i].get(f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = j < s.n ? f[j] - mu[PC == 1 ? 0 : j] : 0.f;
        acc[PC == 1 ? 0 : j] += d * d;
      }
    }
  }
  s.sum(acc, part, stat + kMaxGroups);
}

template <class T, int NT, int R, bool CH>
__global__ __launch_bounds__(NT) void one_pass(DmlGroupNormArgs a, int S) {
  typedef Slab<T, NT, CH> SL;
  constexpr int V = SL::V, PC = SL::PC;
  __shared__ __attribute__((aligned(16))) float part[NT * PC];
  __shared__ float stat[2 * kMaxGroups];
  const int slabs = a.C / S, b = xcd_remap(blockIdx.x, gridDim.x);  // a sample's slabs share DRAM pages and lines
  const int n = b / slabs, c0 = (b - n * slabs) * S;
  const SL s(S, a.C / a.G);
  const int c = c0 + s.col * V;
  Vec16<T> v[R];
  Affine<T, PC> f;
  const float count = (float)a.HW * (float)s.cg;
  read_and_sum<T, NT, R, CH>(s, (const T*)a.x + n * a.xn + c, a.ldx, a.HW, count, v, f.mu, part, stat);
  if (!s.on) return;
  f.load(a, c, s.n);
  float var[PC];
  s.mine(stat + kMaxGroups, var);
#pragma unroll
  for (int j = 0; j < V; ++j) f.scale[j] *= 1.f / sqrtf(var[PC == 1 ? 0 : j] / count + a.eps);
  T* y = (T*)a.y + n * a.yn + c;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = s.rt + i * s.RT;
    if (r < a.HW) {
      f.apply(v[i], a.act);
      s.store(v[i], y + (int64_t)r * a.ldy);
    }
  }
}

// (mean, M2) of each group over one chunk of rows -> ws[(n G + g) chunks + chunk]
template <class T, int NT, int R, bool CH>
__global__ __launch_bounds__(NT) void stats(DmlGroupNormArgs a, int S, int rows, int chunks) {
  typedef Slab<T, NT, CH> SL;
  __shared__ __attribute__((aligned(16))) float part[NT * SL::PC];
  __shared__ float stat[2 * kMaxGroups];
  const int slabs = a.C / S;
  int b = xcd_remap(blockIdx.x, gridDim.x);
  const int slab = b % slabs, chunk = (b /= slabs) % chunks, n = b / chunks;
  const SL s(S, a.C / a.G);
  const int row0 = chunk * rows, mine = min(rows, a.HW - row0);
  Vec16<T> v[R];
  float mu[SL::PC];
  const float count = (float)mine * (float)s.cg;
  read_and_sum<T, NT, R, CH>(s, (const T*)a.x + n * a.xn + row0 * a.ldx + slab * S + s.col * SL::V, a.ldx, mine, count,
                             v, mu, part, stat);
  for (int g = threadIdx.x; g < s.gs; g += NT)
    ((float2*)a.ws)[((int64_t)n * a.G + slab * s.gs + g) * chunks + chunk] =
        make_float2(stat[g] / count, stat[kMaxGroups + g]);
}

template <class T, int NT, int R, bool CH>
__global__ __launch_bounds__(NT) void apply(DmlGroupNormArgs a, int S, int rows, int chunks) {
  typedef Slab<T, NT, CH> SL;
  constexpr int V = SL::V, PC = SL::PC;
  __shared__ float stat[2 * kMaxGroups];
  const int slabs = a.C / S;
  // in the order opposite to the statistics': what those
  // read last is still cached
  int b = xcd_remap(gridDim.x - 1 - blockIdx.x, gridDim.x);
  const int slab = b % slabs, chunk = (b /= slabs) % chunks, n = b / chunks;
  const SL s(S, a.C / a.G);
  const int lane = threadIdx.x & 63;
  const float total = (float)a.HW * (float)s.cg;
  for (int g = threadIdx.x >> 6; g < s.gs; g += NT / 64) {
    const float2* ws = (const float2*)a.ws + ((int64_t)n * a.G + slab * s.gs + g) * chunks;
    float sum = 0.f, m2 = 0.f;
    for (int i = lane; i < chunks; i += 64) sum += ws[i].x * (float)(min(rows, a.HW - i * rows) * s.cg);
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const float mu = sum / total;
    for (int i = lane; i < chunks; i += 64) {
      const float d = ws[i].x - mu;
      m2 += ws[i].y + d * d * (float)(min(rows, a.HW - i * rows) * s.cg);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) m2 += __shfl_xor(m2, o, 64);
    if (lane == 0) {
      stat[g] = mu;
      stat[kMaxGroups + g] = 1.f / sqrtf(m2 / total + a.eps);
    }
  }
  const int c = slab * S + s.col * V, row0 = chunk * rows, mine = min(rows, a.HW - row0);
  const T* x = (const T*)a.x + n * a.xn + row0 * a.ldx + c;
  T* y = (T*)a.y + n * a.yn + row0 * a.ldy + c;
  Vec16<T> v[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = s.rt + i * s.RT;
    if (s.on && r < mine) s.load(v[i], x + (int64_t)r * a.ldx);
  }
  Affine<T, PC> f;
  f.load(a, c, s.on ? s.n : 0);
  __syncthreads();
  if (!s.on) return;
  s.mine(stat, f.mu);
  float rs[PC];
  s.mine(stat + kMaxGroups, rs);
#pragma unroll
  for (int j = 0; j < V; ++j) f.scale[j] *= rs[PC == 1 ? 0 : j];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = s.rt + i * s.RT;
    if (r < mine) {
      f.apply(v[i], a.act);
      s.store(v[i], y + (int64_t)r * a.ldy);
    }
  }
}

// Groups wider than 1024 vectors: a workgroup per (sample, group), three reads.
template <class T>
__global__ __launch_bounds__(256) void wide_groups(DmlGroupNormArgs a) {
  __shared__ float part[4];
  const int g = blockIdx.x % a.G, n = blockIdx.x / a.G;
  const int cg = a.C / a.G, c0 = g * cg;
  const int64_t count = (int64_t)a.HW * cg;
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
  for (int64_t i = threadIdx.x; i < count; i += 256) s += to_f32(x[(i / cg) * a.ldx + i % cg]);
  const float mu = total(s) / (float)count;
  s = 0.f;
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    const float d = to_f32(x[(i / cg) * a.ldx + i % cg]) - mu;
    s += d * d;
  }
  const float rs = 1.f / sqrtf(total(s) / (float)count + a.eps);
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    const int c = (int)(i % cg);
    float v[1] = {(to_f32(x[(i / cg) * a.ldx + c]) - mu) * (rs * (a.weight ? a.weight[c0 + c] : 1.f)) +
                  (a.bias ? a.bias[c0 + c] : 0.f)};
    activate(v, a.act);
    y[(i / cg) * a.ldy + c] = (T)v[0];
  }
}

// The plan of a call: mode 0 = one pass, 1 = statistics and application apart, 2 = wide groups.
struct Plan {
  int mode, S, NT, R, rows, chunks;
  bool ch;
};

static Plan plan(const DmlGroupNormArgs* a) {
  const int es = a->dtype == DML_F32 ? 4 : 2, V = 16 / es, cg = a->C / a->G;
  Plan p = {};
  p.ch = cg % V != 0;
  if ((cg + V - 1) / V > 1024) {
    p.mode = 2;
    return p;
  }
  // A slab is a number of groups that divides G, best with whole vectors (partial ones at a slab's
  // end are loaded by the element). Wanted: runs of 128 bytes (a cache line) a pixel; a slab that
  // fits the registers of a workgroup; 512 workgroups, so that some load while others store.
  auto cost = [&](int k, bool fit_only) -> long {
    const long S = (long)k * cg, cols = (S + V - 1) / V;
    if (cols > 1024) return -1;
    const long cap = (1024 / cols) * 16;  // rows that one_pass<1024, 16> holds
    if (fit_only && a->HW > cap) return -1;
    const long wgs = (long)a->N * (a->C / S);
    long c = 0;
    if (S % V) c += 400;                       // element loads
    if (S * es < 128) c += (128 - S * es) * 2;  // short runs
    if (wgs < 512) c += (512 - wgs);
    c += S * es / 64;                           // else the narrower
    return c;
  };
  int best = 0;
  long bc = 0;
  for (int fit = 1; fit >= 0 && !best; --fit)
    for (int k = 1; k <= a->G && k <= kMaxGroups; ++k) {
      if (a->G % k) continue;
      const long c = cost(k, fit);
      if (c >= 0 && (!best || c < bc)) best = k, bc = c;
    }
  p.S = best * cg;
  const int cols = (p.S + V - 1) / V;
  const long wgs = (long)a->N * (a->C / p.S), slab = (long)a->HW * p.S * es;
  const int RT256 = 256 / cols, RT = 1024 / cols;
  if (cols <= 256 && a->HW <= (long)RT256 * 8) {
    p.NT = 256;
    p.R = a->HW <= RT256 * 2 ? 2 : 8;
    return p;
  }
  p.NT = 1024;
  if (a->HW <= (long)RT * 16 && !(wgs < 128 && slab > 128 * 1024)) {
    p.R = a->HW <= RT * 4 ? 4 : a->HW <= RT * 8 ? 8 : 16;
    return p;
  }
  p.mode = 1;
  p.R = 4;
  p.rows = RT * p.R;
  p.chunks = (a->HW + p.rows - 1) / p.rows;
  return p;
}

template <class T, bool CH>
static int launch(const DmlGroupNormArgs* a, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)((long)a->N * (p.mode == 2 ? a->G : a->C / p.S) * (p.mode == 1 ? p.chunks : 1)));
  if (p.mode == 2) {
    hipLaunchKernelGGL(wide_groups<T>, grid, dim3(256), 0, s, *a);
  } else if (p.mode == 1) {
    hipLaunchKernelGGL((stats<T, 1024, 4, CH>), grid, dim3(1024), 0, s, *a, p.S, p.rows, p.chunks);
    hipLaunchKernelGGL((apply<T, 1024, 4, CH>), grid, dim3(1024), 0, s, *a, p.S, p.rows, p.chunks);
  } else if (p.NT == 256) {
    if (p.R == 2) hipLaunchKernelGGL((one_pass<T, 256, 2, CH>), grid, dim3(256), 0, s, *a, p.S);
    else hipLaunchKernelGGL((one_pass<T, 256, 8, CH>), grid, dim3(256), 0, s, *a, p.S);
  } else {
    if (p.R == 4) hipLaunchKernelGGL((one_pass<T, 1024, 4, CH>), grid, dim3(1024), 0, s, *a, p.S);
    else if (p.R == 8) hipLaunchKernelGGL((one_pass<T, 1024, 8, CH>), grid, dim3(1024), 0, s, *a, p.S);
    else hipLaunchKernelGGL((one_pass<T, 1024, 16, CH>), grid, dim3(1024), 0, s, *a, p.S);
  }
  DML_CHECK_LAUNCH();
  return 0;
}

static int check(const DmlGroupNormArgs* a) {
  if (!a || a->N < 0 || a->HW < 0 || a->C < 1 || a->G < 1 || a->C % a->G) {
    dml_set_error("dml_group_norm: need N, HW >= 0 and a channel count that the groups divide");
    return -1;
  }
  if (a->dtype < DML_BF16 || a->dtype > DML_F32 || a->act < 0 || a->act >= DML_ACT_COUNT) {
    dml_set_error("dml_group_norm: dtype or act out of range");
    return -1;
  }
  if (a->N > 0 && a->HW > 0 && (!a->x || !a->y || a->ldx < 0 || a->ldy < a->C)) {
    dml_set_error("dml_group_norm: null tensor or a pixel stride out of range");
    return -1;
  }
  return 0;
}

}  // namespace gn
}  // namespace dml

extern "C" int64_t dml_group_norm_workspace(const DmlGroupNormArgs* a) {
  using namespace dml::gn;
  if (check(a) != 0) return -1;
  if (a->N == 0 || a->HW == 0) return 0;
  const Plan p = plan(a);
  return p.mode == 1 ? (int64_t)a->N * a->G * p.chunks * 8 : 0;
}

extern "C" int dml_group_norm(const DmlGroupNormArgs* a, hipStream_t s) {
  using namespace dml::gn;
  if (check(a) != 0) return -1;
  if (a->N == 0 || a->HW == 0) return 0;
  const Plan p = plan(a);
  const long per = (long)a->N * (p.mode == 2 ? a->G : a->C / p.S);
  if (per > 0x7fffffffl || (p.mode == 1 && per > 0x7fffffffl / p.chunks)) {
    dml_set_error("dml_group_norm: over 2^31 workgroups");
    return -1;
  }
  if (p.mode == 1 && (!a->ws || a->ws_bytes < (int64_t)a->N * a->G * p.chunks * 8)) {
    dml_set_error("dml_group_norm: workspace missing or smaller than dml_group_norm_workspace says");
    return -1;
  }
  switch (a->dtype) {
    case DML_BF16: return p.ch ? launch<bf16, true>(a, p, s) : launch<bf16, false>(a, p, s);
    case DML_F16: return p.ch ? launch<dml::f16, true>(a, p, s) : launch<dml::f16, false>(a, p, s);
    default: return p.ch ? launch<float, true>(a, p, s) : launch<float, false>(a, p, s);
  }
}
