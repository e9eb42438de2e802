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
//  * one_pass: the slab stays in registers (and, for the longest, LDS) between its one read and
//    its one write: up to 400 KiB in a workgroup.
//  * stats + apply: slabs beyond that, or too few slabs to fill the card. Every chunk of rows
//    yields (mean, sum of squared distances from it) per group in the workspace; the second
//    kernel merges the chunks and reads x again. Between them, where there are many chunks,
//    `join` merges each group's once for all.
//
// Statistics in fp32 from centred values (E[x^2] - mu^2 loses all digits where the mean is
// large against the spread), chunks merged by the parallel form of the same
// (M2 = sum M2_i + n_i (mu_i - mu)^2), all sums in a fixed order.
#include "activation.h"
#include <climits>

namespace dml {
namespace gn {

typedef __attribute__((address_space(3))) void lds_void;
constexpr int kMaxGroups = 256;  // groups of a slab

// t / d for 0 <= t < 2^21: t + 1/2 is at least 1/(2d) away from a multiple of d, the reciprocal's error below that
__device__ __forceinline__ int div_small(int t, float inv) { return (int)(((float)t + 0.5f) * inv); }

// The instruction takes no subnormals: those go through it 2^64 times as large.
__device__ __forceinline__ float inv_sqrt(float v) {
  const bool tiny = v < 0x1p-100f;
  const float r = __builtin_amdgcn_rsqf(tiny ? v * 0x1p64f : v);
  return tiny ? r * 0x1p32f : r;
}

// How a slab of S >= V channels lies over NT threads.
template <class T, int NT, bool CH>
struct Slab {
  static constexpr int V = Vec16<T>::N;
  static constexpr int PC = CH ? V : 1;  // statistics of a thread: per channel, or one where a vector is in one group
  int S, cg, cols, gs, RT;  // channels, group width, vector columns, groups, row threads
  float inv_cg;
  int rt, c, lo;            // this thread's first row, first channel, own channels [lo, V) of the vector there
  bool on;
  __device__ __forceinline__ Slab(int S_, int cg_) : S(S_), cg(cg_) {
    cols = (S + V - 1) / V;
    gs = S / cg;
    inv_cg = __builtin_amdgcn_rcpf((float)cg);
    RT = div_small(NT, __builtin_amdgcn_rcpf((float)cols));
    rt = div_small(threadIdx.x, __builtin_amdgcn_rcpf((float)cols));
    const int col = threadIdx.x - rt * cols;
    on = rt < RT;
    // the last vector ends with the slab: where V does not divide S it shares channels with the one before it (both
    // load and store them, with the same values; the statistics take them from that one)
    c = min(col * V, S - V);
    lo = col * V - c;
  }
  // rows r, r + RT, ... below `rows` (at most 64 a thread)
  __device__ __forceinline__ int rows_of(int r, int rows) const {
    return r < rows ? 1 + div_small(rows - 1 - r, __builtin_amdgcn_rcpf((float)RT)) : 0;
  }
  // The group's statistic at this thread's channels.
  __device__ __forceinline__ void mine(const float* stat, float (&f)[PC]) const {
#pragma unroll
    for (int p = 0; p < PC; ++p) f[p] = stat[min(div_small(c + p, inv_cg), gs - 1)];
  }
};

// A thread's vectors: R in registers, RL in LDS (its own 16 bytes of each row of lds).
template <class T, int NT, int R, int RL>
struct Held {
  Vec16<T> v[R];
  template <class F>
  __device__ __forceinline__ void each(int count, char* lds, F f) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < count) f(v[i], i);
    if constexpr (RL > 0) {
      for (int i = R; i < count; ++i) {
        Vec16<T> t;
        __builtin_memcpy(&t.v, lds + ((i - R) * NT + threadIdx.x) * 16, 16);
        f(t, i);
      }
    }
  }
};

// f(g, lane, L) for each of the gs groups, with L lanes of one wave to a group: a wave each where all groups get one,
// 8 lanes where they are more.
template <int NT, class F>
__device__ __forceinline__ void each_group(int gs, F f) {
  const int t = threadIdx.x;
  if (gs * 64 <= NT) {
    if (t < gs * 64) f(t >> 6, t & 63, std::integral_constant<int, 64>());
  } else {
    for (int g = t >> 3; g < gs; g += NT / 8) f(g, t & 7, std::integral_constant<int, 8>());
  }
}

// v summed over the L lanes of a group
template <int L>
__device__ __forceinline__ float over_lanes(float v) {
#pragma unroll
  for (int o = L >> 1; o; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Rows [0, rows) of the slab into registers and LDS; the groups' means -> stat[0 .. gs), their sums of squared
// distances from it -> stat[kMaxGroups ...). Each thread centres its own values (its mean, then its M2: no
// barrier), leaves the pair in LDS, and each_group merges a group's pairs in a fixed order.
template <class T, int NT, int R, int RL, bool CH, class F>
__device__ __forceinline__ void read_and_sum(const Slab<T, NT, CH>& s, const T* x, int64_t ldx, int rows,
                                             Held<T, NT, R, RL>& h, int count, bool once, char* lds, float2* part,
                                             float* stat, F meanwhile) {
  constexpr int V = Vec16<T>::N, PC = Slab<T, NT, CH>::PC;
  x += s.rt * ldx;
  const int64_t step = s.RT * ldx;
  if (once) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < count) h.v[i].load_once(x + i * step);
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < count) h.v[i].load(x + i * step);
  }
  if constexpr (RL > 0) {
#pragma unroll
    for (int i = R; i < R + RL; ++i) {
      if (i >= count) continue;
      __builtin_amdgcn_global_load_lds((const void*)(x + i * step),
                                       (lds_void*)(lds + ((i - R) * NT + (threadIdx.x & ~63)) * 16), 16, 0, 0);
    }
  }
  if constexpr (RL > 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  float mean[PC] = {}, m2[PC] = {};
  h.each(count, lds, [&](const Vec16<T>& v, int) {
    float f[V];
    v.get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) mean[PC == 1 ? 0 : j] += f[j];
  });
  const float inv = count > 0 ? 1.f / (float)(count * (V / PC)) : 0.f;
#pragma unroll
  for (int p = 0; p < PC; ++p) mean[p] *= inv;
  h.each(count, lds, [&](const Vec16<T>& v, int) {
    float f[V];
    v.get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = f[j] - mean[PC == 1 ? 0 : j];
      m2[PC == 1 ? 0 : j] += d * d;
    }
  });
  meanwhile();  // loads for later, in flight over the barriers
  // What a thread leaves: with CH, a pair per channel, or per group where a group is as wide as a vector (which then
  // holds channels of two groups at most: `cut` channels of the first).
  const bool two = CH && s.cg >= V;
  if (s.on) {
    if constexpr (!CH) {
      part[threadIdx.x] = make_float2(mean[0], m2[0]);
    } else if (two) {
      const int first = s.c + s.lo, cut = min(V, (div_small(first, s.inv_cg) + 1) * s.cg - s.c);
      float n0 = 0.f, s0 = 0.f, s1 = 0.f, q0 = 0.f, q1 = 0.f;
#pragma unroll
      for (int p = 0; p < V; ++p) {
        const bool in0 = p >= s.lo && p < cut, in1 = p >= cut;  // selected: a product with 0 would pass NaN on
        n0 += in0 ? 1.f : 0.f;
        s0 += in0 ? mean[p] : 0.f;
        s1 += in1 ? mean[p] : 0.f;
      }
      const float mu0 = s0 / n0, mu1 = cut < V ? s1 / (float)(V - cut) : 0.f;
#pragma unroll
      for (int p = 0; p < V; ++p) {
        const float d0 = mean[p] - mu0, d1 = mean[p] - mu1;
        q0 += p >= s.lo && p < cut ? m2[p] + d0 * d0 * (float)count : 0.f;
        q1 += p >= cut ? m2[p] + d1 * d1 * (float)count : 0.f;
      }
      part[2 * threadIdx.x] = make_float2(mu0, q0);
      part[2 * threadIdx.x + 1] = make_float2(mu1, q1);
    } else {
#pragma unroll
      for (int p = 0; p < PC; ++p)
        if (p >= s.lo) part[s.rt * s.cols * PC + s.c + p] = make_float2(mean[p], m2[p]);
    }
  }
  __syncthreads();
  const float total = (float)rows * (float)s.cg;
  each_group<NT>(s.gs, [&](int g, int lane, auto lanes) {
    constexpr int L = decltype(lanes)::value;
    // the group's pairs lie in runs of `gw`, one per row thread; `two`: every second from its first column's on
    const int c0 = g * s.cg, c1 = c0 + s.cg, col0 = c0 / V;
    const int gw = two ? (c1 - 1) / V - col0 + 1 : CH ? s.cg : s.cg / V;
    const int at = two ? 2 * col0 : CH ? c0 : col0, SW = two ? 2 * s.cols : s.cols * PC;
    const bool inside = two && (c0 & (V - 1));  // the group begins inside its first column: second pair there
    const float inv_gw = __builtin_amdgcn_rcpf((float)gw);
    const int entries = s.RT * gw;
    auto pair = [&](int t, float& n) {
      const int r = div_small(t, inv_gw), j = t - r * gw;
      n = (float)s.rows_of(r, rows);
      if (two) {
        const int lo = (col0 + j) * V;
        n *= (float)(min(c1, lo + V) - max(c0, lo));
        return part[r * SW + at + 2 * j + (inside && j == 0 ? 1 : 0)];
      }
      n *= (float)(V / PC);
      return part[r * SW + at + j];
    };
    float sum = 0.f, q = 0.f, n;
#pragma unroll 2
    for (int t = lane; t < entries; t += L) {
      const float2 e = pair(t, n);
      sum += e.x * n;
    }
    const float mu = over_lanes<L>(sum) / total;
#pragma unroll 2
    for (int t = lane; t < entries; t += L) {
      const float2 e = pair(t, n);
      q += e.y + (e.x - mu) * (e.x - mu) * n;
    }
    q = over_lanes<L>(q);
    if (lane == 0) {
      stat[g] = mu;
      stat[kMaxGroups + g] = q;
    }
  });
  __syncthreads();
}

// weight and bias of a thread's channels; `scale` = weight / sqrt(var + eps)
template <class T, int PC>
struct Affine {
  static constexpr int V = Vec16<T>::N;
  float scale[V], shift[V], mu[PC];
  __device__ __forceinline__ void load(const DmlGroupNormArgs& a, int c) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      scale[j] = a.weight ? a.weight[c + j] : 1.f;
      shift[j] = a.bias ? a.bias[c + j] : 0.f;
    }
  }
};

// The held vectors through the affine map and the activation -> y
template <int KIND, class T, int NT, int R, int RL, int PC>
__device__ __forceinline__ void write_as(Held<T, NT, R, RL>& h, const Affine<T, PC>& f, Act act, int count, char* lds,
                                         T* y, int64_t step) {
  constexpr int V = Vec16<T>::N;
  h.each(count, lds, [&](const Vec16<T>& v, int i) {
    float u[V];
    v.get(u);
#pragma unroll
    for (int j = 0; j < V; ++j) u[j] = act.run<KIND>((u[j] - f.mu[PC == 1 ? 0 : j]) * f.scale[j] + f.shift[j]);
    Vec16<T> w;
    w.set(u);
    w.store(y + i * step);
  });
}
template <class T, int NT, int R, int RL, int PC>
__device__ __forceinline__ void write(Held<T, NT, R, RL>& h, const Affine<T, PC>& f, int act, int count, char* lds, T* y,
                                      int64_t step) {
  if (act <= DML_ACT_RELU) write_as<kClamp>(h, f, act_parameters(act), count, lds, y, step);
  else if (act == DML_ACT_GELU) write_as<kErf>(h, f, act_parameters(act), count, lds, y, step);
  else write_as<kSwish>(h, f, act_parameters(act), count, lds, y, step);
}

template <class T, int NT, int R, int RL, bool CH>
__global__ __launch_bounds__(NT) void one_pass(DmlGroupNormArgs a, int S, int once) {
  typedef Slab<T, NT, CH> SL;
  constexpr int V = SL::V, PC = SL::PC;
  __shared__ float2 part[NT * PC];
  __shared__ float stat[2 * kMaxGroups];
  __shared__ __attribute__((aligned(16))) char lds[RL > 0 ? RL * NT * 16 : 16];
  const int slabs = a.C / S, b = xcd_remap(blockIdx.x, gridDim.x);  // a sample's slabs share DRAM pages and lines
  const int n = b / slabs, c0 = (b - n * slabs) * S;
  const SL s(S, a.C / a.G);
  const int c = c0 + s.c, count = s.on ? s.rows_of(s.rt, a.HW) : 0;
  Held<T, NT, R, RL> h;
  Affine<T, PC> f;
  read_and_sum<T, NT, R, RL, CH>(s, (const T*)a.x + n * a.xn + c, a.ldx, a.HW, h, count, once, lds, part, stat,
                                 [&] { f.load(a, c); });
  if (!s.on) return;
  s.mine(stat, f.mu);
  float var[PC];
  s.mine(stat + kMaxGroups, var);
  const float inv = 1.f / ((float)a.HW * (float)s.cg);
#pragma unroll
  for (int p = 0; p < PC; ++p) var[p] = inv_sqrt(var[p] * inv + a.eps);
#pragma unroll
  for (int j = 0; j < V; ++j) f.scale[j] *= var[PC == 1 ? 0 : j];
  T* y = (T*)a.y + n * a.yn + c + s.rt * a.ldy;
  const int64_t step = s.RT * a.ldy;
  write(h, f, a.act, count, lds, y, step);
}

// (mean, M2) of each group over one chunk of rows -> ws[(n G + g) chunks + chunk]
template <class T, int NT, int R, bool CH>
__global__ __launch_bounds__(NT) void stats(DmlGroupNormArgs a, int S, int rows, int chunks) {
  typedef Slab<T, NT, CH> SL;
  __shared__ float2 part[NT * SL::PC];
  __shared__ float stat[2 * kMaxGroups];
  const int slabs = a.C / S;
  int b = xcd_remap(blockIdx.x, gridDim.x);
  const int slab = b % slabs, chunk = (b /= slabs) % chunks, n = b / chunks;
  const SL s(S, a.C / a.G);
  const int row0 = chunk * rows, mine = min(rows, a.HW - row0);
  Held<T, NT, R, 0> h;
  read_and_sum<T, NT, R, 0, CH>(s, (const T*)a.x + n * a.xn + row0 * a.ldx + slab * S + s.c, a.ldx, mine, h,
                                s.on ? s.rows_of(s.rt, mine) : 0, false, nullptr, part, stat, [] {});
  for (int g = threadIdx.x; g < s.gs; g += NT)
    ((float2*)a.ws)[((int64_t)n * a.G + slab * s.gs + g) * chunks + chunk] = make_float2(stat[g], stat[kMaxGroups + g]);
}

// All rows' (mean, M2) of a group from its `parts` of `rows` rows each, by L lanes of a wave: every lane has it.
template <int L>
__device__ __forceinline__ float2 joined(const float2* ws, int parts, int rows, int HW, int cg, int lane) {
  // a part may hold 2^31 values and more
  const auto weight = [&](int i) { return (float)min(rows, HW - i * rows) * (float)cg; };
  float sum = 0.f, m2 = 0.f;
#pragma unroll 4
  for (int i = lane; i < parts; i += L) sum += ws[i].x * weight(i);
  const float mu = over_lanes<L>(sum) / ((float)HW * (float)cg);
#pragma unroll 4
  for (int i = lane; i < parts; i += L) {
    const float d = ws[i].x - mu;
    m2 += ws[i].y + d * d * weight(i);
  }
  return make_float2(mu, over_lanes<L>(m2));
}

// Long samples: a group's chunks joined once, and not in each of the chunks' workgroups again (chunks^2 pairs to
// read). Wave w of a group's workgroup joins every 16th run of chunks, its first thread the 16 results.
template <int NT>
__global__ __launch_bounds__(NT) void join(DmlGroupNormArgs a, int rows, int chunks) {
  __shared__ float2 part[NT / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = (chunks + NT / 64 - 1) / (NT / 64), first = min(wave * per, chunks), n = min(per, chunks - first);
  const float2* ws = (const float2*)a.ws + (int64_t)blockIdx.x * chunks + first;
  const int cg = a.C / a.G, span = per * rows;
  const float2 mine = n > 0 ? joined<64>(ws, n, rows, min(span, a.HW - first * rows), cg, lane) : make_float2(0.f, 0.f);
  if (lane == 0) part[wave] = mine;
  __syncthreads();
  if (wave == 0) {
    const int parts = (chunks + per - 1) / per;
    const float2 all = joined<64>(part, parts, span, a.HW, cg, lane);
    if (lane == 0) ((float2*)a.ws)[(int64_t)a.N * a.G * chunks + blockIdx.x] = all;
  }
}

// ws: the groups' pairs, `parts` of `part_rows` rows each
template <class T, int NT, int R, bool CH>
__global__ __launch_bounds__(NT) void apply(DmlGroupNormArgs a, int S, int rows, int chunks, const float2* ws, int parts,
                                            int part_rows) {
  typedef Slab<T, NT, CH> SL;
  constexpr int V = SL::V, PC = SL::PC;
  __shared__ float stat[2 * kMaxGroups];
  const int slabs = a.C / S;
  // in the order opposite to the statistics': what those read last is still cached
  int b = xcd_remap(gridDim.x - 1 - blockIdx.x, gridDim.x);
  const int slab = b % slabs, chunk = (b /= slabs) % chunks, n = b / chunks;
  const SL s(S, a.C / a.G);
  const float total = (float)a.HW * (float)s.cg;
  each_group<NT>(s.gs, [&](int g, int lane, auto lanes) {
    constexpr int L = decltype(lanes)::value;
    const float2 all = joined<L>(ws + ((int64_t)n * a.G + slab * s.gs + g) * parts, parts, part_rows, a.HW, s.cg, lane);
    if (lane == 0) {
      stat[g] = all.x;
      stat[kMaxGroups + g] = inv_sqrt(all.y / total + a.eps);
    }
  });
  const int c = slab * S + s.c, row0 = chunk * rows, mine = min(rows, a.HW - row0);
  const T* x = (const T*)a.x + n * a.xn + row0 * a.ldx + c;
  T* y = (T*)a.y + n * a.yn + row0 * a.ldy + c;
  const int count = s.on ? s.rows_of(s.rt, mine) : 0;
  Held<T, NT, R, 0> h;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i < count) h.v[i].load(x + (int64_t)(s.rt + i * s.RT) * a.ldx);
  Affine<T, PC> f;
  f.load(a, c);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // y may be x, and a slab's last two vectors may share channels
  __syncthreads();
  if (!s.on) return;
  s.mine(stat, f.mu);
  float rs[PC];
  s.mine(stat + kMaxGroups, rs);
#pragma unroll
  for (int j = 0; j < V; ++j) f.scale[j] *= rs[PC == 1 ? 0 : j];
  write(h, f, a.act, count, nullptr, y + s.rt * a.ldy, s.RT * a.ldy);
}

// What no slab fits: fewer channels than a vector has, groups wider than 1024 vectors, and group counts without a
// divisor up to kMaxGroups that makes a vector (521 groups of one channel). A workgroup per (sample, group), element by
// element, three reads: bound by one CU's instructions and latency (1 x 2^22 x 3 in one group: 52 ms). A thread may
// add 2^20 values and more one after the other, so the sums are in 64 bits (in 32, 2^25 x 3 fp16 values at a level of
// 100 and a spread of 1 came out up to 3 times the rounding off).
template <class T>
__global__ __launch_bounds__(256) void by_element(DmlGroupNormArgs a) {
  __shared__ double part[4];
  const int g = blockIdx.x % a.G, n = blockIdx.x / a.G;
  const int cg = a.C / a.G, c0 = g * cg;
  const int64_t count = (int64_t)a.HW * cg;
  const T* x = (const T*)a.x + n * a.xn + c0;
  T* y = (T*)a.y + n * a.yn + c0;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  auto total = [&](double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if (lane == 0) part[wid] = v;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
  };
  double s = 0;
  for (int64_t i = threadIdx.x; i < count; i += 256) s += (double)to_f32(x[(i / cg) * a.ldx + i % cg]);
  const float mu = (float)(total(s) / (double)count);
  s = 0;
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    const float d = to_f32(x[(i / cg) * a.ldx + i % cg]) - mu;
    s += (double)(d * d);
  }
  const float rs = inv_sqrt((float)(total(s) / (double)count) + a.eps);
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    const int c = (int)(i % cg);
    const float v = (to_f32(x[(i / cg) * a.ldx + c]) - mu) * (rs * (a.weight ? a.weight[c0 + c] : 1.f)) +
                    (a.bias ? a.bias[c0 + c] : 0.f);
    y[(i / cg) * a.ldy + c] = (T)activate(v, a.act);
  }
}

// How a call runs: slabs of S channels through one_pass (a row of kShapes), through stats + apply, or element
// by element.
enum { ONE_PASS, SPLIT, ELEMENTS };
struct Plan {
  int mode, S, shape, rows, chunks, once;
  bool ch, join;
};

// one_pass forms: threads, vectors in registers and in LDS. 14 vectors a thread leave two 512-thread or four 256-thread
// workgroups on a CU, and long slabs beat many short ones (256 x 49 x 2048 bf16, 256 threads: 23.1 us at 14 vectors,
// 29.8 at 7, 42 at 4), so a thread holds 14 where there is that much. The last form fills a CU with one workgroup: 400
// KiB, for 128-byte runs where the slab is long (256 x 3136 x 256 bf16: 170 us, against 190 with half the run). It copies
// into LDS directly, which takes 16-byte alignment.
constexpr int kShapes[][3] = {{256, 2, 0}, {256, 6, 0}, {256, 14, 0}, {512, 14, 0}, {1024, 16, 0}, {1024, 16, 9}};

static Plan plan(const DmlGroupNormArgs* a) {
  const int es = a->dtype == DML_F32 ? 4 : 2, V = 16 / es, cg = a->C / a->G;
  const bool aligned = (((uintptr_t)a->x | (uintptr_t)(a->xn * es) | (uintptr_t)(a->ldx * es)) & 15) == 0;
  const double bytes = 2.0 * es * a->N * a->HW * a->C;
  Plan p = {};
  p.ch = cg % V != 0;
  const double ops = (p.ch ? 13 : 10) + (a->act == DML_ACT_GELU ? 18 : a->act >= DML_ACT_SILU ? 11 : 1);
  double best = 1e30;
  // Estimated microseconds of each slab width, from measurements: memory at 5300 bytes/ns for runs of 128 bytes a
  // pixel, less for shorter ones (they cost lines) and off the dword grid; a lone CU's 60 bytes/ns, by the same rule,
  // and `ops` instructions a value on its 64 lanes, one after the other in one workgroup, at once in several on a CU;
  // 4.4 ns a workgroup. stats + apply read twice (the second time partly from cache) and pay a second launch and the
  // groups' merging. Over 75 sizes in every feasible plan the choice was 6.6 % slower than the best in the mean, 61 % at
  // worst (31 x 64 x 384 in 64 groups, odd pitch).
  for (int k = 1; k <= a->G && k <= kMaxGroups; ++k) {
    const long S = (long)k * cg, cols = (S + V - 1) / V;
    if (a->G % k || S < V || cols > 1024) continue;
    const double run = (double)(S * es), eff = (run >= 128 ? 1.0 : run / (run + 24)) * (S * es % 4 ? 0.6 : 1.0);
    const double wgs = (double)a->N * (a->C / S), values = (double)a->HW * S;
    const double stream = bytes / 5.3e6 / eff;
    const double mem = 2 * es * values / (60e3 * (run < 128 ? (run + 16) / 144 : 1.0) * (S * es % 4 ? 0.6 : 1.0)),
                  alu = values * ops / (64 * 2100.0);
    for (int i = 0; i < (int)(sizeof(kShapes) / sizeof(kShapes[0])); ++i) {
      const int* f = kShapes[i];
      if (f[2] && (p.ch || !aligned || run < 64)) continue;
      if (cols > f[0] || a->HW > f[0] / cols * (f[1] + f[2])) continue;
      const double each = (double)(long)((wgs + 255) / 256) * (f[0] == 1024 ? mem + alu : mem > alu ? mem : alu);
      const double own = 3 + (mem + alu > each ? mem + alu : each);
      const double t = (own > stream ? own : stream) + 4.4e-3 * wgs;
      if (t < best) {
        best = t;
        p.mode = ONE_PASS, p.S = (int)S, p.shape = i;
      }
      break;  // the smallest form that holds the slab
    }
    // 8 rows a thread, 4 where that leaves CUs idle; more threads where the rows are wide
    const int RT = (int)(256 / cols);
    const int shape = cols > 256 ? 2 : wgs * ((a->HW + RT * 8 - 1) / (RT * 8)) < 256;
    const int rows = shape == 2 ? (int)(1024 / cols) * 4 : RT * (shape ? 4 : 8), chunks = (a->HW + rows - 1) / rows;
    const double t = 1.55 * stream + 8 + 0.3 * k * chunks / 256;
    if (t < best) {
      best = t;
      p.mode = SPLIT, p.S = (int)S, p.shape = shape, p.rows = rows, p.chunks = chunks;
    }
  }
  // loads marked as not read again where x is beyond the caches anyway and a pixel's run is most of a line (256 x 784 x
  // 512 bf16: 92 -> 82 us; with runs of 32 bytes 15 % slower, and smaller inputs are often still cached)
  p.once = bytes / 2 >= 96e6 && p.S * es >= 64;
  // 2^22 pairs are where joining each group first is worth its launch (1 x 65536 x 512 in 256 chunks: 39.5 us without,
  // 42.5 with; 8 x 65536 x 256: 178 and 159; 1 x 1048576 x 64 in 4096: 261 and 69)
  p.join = p.mode == SPLIT && p.chunks >= 256 && (double)a->N * a->G * p.chunks * p.chunks >= 4194304.0;
  if (best == 1e30) p.mode = ELEMENTS;
  return p;
}

template <class T, int I, bool CH>
static void launch_one(const DmlGroupNormArgs* a, const Plan& p, dim3 grid, hipStream_t s) {
  if constexpr (!(CH && kShapes[I][2])) {
    if (p.shape == I)
      hipLaunchKernelGGL((one_pass<T, kShapes[I][0], kShapes[I][1], kShapes[I][2], CH>), grid, dim3(kShapes[I][0]), 0, s,
                         *a, p.S, p.once);
  }
  if constexpr (I > 0) launch_one<T, I - 1, CH>(a, p, grid, s);
}

template <class T, int NT, int R, bool CH>
static void launch_split(const DmlGroupNormArgs* a, const Plan& p, dim3 grid, hipStream_t s) {
  const float2* ws = (const float2*)a->ws;
  hipLaunchKernelGGL((stats<T, NT, R, CH>), grid, dim3(NT), 0, s, *a, p.S, p.rows, p.chunks);
  if (p.join) {
    hipLaunchKernelGGL(join<1024>, dim3((unsigned)a->N * a->G), dim3(1024), 0, s, *a, p.rows, p.chunks);
    ws += (int64_t)a->N * a->G * p.chunks;
  }
  hipLaunchKernelGGL((apply<T, NT, R, CH>), grid, dim3(NT), 0, s, *a, p.S, p.rows, p.chunks, ws, p.join ? 1 : p.chunks,
                     p.join ? a->HW : p.rows);
}

template <class T, bool CH>
static int launch(const DmlGroupNormArgs* a, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)((long)a->N * (p.mode == ELEMENTS ? a->G : a->C / p.S) * (p.mode == SPLIT ? p.chunks : 1)));
  if (p.mode == ELEMENTS) {
    hipLaunchKernelGGL(by_element<T>, grid, dim3(256), 0, s, *a);
  } else if (p.mode == ONE_PASS) {
    launch_one<T, sizeof(kShapes) / sizeof(kShapes[0]) - 1, CH>(a, p, grid, s);
  } else if (p.shape == 0) {
    launch_split<T, 256, 8, CH>(a, p, grid, s);
  } else if (p.shape == 1) {
    launch_split<T, 256, 4, CH>(a, p, grid, s);
  } else {
    launch_split<T, 1024, 4, CH>(a, p, grid, s);
  }
  DML_CHECK_LAUNCH();
  return 0;
}

static int check(const DmlGroupNormArgs* a) {
  if (!a || a->N < 0 || a->HW < 0 || a->HW > INT_MAX - 4096 || a->C < 1 || a->G < 1 || a->C % a->G) {
    dml_set_error("dml_group_norm: need N >= 0, HW from 0 to 2^31 - 4097 and a channel count that the groups divide");
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

extern "C" int64_t dml_group_norm(const DmlGroupNormArgs* a, hipStream_t s) {
  using namespace dml::gn;
  if (check(a) != 0) return -1;
  if (a->N == 0 || a->HW == 0) return 0;
  const Plan p = plan(a);
  const long per = (long)a->N * (p.mode == ELEMENTS ? a->G : a->C / p.S);
  // a grid has under 2^32 threads
  const long most = UINT_MAX / (p.mode == ELEMENTS ? 256 : p.mode == ONE_PASS ? kShapes[p.shape][0] : p.shape == 2 ? 1024 : 256);
  if (per > (p.mode == SPLIT ? most / p.chunks : most) || (p.join && (long)a->N * a->G > UINT_MAX / 1024)) {
    dml_set_error("dml_group_norm: over 2^32 threads");
    return -1;
  }
  const int64_t need = p.mode == SPLIT ? (int64_t)a->N * a->G * (p.chunks + p.join) * 8 : 0;
  if (need > a->ws_bytes || (need && !a->ws)) return need;
  switch (a->dtype) {
    case DML_BF16: return p.ch ? launch<bf16, true>(a, p, s) : launch<bf16, false>(a, p, s);
    case DML_F16: return p.ch ? launch<dml::f16, true>(a, p, s) : launch<dml::f16, false>(a, p, s);
    default: return p.ch ? launch<float, true>(a, p, s) : launch<float, false>(a, p, s);
  }
}
