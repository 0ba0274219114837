// Group norm with an activation on channel-last rows (graspbal.h gb_group_norm_*), forward and backward.
//
//   mean, var over the rows of a sample and the C / G channels of a group; r = 1 / sqrt(var + eps); xh = (x - mean) r
//   z = w_c xh + b_c (+ residual);  y = act(z) keep / (1 - p)
//   g = dy keep / (1 - p) act'(z);  dres = g;  dw_c = sum g xh;  db_c = sum g   (over all rows)
//   S1 = sum w g, S2 = sum w g xh over a sample's group of n elements;  dx = r (w g - S1 / n - xh S2 / n)
//
// What bounds it: bytes.  The statistics stand between two uses of x, so a sample that does not fit one workgroup's
// registers is read twice (forward 2 reads + 1 write, backward 4 + 1); one that does is read once.
//
// One mapping serves every pass and every channel count: a sample is ONE array of rows * C elements, a lane takes units of N
// consecutive ones (16 bytes), and the lanes that work step by T units, T the largest multiple of C / gcd(C, N) in the
// workgroup.  Then a lane meets the same N channels at every step: its weights stay in registers, its sums need no index,
// loads are full 16-byte accesses for odd C as well, and no lane divides.
#include <type_traits>

#include "row_common.h"

#pragma clang fp contract(on)  // a * b + c in one instruction; the geometry kernels alone need the split form

namespace gb {

static constexpr int GN_MAX_C = 4096;   // two doubles per channel in LDS while a workgroup's sums are joined
static constexpr int GN_DIRECT = 32;    // workgroups per sample up to which every applying one adds their sums for itself:
                                        // a launch less each way (4 x 1024 x 256 bf16: 41 -> 37 us of kernels a pass)
static constexpr int GN_DIRECT_GROUPS = 256;
static constexpr int GN_MIN_STEPS = 4;  // of a workgroup: with fewer, joining the sums costs what the parallelism gains
static constexpr int GN_RUN = 64;       // terms that a lane of the backward pass adds in fp32 before they join a sum in 64 bits

struct GnShape {
  long long R;         // rows of the whole tensor
  long long rows;      // rows per sample (offs == nullptr)
  const long long *offs;
  int S, C, G, cpg;
  int PL, T;           // lanes of one period, lanes that work (a multiple of PL)
  int ns;              // workgroups per sample
};

struct GnArgs {
  GnShape sh;
  const void *x, *res, *dy;
  const float *w, *b;
  void *y, *dx, *dres;
  float *mean, *rstd;  // (S, G)
  float *dw, *db;      // (C)
  double *gpart;       // forward: (S, ns, G, 2) sums of x and x^2
  float *cpart;        // backward: (S, ns, C, 2) sums of g and g xh
  float *csum;         // backward: (S, C, 2)
  const long long *rng;
  long long *used;
  long long seed, call;
  float eps, slope, scale;
  unsigned q;
  int sub;             // columns of a workgroup that holds them in registers
  int direct;          // the applying kernel joins the workgroups' sums itself
  int fold;            // backward: a lane adds more than GN_RUN steps
  int gather, zero;    // dweight / dbias, the rows outside every sample: kernels of their own
  double *zpart;       // gather: (gridDim.y, C, 2) sums over a share of the samples
};

// Rows of sample s.  Offsets come from the device and are taken as they are within [0, R]: no value of theirs leads
// outside the tensor.
__device__ __forceinline__ void sample_rows(const GnShape &sh, int s, long long &lo, long long &hi) {
  if (!sh.offs) {
    lo = sh.rows * s;
    hi = lo + sh.rows;
    return;
  }
  lo = sh.offs[s];
  hi = sh.offs[s + 1];
  lo = lo < 0 ? 0 : lo > sh.R ? sh.R : lo;
  hi = hi < lo ? lo : hi > sh.R ? sh.R : hi;
}

// z = x * sigmoid(x) and friends in fp32; v_exp_f32 / v_rcp_f32 are good to 1 ulp and the argument's rounding adds
// |z| 2^-24: ~1e-7 where the value is not itself vanishing.
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }
// Phi(z) = erfc(-z / sqrt 2) / 2 and e = exp(-z^2 / 2), which the slope needs as well.  erfcx(a) = t P(t), t = 1 / (1 + 0.425 a), P of
// degree 7 fitted for the least relative error over 0 <= a <= 9.3 (1.1e-7); negative z are taken from the tail itself, so
// that gelu keeps its relative error there (8e-7 down to z = -5).  No branch: sixteen erff of a lane's unit twice cost spills.
__device__ __forceinline__ float normal_cdf(float z, float &e) {
  e = __expf(-0.5f * z * z);
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.30052038f * fabsf(z));   // 0.425 / sqrt 2
  float p = 0.07247326f;
  p = p * t - 0.31730647f;
  p = p * t + 0.41477657f;
  p = p * t - 0.10985138f;
  p = p * t + 0.25858663f;
  p = p * t + 0.1996421f;
  p = p * t + 0.24201177f;
  p = p * t + 0.23966741f;
  const float tail = 0.5f * (p * t) * e;
  return z < 0.0f ? tail : 1.0f - tail;
}
template <int ACT>
__device__ __forceinline__ float act_value(float z, float slope) {
  switch (ACT) {
    case GB_ACT_RELU: return z > 0.0f ? z : z != z ? z : 0.0f;
    case GB_ACT_LEAKY_RELU: return z > 0.0f ? z : slope * z;
    case GB_ACT_SILU: return z * sigmoid(z);
    case GB_ACT_GELU: {
      float e;
      return z * normal_cdf(z, e);
    }
    default: return z;
  }
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z, float slope) {
  switch (ACT) {
    case GB_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case GB_ACT_LEAKY_RELU: return z > 0.0f ? 1.0f : slope;
    case GB_ACT_SILU: {
      const float s = sigmoid(z);
      return s * (1.0f + z * (1.0f - s));
    }
    case GB_ACT_GELU: {
      float e;
      const float c = normal_cdf(z, e);
      return c + z * e * 0.39894228f;
    }
    default: return 1.0f;
  }
}

// The lane's place in the period: N channels (N p + k) mod C.
struct Lane {
  int p, r;       // place in the period, row of lanes
  bool on;
};
__device__ __forceinline__ Lane lane_place(const GnShape &sh) {
  Lane l;
  const int t = (int)threadIdx.x;
  l.r = t / sh.PL;
  l.p = t - l.r * sh.PL;
  l.on = t < sh.T;
  return l;
}
template <int N>
__device__ __forceinline__ int channel0(const GnShape &sh, int p) {
  return (N * p) % sh.C;
}
__device__ __forceinline__ int next_channel(const GnShape &sh, int c) { return c + 1 == sh.C ? 0 : c + 1; }

// Joins (v0, v1)[K] of the T working lanes per channel (K = N) or per unit (K = 1) into out0 / out1, in a fixed order.
// buf: half of the lanes' values; out0, out1: C (K = N) or PL (K = 1) entries.  The lanes of one column are added as a
// tree; then the N elements of a lane go to their channels one after another - at each of these steps every lane has
// another channel - because with C not a multiple of N a channel appears at several places of the period.
template <int K, typename A>
__device__ __forceinline__ void join_columns(const GnShape &sh, const Lane &l, A (&v0)[K], A (&v1)[K], A *buf, A *out0,
                                             A *out1) {
  const int RL = sh.T / sh.PL;
  int h = 1;
  while (2 * h < RL) h *= 2;
  if (RL > 1)
    for (; h >= 1; h >>= 1) {
      if (l.on && l.r >= h && l.r < 2 * h) {
        A *to = buf + ((l.r - h) * sh.PL + l.p) * 2 * K;
#pragma unroll
        for (int k = 0; k < K; ++k) to[2 * k] = v0[k], to[2 * k + 1] = v1[k];
      }
      __syncthreads();
      if (l.on && l.r < h && l.r + h < RL) {
        const A *from = buf + (l.r * sh.PL + l.p) * 2 * K;
#pragma unroll
        for (int k = 0; k < K; ++k) v0[k] += from[2 * k], v1[k] += from[2 * k + 1];
      }
      __syncthreads();
    }
  // (out0 / out1 may lie over buf: every lane is past its last read of buf)
  if (K == 1) {
    if (l.on && l.r == 0) out0[l.p] = v0[0], out1[l.p] = v1[0];
  } else {
    for (int c = (int)threadIdx.x; c < sh.C; c += (int)blockDim.x) out0[c] = 0, out1[c] = 0;
    __syncthreads();
    int c = channel0<K>(sh, l.p);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (l.on && l.r == 0) out0[c] += v0[k], out1[c] += v1[k];
      c = next_channel(sh, c);
      if (sh.C % K) __syncthreads();
    }
  }
  __syncthreads();
}

// f(g, sum of a, sum of b) for every group g over its `per` consecutive entries of a, b: one lane per group while groups
// are short, a wave per group from 64 entries on.
template <typename A, typename F>
__device__ __forceinline__ void for_group_sums(const A *a, const A *b, int G, int per, F f) {
  if (per < 64) {
    for (int g = (int)threadIdx.x; g < G; g += (int)blockDim.x) {
      double s0 = 0, s1 = 0;
      for (int i = 0; i < per; ++i) s0 += (double)a[g * per + i], s1 += (double)b[g * per + i];
      f(g, s0, s1);
    }
    return;
  }
  const int lane = (int)threadIdx.x & 63;
  for (int g = (int)threadIdx.x >> 6; g < G; g += (int)blockDim.x >> 6) {
    double s0 = 0, s1 = 0;
    for (int i = lane; i < per; i += 64) s0 += (double)a[g * per + i], s1 += (double)b[g * per + i];
#pragma unroll
    for (int o = 32; o; o >>= 1) s0 += __shfl_xor(s0, o), s1 += __shfl_xor(s1, o);
    if (lane == 0) f(g, s0, s1);
  }
}

// Running count, mean and sum of squared deviations of a lane's N columns (Chan, Golub, LeVeque: "Algorithms for computing
// the sample variance", 1983): four rows at a time, so that an offset of the data costs no bits.
template <int N>
struct Moments {
  float n;
  float mean[N], m2[N];
  __device__ void clear() {
    n = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) mean[k] = m2[k] = 0;
  }
  __device__ void add4(const Vec<N> &a, const Vec<N> &b, const Vec<N> &c, const Vec<N> &d) {
    const float f = 4.0f / (n + 4.0f), e = n * f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float m = 0.25f * ((a.v[k] + b.v[k]) + (c.v[k] + d.v[k]));
      const float da = a.v[k] - m, db = b.v[k] - m, dc = c.v[k] - m, dd = d.v[k] - m, del = m - mean[k];
      mean[k] += del * f;
      m2[k] += ((da * da + db * db) + (dc * dc + dd * dd)) + del * del * e;
    }
    n += 4.0f;
  }
  __device__ void add1(const Vec<N> &a) {
    const float f = 1.0f / (n + 1.0f);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float del = a.v[k] - mean[k];
      mean[k] += del * f;
      m2[k] += del * (a.v[k] - mean[k]);
    }
    n += 1.0f;
  }
};

// Steps of T units [j0, j1) of a sample for workgroup `chunk`: at most ns ranges, of at least GN_MIN_STEPS steps - a short
// packed sample is not spread over the workgroups that the longest possible one would get.  ranges: those that are not
// empty; the first one always counts (it also has the sample's last elements).
__device__ __forceinline__ int chunk_ranges(const GnShape &sh, long long L, int N, long long &per) {
  const long long J = (L / N + sh.T - 1) / sh.T, even = (J + sh.ns - 1) / sh.ns;
  per = even < GN_MIN_STEPS ? GN_MIN_STEPS : even;
  return J <= per ? 1 : (int)((J + per - 1) / per);
}

// Sums of x and x^2 per group from the lanes' columns and `tail`, single elements of them (zeros elsewhere); f as in
// for_group_sums.
template <int N, typename F>
__device__ __forceinline__ void reduce_groups(const GnShape &sh, const Lane &l, const Moments<N> &m, const Vec<N> &tail, double *lds,
                                              F f) {
  if (sh.cpg % N == 0) {  // a lane's channels are one group's (and a sample has no tail)
    double s1[1] = {0}, s2[1] = {0};
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const double t = (double)m.n * m.mean[k];
      s1[0] += t;
      s2[0] += (double)m.m2[k] + t * m.mean[k];
    }
    join_columns<1, double>(sh, l, s1, s2, lds, lds, lds + sh.PL);
    for_group_sums(lds, lds + sh.PL, sh.G, sh.cpg / N, f);
  } else {
    double s1[N], s2[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const double t = (double)m.n * m.mean[k], e = tail.v[k];
      s1[k] = t + e;
      s2[k] = (double)m.m2[k] + t * m.mean[k] + e * e;
    }
    join_columns<N, double>(sh, l, s1, s2, lds, lds, lds + sh.C);
    for_group_sums(lds, lds + sh.C, sh.G, sh.cpg, f);
  }
}

extern __shared__ __attribute__((aligned(16))) unsigned char gn_lds[];

// the units of a workgroup: [first, end) in steps of T, and whether this lane has the sample's last L mod N elements
struct Range {
  long long base, v, end, last;
  int tail;
  bool none;
};
template <int N>
__device__ __forceinline__ Range range_of(const GnShape &sh, int s, int chunk) {
  Range g;
  long long lo, hi, per;
  sample_rows(sh, s, lo, hi);
  const long long L = (hi - lo) * sh.C;
  g.none = chunk >= chunk_ranges(sh, L, N, per);
  g.base = lo * sh.C;
  g.last = L / N;
  g.v = per * chunk * sh.T + threadIdx.x;
  g.end = per * (chunk + 1) * sh.T < g.last ? per * (chunk + 1) * sh.T : g.last;
  g.tail = chunk == 0 && (int)threadIdx.x == (int)(g.last % sh.T) ? (int)(L % N) : 0;
  return g;
}

// (Loads that the caches keep, here and in gn_bwd_stats_kernel, also for tensors past them: the applying kernel finds part of
// the tensors there.  4 x 131072 x 128 fp32 forward 150 -> 132 us, backward 249 -> 238; 8 x 131072 x 128 bf16 160 -> 144, 252 -> 243.)
template <typename T>
__global__ __launch_bounds__(1024) void gn_stats_kernel(GnArgs a) {
  constexpr int N = Unit<T>::N;
  const GnShape &sh = a.sh;
  const int s = (int)blockIdx.y, chunk = (int)blockIdx.x;
  const Lane l = lane_place(sh);
  const Range g = range_of<N>(sh, s, chunk);
  if (g.none) return;
  const T *x = (const T *)a.x + g.base;
  Moments<N> m;
  m.clear();
  VecOf<T> tail = {};
  if (l.on) {
    long long v = g.v;
    const long long step = sh.T;
    for (; v + 3 * step < g.end; v += 4 * step) {
      const Raw<T> r0 = load_raw(x + N * v), r1 = load_raw(x + N * (v + step)), r2 = load_raw(x + N * (v + 2 * step)),
                   r3 = load_raw(x + N * (v + 3 * step));
      m.add4(widen(r0), widen(r1), widen(r2), widen(r3));
    }
    for (; v < g.end; v += step) m.add1(load_unit(x + N * v));
    if (g.tail) tail = load_part(x + N * g.last, g.tail);
  }
  double *out = a.gpart + ((long long)s * sh.ns + chunk) * sh.G * 2;
  reduce_groups<N>(sh, l, m, tail, reinterpret_cast<double *>(gn_lds), [&](int g, double t1, double t2) {
    out[2 * g] = t1;
    out[2 * g + 1] = t2;
  });
}

__device__ __forceinline__ void finish_group(double t1, double t2, double n, float eps, float &mean, float &rstd) {
  const double m = t1 / n;
  double var = t2 / n - m * m;
  if (var < 0) var = 0;  // (NaN stays)
  mean = (float)m;
  rstd = (float)(1.0 / sqrt(var + (double)eps));
}

// mean and rstd of a group from the workgroups' sums, added by the lanes of a wave (lane, lanes) or by one alone (0, 1)
template <int N>
__device__ __forceinline__ void sample_stats(const GnArgs &a, int s, int g, int lane, int lanes, float &mean, float &rstd) {
  const GnShape &sh = a.sh;
  long long lo, hi, per;
  sample_rows(sh, s, lo, hi);
  const int ranges = chunk_ranges(sh, (hi - lo) * sh.C, N, per);
  double t1 = 0, t2 = 0;
#pragma unroll 4
  for (int c = lane; c < ranges; c += lanes) {
    const double *p = a.gpart + (((long long)s * sh.ns + c) * sh.G + g) * 2;
    t1 += p[0];
    t2 += p[1];
  }
  for (int o = lanes >> 1; o; o >>= 1) t1 += __shfl_xor(t1, o), t2 += __shfl_xor(t2, o);
  mean = rstd = 0;
  if (hi > lo) finish_group(t1, t2, (double)(hi - lo) * sh.cpg, a.eps, mean, rstd);
}

// one wave per (sample, group)
template <int N>
__global__ __launch_bounds__(64) void gn_finish_kernel(GnArgs a) {
  const long long at = (long long)blockIdx.y * a.sh.G + blockIdx.x;
  float mean, rstd;
  sample_stats<N>(a, (int)blockIdx.y, (int)blockIdx.x, (int)threadIdx.x, 64, mean, rstd);
  if (threadIdx.x == 0) a.mean[at] = mean, a.rstd[at] = rstd;
}

// A unit from flat index i (of the whole tensor) through norm, activation and dropout; res: zeros where there is no residual.
template <int N>
struct Coef {  // of a lane's channels; a = rstd * w
  float mean[N], rstd[N], a[N], b[N];
};
template <int N>
__device__ __forceinline__ void load_coef(const GnShape &sh, const float *w, const float *b, int p, const float *mean,
                                          const float *rstd, Coef<N> &co) {
  int c = channel0<N>(sh, p);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int g = c / sh.cpg;
    co.mean[k] = mean[g];
    co.rstd[k] = rstd[g];
    co.a[k] = w ? co.rstd[k] * w[c] : co.rstd[k];
    co.b[k] = b ? b[c] : 0.0f;
    c = next_channel(sh, c);
  }
}
template <int ACT, int N>
__device__ __forceinline__ Vec<N> norm_act(const GnArgs &a, const Coef<N> &co, const RowRng &rng, const Vec<N> &x, const Vec<N> &res,
                                           long long i) {
  Vec<N> y;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    float z = (x.v[k] - co.mean[k]) * co.a[k] + co.b[k];
    z += res.v[k];
    y.v[k] = act_value<ACT>(z, a.slope);
  }
  if (a.q) {
    const unsigned m = keep_mask<N>(rng, (unsigned long long)i, a.q);
#pragma unroll
    for (int k = 0; k < N; ++k) y.v[k] = (m >> k & 1) ? y.v[k] * a.scale : 0.0f;
  }
  return y;
}

// g and xh of a unit
template <int ACT, int N>
__device__ __forceinline__ void grad_act(const GnArgs &a, const Coef<N> &co, const RowRng &rng, const Vec<N> &x, const Vec<N> &res,
                                         const Vec<N> &dy, long long i, Vec<N> &g, Vec<N> &xh) {
  unsigned m = (1u << N) - 1;
  if (a.q) m = keep_mask<N>(rng, (unsigned long long)i, a.q);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float d0 = x.v[k] - co.mean[k];
    xh.v[k] = d0 * co.rstd[k];
    float z = d0 * co.a[k] + co.b[k];
    z += res.v[k];
    const float d = (a.q ? dy.v[k] * a.scale : dy.v[k]) * act_slope<ACT>(z, a.slope);
    g.v[k] = m >> k & 1 ? d : 0.0f;   // (a dropped element has no gradient, whatever the residual holds there)
  }
}

// rows before the first and behind the last sample: zeros
template <typename T>
__device__ __forceinline__ void zero_outside(const GnShape &sh, T *y, T *y2, long long part, long long parts) {
  long long lo, hi, lo2, hi2;
  sample_rows(sh, 0, lo, hi);
  sample_rows(sh, sh.S - 1, lo2, hi2);
  const long long n0 = lo * sh.C, n1 = (sh.R - hi2) * sh.C;
  for (long long i = part * blockDim.x + threadIdx.x; i < n0 + n1; i += parts * blockDim.x) {
    const long long e = i < n0 ? i : hi2 * sh.C + (i - n0);
    y[e] = (T)0.0f;
    if (y2) y2[e] = (T)0.0f;
  }
}

template <typename T, int ACT, bool NT>
__global__ __launch_bounds__(1024) void gn_apply_kernel(GnArgs a) {
  constexpr int N = Unit<T>::N;
  const GnShape &sh = a.sh;
  const int s = (int)blockIdx.y, chunk = (int)blockIdx.x;
  const RowRng rng = load_rng(a.rng, a.seed, a.call);
  if (s == 0 && chunk == 0 && threadIdx.x == 0 && a.used) {
    a.used[0] = (long long)rng.seed;
    a.used[1] = (long long)rng.call;
  }
  if (s == sh.S) {
    zero_outside<T>(sh, (T *)a.y, nullptr, chunk, sh.ns);
    return;
  }
  const Lane l = lane_place(sh);
  const Range g = range_of<N>(sh, s, chunk);
  if (g.none) return;
  const float *mean = a.mean + (long long)s * sh.G, *rstd = a.rstd + (long long)s * sh.G;
  __shared__ float stats[2][GN_DIRECT_GROUPS];
  if (a.direct) {
    for (int i = (int)threadIdx.x; i < sh.G; i += (int)blockDim.x) {
      sample_stats<N>(a, s, i, 0, 1, stats[0][i], stats[1][i]);
      if (chunk == 0) {
        a.mean[(long long)s * sh.G + i] = stats[0][i];
        a.rstd[(long long)s * sh.G + i] = stats[1][i];
      }
    }
    __syncthreads();
    mean = stats[0];
    rstd = stats[1];
  }
  if (!l.on) return;
  const T *x = (const T *)a.x + g.base, *res = a.res ? (const T *)a.res + g.base : nullptr;
  T *y = (T *)a.y + g.base;
  Coef<N> co;
  load_coef<N>(sh, a.w, a.b, l.p, mean, rstd, co);
  const long long step = sh.T;
  long long v = g.v;
  for (; v + step < g.end; v += 2 * step) {   // two steps' loads in flight
    const Raw<T> f0 = load_raw<NT>(x + N * v), f1 = load_raw<NT>(x + N * (v + step));
    VecOf<T> r0 = {}, r1 = {};
    if (res) r0 = load_unit<NT>(res + N * v), r1 = load_unit<NT>(res + N * (v + step));
    store_unit<NT>(y + N * v, norm_act<ACT, N>(a, co, rng, widen(f0), r0, g.base + N * v));
    store_unit<NT>(y + N * (v + step), norm_act<ACT, N>(a, co, rng, widen(f1), r1, g.base + N * (v + step)));
  }
  if (v < g.end) {
    VecOf<T> r = {};
    if (res) r = load_unit(res + N * v);
    store_unit(y + N * v, norm_act<ACT, N>(a, co, rng, load_unit(x + N * v), r, g.base + N * v));
  }
  if (g.tail) {
    v = g.last;
    VecOf<T> r = {};
    if (res) r = load_part(res + N * v, g.tail);
    store_part(y + N * v, norm_act<ACT, N>(a, co, rng, load_part(x + N * v, g.tail), r, g.base + N * v), g.tail);
  }
}

// ---- samples whose columns fit a workgroup's registers ----------------------------------------------------------------
// A workgroup takes all rows of a sample and `sub` columns (whole groups: the fewest that make full 128-byte lines), keeps
// its units in registers between the statistics and the output, and reads them once.  The period is that of the columns:
// place p of it is N columns of a row, a step goes down T / PL rows.  With C no multiple of N all columns are one
// workgroup's, as one flat array.
struct Sub {
  GnShape sh;       // the columns as a tensor of their own: C, G, PL, T
  long long base;   // first element
  int c0, g0;
  int first, step;  // of a lane, in elements from base
  int NV, tail;     // units of the workgroup, elements behind the last of them
  double n;         // elements of a group
};
template <int N>
__device__ __forceinline__ Sub sub_of(const GnArgs &a, int s, int part, const Lane &l) {
  Sub u;
  u.sh = a.sh;
  long long lo, hi;
  sample_rows(a.sh, s, lo, hi);
  const int rows = (int)(hi - lo), W = a.sub;
  u.c0 = part * W;
  u.g0 = u.c0 / a.sh.cpg;
  u.base = lo * a.sh.C + u.c0;
  u.sh.C = W;
  u.sh.G = W / a.sh.cpg;
  u.n = (double)rows * a.sh.cpg;
  if (W % N) {
    u.NV = rows * W / N;
    u.tail = rows * W % N;
    u.first = N * (int)threadIdx.x;
    u.step = N * a.sh.T;
  } else {
    u.NV = rows * a.sh.PL;
    u.tail = 0;
    u.first = l.r * a.sh.C + N * l.p;
    u.step = a.sh.T / a.sh.PL * a.sh.C;
  }
  return u;
}
// A lane holds 32 elements, what leaves 1024 lanes of 128 registers without spills.
static constexpr int GN_HELD = 32;

template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_small_kernel(GnArgs a) {
  constexpr int N = Unit<T>::N, H = GN_HELD / N;
  const int s = (int)blockIdx.y, part = (int)blockIdx.x;
  const RowRng rng = load_rng(a.rng, a.seed, a.call);
  if (s == 0 && part == 0 && threadIdx.x == 0 && a.used) {
    a.used[0] = (long long)rng.seed;
    a.used[1] = (long long)rng.call;
  }
  if (s == a.sh.S) {
    zero_outside<T>(a.sh, (T *)a.y, nullptr, part, gridDim.x);
    return;
  }
  const Lane l = lane_place(a.sh);
  const Sub u = sub_of<N>(a, s, part, l);
  const T *x = (const T *)a.x + u.base, *res = a.res ? (const T *)a.res + u.base : nullptr;
  T *y = (T *)a.y + u.base;
  const bool owns_tail = u.tail && l.on && (int)threadIdx.x == u.NV % u.sh.T;
  Raw<T> held[H];
#pragma unroll
  for (int i = 0; i < H; ++i)
    if (l.on && (int)threadIdx.x + i * u.sh.T < u.NV) held[i] = load_raw(x + (u.first + i * u.step));
  VecOf<T> t = {};
  if (owns_tail) t = load_part(x + N * u.NV, u.tail);
  Moments<N> m;
  m.clear();
#pragma unroll
  for (int i = 0; i < H; ++i)
    if (l.on && (int)threadIdx.x + i * u.sh.T < u.NV) m.add1(widen(held[i]));
  float *mean = a.mean + (long long)s * a.sh.G + u.g0, *rstd = a.rstd + (long long)s * a.sh.G + u.g0;
  reduce_groups<N>(u.sh, l, m, t, reinterpret_cast<double *>(gn_lds), [&](int g, double t1, double t2) {
    float mu = 0, r = 0;
    if (u.n > 0) finish_group(t1, t2, u.n, a.eps, mu, r);
    mean[g] = mu;
    rstd[g] = r;
  });
  __threadfence_block();
  __syncthreads();
  if (!l.on) return;
  Coef<N> co;
  load_coef<N>(u.sh, a.w ? a.w + u.c0 : nullptr, a.b ? a.b + u.c0 : nullptr, l.p, mean, rstd, co);
#pragma unroll
  for (int i = 0; i < H; ++i) {
    if ((int)threadIdx.x + i * u.sh.T < u.NV) {
      const int e = u.first + i * u.step;
      VecOf<T> r = {};
      if (res) r = load_unit(res + e);
      store_unit(y + e, norm_act<ACT, N>(a, co, rng, widen(held[i]), r, u.base + e));
    }
    __builtin_amdgcn_sched_barrier(0);   // (one unit widened at a time)
  }
  if (owns_tail) {
    VecOf<T> r = {};
    if (res) r = load_part(res + N * u.NV, u.tail);
    store_part(y + N * u.NV, norm_act<ACT, N>(a, co, rng, t, r, u.base + N * u.NV), u.tail);
  }
}

// ---- backward -------------------------------------------------------------------------------------------------------

template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_bwd_stats_kernel(GnArgs a) {
  constexpr int N = Unit<T>::N;
  const GnShape &sh = a.sh;
  const int s = (int)blockIdx.y, chunk = (int)blockIdx.x;
  const RowRng rng = load_rng(a.rng, a.seed, a.call);
  const Lane l = lane_place(sh);
  const Range u = range_of<N>(sh, s, chunk);
  if (u.none) return;
  const T *x = (const T *)a.x + u.base, *dy = (const T *)a.dy + u.base, *res = a.res ? (const T *)a.res + u.base : nullptr;
  float sg[N] = {}, sx[N] = {};
  double *whole = reinterpret_cast<double *>(gn_lds) + 2 * N * threadIdx.x;   // fold: sums of 64 bits
  if (l.on) {
    Coef<N> co;
    load_coef<N>(sh, a.w, a.b, l.p, a.mean + (long long)s * sh.G, a.rstd + (long long)s * sh.G, co);
    auto add = [&](const VecOf<T> &f, const VecOf<T> &r, const VecOf<T> &d, long long v) {
      VecOf<T> g, xh;
      grad_act<ACT, N>(a, co, rng, f, r, d, u.base + N * v, g, xh);
#pragma unroll
      for (int k = 0; k < N; ++k) sg[k] += g.v[k], sx[k] += g.v[k] * xh.v[k];
    };
    const long long step = sh.T;
    long long v = u.v;
    if (a.fold)
#pragma unroll
      for (int k = 0; k < 2 * N; ++k) whole[k] = 0;
    for (bool more = true; more;) {   // with `fold`, every GN_RUN steps the lane's sums go to its place in LDS
      const long long stop = a.fold && v + GN_RUN * step < u.end ? v + GN_RUN * step : u.end;
      for (; v + step < stop; v += 2 * step) {
        const Raw<T> f0 = load_raw(x + N * v), f1 = load_raw(x + N * (v + step)), d0 = load_raw(dy + N * v),
                     d1 = load_raw(dy + N * (v + step));
        VecOf<T> r0 = {}, r1 = {};
        if (res) r0 = load_unit(res + N * v), r1 = load_unit(res + N * (v + step));
        add(widen(f0), r0, widen(d0), v);
        add(widen(f1), r1, widen(d1), v + step);
      }
      more = stop < u.end;
      if (more)
#pragma unroll
        for (int k = 0; k < N; ++k) {
          whole[2 * k] += sg[k];
          whole[2 * k + 1] += sx[k];
          sg[k] = sx[k] = 0;
        }
    }
    if (v < u.end) {
      VecOf<T> r = {};
      if (res) r = load_unit(res + N * v);
      add(load_unit(x + N * v), r, load_unit(dy + N * v), v);
    }
    if (u.tail) {
      v = u.last;
      VecOf<T> r = {}, g, xh;
      if (res) r = load_part(res + N * v, u.tail);
      grad_act<ACT, N>(a, co, rng, load_part(x + N * v, u.tail), r, load_part(dy + N * v, u.tail), u.base + N * v, g, xh);
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (k < u.tail) sg[k] += g.v[k], sx[k] += g.v[k] * xh.v[k];
    }
    if (a.fold)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        sg[k] = (float)(whole[2 * k] + sg[k]);
        sx[k] = (float)(whole[2 * k + 1] + sx[k]);
      }
  }
  if (a.fold) __syncthreads();   // (the joins take the same LDS)
  float *lds = reinterpret_cast<float *>(gn_lds);
  join_columns<N, float>(sh, l, sg, sx, lds, lds, lds + sh.C);
  float2 *out = reinterpret_cast<float2 *>(a.cpart) + ((long long)s * sh.ns + chunk) * sh.C;
  for (int c = (int)threadIdx.x; c < sh.C; c += (int)blockDim.x) out[c] = make_float2(lds[c], lds[sh.C + c]);
}

// The workgroups' sums of a sample, joined: 8 channels x 32 lanes over the workgroups, in 64 bits.
template <int N>
__global__ __launch_bounds__(256) void gn_bwd_join_kernel(GnArgs a) {
  __shared__ double part[32][8][2];
  const GnShape &sh = a.sh;
  long long lo, hi, per;
  sample_rows(sh, (int)blockIdx.y, lo, hi);
  const int ranges = chunk_ranges(sh, (hi - lo) * sh.C, N, per);
  const int s = (int)blockIdx.y, i = (int)threadIdx.x & 7, c = (int)blockIdx.x * 8 + i, q = (int)threadIdx.x >> 3;
  double s0 = 0, s1 = 0;
  if (c < sh.C)
#pragma unroll 4
    for (int k = q; k < ranges; k += 32) {
      const float2 f = reinterpret_cast<const float2 *>(a.cpart)[((long long)s * sh.ns + k) * sh.C + c];
      s0 += f.x;
      s1 += f.y;
    }
  part[q][i][0] = s0;
  part[q][i][1] = s1;
  __syncthreads();
  if (q == 0 && c < sh.C) {
    for (int k = 1; k < 32; ++k) s0 += part[k][i][0], s1 += part[k][i][1];
    reinterpret_cast<float2 *>(a.csum)[(long long)s * sh.C + c] = make_float2((float)s0, (float)s1);
  }
}

// the sums of a channel over a sample, as the joining kernel left them or from the workgroups'
template <int N>
__device__ __forceinline__ void channel_sums(const GnArgs &a, int s, int c, double &s0, double &s1) {
  const GnShape &sh = a.sh;
  if (!a.direct) {
    const float2 f = reinterpret_cast<const float2 *>(a.csum)[(long long)s * sh.C + c];
    s0 += f.x;
    s1 += f.y;
    return;
  }
  long long lo, hi, per;
  sample_rows(sh, s, lo, hi);
  const int ranges = chunk_ranges(sh, (hi - lo) * sh.C, N, per);
#pragma unroll 8
  for (int k = 0; k < ranges; ++k) {
    const float2 f = reinterpret_cast<const float2 *>(a.cpart)[((long long)s * sh.ns + k) * sh.C + c];
    s0 += f.x;
    s1 += f.y;
  }
}

// dw, db = the samples' sums added, by workgroup `part` of `parts`: 32 channels x blockDim / 32 lanes over the samples
template <int N>
__device__ __forceinline__ void channel_gradients(const GnArgs &a, int part, int parts) {
  const GnShape &sh = a.sh;
  double *lds = reinterpret_cast<double *>(gn_lds);
  const int i = (int)threadIdx.x & 31, q = (int)threadIdx.x >> 5, Q = (int)blockDim.x >> 5;
  for (int c0 = part * 32; c0 < sh.C; c0 += parts * 32) {
    const int c = c0 + i;
    double s0 = 0, s1 = 0;
    if (c < sh.C)
      for (int s = q; s < sh.S; s += Q) channel_sums<N>(a, s, c, s0, s1);
    lds[2 * threadIdx.x] = s0;
    lds[2 * threadIdx.x + 1] = s1;
    __syncthreads();
    if (q == 0 && c < sh.C) {
      for (int j = 1; j < Q; ++j) s0 += lds[2 * (32 * j + i)], s1 += lds[2 * (32 * j + i) + 1];
      if (a.db) a.db[c] = (float)s0;
      if (a.dw) a.dw[c] = (float)s1;
    }
    __syncthreads();
  }
}

// The same where samples are many: 32 channels x 8 lanes over every gridDim.y-th block of eight samples, so that no lane waits
// for more than a few loads one after the other (in the applying kernel's last row, 4096 samples of 64 x 128 kept one workgroup
// busy for 1.2 ms).
template <int N>
__global__ __launch_bounds__(256) void gn_bwd_gather_kernel(GnArgs a) {
  __shared__ double lds[8][32][2];
  const GnShape &sh = a.sh;
  const int i = (int)threadIdx.x & 31, q = (int)threadIdx.x >> 5, c = (int)blockIdx.x * 32 + i;
  double s0 = 0, s1 = 0;
  if (c < sh.C) {
    if (sh.ns == 1) {
#pragma unroll 4
      for (int s = (int)blockIdx.y * 8 + q; s < sh.S; s += 8 * (int)gridDim.y) {
        const float2 f = reinterpret_cast<const float2 *>(a.cpart)[(long long)s * sh.C + c];
        s0 += f.x;
        s1 += f.y;
      }
    } else {
      for (int s = (int)blockIdx.y * 8 + q; s < sh.S; s += 8 * (int)gridDim.y) channel_sums<N>(a, s, c, s0, s1);
    }
  }
  lds[q][i][0] = s0;
  lds[q][i][1] = s1;
  __syncthreads();
  if (q > 0 || c >= sh.C) return;
  for (int j = 1; j < 8; ++j) s0 += lds[j][i][0], s1 += lds[j][i][1];
  if (gridDim.y > 1) {
    double *to = a.zpart + ((long long)blockIdx.y * sh.C + c) * 2;
    to[0] = s0;
    to[1] = s1;
  } else {
    if (a.db) a.db[c] = (float)s0;
    if (a.dw) a.dw[c] = (float)s1;
  }
}
__global__ __launch_bounds__(256) void gn_bwd_channels_kernel(GnArgs a, int parts) {
  __shared__ double lds[8][32][2];
  const int i = (int)threadIdx.x & 31, q = (int)threadIdx.x >> 5, c = (int)blockIdx.x * 32 + i, C = a.sh.C;
  double s0 = 0, s1 = 0;
  if (c < C)
#pragma unroll 4
    for (int z = q; z < parts; z += 8) {
      s0 += a.zpart[((long long)z * C + c) * 2];
      s1 += a.zpart[((long long)z * C + c) * 2 + 1];
    }
  lds[q][i][0] = s0;
  lds[q][i][1] = s1;
  __syncthreads();
  if (q > 0 || c >= C) return;
  for (int j = 1; j < 8; ++j) s0 += lds[j][i][0], s1 += lds[j][i][1];
  if (a.db) a.db[c] = (float)s0;
  if (a.dw) a.dw[c] = (float)s1;
}
template <typename T>
__global__ __launch_bounds__(256) void gn_zero_kernel(GnArgs a, T *y, T *y2) {
  zero_outside<T>(a.sh, y, y2, blockIdx.x, gridDim.x);
}

// S1 / n and S2 / n of every group into k1, k2 (LDS, G entries each) from the channels' sums v0, v1 (LDS, scaled by w here)
__device__ __forceinline__ void group_terms(const GnArgs &a, float *v0, float *v1, float *k1, float *k2, double n) {
  const GnShape &sh = a.sh;
  for (int c = (int)threadIdx.x; c < sh.C; c += (int)blockDim.x) {
    const float w = a.w ? a.w[c] : 1.0f;
    v0[c] *= w;
    v1[c] *= w;
  }
  __syncthreads();
  for_group_sums(v0, v1, sh.G, sh.cpg, [&](int g, double s0, double s1) {
    k1[g] = (float)(s0 / n);
    k2[g] = (float)(s1 / n);
  });
  __syncthreads();
}

template <int N>
__device__ __forceinline__ Vec<N> grad_x(const Coef<N> &co, const Vec<N> &g, const Vec<N> &xh, const float (&c1)[N],
                                         const float (&c2)[N]) {
  Vec<N> o;
#pragma unroll
  for (int k = 0; k < N; ++k) o.v[k] = co.a[k] * g.v[k] - c1[k] - xh.v[k] * c2[k];
  return o;
}

template <typename T, int ACT, bool NT>
__global__ __launch_bounds__(1024) void gn_bwd_apply_kernel(GnArgs a) {
  constexpr int N = Unit<T>::N;
  const GnShape &sh = a.sh;
  const int s = (int)blockIdx.y, chunk = (int)blockIdx.x;
  if (s == sh.S) {
    if (!a.gather) channel_gradients<N>(a, chunk, sh.ns);
    if (sh.offs && !a.zero) zero_outside<T>(sh, (T *)a.dx, (T *)a.dres, chunk, sh.ns);
    return;
  }
  const RowRng rng = load_rng(a.rng, a.seed, a.call);
  const Lane l = lane_place(sh);
  const Range u = range_of<N>(sh, s, chunk);
  if (u.none) return;
  long long lo, hi;
  sample_rows(sh, s, lo, hi);
  if (hi == lo) return;
  float *v0 = reinterpret_cast<float *>(gn_lds), *v1 = v0 + sh.C, *k1 = v1 + sh.C, *k2 = k1 + sh.G;
  for (int c = (int)threadIdx.x; c < sh.C; c += (int)blockDim.x) {
    double s0 = 0, s1 = 0;
    channel_sums<N>(a, s, c, s0, s1);
    v0[c] = (float)s0;
    v1[c] = (float)s1;
  }
  group_terms(a, v0, v1, k1, k2, (double)(hi - lo) * sh.cpg);
  if (!l.on) return;
  Coef<N> co;
  load_coef<N>(sh, a.w, a.b, l.p, a.mean + (long long)s * sh.G, a.rstd + (long long)s * sh.G, co);
  float c1[N], c2[N];
  int c = channel0<N>(sh, l.p);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    c1[k] = co.rstd[k] * k1[c / sh.cpg];
    c2[k] = co.rstd[k] * k2[c / sh.cpg];
    c = next_channel(sh, c);
  }
  const T *x = (const T *)a.x + u.base, *dy = (const T *)a.dy + u.base, *res = a.res ? (const T *)a.res + u.base : nullptr;
  T *dx = (T *)a.dx + u.base, *dres = a.dres ? (T *)a.dres + u.base : nullptr;
  auto put = [&](const VecOf<T> &f, const VecOf<T> &r, const VecOf<T> &d, long long v) {
    VecOf<T> g, xh;
    grad_act<ACT, N>(a, co, rng, f, r, d, u.base + N * v, g, xh);
    store_unit<NT>(dx + N * v, grad_x<N>(co, g, xh, c1, c2));
    if (dres) store_unit<NT>(dres + N * v, g);
  };
  const long long step = sh.T;
  long long v = u.v;
  for (; v + step < u.end; v += 2 * step) {
    const Raw<T> f0 = load_raw<NT>(x + N * v), f1 = load_raw<NT>(x + N * (v + step)), d0 = load_raw<NT>(dy + N * v),
                 d1 = load_raw<NT>(dy + N * (v + step));
    VecOf<T> r0 = {}, r1 = {};
    if (res) r0 = load_unit<NT>(res + N * v), r1 = load_unit<NT>(res + N * (v + step));
    put(widen(f0), r0, widen(d0), v);
    put(widen(f1), r1, widen(d1), v + step);
  }
  if (v < u.end) {
    VecOf<T> r = {};
    if (res) r = load_unit(res + N * v);
    put(load_unit(x + N * v), r, load_unit(dy + N * v), v);
  }
  if (u.tail) {
    v = u.last;
    VecOf<T> r = {}, g, xh;
    if (res) r = load_part(res + N * v, u.tail);
    grad_act<ACT, N>(a, co, rng, load_part(x + N * v, u.tail), r, load_part(dy + N * v, u.tail), u.base + N * v, g, xh);
    store_part(dx + N * v, grad_x<N>(co, g, xh, c1, c2), u.tail);
    if (dres) store_part(dres + N * v, g, u.tail);
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------

static int unit_of(int dtype) { return dtype == GB_T_F32 ? 4 : 8; }
static int period(int c, int unit) {   // lanes: c / gcd(c, unit)
  while (unit > 1 && c % unit) unit /= 2;
  return c / unit;
}

struct GnPlan {
  int block, PL, T;
  int ns;    // workgroups per sample
  int direct;
  int sub;   // columns per workgroup of the one-pass kernel; 0: the sample is read twice
  int fold;
  int gather, zero;   // workgroups over the samples that add dweight / dbias, over the rows outside them; 0: the last row's
  size_t lds, lds_stats, ws, zpart;
};

static int lds_tree(int T, int PL) {  // join_columns: most lanes that give theirs away at a step (RL - h first, then h / 2, ...)
  const int RL = T / PL;
  int h = 1;
  while (2 * h < RL) h *= 2;
  return RL > 1 ? (RL - h > h / 2 ? RL - h : h / 2) * PL : 0;
}

// Workgroups per sample: as many as fill the device with `waves` per SIMD, so that there is no last round of a few.  Where
// bytes alone bind, two waves, each with a long stretch of its own (4 x 131072 x 128 fp32 relu forward / backward: with what
// the registers allow 132 / 238 us, two 127 / 229, one 141 / 256; 8 x 131072 x 128 bf16: 144 / 244, 130 / 232, 159 / 291).  Where
// there is arithmetic to hide - dropout, gelu on 16-bit elements - what the registers allow (4 x 131072 x 128 bf16 gelu +
// residual: 110 / 210 us, two 114 / 214; with dropout 124 / 216, two 133 / 233; but 8 x 131072 x 128 bf16 silu + residual 180 /
// 344, two 171 / 329, and 4 x 65536 x 128 fp32 gelu + residual 90 / 169, two 88 / 162).  What the registers allow: 512 over the
// applying kernels' 60 (fp32) and 78 (16 bits) forward, 94 and 126 backward, in steps of eight; a build that took more would
// have a last round of a few, not other results.  Packed samples may be of very different lengths: as many, cut twice as fine.
// (The plan does not see the lengths: one cloud of 262144 rows x 64 among 1000 of 8 rows gets four workgroups, 6.4 ms a training pass.)
static int spread(const GbGroupNorm *n, long long steps, int block, bool backward) {
  const bool light = n->q == 0 && !(n->act == GB_ACT_GELU && n->dtype != GB_T_F32) && !n->offsets;
  const int waves = light ? 2 : n->dtype == GB_T_F32 ? (backward ? 5 : 8) : (backward ? 4 : 6);
  const long long most = 256ll * 4 * 64 * waves / block * (n->offsets ? 2 : 1) / n->samples, want = (steps + GN_MIN_STEPS - 1) / GN_MIN_STEPS;
  const long long ns = want < most ? want : most;
  return (int)(ns < 1 ? 1 : ns);
}

static GnPlan gn_plan(const GbGroupNorm *n, bool backward) {
  GnPlan p;
  const long long longest = n->offsets ? n->rows : n->rows / n->samples;
  const int C = n->channels, cpg = C / n->groups, N = unit_of(n->dtype), size = 16 / N;
  p.sub = p.fold = p.gather = p.zero = 0;
  if (!backward) {
    // The one-pass kernel wherever a sample's columns fit: no second read and one launch instead of three.  Columns: all
    // of them when C is no multiple of N, else the fewest whole groups that divide C into full 128-byte lines of units, or
    // halves or quarters of lines where only those fit (the other parts' workgroups find the line in L2).
    for (int line = 128; line >= 32 && !p.sub; line /= 2) {
      int sub = C;
      if (C % N == 0)
        for (int gs = 1; gs <= n->groups; ++gs)
          if (n->groups % gs == 0 && gs * cpg % N == 0 && gs * cpg * size >= line) {
            sub = gs * cpg;
            break;
          }
      const int PL = period(sub, N), T = PL <= 1024 ? 1024 / PL * PL : 0;
      if (T && longest * sub / N < (long long)T * (GN_HELD / N)) {
        p.sub = sub;
        p.PL = PL;
        // (lanes for one unit each, in whole waves: latency counts more than what a lane could hold)
        const long long units = (longest * sub + N - 1) / N;
        p.block = PL <= 256 && units <= 256 ? 256 : PL <= 512 && units <= 512 ? 512 : 1024;
        p.ns = C / sub;
      }
    }
  }
  if (!p.sub) {
    // Lanes: 256 where a period fits (more workgroups per CU to change between), else 512 or 1024.
    p.PL = period(C, N);
    p.block = p.PL <= 256 ? 256 : p.PL <= 512 ? 512 : 1024;
    const int T = p.block / p.PL * p.PL;
    const long long units = (longest * C + N - 1) / N, steps = (units + T - 1) / T;
    p.ns = spread(n, steps, p.block, backward);
    // short samples: a few more steps each rather than a launch more
    if (p.ns > GN_DIRECT && steps <= 2ll * GN_DIRECT * GN_MIN_STEPS) p.ns = GN_DIRECT;
    // Steps of the one row of workgroups that would add the samples' sums, some 0.6 us each: from 16 on, two launches are less.
    const long long groups = (C + 31) / 32, lanes = p.block / 32,
                    chain = (groups + p.ns - 1) / p.ns * ((n->samples + lanes - 1) / lanes);
    if (backward && chain > 16) p.gather = n->samples <= 128 ? 1 : n->samples < 256 * 64 ? (n->samples + 63) / 64 : 256;
    if (n->offsets && p.ns < 32 && n->samples >= 64) p.zero = 512;
    p.fold = backward && (steps + p.ns - 1) / p.ns > GN_RUN;
  }
  p.direct = !p.sub && p.ns <= GN_DIRECT && (backward || n->groups <= GN_DIRECT_GROUPS);
  p.T = p.block / p.PL * p.PL;
  const size_t cell = backward ? sizeof(float) : sizeof(double);
  const int K = !backward && cpg % N == 0 ? 1 : N;
  const size_t tree = (size_t)lds_tree(p.T, p.PL) * 2 * K * cell, flat = (size_t)(K == 1 ? p.PL : p.sub ? p.sub : C) * 2 * cell;
  p.lds = tree > flat ? tree : flat;
  if (backward) {
    const size_t apply = (size_t)(C + n->groups) * 2 * sizeof(float);
    if (apply > p.lds) p.lds = apply;
    const size_t joined = (size_t)p.block * 2 * sizeof(double);  // (channel_gradients)
    if (joined > p.lds) p.lds = joined;
    const size_t whole = p.fold ? (size_t)p.block * 2 * N * sizeof(double) : 0;
    p.lds_stats = whole > p.lds ? whole : p.lds;
    p.zpart = ((size_t)n->samples * p.ns + n->samples) * C * 2 * sizeof(float);
    p.ws = p.zpart + (p.gather > 1 ? (size_t)p.gather * C * 2 * sizeof(double) : 0);
  } else {
    p.ws = p.sub ? 0 : (size_t)n->samples * p.ns * n->groups * 2 * sizeof(double);
  }
  return p;
}

static int gn_bad(const GbGroupNorm *n) {
  if (!n || n->rows < 0 || n->samples <= 0 || n->channels <= 0 || n->groups <= 0 || n->channels % n->groups) return GB_EINVAL;
  if (!known_type(n->dtype) || n->act < 0 || n->act > GB_ACT_GELU || n->q < 0 || n->q > 65536 || !(n->eps >= 0)) return GB_EINVAL;
  if (!n->offsets && n->rows % n->samples) return GB_EINVAL;
  if (n->channels > GN_MAX_C || period(n->channels, unit_of(n->dtype)) > 1024 || n->samples > 65534) return GB_ERANGE;
  if (n->rows > (1ll << 62) / n->channels) return GB_ERANGE;
  if ((reinterpret_cast<uintptr_t>(n->offsets) | reinterpret_cast<uintptr_t>(n->rng) | reinterpret_cast<uintptr_t>(n->used)) % 8)
    return GB_EINVAL;
  return GB_OK;
}

template <typename F>
static int with_type_and_act(const GbGroupNorm *n, F f) {
  return with_type(n->dtype, [&](auto z) {
    switch (n->act) {
      case GB_ACT_RELU: return f(z, std::integral_constant<int, GB_ACT_RELU>());
      case GB_ACT_LEAKY_RELU: return f(z, std::integral_constant<int, GB_ACT_LEAKY_RELU>());
      case GB_ACT_SILU: return f(z, std::integral_constant<int, GB_ACT_SILU>());
      case GB_ACT_GELU: return f(z, std::integral_constant<int, GB_ACT_GELU>());
      default: return f(z, std::integral_constant<int, GB_ACT_NONE>());
    }
  });
}

static GnArgs gn_args(const GbGroupNorm *n, const GnPlan &p) {
  GnArgs a = {};
  a.sh.R = n->rows;
  a.sh.rows = n->offsets ? 0 : n->rows / n->samples;
  a.sh.offs = (const long long *)n->offsets;
  a.sh.S = n->samples;
  a.sh.C = n->channels;
  a.sh.G = n->groups;
  a.sh.cpg = n->channels / n->groups;
  a.sh.PL = p.PL;
  a.sh.T = p.T;
  a.sh.ns = p.ns;
  a.sub = p.sub;
  a.direct = p.direct;
  a.fold = p.fold;
  a.gather = p.gather;
  a.zero = p.zero;
  a.x = n->x;
  a.res = n->residual;
  a.w = n->weight;
  a.b = n->bias;
  a.mean = n->mean;
  a.rstd = n->rstd;
  a.rng = (const long long *)n->rng;
  a.used = (long long *)n->used;
  a.seed = n->seed;
  a.call = n->call;
  a.eps = n->eps;
  a.slope = n->slope;
  a.q = (unsigned)n->q;
  a.scale = keep_scale(n->q);
  return a;
}

}  // namespace gb

using namespace gb;

extern "C" int gb_group_norm_workspace(const GbGroupNorm *n, int backward, long long *bytes) {
  const int bad = gn_bad(n);
  if (bad || !bytes) return bad ? bad : GB_EINVAL;
  *bytes = n->rows == 0 ? 0 : (long long)gn_plan(n, backward != 0).ws;
  return GB_OK;
}

extern "C" int gb_group_norm_fwd(const GbGroupNorm *n, void *y, void *ws, long long ws_bytes, void *stream) {
  const int bad = gn_bad(n);
  if (bad) return bad;
  if (n->rows == 0) return GB_OK;
  if (!n->x || !y || !n->mean || !n->rstd) return GB_EINVAL;
  const GnPlan p = gn_plan(n, false);
  if (p.ws && (!ws || ws_bytes < (long long)p.ws || reinterpret_cast<uintptr_t>(ws) % 16)) return GB_EINVAL;
  GnArgs a = gn_args(n, p);
  a.y = y;
  a.gpart = (double *)ws;
  hipStream_t st = as_stream(stream);
  const bool nt = streams(n->rows * n->channels * (16 / unit_of(n->dtype)));
  const dim3 all((unsigned)p.ns, (unsigned)(n->samples + (n->offsets && !p.zero ? 1 : 0)));
  return with_type_and_act(n, [&](auto z, auto act) {
    typedef decltype(z) T;
    constexpr int ACT = decltype(act)::value;
    if (p.sub) {
      gn_small_kernel<T, ACT><<<all, p.block, p.lds, st>>>(a);
    } else {
      const dim3 grid((unsigned)p.ns, (unsigned)n->samples);
      gn_stats_kernel<T><<<grid, p.block, p.lds, st>>>(a);
      if (!p.direct) gn_finish_kernel<Unit<T>::N><<<dim3((unsigned)n->groups, (unsigned)n->samples), 64, 0, st>>>(a);
      if (nt)
        gn_apply_kernel<T, ACT, true><<<all, p.block, 0, st>>>(a);
      else
        gn_apply_kernel<T, ACT, false><<<all, p.block, 0, st>>>(a);
      if (p.zero) gn_zero_kernel<T><<<(unsigned)p.zero, 256, 0, st>>>(a, (T *)y, (T *)nullptr);
    }
    return check_launch("gb_group_norm_fwd");
  });
}

extern "C" int gb_group_norm_bwd(const GbGroupNorm *n, const void *dy, void *dx, void *dresidual, float *dweight, float *dbias,
                                 void *ws, long long ws_bytes, void *stream) {
  const int bad = gn_bad(n);
  if (bad) return bad;
  if (n->rows == 0) return GB_OK;
  if (!n->x || !dy || !dx || !n->mean || !n->rstd) return GB_EINVAL;
  const GnPlan p = gn_plan(n, true);
  if (!ws || ws_bytes < (long long)p.ws || reinterpret_cast<uintptr_t>(ws) % 16) return GB_EINVAL;
  GnArgs a = gn_args(n, p);
  a.dy = dy;
  a.dx = dx;
  a.dres = dresidual;
  a.dw = dweight;
  a.db = dbias;
  a.cpart = (float *)ws;
  a.csum = a.cpart + (size_t)n->samples * p.ns * n->channels * 2;
  a.zpart = (double *)((char *)ws + p.zpart);
  hipStream_t st = as_stream(stream);
  const bool nt = streams(n->rows * n->channels * (16 / unit_of(n->dtype)));
  return with_type_and_act(n, [&](auto z, auto act) {
    typedef decltype(z) T;
    constexpr int ACT = decltype(act)::value;
    const dim3 grid((unsigned)p.ns, (unsigned)n->samples), 
               all((unsigned)p.ns, (unsigned)n->samples + (!p.gather || (n->offsets && !p.zero) ? 1 : 0));
    if (p.lds_stats > 65536) {
      static std::atomic<unsigned long long> done{0};
      allow_dynamic_lds(gn_bwd_stats_kernel<T, ACT>, 131072, done);   // (1024 lanes of 2 x 8 sums)
    }
    gn_bwd_stats_kernel<T, ACT><<<grid, p.block, p.lds_stats, st>>>(a);
    if (!p.direct) gn_bwd_join_kernel<Unit<T>::N><<<dim3((unsigned)((n->channels + 7) / 8), (unsigned)n->samples), 256, 0, st>>>(a);
    if (nt)
      gn_bwd_apply_kernel<T, ACT, true><<<all, p.block, p.lds, st>>>(a);
    else
      gn_bwd_apply_kernel<T, ACT, false><<<all, p.block, p.lds, st>>>(a);
    if (p.gather && (dweight || dbias)) {
      const unsigned groups = (unsigned)((n->channels + 31) / 32);
      gn_bwd_gather_kernel<Unit<T>::N><<<dim3(groups, (unsigned)p.gather), 256, 0, st>>>(a);
      if (p.gather > 1) gn_bwd_channels_kernel<<<groups, 256, 0, st>>>(a, p.gather);
    }
    if (p.zero) gn_zero_kernel<T><<<(unsigned)p.zero, 256, 0, st>>>(a, (T *)dx, (T *)dresidual);
    return check_launch("gb_group_norm_bwd");
  });
}
