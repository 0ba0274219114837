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
// One mapping serves every pass and every channel count: a sample is ONE array of rows * C elements, a lane takes eight
// consecutive ones, and the lanes that work step by T * 8 elements, T the largest multiple of C / gcd(C, 8) in the workgroup.
// Then a lane meets the same eight channels at every step: its weights stay in registers, its sums need no index, loads
// are full 16-byte accesses for odd C as well, and no lane divides.
#include <type_traits>

#include "row_common.h"

#pragma clang fp contract(on)  // a * b + c in one instruction; the geometry kernels alone need the split form

namespace gb {

static constexpr int GN_MAX_C = 4096;   // two doubles per channel in LDS while a workgroup's sums are joined

struct GnShape {
  long long R;         // rows of the whole tensor
  long long rows;      // rows per sample (offs == nullptr)
  const long long *offs;
  int S, C, G, cpg;
  int P8, T;           // lanes of one period, lanes that work (a multiple of P8)
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
template <int ACT>
__device__ __forceinline__ float act_value(float z, float slope) {
  switch (ACT) {
    case GB_ACT_RELU: return z > 0.0f ? z : z != z ? z : 0.0f;
    case GB_ACT_LEAKY_RELU: return z > 0.0f ? z : slope * z;
    case GB_ACT_SILU: return z * sigmoid(z);
    case GB_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678f));
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
    case GB_ACT_GELU: return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * __expf(-0.5f * z * z) * 0.39894228f;
    default: return 1.0f;
  }
}

// The lane's place in the period: eight channels (8 p + k) mod C.
struct Lane {
  int p, r;       // place in the period, row of lanes
  bool on;
};
__device__ __forceinline__ Lane lane_place(const GnShape &sh) {
  Lane l;
  const int t = (int)threadIdx.x;
  l.r = t / sh.P8;
  l.p = t - l.r * sh.P8;
  l.on = t < sh.T;
  return l;
}
__device__ __forceinline__ int channel0(const GnShape &sh, int p) { return (int)((8ll * p) % sh.C); }
__device__ __forceinline__ int next_channel(const GnShape &sh, int c) { return c + 1 == sh.C ? 0 : c + 1; }

// Joins (v0, v1)[K] of the T working lanes per channel (K = 8) or per eight (K = 1) into out0 / out1, in a fixed order.
// buf: half of the lanes' values; out0, out1: C (K = 8) or P8 (K = 1) entries.  The lanes of one column are added as a
// tree; then the eight elements of a lane go to their channels one after another - at each of the eight steps every lane
// has another channel - because with C not a multiple of 8 a channel appears at several places of the period.
template <int K, typename A>
__device__ __forceinline__ void join_columns(const GnShape &sh, const Lane &l, A (&v0)[K], A (&v1)[K], A *buf, A *out0,
                                             A *out1) {
  const int RL = sh.T / sh.P8;
  int h = 1;
  while (2 * h < RL) h *= 2;
  if (RL > 1)
    for (; h >= 1; h >>= 1) {
      if (l.on && l.r >= h && l.r < 2 * h) {
        A *to = buf + (long long)((l.r - h) * sh.P8 + l.p) * 2 * K;
#pragma unroll
        for (int k = 0; k < K; ++k) to[2 * k] = v0[k], to[2 * k + 1] = v1[k];
      }
      __syncthreads();
      if (l.on && l.r < h && l.r + h < RL) {
        const A *from = buf + (long long)(l.r * sh.P8 + l.p) * 2 * K;
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
    int c = channel0(sh, l.p);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (l.on && l.r == 0) out0[c] += v0[k], out1[c] += v1[k];
      c = next_channel(sh, c);
      if (sh.C & 7) __syncthreads();
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

// Running count, mean and sum of squared deviations of a lane's eight columns (Chan, Golub, LeVeque: "Algorithms for
// computing the sample variance", 1983): four rows at a time, so that an offset of the data costs no bits.
struct Moments {
  float n;
  float mean[8], m2[8];
  __device__ void clear() {
    n = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) mean[k] = m2[k] = 0;
  }
  __device__ void add4(const F8 &a, const F8 &b, const F8 &c, const F8 &d) {
    const float f = 4.0f / (n + 4.0f), e = n * f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float m = 0.25f * ((a.v[k] + b.v[k]) + (c.v[k] + d.v[k]));
      const float da = a.v[k] - m, db = b.v[k] - m, dc = c.v[k] - m, dd = d.v[k] - m, del = m - mean[k];
      mean[k] += del * f;
      m2[k] += ((da * da + db * db) + (dc * dc + dd * dd)) + del * del * e;
    }
    n += 4.0f;
  }
  __device__ void add1(const F8 &a) {
    const float f = 1.0f / (n + 1.0f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float del = a.v[k] - mean[k];
      mean[k] += del * f;
      m2[k] += del * (a.v[k] - mean[k]);
    }
    n += 1.0f;
  }
};

// eights [j0, j1) * T of the sample for workgroup `chunk` of ns
__device__ __forceinline__ void chunk_range(const GnShape &sh, long long L, int chunk, long long &j0, long long &j1) {
  const long long J = ((L >> 3) + sh.T - 1) / sh.T, per = (J + sh.ns - 1) / sh.ns;
  j0 = per * chunk < J ? per * chunk : J;
  j1 = j0 + per < J ? j0 + per : J;
}

// Sums of x and x^2 per group from the lanes' columns and `tail`, single elements of them (zeros elsewhere); f as in
// for_group_sums.
template <typename F>
__device__ __forceinline__ void reduce_groups(const GnShape &sh, const Lane &l, const Moments &m, const F8 &tail, double *lds,
                                              F f) {
  if ((sh.cpg & 7) == 0) {  // a lane's eight channels are one group's (and a sample has no tail)
    double s1[1] = {0}, s2[1] = {0};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const double t = (double)m.n * m.mean[k];
      s1[0] += t;
      s2[0] += (double)m.m2[k] + t * m.mean[k];
    }
    join_columns<1, double>(sh, l, s1, s2, lds, lds, lds + sh.P8);
    for_group_sums(lds, lds + sh.P8, sh.G, sh.cpg >> 3, f);
  } else {
    double s1[8], s2[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const double t = (double)m.n * m.mean[k], e = tail.v[k];
      s1[k] = t + e;
      s2[k] = (double)m.m2[k] + t * m.mean[k] + e * e;
    }
    join_columns<8, double>(sh, l, s1, s2, lds, lds, lds + sh.C);
    for_group_sums(lds, lds + sh.C, sh.G, sh.cpg, f);
  }
}

extern __shared__ __attribute__((aligned(16))) unsigned char gn_lds[];

template <typename T>
__global__ __launch_bounds__(1024) void gn_stats_kernel(GnArgs a) {
  const GnShape &sh = a.sh;
  const int s = (int)blockIdx.y, chunk = (int)blockIdx.x;
  const Lane l = lane_place(sh);
  long long lo, hi, j0, j1;
  sample_rows(sh, s, lo, hi);
  const long long L = (hi - lo) * sh.C, NV = L >> 3;
  chunk_range(sh, L, chunk, j0, j1);
  const T *x = (const T *)a.x + lo * sh.C;
  Moments m;
  m.clear();
  if (l.on) {
    long long v = j0 * sh.T + threadIdx.x;
    const long long end = j1 * sh.T < NV ? j1 * sh.T : NV, step = sh.T;
    for (; v + 3 * step < end; v += 4 * step) {
      const Raw8<T> r0 = load_raw8(x + 8 * v), r1 = load_raw8(x + 8 * (v + step)), r2 = load_raw8(x + 8 * (v + 2 * step)),
                    r3 = load_raw8(x + 8 * (v + 3 * step));
      m.add4(widen(r0), widen(r1), widen(r2), widen(r3));
    }
    for (; v < end; v += step) m.add1(load8(x + 8 * v));
  }
  F8 tail = {};  // the sample's last L mod 8 elements
  if (chunk == 0 && (L & 7) && l.on && (int)threadIdx.x == (int)(NV % sh.T)) tail = load_tail(x + 8 * NV, (int)(L & 7));
  double *out = a.gpart + ((long long)s * sh.ns + chunk) * sh.G * 2;
  reduce_groups(sh, l, m, tail, reinterpret_cast<double *>(gn_lds), [&](int g, double t1, double t2) {
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

// one wave per (sample, group)
__global__ __launch_bounds__(64) void gn_finish_kernel(GnArgs a) {
  const GnShape &sh = a.sh;
  const int g = (int)blockIdx.x, s = (int)blockIdx.y, lane = (int)threadIdx.x;
  double t1 = 0, t2 = 0;
  for (int c = lane; c < sh.ns; c += 64) {
    const double *p = a.gpart + (((long long)s * sh.ns + c) * sh.G + g) * 2;
    t1 += p[0];
    t2 += p[1];
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) t1 += __shfl_xor(t1, o), t2 += __shfl_xor(t2, o);
  if (lane == 0) {
    long long lo, hi;
    sample_rows(sh, s, lo, hi);
    float mean = 0, rstd = 0;
    if (hi > lo) finish_group(t1, t2, (double)(hi - lo) * sh.cpg, a.eps, mean, rstd);
    a.mean[(long long)s * sh.G + g] = mean;
    a.rstd[(long long)s * sh.G + g] = rstd;
  }
}

// Eight elements from flat index i (of the whole tensor) through norm, activation and dropout; res: zeros where there is
// no residual.
struct Coef {  // of a lane's eight channels; a = rstd * w
  float mean[8], rstd[8], a[8], b[8];
};
__device__ __forceinline__ void load_coef(const GnShape &sh, const float *w, const float *b, int p, const float *mean,
                                          const float *rstd, Coef &co) {
  int c = channel0(sh, p);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int g = c / sh.cpg;
    co.mean[k] = mean[g];
    co.rstd[k] = rstd[g];
    co.a[k] = w ? co.rstd[k] * w[c] : co.rstd[k];
    co.b[k] = b ? b[c] : 0.0f;
    c = next_channel(sh, c);
  }
}
template <int ACT>
__device__ __forceinline__ F8 norm_act(const GnArgs &a, const Coef &co, const RowRng &rng, const F8 &x, const F8 &res,
                                       long long i) {
  F8 y;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float z = (x.v[k] - co.mean[k]) * co.a[k] + co.b[k];
    z += res.v[k];
    y.v[k] = act_value<ACT>(z, a.slope);
  }
  if (a.q) {
    const unsigned m = keep8(rng, (unsigned long long)i, a.q);
#pragma unroll
    for (int k = 0; k < 8; ++k) y.v[k] = (m >> k & 1) ? y.v[k] * a.scale : 0.0f;
  }
  return y;
}

// g and xh of eight elements
template <int ACT>
__device__ __forceinline__ void grad_act(const GnArgs &a, const Coef &co, const RowRng &rng, const F8 &x, const F8 &res,
                                         const F8 &dy, long long i, F8 &g, F8 &xh) {
  unsigned m = 0xff;
  if (a.q) m = keep8(rng, (unsigned long long)i, a.q);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float d0 = x.v[k] - co.mean[k];
    xh.v[k] = d0 * co.rstd[k];
    float z = d0 * co.a[k] + co.b[k];
    z += res.v[k];
    const float d = a.q ? ((m >> k & 1) ? dy.v[k] * a.scale : 0.0f) : dy.v[k];
    g.v[k] = d * act_slope<ACT>(z, a.slope);
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

template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_apply_kernel(GnArgs a) {
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
  if (!l.on) return;
  long long lo, hi, j0, j1;
  sample_rows(sh, s, lo, hi);
  const long long L = (hi - lo) * sh.C, NV = L >> 3, base = lo * sh.C;
  chunk_range(sh, L, chunk, j0, j1);
  const T *x = (const T *)a.x + base, *res = a.res ? (const T *)a.res + base : nullptr;
  T *y = (T *)a.y + base;
  Coef co;
  load_coef(sh, a.w, a.b, l.p, a.mean + (long long)s * sh.G, a.rstd + (long long)s * sh.G, co);
  const long long end = j1 * sh.T < NV ? j1 * sh.T : NV;
  for (long long v = j0 * sh.T + threadIdx.x; v < end; v += sh.T) {
    const F8 f = load8(x + 8 * v);
    F8 r = {};
    if (res) r = load8(res + 8 * v);
    store8(y + 8 * v, norm_act<ACT>(a, co, rng, f, r, base + 8 * v));
  }
  if (chunk == 0 && (L & 7) && (int)threadIdx.x == (int)(NV % sh.T)) {  // the sample's last L mod 8 elements
    const int n = (int)(L & 7);
    F8 r = {};
    if (res) r = load_tail(res + 8 * NV, n);
    store_tail(y + 8 * NV, norm_act<ACT>(a, co, rng, load_tail(x + 8 * NV, n), r, base + 8 * NV), n);
  }
}

// ---- samples whose columns fit a workgroup's registers ----------------------------------------------------------------
// A workgroup takes all rows of a sample and `sub` columns (whole groups: the fewest that make full 128-byte lines), keeps
// its eights in registers between the statistics and the output, and reads them once.  The period is that of the columns:
// place p of it is eight columns of a row, a step goes down T / P8 rows.  With C no multiple of 8 all columns are one
// workgroup's, as one flat array.
struct Sub {
  GnShape sh;       // the columns as a tensor of their own: C, G, P8, T
  long long base;   // first element
  int c0, g0;
  int first, step;  // of a lane, in elements from base
  int NV, tail;     // eights of the workgroup, elements behind the last of them
  double n;         // elements of a group
};
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
  if (W & 7) {
    u.NV = rows * W >> 3;
    u.tail = rows * W & 7;
    u.first = 8 * (int)threadIdx.x;
    u.step = 8 * a.sh.T;
  } else {
    u.NV = rows * a.sh.P8;
    u.tail = 0;
    u.first = l.r * a.sh.C + 8 * l.p;
    u.step = a.sh.T / a.sh.P8 * a.sh.C;
  }
  return u;
}
// Eights per lane: 32 registers of elements, what leaves 1024 lanes of 128 registers without spills.
template <typename T>
struct Held {
  static constexpr int N = 16 / (int)sizeof(T);
};

template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_small_kernel(GnArgs a) {
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
  constexpr int H = Held<T>::N;
  const Lane l = lane_place(a.sh);
  const Sub u = sub_of(a, s, part, l);
  const T *x = (const T *)a.x + u.base, *res = a.res ? (const T *)a.res + u.base : nullptr;
  T *y = (T *)a.y + u.base;
  const bool owns_tail = u.tail && l.on && (int)threadIdx.x == u.NV % u.sh.T;
  Raw8<T> held[H];
#pragma unroll
  for (int i = 0; i < H; ++i)
    if (l.on && (int)threadIdx.x + i * u.sh.T < u.NV) held[i] = load_raw8(x + (u.first + i * u.step));
  F8 t = {};
  if (owns_tail) t = load_tail(x + 8 * u.NV, u.tail);
  Moments m;
  m.clear();
#pragma unroll
  for (int i = 0; i < H; ++i)
    if (l.on && (int)threadIdx.x + i * u.sh.T < u.NV) m.add1(widen(held[i]));
  float *mean = a.mean + (long long)s * a.sh.G + u.g0, *rstd = a.rstd + (long long)s * a.sh.G + u.g0;
  reduce_groups(u.sh, l, m, t, reinterpret_cast<double *>(gn_lds), [&](int g, double t1, double t2) {
    float mu = 0, r = 0;
    if (u.n > 0) finish_group(t1, t2, u.n, a.eps, mu, r);
    mean[g] = mu;
    rstd[g] = r;
  });
  __threadfence_block();
  __syncthreads();
  if (!l.on) return;
  Coef co;
  load_coef(u.sh, a.w ? a.w + u.c0 : nullptr, a.b ? a.b + u.c0 : nullptr, l.p, mean, rstd, co);
#pragma unroll
  for (int i = 0; i < H; ++i)
    if ((int)threadIdx.x + i * u.sh.T < u.NV) {
      const int e = u.first + i * u.step;
      F8 r = {};
      if (res) r = load8(res + e);
      store8(y + e, norm_act<ACT>(a, co, rng, widen(held[i]), r, u.base + e));
    }
  if (owns_tail) {
    F8 r = {};
    if (res) r = load_tail(res + 8 * u.NV, u.tail);
    store_tail(y + 8 * u.NV, norm_act<ACT>(a, co, rng, t, r, u.base + 8 * u.NV), u.tail);
  }
}

// ---- backward -------------------------------------------------------------------------------------------------------

template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_bwd_stats_kernel(GnArgs a) {
  const GnShape &sh = a.sh;
  const int s = (int)blockIdx.y, chunk = (int)blockIdx.x;
  const RowRng rng = load_rng(a.rng, a.seed, a.call);
  const Lane l = lane_place(sh);
  long long lo, hi, j0, j1;
  sample_rows(sh, s, lo, hi);
  const long long L = (hi - lo) * sh.C, NV = L >> 3, base = lo * sh.C;
  chunk_range(sh, L, chunk, j0, j1);
  const T *x = (const T *)a.x + base, *dy = (const T *)a.dy + base, *res = a.res ? (const T *)a.res + base : nullptr;
  float sg[8] = {}, sx[8] = {};
  if (l.on) {
    Coef co;
    load_coef(sh, a.w, a.b, l.p, a.mean + (long long)s * sh.G, a.rstd + (long long)s * sh.G, co);
    const long long end = j1 * sh.T < NV ? j1 * sh.T : NV;
    for (long long v = j0 * sh.T + threadIdx.x; v < end; v += sh.T) {
      const F8 f = load8(x + 8 * v), d = load8(dy + 8 * v);
      F8 r = {}, g, xh;
      if (res) r = load8(res + 8 * v);
      grad_act<ACT>(a, co, rng, f, r, d, base + 8 * v, g, xh);
#pragma unroll
      for (int k = 0; k < 8; ++k) sg[k] += g.v[k], sx[k] += g.v[k] * xh.v[k];
    }
    if (chunk == 0 && (L & 7) && (int)threadIdx.x == (int)(NV % sh.T)) {
      const int n = (int)(L & 7);
      F8 r = {}, g, xh;
      if (res) r = load_tail(res + 8 * NV, n);
      grad_act<ACT>(a, co, rng, load_tail(x + 8 * NV, n), r, load_tail(dy + 8 * NV, n), base + 8 * NV, g, xh);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < n) sg[k] += g.v[k], sx[k] += g.v[k] * xh.v[k];
    }
  }
  float *lds = reinterpret_cast<float *>(gn_lds);
  join_columns<8, float>(sh, l, sg, sx, lds, lds, lds + sh.C);
  float2 *out = reinterpret_cast<float2 *>(a.cpart) + ((long long)s * sh.ns + chunk) * sh.C;
  for (int c = (int)threadIdx.x; c < sh.C; c += (int)blockDim.x) out[c] = make_float2(lds[c], lds[sh.C + c]);
}

// The workgroups' sums of a sample, joined: 32 channels x 8 lanes over the workgroups, in 64 bits.
__global__ __launch_bounds__(256) void gn_bwd_join_kernel(GnArgs a) {
  __shared__ double part[2][8][32];
  const GnShape &sh = a.sh;
  const int s = (int)blockIdx.y, c = (int)blockIdx.x * 32 + ((int)threadIdx.x & 31), q = (int)threadIdx.x >> 5;
  double s0 = 0, s1 = 0;
  if (c < sh.C)
    for (int i = q; i < sh.ns; i += 8) {
      const float2 f = reinterpret_cast<const float2 *>(a.cpart)[((long long)s * sh.ns + i) * sh.C + c];
      s0 += f.x;
      s1 += f.y;
    }
  part[0][q][threadIdx.x & 31] = s0;
  part[1][q][threadIdx.x & 31] = s1;
  __syncthreads();
  if (q == 0 && c < sh.C) {
    for (int i = 1; i < 8; ++i) s0 += part[0][i][threadIdx.x], s1 += part[1][i][threadIdx.x];
    reinterpret_cast<float2 *>(a.csum)[(long long)s * sh.C + c] = make_float2((float)s0, (float)s1);
  }
}

// dw, db = the samples' sums added, by workgroup `part` of `parts`: 32 channels x blockDim / 32 lanes over the samples
__device__ __forceinline__ void channel_gradients(const GnArgs &a, int part, int parts) {
  const GnShape &sh = a.sh;
  double *lds = reinterpret_cast<double *>(gn_lds);
  const int i = (int)threadIdx.x & 31, q = (int)threadIdx.x >> 5, Q = (int)blockDim.x >> 5;
  for (int c0 = part * 32; c0 < sh.C; c0 += parts * 32) {
    const int c = c0 + i;
    double s0 = 0, s1 = 0;
    if (c < sh.C)
      for (int s = q; s < sh.S; s += Q) {
        const float2 f = reinterpret_cast<const float2 *>(a.csum)[(long long)s * sh.C + c];
        s0 += f.x;
        s1 += f.y;
      }
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

__device__ __forceinline__ F8 grad_x(const Coef &co, const F8 &g, const F8 &xh, const float (&c1)[8], const float (&c2)[8]) {
  F8 o;
#pragma unroll
  for (int k = 0; k < 8; ++k) o.v[k] = co.a[k] * g.v[k] - c1[k] - xh.v[k] * c2[k];
  return o;
}

template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_bwd_apply_kernel(GnArgs a) {
  const GnShape &sh = a.sh;
  const int s = (int)blockIdx.y, chunk = (int)blockIdx.x;
  if (s == sh.S) {
    channel_gradients(a, chunk, sh.ns);
    if (sh.offs) zero_outside<T>(sh, (T *)a.dx, (T *)a.dres, chunk, sh.ns);
    return;
  }
  const RowRng rng = load_rng(a.rng, a.seed, a.call);
  const Lane l = lane_place(sh);
  long long lo, hi, j0, j1;
  sample_rows(sh, s, lo, hi);
  const long long L = (hi - lo) * sh.C, NV = L >> 3, base = lo * sh.C;
  chunk_range(sh, L, chunk, j0, j1);
  if (L == 0) return;
  float *v0 = reinterpret_cast<float *>(gn_lds), *v1 = v0 + sh.C, *k1 = v1 + sh.C, *k2 = k1 + sh.G;
  for (int c = (int)threadIdx.x; c < sh.C; c += (int)blockDim.x) {
    const float2 f = reinterpret_cast<const float2 *>(a.csum)[(long long)s * sh.C + c];
    v0[c] = f.x;
    v1[c] = f.y;
  }
  group_terms(a, v0, v1, k1, k2, (double)(hi - lo) * sh.cpg);
  if (!l.on) return;
  Coef co;
  load_coef(sh, a.w, a.b, l.p, a.mean + (long long)s * sh.G, a.rstd + (long long)s * sh.G, co);
  float c1[8], c2[8];
  int c = channel0(sh, l.p);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    c1[k] = co.rstd[k] * k1[c / sh.cpg];
    c2[k] = co.rstd[k] * k2[c / sh.cpg];
    c = next_channel(sh, c);
  }
  const T *x = (const T *)a.x + base, *dy = (const T *)a.dy + base, *res = a.res ? (const T *)a.res + base : nullptr;
  T *dx = (T *)a.dx + base, *dres = a.dres ? (T *)a.dres + base : nullptr;
  const long long end = j1 * sh.T < NV ? j1 * sh.T : NV;
  for (long long v = j0 * sh.T + threadIdx.x; v < end; v += sh.T) {
    const F8 f = load8(x + 8 * v), d = load8(dy + 8 * v);
    F8 r = {}, g, xh;
    if (res) r = load8(res + 8 * v);
    grad_act<ACT>(a, co, rng, f, r, d, base + 8 * v, g, xh);
    store8(dx + 8 * v, grad_x(co, g, xh, c1, c2));
    if (dres) store8(dres + 8 * v, g);
  }
  if (chunk == 0 && (L & 7) && (int)threadIdx.x == (int)(NV % sh.T)) {
    const int n = (int)(L & 7);
    F8 r = {}, g, xh;
    if (res) r = load_tail(res + 8 * NV, n);
    grad_act<ACT>(a, co, rng, load_tail(x + 8 * NV, n), r, load_tail(dy + 8 * NV, n), base + 8 * NV, g, xh);
    store_tail(dx + 8 * NV, grad_x(co, g, xh, c1, c2), n);
    if (dres) store_tail(dres + 8 * NV, g, n);
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------

static int gcd8(int c) { return c % 8 == 0 ? 8 : c % 4 == 0 ? 4 : c % 2 == 0 ? 2 : 1; }

struct GnPlan {
  int block, P8, T, ns;
  int sub;   // columns per workgroup of the one-pass kernel; 0: the sample is read twice
  size_t lds, ws;
};

static int lds_tree(int T, int P8) {  // join_columns: most lanes that give theirs away at a step (RL - h first, then h / 2, ...)
  const int RL = T / P8;
  int h = 1;
  while (2 * h < RL) h *= 2;
  return RL > 1 ? (RL - h > h / 2 ? RL - h : h / 2) * P8 : 0;
}

static GnPlan gn_plan(const GbGroupNorm *n, bool backward) {
  GnPlan p;
  const long long longest = n->offsets ? n->rows : n->rows / n->samples;
  const int C = n->channels, cpg = C / n->groups, size = n->dtype == GB_T_F32 ? 4 : 2;
  p.sub = 0;
  if (!backward) {
    // The one-pass kernel wherever a sample's columns fit: no second read and one launch instead of three.  Columns: all
    // of them when C is no multiple of 8, else the fewest whole groups that divide C into full 128-byte lines of eights.
    int sub = C;
    if (C % 8 == 0)
      for (int gs = 1; gs <= n->groups; ++gs)
        if (n->groups % gs == 0 && gs * cpg % 8 == 0 && gs * cpg * size >= 128) {
          sub = gs * cpg;
          break;
        }
    const int P8 = sub / gcd8(sub), T = P8 <= 1024 ? 1024 / P8 * P8 : 0;
    if (T && longest * sub / 8 < (long long)T * (16 / size)) {
      p.sub = sub;
      p.P8 = P8;
      // (lanes for one eight each, in whole waves: latency counts more than what a lane could hold)
      const long long eights = (longest * sub + 7) / 8;
      p.block = P8 <= 256 && eights <= 256 ? 256 : P8 <= 512 && eights <= 512 ? 512 : 1024;
      p.ns = C / sub;
    }
  }
  if (!p.sub) {
    // Lanes: 256 where a period fits (more workgroups per CU to change between), else 512 or 1024.  A sample is spread
    // over enough workgroups that a lane meets ~16 eights (64 KB of fp32 per workgroup keep the joining of the sums below
    // 2 % of the pass) but the device has ~2048 in all; packed samples may be of very different lengths and are cut finer.
    p.P8 = C / gcd8(C);
    p.block = p.P8 <= 256 ? 256 : p.P8 <= 512 ? 512 : 1024;
    const int T = p.block / p.P8 * p.P8;
    const long long eights = (longest * C + 7) / 8, steps = (eights + T - 1) / T;
    long long ns = (steps + 15) / 16;
    const long long fill = n->offsets ? 8192 : 2048, most = (fill + n->samples - 1) / n->samples;
    if (ns > most) ns = most;
    p.ns = (int)(ns < 1 ? 1 : ns);
  }
  p.T = p.block / p.P8 * p.P8;
  const size_t cell = backward ? sizeof(float) : sizeof(double);
  const int K = !backward && cpg % 8 == 0 ? 1 : 8;
  const size_t tree = (size_t)lds_tree(p.T, p.P8) * 2 * K * cell, flat = (size_t)(K == 1 ? p.P8 : p.sub ? p.sub : C) * 2 * cell;
  p.lds = tree > flat ? tree : flat;
  if (backward) {
    const size_t apply = (size_t)(C + n->groups) * 2 * sizeof(float);
    if (apply > p.lds) p.lds = apply;
    const size_t joined = (size_t)p.block * 2 * sizeof(double);  // (channel_gradients)
    if (joined > p.lds) p.lds = joined;
    p.ws = ((size_t)n->samples * p.ns + n->samples) * C * 2 * sizeof(float);
  } else {
    p.ws = p.sub ? 0 : (size_t)n->samples * p.ns * n->groups * 2 * sizeof(double);
  }
  return p;
}

static int gn_bad(const GbGroupNorm *n) {
  if (!n || n->rows < 0 || n->samples <= 0 || n->channels <= 0 || n->groups <= 0 || n->channels % n->groups) return GB_EINVAL;
  if (!known_type(n->dtype) || n->act < 0 || n->act > GB_ACT_GELU || n->q < 0 || n->q > 65536 || !(n->eps >= 0)) return GB_EINVAL;
  if (!n->offsets && n->rows % n->samples) return GB_EINVAL;
  if (n->channels > GN_MAX_C || n->channels / gcd8(n->channels) > 1024 || n->samples > 65534) return GB_ERANGE;
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
  a.sh.P8 = p.P8;
  a.sh.T = p.T;
  a.sh.ns = p.ns;
  a.sub = p.sub;
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
  const dim3 all((unsigned)p.ns, (unsigned)(n->samples + (n->offsets ? 1 : 0)));
  return with_type_and_act(n, [&](auto z, auto act) {
    typedef decltype(z) T;
    constexpr int ACT = decltype(act)::value;
    if (p.sub) {
      gn_small_kernel<T, ACT><<<all, p.block, p.lds, st>>>(a);
    } else {
      gn_stats_kernel<T><<<dim3((unsigned)p.ns, (unsigned)n->samples), p.block, p.lds, st>>>(a);
      gn_finish_kernel<<<dim3((unsigned)n->groups, (unsigned)n->samples), 64, 0, st>>>(a);
      gn_apply_kernel<T, ACT><<<all, p.block, 0, st>>>(a);
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
  hipStream_t st = as_stream(stream);
  return with_type_and_act(n, [&](auto z, auto act) {
    typedef decltype(z) T;
    constexpr int ACT = decltype(act)::value;
    gn_bwd_stats_kernel<T, ACT><<<dim3((unsigned)p.ns, (unsigned)n->samples), p.block, p.lds, st>>>(a);
    gn_bwd_join_kernel<<<dim3((unsigned)((n->channels + 31) / 32), (unsigned)n->samples), 256, 0, st>>>(a);
    gn_bwd_apply_kernel<T, ACT><<<dim3((unsigned)p.ns, (unsigned)n->samples + 1), p.block, p.lds, st>>>(a);
    return check_launch("gb_group_norm_bwd");
  });
}
