// Products in 8-bit floats with a power-of-two scale for each block of 128 (graspbal.h gb_fp8_*).
//
//   Y = deq(Q(X)) deq(Q(W))^T + bias;   dX = deq(Q(dY)) deq(Q(W));   dW = deq(Q(dY))^T deq(Q(X));   db = sum of dY
//
// Q of a block: e = the least integer with max|x| <= 448 2^e over the block's finite values (at least -126; 0 for a block of
// zeros), codes = e4m3(x 2^-e).  X and dY have a block per 128 elements of a row, W per 128 x 128.  A power of two costs a
// floating format nothing (scaling by it is exact), is what the matrix instructions take beside their operands, and is
// exact in bf16.
//
// Two inner products:
//   EXACT (fp32 outputs, and 16-bit ones unless the caller asks for the other): the codes are turned into bf16 (exact) in
//     registers, scale included, and go through v_mfma_f32_32x32x16_bf16, whose sums are fp32 (1.76 PFLOP/s on this card with
//     random values; 8e-8 of the result's norm).
//   GB_FP8_SHORT_SUMS (16-bit outputs): v_mfma_scale_f32_32x32x64_f8f6f4 - 4.0 PFLOP/s with random codes (4.7 with zeros: the
//     clock falls with the power), scales applied by the instruction.  It adds the products of a step of 64 or 128 with
//     about 14 bits below the largest one, then accumulates in fp32: measured 5e-5 of the result's norm for codes over the
//     whole range, 0 where they span 2^4 - a twentieth of bf16's half step, a quarter of fp16's.  Fewer than 32 bits of a sum
//     are the caller's choice, so this form is never taken unasked.
#include <type_traits>

#include "row_common.h"

#pragma clang fp contract(on)

namespace gb {

// the quantisers' eight elements per lane (sixteen lanes = a block of 128)
typedef Vec<8> F8;
template <typename T>
__device__ __forceinline__ F8 load_upto8(const T *p, int n) {   // n <= 0: nothing is read
  F8 f = {};
  if (n >= 8) {
    T v[8];
    __builtin_memcpy(v, p, sizeof(v));
#pragma unroll
    for (int k = 0; k < 8; ++k) f.v[k] = (float)v[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) f.v[k] = (float)p[k];
  }
  return f;
}

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

static constexpr int FP8_FEW_ROWS = 64;          // rows up to which the products run without LDS tiles
static constexpr int FP8_FUSED_CODES = 16384;    // bytes of codes a workgroup quantises for itself
static constexpr int FP8_FUSED_ROWS = 16;

__host__ __device__ inline int blocks128(int k) { return (k + 127) / 128; }
__host__ __device__ inline int scale_stride(int k) { return (blocks128(k) + 3) / 4 * 4; }   // whole dwords per row

// ---- quantisers -----------------------------------------------------------------------------------------------------

// biased exponent (e + 127) of a block whose largest finite magnitude is `top`: 448 = 1.75 * 2^8
__device__ __forceinline__ int block_exponent(float top) {
  const unsigned b = __float_as_uint(top);
  if (b == 0) return 127;
  const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < 1 ? 1 : e;
}
__device__ __forceinline__ float power_of(int biased) { return __uint_as_float((unsigned)biased << 23); }  // 1 <= biased <= 254
__device__ __forceinline__ float finite_magnitude(float x) {
  const float a = fabsf(x);
  return a <= 3.4028235e38f ? a : 0.0f;
}
__device__ __forceinline__ float top8(const F8 &f) {
  float m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_magnitude(f.v[k]));
  return m;
}
// eight codes; x * 2^-e is exact wherever it reaches the codes' range; what is not finite becomes NaN
__device__ __forceinline__ uint2 encode8(const F8 &f, int biased) {
  const float inv = power_of(254 - biased);
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = fabsf(f.v[k]) <= 3.4028235e38f ? f.v[k] * inv : __uint_as_float(0x7fc00000u);
  uint2 r;
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  r.x = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  r.y = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  return r;
}
// Rows [r0, r0 + per) x block kb of 128 columns: sixteen lanes x eight elements a row.  SUM: also the column sums of these
// rows, fp32 over per / 16 rows a lane (64 at most) joined in 64 bits, to part[chunk][K].
template <typename T, bool SUM>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T *__restrict__ x, long long P, int K, unsigned char *__restrict__ codes,
                                                       unsigned char *__restrict__ scales, int per, float *__restrict__ part) {
  const int cl = (int)threadIdx.x & 15, rl = (int)threadIdx.x >> 4, kb = (int)blockIdx.y, col = kb * 128 + cl * 8;
  const long long r0 = (long long)blockIdx.x * per, r1 = r0 + per < P ? r0 + per : P;
  const int Kp = blocks128(K) * 128, ss = scale_stride(K), n = K - col;
  F8 sum = {};
  for (long long r = r0 + rl; r < r1; r += 16) {
    const F8 f = load_upto8(x + r * K + col, n);
    const int e = block_exponent(row_max_f32(top8(f)));
    *reinterpret_cast<uint2 *>(codes + r * Kp + col) = encode8(f, e);
    if (cl == 0) scales[r * ss + kb] = (unsigned char)e;
    if (SUM)
#pragma unroll
      for (int k = 0; k < 8; ++k) sum.v[k] += f.v[k];
  }
  if (SUM) {
    __shared__ float lds[16][128];
#pragma unroll
    for (int k = 0; k < 8; ++k) lds[rl][cl * 8 + k] = sum.v[k];
    __syncthreads();
    const int c = (int)threadIdx.x;
    if (c < 128 && kb * 128 + c < K) {
      double s = 0;
      for (int i = 0; i < 16; ++i) s += lds[i][c];
      part[(long long)blockIdx.x * K + kb * 128 + c] = (float)s;
    }
  }
}

// the workgroups' sums of a column, joined: 8 columns x 32 lanes, in 64 bits
__global__ __launch_bounds__(256) void fp8_colsum_kernel(const float *__restrict__ part, int chunks, int K, float *__restrict__ out) {
  __shared__ double lds[32][8];
  const int i = (int)threadIdx.x & 7, q = (int)threadIdx.x >> 3, c = (int)blockIdx.x * 8 + i;
  double s = 0;
  if (c < K)
#pragma unroll 4
    for (int j = q; j < chunks; j += 32) s += part[(long long)j * K + c];
  lds[q][i] = s;
  __syncthreads();
  if (q == 0 && c < K) {
    for (int j = 1; j < 32; ++j) s += lds[j][i];
    out[c] = (float)s;
  }
}

// One 128 x 128 block of a weight: codes (N, Kp) and, for the product with dY, codes_t (K, Np); one exponent.
template <typename T>
__global__ __launch_bounds__(256) void fp8_weight_kernel(const T *__restrict__ w, int N, int K, unsigned char *__restrict__ codes,
                                                         unsigned char *__restrict__ codes_t, unsigned char *__restrict__ scales) {
  __shared__ float top[4];
  __shared__ unsigned char tile[128][136];
  const int cl = (int)threadIdx.x & 15, rl = (int)threadIdx.x >> 4, kb = (int)blockIdx.x, nb = (int)blockIdx.y;
  const int Kb = blocks128(K), Np = blocks128(N) * 128, col = kb * 128 + cl * 8;
  F8 f[8];
  float m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = nb * 128 + i * 16 + rl;
    f[i] = load_upto8(w + (long long)n * K + col, n < N ? K - col : 0);
    m = fmaxf(m, top8(f[i]));
  }
  m = wave_max_f32(m);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
  const int e = block_exponent(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
  if (threadIdx.x == 0) scales[nb * Kb + kb] = (unsigned char)e;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = i * 16 + rl;
    const uint2 c = encode8(f[i], e);
    if (nb * 128 + n < N) *reinterpret_cast<uint2 *>(codes + (long long)(nb * 128 + n) * (Kb * 128) + col) = c;
    if (codes_t) *reinterpret_cast<uint2 *>(&tile[n][cl * 8]) = c;
  }
  if (!codes_t) return;
  __syncthreads();
  const int k = (int)threadIdx.x >> 1, h = ((int)threadIdx.x & 1) * 64;
  if (kb * 128 + k < K)
    for (int j = 0; j < 64; j += 16) {
      unsigned v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = h + j + 4 * q;
        v[q] = tile[n][k] | tile[n + 1][k] << 8 | tile[n + 2][k] << 16 | (unsigned)tile[n + 3][k] << 24;
      }
      *reinterpret_cast<uint4 *>(codes_t + (long long)(kb * 128 + k) * Np + nb * 128 + h + j) = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

// ---- fragments ------------------------------------------------------------------------------------------------------

// Codes 8j .. 8j+7 of a lane's 32 as bf16 times 2^scale (exact): one operand of a 32x32x16 / 16x16x32 bf16 step.  Which
// element of the reduction a lane holds does not matter as long as both operands hold the same one.
__device__ __forceinline__ bf16x8 decode8(unsigned lo, unsigned hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true),
               c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  bf16x8 r;
  r[0] = a[0], r[1] = a[1], r[2] = b[0], r[3] = b[1], r[4] = c[0], r[5] = c[1], r[6] = d[0], r[7] = d[1];
  return r;
}

// 64 codes of the reduction into TM x TN tiles: fa, fb are a lane's 32 codes of its rows, sa, sb their biased exponents
template <bool EXACT, int TM, int TN>
__device__ __forceinline__ void multiply64(f32x16 (&acc)[TM][TN], const i32x4 (&fa)[TM][2], const i32x4 (&fb)[TN][2], const int (&sa)[TM],
                                           int sb) {
  if (EXACT) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      bf16x8 db[TN];
#pragma unroll
      for (int n = 0; n < TN; ++n)
        db[n] = decode8((unsigned)fb[n][q / 2][q % 2 * 2], (unsigned)fb[n][q / 2][q % 2 * 2 + 1], power_of(sb));
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        const bf16x8 da = decode8((unsigned)fa[m][q / 2][q % 2 * 2], (unsigned)fa[m][q / 2][q % 2 * 2 + 1], power_of(sa[m]));
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(da, db[n], acc[m][n], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const i32x8 va = __builtin_shufflevector(fa[m][0], fa[m][1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int n = 0; n < TN; ++n) {
        const i32x8 vb = __builtin_shufflevector(fb[n][0], fb[n][1], 0, 1, 2, 3, 4, 5, 6, 7);
        acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, acc[m][n], 0, 0, 0, sa[m], 0, sb);
      }
    }
  }
}

// The same for 128 codes from LDS: la, lb are the lane's rows of the operands (128 bytes each, chunks permuted as below).
template <bool EXACT, int TM, int TN>
__device__ __forceinline__ void multiply128(f32x16 (&acc)[TM][TN], const unsigned char *la, const unsigned char *lb, int lane,
                                            const int (&sa)[TM], int sb) {
  const int h = lane >> 5, x = lane >> 1 & 7;
#pragma unroll
  for (int s = 0; s < 2; ++s) {   // 64 codes: lane half h holds 32 of them
    const int c0 = ((4 * s + 2 * h) ^ x) * 16, c1 = ((4 * s + 2 * h + 1) ^ x) * 16;
    i32x4 fa[TM][2], fb[TN][2];
#pragma unroll
    for (int n = 0; n < TN; ++n) {
      const unsigned char *r = lb + 32 * n * 128;
      fb[n][0] = *reinterpret_cast<const i32x4 *>(r + c0);
      fb[n][1] = *reinterpret_cast<const i32x4 *>(r + c1);
    }
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const unsigned char *r = la + 32 * m * 128;
      fa[m][0] = *reinterpret_cast<const i32x4 *>(r + c0);
      fa[m][1] = *reinterpret_cast<const i32x4 *>(r + c1);
    }
    multiply64<EXACT, TM, TN>(acc, fa, fb, sa, sb);
  }
}

// A wave's results to memory: lane j of a pair of tiles has columns 2 j, 2 j + 1 of 64 (from col0 of N) and, of every eight
// rows, 4 h .. 4 h + 3.  Eight rows at a time go through the wave's own LDS cell and leave as 16 bytes per lane, whole
// 128-byte lines: stored from where they are (4 bytes a lane) they took 75 of the 120 us of 524288 x 128 -> 256 bf16.
// `rows` of the tile exist.  (A tile's offsets fit 32 unsigned bits: 256 rows of 2^22 fp32.)
template <typename T>
struct Cell {
  static constexpr int ROW = 64 * (int)sizeof(T) + 16, BYTES = 8 * ROW;
};
template <typename T, int TM, int TN, bool NT>
__device__ __forceinline__ void store_tiles(const f32x16 (&acc)[TM][TN], T *y, const float *bias, int N, int col0, int row0, int lane, int rows,
                                            unsigned char *cell) {
  constexpr int ROW = Cell<T>::ROW, E = 16 / (int)sizeof(T), CH = 64 / E;   // elements of an access, accesses of a row
  const int j = lane & 31, h = lane >> 5;
#pragma unroll
  for (int n = 0; n < TN; n += 2) {
    const int base = col0 + 32 * n, col = base + 2 * j;
    if (base >= N) break;
    const float b0 = bias && col < N ? bias[col] : 0.0f, b1 = bias && col + 1 < N ? bias[col + 1] : 0.0f;
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const T v[2] = {(T)(acc[m][n][4 * q + i] + b0), (T)(acc[m][n + 1][4 * q + i] + b1)};
          __builtin_memcpy(cell + (4 * h + i) * ROW + 2 * j * (int)sizeof(T), v, sizeof(v));
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int t = 0; t < 8 * CH / 64; ++t) {
          const int at = t * 64 + lane, r = at / CH, c = base + at % CH * E, row = row0 + 32 * m + 8 * q + r;
          typedef unsigned u4 __attribute__((ext_vector_type(4)));
          const u4 w = *reinterpret_cast<const u4 *>(cell + r * ROW + at % CH * 16);
          if (row >= rows || c >= N) continue;
          T *to = reinterpret_cast<T *>(reinterpret_cast<unsigned char *>(y) + ((unsigned)row * (unsigned)N + (unsigned)c) * (unsigned)sizeof(T));
          if (c + E <= N) {
            if (NT)
              __builtin_nontemporal_store((u32x4_any)w, reinterpret_cast<u32x4_any *>(to));
            else
              __builtin_memcpy(to, &w, 16);
          } else {
            T v[E];
            __builtin_memcpy(v, &w, 16);
#pragma unroll
            for (int k = 0; k < E; ++k)
              if (c + k < N) to[k] = v[k];
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
  }
}

// ---- tiles ----------------------------------------------------------------------------------------------------------
// A workgroup of WM x WN waves, each with TM x TN tiles of 32 x 32, steps through the reduction 128 codes (one scale block)
// at a time: two LDS stages filled by LDS-DMA, the next one in flight while this one is multiplied.  An LDS row is 128
// codes, eight chunks of 16 bytes; chunk c of row r lies at place c ^ (r >> 1 & 7) (the DMA writes lane-linearly, so the
// lane's SOURCE is permuted), which spreads the sixteen rows that are read in a cycle over all 64 banks.  The tiles of W come
// in pairs, and lane j of a pair takes rows 2j and 2j + 1 of its 64, so that a lane ends up with two neighbouring outputs: in
// LDS the even rows of each 64 come first.

struct GemmArgs8 {
  const unsigned char *a, *a_scales, *b, *b_scales;  // a (P, Kp), b (N, Kp); a_scales (P, stride), b_scales by block
  const float *bias;
  void *y;
  long long P;
  int N, Kb, a_stride, bs_n, bs_k, tiles_n;
  long long tiles;
};

__device__ __forceinline__ void dma16(const unsigned char *src, unsigned char *lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src, (__attribute__((address_space(3))) void *)lds,
                                   16, 0, 0);
}

// the row of W at place `at` of LDS
__device__ __forceinline__ int weight_row(int at) { return (at & ~63) + 2 * (at & 31) + (at >> 5 & 1); }

// G > 1 (few tiles, a long reduction): G groups of WM x WN waves with stages of their own take a range of the steps each, and
// their sums meet in LDS, added in the groups' order.  A lone group is bound by its own steps, one after the other (~0.6 us
// each: waits for LDS and the matrix pipe; four stages in flight instead of two gained 3 us in 21 with the 8-bit instructions and
// lost as much with bf16 products).  128 x 4096 -> 4096 with its quantiser bf16 25.3 -> 16.1 us, fp32 26.1 -> 16.7; 512 x 1024 -> 1024
// bf16 9.8 -> 8.5.
template <typename T, bool EXACT, int TM, int TN, int WM, int WN, int G, bool NT>
__global__ __launch_bounds__(64 * WM * WN * G) void fp8_gemm_kernel(GemmArgs8 g) {
  constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, WAVES = WM * WN, ROWS = BM + BN, LOADS = ROWS / (8 * WAVES);
  static_assert(TN % 2 == 0 && ROWS % (8 * WAVES) == 0 && (32 * TN) <= 128, "tile");
  static_assert((G - 1) * WAVES * TM * TN * 4096 + WAVES * Cell<T>::BYTES <= G * 2 * ROWS * 128, "the groups' sums");
  extern __shared__ __attribute__((aligned(128))) unsigned char lds[];   // per group: one stage, or two where there is a second step
  const int lane = (int)threadIdx.x & 63, at = (int)threadIdx.x >> 6, group = at / WAVES, wave = at % WAVES, wm = wave / WN, wn = wave % WN,
            j = lane & 31;
  unsigned char *stages = lds + group * (2 * ROWS * 128);
  // neighbouring tiles on one XCD (workgroups go to the eight XCDs in turn): its L2 then holds their common rows
  const long long per = g.tiles >> 3, extra = g.tiles & 7, x = blockIdx.x & 7;
  const long long tile = x * per + (x < extra ? x : extra) + (blockIdx.x >> 3);
  const long long p0 = tile / g.tiles_n * BM;
  const int n0 = (int)(tile % g.tiles_n) * BN, Kp = g.Kb * 128;
  const unsigned char *a = g.a + p0 * Kp, *b = g.b + (long long)n0 * Kp;
  const int last_a = (int)(g.P - p0 < BM ? g.P - p0 : BM) - 1, last_b = (g.N - n0 < BN ? g.N - n0 : BN) - 1;

  // the lane's share of a stage: 16 bytes of LOADS rows (rows behind the last repeat it; their outputs are not stored)
  int off[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = (i * WAVES + wave) * 8 + (lane >> 3);
    const bool of_a = row < BM;
    const int at = of_a ? row : row - BM, r = of_a ? at : weight_row(at), last = of_a ? last_a : last_b;
    off[i] = (r < last ? r : last) * Kp + ((lane & 7) ^ (at >> 1 & 7)) * 16;
  }
  auto request = [&](int kb, unsigned char *stage) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int first = (i * WAVES + wave) * 8;
      dma16((first < BM ? a : b) + off[i] + kb * 128, stage + first * 128);
    }
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int n = 0; n < TN; ++n) acc[m][n] = f32x16{};
  const int steps = G > 1 ? ((g.Kb + G - 1) / G + 3) / 4 * 4 : g.Kb;   // (a range starts with a dword of four exponents)
  const int k0 = G > 1 ? group * steps : 0, k1 = G > 1 && k0 + steps < g.Kb ? k0 + steps : g.Kb;
  const unsigned char *as[TM];
  unsigned sa[TM], sa_next[TM];
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int r = wm * 32 * TM + 32 * m + j;
    as[m] = g.a_scales + (p0 + (r < last_a ? r : last_a)) * g.a_stride;
  }
  const int nb = (n0 + wn * 32 * TN) / 128, nbs = nb < (g.N + 127) / 128 ? nb : (g.N + 127) / 128 - 1;
  const unsigned char *bs = g.b_scales + (long long)nbs * g.bs_n;
  unsigned sb_next = 0;
  if (k0 < k1) {
    request(k0, stages);
#pragma unroll
    for (int m = 0; m < TM; ++m) sa_next[m] = *reinterpret_cast<const unsigned *>(as[m] + k0);
    sb_next = bs[(long long)k0 * g.bs_k];
  }
  for (int i = 0; i < steps; ++i) {
    const int kb = k0 + i;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();   // this stage is complete, and nobody reads the other one any more
    if (G > 1 && kb >= k1) continue;   // (the last group's range may be shorter)
    const unsigned sb = sb_next;
    if ((kb & 3) == 0)
#pragma unroll
      for (int m = 0; m < TM; ++m) sa[m] = sa_next[m];
    if (kb + 1 < k1) {   // the next step's codes and exponents travel while this one is multiplied
      request(kb + 1, stages + ((i + 1) & 1) * (ROWS * 128));
      sb_next = bs[(long long)(kb + 1) * g.bs_k];
      if ((kb & 3) == 3)
#pragma unroll
        for (int m = 0; m < TM; ++m) sa_next[m] = *reinterpret_cast<const unsigned *>(as[m] + kb + 1);
    }
    const unsigned char *st = stages + (i & 1) * (ROWS * 128);
    int s8[TM];
#pragma unroll
    for (int m = 0; m < TM; ++m) s8[m] = (int)(sa[m] >> (8 * (kb & 3)) & 0xff);
    multiply128<EXACT, TM, TN>(acc, st + (wm * 32 * TM + j) * 128, st + (BM + wn * 32 * TN + j) * 128, lane, s8, (int)sb);
  }
  __syncthreads();   // (the stages become the groups' sums, then the waves' cells)
  if (G > 1) {
    f32x4 *sums = reinterpret_cast<f32x4 *>(lds) + wave * (TM * TN * 256) + lane;   // [group - 1][wave][tile][quarter][lane]
    if (group > 0)
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            sums[(group - 1) * (WAVES * TM * TN * 256) + ((m * TN + n) * 4 + q) * 64] =
                f32x4{acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]};
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int o = 0; o < G - 1; ++o)
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 v = sums[o * (WAVES * TM * TN * 256) + ((m * TN + n) * 4 + q) * 64];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][n][4 * q + i] += v[i];
          }
  }
  store_tiles<T, TM, TN, NT>(acc, (T *)g.y + p0 * g.N, g.bias, g.N, n0 + wn * 32 * TN, wm * 32 * TM, lane, last_a + 1,
                             lds + (G > 1 ? (G - 1) * WAVES * TM * TN * 4096 : 0) + wave * Cell<T>::BYTES);
}

// ---- streamed rows --------------------------------------------------------------------------------------------------
// Many rows and a weight that fits LDS (64 KB: 512 x 128, 128 x 512, ...): bound by reading X and writing Y.  A workgroup
// keeps the weight and walks over tiles of 64 rows, 128 columns of X at a step: the next step's rows travel in registers
// while this one is multiplied, are quantised into the other LDS buffer, and go to memory as codes only where the backward
// pass wants them.  Against a quantising kernel and the tiles above: X's codes are not read back and there is one launch
// (524288 x 256 -> 128 bf16: 137 us in two launches, 107 here: 403 MB at 3.8 TB/s; 524288 x 128 -> 256: 92, 86).  SUM: also the
// column sums of X, a tile's four rows of a lane in registers, then fp32 in the lane's LDS cells over STREAM_RUN tiles at most.
static constexpr int STREAM_RUN = 60;
struct StreamArgs8 {
  const void *x;
  const unsigned char *w, *w_scales;
  const float *bias;
  void *y;
  unsigned char *codes, *scales;
  float *part;         // (workgroups, K)
  long long P, tiles;
  int N, K, bs_n, bs_k;
};
template <typename T>
struct Eight {
  T v[8];
};

template <typename T, bool EXACT, int TM, int TN, int WM, int WN, bool SUM, bool NT>
__global__ __launch_bounds__(256, 2) void fp8_stream_kernel(StreamArgs8 g) {
  constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, SLOTS = BM / 16;
  static_assert(WM * WN == 4 && BM == 64 && TN % 2 == 0 && 32 * TN <= 128, "tile");
  extern __shared__ __attribute__((aligned(128))) unsigned char smem[];
  const int Kb = blocks128(g.K), Kp = Kb * 128, ss = scale_stride(g.K);
  unsigned char *ws = smem, *xs = ws + Kb * BN * 128, *es = xs + 2 * BM * 128;
  float *sums = reinterpret_cast<float *>(es + 2 * BM + 4 * Cell<T>::BYTES);   // SUM: [16][Kp]
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, wm = wave / WN, wn = wave % WN, j = lane & 31;
  const int cl = (int)threadIdx.x & 15, rl = (int)threadIdx.x >> 4;
  const T *x = (const T *)g.x;

  for (int i = wave * 8; i < Kb * BN; i += 32) {   // the weight: eight rows of 128 codes per access (see above for the order)
    const int kb = i / BN, at = i - kb * BN + (lane >> 3), r = weight_row(at), n = r < g.N ? r : g.N - 1;
    dma16(g.w + (long long)n * Kp + kb * 128 + ((lane & 7) ^ (at >> 1 & 7)) * 16, ws + i * 128);
  }
  if (SUM)
    for (int i = 0; i < Kp / 128; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) sums[rl * Kp + i * 128 + cl * 8 + k] = 0;

  Eight<T> raw[SLOTS];
  auto fetch = [&](long long tile, int kb) {
    const int col = kb * 128 + cl * 8, n = g.K - col, rows = (int)(g.P - tile * BM < BM ? g.P - tile * BM : BM);
    const T *base = x + tile * BM * g.K;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const T *p = base + (unsigned)((s * 16 + rl) * g.K + col);
#pragma unroll
      for (int k = 0; k < 8; ++k) raw[s].v[k] = (T)0.0f;
      if (s * 16 + rl < rows) {
        if (n >= 8) {
          if (NT) {
            typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(1)));
            u4 v[sizeof(raw[s]) / 16];
#pragma unroll
            for (int i = 0; i < (int)(sizeof(raw[s]) / 16); ++i) v[i] = __builtin_nontemporal_load(reinterpret_cast<const u4 *>(p) + i);
            __builtin_memcpy(&raw[s], v, sizeof(raw[s]));
          } else {
            __builtin_memcpy(&raw[s], p, sizeof(raw[s]));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < n) raw[s].v[k] = p[k];
        }
      }
    }
  };
  auto put = [&](long long tile, int kb, int buf) {
    F8 sum = {};
    const int rows = (int)(g.P - tile * BM < BM ? g.P - tile * BM : BM);
    unsigned char *codes = g.codes + tile * BM * Kp + kb * 128, *scales = g.scales + tile * BM * ss + kb;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      F8 f;
#pragma unroll
      for (int k = 0; k < 8; ++k) f.v[k] = (float)raw[s].v[k];
      const int row = s * 16 + rl, e = block_exponent(row_max_f32(top8(f)));
      const uint2 c = encode8(f, e);
      *reinterpret_cast<uint2 *>(xs + (buf * BM + row) * 128 + ((cl >> 1) ^ (row >> 1 & 7)) * 16 + (cl & 1) * 8) = c;
      if (cl == 0) es[buf * BM + row] = (unsigned char)e;
      if (g.codes && row < rows) {
        *reinterpret_cast<uint2 *>(codes + (unsigned)(row * Kp + cl * 8)) = c;
        if (cl == 0) scales[(unsigned)(row * ss)] = (unsigned char)e;
      }
      if (SUM)
#pragma unroll
        for (int k = 0; k < 8; ++k) sum.v[k] += f.v[k];
    }
    if (SUM)
#pragma unroll
      for (int k = 0; k < 8; ++k) sums[rl * Kp + kb * 128 + cl * 8 + k] += sum.v[k];
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int n = 0; n < TN; ++n) acc[m][n] = f32x16{};
  const int nb = wn * 32 * TN / 128, last_nb = (g.N - 1) / 128;
  const unsigned char *bs = g.w_scales + (long long)(nb < last_nb ? nb : last_nb) * g.bs_n;

  long long tile = blockIdx.x;
  int kb = 0, buf = 0;
  if (tile < g.tiles) {
    fetch(tile, 0);
    put(tile, 0, 0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  while (tile < g.tiles) {
    const bool last = kb + 1 == Kb;
    const long long next = last ? tile + gridDim.x : tile;
    const int next_kb = last ? 0 : kb + 1;
    if (next < g.tiles) fetch(next, next_kb);
    const unsigned char *la = xs + (buf * BM + wm * 32 * TM + j) * 128, *lb = ws + (kb * BN + wn * 32 * TN + j) * 128;
    const int sb = bs[(long long)kb * g.bs_k];
    int sa[TM];
#pragma unroll
    for (int m = 0; m < TM; ++m) sa[m] = es[buf * BM + wm * 32 * TM + 32 * m + j];
    multiply128<EXACT, TM, TN>(acc, la, lb, lane, sa, sb);
    if (last) {
      T *y = (T *)g.y + tile * BM * g.N;
      const int rows = (int)(g.P - tile * BM < BM ? g.P - tile * BM : BM);
      int ll = lane;   // (opaque: the offsets of the stores are the same for every tile and would live in registers)
      asm volatile("" : "+v"(ll));
      store_tiles<T, TM, TN, NT>(acc, y, g.bias, g.N, wn * 32 * TN, wm * 32 * TM, ll, rows, es + 2 * BM + wave * Cell<T>::BYTES);
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = f32x16{};
    }
    if (next < g.tiles) put(next, next_kb, buf ^ 1);
    __syncthreads();
    tile = next;
    kb = next_kb;
    buf ^= 1;
  }
  if (SUM)
    for (int c = (int)threadIdx.x; c < g.K; c += 256) {
      double s = 0;
      for (int i = 0; i < 16; ++i) s += sums[i * Kp + c];
      g.part[(long long)blockIdx.x * g.K + c] = (float)s;
    }
}

// ---- few rows -------------------------------------------------------------------------------------------------------
// Up to 64 rows: bound by reading W once.  A workgroup takes 16 outputs; its waves take the blocks of 128 in turn, a lane
// reads 32 codes of W straight into the operand of a 16-row step (the four lanes of a row read one 128-byte line), and the
// waves' sums meet in LDS.  FUSED: every workgroup quantises the few rows of X for itself (one launch instead of two); the
// first one stores the codes where somebody wants them.
template <typename T, bool EXACT, int PT, int NW, bool FUSED>
__global__ __launch_bounds__(64 * NW) void fp8_few_kernel(GemmArgs8 g, const T *__restrict__ x, int K, unsigned char *__restrict__ codes_out,
                                                      unsigned char *__restrict__ scales_out) {
  __shared__ float sums[NW][PT][64][4];
  extern __shared__ __attribute__((aligned(16))) unsigned char codes[];   // FUSED: P x Kp codes, P x Kb exponents
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, j = lane & 15, q = lane >> 4;
  const int n0 = (int)blockIdx.x * 16, Kp = g.Kb * 128, P = (int)g.P;
  const unsigned char *ex = codes + P * Kp;
  if (FUSED) {
    const int cl = (int)threadIdx.x & 15;
    for (int i = (int)threadIdx.x >> 4; i < P * g.Kb; i += 4 * NW) {
      const int r = i / g.Kb, kb = i - r * g.Kb, col = kb * 128 + cl * 8;
      const F8 f = load_upto8(x + (long long)r * K + col, K - col);
      const int e = block_exponent(row_max_f32(top8(f)));
      const uint2 c = encode8(f, e);
      *reinterpret_cast<uint2 *>(codes + r * Kp + col) = c;
      if (cl == 0) codes[P * Kp + r * g.Kb + kb] = (unsigned char)e;
      if (codes_out && blockIdx.x == 0) {
        *reinterpret_cast<uint2 *>(codes_out + r * Kp + col) = c;
        if (cl == 0) scales_out[r * scale_stride(K) + kb] = (unsigned char)e;
      }
    }
    __syncthreads();
  }
  const int n = n0 + j < g.N ? n0 + j : g.N - 1;
  const unsigned char *w = g.b + (long long)n * Kp + q * 32, *bs = g.b_scales + (long long)(n0 / 128) * g.bs_n;
  f32x4 acc[PT];
  int row[PT];
#pragma unroll
  for (int t = 0; t < PT; ++t) {
    acc[t] = f32x4{};
    row[t] = 16 * t + j < P ? 16 * t + j : P - 1;
  }
  for (int kb = wave; kb < g.Kb; kb += NW) {
    const i32x4 w0 = *reinterpret_cast<const i32x4 *>(w + kb * 128), w1 = *reinterpret_cast<const i32x4 *>(w + kb * 128 + 16);
    const int sw = bs[(long long)kb * g.bs_k];
#pragma unroll
    for (int t = 0; t < PT; ++t) {
      const unsigned char *c = (FUSED ? codes : g.a) + (long long)row[t] * Kp + kb * 128 + q * 32;
      const int sx = FUSED ? ex[row[t] * g.Kb + kb] : g.a_scales[(long long)row[t] * g.a_stride + kb];
      const i32x4 x0 = *reinterpret_cast<const i32x4 *>(c), x1 = *reinterpret_cast<const i32x4 *>(c + 16);
      if (EXACT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const i32x4 &wq = i < 2 ? w0 : w1, &xq = i < 2 ? x0 : x1;
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              decode8((unsigned)wq[i % 2 * 2], (unsigned)wq[i % 2 * 2 + 1], power_of(sw)),
              decode8((unsigned)xq[i % 2 * 2], (unsigned)xq[i % 2 * 2 + 1], power_of(sx)), acc[t], 0, 0, 0);
        }
      } else {
        acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(w0, w1, 0, 1, 2, 3, 4, 5, 6, 7),
                                                                  __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7), acc[t], 0,
                                                                  0, 0, sw, 0, sx);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < PT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][t][lane][i] = acc[t][i];
  __syncthreads();
  for (int t = wave; t < PT; t += NW) {   // lane: row 16 t + j, outputs n0 + 4 q ..
    const int r = 16 * t + j;
    if (r >= P) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = n0 + 4 * q + i;
      if (c >= g.N) break;
      float s = sums[0][t][lane][i];
#pragma unroll
      for (int w = 1; w < NW; ++w) s += sums[w][t][lane][i];
      ((T *)g.y)[(long long)r * g.N + c] = (T)(s + (g.bias ? g.bias[c] : 0.0f));
    }
  }
}

// ---- weight gradient ------------------------------------------------------------------------------------------------
// dW[n][k] = sum over rows p of deq(dY)[p][n] deq(X)[p][k].  The scales belong to rows, i.e. to the reduction, and cannot leave
// the sum: the codes become bf16 with their scale (exact) on the way into LDS, and the bf16 matrix instructions do the
// rest in fp32.  Both operands lie in memory with the reduction as the slow index; ds_read_b64_tr_b16 hands every lane four
// rows of its column.  An LDS row is padded by 64 bytes: the four rows that sixteen lanes read then start 16 banks apart.
// Many rows and few outputs: the rows are cut into `splits` ranges, each range's sum goes to the workspace and a second
// kernel adds them in order.
struct WgradArgs8 {
  const unsigned char *dy, *dys, *x, *xs;
  float *out;
  long long P, rows;   // rows per split (a multiple of the step)
  int N, K, tiles_k;
};

typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4;

template <int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void fp8_wgrad_kernel(WgradArgs8 g) {
  constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, THREADS = 64 * WM * WN, STEP = 32;
  constexpr int CA = BM / 16, CH = (BM + BN) / 16, LOADS = STEP * CH / THREADS;
  constexpr int SA = BM * 2 + 64, SB = BN * 2 + 64, STAGE = STEP * (SA + SB);
  static_assert(STEP * CH % THREADS == 0, "loads");
  __shared__ __attribute__((aligned(16))) unsigned char lds[2][STAGE];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
  const int n0 = (int)(blockIdx.x / g.tiles_k) * BM, k0 = (int)(blockIdx.x % g.tiles_k) * BN;
  const int Np = blocks128(g.N) * 128, Kp = blocks128(g.K) * 128, sn = scale_stride(g.N), sk = scale_stride(g.K);
  const long long p0 = g.rows * blockIdx.y, p1 = p0 + g.rows < g.P ? p0 + g.rows : g.P;

  // the lane's share of a step: sixteen codes of LOADS rows, as they are in memory
  int row[LOADS], to[LOADS];
  const unsigned char *src[LOADS], *scl[LOADS];
  int ld[LOADS], sld[LOADS];
  bool in[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int c = i * THREADS + (int)threadIdx.x, cc = c % CH;
    row[i] = c / CH;
    const bool of_a = cc < CA;
    const int col = of_a ? n0 + cc * 16 : k0 + (cc - CA) * 16, width = of_a ? Np : Kp;
    in[i] = col < width;
    const int at = in[i] ? col : 0;
    ld[i] = width;
    sld[i] = of_a ? sn : sk;
    src[i] = (of_a ? g.dy : g.x) + (p0 + row[i]) * width + at;
    scl[i] = (of_a ? g.dys : g.xs) + (p0 + row[i]) * sld[i] + at / 128;
    to[i] = of_a ? row[i] * SA + cc * 32 : STEP * SA + row[i] * SB + (cc - CA) * 32;
  }
  struct Codes {
    uint4 code[LOADS];
    unsigned scale[LOADS];
  };
  auto fetch = [&](long long p, Codes &f) {   // (called for p0, p0 + STEP, ... in turn)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      f.code[i] = make_uint4(0, 0, 0, 0);
      f.scale[i] = 127;
      if (in[i] && p + row[i] < p1) {
        f.code[i] = *reinterpret_cast<const uint4 *>(src[i]);
        f.scale[i] = *scl[i];
      }
      src[i] += (long long)STEP * ld[i];
      scl[i] += STEP * sld[i];
    }
  };
  auto put = [&](unsigned char *stage, const Codes &f) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const float s = power_of((int)f.scale[i]);
      *reinterpret_cast<bf16x8 *>(stage + to[i]) = decode8(f.code[i].x, f.code[i].y, s);
      *reinterpret_cast<bf16x8 *>(stage + to[i] + 16) = decode8(f.code[i].z, f.code[i].w, s);
    }
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int n = 0; n < TN; ++n) acc[m][n] = f32x16{};
  const int sub = lane & 15, right = (lane >> 4 & 1) * 16 + (sub & 3) * 4, down = (lane >> 5) * 8 + (sub >> 2);
  const int fa = down * SA + (wm * 32 * TM + right) * 2, fb = STEP * SA + down * SB + (wn * 32 * TN + right) * 2;
  auto multiply = [&](unsigned char *st) {
#pragma unroll
    for (int s = 0; s < STEP / 16; ++s) {
      bf16x8 a[TM], b[TN];
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        unsigned char *at = st + fa + s * 16 * SA + m * 64;
        a[m] = __builtin_shufflevector(__builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4 *)(at)),
                                       __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4 *)(at + 4 * SA)), 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int n = 0; n < TN; ++n) {
        unsigned char *at = st + fb + s * 16 * SB + n * 64;
        b[n] = __builtin_shufflevector(__builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4 *)(at)),
                                       __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4 *)(at + 4 * SB)), 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[m], b[n], acc[m][n], 0, 0, 0);
    }
  };
  // A step's codes are requested two steps before they are needed: one step multiplies for ~1000 cycles, less than the
  // memory takes to answer.  Behind the range there are zeros.
  if (p0 < p1) {
    Codes even, odd;
    fetch(p0, even);
    put(lds[0], even);
    fetch(p0 + STEP, odd);
    fetch(p0 + 2 * STEP, even);
    __syncthreads();
    for (long long p = p0; p < p1; p += 2 * STEP) {
      multiply(lds[0]);
      put(lds[1], odd);
      fetch(p + 3 * STEP, odd);
      __syncthreads();
      multiply(lds[1]);   // (zeros where the range ends with an odd step)
      put(lds[0], even);
      fetch(p + 4 * STEP, even);
      __syncthreads();
    }
  }
  float *out = g.out + (long long)blockIdx.y * g.N * g.K;
  const int j = lane & 31, h = lane >> 5;
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int n = 0; n < TN; ++n) {
      const int col = k0 + wn * 32 * TN + 32 * n + j;
      if (col >= g.K) continue;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = n0 + wm * 32 * TM + 32 * m + i / 4 * 8 + h * 4 + i % 4;
        if (r < g.N) out[(long long)r * g.K + col] = acc[m][n][i];
      }
    }
}

// out[i] = the splits' sums added in order: 32 elements x 8 lanes over the splits
__global__ __launch_bounds__(256) void fp8_wgrad_join_kernel(const float *__restrict__ part, int splits, long long n,
                                                             float *__restrict__ out) {
  __shared__ float lds[8][32];
  const int i = (int)threadIdx.x & 31, q = (int)threadIdx.x >> 5;
  const long long e = (long long)blockIdx.x * 32 + i;
  float s = 0;
  if (e < n)
#pragma unroll 8
    for (int k = q; k < splits; k += 8) s += part[(long long)k * n + e];
  lds[q][i] = s;
  __syncthreads();
  if (q == 0 && e < n) {
    for (int j = 1; j < 8; ++j) s += lds[j][i];
    out[e] = s;
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------

template <typename T, bool EXACT, int TM, int TN, int WM, int WN, int G, bool NT>
static int launch_tiles(GemmArgs8 g, hipStream_t st) {
  constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, STAGE = (BM + BN) * 128;
  g.tiles_n = (g.N + BN - 1) / BN;
  g.tiles = (g.P + BM - 1) / BM * g.tiles_n;
  if (g.tiles > 0x7fffffffll) return GB_ERANGE;
  if (2 * G * STAGE > 65536) {
    static std::atomic<unsigned long long> done{0};
    allow_dynamic_lds(fp8_gemm_kernel<T, EXACT, TM, TN, WM, WN, G, NT>, 2 * G * STAGE, done);
  }
  fp8_gemm_kernel<T, EXACT, TM, TN, WM, WN, G, NT><<<(unsigned)g.tiles, 64 * WM * WN * G, (g.Kb > 1 ? 2 * G : 1) * STAGE, st>>>(g);
  return check_launch("gb_fp8_linear");
}

static long long tiles_of(long long P, int N, int b) { return ((P + b - 1) / b) * ((N + b - 1) / b); }
template <typename T, bool EXACT, int PT, bool FUSED>
static void launch_few(const GemmArgs8 &g, const T *x, int K, unsigned char *codes, unsigned char *scales, size_t lds, hipStream_t st) {
  const unsigned grid = (unsigned)((g.N + 15) / 16);
  if (g.Kb >= 8)   // (a wave per block of a long reduction: 4 x 4096 -> 4096 fp32 9.7 us with four waves, 6.7 with eight)
    fp8_few_kernel<T, EXACT, PT, 8, FUSED><<<grid, 512, lds, st>>>(g, x, K, codes, scales);
  else
    fp8_few_kernel<T, EXACT, PT, 4, FUSED><<<grid, 256, lds, st>>>(g, x, K, codes, scales);
}

// y from codes and exponents in memory
template <typename T, bool EXACT>
static int multiply_codes(const GemmArgs8 &g, int K, hipStream_t st) {
  // (64 x 4096 -> 4096 bf16: 18.6 us without tiles, 14.9 with four groups of waves a tile; 64 x 1024 -> 1024: 7.3, 8.4)
  if (g.P <= FP8_FEW_ROWS && !(g.P > 32 && g.Kb >= 32)) {
    if (g.P <= 16)
      launch_few<T, EXACT, 1, false>(g, nullptr, K, nullptr, nullptr, 0, st);
    else if (g.P <= 32)
      launch_few<T, EXACT, 2, false>(g, nullptr, K, nullptr, nullptr, 0, st);
    else
      launch_few<T, EXACT, 4, false>(g, nullptr, K, nullptr, nullptr, 0, st);
    return check_launch("gb_fp8_linear");
  }
  // 256 x 256 where that still gives every CU a tile, the columns fill it as well as 128 do to a fifth, and there are steps
  // enough to work through; short reductions live from several workgroups per CU, which only smaller tiles leave room for.  Tiles of 64 x 64 that leave
  // CUs idle get groups of waves: four up to a tile per CU, two up to two tiles (1024 x 4096 -> 4096 bf16: 45.6 us in tiles
  // of 128 x 128, 48.4 in 1024 of these; with the 8-bit instructions 34, 46).
  const bool nt = streams(g.P * g.N * (long long)sizeof(T));
  if (g.Kb >= 4 && tiles_of(g.P, g.N, 256) >= 256 && 5 * blocks128(g.N) >= 8 * ((g.N + 255) / 256))
    return nt ? launch_tiles<T, EXACT, 4, 2, 2, 4, 1, true>(g, st) : launch_tiles<T, EXACT, 4, 2, 2, 4, 1, false>(g, st);
  if (tiles_of(g.P, g.N, 128) >= 256) return nt ? launch_tiles<T, EXACT, 2, 2, 2, 2, 1, true>(g, st) : launch_tiles<T, EXACT, 2, 2, 2, 2, 1, false>(g, st);
  const long long tiles = tiles_of(g.P, g.N, 64);
  if (g.Kb >= 8 && tiles <= 512)
    return tiles <= 256 ? launch_tiles<T, EXACT, 1, 2, 2, 1, 4, false>(g, st) : launch_tiles<T, EXACT, 1, 2, 2, 1, 2, false>(g, st);
  return launch_tiles<T, EXACT, 1, 2, 2, 1, 1, false>(g, st);
}

// Columns of the streaming kernel's variant; 0: not one of its shapes.  A weight of 128 x 128 is in LDS at once, and one
// launch beats two from the first rows on (1024 rows fp32: 5.2 us against 5.8; 16384: 6.4, 8.7); a larger one has to be worth
// its loading by every workgroup (8192 x 512 -> 128 bf16: 12.8 against 10.6, 16384 x 256 -> 256 fp32: 12.2 against 14.0,
// 524288 x 256 -> 128 bf16: 107 against 137, fp32 165 against 211; the worst is 65536 x 256 -> 256: bf16 34 against 26, fp32 35
// against 33).
static int stream_columns(long long P, int N, int K) {
  if (P <= FP8_FEW_ROWS || N > 512) return 0;
  const int cols = N <= 128 ? 128 : N <= 256 ? 256 : 512;
  const long long bytes = (long long)cols * blocks128(K) * 128;
  return bytes <= 16384 || (bytes <= 65536 && P >= 16384) ? cols : 0;
}
struct StreamPlan8 {
  size_t lds;
  int grid;
};
// Workgroups per CU that walk over the tiles.  A 128 x 128 weight: three for fp32, four for 16 bits (700001 rows bf16: two 82 us, three
// 72, four 67); larger ones: two, although registers and LDS would often hold three (524288 x 128 -> 256 bf16: two 86 us, three
// 96, four in turns 88; 524288 x 256 -> 128: 107, 121, 108; 100000 x 128 -> 256: 24.6, 27.3, 25.5; a training pass of
// 524288 x 128 -> 256: 262, 290, 276).
static StreamPlan8 stream_plan(long long P, int cols, int K, int dtype, bool sum) {
  StreamPlan8 p;
  const int Kp = blocks128(K) * 128;
  p.lds = (size_t)cols * Kp + 2 * 64 * 128 + 2 * 64 + 4 * (dtype == GB_T_F32 ? Cell<float>::BYTES : Cell<__bf16>::BYTES) + (sum ? (size_t)16 * Kp * 4 : 0);
  const int by_lds = (int)(163840 / p.lds), want = cols * Kp <= 16384 ? (dtype == GB_T_F32 ? 3 : 4) : 2, per_cu = by_lds < want ? by_lds : want;
  const long long tiles = (P + 63) / 64, fill = 256ll * (per_cu < 1 ? 1 : per_cu), runs = sum ? (tiles + STREAM_RUN - 1) / STREAM_RUN : 0,
                  most = fill > runs ? fill : runs;
  p.grid = (int)(tiles < most ? tiles : most);
  return p;
}
template <typename T, bool EXACT, int TM, int TN, int WM, int WN, bool SUM>
static int launch_stream(const StreamArgs8 &g, const StreamPlan8 &p, hipStream_t st) {
  const bool nt = streams(g.P * (g.N < g.K ? g.N : g.K) * (long long)sizeof(T));
  static std::atomic<unsigned long long> done[2];
  if (nt) {
    allow_dynamic_lds(fp8_stream_kernel<T, EXACT, TM, TN, WM, WN, SUM, true>, 163840, done[1]);
    fp8_stream_kernel<T, EXACT, TM, TN, WM, WN, SUM, true><<<(unsigned)p.grid, 256, p.lds, st>>>(g);
  } else {
    allow_dynamic_lds(fp8_stream_kernel<T, EXACT, TM, TN, WM, WN, SUM, false>, 163840, done[0]);
    fp8_stream_kernel<T, EXACT, TM, TN, WM, WN, SUM, false><<<(unsigned)p.grid, 256, p.lds, st>>>(g);
  }
  return check_launch("gb_fp8_linear");
}
template <typename T, bool EXACT, bool SUM>
static int stream_rows(const StreamArgs8 &g, const StreamPlan8 &p, int cols, hipStream_t st) {
  return cols == 128   ? launch_stream<T, EXACT, 1, 2, 2, 2, SUM>(g, p, st)
         : cols == 256 ? launch_stream<T, EXACT, 2, 2, 1, 4, SUM>(g, p, st)
                       : launch_stream<T, EXACT, 2, 4, 1, 4, SUM>(g, p, st);
}


// f(T(), EXACT) of a product's output type and GB_FP8_SHORT_SUMS
template <typename F>
static int with_form(int dtype, int flags, F f) {
  return with_type(dtype, [&](auto z) {
    typedef decltype(z) T;
    if constexpr (sizeof(T) == 2)
      if (flags & GB_FP8_SHORT_SUMS) return f(z, std::false_type());
    return f(z, std::true_type());
  });
}

static bool fp8_dims_bad(long long P, int N, int K) { return P < 0 || N <= 0 || K <= 0; }
static bool fp8_dims_large(long long P, int N, int K) {   // int tile offsets: 256 rows of Kp bytes; 65535 blocks a grid axis
  return N > (1 << 22) || K > (1 << 22) || P > (1ll << 40);
}

// Rows of a workgroup: sixteen (one access a lane) until that fills the device, then 64 (8192 x 128 fp32 in chunks of 64 rows
// 4.8 us, of sixteen 3.7); with column sums as many as leave at most 512 partial ones, but no lane adds more than 64.
static int rows_per_chunk(long long P, int K, bool sum) {
  if (!sum) {
    if (P / 16 * blocks128(K) < 8192) return 16;
    const long long per = (P >> 23) / 16 * 16 + 16;   // (a launch has fewer than 2^32 lanes)
    return per < 64 ? 64 : (int)per;
  }
  const long long per = (P + 511) / 512;
  return (int)(per < 16 ? 16 : per > 1024 ? 1024 : (per + 15) / 16 * 16);
}

struct WgradPlan8 {
  bool big;
  int tiles_n, tiles_k, splits;
  long long rows;
};
// 256 x 256 outputs per workgroup where both sides fill them, else 128 x 128; the rows are cut until there is a workgroup
// of the large kind for every CU, or two of the small, into ranges of 512 rows at least (a range writes its outputs once more and has them read once more).
static WgradPlan8 wgrad_plan(long long P, int N, int K) {
  WgradPlan8 p;
  p.big = N > 192 && K > 192;
  const int b = p.big ? 256 : 128;
  p.tiles_n = (N + b - 1) / b;
  p.tiles_k = (K + b - 1) / b;
  const long long tiles = (long long)p.tiles_n * p.tiles_k, want = ((p.big ? 256 : 512) + tiles - 1) / tiles, most = (P + 511) / 512;
  long long splits = want < most ? want : most;
  if (splits < 1) splits = 1;
  p.rows = ((P + splits - 1) / splits + 31) / 32 * 32;
  p.splits = p.rows ? (int)((P + p.rows - 1) / p.rows) : 0;
  return p;
}

}  // namespace gb

using namespace gb;

extern "C" int gb_fp8_quant_rows(const void *x, int dtype, long long P, int K, void *codes, void *scales, float *colsum, void *ws,
                                 long long ws_bytes, void *stream) {
  if (fp8_dims_bad(P, 1, K) || !known_type(dtype)) return GB_EINVAL;
  if (fp8_dims_large(P, 1, K)) return GB_ERANGE;
  const int per = rows_per_chunk(P, K, colsum != nullptr);
  const long long chunks = (P + per - 1) / per;
  if (chunks > 0x7fffffffll || blocks128(K) > 65535) return GB_ERANGE;
  if (P == 0 && !colsum) return GB_OK;
  if (P > 0 && (!x || !codes || !scales || (reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) % 16)) return GB_EINVAL;
  if (colsum && chunks > 0 && (!ws || ws_bytes < chunks * K * 4 || reinterpret_cast<uintptr_t>(ws) % 16)) return GB_EINVAL;
  hipStream_t st = as_stream(stream);
  return with_type(dtype, [&](auto z) {
    typedef decltype(z) T;
    const dim3 grid((unsigned)chunks, (unsigned)blocks128(K));
    if (colsum) {
      if (P > 0)
        fp8_rows_kernel<T, true><<<grid, 256, 0, st>>>((const T *)x, P, K, (unsigned char *)codes, (unsigned char *)scales, per, (float *)ws);
      fp8_colsum_kernel<<<(K + 7) / 8, 256, 0, st>>>((const float *)ws, (int)chunks, K, colsum);
    } else {
      fp8_rows_kernel<T, false><<<grid, 256, 0, st>>>((const T *)x, P, K, (unsigned char *)codes, (unsigned char *)scales, per, nullptr);
    }
    return check_launch("gb_fp8_quant_rows");
  });
}

extern "C" int gb_fp8_quant_weight(const void *w, int dtype, int N, int K, void *codes, void *codes_t, void *scales, void *stream) {
  if (fp8_dims_bad(0, N, K) || !known_type(dtype)) return GB_EINVAL;
  if (fp8_dims_large(0, N, K)) return GB_ERANGE;
  if (!w || !codes || !scales || (reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(codes_t)) % 16) return GB_EINVAL;
  return with_type(dtype, [&](auto z) {
    typedef decltype(z) T;
    fp8_weight_kernel<T><<<dim3((unsigned)blocks128(K), (unsigned)blocks128(N)), 256, 0, as_stream(stream)>>>(
        (const T *)w, N, K, (unsigned char *)codes, (unsigned char *)codes_t, (unsigned char *)scales);
    return check_launch("gb_fp8_quant_weight");
  });
}

// Which way a product goes: quantised by every workgroup for itself (few), streamed, or quantised by a kernel of its own
// before the tiles.
enum { FP8_FEW, FP8_STREAM, FP8_TILES };
static int linear_route(long long P, int N, int K) {
  if (P <= FP8_FUSED_ROWS && P * blocks128(K) * 128 <= FP8_FUSED_CODES) return FP8_FEW;
  return stream_columns(P, N, K) ? FP8_STREAM : FP8_TILES;
}
static long long up16(long long n) { return (n + 15) / 16 * 16; }
// (the 16-bit plan has at least as many workgroups as the fp32 one)
// bytes: column sums' partials, then the codes and exponents of the tiles' route where the caller keeps none
static long long linear_workspace(long long P, int N, int K, bool keeps, bool sum) {
  const int route = linear_route(P, N, K);
  long long b = 0;
  if (sum) {
    const long long per = rows_per_chunk(P, K, true),
                    chunks = route == FP8_STREAM ? stream_plan(P, stream_columns(P, N, K), K, GB_T_BF16, true).grid : (P + per - 1) / per;
    b += up16(chunks * K * 4);
  }
  if ((route == FP8_TILES || (route == FP8_FEW && sum)) && !keeps) b += P * (blocks128(K) * 128ll) + up16(P * scale_stride(K));
  return b;
}

extern "C" int gb_fp8_linear(const void *x, int dtype, long long P, int K, const void *w, const void *w_scales, int flags, int N,
                             const float *bias, void *y, void *codes, void *scales, float *colsum, void *ws, long long ws_bytes,
                             void *stream) {
  if (fp8_dims_bad(P, N, K) || !known_type(dtype) || !codes != !scales || (flags & ~(GB_FP8_TRANSPOSED | GB_FP8_SHORT_SUMS))) return GB_EINVAL;
  if (fp8_dims_large(P, N, K)) return GB_ERANGE;
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(ws) |
       reinterpret_cast<uintptr_t>(w)) % 16)
    return GB_EINVAL;
  if (P > 0 && (!x || !y || !w || !w_scales)) return GB_EINVAL;
  const long long need = linear_workspace(P, N, K, codes != nullptr, colsum != nullptr);
  if (need > 0 && (!ws || ws_bytes < need)) return GB_EINVAL;
  hipStream_t st = as_stream(stream);
  if (P == 0) {
    if (!colsum) return GB_OK;
    fp8_colsum_kernel<<<(K + 7) / 8, 256, 0, st>>>((const float *)ws, 0, K, colsum);
    return check_launch("gb_fp8_linear");
  }
  const int route = linear_route(P, N, K), Kb = blocks128(K), bs_n = flags & GB_FP8_TRANSPOSED ? 1 : Kb,
            bs_k = flags & GB_FP8_TRANSPOSED ? blocks128(N) : 1;
  if (route == FP8_STREAM) {
    const int cols = stream_columns(P, N, K);
    const StreamPlan8 p = stream_plan(P, cols, K, dtype, colsum != nullptr);
    StreamArgs8 g = {};
    g.x = x;
    g.w = (const unsigned char *)w;
    g.w_scales = (const unsigned char *)w_scales;
    g.bias = bias;
    g.y = y;
    g.codes = (unsigned char *)codes;
    g.scales = (unsigned char *)scales;
    g.part = (float *)ws;
    g.P = P;
    g.tiles = (P + 63) / 64;
    g.N = N;
    g.K = K;
    g.bs_n = bs_n;
    g.bs_k = bs_k;
    const int rc = with_form(dtype, flags, [&](auto z, auto exact) {
      typedef decltype(z) T;
      constexpr bool EXACT = decltype(exact)::value;
      return colsum ? stream_rows<T, EXACT, true>(g, p, cols, st) : stream_rows<T, EXACT, false>(g, p, cols, st);
    });
    if (rc || !colsum) return rc;
    fp8_colsum_kernel<<<(K + 7) / 8, 256, 0, st>>>((const float *)ws, p.grid, K, colsum);
    return check_launch("gb_fp8_linear");
  }
  GemmArgs8 g = {};
  g.b = (const unsigned char *)w;
  g.b_scales = (const unsigned char *)w_scales;
  g.bias = bias;
  g.y = y;
  g.P = P;
  g.N = N;
  g.Kb = Kb;
  g.a_stride = scale_stride(K);
  g.bs_n = bs_n;
  g.bs_k = bs_k;
  if (route == FP8_FEW && !colsum) {
    const size_t lds = (size_t)up16(P * Kb * 129);
    return with_form(dtype, flags, [&](auto z, auto exact) {
      typedef decltype(z) T;
      launch_few<T, decltype(exact)::value, 1, true>(g, (const T *)x, K, (unsigned char *)codes, (unsigned char *)scales, lds, st);
      return check_launch("gb_fp8_linear");
    });
  }
  unsigned char *at = (unsigned char *)ws;
  const long long sums = colsum ? linear_workspace(P, N, K, true, true) : 0;
  if (!codes) {
    codes = at + sums;
    scales = (unsigned char *)codes + P * (Kb * 128ll);
  }
  const int rc = gb_fp8_quant_rows(x, dtype, P, K, codes, scales, colsum, ws, sums, stream);
  if (rc) return rc;
  g.a = (const unsigned char *)codes;
  g.a_scales = (const unsigned char *)scales;
  return with_form(dtype, flags, [&](auto z, auto exact) {
    typedef decltype(z) T;
    return multiply_codes<T, decltype(exact)::value>(g, K, st);
  });
}

extern "C" int gb_fp8_workspace(int what, long long P, int N, int K, long long *bytes) {
  if (fp8_dims_bad(P, N, K) || !bytes || (what != GB_FP8_WS_COLSUM && what != GB_FP8_WS_WGRAD && (what < GB_FP8_WS_LINEAR || what >= GB_FP8_WS_LINEAR + 4))) return GB_EINVAL;
  if (fp8_dims_large(P, N, K)) return GB_ERANGE;
  if (what == GB_FP8_WS_COLSUM) {
    const int per = rows_per_chunk(P, K, true);
    *bytes = (P + per - 1) / per * N * 4;
  } else if (what >= GB_FP8_WS_LINEAR) {
    *bytes = linear_workspace(P, N, K, (what - GB_FP8_WS_LINEAR) & GB_FP8_KEEP, (what - GB_FP8_WS_LINEAR) & GB_FP8_SUM);
  } else {
    const WgradPlan8 p = wgrad_plan(P, N, K);
    *bytes = p.splits > 1 ? (long long)p.splits * N * K * 4 : 0;
  }
  return GB_OK;
}

extern "C" int gb_fp8_wgrad(const void *dy, const void *dy_scales, const void *x, const void *x_scales, float *dw, long long P, int N, int K,
                            void *ws, long long ws_bytes, void *stream) {
  if (fp8_dims_bad(P, N, K)) return GB_EINVAL;
  if (fp8_dims_large(P, N, K)) return GB_ERANGE;
  if (!dw || (P > 0 && (!dy || !dy_scales || !x || !x_scales || (reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(x)) % 16)))
    return GB_EINVAL;
  const WgradPlan8 p = wgrad_plan(P, N, K);
  const long long n = (long long)N * K;
  if (p.splits > 1 && (!ws || ws_bytes < p.splits * n * 4 || reinterpret_cast<uintptr_t>(ws) % 16)) return GB_EINVAL;
  if ((long long)p.tiles_n * p.tiles_k > 0x7fffffffll || (n + 31) / 32 > 0x7fffffffll) return GB_ERANGE;
  hipStream_t st = as_stream(stream);
  WgradArgs8 g = {};
  g.dy = (const unsigned char *)dy;
  g.dys = (const unsigned char *)dy_scales;
  g.x = (const unsigned char *)x;
  g.xs = (const unsigned char *)x_scales;
  g.out = p.splits > 1 ? (float *)ws : dw;
  g.P = P;
  g.rows = p.rows;
  g.N = N;
  g.K = K;
  g.tiles_k = p.tiles_k;
  const dim3 grid((unsigned)(p.tiles_n * p.tiles_k), (unsigned)p.splits);
  if (p.splits > 0) {
    if (p.big)
      fp8_wgrad_kernel<4, 2, 2, 4><<<grid, 512, 0, st>>>(g);
    else
      fp8_wgrad_kernel<2, 2, 2, 2><<<grid, 256, 0, st>>>(g);
  }
  if (p.splits != 1) fp8_wgrad_join_kernel<<<(unsigned)((n + 31) / 32), 256, 0, st>>>((const float *)ws, p.splits, n, dw);
  return check_launch("gb_fp8_wgrad");
}
