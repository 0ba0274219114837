// Shared helpers of the channel-last row operators (row_norm.hip, row_dropout.hip, fp8.hip): element types, 16
// bytes of consecutive elements per lane, the counter-based generator.
#pragma once
#include "gb_common.h"

namespace gb {

// A lane's unit of work: the 16 bytes of one access, N = 4 fp32 or 8 16-bit elements, widened to fp32.  Neighbouring lanes
// take neighbouring units, so that a wave's access covers whole lines (fp32 in eights per lane, two accesses of every
// other 16 bytes, copied 268 MB at 3.8 - 5.0 TB/s; in units 5.3 - 6.1).  The accesses carry no alignment: tensors that start
// inside another one are legal, and the hardware takes any address.
template <typename T>
struct Unit {
  static constexpr int N = 16 / (int)sizeof(T);
};
template <typename T>
struct Raw {
  T v[Unit<T>::N];
};
template <int N>
struct Vec {
  float v[N];
};
template <typename T>
using VecOf = Vec<Unit<T>::N>;
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// NT: the tensors are far larger than the caches, and a line that nobody will find there again is kept out of them (268 MB:
// reads 5.6 -> 6.4 TB/s, copies 5.4 -> 5.9).
template <bool NT = false, typename T>
__device__ __forceinline__ Raw<T> load_raw(const T *p) {
  Raw<T> r;
  if (NT) {
    const u32x4_any w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p));
    __builtin_memcpy(&r, &w, 16);
  } else {
    __builtin_memcpy(&r, p, 16);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ VecOf<T> widen(const Raw<T> &r) {
  VecOf<T> f;
#pragma unroll
  for (int k = 0; k < Unit<T>::N; ++k) f.v[k] = (float)r.v[k];
  return f;
}
template <bool NT = false, typename T>
__device__ __forceinline__ VecOf<T> load_unit(const T *p) {
  return widen(load_raw<NT>(p));
}
template <bool NT = false, typename T>
__device__ __forceinline__ void store_unit(T *p, const VecOf<T> &f) {  // the one rounding of a result: nearest, ties to even
  Raw<T> r;
#pragma unroll
  for (int k = 0; k < Unit<T>::N; ++k) r.v[k] = (T)f.v[k];
  if (NT) {
    u32x4_any w;
    __builtin_memcpy(&w, &r, 16);
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any *>(p));
  } else {
    __builtin_memcpy(p, &r, 16);
  }
}
// the first n of a unit's elements; the others read as zero
template <typename T>
__device__ __forceinline__ VecOf<T> load_part(const T *p, int n) {
  VecOf<T> f = {};
#pragma unroll
  for (int k = 0; k < Unit<T>::N; ++k)
    if (k < n) f.v[k] = (float)p[k];
  return f;
}
template <typename T>
__device__ __forceinline__ void store_part(T *p, const VecOf<T> &f, int n) {
#pragma unroll
  for (int k = 0; k < Unit<T>::N; ++k)
    if (k < n) p[k] = (T)f.v[k];
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten rounds of two
// 32x32 -> 64 products on the counter (block, call) under the key `seed`.
struct RowRng {
  unsigned long long seed, call;
};
__device__ __forceinline__ void philox_block(const RowRng &g, unsigned long long block, unsigned (&w)[4]) {
  unsigned k0 = (unsigned)g.seed, k1 = (unsigned)(g.seed >> 32);
  w[0] = (unsigned)block;
  w[1] = (unsigned)(block >> 32);
  w[2] = (unsigned)g.call;
  w[3] = (unsigned)(g.call >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p0 = 0xD2511F53ull * w[0], p1 = 0xCD9E8D57ull * w[2];
    const unsigned n0 = (unsigned)(p1 >> 32) ^ w[1] ^ k0, n2 = (unsigned)(p0 >> 32) ^ w[3] ^ k1;
    w[0] = n0;
    w[1] = (unsigned)p1;
    w[2] = n2;
    w[3] = (unsigned)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}
// Element i of a call takes the 16-bit number i & 7 (low half of word 0 first) of block i >> 3 and is kept when that
// number is >= q: p = q / 65536.  Sixteen bits per element halve the integer products per element against 32 and cost a
// resolution of p of 2^-16.  Bit k of the result: element i + k is kept.
__device__ __forceinline__ unsigned block_mask(const unsigned (&w)[4], unsigned q) {
  unsigned m = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    m |= ((w[k] & 0xffffu) >= q ? 1u : 0u) << (2 * k) | ((w[k] >> 16) >= q ? 1u : 0u) << (2 * k + 1);
  return m;
}
// the N elements from element i on
template <int N>
__device__ __forceinline__ unsigned keep_mask(const RowRng &g, unsigned long long i, unsigned q) {
  unsigned w[4];
  philox_block(g, i >> 3, w);
  unsigned m = block_mask(w, q);
  const int r = (int)(i & 7);
  if (r + N > 8) {  // a packed cloud that starts inside a block: the rest of the elements are in the next one
    philox_block(g, (i >> 3) + 1, w);
    m |= block_mask(w, q) << 8;
  }
  return m >> r & ((1u << N) - 1);
}

// [seed, call] from the device (a captured graph's next replay sees what its owner wrote there) or by value; the pair
// that was used goes to `used`, from where the backward pass reads it.
__device__ __forceinline__ RowRng load_rng(const long long *rng, long long seed, long long call) {
  RowRng g;
  g.seed = (unsigned long long)(rng ? rng[0] : seed);
  g.call = (unsigned long long)(rng ? rng[1] : call);
  return g;
}

// q = p * 65536 is checked to be in [0, 65536] on the host; everything is dropped at 65536 and the factor is unused.
inline float keep_scale(int q) { return q < 65536 ? (float)(65536.0 / (65536 - q)) : 0.0f; }

inline bool known_type(int t) { return t == GB_T_F32 || t == GB_T_BF16 || t == GB_T_F16; }

// Tensors that no cache keeps until somebody reads them again (the last level holds 256 MB)
inline bool streams(long long bytes) { return bytes >= (96ll << 20); }

// f(T()) for the element type behind a GB_T_* code
template <typename F>
inline int with_type(int t, F f) {
  if (t == GB_T_F32) return f((float)0);
  if (t == GB_T_BF16) return f((__bf16)0.0f);
  return f((_Float16)0.0f);
}

}  // namespace gb
