// Shared helpers of the channel-last row operators (row_norm.hip, row_dropout.hip, fp8.hip): element types, eight
// consecutive elements per lane, the counter-based generator.
#pragma once
#include "gb_common.h"

namespace gb {

// Eight consecutive elements as fp32.  A lane always works on eight: one 16-byte access for the 16-bit types, two for
// fp32, and exactly the eight 16-bit numbers that one block of the generator gives.  The accesses carry no alignment
// (tensors that start inside another one are legal; the hardware takes any byte address).
struct F8 {
  float v[8];
};
template <typename T>
struct Raw8 {
  T v[8];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T *p) {
  Raw8<T> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T>
__device__ __forceinline__ F8 widen(const Raw8<T> &r) {
  F8 f;
#pragma unroll
  for (int k = 0; k < 8; ++k) f.v[k] = (float)r.v[k];
  return f;
}
template <typename T>
__device__ __forceinline__ F8 load8(const T *p) {
  return widen(load_raw8(p));
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const F8 &f) {  // the one rounding of a result: nearest, ties to even
  Raw8<T> r;
#pragma unroll
  for (int k = 0; k < 8; ++k) r.v[k] = (T)f.v[k];
  __builtin_memcpy(p, &r, sizeof(r));
}

// the first n < 8 of eight elements; the others read as zero
template <typename T>
__device__ __forceinline__ F8 load_tail(const T *p, int n) {
  F8 f = {};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) f.v[k] = (float)p[k];
  return f;
}
template <typename T>
__device__ __forceinline__ void store_tail(T *p, const F8 &f, int n) {
#pragma unroll
  for (int k = 0; k < 8; ++k)
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
__device__ __forceinline__ unsigned keep8(const RowRng &g, unsigned long long i, unsigned q) {
  unsigned w[4];
  philox_block(g, i >> 3, w);
  unsigned m = block_mask(w, q);
  const int r = (int)(i & 7);
  if (r) {  // eight elements of a packed cloud that starts inside a block: the rest of them are in the next block
    philox_block(g, (i >> 3) + 1, w);
    m = (m | block_mask(w, q) << 8) >> r;
  }
  return m & 0xffu;
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

// f(T()) for the element type behind a GB_T_* code
template <typename F>
inline int with_type(int t, F f) {
  if (t == GB_T_F32) return f((float)0);
  if (t == GB_T_BF16) return f((__bf16)0.0f);
  return f((_Float16)0.0f);
}

}  // namespace gb
