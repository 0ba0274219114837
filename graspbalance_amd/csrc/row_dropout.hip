// Dropout from a counter-based generator (graspbal.h gb_dropout): y = x * keep / (1 - p) (+ residual), keep recomputed from
// (seed, call, element index) wherever it is needed - the backward pass is the same kernel on dy - and never stored.
#include "row_common.h"

#pragma clang fp contract(on)  // x * scale + residual in one instruction

namespace gb {

// A lane takes eight consecutive elements = one block of the generator = 16 bytes (two times 16 for fp32) per tensor.
// `full`: blocks of eight that lie wholly inside n; the last lane takes the rest element by element.
template <typename T, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const T *__restrict__ x, const T *__restrict__ res, T *__restrict__ y,
                                                      long long n, unsigned q, float scale, const long long *__restrict__ rng,
                                                      long long seed, long long call, long long *__restrict__ used) {
  const RowRng g = load_rng(rng, seed, call);
  const long long t0 = (long long)blockIdx.x * 256 + threadIdx.x, stride = (long long)gridDim.x * 256;
  if (t0 == 0 && used) {
    used[0] = (long long)g.seed;
    used[1] = (long long)g.call;
  }
  const long long full = n >> 3;
  for (long long b = t0; b < full; b += stride) {
    F8 f = load8(x + 8 * b);
    F8 r;
    if (RES) r = load8(res + 8 * b);
    unsigned w[4];
    philox_block(g, (unsigned long long)b, w);
    const unsigned m = block_mask(w, q);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f.v[k] = (m >> k & 1) ? f.v[k] * scale : 0.0f;
      if (RES) f.v[k] += r.v[k];
    }
    store8(y + 8 * b, f);
  }
  if (t0 == 0 && (n & 7)) {
    unsigned w[4];
    philox_block(g, (unsigned long long)full, w);
    const unsigned m = block_mask(w, q);
    for (int k = 0; k < (int)(n & 7); ++k) {
      const long long i = 8 * full + k;
      float f = (m >> k & 1) ? (float)x[i] * scale : 0.0f;
      if (RES) f += (float)res[i];
      y[i] = (T)f;
    }
  }
}

}  // namespace gb

using namespace gb;

extern "C" int gb_dropout(const void *x, const void *residual, void *y, long long n, int dtype, int q, const int64_t *rng,
                          long long seed, long long call, int64_t *used, void *stream) {
  if (n < 0 || !known_type(dtype) || q < 0 || q > 65536) return GB_EINVAL;
  if (n == 0 && !used) return GB_OK;
  if (n > 0 && (!x || !y)) return GB_EINVAL;
  if ((reinterpret_cast<uintptr_t>(rng) | reinterpret_cast<uintptr_t>(used)) % 8 != 0) return GB_EINVAL;
  const long long blocks = ((n >> 3) + 255) / 256;
  const int grid = (int)(blocks < 1 ? 1 : blocks > 8192 ? 8192 : blocks);
  const float scale = keep_scale(q);
  return with_type(dtype, [&](auto z) {
    typedef decltype(z) T;
    if (residual)
      dropout_kernel<T, true><<<grid, 256, 0, as_stream(stream)>>>(
          (const T *)x, (const T *)residual, (T *)y, n, (unsigned)q, scale, (const long long *)rng, seed, call, (long long *)used);
    else
      dropout_kernel<T, false><<<grid, 256, 0, as_stream(stream)>>>(
          (const T *)x, nullptr, (T *)y, n, (unsigned)q, scale, (const long long *)rng, seed, call, (long long *)used);
    return check_launch("gb_dropout");
  });
}
