// Dropout from a counter-based generator (graspbal.h gb_dropout): y = x * keep / (1 - p) (+ residual), keep recomputed from
// (seed, call, element index) wherever it is needed - the backward pass is the same kernel on dy - and never stored.
#include "row_common.h"

#pragma clang fp contract(on)  // x * scale + residual in one instruction

namespace gb {

// A lane takes units of 16 bytes.  For the 16-bit types that is one block of the generator; for fp32 two lanes compute the
// same block - 40 integer products for four elements are a third of what the bytes take.
template <typename T, bool RES, bool NT>
__global__ __launch_bounds__(256) void dropout_kernel(const T *__restrict__ x, const T *__restrict__ res, T *__restrict__ y,
                                                      long long n, unsigned q, float scale, const long long *__restrict__ rng,
                                                      long long seed, long long call, long long *__restrict__ used) {
  constexpr int N = Unit<T>::N;
  const RowRng g = load_rng(rng, seed, call);
  const long long t0 = (long long)blockIdx.x * 256 + threadIdx.x, stride = (long long)gridDim.x * 256;
  if (t0 == 0 && used) {
    used[0] = (long long)g.seed;
    used[1] = (long long)g.call;
  }
  const long long full = n / N;
  for (long long u = t0; u < full; u += stride) {
    VecOf<T> f = load_unit<NT>(x + N * u);
    VecOf<T> r;
    if (RES) r = load_unit<NT>(res + N * u);
    const unsigned m = keep_mask<N>(g, (unsigned long long)(N * u), q);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      f.v[k] = (m >> k & 1) ? f.v[k] * scale : 0.0f;
      if (RES) f.v[k] += r.v[k];
    }
    store_unit<NT>(y + N * u, f);
  }
  if (t0 == 0 && n % N) {
    const unsigned m = keep_mask<N>(g, (unsigned long long)(N * full), q);
    for (int k = 0; k < (int)(n % N); ++k) {
      const long long i = N * full + k;
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
  const float scale = keep_scale(q);
  return with_type(dtype, [&](auto z) {
    typedef decltype(z) T;
    const long long blocks = (n / Unit<T>::N + 255) / 256;
    const int grid = (int)(blocks < 1 ? 1 : blocks > 8192 ? 8192 : blocks);
    auto launch = [&](auto kernel) {
      kernel<<<grid, 256, 0, as_stream(stream)>>>((const T *)x, (const T *)residual, (T *)y, n, (unsigned)q, scale,
                                                  (const long long *)rng, seed, call, (long long *)used);
    };
    const bool nt = streams(n * (long long)sizeof(T));
    if (residual)
      nt ? launch(dropout_kernel<T, true, true>) : launch(dropout_kernel<T, true, false>);
    else
      nt ? launch(dropout_kernel<T, false, true>) : launch(dropout_kernel<T, false, false>);
    return check_launch("gb_dropout");
  });
}
