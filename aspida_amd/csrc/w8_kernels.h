// w8_kernels.h -- what the kernels of products with 8-bit integer weights
// share: results from sums, and which of them takes a call.
#pragma once
#include "w8.h"

namespace kq {

// Whether the kernel for few tokens takes a call, and finds the tokens' codes itself.
bool w8_rows_takes(const W8Args& a);
bool w8_rows_fuse(const W8Args& a);
hipError_t launch_w8_rows(int type, const W8Args& a, hipStream_t s);

#ifdef __HIPCC__
// Token t's results o .. o + 3 (o a multiple of 4) from the sums of the
// weights' and (gated) the up projection's rows.
template <class T, bool GATED>
__device__ __forceinline__ void w8_finish(const W8Args& a, int t, int o, w8i4 sum, w8i4 up, const W8Unit& ux) {
  const float* const sw = w8_scales(a.w, a.in_dim, a.out_dim) + o;
  T* const y = (T*)a.y + (long long)t * a.y_stride + o;
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = w8_value(sum[e], W8Unit(sw[e]), ux);
    if constexpr (GATED)
      v[e] = w8_gate(v[e], w8_value(up[e], W8Unit(w8_scales(a.up, a.in_dim, a.out_dim)[o + e]), ux), a.act);
  }
  if (o + 4 <= a.out_dim) {
    struct { T t[4]; } r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r.t[e] = (T)v[e];
    __builtin_memcpy(y, &r, sizeof(r));
  } else {
    for (int e = 0; e < a.out_dim - o; ++e) y[e] = (T)v[e];
  }
}
#endif

}  // namespace kq
