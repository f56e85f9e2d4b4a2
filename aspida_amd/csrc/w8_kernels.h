// w8_kernels.h -- what the kernels of products with 8-bit integer weights
// share: results from sums, and which of them takes a call.
#pragma once
#include "w8.h"

namespace kq {

// Whether the kernel for few tokens takes a call, and finds the tokens' codes itself.
bool w8_rows_takes(const W8Args& a);
bool w8_rows_fuse(const W8Args& a);
hipError_t launch_w8_rows(int type, const W8Args& a, hipStream_t s);

// LDS that a launch asks for: at least so much that no compute unit takes more
// than its share of the workgroups, at most `room`, while others have none.
inline int w8_spread(int lds, int groups, int room) {
  const int each = groups <= 256 ? 1 : room;
  const int least = 160 * 1024 / (each + 1) + 1024;  // 1 + each of these do not fit
  return lds > least ? lds : least;
}

#ifdef __HIPCC__
// Memory from p on; offsets are bounded by the kernels.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w8_buffer(const uint8_t* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), (short)0, 0x7FFFFFFF, 0x00020000);
}
// 16 bytes per lane to LDS (lane l's at lds + 16 l).  Loads come in order: a
// wait for at most n outstanding ones covers all with n later ones.  AUX 2:
// read once, to leave the caches alone.
template <int AUX> __device__ __forceinline__ void w8_to_lds(__amdgpu_buffer_rsrc_t r, int lane_off, int off, uint32_t lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(uintptr_t)lds, 16, lane_off, off, 0, AUX);
}

// The scales of rows o .. o + 3 (o a multiple of 4) of the weights and (gated)
// of the up projection, and those rows' results for token t from their sums.
template <bool GATED> struct W8Rows {
  float m[GATED ? 2 : 1][4];
  int e[GATED ? 2 : 1][4];
  __device__ __forceinline__ W8Rows(const W8Args& a, int o) {
#pragma unroll
    for (int p = 0; p < (GATED ? 2 : 1); ++p) {
      const float* const s = w8_scales(p ? a.up : a.w, a.in_dim, a.out_dim) + o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const W8Unit u(s[i]);
        m[p][i] = u.m;
        e[p][i] = u.e;
      }
    }
  }
  // The same of lane group `kg` of a tile (wave-uniform), by scalar loads: they
  // do not wait for vector loads on their way.
  __device__ __forceinline__ W8Rows(const W8Args& a, int tile, int kg) {
    typedef const __attribute__((address_space(4))) float* Scalar;
#pragma unroll
    for (int p = 0; p < (GATED ? 2 : 1); ++p) {
      const Scalar s = (Scalar)(uintptr_t)(w8_scales(p ? a.up : a.w, a.in_dim, a.out_dim) + 16 * tile);
      uint32_t x16[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x16[i] = __builtin_bit_cast(uint32_t, s[i]);
        asm volatile("" : "+s"(x16[i]));  // (or the choice below becomes one vector load)
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t bits = kg < 2 ? (kg == 0 ? x16[i] : x16[4 + i]) : (kg == 2 ? x16[8 + i] : x16[12 + i]);
        const float x = __builtin_bit_cast(float, bits);
        const W8Unit u(x);
        m[p][i] = u.m;
        e[p][i] = u.e;
      }
    }
  }
  template <class T>
  __device__ __forceinline__ void finish(const W8Args& a, int t, int o, w8i4 sum, w8i4 up, const W8Unit& ux) const {
    T* const y = (T*)a.y + (long long)t * a.y_stride + o;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = w8_value(sum[i], m[0][i], e[0][i], ux);
      if constexpr (GATED) v[i] = w8_gate(v[i], w8_value(up[i], m[1][i], e[1][i], ux), a.act);
    }
    if (o + 4 <= a.out_dim) {
      struct { T t[4]; } r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r.t[i] = (T)v[i];
      __builtin_memcpy(y, &r, sizeof(r));
    } else {
      for (int i = 0; i < a.out_dim - o; ++i) y[i] = (T)v[i];
    }
  }
};
#endif

}  // namespace kq
