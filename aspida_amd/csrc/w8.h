// w8.h -- products with 8-bit integer weights: layout and launchers.
//
// A weight row has int8 codes c_w and an f32 scale s_w, a token's activations
// codes c_x and a scale s_x of their own, found when the product is called:
//   s_x = f32(max |x| / 127),   c_x = x / s_x rounded to nearest, ties to even,
//   y = s_x s_w sum_k c_x c_w,
// the sum exact in int32 (in_dim <= 131072: at most 131072 * 127 * 128 < 2^31).
// A token whose largest magnitude is below 2^-100 counts as zeros, so that s_x
// is a normal number; one with a value that is not finite gets the scale NaN.
//
// Codes of weights (packed once) and of tokens (in the caller's workspace) lie
// in tiles of 16 rows x 64 k, [tile][k block][lane 64][16 bytes], lane = 16 (k
// / 16 % 4) + row % 16: what a lane of v_mfma_i32_16x16x64_i8 takes, so a
// tile's load is one line of 1 KB for registers and for LDS alike.  The blocks
// are an even number.  Packed weights are zero past in_dim; rows past the last
// and tokens past in_dim may be anything (their products are dropped, or zero).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "rope.h"

namespace kq {

constexpr int W8_MAX_IN = 131072;
constexpr int W8_TILE = 1024;  // bytes of a tile

__host__ __device__ inline int w8_blocks(int in_dim) { return (in_dim + 127) / 128 * 2; }
__host__ __device__ inline int w8_tiles(int rows) { return (rows + 15) / 16; }
__host__ __device__ inline size_t w8_code_bytes(int in_dim, int rows) {
  return (size_t)w8_tiles(rows) * w8_blocks(in_dim) * W8_TILE;
}
// Codes, then a scale per row of every tile.
inline size_t w8_bytes(int in_dim, int rows) {
  return (w8_code_bytes(in_dim, rows) + (size_t)w8_tiles(rows) * 64 + 255) / 256 * 256;
}

// Weights: from int8 rows and scales, or from rows of a quantised kind (kq_common.h) or of f32 (kind -1).
hipError_t launch_w8_pack(const int8_t* codes, long long stride, const float* scale, int in_dim, int out_dim,
                          uint8_t* packed, hipStream_t s);
hipError_t launch_w8_convert(int kind, const void* w, int in_dim, int out_dim, uint8_t* packed, hipStream_t s);
hipError_t launch_w8_unpack(const uint8_t* packed, int in_dim, int out_dim, float* w, hipStream_t s);

struct W8Args {
  const uint8_t* w;   // packed weights, of the gate projection in a gated block
  const uint8_t* up;  // null in a plain product
  int in_dim, out_dim, n_tok;
  const void* x;
  long long x_stride;
  void* y;
  long long y_stride;
  uint8_t* work;      // w8_bytes(in_dim, n_tok)
  int act;            // of a gated block: 0 silu, 1 gelu (tanh form)
};
hipError_t launch_w8(int type, const W8Args& a, hipStream_t s);

#ifdef __HIPCC__
typedef int w8i4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ w8i4 w8_mfma(w8i4 a, w8i4 b, w8i4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// A row's scale from its largest magnitude (NaN where a value is not finite:
// `top` is then not finite), and 1 / scale or 0.
struct W8Scale {
  float s, inv;
  __device__ __forceinline__ explicit W8Scale(float top) {
    s = top / 127.f;
    inv = 1.f / s;
    if (top < 0x1p-100f) s = inv = 0.f;
    if (!(top <= 3.402823466e38f)) { s = __builtin_nanf(""); inv = 0.f; }
  }
  // The nearest code.  x * inv is off by less than a step, so the remainder
  // x - s r (exact: it has at most 24 bits) tells which neighbour is nearer.
  __device__ __forceinline__ int code(float x) const {
    float r = __builtin_rintf(x * inv);
    const float t = __builtin_fmaf(-s, r, x), a = __builtin_fabsf(t), half = 0.5f * s;
    const float one = __builtin_copysignf(1.f, t);
    const bool odd = __builtin_fabsf(__builtin_fmaf(-2.f, __builtin_rintf(0.5f * r), r)) > 0.5f;
    if (a > half || (a == half && odd)) r += one;
    return inv == 0.f ? 0 : (int)r;
  }
};

__device__ __forceinline__ uint32_t w8_four(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

// s_x s_w sum: as significands and exponents, so that the product of two tiny
// (or a large and a tiny) scales loses nothing before the sum is in it.
struct W8Unit {
  float m;
  int e;
  __device__ __forceinline__ explicit W8Unit(float s) : m(__builtin_amdgcn_frexp_mantf(s)), e(__builtin_amdgcn_frexp_expf(s)) {}
};
__device__ __forceinline__ float w8_value(int sum, float m, int e, const W8Unit& b) {
  return __builtin_ldexpf((float)sum * m * b.m, e + b.e);
}

// act(g) u, act(g) = g / (1 + e^-t): t = g is silu, t = 2 sqrt(2 / pi) (g +
// 0.044715 g^3) gelu in its tanh form.  For t < 0 it is g e^t / (1 + e^t), e^t
// multiplied in as two roots, so that nothing but the result leaves f32's
// range (down to t = -174, where the roots do).  exp2 and the reciprocal of a
// number in [1, 2] are the instructions', good to an ulp: a prompt's 30 million
// results would otherwise spend as long here as an eighth of their products.
__device__ __forceinline__ float w8_gate(float g, float u, int act) {
  const float t = act == 0 ? g : 1.5957691216057308f * __builtin_fmaf(0.044715f * g * g, g, g);
  const float h = __builtin_amdgcn_exp2f(-0.72134752044448170368f * __builtin_fabsf(t));
  const float p = t < 0.f ? h : 1.f;
  return g * p * u * p * __builtin_amdgcn_rcpf(__builtin_fmaf(h, h, 1.f));
}

// Runs of 16 consecutive activations.  w8_run: a whole one, at any alignment
// of the type; w8_rest: the one that in_dim ends in, zeros behind it.
template <class T> struct W8Run {
  T t[16];
  __device__ __forceinline__ void values(float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = (float)t[i];
  }
};
template <class T> __device__ __forceinline__ W8Run<T> w8_run(const T* x) {
  W8Run<T> r;
  __builtin_memcpy(&r, x, sizeof(r));
  return r;
}
template <class T> __device__ __forceinline__ W8Run<T> w8_rest(const T* x, int n) {
  W8Run<T> r;
#pragma unroll
  for (int i = 0; i < 16; ++i) r.t[i] = i < n ? x[i] : (T)0.f;
  return r;
}
// The larger magnitude; infinite where one is not finite.
__device__ __forceinline__ float w8_top(float top, float v) {
  const float a = __builtin_fabsf(v);
  return a <= 3.402823466e38f ? __builtin_fmaxf(top, a) : __builtin_inff();
}
// Magnitudes as bits, which order as the numbers do; NaN above infinity.
template <class T> __device__ __forceinline__ uint32_t w8_top16(const W8Run<T>& r, uint32_t top) {
  float v[16];
  r.values(v);
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
  return top;
}
// 16 codes of a wave's lanes at a time.  x inv + 1.5 2^23, rounded once, has
// the code in its lowest byte; x inv is off by at most 127 2^-24, so only
// where one comes within 2^-16 of a half are the lane's codes settled one by
// one (three steps of 1024 values in a hundred).  That is 5 instructions a
// value in place of about 20, which were most of the time of long rows.
template <class T> __device__ __forceinline__ uint4 w8_codes16(const W8Run<T>& run, const W8Scale& s) {
  constexpr float M = 12582912.f;
  float v[16], r[16], far = 0.f;
  run.values(v);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    r[i] = __builtin_fmaf(v[i], s.inv, M);
    far = __builtin_fmaxf(far, __builtin_fabsf(__builtin_fmaf(v[i], s.inv, M - r[i])));
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    auto bits = [&](int j) { return __builtin_bit_cast(uint32_t, r[4 * i + j]); };
    // Bytes of (a, b): 0..3 are b's, 4..7 a's.
    const uint32_t lo = __builtin_amdgcn_perm(bits(1), bits(0), 0x0C0C0400u), hi = __builtin_amdgcn_perm(bits(3), bits(2), 0x04000C0Cu);
    w[i] = lo | hi;
  }
  if (__ballot(far > 0.5f - 0x1p-16f)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = w8_four(s.code(v[4 * i]), s.code(v[4 * i + 1]), s.code(v[4 * i + 2]), s.code(v[4 * i + 3]));
  }
  return s.inv == 0.f ? make_uint4(0, 0, 0, 0) : make_uint4(w[0], w[1], w[2], w[3]);
}

// Where codes k .. k + 15 (k a multiple of 16) of a row stand.
__device__ __forceinline__ size_t w8_place(int row, int k, int blocks) {
  return ((size_t)(row >> 4) * blocks + (k >> 6)) * W8_TILE + ((k >> 4 & 3) * 16 + (row & 15)) * 16;
}
__device__ __forceinline__ float* w8_scales(const uint8_t* packed, int in_dim, int rows) {
  return reinterpret_cast<float*>(const_cast<uint8_t*>(packed) + w8_code_bytes(in_dim, rows));
}

// Largest value over a wave, and over a workgroup of NW waves, in every thread.
template <class V> __device__ __forceinline__ V w8_wave_max(V v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max(v, (V)__shfl_xor(v, o, 64));
  return v;
}
template <int NW, class V>
__device__ __forceinline__ V w8_group_max(V v, V* lds) {
  v = w8_wave_max(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) v = max(v, lds[i]);
  return v;
}
#endif

}  // namespace kq
