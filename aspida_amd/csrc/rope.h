// rope.h -- rotary positions: the rotation table and its device math.
//
// A rotation turns pair i of a head (i < rot_dim / 2) by theta = pos * f_i:
//   (a, b) -> mag (a cos theta - b sin theta, a sin theta + b cos theta).
// theta is formed in f64 (one rounding of pos * f_i), since at position 10^5
// an f32 angle is off by a hundredth of a radian.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kq {

constexpr int ROPE_MAX_ROT = 256;
constexpr double ROPE_MAX_FREQ = 524288.0;  // |pos f| <= 2^50, as sincos_f64 needs

// Passed to the kernels by value (1 KB of arguments), so a captured graph
// holds the table itself and no device memory belongs to a rotation.
struct RopeTable {
  double freq[ROPE_MAX_ROT / 2];
  double mag;
  int rot_dim, interleaved;
};

enum ActType : int { ACT_F32 = 0, ACT_F16 = 1, ACT_BF16 = 2 };

// Whether launch_rope has a form for these runs: a head of at most 256 pieces
// of 16 bytes, two values or one (half layout), whichever divides it.
bool rope_takes(const RopeTable& t, int type, int head_dim);
hipError_t launch_rope(const RopeTable& t, int type, const void* x, long long x_stride, int n_tok, int n_heads,
                       int head_dim, const int* pos, bool inverse, void* y, long long y_stride, hipStream_t s);

#ifdef __HIPCC__
typedef __bf16 bf16_t;

template <class T> __device__ __forceinline__ float act_f32(T v) { return (float)v; }

// sin and cos of theta to about an ulp of f64 for |theta| <= 2^50: theta less
// the nearest multiple n of pi/2 in two fma steps (pi/2 as a sum of two f64;
// n times what a third would add is below 2^-59), then the Taylor series at
// |r| <= pi/4 (0.86 at 2^50, where n may be the second nearest), whose first
// dropped terms are r^19/19! and r^18/18! (below 2^-56).
__device__ __forceinline__ void sincos_f64(double theta, double& s, double& c) {
  // n + 1.5 2^52 has n's low bits at the end of its significand.
  const double at = __builtin_fma(theta, 0.63661977236758134308, 6755399441055744.0);
  const double n = at - 6755399441055744.0;
  double r = __builtin_fma(-n, 1.5707963267948965580, theta);
  r = __builtin_fma(-n, 6.1232339957367660359e-17, r);
  const double z = r * r;
  double p = 1.0 / 355687428096000.0;
  p = __builtin_fma(p, z, -1.0 / 1307674368000.0);
  p = __builtin_fma(p, z, 1.0 / 6227020800.0);
  p = __builtin_fma(p, z, -1.0 / 39916800.0);
  p = __builtin_fma(p, z, 1.0 / 362880.0);
  p = __builtin_fma(p, z, -1.0 / 5040.0);
  p = __builtin_fma(p, z, 1.0 / 120.0);
  p = __builtin_fma(p, z, -1.0 / 6.0);
  const double sn = __builtin_fma(p * z, r, r);
  double q = 1.0 / 20922789888000.0;
  q = __builtin_fma(q, z, -1.0 / 87178291200.0);
  q = __builtin_fma(q, z, 1.0 / 479001600.0);
  q = __builtin_fma(q, z, -1.0 / 3628800.0);
  q = __builtin_fma(q, z, 1.0 / 40320.0);
  q = __builtin_fma(q, z, -1.0 / 720.0);
  q = __builtin_fma(q, z, 1.0 / 24.0);
  q = __builtin_fma(q, z, -0.5);
  const double cs = __builtin_fma(q, z, 1.0);
  const int k = (int)__builtin_bit_cast(uint64_t, at) & 3;
  const double u = (k & 1) ? cs : sn, w = (k & 1) ? sn : cs;
  s = (k & 2) ? -u : u;
  c = (k == 1 || k == 2) ? -w : w;
}
#endif

}  // namespace kq
