// rope.hip -- rotary positions on the heads of some tokens.
//
// Bound by bytes: every value is read and written once, the angles are shared
// by all heads of a token.  A workgroup takes some tokens and some of their
// heads: it forms the tokens' sin and cos once (f64 angles, f32 results) in
// LDS, then each thread rotates 16 bytes of one half and 16 of the other
// (half layout) or 16 bytes of neighbours (interleaved) at a time.  4001 tokens
// of 72 heads of 128 (bf16, 64 values of each rotated, 147 MB) take 31 us,
// 4.7 TB/s, of 29 at the rate of a large copy.
#include "rope.h"

#include <algorithm>

namespace kq {

template <class T, int V> struct RVec { T v[V]; };

struct RopeArgs {
  RopeTable t;
  const void* x;
  void* y;
  long long xs, ys;
  const int* pos;
  int n_tok, n_heads, head_dim, tpb, hpb, rot_units, units;
  float sign;
};

template <class T, int V, bool INTER>
__global__ __launch_bounds__(256) void rope_rotate(RopeArgs a) {
  extern __shared__ float2 cs[];  // [token][rot / 2]
  const int half = a.t.rot_dim >> 1;
  const int t0 = blockIdx.x * a.tpb, nt = min(a.tpb, a.n_tok - t0);
  const int h0 = blockIdx.y * a.hpb, nh = min(a.hpb, a.n_heads - h0);
  for (int i = threadIdx.x; i < nt * half; i += 256) {
    const int t = i / half, p = i - t * half;
    double s, c;
    sincos_f64((double)a.pos[t0 + t] * a.t.freq[p], s, c);
    cs[i] = make_float2((float)(c * a.t.mag), (float)(s * a.t.mag) * a.sign);
  }
  __syncthreads();
  const int per = 256 / a.units;  // (token, head) pairs at a time
  const int slot = threadIdx.x / a.units, u = threadIdx.x - slot * a.units;
  if (slot >= per) return;
  int t = slot / nh, h = slot - t * nh;
  while (t < nt) {
    const T* x = (const T*)a.x + (size_t)(t0 + t) * a.xs + (size_t)(h0 + h) * a.head_dim;
    T* y = (T*)a.y + (size_t)(t0 + t) * a.ys + (size_t)(h0 + h) * a.head_dim;
    const float2* w = cs + t * half;
    if (u < a.rot_units) {
      if constexpr (INTER) {
        static_assert(V % 2 == 0, "pairs stay together");
        RVec<T, V> r;
        __builtin_memcpy(&r, x + u * V, sizeof(r));
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float2 k = w[u * (V / 2) + e / 2];
          const float p = (float)r.v[e], q = (float)r.v[e + 1];
          r.v[e] = (T)__builtin_fmaf(p, k.x, -(q * k.y));
          r.v[e + 1] = (T)__builtin_fmaf(p, k.y, q * k.x);
        }
        __builtin_memcpy(y + u * V, &r, sizeof(r));
      } else {
        RVec<T, V> r, s;
        __builtin_memcpy(&r, x + u * V, sizeof(r));
        __builtin_memcpy(&s, x + half + u * V, sizeof(s));
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 k = w[u * V + e];
          const float p = (float)r.v[e], q = (float)s.v[e];
          r.v[e] = (T)__builtin_fmaf(p, k.x, -(q * k.y));
          s.v[e] = (T)__builtin_fmaf(p, k.y, q * k.x);
        }
        __builtin_memcpy(y + u * V, &r, sizeof(r));
        __builtin_memcpy(y + half + u * V, &s, sizeof(s));
      }
    } else {  // the part of the head behind rot_dim passes through
      RVec<T, V> r;
      __builtin_memcpy(&r, x + a.t.rot_dim + (u - a.rot_units) * V, sizeof(r));
      __builtin_memcpy(y + a.t.rot_dim + (u - a.rot_units) * V, &r, sizeof(r));
    }
    for (h += per; h >= nh && t < nt; h -= nh) ++t;
  }
}

template <class T, int V, bool INTER>
static void rope_go(RopeArgs& a, hipStream_t s) {
  const int half = a.t.rot_dim / 2;
  a.rot_units = (INTER ? a.t.rot_dim : half) / V;
  a.units = a.rot_units + (a.x == a.y ? 0 : (a.head_dim - a.t.rot_dim) / V);
  // Tokens that fill a workgroup's sincos, then heads for about four units a
  // thread.
  a.tpb = std::max(1, std::min(a.n_tok, 256 / half));
  a.hpb = std::max(1, std::min(a.n_heads, 1024 / (a.tpb * a.units)));
  const dim3 grid((a.n_tok + a.tpb - 1) / a.tpb, (a.n_heads + a.hpb - 1) / a.hpb);
  hipLaunchKernelGGL((rope_rotate<T, V, INTER>), grid, dim3(256), (size_t)a.tpb * half * sizeof(float2), s, a);
}

// The widest vector, up to 16 bytes, that divides the runs of a head; 0 where
// that leaves more than one unit per thread.
static int rope_width(const RopeTable& t, int type, int head_dim) {
  const int run = t.interleaved ? t.rot_dim : t.rot_dim / 2, rest = head_dim - t.rot_dim;
  const int wide = type == ACT_F32 ? 4 : 8;
  for (int v : {wide, 2, t.interleaved ? 2 : 1})
    if (run % v == 0 && rest % v == 0) return run / v + rest / v <= 256 ? v : 0;
  return 0;
}

bool rope_takes(const RopeTable& t, int type, int head_dim) { return rope_width(t, type, head_dim) != 0; }

template <class T>
static bool rope_typed(RopeArgs& a, int v, hipStream_t s) {
  constexpr int W = 16 / sizeof(T);
  if (a.t.interleaved) {
    if (v == W) rope_go<T, W, true>(a, s);
    else if (v == 2) rope_go<T, 2, true>(a, s);
    else return false;
  } else {
    if (v == W) rope_go<T, W, false>(a, s);
    else if (v == 2) rope_go<T, 2, false>(a, s);
    else if (v == 1) rope_go<T, 1, false>(a, s);
    else return false;
  }
  return true;
}

hipError_t launch_rope(const RopeTable& t, int type, const void* x, long long x_stride, int n_tok, int n_heads,
                       int head_dim, const int* pos, bool inverse, void* y, long long y_stride, hipStream_t s) {
  RopeArgs a{};
  a.t = t;
  a.x = x;
  a.y = y;
  a.xs = x_stride;
  a.ys = y_stride;
  a.pos = pos;
  a.n_tok = n_tok;
  a.n_heads = n_heads;
  a.head_dim = head_dim;
  a.sign = inverse ? -1.f : 1.f;
  const int v = rope_width(t, type, head_dim);
  const bool ok = type == ACT_F32 ? rope_typed<float>(a, v, s)
                : type == ACT_F16 ? rope_typed<_Float16>(a, v, s) : rope_typed<bf16_t>(a, v, s);
  return ok ? hipGetLastError() : hipErrorInvalidValue;
}

}  // namespace kq
