// kv4_mma.h -- the 4-bit cache as operands of the matrix instructions, and
// queries as theirs; shared by the attention and weight kernels.
#pragma once
#include "kq_common.h"
#include "kv4.h"

namespace kq {

__device__ __forceinline__ kvf4 kv_mfma(kvh8 a, kvh8 b, kvf4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ kvh2 kv_h2(uint32_t v) { return __builtin_bit_cast(kvh2, v); }
__device__ __forceinline__ kvh2 kv_fma2(kvh2 a, kvh2 b, kvh2 c) { return __builtin_elementwise_fma(a, b, c); }

// The eight codes of a dword times their steps, exact in f16: masked codes
// with the bits of 16.0 or 256.0 are 16 + q or 256 + q, and one fma takes the
// offset off again (d q has at most 11 bits).  dj: steps of codes (0, 1),
// (2, 3), (4, 5), (6, 7); nj: -16, -256, -16 and -256 times them.
__device__ __forceinline__ kvh8 kv4_unpack(uint32_t w, kvh2 d0, kvh2 d1, kvh2 d2, kvh2 d3, kvh2 n0, kvh2 n1, kvh2 n2,
                                           kvh2 n3) {
  const uint32_t r = __builtin_amdgcn_alignbit(w, w, 8);
  const kvh2 a = kv_fma2(kv_h2((w & 0x03C003C0u) | 0x4C004C00u), d0, n0);
  const kvh2 b = kv_fma2(kv_h2((w & 0x003C003Cu) | 0x5C005C00u), d1, n1);
  const kvh2 c = kv_fma2(kv_h2((r & 0x03C003C0u) | 0x4C004C00u), d2, n2);
  const kvh2 e = kv_fma2(kv_h2((r & 0x003C003Cu) | 0x5C005C00u), d3, n3);
  return kvh8{a.x, a.y, b.x, b.y, c.x, c.y, e.x, e.y};
}
__device__ __forceinline__ kvh2 kv_times(kvh2 a, float s) { return a * kvh2{(_Float16)s, (_Float16)s}; }

// The same less 8 steps, d (q - 8): -24 d takes the offset off, so every code
// stands at the bits of 16 + q.
__device__ __forceinline__ kvh8 kv4_unpack_centered(uint32_t w, kvh2 d0, kvh2 d1, kvh2 d2, kvh2 d3) {
  const uint32_t r = __builtin_amdgcn_alignbit(w, w, 8);
  const kvh2 a = kv_fma2(kv_h2((w & 0x03C003C0u) | 0x4C004C00u), d0, kv_times(d0, -24.f));
  const kvh2 b = kv_fma2(kv_h2(((w << 4) & 0x03C003C0u) | 0x4C004C00u), d1, kv_times(d1, -24.f));
  const kvh2 c = kv_fma2(kv_h2((r & 0x03C003C0u) | 0x4C004C00u), d2, kv_times(d2, -24.f));
  const kvh2 e = kv_fma2(kv_h2(((r << 4) & 0x03C003C0u) | 0x4C004C00u), d3, kv_times(d3, -24.f));
  return kvh8{a.x, a.y, b.x, b.y, c.x, c.y, e.x, e.y};
}

// Eight codes that share the step d2 = (d, d).
__device__ __forceinline__ kvh8 kv4_unpack1(uint32_t w, kvh2 d2) {
  const kvh2 n16 = kv_times(d2, -16.f), n256 = kv_times(d2, -256.f);
  return kv4_unpack(w, d2, d2, d2, d2, n16, n256, n16, n256);
}

// The score up to which exp2(c u - ref), its product not rounded, is sure to
// stay below 2^16 and so in f16: ref + 15 while products round by 1/4 at most.
// Beyond that none is: the product is rounded first, as the maximum was.
__device__ __forceinline__ float kv4_limit(float ref) {
  return __builtin_fabsf(ref) < 0x1p22f ? ref + 15.f : -__builtin_inff();
}

// The page ids of a sequence, 64 at a time in a wave's lanes: a lookup in a
// loop is a lane read, where a scalar load would make every LDS wait of the
// loop wait for it too.  Wave-uniform arguments.
struct PageIds {
  int ids, base;
  __device__ __forceinline__ void fill(const Kv4View& c, int b, int p, int lane) {
    base = p;
    ids = p + lane < c.max_pages ? c.table[(size_t)b * c.max_pages + p + lane] : -1;
  }
  // kv4_block for base <= p < base + 64.
  __device__ __forceinline__ uint8_t* at(const Kv4View& c, int p, int hk, int head_bytes) const {
    const int id = __builtin_amdgcn_readlane(ids, p - base);
    return (unsigned)id < (unsigned)c.n_pages ? c.pages + ((size_t)id * c.n_kv + hk) * head_bytes : nullptr;
  }
  // The same for ascending p from the first base on.  The refill's wait counts
  // every load in flight, so loops with loads ahead refill outside.
  __device__ __forceinline__ uint8_t* block(const Kv4View& c, int b, int p, int hk, int head_bytes, int lane) {
    if (p - base >= 64) fill(c, b, p, lane);
    return at(c, p, hk, head_bytes);
  }
};

// A load that leaves nothing in the caches: a cache is read once a step (64
// lanes of up to 8000 slots 85 -> 80 us; heads of 256 that the caches could
// have held, 8 lanes of 8000, 35 -> 37).
template <class V> __device__ __forceinline__ V kv_stream(const uint8_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
}

// A lane's words of a 16-token key tile: token lane % 16, lane group kg =
// lane / 16 of each group's dims; scales: all d of the token, then all m.
template <int D> struct KeyTile {
  static constexpr int NG = D / 32;
  uint32_t w[NG];
  uint32_t s[NG];
  __device__ __forceinline__ void load(const uint8_t* blk, int tile, int lane) {
    using L = Kv4L<D>;
    const uint8_t* p = blk + tile * L::KT + lane * (4 * L::QG);
    const uint8_t* q = blk + L::KS0 + (tile * 16 + (lane & 15)) * (4 * NG);
    if constexpr (NG == 2) {
      const kvu2 a = kv_stream<kvu2>(p), b = kv_stream<kvu2>(q);
      w[0] = a.x; w[1] = a.y; s[0] = b.x; s[1] = b.y;
    } else {
#pragma unroll
      for (int c = 0; c < NG / 4; ++c) {
        const kvu4 a = kv_stream<kvu4>(p + 1024 * c), b = kv_stream<kvu4>(q + 16 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) { w[4 * c + i] = a[i]; s[4 * c + i] = b[i]; }
      }
    }
  }
  __device__ __forceinline__ kvh2 d(int g) const {
    const kvh2 pair = kv_h2(s[g >> 1]);
    return (g & 1) ? __builtin_shufflevector(pair, pair, 1, 1) : __builtin_shufflevector(pair, pair, 0, 0);
  }
  // The operand of group g's code part: rows = tokens, k = dims.
  __device__ __forceinline__ kvh8 codes(int g) const { return kv4_unpack1(w[g], d(g)); }
  // The operand of the minima: k = groups in every lane group (the other
  // operand says which count).
  __device__ __forceinline__ kvh8 minima() const {
    uint32_t r[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NG / 2; ++i) r[i] = s[NG / 2 + i];
    return __builtin_bit_cast(kvh8, kvu4{r[0], r[1], r[2], r[3]});
  }
};

// A lane's words of a 32-token value block: dims 16 n + lane % 16, tokens 4 rg
// + 0..3 of both halves (rg = lane / 16); steps of those tokens per group and
// (group (lane % 16) % NG) their minima.
template <int D> struct ValueBlock {
  static constexpr int NG = D / 32;
  kvu4 w[D / 64];
  kvu4 d[NG];
  kvu4 m;
  __device__ __forceinline__ void load(const uint8_t* blk, int half, int lane) {
    using L = Kv4L<D>;
    const uint8_t* p = blk + L::V0 + half * L::VB + lane * 16;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) w[c] = kv_stream<kvu4>(p + 1024 * c);
    const uint8_t* s = blk + L::VS0 + half * L::VSB + (lane >> 4) * 16;
#pragma unroll
    for (int g = 0; g < NG; ++g) d[g] = kv_stream<kvu4>(s + 64 * g);
    m = kv_stream<kvu4>(s + 64 * NG + 64 * (lane & (NG - 1)));
  }
  // Steps and minima of the tokens whose bit of `keep` is clear become 0 (bit
  // j: the lane's token j).
  __device__ __forceinline__ void drop(uint32_t keep) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t mask = ((keep >> (2 * j)) & 1 ? 0x0000FFFFu : 0u) | ((keep >> (2 * j + 1)) & 1 ? 0xFFFF0000u : 0u);
#pragma unroll
      for (int g = 0; g < NG; ++g) d[g][j] &= mask;
      m[j] &= mask;
    }
  }
};

// Eight consecutive activations from p as f32.
template <class T>
__device__ __forceinline__ void kv_load8(const T* p, float (&x)[8]) {
  struct { T v[8]; } r;
  __builtin_memcpy(&r, p, sizeof(r));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)r.v[i];
}

// One query row as the other operand (cols = rows of q; lane % 16), scaled by
// a power of two so that its largest value is in [2^9, 2^10): hi is its f16,
// lo (f32 activations) what hi leaves.  bf16 and f16 values are exact in hi.
// sums: the groups' sums, hi in lane group 0, lo in lane group 1, which meet
// the key's minima.  unit: what a product must be multiplied by.
template <int D, bool TWO> struct Query {
  static constexpr int NG = D / 32;
  kvh8 hi[NG], lo[TWO ? NG : 1], sums;
  float unit;
  // turn: 1, or -1 for a negative scale.
  template <class T> __device__ __forceinline__ void load(const T* row, bool valid, int lane, float turn = 1.f) {
    const int kg = lane >> 4;
    float x[NG][8], top = 0.f;
    bool finite = true;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[g][j] = 0.f;
      if (valid) kv_load8(row + 32 * g + 8 * kg, x[g]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top = fmaxf(top, fabsf(x[g][j]));
        finite = finite && __builtin_isfinite(x[g][j]);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int e = 10;
    if (top > 0.f && top <= 3.402823466e38f) e = __builtin_amdgcn_frexp_expf(top);
    unit = ldexpf(1.f, e - 10);
    // What is not finite stays so: its row's scores are NaN.
    if (!finite) unit = __builtin_nanf("");
    unit += 0.f * __shfl_xor(unit, 16, 64);
    unit += 0.f * __shfl_xor(unit, 32, 64);
    float sg[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = ldexpf(finite ? x[g][j] : 0.f, 10 - e) * turn;
        const _Float16 h = (_Float16)c;
        hi[g][j] = h;
        if constexpr (TWO) lo[g][j] = (_Float16)(c - (float)h);
        sum += c;
      }
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      const _Float16 h = (_Float16)sum;
      sg[g] = kg == 0 ? (float)h : kg == 1 ? sum - (float)h : 0.f;
    }
#pragma unroll
    for (int g = 0; g < 8; ++g) sums[g] = (_Float16)sg[g];
  }
  // Code and minimum products of a key tile: C[token][row], lane: row lane %
  // 16, tokens 4 (lane / 16) + 0..3; to be multiplied by unit.
  __device__ __forceinline__ kvf4 scores(const KeyTile<D>& k) const {
    kvf4 c = kv_mfma(k.minima(), sums, kvf4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const kvh8 a = k.codes(g);
      if constexpr (TWO) c = kv_mfma(a, lo[g], c);
      c = kv_mfma(a, hi[g], c);
    }
    return c;
  }
};

}  // namespace kq
