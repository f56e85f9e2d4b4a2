// kv4_stage.h -- 32 tokens of the 4-bit cache as operands of the 32x32x16
// matrix instructions in LDS, for kernels whose waves share them
// (kv4_prefill.hip, kv4_tree.hip).
#pragma once
#include "kv4_mma.h"

namespace kq {

__device__ __forceinline__ kvf16 kv_mfma32(kvh8 a, kvh8 b, kvf16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// LDS of one stage, 32 tokens: operands of 1 KB (a lane's eight halves at 16 lane).
template <int D, bool TWO> struct StageLds {
  static constexpr int NG = D / 32;
  static constexpr int K = 0;                    // [D / 16 steps]
  static constexpr int V = K + 64 * D;           // [D / 32 dim tiles][2 steps]
  static constexpr int KM = V + 64 * D;          // minima of keys: [32 tokens][8]
  static constexpr int VM = KM + 512;            // of values: [2 steps][2 lane halves][16 rows][8]
  static constexpr int VL = VM + 1024;           // what m + 8 d leaves after its f16 (f32 activations)
  static constexpr int BYTES = VL + (TWO ? 1024 : 0);
};

// What a thread loads of a stage and later writes to LDS.  128 threads have
// the keys, 128 the values; with eight waves, four take the even stages and
// four the odd ones, so of the two waves of a SIMD one unpacks at a time.
// Both halves load by the same instructions at offsets of their own: with a
// branch the compiler joins the two halves' registers by moves, which wait
// for the loads at once.
template <int D, bool TWO> struct StageLoad {
  static constexpr int NG = D / 32, QG = Kv4L<D>::QG, HALF = 128;
  static constexpr int KTASKS = 2 * 64 * (NG / QG), VTASKS = D;
  static constexpr int KN = KTASKS / HALF, VN = (VTASKS + HALF - 1) / HALF, N = KN > VN ? KN : VN;
  // Keys: w the code words, d the steps of their token (from group 0).
  // Values: w the code words of four 16-dim tiles, d and d2 the tokens' steps
  // of their two groups.
  kvu4 w[N], d[N], d2[N];
  kvu4 m, md;  // a piece of the minima (and of the steps that go with it)
  int ow[N], od[N], om;
  bool there;

  __device__ __forceinline__ void place(bool values, int tid) {
    using L = Kv4L<D>;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = tid + i * HALF, lane = t & 63, quad = (t >> 6) % (NG / QG), tile = (t >> 6) / (NG / QG);
      const int ch = (t >> 6) % (D / 64);
      ow[i] = values ? L::V0 + ch * 1024 + lane * 16 : tile * L::KT + quad * (256 * QG) + lane * (4 * QG);
      od[i] = values ? L::VS0 + 2 * ch * 64 + (lane >> 4) * 16 : L::KS0 + (tile * 16 + (lane & 15)) * (4 * NG);
    }
    om = values ? L::VS0 + ((tid >> 2) % NG) * 64 + (tid & 3) * 16 + 64 * NG : L::KS0 + (tid & 31) * (4 * NG) + 2 * NG;
  }
  // blk: the stage's page, null where there is none.  (The second half of a
  // page lies 16 D bytes on in the codes, 4 D in the scales, and 16 bytes from
  // any of these offsets are in the block.)
  __device__ __forceinline__ void load(const uint8_t* blk, const uint8_t* any, int half) {
    there = blk != nullptr;
    if (!blk) blk = any;  // its steps and minima become 0 below
    const uint8_t *pw = blk + half * (16 * D), *ps = blk + half * (4 * D);
    auto at = [](const uint8_t* q) {
      kvu4 v;
      __builtin_memcpy(&v, __builtin_assume_aligned(q, 4), 16);
      return v;
    };
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i] = at(pw + ow[i]);
      d[i] = at(ps + od[i]);
      d2[i] = at(ps + od[i] + 64);
    }
    m = at(ps + om);
    if constexpr (TWO) md = at(ps + om - 64 * NG + (om < Kv4L<D>::VS0 ? 64 * NG : 0));
  }

  // Steps and minima of value tokens outside [lo, hi) (of the stage) become 0.
  static __device__ __forceinline__ kvu4 keep(kvu4 x, int rg, int lo, int hi) {
    uint32_t r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = 16 * (j >> 1) + 4 * rg + 2 * (j & 1);
      r[j] = x[j] & ((t >= lo && t < hi ? 0x0000FFFFu : 0u) | (t + 1 >= lo && t + 1 < hi ? 0xFFFF0000u : 0u));
    }
    return kvu4{r[0], r[1], r[2], r[3]};
  }

  __device__ __forceinline__ void store(uint8_t* lds, int lo, int hi, bool values, int tid) {
    using P = StageLds<D, TWO>;
    if (!values) {
#pragma unroll
      for (int i = 0; i < KN; ++i) {
        const int t = tid + i * HALF, lane = t & 63, quad = (t >> 6) % (NG / QG), tile = (t >> 6) / (NG / QG);
        const int tok = tile * 16 + (lane & 15), kg = lane >> 4;
        // Token tok's dims 32 g + 8 kg ..: step 2 g + kg / 2, lane half kg % 2.
        uint8_t* to = lds + P::K + ((kg & 1) * 32 + tok) * 16 + (kg >> 1) * 1024;
#pragma unroll
        for (int g = 0; g < QG; ++g) {
          const uint32_t two = NG == 8 && quad ? d[i][2 + (g >> 1)] : d[i][g >> 1];
          const kvh2 pair = kv_h2(two);
          const kvh2 dd = (g & 1) ? __builtin_shufflevector(pair, pair, 1, 1) : __builtin_shufflevector(pair, pair, 0, 0);
          *reinterpret_cast<kvh8*>(to + 2 * (quad * QG + g) * 1024) = kv4_unpack1(w[i][g], dd);
        }
      }
      // (What follows a token's minima is not its own.)  The scores of a page
      // that is not there are NaN.
      if constexpr (NG == 4) m = kvu4{m.x, m.y, 0, 0};
      if constexpr (NG == 2) m = kvu4{m.x, 0, 0, 0};
      if (!there) m = kvu4{0x7E007E00u, 0x7E007E00u, 0x7E007E00u, 0x7E007E00u};
      if (tid < 32) *reinterpret_cast<kvu4*>(lds + P::KM + tid * 16) = m;
      return;
    }
    if (!there) hi = 0;
    const bool cut = lo > 0 || hi < 32;
    if (cut) {
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const int rg = (tid & 63) >> 4;
        d[i] = keep(d[i], rg, lo, hi);
        d2[i] = keep(d2[i], rg, lo, hi);
      }
      m = keep(m, tid & 3, lo, hi);
      if constexpr (TWO) md = keep(md, tid & 3, lo, hi);
    }
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      const int t = tid + i * HALF;
      if (VTASKS % HALF && t >= VTASKS) continue;
      const int lane = t & 63, ch = t >> 6, rg = lane >> 4;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const kvu4 dd = e ? d2[i] : d[i];
        const kvh2 d0 = kv_h2(dd[0]), d1 = kv_h2(dd[1]), dd2 = kv_h2(dd[2]), d3 = kv_h2(dd[3]);
        // Dims 64 ch + 32 e + 16 f + lane % 16 are dim tile 2 ch + e; tokens 4 rg .. of the first 16 are
        // lane half rg % 2's, place rg / 2, of step 0, those of the other 16 of step 1.
        uint8_t* to = lds + P::V + (2 * ch + e) * 2048 + ((rg & 1) * 32 + (lane & 15)) * 16 + (rg >> 1) * 8;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const kvh8 v = TWO ? kv4_unpack_centered(w[i][2 * e + f], d0, d1, dd2, d3)
                             : kv4_unpack(w[i][2 * e + f], d0, d1, dd2, d3, kv_times(d0, -16.f), kv_times(d1, -256.f),
                                          kv_times(dd2, -16.f), kv_times(d3, -256.f));
          *reinterpret_cast<kvh4*>(to + f * 256) = __builtin_shufflevector(v, v, 0, 1, 2, 3);
          *reinterpret_cast<kvh4*>(to + f * 256 + 1024) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
        }
      }
    }
    if (tid < 4 * NG) {
      const int rg = tid & 3, g = tid >> 2;
      kvu4 mm = m;
      uint8_t* to = lds + P::VM + ((rg & 1) * 16 + g) * 16 + (rg >> 1) * 8;
      if constexpr (TWO) {
        uint32_t low[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const kvh2 mj = kv_h2(mm[j]), dj = kv_h2(md[j]);
          const float a = __builtin_fmaf(8.f, (float)dj.x, (float)mj.x), b = __builtin_fmaf(8.f, (float)dj.y, (float)mj.y);
          // m + 8 d may pass f16's largest value by 2032, which the low number then holds.
          const kvh2 hi2 = {(_Float16)fminf(a, 65504.f), (_Float16)fminf(b, 65504.f)};
          const kvh2 lo2 = {(_Float16)(a - (float)hi2.x), (_Float16)(b - (float)hi2.y)};
          mm[j] = __builtin_bit_cast(uint32_t, hi2);
          low[j] = __builtin_bit_cast(uint32_t, lo2);
        }
        *reinterpret_cast<kvu2*>(to + 1024) = kvu2{low[0], low[1]};
        *reinterpret_cast<kvu2*>(to + 1024 + 512) = kvu2{low[2], low[3]};
      }
      *reinterpret_cast<kvu2*>(to) = kvu2{mm[0], mm[1]};
      *reinterpret_cast<kvu2*>(to + 512) = kvu2{mm[2], mm[3]};
    }
  }
};

}  // namespace kq
