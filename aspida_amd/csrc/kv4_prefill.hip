// kv4_prefill.hip -- attention of many rows over the 4-bit cache.
//
// A workgroup takes 32 columns (rows times query heads of one kv head) per
// wave and walks the slots that they see in stages of 32 tokens.  The waves
// turn a stage's codes into f16 operands in LDS once (exact, kv4_mma.h), in
// the order the 32x32x16 instructions read them, two stages ahead; per stage
//   S[token][col] = K Q^T      D / 16 steps, and one for the minima
//   P = exp2(S - ref)          ref moves when a score passes it by 15
//   O[dim][col] += V^T P       P in S's own registers: the steps' token order
//                              is the one in which S's lanes hold them
//   M[g][col] += m^T P         the minima, with a row of ones that sums P
// P is two f16 planes, each in turn, for every type (one leaves 2^-11 of a
// weight, as much as an f16 result's own rounding).  f32 activations: two of Q
// as well, and value codes less 8 (d (q - 8), with m + 8 d as two f16 in place
// of m): the sums over thousands of slots then stay near the result instead of
// cancelling against the minima (6000 slots: error 3.1e-6 before, of 1.5e-6 in
// plain f32).
// Bound by waiting: of a busy compute unit's cycles the matrix cores work 51%
// (f32 60%), the vector units 52% (44%: unpacking, exp2, the planes of P),
// LDS 30%, and each of the two waves a SIMD waits a third of its time for data
// and the barrier of every 32 tokens.  2000 rows behind 4000 slots (32/8 heads
// of 128, f32, 164 GFLOP, twice with both planes) 397 us, 830 TFLOP/s of them;
// prompts up to 4097 rows (bf16, 391 GFLOP, half as many again for P's low
// plane) 688 us, 850 TFLOP/s; a large f16 product reaches 1108.  Measured and
// not taken: four waves a workgroup, priorities of waves, dwords instead of
// 16-byte pieces per unpacking thread (with one plane of P 598 us for 557).
#include <algorithm>

#include "kv4_stage.h"

namespace kq {

struct PrefillArgs {
  Kv4View c;
  Kv4Rows rows;
  Kv4Attn a;
  int group;
};

constexpr float PF_LOG2E = 1.4426950408889634f, PF_LN2 = 0.6931471805599453f;

template <int D, class T, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 ? 2 : 1) void kv4_prefill(PrefillArgs s) {
  constexpr bool TWO = sizeof(T) == 4;
  using P = StageLds<D, TWO>;
  constexpr int NG = D / 32, NS = D / 16, THREADS = 64 * WAVES, COLS = 32 * WAVES;
  extern __shared__ uint8_t lds[];  // three stages, and the low plane of Q
  const int lane = threadIdx.x & 63, col = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.x % s.c.n_kv, b = blockIdx.z;
  const Kv4Span sp = kv4_span(s.rows, b);
  const int n = sp.r1 - sp.r0, nr = min(n, s.a.max_rows);
  // The last rows, which see most, come first.
  const int tiles = (int)(((long long)nr * s.group + COLS - 1) / COLS), tile = tiles - 1 - (int)(blockIdx.x / s.c.n_kv);
  if (tile < 0) return;
  const int c0 = tile * COLS, c1 = min(c0 + COLS, nr * s.group);  // the workgroup's columns
  const int first = sp.len - n;                                   // slot of row 0
  const int max_slots = s.c.max_pages * KV4_PAGE, reach = kv4_reach(s.a.window);
  const int any_hi = min(first + (c1 - 1) / s.group + 1, max_slots);
  const int any_lo = kv4_lowest(first + c0 / s.group, reach);

  // This lane's column, and what the wave's columns all see and see at all.
  const int w0 = c0 + 32 * wave, w1 = min(w0 + 32, c1) - 1;
  const int ci = w0 + col, row = ci / s.group, head = hk * s.group + ci % s.group;
  const bool valid = ci < c1;
  const int pos = first + row;
  const int chi = valid ? max(pos + 1, 0) : 0, clo = kv4_lowest(pos, reach);
  const int all_hi = first + w0 / s.group + 1;
  const int all_lo = kv4_lowest(first + max(w1, w0) / s.group, reach);

  // f32 activations with a head of 128: the low plane of Q would not fit in
  // the registers of two waves per SIMD and is read from LDS.
  constexpr bool QL_LDS = TWO && WAVES == 8;
  uint8_t* const qlds = lds + 3 * P::BYTES + wave * (NS * 1024) + lane * 16;
  kvh8 qh[NS], ql[TWO && !QL_LDS ? NS : 1], qs;
  float unit;
  {
    const T* q = (const T*)s.a.q + (size_t)(sp.r0 + (valid ? row : 0)) * s.a.q_stride + (size_t)head * D + 8 * hl;
    float top = 0.f;
    bool finite = true;
    if (valid) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        float x[8];
        kv_load8(q + 16 * i, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          top = fmaxf(top, fabsf(x[j]));
          finite = finite && __builtin_isfinite(x[j]);
        }
      }
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int e = 10;
    if (top > 0.f && top <= 3.402823466e38f) e = __builtin_amdgcn_frexp_expf(top);
    unit = finite ? ldexpf(1.f, e - 10) : __builtin_nanf("");
    unit += 0.f * __shfl_xor(unit, 32, 64);
    // unit stays positive (the largest score is the largest product): a
    // negative scale turns the query round.
    unit *= fabsf(s.a.scale) * PF_LOG2E;
    const float turn = s.a.scale < 0.f ? -1.f : 1.f;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) qs[j] = (_Float16)0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      kvh8 low;
      if (valid) kv_load8(q + 16 * i, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = ldexpf(finite ? x[j] : 0.f, 10 - e) * turn;
        qh[i][j] = (_Float16)c;
        if constexpr (TWO) low[j] = (_Float16)(c - (float)qh[i][j]);
        sum += c;
      }
      if constexpr (QL_LDS) *reinterpret_cast<kvh8*>(qlds + i * 1024) = low;
      else if constexpr (TWO) ql[i] = low;
      if (i & 1) {
        sum += __shfl_xor(sum, 32, 64);
        const _Float16 h = (_Float16)sum;
        qs[i >> 1] = hl == 0 ? h : (_Float16)(sum - (float)h);
        sum = 0.f;
      }
    }
  }

  kvf16 o[NG], om;
#pragma unroll
  for (int i = 0; i < 16; ++i) om[i] = 0.f;
#pragma unroll
  for (int i = 0; i < NG; ++i) o[i] = om;
  // A row past the table sees its own slot there: NaN.
  float ref = -3.402823466e38f;
  const bool past = chi > max_slots;

  // Rows of the value minima that no group has: zeros, and ones in row 8.
  for (int i = threadIdx.x; i < 3 * 64; i += THREADS) {
    const int r = i & 15, u = (i >> 4) & 3, buf = i >> 6;
    const uint32_t v = r == 8 ? 0x3C003C00u : 0u;
    if (r >= NG) {
      uint8_t* to = lds + buf * P::BYTES + P::VM + (u * 16 + r) * 16;
      *reinterpret_cast<kvu4*>(to) = kvu4{v, v, v, v};
      if constexpr (TWO) *reinterpret_cast<kvu4*>(to + 1024) = kvu4{0, 0, 0, 0};
    }
  }
  // Stages [s0, s1), an even number (one past the end is all masked).  While
  // stage s is multiplied by its weights, the scores of s + 1 are formed and
  // stage s + 2 is unpacked into the buffer of s - 1.
  const int s0 = any_lo / 32, s1 = any_hi > any_lo ? s0 + (((any_hi - 1) / 32 + 2 - s0) & ~1) : s0;
  constexpr int TURNS = WAVES / 4;  // groups of four waves that take turns
  StageLoad<D, TWO> raw;
  const int turn = wave >> 2, tid = threadIdx.x & 127;
  const bool values = wave & 2;
  raw.place(values, tid);
  auto store = [&](int st) {
    raw.store(lds + (st % 3) * P::BYTES, any_lo - 32 * st, any_hi - 32 * st, values, tid);
  };
  PageIds ids;
  ids.fill(s.c, b, s0 >> 1, lane);
  auto fetch = [&](int st) {
    raw.load(st < s1 ? ids.block(s.c, b, st >> 1, hk, Kv4L<D>::BYTES, lane) : nullptr, s.c.pages, st & 1);
  };
  auto scores = [&](int st) {
    const uint8_t* pg = lds + (st % 3) * P::BYTES;
    kvf16 c;
#pragma unroll
    for (int i = 0; i < 16; ++i) c[i] = 0.f;
    c = kv_mfma32(*reinterpret_cast<const kvh8*>(pg + P::KM + col * 16), qs, c);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const kvh8 k = *reinterpret_cast<const kvh8*>(pg + P::K + i * 1024 + lane * 16);
      if constexpr (QL_LDS) c = kv_mfma32(k, *reinterpret_cast<const kvh8*>(qlds + i * 1024), c);
      else if constexpr (TWO) c = kv_mfma32(k, ql[i], c);
      c = kv_mfma32(k, qh[i], c);
    }
    return c;
  };
  float u = unit;  // what c is to be multiplied by
  // Masks the scores of a stage that not every column sees whole, and moves
  // ref where a score passes it.
  auto settle = [&](kvf16& c, int st) {
    const int at = 32 * st;
    u = unit;
    if (at + 32 > all_hi || at < all_lo) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int slot = at + 8 * (i >> 2) + 4 * hl + (i & 3);
        c[i] = slot >= clo && slot < chi ? c[i] * unit : -INFINITY;
      }
      u = 1.f;
    }
    float top = c[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, c[i]);
    top *= u;
    if (__ballot(top > kv4_limit(ref))) {
      // (Large scores are rounded before ref is taken off.)
#pragma unroll
      for (int i = 0; i < 16; ++i) c[i] *= u;
      u = 1.f;
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float next = fmaxf(ref, top - 7.f), f = __builtin_amdgcn_exp2f(ref - next);
      ref = next;
#pragma unroll
      for (int i = 0; i < NG; ++i) o[i] *= f;
      om *= f;
    }
  };
  // One stage: its weights from the scores c, the next one's scores into c2.
  auto step = [&](int st, const kvf16& c, kvf16& c2) {
    const uint8_t* pg = lds + (st % 3) * P::BYTES;
    c2 = scores(min(st + 1, s1 - 1));
    kvh8 ph[2], pl[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(c[8 * e + j], u, -ref));
        ph[e][j] = (_Float16)x[j];
        pl[e][j] = (_Float16)(x[j] - (float)ph[e][j]);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const kvh8 vm = *reinterpret_cast<const kvh8*>(pg + P::VM + e * 512 + (hl * 16 + (col & 15)) * 16);
      if constexpr (TWO) {
        const kvh8 vl = *reinterpret_cast<const kvh8*>(pg + P::VL + e * 512 + (hl * 16 + (col & 15)) * 16);
        om = kv_mfma32(vl, pl[e], om);
        om = kv_mfma32(vl, ph[e], om);
      }
      om = kv_mfma32(vm, pl[e], om);
      om = kv_mfma32(vm, ph[e], om);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const kvh8 v = *reinterpret_cast<const kvh8*>(pg + P::V + g * 2048 + e * 1024 + lane * 16);
        o[g] = kv_mfma32(v, pl[e], o[g]);
        o[g] = kv_mfma32(v, ph[e], o[g]);
      }
    }
    __syncthreads();
    settle(c2, min(st + 1, s1 - 1));
  };
  kvf16 ca, cb;
  if (s0 < s1) {
    if constexpr (TURNS == 1) {
      fetch(s0);
      store(s0);
      fetch(s0 + 1);
      store(s0 + 1);
      fetch(s0 + 2);
    } else {
      fetch(s0 + turn);
      store(s0 + turn);
      fetch(s0 + 2 + turn);
    }
  }
  __syncthreads();
  if (s0 < s1) {
    ca = scores(s0);
    settle(ca, s0);
  }
  for (int st = s0; st < s1; st += 2) {
    // The loads of both groups stand where each finds its registers free: the
    // first group's have this stage to arrive, the second's two.
    if (TURNS == 1 || turn == 0) store(st + 2);
    if constexpr (TURNS == 1) fetch(st + 3);
    step(st, ca, cb);
    if (TURNS == 1 || turn == 1) store(st + 3);
    fetch(TURNS == 1 ? st + 4 : st + 4 + turn);
    step(st + 1, cb, ca);
  }

  // l is row 8 of om (lane half 0, register 4), group g's minima row g.
  float l = __shfl(om[4], col, 64);
  if (past) l = __builtin_nanf("");
  const float inv = l != 0.f ? 1.f / l : 0.f;
  T* out = (T*)s.a.out + (size_t)(sp.r0 + row) * s.a.out_stride + (size_t)head * D + 4 * hl;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float m = __shfl(om[g & 3], ((g >> 2) & 1) * 32 + col, 64);
    if (!valid) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      struct { T v[4]; } r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r.v[j] = (T)((o[g][4 * i + j] + m) * inv);
      __builtin_memcpy(out + 32 * g + 8 * i, &r, sizeof(r));
    }
  }
  if (valid && s.a.lse && hl == 0)
    s.a.lse[(size_t)(sp.r0 + row) * s.a.n_heads + head] = l != 0.f ? (ref + __builtin_amdgcn_logf(l)) * PF_LN2 : -INFINITY;
  // Rows past max_rows have no workgroup: NaN, by the first tile's.
  if (n > nr && tile == 0) {
    const int w = s.group * D;
    for (int r = sp.r0 + nr; r < sp.r1; ++r) {
      for (int i = threadIdx.x; i < w; i += THREADS)
        ((T*)s.a.out)[(size_t)r * s.a.out_stride + (size_t)hk * w + i] = (T)__builtin_nanf("");
      if (s.a.lse && (int)threadIdx.x < s.group)
        for (int i = threadIdx.x; i < s.group; i += THREADS)
          s.a.lse[(size_t)r * s.a.n_heads + hk * s.group + i] = __builtin_nanf("");
    }
  }
}

template <int D, class T, int WAVES>
static hipError_t prefill_go(const PrefillArgs& s, hipStream_t st) {
  constexpr int lds = 3 * StageLds<D, sizeof(T) == 4>::BYTES + (sizeof(T) == 4 && WAVES == 8 ? WAVES * D * 64 : 0);
  const hipError_t e = hipFuncSetAttribute((const void*)&kv4_prefill<D, T, WAVES>,
                                           hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  const long long tiles = ((long long)std::min(s.a.max_rows, s.rows.n_rows) * s.group + 32 * WAVES - 1) / (32 * WAVES);
  // Tiles and kv heads share x.  (Its limit is 2^32 threads, 300 GB of queries.)
  if (tiles * s.c.n_kv >= (1ll << 32) / (64 * WAVES)) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)(tiles * s.c.n_kv), 1, s.rows.n_seq);
  hipLaunchKernelGGL((kv4_prefill<D, T, WAVES>), grid, dim3(64 * WAVES), lds, st, s);
  return hipGetLastError();
}

template <class T>
static hipError_t prefill_typed(int head_dim, const PrefillArgs& s, hipStream_t st) {
  if (head_dim == 64) return prefill_go<64, T, 8>(s, st);
  if (head_dim == 128) return prefill_go<128, T, 8>(s, st);
  return prefill_go<256, T, 4>(s, st);
}

// The host knows rows, not lengths.  A workgroup here walks all slots of 256
// columns; the split kernel (kv4_attn.hip) cuts the slots, and reads them once
// per 16 columns.  So this one is for sequences of many columns, and for
// enough of them in all that most compute units have some:
//   columns of a (sequence, kv head), card full (64 sequences of 3000 slots,
//   32/8 heads, bf16): 48 here 287 us, split 207; 64: 285 and 227; 80: 300 and
//   305; 96: 299 and 383 (f32 80: 386 and 317; 96: 383 and 400; heads of 256,
//   80: 253 and 319; of 64, 80: 226 and 208);
//   rows x heads in all (six sequences, 20000 slots, bf16): 12288 here 819 us,
//   split 447; 18432: 816 and 805; 24576: 820 and 822; 30720: 823 and 1610
//   (f32 24576: 1130 and 869; 30720: 1127 and 1673; heads of 64, 24576: 691
//   and 563; of 256, 24576: 1469 and 1701).
// All of it for sequences alike.  A sequence of a few rows beside a long one
// goes where that one does: its slots are not cut here, and there fewer
// workgroups share the axis (64/8 heads, bf16: 63 lanes of up to 8000 slots 94
// us and 200 rows 39, together 2630; a lane of 130001 slots 42 and 2000 rows
// 146, together 5120).
// What the split kernel's launch has no room for comes here in any case.
bool kv4_prefill_takes(const Kv4View& c, const Kv4Rows& rows, const Kv4Attn& a) {
  const long long cols = (long long)std::min(a.max_rows, rows.n_rows) * (a.n_heads / c.n_kv);
  return (cols + 15) / 16 * c.n_kv > 65535 || (cols >= 80 && (long long)rows.n_rows * a.n_heads >= 20480);
}

hipError_t launch_kv4_prefill(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Attn& a,
                              hipStream_t st) {
  const PrefillArgs s{c, rows, a, a.n_heads / c.n_kv};
  if (type == ACT_F32) return prefill_typed<float>(head_dim, s, st);
  if (type == ACT_F16) return prefill_typed<_Float16>(head_dim, s, st);
  return prefill_typed<bf16_t>(head_dim, s, st);
}

}  // namespace kq
