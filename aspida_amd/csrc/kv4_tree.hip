// kv4_tree.hip -- attention of trees of drafted tokens over the 4-bit cache.
//
// A row at tree place i sees every slot before the tree and the rows that its
// mask names (TreeSeen, kv4_split.h).  Trees of many columns (rows times query
// heads of a kv head) behind many slots come here (tree_takes); the others take
// kv4_attn_split.
//
// A workgroup takes 32 columns per wave, 128 or 256 in all, and a share of the
// axis of all sequences' slots (kv4_split.h).  It walks the share in stages of
// 32 tokens, turned into f16 operands in LDS once for all waves, two stages
// ahead (kv4_stage.h); per stage S = K Q^T, P = exp2(S - ref) in two f16
// planes, O += V^T P, as in kv4_prefill.hip.  So a slot is unpacked once for
// all rows of its tree, where tiles of 16 columns unpack it for each, and few
// trees behind long caches still fill the card.  Masks are looked up in stages
// that reach into the tree or out of the window alone.  A second launch joins
// the parts of a sequence.
//
// Bound by waiting at the barrier of every stage and for its data (45% of wave
// time; vector units 50% busy, matrix cores 43%): 256 columns behind 32000
// slots (32/8 heads of 128, bf16) take 83 us, 404 TFLOP/s of the products that
// the formula has; the two planes of P and the minima make 1.6 times as many.
// In tiles of 16 columns, which unpack every slot 16 times: 124 us; in tiles of
// 32 and 64 columns unpacked straight into registers: 157 us (two waves a SIMD,
// registers spilled) and 102 (one wave).
#include <algorithm>

#include "kv4_split.h"
#include "kv4_stage.h"

namespace kq {

// Value steps and minima that a token in the cache cannot have become 0: rows
// of a tree that no mask names may never have been written, and their weight
// of 0 must meet finite values.
__device__ __forceinline__ uint32_t kv4_sane(uint32_t pair, uint32_t top) {
  const uint32_t lo = pair & 0x7FFFu, hi = pair >> 16 & 0x7FFFu;
  return pair & ((lo <= top ? 0x0000FFFFu : 0u) | (hi <= top ? 0xFFFF0000u : 0u));
}

template <int D, class T, int WAVES>
__global__ __launch_bounds__(64 * WAVES, D == 256 ? 1 : 2) void kv4_tree(SplitArgs s) {
  constexpr bool TWO = sizeof(T) == 4;
  using P = StageLds<D, TWO>;
  constexpr int NG = D / 32, NS = D / 16, THREADS = 64 * WAVES, COLS = 32 * WAVES;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];  // three stages, and the low plane of Q
  const int lane = threadIdx.x & 63, col = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.y / s.tiles, tile = blockIdx.y % s.tiles;
  const int max_slots = s.c.max_pages * KV4_PAGE;
  Kv4Span own = {0, 0, 0};
  if (lane < s.rows.n_seq) own = kv4_span(s.rows, lane);
  AxisPlace place = axis_place<true>(s.rows, own, s.a.window, max_slots, s.groups, blockIdx.x);
  const long long x1 = place.x0 + place.share;

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
  constexpr bool QL_LDS = TWO && WAVES == 8;  // the low plane of Q would not fit in the registers
  uint8_t* const qlds = lds + 3 * P::BYTES + wave * (NS * 1024) + lane * 16;
  constexpr int TURNS = WAVES / 4;  // groups of four waves that take turns
  StageLoad<D, TWO> raw;
  const int turn = wave >> 2, tid = threadIdx.x & 127;
  const bool values = wave & 2;
  raw.place(values, tid);

  for (int b = place.seq; b < s.rows.n_seq && place.start < x1; ++b) {
    const Kv4Span sp = kv4_span(s.rows, b);
    const SeenRange seen = seen_range<true>(sp, s.a.window, max_slots);
    const int length = rounds_of<true>(sp, s.a.window, max_slots);
    const long long at0 = place.start + AXIS_EXTRA;
    place.start = at0 + length;
    const int u0 = (int)max(0ll, place.x0 - at0), u1 = (int)min((long long)length, x1 - at0);
    if (u0 >= u1) continue;
    const bool whole = u0 == 0 && u1 == length;
    const int n = sp.r1 - sp.r0, nr = min(n, s.a.max_rows), base = sp.len - n;
    if (n > s.a.max_rows && u0 == 0 && tile == 0) fill_excess<T>(s, sp, hk, D);
    const int c0 = tile * COLS, c1 = min(c0 + COLS, nr * s.group);
    if (c1 <= c0) continue;
    // The share's slots [t0, t1), and this lane's column.
    const int t0 = seen.lo + u0 * ATTN_STEP, t1 = (int)min((long long)seen.hi, seen.lo + (long long)u1 * ATTN_STEP);
    const int w0 = c0 + 32 * wave;
    const bool works = w0 < c1;
    // A lane's column, formed anew (opaquely) where it is needed: kept over the
    // loop, it and what follows from it cost registers that stages need.
    struct Column { int ci, row; bool valid; };
    auto column = [&] {
      int l = lane;
      asm volatile("" : "+v"(l));
      Column x;
      x.ci = w0 + (l & 31);
      x.row = x.ci / s.group;
      x.valid = x.ci < c1;
      if (!x.valid) x.row = 0;
      return x;
    };
    int low;  // of its TreeSeen
    {
      const Column x = column();
      low = TreeSeen(s.a, sp.r0, x.row, n, base, x.valid).lo;
    }
    int all_lo = w0 + col < c1 ? low : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) all_lo = max(all_lo, __shfl_xor(all_lo, o, 64));
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);

    kvh8 qh[NS], ql[TWO && !QL_LDS ? NS : 1], qs;
    float unit = 0.f;
    {
      const Column x0 = column();
      const bool valid = x0.valid;
      const int head = hk * s.group + (valid ? x0.ci % s.group : 0);
      const T* q = (const T*)s.a.q + (size_t)(sp.r0 + x0.row) * s.a.q_stride + (size_t)head * D + 8 * hl;
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
      unit *= fabsf(s.a.scale) * LOG2E;
      const float turned = s.a.scale < 0.f ? -1.f : 1.f;
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
          const float c = ldexpf(finite ? x[j] : 0.f, 10 - e) * turned;
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
    float ref = REF0;

    // Stages [s0, s1), an even number (one past the end is all masked).  While
    // stage s is multiplied by its weights, the scores of s + 1 are formed and
    // stage s + 2 is unpacked into the buffer of s - 1.
    const int s0 = t0 / 32, s1 = t1 > t0 ? s0 + (((t1 - 1) / 32 + 2 - s0) & ~1) : s0;
    PageIds ids;
    ids.fill(s.c, b, s0 >> 1, lane);
    auto fetch = [&](int st) {
      raw.load(st < s1 ? ids.block(s.c, b, st >> 1, hk, Kv4L<D>::BYTES, lane) : nullptr, s.c.pages, st & 1);
    };
    auto store = [&](int st) {
      if (values && 32 * st + 32 > base) {
#pragma unroll
        for (int i = 0; i < StageLoad<D, TWO>::N; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            raw.d[i][k] = kv4_sane(raw.d[i][k], 0x5BF0u);  // 254
            raw.d2[i][k] = kv4_sane(raw.d2[i][k], 0x5BF0u);
          }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          raw.m[k] = kv4_sane(raw.m[k], 0x7BFFu);  // finite
          if constexpr (TWO) raw.md[k] = kv4_sane(raw.md[k], 0x5BF0u);
        }
      }
      raw.store(lds + (st % 3) * P::BYTES, t0 - 32 * st, t1 - 32 * st, values, tid);
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
      if (at + 32 > base || at < all_lo || at + 32 > t1) {
        const Column x = column();
        const TreeSeen tree(s.a, sp.r0, x.row, n, base, x.valid, low);
        uint32_t sees = 0;
        if (at + 32 > base) sees = tree.rows(at - base);
        const int lo = tree.lo - at, hi = base - at;
        if (hi > 0 && lo < 32 && lo < hi) sees |= (hi < 32 ? ~(~0u << hi) : ~0u) & (lo > 0 ? ~0u << lo : ~0u);
        if (at + 32 > t1) sees &= t1 > at ? ~0u >> (at + 32 - t1) : 0u;
        sees >>= 4 * hl;
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] = sees & 1u << (8 * (i >> 2) + (i & 3)) ? c[i] * unit : -INFINITY;
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
    // The loads of both groups stand where each finds its registers free: the
    // first group's have this stage to arrive, the second's two.
    auto first_half = [&](int st) {
      if (TURNS == 1 || turn == 0) store(st + 2);
      if constexpr (TURNS == 1) fetch(st + 3);
    };
    auto second_half = [&](int st) {
      if (TURNS == 1 || turn == 1) store(st + 3);
      fetch(TURNS == 1 ? st + 4 : st + 4 + turn);
    };
    if (works) {
      kvf16 ca, cb;
      if (s0 < s1) {
        ca = scores(s0);
        settle(ca, s0);
      }
      for (int st = s0; st < s1; st += 2) {
        first_half(st);
        step(st, ca, cb);
        second_half(st);
        step(st + 1, cb, ca);
      }
    } else {  // a wave without columns has its part in unpacking alone
      for (int st = s0; st < s1; st += 2) {
        first_half(st);
        __syncthreads();
        second_half(st);
        __syncthreads();
      }
    }
    // (The stores past s1 reached buffers that the next sequence's first stages
    // take: not before every wave is here.)
    __syncthreads();

    // l is row 8 of om (lane half 0, register 4), group g's minima row g.
    float l = __shfl(om[4], col, 64);
    const Column x = column();
    const bool valid = x.valid;
    const int row = x.row, head = hk * s.group + x.ci % s.group;
    if (u0 == 0 && TreeSeen(s.a, sp.r0, row, n, base, valid, low).past(base, max_slots)) l = __builtin_nanf("");
    const float inv = whole ? (l != 0.f ? 1.f / l : 0.f) : 1.f;
    T* out = (T*)s.a.out + (size_t)(sp.r0 + row) * s.a.out_stride + (size_t)head * D + 4 * hl;
    AttnPart<D, COLS>* part =
        (AttnPart<D, COLS>*)s.a.work + (2 * (size_t)blockIdx.x + (u0 == 0)) * gridDim.y + blockIdx.y;
    float* sums = &part->o[32 * wave + col][4 * hl];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float m = __shfl(om[g & 3], ((g >> 2) & 1) * 32 + col, 64);
      if (!valid) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y[4] = {(o[g][4 * i] + m) * inv, (o[g][4 * i + 1] + m) * inv, (o[g][4 * i + 2] + m) * inv,
                            (o[g][4 * i + 3] + m) * inv};
        if (whole) store4(out + 32 * g + 8 * i, y);
        else *reinterpret_cast<kvf4*>(sums + 32 * g + 8 * i) = kvf4{y[0], y[1], y[2], y[3]};
      }
    }
    if (valid && hl == 0) {
      if (!whole) {
        part->ref[32 * wave + col] = ref;
        part->l[32 * wave + col] = l;
      } else if (s.a.lse) {
        s.a.lse[(size_t)(sp.r0 + row) * s.a.n_heads + head] = l != 0.f ? (ref + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
      }
    }
  }
}

// Joins the parts of a sequence, as kv4_attn_join does, but with a wave a
// column: trees have hundreds of columns and few parts, and what a workgroup
// spends on finding its parts is most of a join's time (16 trees of up to 104
// columns and 8 kv heads: 19 us with a workgroup a column, 10 here).
template <int D, class T, int COLS>
__global__ __launch_bounds__(256) void kv4_tree_join(SplitArgs s) {
  constexpr int E = D / 64;
  struct Dims { float v[E]; };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.z, hk = blockIdx.y / s.tiles, tile = blockIdx.y % s.tiles, col = 4 * blockIdx.x + wave;
  const Kv4Span sp = kv4_span(s.rows, b);
  const int ncol = min(COLS, min(sp.r1 - sp.r0, s.a.max_rows) * s.group - tile * COLS);
  if (col >= ncol) return;
  const int max_slots = s.c.max_pages * KV4_PAGE, length = rounds_of<true>(sp, s.a.window, max_slots);
  int first, count;  // of the workgroups that share it
  if (s.rows.n_seq <= 64) {  // (sums below 2^30)
    int n = 0;
    if (lane < s.rows.n_seq) n = rounds_of<true>(kv4_span(s.rows, lane), s.a.window, max_slots) + AXIS_EXTRA;
    const int upto = wave_scan_add(n);
    const uint32_t share = ((uint32_t)__builtin_amdgcn_readlane(upto, 63) + s.groups - 1) / (uint32_t)s.groups;
    const uint32_t start = __builtin_amdgcn_readlane(upto, b) - length;
    first = (int)(start / share);
    count = (int)((start + length - 1) / share) - first + 1;
  } else {
    Kv4Span own = {0, 0, 0};
    if (lane < s.rows.n_seq) own = kv4_span(s.rows, lane);
    const long long share = (axis_total<true>(s.rows, own, s.a.window, max_slots) + s.groups - 1) / s.groups;
    long long start = 0;
    for (int i = lane; i < b; i += 64) start += rounds_of<true>(kv4_span(s.rows, i), s.a.window, max_slots) + AXIS_EXTRA;
#pragma unroll
    for (int o = 32; o; o >>= 1) start += __shfl_xor(start, o, 64);
    start += AXIS_EXTRA;
    first = (int)(start / share);
    count = (int)((start + length - 1) / share) - first + 1;
  }
  if (count == 1) return;
  // Its parts: number 2 first + 1, then 2 x of the workgroups behind.
  const size_t step = gridDim.y;
  const AttnPart<D, COLS>* parts = (const AttnPart<D, COLS>*)s.a.work + 2 * (size_t)first * step + blockIdx.y;
  auto part = [&](int i) -> const AttnPart<D, COLS>& { return parts[(i ? 2 * (size_t)i : 1) * step]; };
  float ref = REF0;
  for (int i = lane; i < count; i += 64) ref = fmaxf(ref, part(i).ref[col]);
#pragma unroll
  for (int o = 32; o; o >>= 1) ref = fmaxf(ref, __shfl_xor(ref, o, 64));
  float l = 0.f, y[E] = {};
  for (int c0 = 0; c0 < count; c0 += 64) {
    const int here = min(count - c0, 64);
    const AttnPart<D, COLS>& own = part(c0 + min(lane, here - 1));
    const float f = lane < here ? __builtin_amdgcn_exp2f(own.ref[col] - ref) : 0.f;
    if (lane < here) l += own.l[col] * f;
    for (int i = 0; i < here; i += 8) {  // (past the last part it is the last one again, with a weight of 0)
      Dims o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        o[j] = *reinterpret_cast<const Dims*>(&part(c0 + min(i + j, here - 1)).o[col][lane * E]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float fj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i + j));
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = __builtin_fmaf(o[j].v[e], fj, y[e]);
      }
    }
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o, 64);
  const int ci = tile * COLS + col, row = sp.r0 + ci / s.group, head = hk * s.group + ci % s.group;
  T* out = (T*)s.a.out + (size_t)row * s.a.out_stride + (size_t)head * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = (T)(l != 0.f ? y[e] / l : 0.f);
  if (s.a.lse && lane == 0)
    s.a.lse[(size_t)row * s.a.n_heads + head] = l != 0.f ? (ref + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
}

// Workgroups that fit at once: one of eight waves a compute unit, two of four
// (one for heads of 256, whose stages take 103 KB).
template <int D, int WAVES> constexpr int TREE_ROOM = WAVES == 4 && D != 256 ? 512 : 256;

template <int D, int WAVES>
static size_t tree_work() { return 2 * (size_t)TREE_ROOM<D, WAVES> * sizeof(AttnPart<D, 32 * WAVES>); }

template <int D, class T, int WAVES>
static hipError_t tree_go(SplitArgs s, hipStream_t st) {
  constexpr int lds = 3 * StageLds<D, sizeof(T) == 4>::BYTES + (sizeof(T) == 4 && WAVES == 8 ? WAVES * D * 64 : 0);
  const hipError_t e = hipFuncSetAttribute((const void*)&kv4_tree<D, T, WAVES>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  const long long cols = (long long)s.a.max_rows * s.group;
  s.tiles = (int)((cols + 32 * WAVES - 1) / (32 * WAVES));
  const int per_seq = s.c.n_kv * s.tiles;
  s.groups = std::max(1, TREE_ROOM<D, WAVES> / per_seq);
  hipLaunchKernelGGL((kv4_tree<D, T, WAVES>), dim3(s.groups, per_seq), dim3(64 * WAVES), lds, st, s);
  if (s.groups > 1)
    hipLaunchKernelGGL((kv4_tree_join<D, T, 32 * WAVES>), dim3((unsigned)(std::min<long long>(32 * WAVES, cols) + 3) / 4, per_seq, s.rows.n_seq), dim3(256), 0, st, s);
  return hipGetLastError();
}

// Eight waves above 128 columns, and for f32 (its two planes of Q leave four
// waves one to a SIMD); heads of 256 have room for four alone.  16 trees
// behind 4000 slots each, 32/8 heads of 128, bf16, four and eight: 96 columns
// 102 and 118 us, 128 columns 117 and 127, 192 columns 180 and 164, 400
// columns 299 and 275.
template <class T>
static hipError_t tree_typed(int head_dim, const SplitArgs& s, hipStream_t st) {
  if (head_dim == 256) return tree_go<256, T, 4>(s, st);
  if constexpr (sizeof(T) == 2) {
    if ((long long)s.a.max_rows * s.group <= 128) return head_dim == 64 ? tree_go<64, T, 4>(s, st) : tree_go<128, T, 4>(s, st);
  }
  return head_dim == 64 ? tree_go<64, T, 8>(s, st) : tree_go<128, T, 8>(s, st);
}

// Whether trees of so many columns behind so many slots (the page table's
// bound) come here.  kv4_attn_split and this kernel, 16 trees behind 4000
// slots each, us: heads of 128, bf16, 64 columns 73 and 90, 96 columns 129 and
// 102, 256 columns 274 and 190; f32 128 columns 146 and 145, 192 columns 258
// and 187; heads of 256, bf16, 64 columns 74 and 111, 128 columns 141 and 124;
// heads of 64, bf16, 96 columns 71 and 81, 128 columns 102 and 91.  Behind few
// slots its start costs more than its stages save: one tree behind 2000 slots
// takes 21 and 32 us with 128 columns, 36 and 42 with 400; both take the same
// where columns times slots are 1.5 to 3 million.
static bool tree_takes(int head_dim, int type, long long cols, long long slots) {
  const int least = type == ACT_F32 ? 128 : head_dim == 128 ? 64 : 96;
  return cols > least && slots > (1 << 21) / cols;
}

size_t kv4_tree_work_bytes(int head_dim, int rows, int group) {
  const size_t few = kv4_attn_work_bytes(head_dim);
  if (!tree_takes(head_dim, ACT_BF16, (long long)rows * group, 1ll << 40)) return few;
  return std::max(few, head_dim == 64    ? std::max(tree_work<64, 8>(), tree_work<64, 4>())
                       : head_dim == 128 ? std::max(tree_work<128, 8>(), tree_work<128, 4>())
                                         : tree_work<256, 4>());
}

hipError_t launch_kv4_tree(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Attn& a,
                           hipStream_t st) {
  const int group = a.n_heads / c.n_kv;
  const long long slots = (long long)rows.n_seq * c.max_pages * KV4_PAGE;
  if (!tree_takes(head_dim, type, (long long)a.max_rows * group, slots))
    return launch_kv4_attn(head_dim, c, type, rows, a, st);
  const SplitArgs s{c, rows, a, group, 0, 0};
  if (type == ACT_F32) return tree_typed<float>(head_dim, s, st);
  if (type == ACT_F16) return tree_typed<_Float16>(head_dim, s, st);
  return tree_typed<bf16_t>(head_dim, s, st);
}

}  // namespace kq
