// kv4_attn.hip -- attention over the paged 4-bit cache.
//
// Row i of a sequence's n new rows sits at slot p = kv_len - n + i and sees
// the slots j <= p (and j > p - window):
//   o = sum_j softmax_j(scale q . k_j) v_j,   lse = log sum_j exp(scale q . k_j).
// A row that sees nothing gets o = 0 and lse = -inf.
//
// kv4_attn_split: the rows of a sequence times the query heads of a kv head
// are columns, 16 to a tile.  A wave takes 32 tokens at a time:
//   S[token][col] = K Q^T   16x16x32, K's codes as exact f16 (kv4_mma.h), one
//                           more step for the minima; two planes of Q for f32
//   P = exp2(S - ref)       ref follows the running maximum per column, moved
//                           only when a score passes it by 15
//   O[dim][col] += V^T P    P in S's own registers: S's lane holds tokens 4 rg
//                           + 0..3 of two tiles for one column, which is how
//                           the value dwords are ordered; one more step for
//                           the minima; P is two f16 numbers for every type
//                           (one leaves 2^-11 of a weight, as much as an f16
//                           result's own rounding)
// so nothing passes through LDS until the waves of a workgroup are joined.
// The sequences' slots stand one after the other on one axis, which is cut
// into equal shares, one for each workgroup that fits on the card at once: a
// workgroup takes what of one sequence or of several lies in its share, and a
// second launch joins the parts of a sequence.  All of it follows from the
// lengths on the device, which the host does not know.
// Bound by the vector units: a wave's round of 32 tokens is about 300 of their
// instructions (unpacking, exp2, the two planes of P) in 1800 cycles, with
// two waves a SIMD, and 45 matrix instructions beside them (64 lanes: vector
// units 73% busy, matrix cores 18%).  130001 slots of 8 kv heads of 128 (f32,
// 166 MB) take 42 us, 4.0 TB/s, of 32 at the rate of a large copy; 64 lanes of
// up to 8000 slots (bf16, 330 MB) 79 us, 4.2 TB/s.
#include <algorithm>

#include "kv4_mma.h"

namespace kq {

constexpr int ATTN_WAVES = 4;
constexpr int ATTN_STEP = 32 * ATTN_WAVES;  // tokens of a workgroup's round
// Tokens whose page ids a wave holds at once: whole rounds, within 64 pages
// wherever in a page they start.
constexpr int ATTN_SEGMENT = (4096 - 32) / ATTN_STEP * ATTN_STEP;
// Workgroups that fit at once: 256 CUs times what their registers allow (under
// 168, 256 and 512 for heads of 64, 128 and 256).  One round of equal shares
// measured against 1.5 and 2 rounds (32/8 heads, f32): 130001 slots 47, 59
// and 57 us; 16 lanes of 8000 45, 56 and 54 us.
template <int D> constexpr int ATTN_GROUPS = D == 64 ? 768 : D == 128 ? 512 : 256;
constexpr float REF0 = -3.402823466e38f;  // below every score
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// Slots that a sequence's rows see together: [lo, hi), lo a multiple of 32.
struct SeenRange { int lo, hi; };
__device__ __forceinline__ SeenRange seen_range(const Kv4Span& s, int window, int max_slots) {
  const int first = s.len - (s.r1 - s.r0);  // the first row's slot
  SeenRange r;
  r.hi = s.r1 > s.r0 ? min(s.len, max_slots) : 0;
  r.lo = min(kv4_lowest(first, kv4_reach(window)), r.hi) & ~31;
  return r;
}

// A sequence's rounds (one at least: one whose rows see nothing has outputs
// too), and its length on the axis, which counts what a workgroup spends on a
// sequence besides: its rows, page ids and sums, about 8000 cycles where a
// round takes 1800.
constexpr int AXIS_EXTRA = 4;
__device__ __forceinline__ int rounds_of(const Kv4Span& s, int window, int max_slots) {
  const SeenRange r = seen_range(s, window, max_slots);
  return max(1, (r.hi - r.lo + ATTN_STEP - 1) / ATTN_STEP);
}

// Where workgroup x's share starts: [x0, x0 + share) of the axis, sequence seq
// (n_seq: none) from `start` of it on.
struct AxisPlace { long long x0, share, start; int seq; };

// Inclusive sum over the lanes.
__device__ __forceinline__ long long wave_scan64(long long v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

// own: the span of sequence `lane`, which the first 64 sequences' lengths come
// from.
__device__ __forceinline__ long long axis_total(const Kv4Rows& rows, const Kv4Span& own, int window, int max_slots) {
  const int lane = threadIdx.x & 63;
  long long total = lane < rows.n_seq ? rounds_of(own, window, max_slots) + AXIS_EXTRA : 0;
  for (int b = 64 + lane; b < rows.n_seq; b += 64) total += rounds_of(kv4_span(rows, b), window, max_slots) + AXIS_EXTRA;
#pragma unroll
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o, 64);
  return total;
}

__device__ __forceinline__ AxisPlace axis_place(const Kv4Rows& rows, const Kv4Span& own, int window, int max_slots,
                                                int groups, int x) {
  const int lane = threadIdx.x & 63;
  AxisPlace p;
  if (rows.n_seq <= 64) {  // one lane each, and sums below 2^30
    const int n = lane < rows.n_seq ? rounds_of(own, window, max_slots) + AXIS_EXTRA : 0;
    const int end = wave_scan_add(n);
    p.share = (__builtin_amdgcn_readlane(end, 63) + groups - 1) / groups;
    p.x0 = x * p.share;
    const uint64_t over = __ballot(end > p.x0);
    const int l = over ? __builtin_ctzll(over) : 63;
    p.seq = over ? l : rows.n_seq;
    p.start = __builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(n, l);
    return p;
  }
  p.share = (axis_total(rows, own, window, max_slots) + groups - 1) / groups;
  p.x0 = x * p.share;
  long long before = 0;
  for (int b0 = 0; b0 < rows.n_seq; b0 += 64) {
    const int b = b0 + lane;
    const int n = b < rows.n_seq ? rounds_of(b0 ? kv4_span(rows, b) : own, window, max_slots) + AXIS_EXTRA : 0;
    const long long end = before + wave_scan64(n);
    const uint64_t over = __ballot(end > p.x0);
    if (over) {
      const int l = __builtin_ctzll(over);
      p.seq = b0 + l;
      p.start = __shfl(end, l, 64) - __shfl(n, l, 64);
      return p;
    }
    before = __shfl(end, 63, 64);
  }
  p.seq = rows.n_seq;
  p.start = before;
  return p;
}

// Workspace: per part, kv head and column tile the columns' sums [16][D] and
// (ref, l) [16].  A workgroup has at most two sequences in part: one that
// began in a share before its own (number 2 x) and one that goes on in the
// next (2 x + 1), so parts number as the workgroups do, not as the sequences.
template <int D> struct AttnPart {
  float o[16][D];
  float ref[16], l[16];
};

struct SplitArgs {
  Kv4View c;
  Kv4Rows rows;
  Kv4Attn a;
  int group, tiles;  // query heads of a kv head, column tiles
  int groups;        // workgroups that share the axis
};

template <class T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4]) {
  struct { T v[4]; } r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = (T)x[i];
  __builtin_memcpy(p, &r, sizeof(r));
}

// Rows past max_rows have no workgroup: NaN, by all threads of one.
template <class T>
__device__ void fill_excess(const SplitArgs& s, const Kv4Span& sp, int hk, int d) {
  const int w = s.group * d;
  for (int row = sp.r0 + s.a.max_rows; row < sp.r1; ++row) {
    T* out = (T*)s.a.out + (size_t)row * s.a.out_stride + (size_t)hk * w;
    for (int i = threadIdx.x; i < w; i += blockDim.x) out[i] = (T)__builtin_nanf("");
    if (s.a.lse)
      for (int i = threadIdx.x; i < s.group; i += blockDim.x)
        s.a.lse[(size_t)row * s.a.n_heads + hk * s.group + i] = __builtin_nanf("");
  }
}

template <int D, class T>
__global__ __launch_bounds__(64 * ATTN_WAVES, D == 64 ? 3 : D == 128 ? 2 : 1) void kv4_attn_split(SplitArgs s) {
  using L = Kv4L<D>;
  constexpr bool TWO = sizeof(T) == 4;
  constexpr int NG = D / 32, NT = D / 16;
  __shared__ float so[2][16][D];
  __shared__ float sr[2][16], sl[2][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.y / s.tiles, tile = blockIdx.y % s.tiles;
  const int max_slots = s.c.max_pages * KV4_PAGE;
  // The first 64 sequences' spans, a lane each.
  const int mine = threadIdx.x & 63;
  Kv4Span own = {0, 0, 0};
  if (mine < s.rows.n_seq) own = kv4_span(s.rows, mine);
  AxisPlace place = axis_place(s.rows, own, s.a.window, max_slots, s.groups, blockIdx.x);
  const long long x1 = place.x0 + place.share;
  for (int b = place.seq; b < s.rows.n_seq && place.start < x1; ++b) {
    // (Opaque, so that what follows from it is not kept in registers from one
    // sequence to the next: 251 of them against 198.)
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int col = lane & 15, rg = lane >> 4;
    Kv4Span sp;
    if (b < 64) {
      sp.r0 = __builtin_amdgcn_readlane(own.r0, b);
      sp.r1 = __builtin_amdgcn_readlane(own.r1, b);
      sp.len = __builtin_amdgcn_readlane(own.len, b);
    } else {
      sp = kv4_span(s.rows, b);
    }
    const SeenRange seen = seen_range(sp, s.a.window, max_slots);
    const int length = rounds_of(sp, s.a.window, max_slots);
    // Its rounds [u0, u1) are in this share.
    const long long at = place.start + AXIS_EXTRA;
    place.start = at + length;
    const int u0 = (int)max(0ll, place.x0 - at), u1 = (int)min((long long)length, x1 - at);
    const bool whole = u0 == 0 && u1 == length;
    if (u0 >= u1) continue;
    const int n = sp.r1 - sp.r0;
    if (n > s.a.max_rows && u0 == 0 && tile == 0) fill_excess<T>(s, sp, hk, D);
    const int ncol = min(16, min(n, s.a.max_rows) * s.group - tile * 16);
    if (ncol <= 0) continue;
    // This lane's column: its row, head, and the slots [clo, chi) it sees.
    const int reach = kv4_reach(s.a.window);
    const int ci = tile * 16 + col, row = ci / s.group, head = hk * s.group + ci % s.group;
    const bool valid = col < ncol;
    const int pos = sp.len - n + row;
    const int chi = valid ? max(pos + 1, 0) : 0, clo = kv4_lowest(pos, reach);
    // The share's slots, and those of them that every column sees.
    const int t0 = seen.lo + u0 * ATTN_STEP, t1 = (int)min((long long)seen.hi, seen.lo + (long long)u1 * ATTN_STEP);
    const int row_last = (tile * 16 + ncol - 1) / s.group, row_first = tile * 16 / s.group;
    const int all_hi = sp.len - n + row_first + 1;                                       // below: seen by every column
    const int all_lo = kv4_lowest(sp.len - n + row_last, reach);
    const int any_hi = min(t1, sp.len - n + row_last + 1);
    const int any_lo = kv4_lowest(sp.len - n + row_first, reach);

    kvf4 o[NT], om = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] = om;
    // A row past the table sees its own slot there: NaN.
    float ref = REF0, l = chi > max_slots && u0 == 0 && wave == 0 ? __builtin_nanf("") : 0.f;

    // Two sets of registers: one is multiplied while the other arrives.  The
    // loads are the same every time (past the end they read any page again), so
    // nothing makes the compiler move, and wait for, what is on its way.
    struct Set {
      KeyTile<D> k[2];
      ValueBlock<D> v;
      bool there;
    };
    PageIds ids;
    int end = 0;
    auto load = [&](Set& x, int at) {
      const uint8_t* blk = at < end ? ids.at(s.c, at >> 6, hk, L::BYTES) : nullptr;
      x.there = blk != nullptr;
      if (!blk) blk = s.c.pages;  // any page: what is read there is not used
      const int half = (at >> 5) & 1;
      x.k[0].load(blk, 2 * half, lane);
      x.k[1].load(blk, 2 * half + 1, lane);
      x.v.load(blk, half, lane);
    };
    Query<D, TWO> q;
    float unit;
    auto step = [&](Set& y, int at) {
      kvf4 c[2] = {q.scores(y.k[0]), q.scores(y.k[1])};
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = c[j >> 2][j & 3];
      float u = unit;
      if (!y.there || at + 32 > all_hi || at < all_lo) {
        // Slots that this column does not see get no weight; the steps and
        // minima of slots that no column sees may be anything and become 0.
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int slot = at + 16 * (j >> 2) + 4 * rg + (j & 3);
          const bool see = slot >= clo && slot < chi;
          x[j] = see ? (y.there ? x[j] * unit : __builtin_nanf("")) : -INFINITY;
          if (y.there && slot < any_hi && slot >= any_lo) keep |= 1u << j;
        }
        y.v.drop(keep);
        u = 1.f;
      }
      float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * u;
      if (__ballot(top > kv4_limit(ref))) {
        // P' = exp2(x - ref) is kept below 2^15; after a move the maximum of the
        // column is at 2^7.  Large scores are rounded before ref is taken off.
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= u;
        u = 1.f;
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float next = fmaxf(ref, top - 7.f);
        const float f = __builtin_amdgcn_exp2f(ref - next);
        ref = next;
        l *= f;
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i] *= f;
        om *= f;
      }
      kvh8 ph, pl;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], u, -ref));
        l += p;
        ph[j] = (_Float16)p;
        pl[j] = (_Float16)(p - (float)ph[j]);
      }
      const kvh8 vm = __builtin_bit_cast(kvh8, y.v.m);
      om = kv_mfma(vm, pl, om);
      om = kv_mfma(vm, ph, om);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const kvh2 d0 = kv_h2(y.v.d[g][0]), d1 = kv_h2(y.v.d[g][1]), d2 = kv_h2(y.v.d[g][2]), d3 = kv_h2(y.v.d[g][3]);
        const kvh2 n0 = kv_times(d0, -16.f), n1 = kv_times(d1, -256.f);
        const kvh2 n2 = kv_times(d2, -16.f), n3 = kv_times(d3, -256.f);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * g + e;
          const kvh8 a = kv4_unpack(y.v.w[i >> 2][i & 3], d0, d1, d2, d3, n0, n1, n2, n3);
          o[i] = kv_mfma(a, pl, o[i]);
          o[i] = kv_mfma(a, ph, o[i]);
        }
      }
    };
    // The page ids, and the first tokens' words, are on their way while the
    // rows are read.
    Set xa, xb;
    ids.fill(s.c, b, t0 >> 6, lane);
    end = min(any_hi, t0 + ATTN_SEGMENT);
    load(xa, t0 + 32 * wave);
    q.load((const T*)s.a.q + (size_t)(sp.r0 + (valid ? row : 0)) * s.a.q_stride + (size_t)head * D, valid, lane,
           s.a.scale < 0.f ? -1.f : 1.f);
    // Not negative, so that the largest product is the largest score.
    unit = q.unit * (fabsf(s.a.scale) * LOG2E);
    for (int from = t0; from < any_hi; from += ATTN_SEGMENT) {
      int t = from + 32 * wave;
      if (from != t0) {
        ids.fill(s.c, b, from >> 6, lane);
        end = min(any_hi, from + ATTN_SEGMENT);
        load(xa, t);
      }
      for (; t < end; t += 2 * ATTN_STEP) {
        load(xb, t + ATTN_STEP);
        step(xa, t);
        if (t + ATTN_STEP >= end) break;
        load(xa, t + 2 * ATTN_STEP);
        step(xb, t + ATTN_STEP);
      }
    }

    // The wave's column sums: l over the lane groups, and the minima's part of
    // dim group g (row g of om) added to its dims.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float part = __shfl(om[g & 3], (g >> 2) * 16 + col, 64);
      o[2 * g] += part;
      o[2 * g + 1] += part;
    }
    // Join the waves, pairs first: the upper of a pair hands over its sums.
#pragma unroll
    for (int half = ATTN_WAVES / 2; half >= 1; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
        const int w = wave - half;
#pragma unroll
        for (int i = 0; i < NT; ++i) *reinterpret_cast<kvf4*>(&so[w][col][16 * i + 4 * rg]) = o[i];
        if (rg == 0) { sr[w][col] = ref; sl[w][col] = l; }
      }
      __syncthreads();
      if (wave < half) {
        const float r2 = sr[wave][col], next = fmaxf(ref, r2);
        const float f = __builtin_amdgcn_exp2f(ref - next), f2 = __builtin_amdgcn_exp2f(r2 - next);
        ref = next;
        l = l * f + sl[wave][col] * f2;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          o[i] = o[i] * f + *reinterpret_cast<const kvf4*>(&so[wave][col][16 * i + 4 * rg]) * f2;
      }
    }
    if (wave != 0 || !valid) continue;
    if (whole) {
      const float inv = l != 0.f ? 1.f / l : 0.f;  // NaN stays
      T* out = (T*)s.a.out + (size_t)(sp.r0 + row) * s.a.out_stride + (size_t)head * D;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float y[4] = {o[i][0] * inv, o[i][1] * inv, o[i][2] * inv, o[i][3] * inv};
        store4(out + 16 * i + 4 * rg, y);
      }
      if (s.a.lse && rg == 0)
        s.a.lse[(size_t)(sp.r0 + row) * s.a.n_heads + head] = l != 0.f ? (ref + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
      continue;
    }
    AttnPart<D>* part = (AttnPart<D>*)s.a.work + (2 * (size_t)blockIdx.x + (u0 == 0)) * gridDim.y + blockIdx.y;
#pragma unroll
    for (int i = 0; i < NT; ++i) *reinterpret_cast<kvf4*>(&part->o[col][16 * i + 4 * rg]) = o[i];
    if (rg == 0) { part->ref[col] = ref; part->l[col] = l; }
  }
}

// Joins the parts of a sequence: a workgroup per (column of a kv head's
// tile, sequence).  Each of its waves takes every fourth part, 64 lanes over
// the dims; LDS adds the four up.
template <int D, class T>
__global__ __launch_bounds__(256) void kv4_attn_join(SplitArgs s) {
  constexpr int E = D / 64;
  __shared__ float so[4][D], sl[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.z, hk = blockIdx.y / s.tiles, tile = blockIdx.y % s.tiles, col = blockIdx.x;
  const Kv4Span sp = kv4_span(s.rows, b);
  const int ncol = min(16, min(sp.r1 - sp.r0, s.a.max_rows) * s.group - tile * 16);
  if (col >= ncol) return;
  const int max_slots = s.c.max_pages * KV4_PAGE;
  Kv4Span own = {0, 0, 0};
  if (lane < s.rows.n_seq) own = kv4_span(s.rows, lane);
  long long total, start;  // the axis, and where this sequence begins on it
  if (s.rows.n_seq <= 64) {
    const int n = lane < s.rows.n_seq ? rounds_of(own, s.a.window, max_slots) + AXIS_EXTRA : 0;
    const int upto = wave_scan_add(n);
    total = __builtin_amdgcn_readlane(upto, 63);
    start = __builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(n, b);
  } else {
    total = axis_total(s.rows, own, s.a.window, max_slots);
    start = lane < b ? rounds_of(own, s.a.window, max_slots) + AXIS_EXTRA : 0;
    for (int i = 64 + lane; i < b; i += 64)
      start += rounds_of(kv4_span(s.rows, i), s.a.window, max_slots) + AXIS_EXTRA;
#pragma unroll
    for (int o = 32; o; o >>= 1) start += __shfl_xor(start, o, 64);
  }
  const long long share = (total + s.groups - 1) / s.groups;
  start += AXIS_EXTRA;
  const long long first = start / share, last = (start + rounds_of(sp, s.a.window, max_slots) - 1) / share;
  const int count = (int)(last - first) + 1;
  if (count == 1) return;
  // Its parts: number 2 first + 1, then 2 x of the workgroups behind.
  const size_t step = gridDim.y;
  const AttnPart<D>* parts = (const AttnPart<D>*)s.a.work + 2 * (size_t)first * step + blockIdx.y;
  auto part = [&](int i) -> const AttnPart<D>& { return parts[(i ? 2 * (size_t)i : 1) * step]; };
  float ref = REF0;
  for (int i = lane; i < count; i += 64) ref = fmaxf(ref, part(i).ref[col]);
  for (int o = 32; o; o >>= 1) ref = fmaxf(ref, __shfl_xor(ref, o, 64));
  float l = 0.f, y[E] = {};
#pragma unroll 8
  for (int i = wave; i < count; i += 4) {
    const AttnPart<D>& p = part(i);
    const float f = __builtin_amdgcn_exp2f(p.ref[col] - ref);
    l += p.l[col] * f;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] += p.o[col][lane * E + e] * f;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[wave][lane * E + e] = y[e];
  if (lane == 0) sl[wave] = l;
  __syncthreads();
  const int i = threadIdx.x;
  if (i >= D) return;
  l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
  const float v = (so[0][i] + so[1][i]) + (so[2][i] + so[3][i]);
  const int ci = tile * 16 + col, row = sp.r0 + ci / s.group, head = hk * s.group + ci % s.group;
  ((T*)s.a.out)[(size_t)row * s.a.out_stride + (size_t)head * D + i] = (T)(l != 0.f ? v / l : 0.f);
  if (s.a.lse && i == 0)
    s.a.lse[(size_t)row * s.a.n_heads + head] = l != 0.f ? (ref + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
}

// (kv4_prefill_takes leaves at most 65535 of all kv heads.)
static int attn_tiles(int group, int max_rows) {
  return (int)(((long long)max_rows * group + 15) / 16);
}
// Workgroups that share the axis, of each kv head and column tile.
template <int D> static int attn_groups(int per_seq) { return std::max(1, ATTN_GROUPS<D> / per_seq); }

// Two parts of each workgroup, and workgroups times column tiles are at most
// ATTN_GROUPS: with more tiles one workgroup walks the whole axis, and there
// are no parts.
size_t kv4_attn_work_bytes(int head_dim) {
  return head_dim == 64    ? 2 * ATTN_GROUPS<64> * sizeof(AttnPart<64>)
         : head_dim == 128 ? 2 * ATTN_GROUPS<128> * sizeof(AttnPart<128>)
                           : 2 * ATTN_GROUPS<256> * sizeof(AttnPart<256>);
}

template <int D, class T>
static void attn_go(SplitArgs s, hipStream_t st) {
  const int per_seq = s.c.n_kv * s.tiles;
  s.groups = attn_groups<D>(per_seq);
  hipLaunchKernelGGL((kv4_attn_split<D, T>), dim3(s.groups, per_seq), dim3(64 * ATTN_WAVES), 0, st, s);
  const int cols = (int)std::min<long long>(16, (long long)s.a.max_rows * s.group);
  hipLaunchKernelGGL((kv4_attn_join<D, T>), dim3(cols, per_seq, s.rows.n_seq), dim3(256), 0, st, s);
}

template <class T>
static void attn_typed(int head_dim, const SplitArgs& s, hipStream_t st) {
  if (head_dim == 64) attn_go<64, T>(s, st);
  else if (head_dim == 128) attn_go<128, T>(s, st);
  else attn_go<256, T>(s, st);
}

hipError_t launch_kv4_attn(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Attn& a,
                           hipStream_t st) {
  if (kv4_prefill_takes(c, rows, a)) return launch_kv4_prefill(head_dim, c, type, rows, a, st);
  SplitArgs s{c, rows, a, a.n_heads / c.n_kv, attn_tiles(a.n_heads / c.n_kv, a.max_rows), 0};
  if (type == ACT_F32) attn_typed<float>(head_dim, s, st);
  else if (type == ACT_F16) attn_typed<_Float16>(head_dim, s, st);
  else attn_typed<bf16_t>(head_dim, s, st);
  return hipGetLastError();
}

}  // namespace kq
