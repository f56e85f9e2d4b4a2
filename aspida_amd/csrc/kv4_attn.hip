// kv4_attn.hip -- attention over the paged 4-bit cache.
//
// Row i of a sequence's n new rows sits at slot p = kv_len - n + i and sees
// the slots j <= p (and j > p - window):
//   o = sum_j softmax_j(scale q . k_j) v_j,   lse = log sum_j exp(scale q . k_j).
// A row that sees nothing gets o = 0 and lse = -inf.  Rows that are a tree
// (TREE) see the slots j < kv_len - n, and of the n rows those that their mask
// names; with a window, so many of the former that it sees `window` in all.
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

#include "kv4_split.h"

namespace kq {

constexpr int ATTN_WAVES = 4;
static_assert(ATTN_STEP == 32 * ATTN_WAVES);  // a workgroup's round
// Tokens whose page ids a wave holds at once: whole rounds, within 64 pages
// wherever in a page they start.
constexpr int ATTN_SEGMENT = (4096 - 32) / ATTN_STEP * ATTN_STEP;
// Workgroups that fit at once: 256 CUs times what their registers allow (under
// 168, 256 and 512 for heads of 64, 128 and 256).  One round of equal shares
// measured against 1.5 and 2 rounds (32/8 heads, f32): 130001 slots 47, 59
// and 57 us; 16 lanes of 8000 45, 56 and 54 us.
template <int D> constexpr int ATTN_GROUPS = D == 64 ? 768 : D == 128 ? 512 : 256;

template <int D, class T, bool TREE>
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
  AxisPlace place = axis_place<TREE>(s.rows, own, s.a.window, max_slots, s.groups, blockIdx.x);
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
    const SeenRange seen = seen_range<TREE>(sp, s.a.window, max_slots);
    const int length = rounds_of<TREE>(sp, s.a.window, max_slots);
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
    int all_hi = sp.len - n + row_first + 1;  // below: seen by every column
    int all_lo = kv4_lowest(sp.len - n + row_last, reach);
    int any_hi = min(t1, sp.len - n + row_last + 1);
    int any_lo = kv4_lowest(sp.len - n + row_first, reach);
    const int base = sp.len - n;
    const TreeSeen tree = TREE ? TreeSeen(s.a, sp.r0, row, n, base, valid) : TreeSeen();
    if constexpr (TREE) {
      any_lo = valid ? tree.lo : base;
      all_lo = valid ? tree.lo : 0;
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) {
        any_lo = min(any_lo, __shfl_xor(any_lo, o, 64));
        all_lo = max(all_lo, __shfl_xor(all_lo, o, 64));
      }
      any_lo = __builtin_amdgcn_readfirstlane(any_lo);
      all_lo = __builtin_amdgcn_readfirstlane(all_lo);
      all_hi = base;
      any_hi = t1;
    }

    kvf4 o[NT], om = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] = om;
    // A row past the table sees its own slot there: NaN.
    const bool past = TREE ? u0 == 0 && wave == 0 && tree.past(base, max_slots) : chi > max_slots && u0 == 0 && wave == 0;
    float ref = REF0, l = past ? __builtin_nanf("") : 0.f;

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
        // A tree: bit i of sees is slot at + i for this column, of some for any of them.
        uint32_t sees = 0, some = 0;
        if constexpr (TREE) {
          if (at + 32 > base) sees = tree.rows(at - base);
          const int lo = tree.lo - at, hi = base - at;
          if (hi > 0 && lo < 32 && lo < hi) sees |= (hi < 32 ? ~(~0u << hi) : ~0u) & (lo > 0 ? ~0u << lo : ~0u);
          some = sees;
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) some |= (uint32_t)__shfl_xor((int)some, o, 64);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int in = 16 * (j >> 2) + 4 * rg + (j & 3), slot = at + in;
          const bool see = TREE ? sees >> in & 1 : slot >= clo && slot < chi;
          x[j] = see ? (y.there ? x[j] * unit : __builtin_nanf("")) : -INFINITY;
          if (y.there && (TREE ? some >> in & 1 : slot < any_hi && slot >= any_lo)) keep |= 1u << j;
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
    AttnPart<D, 16>* part = (AttnPart<D, 16>*)s.a.work + (2 * (size_t)blockIdx.x + (u0 == 0)) * gridDim.y + blockIdx.y;
#pragma unroll
    for (int i = 0; i < NT; ++i) *reinterpret_cast<kvf4*>(&part->o[col][16 * i + 4 * rg]) = o[i];
    if (rg == 0) { part->ref[col] = ref; part->l[col] = l; }
  }
}

// Joins the parts of a sequence: a workgroup per (column of a kv head's
// tile, sequence).  Each of its waves takes every fourth part, 64 lanes over
// the dims; LDS adds the four up.
template <int D, class T, bool TREE>
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
    const int n = lane < s.rows.n_seq ? rounds_of<TREE>(own, s.a.window, max_slots) + AXIS_EXTRA : 0;
    const int upto = wave_scan_add(n);
    total = __builtin_amdgcn_readlane(upto, 63);
    start = __builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(n, b);
  } else {
    total = axis_total<TREE>(s.rows, own, s.a.window, max_slots);
    start = lane < b ? rounds_of<TREE>(own, s.a.window, max_slots) + AXIS_EXTRA : 0;
    for (int i = 64 + lane; i < b; i += 64)
      start += rounds_of<TREE>(kv4_span(s.rows, i), s.a.window, max_slots) + AXIS_EXTRA;
#pragma unroll
    for (int o = 32; o; o >>= 1) start += __shfl_xor(start, o, 64);
  }
  const long long share = (total + s.groups - 1) / s.groups;
  start += AXIS_EXTRA;
  const long long first = start / share, last = (start + rounds_of<TREE>(sp, s.a.window, max_slots) - 1) / share;
  const int count = (int)(last - first) + 1;
  if (count == 1) return;
  // Its parts: number 2 first + 1, then 2 x of the workgroups behind.
  const size_t step = gridDim.y;
  const AttnPart<D, 16>* parts = (const AttnPart<D, 16>*)s.a.work + 2 * (size_t)first * step + blockIdx.y;
  auto part = [&](int i) -> const AttnPart<D, 16>& { return parts[(i ? 2 * (size_t)i : 1) * step]; };
  float ref = REF0;
  for (int i = lane; i < count; i += 64) ref = fmaxf(ref, part(i).ref[col]);
  for (int o = 32; o; o >>= 1) ref = fmaxf(ref, __shfl_xor(ref, o, 64));
  float l = 0.f, y[E] = {};
#pragma unroll 8
  for (int i = wave; i < count; i += 4) {
    const AttnPart<D, 16>& p = part(i);
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
  return head_dim == 64    ? 2 * ATTN_GROUPS<64> * sizeof(AttnPart<64, 16>)
         : head_dim == 128 ? 2 * ATTN_GROUPS<128> * sizeof(AttnPart<128, 16>)
                           : 2 * ATTN_GROUPS<256> * sizeof(AttnPart<256, 16>);
}

template <int D, class T, bool TREE>
static void attn_go(SplitArgs s, hipStream_t st) {
  const int per_seq = s.c.n_kv * s.tiles;
  s.groups = attn_groups<D>(per_seq);
  hipLaunchKernelGGL((kv4_attn_split<D, T, TREE>), dim3(s.groups, per_seq), dim3(64 * ATTN_WAVES), 0, st, s);
  const int cols = (int)std::min<long long>(16, (long long)s.a.max_rows * s.group);
  hipLaunchKernelGGL((kv4_attn_join<D, T, TREE>), dim3(cols, per_seq, s.rows.n_seq), dim3(256), 0, st, s);
}

template <class T, bool TREE>
static void attn_typed(int head_dim, const SplitArgs& s, hipStream_t st) {
  if (head_dim == 64) attn_go<64, T, TREE>(s, st);
  else if (head_dim == 128) attn_go<128, T, TREE>(s, st);
  else attn_go<256, T, TREE>(s, st);
}

hipError_t launch_kv4_attn(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Attn& a,
                           hipStream_t st) {
  if (!a.mask && kv4_prefill_takes(c, rows, a)) return launch_kv4_prefill(head_dim, c, type, rows, a, st);
  SplitArgs s{c, rows, a, a.n_heads / c.n_kv, attn_tiles(a.n_heads / c.n_kv, a.max_rows), 0};
  if (a.mask) {
    if (type == ACT_F32) attn_typed<float, true>(head_dim, s, st);
    else if (type == ACT_F16) attn_typed<_Float16, true>(head_dim, s, st);
    else attn_typed<bf16_t, true>(head_dim, s, st);
  } else {
    if (type == ACT_F32) attn_typed<float, false>(head_dim, s, st);
    else if (type == ACT_F16) attn_typed<_Float16, false>(head_dim, s, st);
    else attn_typed<bf16_t, false>(head_dim, s, st);
  }
  return hipGetLastError();
}

}  // namespace kq
