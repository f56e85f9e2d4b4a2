// kv4_split.h -- attention over the 4-bit cache by shares of the slots: the
// axis that all sequences' slots make, its shares, their parts and the join;
// what the rows of a tree see.  Shared by kv4_attn.hip and kv4_tree.hip.
#pragma once
#include "kv4_mma.h"

namespace kq {

constexpr int ATTN_STEP = 128;  // tokens of a round, the axis's unit
constexpr float REF0 = -3.402823466e38f;  // below every score
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// Slots that a sequence's rows see together: [lo, hi), lo a multiple of 32.
struct SeenRange { int lo, hi; };
template <bool TREE>
__device__ __forceinline__ SeenRange seen_range(const Kv4Span& s, int window, int max_slots) {
  const int first = s.len - (s.r1 - s.r0);  // the first row's slot
  SeenRange r;
  r.hi = s.r1 > s.r0 ? min(s.len, max_slots) : 0;
  const int lowest = TREE ? (window > 0 ? max(0, max(first, 0) - window) : 0) : kv4_lowest(first, kv4_reach(window));
  r.lo = min(lowest, r.hi) & ~31;
  return r;
}

// A sequence's rounds (one at least: one whose rows see nothing has outputs
// too), and its length on the axis, which counts what a workgroup spends on a
// sequence besides: its rows, page ids and sums, about 8000 cycles where a
// round takes 1800.
constexpr int AXIS_EXTRA = 4;
template <bool TREE>
__device__ __forceinline__ int rounds_of(const Kv4Span& s, int window, int max_slots) {
  const SeenRange r = seen_range<TREE>(s, window, max_slots);
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
template <bool TREE>
__device__ __forceinline__ long long axis_total(const Kv4Rows& rows, const Kv4Span& own, int window, int max_slots) {
  const int lane = threadIdx.x & 63;
  long long total = lane < rows.n_seq ? rounds_of<TREE>(own, window, max_slots) + AXIS_EXTRA : 0;
  for (int b = 64 + lane; b < rows.n_seq; b += 64) total += rounds_of<TREE>(kv4_span(rows, b), window, max_slots) + AXIS_EXTRA;
#pragma unroll
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o, 64);
  return total;
}

template <bool TREE>
__device__ __forceinline__ AxisPlace axis_place(const Kv4Rows& rows, const Kv4Span& own, int window, int max_slots,
                                                int groups, int x) {
  const int lane = threadIdx.x & 63;
  AxisPlace p;
  if (rows.n_seq <= 64) {  // one lane each, and sums below 2^30
    const int n = lane < rows.n_seq ? rounds_of<TREE>(own, window, max_slots) + AXIS_EXTRA : 0;
    const int end = wave_scan_add(n);
    p.share = (__builtin_amdgcn_readlane(end, 63) + groups - 1) / groups;
    p.x0 = x * p.share;
    const uint64_t over = __ballot(end > p.x0);
    const int l = over ? __builtin_ctzll(over) : 63;
    p.seq = over ? l : rows.n_seq;
    p.start = __builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(n, l);
    return p;
  }
  p.share = (axis_total<TREE>(rows, own, window, max_slots) + groups - 1) / groups;
  p.x0 = x * p.share;
  long long before = 0;
  for (int b0 = 0; b0 < rows.n_seq; b0 += 64) {
    const int b = b0 + lane;
    const int n = b < rows.n_seq ? rounds_of<TREE>(b0 ? kv4_span(rows, b) : own, window, max_slots) + AXIS_EXTRA : 0;
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

// Workspace: per part, kv head and column tile the columns' sums [COLS][D] and
// (ref, l) [COLS].  A workgroup has at most two sequences in part: one that
// began in a share before its own (number 2 x) and one that goes on in the
// next (2 x + 1), so parts number as the workgroups do, not as the sequences.
template <int D, int COLS> struct AttnPart {
  float o[COLS][D];
  float ref[COLS], l[COLS];
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

// What a column of a tree sees: the slots [lo, base) and the rows [r0, r1)
// that its mask names.
struct TreeSeen {
  const uint32_t* mask;
  int lo, r0, r1;
  __device__ __forceinline__ uint32_t word(int w) const {
    uint32_t v = 32 * w < r1 && 32 * w + 32 > r0 ? mask[w] : 0u;
    if (32 * w + 32 > r1) v &= r1 - 32 * w > 0 ? ~0u >> (32 * w + 32 - r1) : 0u;
    if (32 * w < r0) v &= r0 - 32 * w < 32 ? ~0u << (r0 - 32 * w) : 0u;
    return v;
  }
  // Bits of the rows j .. j + 31 (j may be below 0).
  __device__ __forceinline__ uint32_t rows(int j) const {
    const int w = j >> 5;
    return __builtin_amdgcn_alignbit(word(w + 1), word(w), (uint32_t)(j & 31));
  }
  // The same with what it found for lo, which takes a walk over the mask.
  __device__ __forceinline__ TreeSeen(const Kv4Attn& a, int row0, int row, int n, int base, bool valid, int low) {
    r0 = max(0, -base);
    r1 = valid && base + row >= 0 ? min(n, 32 * a.mask_words) : 0;
    mask = a.mask + (size_t)(row0 + (r1 > 0 ? row : 0)) * a.mask_words;
    lo = low;
  }
  __device__ __forceinline__ TreeSeen() : mask(nullptr), lo(0), r0(0), r1(0) {}
  // n rows at slots from base on, of which those at slots below 0 do not count.
  __device__ __forceinline__ TreeSeen(const Kv4Attn& a, int row0, int row, int n, int base, bool valid) {
    r0 = max(0, -base);
    r1 = valid && base + row >= 0 ? min(n, 32 * a.mask_words) : 0;
    mask = a.mask + (size_t)(row0 + (r1 > 0 ? row : 0)) * a.mask_words;
    int shown = 0;
    if (a.window > 0)
      for (int w = 0; 32 * w < r1; ++w) shown += __popc(word(w));
    lo = r1 <= 0 ? max(base, 0) : a.window > 0 ? max(0, max(base, 0) - max(a.window - shown, 0)) : 0;
  }
  // Whether it sees a slot from max_slots on.
  __device__ __forceinline__ bool past(int base, int max_slots) const {
    if (lo < base && base > max_slots) return true;
    bool any = false;
    for (int j = max(0, max_slots - base); j < r1; j += 32) any |= rows(j) != 0;
    return any;
  }
};

}  // namespace kq
