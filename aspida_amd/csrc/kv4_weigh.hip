// kv4_weigh.hip -- the attention weight each cached slot received:
//   acc_out[b][hk][j] = acc_in[b][hk][j]
//                     + sum over rows and the query heads of hk of exp(scale q . k_j - lse)
// for the slots j a row sees (acc_out = acc_in for the others).
//
// The columns are rows times query heads, 16 to a tile; a wave turns keys into
// f16 operands (kv4_mma.h), S[token][col] as in the attention, exp2, and adds
// the columns of a token by a fixed order of lane moves.  No atomics, the
// same bits every time.
//   kv4_weigh_one   one tile of columns (decode lanes): its operands stay in
//                   registers, a wave walks pages with the next one in
//                   flight.  32 lanes of 8 kv heads of 128 (f32, 113 MB) 33
//                   us, 3.4 TB/s, of 22 at the rate of a large copy: bound
//                   by the vector units, 74% busy (unpacking, exp2, sums over
//                   columns).  (Loads without a branch, ids a step ahead: 34.)
//   kv4_weigh_many  a wave turns its page's keys into operands once; column
//                   tiles pass through LDS, each made by one wave and used by
//                   all.  64 rows over 32000 slots (64/8 heads of 128,
//                   bf16, 33.5 GFLOP) 77 us, of 29 at the rate of a large
//                   product.  No unit is full (vector units 53%, matrix
//                   cores 23%): a tile's operands are read, multiplied, raised
//                   and summed one after the other, and waves wait 43%.
#include <algorithm>

#include "kv4_mma.h"

namespace kq {

constexpr float WEIGH_LOG2E = 1.4426950408889634f;

template <int D> struct KeyOps {
  static constexpr int NG = D / 32;
  kvh8 a[NG], m;
  __device__ __forceinline__ void unpack(const KeyTile<D>& k) {
#pragma unroll
    for (int g = 0; g < NG; ++g) a[g] = k.codes(g);
    m = k.minima();
  }
  template <bool TWO>
  __device__ __forceinline__ kvf4 scores(const Query<D, TWO>& q) const {
    kvf4 c = kv_mfma(m, q.sums, kvf4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if constexpr (TWO) c = kv_mfma(a[g], q.lo[g], c);
      c = kv_mfma(a[g], q.hi[g], c);
    }
    return c;
  }
};

struct WeighArgs {
  Kv4View c;
  Kv4Rows rows;
  Kv4Weigh w;
  int group;
};

// The sum over the 16 lanes of a row, in each of them.
__device__ __forceinline__ float row_sum(float v) {
  v += dpp_from<0xB1>(v, 0.f);   // lane ^ 1
  v += dpp_from<0x4E>(v, 0.f);   // lane ^ 2
  v += dpp_from<0x141>(v, 0.f);  // mirrored within 8
  return v + dpp_from<0x140>(v, 0.f);  // mirrored within 16
}

// Lane l of a wave writes token 16 (l % 16 / 4) + 4 (l / 16) + l % 4 of its 64:
// the value among its sums[tile][j] that belongs there.
template <int H>
__device__ __forceinline__ float own_sum(const kvf4 (&sum)[H], int col) {
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < H; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float r = row_sum(sum[i][j]);
      if (col == 4 * i + j) v = r;
    }
  return v;
}

constexpr int ONE_WAVES = 4;

template <int D, class T>
__global__ __launch_bounds__(64 * ONE_WAVES) void kv4_weigh_one(WeighArgs s) {
  using L = Kv4L<D>;
  constexpr bool TWO = sizeof(T) == 4;
  constexpr int H = D == 256 ? 2 : 4, TOK = 16 * H;  // tiles of a step, its tokens
  const int lane = threadIdx.x & 63, col = lane & 15, rg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.y, b = blockIdx.z;
  const Kv4Span sp = kv4_span(s.rows, b);
  const int n = sp.r1 - sp.r0, first = sp.len - n, reach = kv4_reach(s.w.window);
  const int any_lo = kv4_lowest(first, reach), any_hi = n > 0 ? sp.len : 0;
  const size_t at = ((size_t)b * s.c.n_kv + hk) * s.w.acc_stride;
  const float* in = s.w.acc_in ? s.w.acc_in + at : nullptr;
  float* out = s.w.acc_out + at;
  const int row = col / s.group, head = hk * s.group + col % s.group;
  const bool valid = row < n;
  const int chi = valid ? max(first + row + 1, 0) : 0, clo = kv4_lowest(first + row, reach);
  // What every column that counts sees (columns that are none have lse inf).
  const int all_hi = first + 1, all_lo = kv4_lowest(first + min(n - 1, 15 / s.group), reach);

  const long long step = (long long)gridDim.x * ONE_WAVES * TOK;
  long long t0 = ((long long)blockIdx.x * ONE_WAVES + wave) * TOK;
  KeyTile<D> k[H];
  float acc = 0.f;
  bool there = false;
  const int mine = 16 * (col >> 2) + 4 * rg + (col & 3);  // the token of a step that this lane writes
  const bool writes = (col >> 2) < H;
  auto seen = [&](long long t) { return t + TOK > any_lo && t < any_hi; };
  auto load = [&](long long t) {
    acc = in && writes && t + mine < s.w.acc_stride ? in[t + mine] : 0.f;
    if (!seen(t)) return;
    const uint8_t* blk = kv4_block(s.c, b, (int)(t / KV4_PAGE), hk, L::BYTES);
    there = blk != nullptr;
    if (!blk) blk = s.c.pages;
#pragma unroll
    for (int i = 0; i < H; ++i) k[i].load(blk, (int)(t % KV4_PAGE) / 16 + i, lane);
  };
  load(t0);
  Query<D, TWO> q;
  q.load((const T*)s.w.q + (size_t)(sp.r0 + (valid ? row : 0)) * s.w.q_stride + (size_t)head * D,
         valid && any_hi > 0, lane);
  const float unit = q.unit * (s.w.scale * WEIGH_LOG2E);
  // A row that saw nothing (lse -inf) gives nothing, nor does a column that is none.
  const float lse = valid ? s.w.lse[(size_t)(sp.r0 + row) * s.w.n_heads + head] : -INFINITY;
  const float off = lse == -INFINITY ? INFINITY : lse * WEIGH_LOG2E;
  for (; t0 < s.w.acc_stride; t0 += step) {
    kvf4 c[H];
    const bool see = seen(t0), ok = there;
    if (see) {
#pragma unroll
      for (int i = 0; i < H; ++i) c[i] = q.scores(k[i]);
    }
    const float base = acc;
    if (t0 + step < s.w.acc_stride) load(t0 + step);
    float v = 0.f;
    if (see) {
      const bool whole = ok && t0 >= all_lo && t0 + TOK <= all_hi;
#pragma unroll
      for (int i = 0; i < H; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = __builtin_fmaf(c[i][j], unit, -off);
          if (!whole) {
            const int slot = (int)t0 + 16 * i + 4 * rg + j;
            x = slot >= clo && slot < chi ? (ok ? x : __builtin_nanf("")) : -INFINITY;
          }
          c[i][j] = __builtin_amdgcn_exp2f(x);
        }
      v = own_sum(c, col);
    }
    if (writes && t0 + mine < s.w.acc_stride) out[t0 + mine] = base + v;
  }
  // Rows past max_rows may have no column: NaN in all slots seen, by the lanes
  // that wrote them.  (Decided in the loop above: 36 us for 33.)
  if (n <= s.w.max_rows) return;
  const long long end = min((long long)any_hi, s.w.acc_stride);
  for (t0 = ((long long)blockIdx.x * ONE_WAVES + wave) * TOK; t0 < end; t0 += step)
    if (writes && t0 + mine >= any_lo && t0 + mine < end) out[t0 + mine] = __builtin_nanf("");
}

constexpr int WEIGH_WAVES = 8;

// What a wave holds and what a workgroup prepares: 16-token tiles of a page at
// a time (all four would not fit beside the operands of a head of 256), and
// column tiles in LDS.
template <int D, class T> struct WeighShape {
  static constexpr bool TWO = sizeof(T) == 4;
  static constexpr int NG = D / 32, HOLD = D == 256 ? 2 : 4, TILES = D == 256 ? 4 : 8;
  static constexpr int OPS = NG * (TWO ? 2 : 1) + 1;  // 1 KB operands of a column tile
  static constexpr size_t LDS = (size_t)TILES * (OPS * 1024 + 16 * 16);
};

template <int D, class T>
__global__ __launch_bounds__(64 * WEIGH_WAVES) void kv4_weigh_many(WeighArgs s) {
  using L = Kv4L<D>;
  using W = WeighShape<D, T>;
  constexpr bool TWO = W::TWO;
  constexpr int NG = W::NG;
  extern __shared__ kvu4 lds[];
  kvu4* cols = lds + W::TILES * W::OPS * 64;  // unit, lse (f32), clo, chi of a column
  const int lane = threadIdx.x & 63, col = lane & 15, rg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.y, b = blockIdx.z;
  const Kv4Span sp = kv4_span(s.rows, b);
  const int n = sp.r1 - sp.r0, first = sp.len - n, reach = kv4_reach(s.w.window);  // first: the first row's slot
  const int tiles = (int)(((long long)n * s.group + 15) / 16);
  const int any_lo = kv4_lowest(first, reach), any_hi = n > 0 ? sp.len : 0;
  const size_t at = ((size_t)b * s.c.n_kv + hk) * s.w.acc_stride;
  const float* in = s.w.acc_in ? s.w.acc_in + at : nullptr;
  float* out = s.w.acc_out + at;

  // Operands of column tile c, by one wave, into place i.
  auto prepare = [&](int c, int i) {
    const int ci = c * 16 + col, row = ci / s.group, head = hk * s.group + ci % s.group;
    const bool valid = row < n;
    const int pos = first + row;
    Query<D, TWO> q;
    q.load((const T*)s.w.q + (size_t)(sp.r0 + (valid ? row : 0)) * s.w.q_stride + (size_t)head * D, valid, lane);
    kvu4* to = lds + i * W::OPS * 64 + lane;
    to[0] = __builtin_bit_cast(kvu4, q.sums);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      to[(1 + g) * 64] = __builtin_bit_cast(kvu4, q.hi[g]);
      if constexpr (TWO) to[(1 + NG + g) * 64] = __builtin_bit_cast(kvu4, q.lo[g]);
    }
    if (rg == 0) {
      // A row that saw nothing (lse -inf) gives nothing, nor does a column that is none.
      const float lse = valid ? s.w.lse[(size_t)(sp.r0 + row) * s.w.n_heads + head] : -INFINITY;
      const int chi = valid ? max(pos + 1, 0) : 0, clo = kv4_lowest(pos, reach);
      const float unit = n > s.w.max_rows ? __builtin_nanf("") : q.unit * (s.w.scale * WEIGH_LOG2E);
      cols[i * 16 + col] = kvu4{__builtin_bit_cast(uint32_t, unit),
                                __builtin_bit_cast(uint32_t, lse == -INFINITY ? INFINITY : lse * WEIGH_LOG2E),
                                (uint32_t)clo, (uint32_t)chi};
    }
  };

  int ready = -1;  // first column tile of those in LDS
  const long long step = (long long)gridDim.x * WEIGH_WAVES;
  for (long long p0 = (long long)blockIdx.x * WEIGH_WAVES; p0 * KV4_PAGE < s.w.acc_stride; p0 += step) {
    const long long t0 = (p0 + wave) * KV4_PAGE;
    if (t0 + KV4_PAGE <= any_lo || t0 >= any_hi)  // a page that no row sees
      if (t0 + lane < s.w.acc_stride) out[t0 + lane] = in ? in[t0 + lane] : 0.f;
    // The same for all waves, which meet in LDS: does any of their pages matter?
    if ((p0 + WEIGH_WAVES) * KV4_PAGE <= any_lo || p0 * KV4_PAGE >= any_hi) continue;
    const bool mine = t0 + KV4_PAGE > any_lo && t0 < any_hi;
    const uint8_t* blk = mine ? kv4_block(s.c, b, (int)(p0 + wave), hk, L::BYTES) : nullptr;
    const bool there = blk != nullptr;
    if (!there) blk = s.c.pages;
    for (int h = 0; h < 4; h += W::HOLD) {
      KeyOps<D> k[W::HOLD];
      kvf4 sum[W::HOLD] = {};
      if (mine) {
#pragma unroll
        for (int i = 0; i < W::HOLD; ++i) {
          KeyTile<D> kt;
          kt.load(blk, h + i, lane);
          k[i].unpack(kt);
        }
      }
      for (int c0 = 0; c0 < tiles; c0 += W::TILES) {
        if (ready != c0) {
          __syncthreads();
          if (wave < W::TILES && c0 + wave < tiles) prepare(c0 + wave, wave);
          __syncthreads();
          ready = c0;
        }
        if (!mine) continue;
        for (int i = 0; i < min(W::TILES, tiles - c0); ++i) {
          const int r0 = (c0 + i) * 16 / s.group, r1 = min(n - 1, ((c0 + i) * 16 + 15) / s.group);
          // No row of the tile sees the page: all below it, or their windows past it.
          if (first + r1 < t0 || max(first + r0, 0) - reach >= t0 + KV4_PAGE) continue;
          const bool whole = there && first + r0 + 1 >= t0 + KV4_PAGE && max(first + r1, 0) - reach <= t0;
          const kvu4* from = lds + i * W::OPS * 64 + lane;
          Query<D, TWO> q;
          q.sums = __builtin_bit_cast(kvh8, from[0]);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            q.hi[g] = __builtin_bit_cast(kvh8, from[(1 + g) * 64]);
            if constexpr (TWO) q.lo[g] = __builtin_bit_cast(kvh8, from[(1 + NG + g) * 64]);
          }
          const kvu4 cc = cols[i * 16 + col];
          const uint32_t bits[2] = {cc.x, cc.y};
          const float unit = __builtin_bit_cast(float, bits[0]), off = __builtin_bit_cast(float, bits[1]);
#pragma unroll
          for (int e = 0; e < W::HOLD; ++e) {
            const kvf4 c = k[e].scores(q);
            if (whole) {
#pragma unroll
              for (int j = 0; j < 4; ++j) sum[e][j] += __builtin_amdgcn_exp2f(__builtin_fmaf(c[j], unit, -off));
            } else {
              const int clo = (int)cc.z, chi = (int)cc.w;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int slot = (int)t0 + 16 * (h + e) + 4 * rg + j;
                const float x = there ? __builtin_fmaf(c[j], unit, -off) : __builtin_nanf("");
                sum[e][j] += slot >= clo && slot < chi ? __builtin_amdgcn_exp2f(x) : 0.f;
              }
            }
          }
        }
      }
      if (!mine) continue;
      const float v = own_sum(sum, col);
      const long long t = t0 + 16 * (h + (col >> 2)) + 4 * rg + (col & 3);
      if ((col >> 2) < W::HOLD && t < s.w.acc_stride) out[t] = (in ? in[t] : 0.f) + v;
    }
  }
}

template <int D, class T>
static hipError_t weigh_go(const WeighArgs& s, hipStream_t st) {
  using W = WeighShape<D, T>;
  if ((long long)s.w.max_rows * s.group <= 16) {
    constexpr int tokens = ONE_WAVES * (D == 256 ? 32 : 64);
    const long long most = (s.w.acc_stride + tokens - 1) / tokens;
    const long long want = (1024 + (long long)s.c.n_kv * s.rows.n_seq - 1) / ((long long)s.c.n_kv * s.rows.n_seq);
    hipLaunchKernelGGL((kv4_weigh_one<D, T>), dim3((unsigned)std::min(most, want), s.c.n_kv, s.rows.n_seq),
                       dim3(64 * ONE_WAVES), 0, st, s);
    return hipGetLastError();
  }
  // About four workgroups per CU, fewer where there are fewer pages.
  const long long pages = (s.w.acc_stride + KV4_PAGE - 1) / KV4_PAGE;
  const long long most = (pages + WEIGH_WAVES - 1) / WEIGH_WAVES;
  const long long want = (1024 + (long long)s.c.n_kv * s.rows.n_seq - 1) / ((long long)s.c.n_kv * s.rows.n_seq);
  const hipError_t e = hipFuncSetAttribute((const void*)&kv4_weigh_many<D, T>,
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)W::LDS);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((kv4_weigh_many<D, T>), dim3((unsigned)std::min(most, want), s.c.n_kv, s.rows.n_seq),
                     dim3(64 * WEIGH_WAVES), W::LDS, st, s);
  return hipGetLastError();
}

template <class T>
static hipError_t weigh_typed(int head_dim, const WeighArgs& s, hipStream_t st) {
  if (head_dim == 64) return weigh_go<64, T>(s, st);
  if (head_dim == 128) return weigh_go<128, T>(s, st);
  return weigh_go<256, T>(s, st);
}

hipError_t launch_kv4_weigh(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Weigh& w,
                            hipStream_t st) {
  const WeighArgs s{c, rows, w, w.n_heads / c.n_kv};
  if (type == ACT_F32) return weigh_typed<float>(head_dim, s, st);
  if (type == ACT_F16) return weigh_typed<_Float16>(head_dim, s, st);
  return weigh_typed<bf16_t>(head_dim, s, st);
}

}  // namespace kq
