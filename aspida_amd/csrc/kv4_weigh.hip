// kv4_weigh.hip -- the attention weight each cached slot received:
//   acc_out[b][hk][j] = acc_in[b][hk][j]
//                     + sum over rows and the query heads of hk of exp(scale q . k_j - lse)
// for the slots j a row sees (acc_out = acc_in for the others).
//
// A wave takes 64 slots, whose keys it unpacks into f16 operands once
// (kv4_mma.h), and goes through the columns (rows times query heads, 16 to a
// tile) with them: S[token][col] as in the attention, exp2, and a sum per
// token in registers; the columns of a tile are added at the end by a fixed
// order of lane exchanges.  No atomics, the same bits every time.
// Bound by the keys' bytes for the single rows of decode lanes, by the matrix
// cores for many rows.
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

template <int D, class T>
__global__ __launch_bounds__(256) void kv4_weigh(WeighArgs s) {
  using L = Kv4L<D>;
  constexpr bool TWO = sizeof(T) == 4;
  const int lane = threadIdx.x & 63, col = lane & 15, rg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.y, b = blockIdx.z;
  const Kv4Span sp = kv4_span(s.rows, b);
  const int n = sp.r1 - sp.r0, first = sp.len - n;  // the first row's slot
  const int any_lo = s.w.window > 0 ? max(0, first - s.w.window + 1) : 0, any_hi = n > 0 ? sp.len : 0;
  const size_t at = ((size_t)b * s.c.n_kv + hk) * s.w.acc_stride;
  const float* in = s.w.acc_in ? s.w.acc_in + at : nullptr;
  float* out = s.w.acc_out + at;
  for (long long p = (long long)blockIdx.x * 4 + wave; p * KV4_PAGE < s.w.acc_stride; p += (long long)gridDim.x * 4) {
    const long long t0 = p * KV4_PAGE;
    if (t0 + KV4_PAGE <= any_lo || t0 >= any_hi) {  // a page that no row sees
      if (t0 + lane < s.w.acc_stride) out[t0 + lane] = in ? in[t0 + lane] : 0.f;
      continue;
    }
    const uint8_t* blk = kv4_block(s.c, b, (int)p, hk, L::BYTES);
    const bool there = blk != nullptr;
    if (!there) blk = s.c.pages;
    KeyOps<D> k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      KeyTile<D> kt;
      kt.load(blk, i, lane);
      k[i].unpack(kt);
    }
    kvf4 sum[4] = {};
    for (int c0 = 0; c0 < n * s.group; c0 += 16) {
      const int ci = c0 + col, row = ci / s.group, head = hk * s.group + ci % s.group;
      const bool valid = ci < n * s.group;
      const int pos = first + row;
      const int chi = valid ? max(pos + 1, 0) : 0, clo = s.w.window > 0 ? max(0, pos - s.w.window + 1) : 0;
      // Rows ascend: past the last that sees the page none of the others does, and back.
      if (s.w.window > 0 && first + c0 / s.group - s.w.window + 1 >= t0 + KV4_PAGE) break;
      if (first + min(n - 1, (c0 + 15) / s.group) < t0) continue;
      Query<D, TWO> q;
      q.load((const T*)s.w.q + (size_t)(sp.r0 + (valid ? row : 0)) * s.w.q_stride + (size_t)head * D, valid, lane);
      const float unit = q.unit * (s.w.scale * WEIGH_LOG2E);
      const float lse = valid ? s.w.lse[(size_t)(sp.r0 + row) * s.w.n_heads + head] : -INFINITY;
      const float off = lse == -INFINITY ? INFINITY : lse * WEIGH_LOG2E;  // a row that saw nothing gives nothing
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const kvf4 c = k[i].scores(q);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int slot = (int)t0 + 16 * i + 4 * rg + j;
          const float x = there ? __builtin_fmaf(c[j], unit, -off) : __builtin_nanf("");
          sum[i][j] += slot >= clo && slot < chi ? __builtin_amdgcn_exp2f(x) : 0.f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v = sum[i][j];
        v += __shfl_xor(v, 1, 64);
        v += __shfl_xor(v, 2, 64);
        v += __shfl_xor(v, 4, 64);
        v += __shfl_xor(v, 8, 64);
        // Lane group rg now holds tokens 4 rg + j; lane (4 i + j) of it writes one.
        const long long t = t0 + 16 * i + 4 * rg + j;
        if (col == 4 * i + j && t < s.w.acc_stride) out[t] = (in ? in[t] : 0.f) + v;
      }
  }
}

template <int D, class T>
static void weigh_go(const WeighArgs& s, hipStream_t st) {
  const long long pages = (s.w.acc_stride + KV4_PAGE - 1) / KV4_PAGE;
  const dim3 grid((unsigned)std::min<long long>(4096, (pages + 3) / 4), s.c.n_kv, s.rows.n_seq);
  hipLaunchKernelGGL((kv4_weigh<D, T>), grid, dim3(256), 0, st, s);
}

template <class T>
static void weigh_typed(int head_dim, const WeighArgs& s, hipStream_t st) {
  if (head_dim == 64) weigh_go<64, T>(s, st);
  else if (head_dim == 128) weigh_go<128, T>(s, st);
  else weigh_go<256, T>(s, st);
}

hipError_t launch_kv4_weigh(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Weigh& w,
                            hipStream_t st) {
  const WeighArgs s{c, rows, w, w.n_heads / c.n_kv};
  if (type == ACT_F32) weigh_typed<float>(head_dim, s, st);
  else if (type == ACT_F16) weigh_typed<_Float16>(head_dim, s, st);
  else weigh_typed<bf16_t>(head_dim, s, st);
  return hipGetLastError();
}

}  // namespace kq
