// w8_rows.hip -- products of few tokens (up to 128) with 8-bit integer
// weights, plain and gated (the format and formulas: w8.h, w8_gemm.hip).
//
// A workgroup of eight waves takes one tile of 16 rows (of a gated block one
// of the gate and the same of the up projection) and all tokens, 16 to a
// column tile; its waves share k, a block of 64 in turn, and add their int32
// sums in LDS.  Weights go from memory to registers as the matrix
// instructions take them, two sets in turn, and are read once; the tokens'
// codes come from L2.  The few tokens of a decode step are quantised by every
// workgroup for itself, into LDS, while its first weights are on their way
// (FUSED): that saves a launch.
// Bound by the weights' bytes.
#include <algorithm>

#include "kq_common.h"
#include "w8.h"
#include "w8_kernels.h"

namespace kq {

constexpr int W8R_WAVES = 8;

// Blocks of a set: what keeps its operands within 64 registers.
template <int BT, bool GATED> constexpr int W8R_SET = BT == 1 ? (GATED ? 4 : 8) : BT == 2 ? 4 : BT == 4 ? 2 : 1;

template <class T, int BT, bool GATED, bool FUSED>
__global__ __launch_bounds__(64 * W8R_WAVES) void w8_rows(W8Args a) {
  constexpr int NP = GATED ? 2 : 1, U = W8R_SET<BT, GATED>;
  extern __shared__ uint8_t lds[];  // the waves' sums; FUSED: scales, then codes [token][64 blocks], before them
  __shared__ float part[W8R_WAVES], scale[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blocks = w8_blocks(a.in_dim), tile = blockIdx.x;
  const int row = 64 * blocks;  // bytes of a token's codes in LDS
  __amdgpu_buffer_rsrc_t w[NP], x[BT];
  auto buffer = [&](const uint8_t* p, int t) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p) + (size_t)t * blocks * W8_TILE, (short)0,
                                             blocks * W8_TILE, 0x00020000);
  };
  w[0] = buffer(a.w, tile);
  if constexpr (GATED) w[1] = buffer(a.up, tile);
#pragma unroll
  for (int j = 0; j < BT; ++j) x[j] = buffer(a.work, min(j, w8_tiles(a.n_tok) - 1));
  struct Set { w8i4 a[U][NP], b[U][BT]; };
  // Blocks past the end read as zeros.
  auto load_w = [&](Set& f, int i) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < NP; ++p)
        f.a[u][p] = __builtin_bit_cast(w8i4, __builtin_amdgcn_raw_buffer_load_b128(w[p], (wave + W8R_WAVES * (i + u)) * W8_TILE + lane * 16, 0, 2));
  };
  auto load_x = [&](Set& f, int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = wave + W8R_WAVES * (i + u);
      if constexpr (FUSED) {
        f.b[u][0] = *reinterpret_cast<const w8i4*>(lds + min(lane & 15, a.n_tok - 1) * row + min(kb, blocks - 1) * 64 + (lane >> 4) * 16);
      } else {
#pragma unroll
        for (int j = 0; j < BT; ++j)
          f.b[u][j] = __builtin_bit_cast(w8i4, __builtin_amdgcn_raw_buffer_load_b128(x[j], kb * W8_TILE + lane * 16, 0, 0));
      }
    }
  };
  w8i4 acc[NP][BT];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int j = 0; j < BT; ++j) acc[p][j] = w8i4{0, 0, 0, 0};
  auto multiply = [&](const Set& f) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int j = 0; j < BT; ++j) acc[p][j] = w8_mfma(f.a[u][p], f.b[u][j], acc[p][j]);
  };
  Set f, g;
  load_w(f, 0);
  if constexpr (FUSED) {
    for (int t = 0; t < a.n_tok; ++t) {
      const T* const from = (const T*)a.x + (long long)t * a.x_stride;
      float top = 0.f;
      for (int k = 16 * threadIdx.x; k < a.in_dim; k += 16 * 64 * W8R_WAVES) {
        float v[16];
        w8_load16(from, k, a.in_dim, v);
        top = w8_top16(v, top);
      }
      const W8Scale s(w8_group_max<W8R_WAVES>(top, part));
      if (threadIdx.x == 0) scale[t] = s.s;
      for (int k = 16 * threadIdx.x; k < row; k += 16 * 64 * W8R_WAVES) {
        float v[16];
        w8_load16(from, k, a.in_dim, v);
        *reinterpret_cast<uint4*>(lds + t * row + k) = w8_codes16(v, s);
      }
      __syncthreads();
    }
  }
  load_x(f, 0);
  const int mine = (blocks - wave + W8R_WAVES - 1) / W8R_WAVES;  // this wave's blocks
  for (int i = 0; i < mine; i += 2 * U) {
    load_w(g, i + U);
    load_x(g, i + U);
    multiply(f);
    load_w(f, i + 2 * U);
    load_x(f, i + 2 * U);
    multiply(g);
  }

  // The waves' sums: [wave][product][token tile][lane] of four rows.
  if constexpr (FUSED) __syncthreads();
  w8i4* const sums = reinterpret_cast<w8i4*>(lds);
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int j = 0; j < BT; ++j) sums[((wave * NP + p) * BT + j) * 64 + lane] = acc[p][j];
  __syncthreads();
  for (int q = threadIdx.x; q < 64 * BT; q += 64 * W8R_WAVES) {
    const int t = 16 * (q >> 6) + (q & 15), o = 16 * tile + 4 * (q >> 4 & 3);
    if (t >= a.n_tok || o >= a.out_dim) continue;
    w8i4 sum[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      sum[p] = sums[p * BT * 64 + q];
#pragma unroll
      for (int v = 1; v < W8R_WAVES; ++v) sum[p] += sums[(v * NP + p) * BT * 64 + q];
    }
    const W8Unit ux(FUSED ? scale[t & 15] : w8_scales(a.work, a.in_dim, a.n_tok)[t]);
    w8_finish<T, GATED>(a, t, o, sum[0], sum[NP - 1], ux);
  }
}

template <class T, int BT, bool GATED, bool FUSED>
static hipError_t rows_go(const W8Args& a, hipStream_t st) {
  constexpr int sums = W8R_WAVES * (GATED ? 2 : 1) * BT * 1024;
  const int lds = std::max(sums, FUSED ? a.n_tok * 64 * w8_blocks(a.in_dim) : 0);
  auto* k = &w8_rows<T, BT, GATED, FUSED>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k, dim3(w8_tiles(a.out_dim)), dim3(64 * W8R_WAVES), lds, st, a);
  return hipGetLastError();
}

// One workgroup's share of finding codes, against a launch for it.
bool w8_rows_fuse(const W8Args& a) { return a.n_tok <= 16 && (long long)a.n_tok * a.in_dim <= 16384; }
bool w8_rows_takes(const W8Args& a) { return a.n_tok <= 128; }

template <class T, bool GATED> static hipError_t rows_typed(const W8Args& a, hipStream_t st) {
  if (w8_rows_fuse(a)) return rows_go<T, 1, GATED, true>(a, st);
  if (a.n_tok <= 16) return rows_go<T, 1, GATED, false>(a, st);
  if (a.n_tok <= 32) return rows_go<T, 2, GATED, false>(a, st);
  if (a.n_tok <= 64) return rows_go<T, 4, GATED, false>(a, st);
  return rows_go<T, 8, GATED, false>(a, st);
}

hipError_t launch_w8_rows(int type, const W8Args& a, hipStream_t st) {
  if (type == ACT_F32) return a.up ? rows_typed<float, true>(a, st) : rows_typed<float, false>(a, st);
  if (type == ACT_F16) return a.up ? rows_typed<_Float16, true>(a, st) : rows_typed<_Float16, false>(a, st);
  return a.up ? rows_typed<bf16_t, true>(a, st) : rows_typed<bf16_t, false>(a, st);
}

}  // namespace kq
