// w8_gemm.hip -- products of many tokens with 8-bit integer weights, plain and
// gated, and the codes of tokens (the format: w8.h).
//
//   y[t][o] = s_x[t] s_w[o] sum_k c_x[t][k] c_w[o][k]
//   gated:  act(gate[t][o]) up[t][o], both products in one pass over x
//
// w8_tokens finds the tokens' scales and codes.  w8_gemm: a workgroup takes
// NA row tiles by NB token tiles (16 x 16 each) and walks k in stages of 64.
// The tiles of both sides lie in memory as the matrix instructions take them,
// so a stage goes to LDS by loads that bypass the registers, 1 KB an
// instruction, into a ring of four; a wave reads the operands of stage s + 1
// while it multiplies those of stage s, so a barrier (one a stage) finds
// matrix work in hand.  In a gated block a wave has as many row tiles of the
// gate as of the up projection, and forms their product in its registers.
#include <algorithm>

#include "kq_common.h"
#include "w8.h"
#include "w8_kernels.h"

namespace kq {

// ---- tokens' codes -------------------------------------------------------------

// A workgroup of TOK = 1 token (few tokens) or of the 16 of a tile (whole
// lines are written).  A thread's 16 values of the first KEEP turns stay in
// registers between the two passes; longer rows are read twice.
template <class T, int TOK, int THREADS>
__global__ __launch_bounds__(THREADS) void w8_tokens(const T* x, long long stride, int n_tok, int in_dim, uint8_t* work) {
  constexpr int KEEP = 4, RUNS = THREADS / TOK;  // runs of 16 values a turn
  __shared__ float part[TOK][THREADS / 64];
  const int tid = threadIdx.x, blocks = w8_blocks(in_dim);
  const int t = TOK == 1 ? 0 : tid & 15, run = TOK == 1 ? tid : tid >> 4;
  const int row = blockIdx.x * TOK + t, turns = (4 * blocks + RUNS - 1) / RUNS;
  const T* const from = x + (long long)min(row, n_tok - 1) * stride;
  float kept[KEEP][16], top = 0.f;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int k = 16 * (run + i * RUNS);
    if (k >= in_dim) break;
    w8_load16(from, k, in_dim, kept[i]);
    top = w8_top16(kept[i], top);
  }
  for (int i = KEEP; i < turns; ++i) {
    float v[16];
    const int k = 16 * (run + i * RUNS);
    if (k >= in_dim) break;
    w8_load16(from, k, in_dim, v);
    top = w8_top16(v, top);
  }
  if constexpr (TOK == 1) {
    top = w8_group_max<THREADS / 64>(top, part[0]);
  } else {
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if ((tid & 63) < 16) part[t][tid >> 6] = top;
    __syncthreads();
    for (int i = 0; i < THREADS / 64; ++i) top = fmaxf(top, part[t][i]);
  }
  if (row >= n_tok) return;
  const W8Scale s(top);
  if (run == 0) w8_scales(work, in_dim, n_tok)[row] = s.s;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int k = 16 * (run + i * RUNS);
    if (k >= in_dim) break;
    *reinterpret_cast<uint4*>(work + w8_place(row, k, blocks)) = w8_codes16(kept[i], s);
  }
  for (int i = KEEP; i < turns; ++i) {
    float v[16];
    const int k = 16 * (run + i * RUNS);
    if (k >= in_dim) break;
    w8_load16(from, k, in_dim, v);
    *reinterpret_cast<uint4*>(work + w8_place(row, k, blocks)) = w8_codes16(v, s);
  }
}

// ---- products --------------------------------------------------------------------

__device__ __forceinline__ __amdgpu_buffer_rsrc_t w8_buffer(const uint8_t* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), (short)0, 0x7FFFFFFF, 0x00020000);
}
__device__ __forceinline__ void w8_to_lds(__amdgpu_buffer_rsrc_t r, int lane_off, int off, uint32_t lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(uintptr_t)lds, 16, lane_off, off, 0, 0);
}
// At most N of this wave's loads outstanding, then the workgroup's barrier.
template <int N> __device__ __forceinline__ void w8_wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

// WR x WT waves, each AR row tiles (of a gated block: AR / 2 of the gate, AR /
// 2 of the up projection) by BT token tiles.
template <class T, int WR, int WT, int AR, int BT, bool GATED>
__global__ __launch_bounds__(64 * WR * WT, WR * WT >= 8 ? 2 : 1) void w8_gemm(W8Args a) {
  constexpr int W = WR * WT, NA = WR * AR, NB = WT * BT, PER = (NA + NB) / W, STAGE = (NA + NB) * W8_TILE, RING = 4;
  constexpr int OUTS = GATED ? AR / 2 : AR;  // row tiles of the result a wave
  static_assert((NA + NB) % W == 0);
  extern __shared__ uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave / WT, wt = wave % WT;
  const int blocks = w8_blocks(a.in_dim), row_tiles = w8_tiles(a.out_dim), tok_tiles = w8_tiles(a.n_tok);
  const int gr = (row_tiles + WR * OUTS - 1) / (WR * OUTS), gt = (tok_tiles + NB - 1) / NB;
  // Workgroups go round the XCDs in turn; each XCD takes a run of the tiles,
  // in bands of 4 token tiles, so that those at work at a time share lines.
  const int total = gr * gt, per = (total + 7) / 8;
  const int at = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || at >= total) return;
  const int band = at / (4 * gr), in_band = at - band * 4 * gr, height = min(4, gt - 4 * band);
  const int bt0 = (4 * band + in_band % height) * NB, br0 = in_band / height * (WR * OUTS);

  // This wave's loads of a stage: PER tiles of the NA + NB.
  __amdgpu_buffer_rsrc_t from[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = wave * PER + i;
    const uint8_t* p;
    if (t < NA) {
      const int w = t / AR, j = t % AR;
      const bool up = GATED && j >= OUTS;
      p = (up ? a.up : a.w) + (size_t)min(br0 + w * OUTS + (up ? j - OUTS : j), row_tiles - 1) * blocks * W8_TILE;
    } else {
      p = a.work + (size_t)min(bt0 + t - NA, tok_tiles - 1) * blocks * W8_TILE;
    }
    from[i] = w8_buffer(p);
  }
  const uint32_t base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)lds;
  auto fetch = [&](int s) {
    const int off = min(s, blocks - 1) * W8_TILE;
#pragma unroll
    for (int i = 0; i < PER; ++i) w8_to_lds(from[i], lane * 16, off, base + (s % RING) * STAGE + (wave * PER + i) * W8_TILE);
  };
  const uint8_t* const la = lds + (wr * AR) * W8_TILE + lane * 16;
  const uint8_t* const lb = lds + (NA + wt * BT) * W8_TILE + lane * 16;
  auto operand = [](const uint8_t* p, int s, int i) {
    return *reinterpret_cast<const w8i4*>(p + (s % RING) * STAGE + i * W8_TILE);
  };
  w8i4 acc[AR][BT], ra[AR], rb[2][BT];
#pragma unroll
  for (int i = 0; i < AR; ++i)
#pragma unroll
    for (int j = 0; j < BT; ++j) acc[i][j] = w8i4{0, 0, 0, 0};
  // Stage s + 3 goes where s - 1 was, whose operands every wave has multiplied,
  // and so has read, before the barrier of step s.  Past the end the last stage is loaded again.  A row
  // tile's operand is replaced by the next stage's as soon as it is used.
  auto step = [&](int s, const w8i4 (&b)[BT], w8i4 (&next)[BT]) {
    w8_wait_barrier<PER>();
    fetch(s + 3);
#pragma unroll
    for (int j = 0; j < BT; ++j) next[j] = operand(lb, s + 1, j);
#pragma unroll
    for (int i = 0; i < AR; ++i) {
#pragma unroll
      for (int j = 0; j < BT; ++j) acc[i][j] = w8_mfma(ra[i], b[j], acc[i][j]);
      ra[i] = operand(la, s + 1, i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  fetch(0);
  fetch(1);
  fetch(2);
  w8_wait_barrier<2 * PER>();
#pragma unroll
  for (int j = 0; j < BT; ++j) rb[0][j] = operand(lb, 0, j);
#pragma unroll
  for (int i = 0; i < AR; ++i) ra[i] = operand(la, 0, i);
  for (int s = 0; s < blocks; s += 2) {
    step(s, rb[0], rb[1]);
    step(s + 1, rb[1], rb[0]);
  }
  w8_wait_barrier<0>();  // nothing is on its way to LDS when the workgroup ends

  const float* sx = w8_scales(a.work, a.in_dim, a.n_tok);
#pragma unroll
  for (int j = 0; j < BT; ++j) {
    const int t = (bt0 + wt * BT + j) * 16 + (lane & 15);
    if (t >= a.n_tok) continue;
    const W8Unit ux(sx[t]);
#pragma unroll
    for (int i = 0; i < OUTS; ++i) {
      const int o = (br0 + wr * OUTS + i) * 16 + 4 * (lane >> 4);
      if (o < a.out_dim) w8_finish<T, GATED>(a, t, o, acc[i][j], acc[i + (GATED ? OUTS : 0)][j], ux);
    }
  }
}

template <class T, int WR, int WT, int AR, int BT, bool GATED>
static hipError_t gemm_go(const W8Args& a, hipStream_t st) {
  constexpr int lds = 4 * (WR * AR + WT * BT) * W8_TILE;
  auto* k = &w8_gemm<T, WR, WT, AR, BT, GATED>;
  const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  const int outs = WR * (GATED ? AR / 2 : AR);
  const long long total = (long long)((w8_tiles(a.out_dim) + outs - 1) / outs) * ((w8_tiles(a.n_tok) + WT * BT - 1) / (WT * BT));
  hipLaunchKernelGGL(k, dim3((unsigned)((total + 7) / 8 * 8)), dim3(64 * WR * WT), lds, st, a);
  return hipGetLastError();
}

template <class T> static hipError_t w8_typed(int type, const W8Args& a, hipStream_t st) {
  if (w8_rows_takes(a) && w8_rows_fuse(a)) return launch_w8_rows(type, a, st);
  if (a.n_tok < 64)
    hipLaunchKernelGGL((w8_tokens<T, 1, 256>), dim3(a.n_tok), dim3(256), 0, st, (const T*)a.x, a.x_stride, a.n_tok, a.in_dim, a.work);
  else
    hipLaunchKernelGGL((w8_tokens<T, 16, 1024>), dim3(w8_tiles(a.n_tok)), dim3(1024), 0, st, (const T*)a.x, a.x_stride, a.n_tok, a.in_dim, a.work);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (w8_rows_takes(a)) return launch_w8_rows(type, a, st);
  const bool big = a.n_tok > 512;
  if (a.up) return big ? gemm_go<T, 2, 4, 8, 4, true>(a, st) : gemm_go<T, 2, 2, 4, 4, true>(a, st);
  return big ? gemm_go<T, 2, 4, 8, 4, false>(a, st) : gemm_go<T, 2, 2, 4, 4, false>(a, st);
}

hipError_t launch_w8(int type, const W8Args& a, hipStream_t st) {
  if (type == ACT_F32) return w8_typed<float>(type, a, st);
  if (type == ACT_F16) return w8_typed<_Float16>(type, a, st);
  return w8_typed<bf16_t>(type, a, st);
}

}  // namespace kq
