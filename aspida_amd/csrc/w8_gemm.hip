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
// instruction, into a ring of 4 to 20 of them; a wave reads the operands of
// stage s + 1 while it multiplies those of stage s, so a barrier (one a stage)
// finds matrix work in hand.  In a gated block a wave has as many row tiles of
// the gate as of the up projection, and forms their product in its registers.
// Bound by the matrix cores where tokens are many: 4001 tokens, 14336 inputs,
// 4096 rows 213 us (codes 17 more), 2200 TOP/s; gated, 2001 tokens, 4096
// inputs, twice 14336 rows 204 us, 2300; an 8192^3 product of a library
// reaches 2079.  Bound by waiting where they are few: 60 tokens, 14336 inputs,
// 4096 rows 16 us, 3.7 TB/s of the weights.
#include <algorithm>

#include "kq_common.h"
#include "w8.h"
#include "w8_kernels.h"

namespace kq {

// ---- tokens' codes -------------------------------------------------------------

// A workgroup takes TOK tokens, KEEP runs of 16 values a thread at a time: rows
// of up to 16 KEEP THREADS / TOK values stay in registers between the pass
// that finds the scale and the one that writes codes, longer ones are read
// again.  The loads of a turn leave together: runs past the end are the last
// whole one again.  The run that in_dim ends in, if it does, is a turn of its own.
template <class T, int TOK, int THREADS, int KEEP>
__global__ __launch_bounds__(THREADS) void w8_tokens(const T* x, long long stride, int n_tok, int in_dim, uint8_t* work) {
  constexpr int RUNS = THREADS / TOK, STEP = 16 * KEEP * RUNS;
  __shared__ uint32_t part[TOK][THREADS / 64];
  const int tid = threadIdx.x, blocks = w8_blocks(in_dim);
  const int t = tid % TOK, run = tid / TOK, first = __builtin_amdgcn_readfirstlane(run);  // (the wave's first)
  const int row = blockIdx.x * TOK + t;
  const T* const from = x + (long long)min(row, n_tok - 1) * stride;
  const int whole = in_dim & ~15;
  const bool last = in_dim > whole && run == (whole >> 4) % RUNS;
  W8Run<T> v[KEEP], rest;
  uint32_t top = 0;
  if (last) {
    rest = w8_rest(from + whole, in_dim - whole);
    top = w8_top16(rest, top);
  }
  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i) v[i] = w8_run(from + min(k0 + 16 * (run + i * RUNS), whole - 16));
  };
  for (int k0 = 0; k0 + 16 * first < whole; k0 += STEP) {
    load(k0);
#pragma unroll
    for (int i = 0; i < KEEP; ++i) top = w8_top16(v[i], top);
  }
  if constexpr (TOK == 1) {
    top = w8_group_max<THREADS / 64>(top, part[0]);
  } else {
#pragma unroll
    for (int o = TOK; o < 64; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if ((tid & 63) < TOK) part[t][tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) top = max(top, part[t][i]);
  }
  if (row >= n_tok) return;
  const W8Scale s(__builtin_bit_cast(float, top));
  if (run == 0) w8_scales(work, in_dim, n_tok)[row] = s.s;
  for (int k0 = 0; k0 + 16 * first < whole; k0 += STEP) {
    if (STEP < whole) load(k0);
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      if (k0 + 16 * (first + i * RUNS) >= whole) break;
      const uint4 c = w8_codes16(v[i], s);
      const int k = k0 + 16 * (run + i * RUNS);
      if (k < whole) *reinterpret_cast<uint4*>(work + w8_place(row, k, blocks)) = c;
    }
  }
  if (last) *reinterpret_cast<uint4*>(work + w8_place(row, whole, blocks)) = w8_codes16(rest, s);
}

// ---- products --------------------------------------------------------------------

// At most N of this wave's loads outstanding, then the workgroup's barrier.
template <int N> __device__ __forceinline__ void w8_wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

// WR x WT waves, each AR row tiles (of a gated block: AR / 2 of the gate, AR /
// 2 of the up projection) by BT token tiles.
template <class T, int WR, int WT, int AR, int BT, int RING, bool GATED>
__global__ __launch_bounds__(64 * WR * WT, WR * WT >= 8 ? 2 : 1) void w8_gemm(W8Args a) {
  constexpr int W = WR * WT, NA = WR * AR, NB = WT * BT, PER = (NA + NB) / W, STAGE = (NA + NB) * W8_TILE;
  constexpr int OUTS = GATED ? AR / 2 : AR;  // row tiles of the result a wave
  static_assert((NA + NB) % W == 0);
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
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
  // `to` and `slot`: byte offsets of ring slots.
  auto fetch = [&](int s, int to, int i) {
    w8_to_lds<0>(from[i], lane * 16, min(s, blocks - 1) * W8_TILE, base + to + (wave * PER + i) * W8_TILE);
  };
  auto after = [](int slot) { return slot == (RING - 1) * STAGE ? 0 : slot + STAGE; };
  const uint8_t* const la = lds + (wr * AR) * W8_TILE + lane * 16;
  const uint8_t* const lb = lds + (NA + wt * BT) * W8_TILE + lane * 16;
  auto operand = [](const uint8_t* p, int slot, int i) { return *reinterpret_cast<const w8i4*>(p + slot + i * W8_TILE); };
  w8i4 acc[AR][BT], ra[AR], rb[2][BT];
#pragma unroll
  for (int i = 0; i < AR; ++i)
#pragma unroll
    for (int j = 0; j < BT; ++j) acc[i][j] = w8i4{0, 0, 0, 0};
  // Stage s + RING - 1 goes where s - 1 was, whose operands every wave has
  // multiplied, and so has read, before the barrier of step s.  Past the end
  // the last stage is loaded again.  A row tile's operand is replaced by the
  // next stage's as soon as it is used.
  int next_slot = STAGE, free_slot = (RING - 1) * STAGE;  // of stages s + 1 and s + RING - 1
  auto step = [&](int s, const w8i4 (&b)[BT], w8i4 (&next)[BT]) {
    constexpr int HEAD = AR == 1 ? 0 : AR / 4 > 0 ? AR / 4 : 1, REST = AR - HEAD;
#pragma unroll
    for (int i = 0; i < AR; ++i) {
      if (i == HEAD) w8_wait_barrier<PER * (RING - 3)>();
#pragma unroll
      for (int j = 0; j < BT; ++j) acc[i][j] = w8_mfma(ra[i], b[j], acc[i][j]);
      if (i >= HEAD) {
        const int k = i - HEAD;
        if (k == 0) {
#pragma unroll
          for (int h = 0; h < HEAD; ++h) ra[h] = operand(la, next_slot, h);
        }
        ra[i] = operand(la, next_slot, i);
#pragma unroll
        for (int j = k * BT / REST; j < (k + 1) * BT / REST; ++j) next[j] = operand(lb, next_slot, j);
#pragma unroll
        for (int j = k * PER / REST; j < (k + 1) * PER / REST; ++j) fetch(s + RING - 1, free_slot, j);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    next_slot = after(next_slot);
    free_slot = after(free_slot);
  };
#pragma unroll
  for (int s = 0; s < RING - 1; ++s)
#pragma unroll
    for (int i = 0; i < PER; ++i) fetch(s, s * STAGE, i);
  w8_wait_barrier<PER * (RING - 2)>();
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
  float units[BT];
#pragma unroll
  for (int j = 0; j < BT; ++j) units[j] = sx[min((bt0 + wt * BT + j) * 16 + (lane & 15), a.n_tok - 1)];
#pragma unroll
  for (int i = 0; i < OUTS; ++i) {
    const int o = (br0 + wr * OUTS + i) * 16 + 4 * (lane >> 4);
    if (o >= a.out_dim) continue;
    const W8Rows<GATED> rows(a, o);
#pragma unroll
    for (int j = 0; j < BT; ++j) {
      const int t = (bt0 + wt * BT + j) * 16 + (lane & 15);
      if (t < a.n_tok) rows.template finish<T>(a, t, o, acc[i][j], acc[i + (GATED ? OUTS : 0)][j], W8Unit(units[j]));
    }
  }
}

template <class T, int WR, int WT, int AR, int BT, int RING, bool GATED>
static hipError_t gemm_go(const W8Args& a, hipStream_t st) {
  constexpr int ring = RING * (WR * AR + WT * BT) * W8_TILE;
  auto* k = &w8_gemm<T, WR, WT, AR, BT, RING, GATED>;
  const int outs = WR * (GATED ? AR / 2 : AR);
  const long long total = (long long)((w8_tiles(a.out_dim) + outs - 1) / outs) * ((w8_tiles(a.n_tok) + WT * BT - 1) / (WT * BT));
  const int lds = w8_spread(ring, (int)std::min(total, 1ll << 30), 160 * 1024 / ring);
  const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3((unsigned)((total + 7) / 8 * 8)), dim3(64 * WR * WT), lds, st, a);
  return hipGetLastError();
}

// A token a workgroup, or four (64 bytes of a tile's line are written
// together): from 2048 tokens on the latter is faster (bf16, 4096 inputs:
// 1024 tokens 8.3 against 11.3 us, 2001 11.9 and 12.8, 4001 21.3 and 17.5;
// 14336 inputs: 2001 31.6 and 32.4, 4001 56.8 and 49.2).  Wide rows of tokens
// that do not fill the card have four times the threads (product with 1024
// rows, bf16, 14336 inputs, 256 and 1024 threads: 60 tokens 21.9 and 19.8 us,
// 256 tokens 23.9 and 21.6, 512 tokens 31.9 and 33.2).
template <class T> static void launch_tokens(const W8Args& a, hipStream_t st) {
  auto go = [&](auto* k, int tok, int threads = 256) {
    hipLaunchKernelGGL(k, dim3((a.n_tok + tok - 1) / tok), dim3(threads), 0, st, (const T*)a.x, a.x_stride, a.n_tok, a.in_dim, a.work);
  };
  if (a.n_tok >= 2048) go(&w8_tokens<T, 4, 256, 8 / (int)sizeof(T) == 4 ? 2 : 4>, 4);
  else if (a.in_dim <= 4096) go(&w8_tokens<T, 1, 256, 1>, 1);
  else if (a.n_tok <= 256) go(&w8_tokens<T, 1, 1024, 1>, 1, 1024);
  else go(&w8_tokens<T, 1, 256, 4>, 1);
}

// Tiles that a workgroup takes, its ring, how many fit on a compute unit, and
// what a stage of 64 k takes (us) with one and with as many as fit on every
// compute unit, from products of 129 to 4001 tokens with 1024 to 14336 rows
// (bf16): e.g. 4096 inputs and rows, 512 tokens: 53.7, 34.7, 27.3, 22.2 and
// 22.4 us from the first form to the fifth, 4001 tokens: 78, 89, 92, 104 and
// 121; 16 tokens: the last 10, the fifth 12.
struct W8Form { int rows, toks, room; float one, full; };
constexpr W8Form W8_FORMS[] = {{16, 16, 1, .80f, .80f}, {8, 16, 1, .55f, .55f}, {8, 8, 2, .29f, .53f},
                               {4, 8, 2, .20f, .335f},  {4, 4, 2, .14f, .21f},  {2, 2, 2, .085f, .15f}};

// The form whose rounds of workgroups take least; `both`: a gated block has
// half the rows to a workgroup.
static int w8_form(const W8Args& a) {
  int best = 0;
  float least = 0.f;
  for (int f = 0; f < (int)(sizeof(W8_FORMS) / sizeof(W8_FORMS[0])); ++f) {
    const W8Form& w = W8_FORMS[f];
    const int rows = a.up ? w.rows / 2 : w.rows;
    const long long groups = (long long)((w8_tiles(a.out_dim) + rows - 1) / rows) * ((w8_tiles(a.n_tok) + w.toks - 1) / w.toks);
    const long long fit = 256 * w.room, whole = groups / fit, rest = groups % fit;
    const float stage = (float)whole * w.full + (rest == 0 ? 0.f : rest > 256 ? w.full : whole ? .75f * w.full : w.one);
    const float us = stage * (float)w8_blocks(a.in_dim) + 2.f * (float)(whole + (rest > 0));
    if (f == 0 || us < least) { best = f; least = us; }
  }
  return best;
}

template <class T, bool GATED> static hipError_t gemm_typed(const W8Args& a, hipStream_t st) {
  switch (w8_form(a)) {
    case 0: return gemm_go<T, 2, 4, 8, 4, 4, GATED>(a, st);
    case 1: return gemm_go<T, 2, 4, 4, 4, 6, GATED>(a, st);
    case 2: return gemm_go<T, 2, 2, 4, 4, 5, GATED>(a, st);
    case 3: return gemm_go<T, 2, 2, 2, 4, 6, GATED>(a, st);
    case 4: return gemm_go<T, 2, 2, 2, 2, 10, GATED>(a, st);
    default:
      if constexpr (GATED) return gemm_go<T, 1, 2, 2, 1, 20, true>(a, st);
      else return gemm_go<T, 2, 2, 1, 1, 20, false>(a, st);
  }
}

template <class T> static hipError_t w8_typed(int type, const W8Args& a, hipStream_t st) {
  if (w8_rows_fuse(a)) return launch_w8_rows(type, a, st);
  launch_tokens<T>(a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (w8_rows_takes(a)) return launch_w8_rows(type, a, st);
  return a.up ? gemm_typed<T, true>(a, st) : gemm_typed<T, false>(a, st);
}

hipError_t launch_w8(int type, const W8Args& a, hipStream_t st) {
  if (type == ACT_F32) return w8_typed<float>(type, a, st);
  if (type == ACT_F16) return w8_typed<_Float16>(type, a, st);
  return w8_typed<bf16_t>(type, a, st);
}

}  // namespace kq
