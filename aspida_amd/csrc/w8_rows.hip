// w8_rows.hip -- products of few tokens (up to 32) with 8-bit integer
// weights, plain and gated (the format and formulas: w8.h, w8_gemm.hip).
//
// A workgroup takes tiles of 16 rows (of a gated block one of the gate and the
// same of the up projection), one after the other, with all tokens, 16 to a
// column tile; its four waves share k, a block of 64 in turn.  Each wave
// streams its blocks through a ring of its own in LDS by loads that bypass the
// registers, so that 64 KB and more of a compute unit are on their way at any
// time, over the ends of tiles too, and no wave waits for another but to add
// up a tile: int32 sums, by LDS atomics (any order gives the same).  The few
// tokens of a decode step are quantised by every workgroup for itself while
// its first weights are on their way (FUSED), which saves a launch; the codes
// of more go through the ring, from L2.
// Bound by the weights' bytes: 4096 x 4096 weights and one token 6.7 us, 2.5
// TB/s with the launch; twice 14336 x 4096, gated, 18.5 us, 6.3 TB/s (in part
// from the memory-side cache).
#include <algorithm>

#include "kq_common.h"
#include "w8.h"
#include "w8_kernels.h"

namespace kq {

constexpr int W8R_WAVES = 4;
constexpr int W8R_TURN = 16 * 64 * W8R_WAVES;  // activations that the threads quantise at a time, 16 each
constexpr int W8R_KEEP = 8;                    // turns at most (FUSED)

// Ring depth by tiles of weights and of tokens a block: LDS for two workgroups
// a compute unit.
template <int NP, int BT, bool FUSED> struct W8Ring {
  static constexpr int PER = NP + (FUSED ? 0 : BT);  // loads of a block
  static constexpr int DEPTH = FUSED ? (NP == 1 ? 11 : 5) : PER == 2 ? 9 : PER == 3 ? 6 : 4;
  static constexpr int SUMS = 2 * NP * BT * 1024;    // of a tile, and of the next
  static constexpr int RING = W8R_WAVES * DEPTH * PER * W8_TILE;
};

template <int N> __device__ __forceinline__ void w8_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// The wave's LDS accesses are done, then the workgroup's barrier (loads to
// LDS stay on their way).
__device__ __forceinline__ void w8_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Sums in LDS, [4][64] dwords, lane's from byte `at` on.  (For its own writes
// to LDS the compiler waits for every load on its way there; so these are
// written here, behind the wait that reading a matrix result takes.)
__device__ __forceinline__ void w8_lds_add(uint32_t at, w8i4 v) {
  asm volatile(
      "s_nop 15\n\ts_nop 15\n\tds_add_u32 %0, %1\n\tds_add_u32 %0, %2 offset:256\n\tds_add_u32 %0, %3 offset:512\n\t"
      "ds_add_u32 %0, %4 offset:768" ::"v"(at), "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]) : "memory");
}
__device__ __forceinline__ void w8_lds_zero(uint32_t at) {
  asm volatile("ds_write_b32 %0, %1\n\tds_write_b32 %0, %1 offset:256\n\tds_write_b32 %0, %1 offset:512\n\t"
               "ds_write_b32 %0, %1 offset:768" ::"v"(at), "v"(0) : "memory");
}

// FUSED: how many turns it takes to quantise the tokens, 0 where they are.
template <class T, int BT, bool GATED, int FUSED>
__global__ __launch_bounds__(64 * W8R_WAVES, 2) void w8_rows(W8Args a) {
  constexpr int NP = GATED ? 2 : 1;
  using R = W8Ring<NP, BT, (FUSED > 0)>;
  constexpr int W = W8R_WAVES, D = R::DEPTH, PER = R::PER;
  // Rings, two buffers of sums, FUSED: codes [token][64 blocks].  (Behind other
  // variables, 16-byte accesses that are not aligned took half as long again.)
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  __shared__ uint32_t part[W];
  __shared__ float scale[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blocks = w8_blocks(a.in_dim), tiles = w8_tiles(a.out_dim), turns = (blocks + W - 1) / W, row = 64 * blocks;
  int* const sums = reinterpret_cast<int*>(lds + R::RING);
  uint8_t* const codes = lds + R::RING + R::SUMS;
  const uint8_t* const ring = lds + wave * (D * PER * W8_TILE);
  const uint32_t ring_at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)ring;

  __amdgpu_buffer_rsrc_t x[BT];
#pragma unroll
  for (int j = 0; j < BT; ++j) x[j] = w8_buffer(a.work + (size_t)min(j, w8_tiles(a.n_tok) - 1) * blocks * W8_TILE);
  // The next block to load: turn `ahead` of tile `to_tile`.  Past the last
  // tile its blocks are loaded again.
  int to_tile = blockIdx.x, ahead = 0, to_slot = 0;
  __amdgpu_buffer_rsrc_t w[NP];
  auto open = [&] {
    const size_t at = (size_t)min(to_tile, tiles - 1) * blocks * W8_TILE;
    w[0] = w8_buffer(a.w + at);
    if constexpr (GATED) w[1] = w8_buffer(a.up + at);
  };
  open();
  auto fetch = [&] {
    const int off = min(wave + W * ahead, blocks - 1) * W8_TILE;
    const uint32_t to = ring_at + to_slot;
#pragma unroll
    for (int p = 0; p < NP; ++p) w8_to_lds<2>(w[p], lane * 16, off, to + p * W8_TILE);
    if constexpr (FUSED == 0) {
#pragma unroll
      for (int j = 0; j < BT; ++j) w8_to_lds<0>(x[j], lane * 16, off, to + (NP + j) * W8_TILE);
    }
    to_slot = to_slot == (D - 1) * PER * W8_TILE ? 0 : to_slot + PER * W8_TILE;
    if (++ahead == turns) {
      ahead = 0;
      to_tile += gridDim.x;
      open();
    }
  };
  // FUSED: all threads have the token, or half of them one of two.  Their
  // activations are asked for first, since loads arrive in order, and without
  // branches, which would wait for them (runs past the end are the last whole
  // one again; where there is none, memory of ours).
  const int share = FUSED && a.n_tok == 1 ? 64 * W : 32 * W;
  const int tok = (int)threadIdx.x / share, own = (int)threadIdx.x % share, whole = a.in_dim & ~15;
  const T* const from = (const T*)a.x + (long long)min(tok, a.n_tok - 1) * a.x_stride;
  const bool last = FUSED && a.in_dim > whole && own == (whole >> 4) % share;
  W8Run<T> v[FUSED ? FUSED : 1], rest;
  if constexpr (FUSED > 0) {
#pragma unroll
    for (int i = 0; i < FUSED; ++i)
      v[i] = w8_run(whole ? from + min(16 * (own + i * share), whole - 16) : reinterpret_cast<const T*>(a.work));
    if (last) rest = w8_rest(from + whole, a.in_dim - whole);
    __builtin_amdgcn_sched_barrier(0);
  }
  // This thread's token in the results (of the first BT waves).
  const int t = 16 * wave + (lane & 15);
  const float token_scale = FUSED ? 0.f : w8_scales(a.work, a.in_dim, a.n_tok)[min(t, a.n_tok - 1)];
#pragma unroll
  for (int d = 0; d < D; ++d) fetch();
  for (int i = threadIdx.x; i < R::SUMS / 4; i += 64 * W) sums[i] = 0;
  if constexpr (FUSED > 0) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < FUSED; ++i)
      if (whole) top = w8_top16(v[i], top);
    if (last) top = w8_top16(rest, top);
#pragma unroll
    for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if (lane == 0) part[wave] = top;
    w8_barrier();
    for (int i = 0; i < share / 64; ++i) top = max(top, part[tok * (share / 64) + i]);
    const W8Scale s(__builtin_bit_cast(float, top));
    if (tok < a.n_tok) {
      if (own == 0) scale[tok] = s.s;
#pragma unroll
      for (int i = 0; i < FUSED; ++i) {
        if (16 * i * share >= whole) break;
        const int k = 16 * (own + i * share);
        const uint4 c = w8_codes16(v[i], s);
        if (k < whole) *reinterpret_cast<uint4*>(codes + tok * row + k) = c;
      }
      if (last) *reinterpret_cast<uint4*>(codes + tok * row + whole) = w8_codes16(rest, s);
    }
  }
  w8_barrier();

  const uint32_t sums_at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) int*)sums;
  const W8Unit ux(FUSED ? scale[t & 1] : token_scale);
  int slot = 0, buf = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, buf ^= 1) {
    w8i4 acc[NP][BT];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int j = 0; j < BT; ++j) acc[p][j] = w8i4{0, 0, 0, 0};
    for (int i = 0; i < turns; ++i) {
      const int kb = wave + W * i;
      w8_wait<(D - 1) * PER>();
      w8i4 f[NP], g[BT];
#pragma unroll
      for (int p = 0; p < NP; ++p) f[p] = *reinterpret_cast<const w8i4*>(ring + slot + p * W8_TILE + lane * 16);
#pragma unroll
      for (int j = 0; j < BT; ++j)
        g[j] = FUSED ? *reinterpret_cast<const w8i4*>(codes + min(lane & 15, a.n_tok - 1) * row + min(kb, blocks - 1) * 64 + (lane >> 4) * 16)
                     : *reinterpret_cast<const w8i4*>(ring + slot + (NP + j) * W8_TILE + lane * 16);
      // Read before its place is loaded anew.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      fetch();
      slot = slot == (D - 1) * PER * W8_TILE ? 0 : slot + PER * W8_TILE;
      if (kb < blocks) {
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int j = 0; j < BT; ++j) acc[p][j] = w8_mfma(f[p], g[j], acc[p][j]);
      }
    }
    // Sums [product][token tile][lane] of four rows, of one tile and the next in
    // turn: one is added up while the other is read and cleared.
    const uint32_t to = sums_at + buf * (NP * BT * 1024) + lane * 4;
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int j = 0; j < BT; ++j)
        if (16 * j + (lane & 15) < a.n_tok) w8_lds_add(to + (p * BT + j) * 1024, acc[p][j]);
    w8_barrier();
    if (wave < BT) {
      w8i4 sum[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int* const at = sums + (buf * NP * BT + p * BT + wave) * 256 + lane;
        sum[p] = w8i4{at[0], at[64], at[128], at[192]};
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int p = 0; p < NP; ++p) w8_lds_zero(to + (p * BT + wave) * 1024);
      const int o = 16 * tile + 4 * (lane >> 4);
      const W8Rows<GATED> rows(a, tile, lane >> 4);
      if (t < a.n_tok && o < a.out_dim) rows.template finish<T>(a, t, o, sum[0], sum[NP - 1], ux);
    }
  }
  w8_wait<0>();  // nothing is on its way to LDS when the workgroup ends
}

template <class T, int BT, bool GATED, int FUSED>
static hipError_t rows_go(const W8Args& a, hipStream_t st) {
  using R = W8Ring<GATED ? 2 : 1, BT, (FUSED > 0)>;
  // As many workgroups as fit at once, with equal shares of the tiles.
  const int tiles = w8_tiles(a.out_dim), room = 512, each = (tiles + room - 1) / room;
  const int groups = (tiles + each - 1) / each;
  const int lds = w8_spread(R::RING + R::SUMS + (FUSED ? a.n_tok * 64 * w8_blocks(a.in_dim) : 0), groups, 2);
  auto* k = &w8_rows<T, BT, GATED, FUSED>;
  const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(groups), dim3(64 * W8R_WAVES), lds, st, a);
  return hipGetLastError();
}

static int w8_rows_turns(const W8Args& a) { return (int)(((long long)a.n_tok * a.in_dim + W8R_TURN - 1) / W8R_TURN); }
// A launch for the codes against codes found by every workgroup (bf16, 4096
// inputs; 4096 rows: 1 token 10.2 and 7.6 us, 2 tokens 9.8 and 8.9, 4 tokens
// 9.9 and 10.5; 14336 rows: 16.5 and 12.7, 16.4 and 14.1, 16.4 and 17.2).
bool w8_rows_fuse(const W8Args& a) { return a.n_tok <= 2 && w8_rows_turns(a) <= W8R_KEEP; }
// Besides, long rows of few outputs, of which the tile kernel's workgroups
// would be too few (bf16, 14336 inputs, 4096 rows: 16 tokens 19.9 here, 24.4
// there; 32 tokens 24.0 and 28.1; 60: 29.9 and 29.0; 8192 inputs and rows, 16
// tokens: 20.5 and 19.5; 4096 inputs, 14336 rows: 18.3 and 16.6).
bool w8_rows_takes(const W8Args& a) {
  return w8_rows_fuse(a) || (a.n_tok <= 32 && a.out_dim <= 6144 && a.in_dim >= 8192);
}

template <class T, bool GATED> static hipError_t rows_typed(const W8Args& a, hipStream_t st) {
  if (w8_rows_fuse(a)) {
    const int turns = w8_rows_turns(a);
    return turns <= 1 ? rows_go<T, 1, GATED, 1>(a, st) : turns <= 4 ? rows_go<T, 1, GATED, 4>(a, st) : rows_go<T, 1, GATED, W8R_KEEP>(a, st);
  }
  return a.n_tok <= 16 ? rows_go<T, 1, GATED, 0>(a, st) : rows_go<T, 2, GATED, 0>(a, st);
}

hipError_t launch_w8_rows(int type, const W8Args& a, hipStream_t st) {
  if (type == ACT_F32) return a.up ? rows_typed<float, true>(a, st) : rows_typed<float, false>(a, st);
  if (type == ACT_F16) return a.up ? rows_typed<_Float16, true>(a, st) : rows_typed<_Float16, false>(a, st);
  return a.up ? rows_typed<bf16_t, true>(a, st) : rows_typed<bf16_t, false>(a, st);
}

}  // namespace kq
