// kv4_keep.hip -- the accepted rows of a tree moved together in the 4-bit
// cache: slot base + i takes what slot base + path[i] holds, base being the
// slot of the sequence's row 0.
//
// A workgroup per kv head and sequence takes the blocks of 32 new slots in
// ascending order: it reads all that a block will hold, waits, and writes.
// The path ascends, path[i] >= i, so what later blocks take lies behind what
// has been written.  A value dword and the 16 bytes of its scales hold eight
// tokens, each from its old place or, if it stays, from its own.  The codes
// and scales are moved as they are: nothing is rounded again.
// Bound by waiting (84% of wave time): a page id, a path entry and a word one
// after the other, then the next block.  8 rows of one sequence 5 us, 32
// sequences of up to 26 rows (8 kv heads of 128) 9 us.
#include "kv4.h"
#include "tree.h"

namespace kq {

template <int D>
__global__ __launch_bounds__(256) void kv4_keep(Kv4View c, Kv4Rows rows, const int* path, const int* count) {
  using L = Kv4L<D>;
  constexpr int NG = L::NG;
  typedef uint32_t Quad __attribute__((ext_vector_type(L::QG)));
  __shared__ const uint8_t* from[32];  // the block that a new slot's token is in (or any memory of ours, unused)
  __shared__ int slot[32];             // its slot there, -1: it stays, -2: its page is missing
  __shared__ int good;
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const Kv4Span sp = kv4_span(rows, b);
  const int n = sp.r1 - sp.r0, base = sp.len - n;
  const int* const p = path + sp.r0;
  // The rows that are kept: up to the first entry that does not ascend within
  // the sequence.  What is where it was already is not moved.
  const int asked = min(max(count[b], 0), n);
  if (tid == 0) good = asked;
  __syncthreads();
  int first = asked;
  for (int i = tid; i < asked; i += 256) {
    const int v = p[i], before = i ? p[i - 1] : -1;
    if (v <= before || v >= n) atomicMin(&good, i);
    if (v != i) first = min(first, i);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
  __shared__ int firsts[4];
  if ((tid & 63) == 0) firsts[tid >> 6] = first;
  __syncthreads();
  const int kept = good;
  first = min(min(firsts[0], firsts[1]), min(firsts[2], firsts[3]));
  const int s0 = max(base + first, 0), s1 = min(base + kept, min(sp.len, c.max_pages * KV4_PAGE));
  for (int at = s0 & ~31; at < s1; at += 32) {
    uint8_t* const to = kv4_block(c, b, at / KV4_PAGE, hk, L::BYTES);
    const int h = at & 32;  // the block's first slot in its page
    __syncthreads();        // the last block is written, its table no longer read
    if (tid < 32) {
      const int s = at + tid;
      const bool moves = s >= s0 && s < s1 && p[s - base] != s - base;
      const int f = moves ? base + p[s - base] : s;
      const uint8_t* src = moves && f >= 0 ? kv4_block(c, b, f / KV4_PAGE, hk, L::BYTES) : nullptr;
      from[tid] = src ? src : to ? to : c.pages;
      slot[tid] = !moves ? -1 : src ? f % KV4_PAGE : -2;
    }
    __syncthreads();
    if (!to) continue;
    // Token t of the block: its slot in from[t], and whether it comes from a page.
    auto old = [&](int t) { return slot[t] == -1 ? h + t : max(slot[t], 0); };
    // Key codes: token, lane group, quad.
    const int kt = tid & 31, kg = (tid >> 5) & 3, kq = (tid >> 7) * L::QG;
    Quad key = 0, scale = 0;
    if (kq < NG) key = *reinterpret_cast<const Quad*>(from[kt] + L::key_word(old(kt), kq, kg));
    // Key scales of a token: NG dwords, steps and then minima.
    const int sc = tid >> 5;
    if (sc < NG / L::QG) scale = *reinterpret_cast<const Quad*>(from[kt] + L::key_d(old(kt), 0) + 4 * L::QG * sc);
    // Value dwords, four dims (16 apart) together.
    const int rg = (tid >> 4) & 3, dim = 64 * (tid >> 6) + (tid & 15);
    kvu4 value = {0, 0, 0, 0};
    if (tid < D) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = 16 * (j >> 2) + 4 * rg + (j & 3), f = old(t);
        const kvu4 w = *reinterpret_cast<const kvu4*>(from[t] + L::value_word(f, dim));
        const uint32_t fj = (uint32_t)L::value_j(f), four = slot[t] == -2 ? 0u : 15u;
        // kv4_bit of a run-time j: 6, 22, 2, 18, 14, 30, 10, 26.
        const uint32_t bit = ((fj & 1) << 4) + ((0xAE26u >> ((fj >> 1) << 2)) & 15u);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t word = w[k], code = __builtin_amdgcn_alignbit(word, word, bit) & four;
          value[k] |= __builtin_amdgcn_alignbit(code, code, (uint32_t)((32 - kv4_bit(j)) & 31));
        }
      }
    }
    // Value scales: group, step or minimum, lane group.
    const int vr = tid & 3, vg = (tid >> 2) % NG, vm = (tid / (4 * NG)) & 1;
    uint16_t half[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) half[j] = 0;
    if (tid < 8 * NG) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = 16 * (j >> 2) + 4 * vr + (j & 3);
        if (slot[t] != -2) half[j] = *reinterpret_cast<const uint16_t*>(from[t] + L::value_d(old(t), vg) + 64 * NG * vm);
      }
    }
    __syncthreads();
    // A token whose page is missing reads as NaN from here on: key steps of
    // NaN, all else 0.
    if (kq < NG && slot[kt] != -1)
      *reinterpret_cast<Quad*>(to + L::key_word(h + kt, kq, kg)) = slot[kt] == -2 ? Quad(0) : key;
    if (sc < NG / L::QG && slot[kt] != -1) {
      if (slot[kt] == -2) {
#pragma unroll
        for (int k = 0; k < L::QG; ++k) scale[k] = L::QG * sc + k < NG / 2 ? 0x7E007E00u : 0u;
      }
      *reinterpret_cast<Quad*>(to + L::key_d(h + kt, 0) + 4 * L::QG * sc) = scale;
    }
    if (tid < D) *reinterpret_cast<kvu4*>(to + L::value_word(h + 4 * rg, dim)) = value;
    if (tid < 8 * NG) {
      kvu4 w;
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = half[2 * k] | (uint32_t)half[2 * k + 1] << 16;
      *reinterpret_cast<kvu4*>(to + L::value_d(h + 4 * vr, vg) + 64 * NG * vm) = w;
    }
  }
}

hipError_t launch_kv4_keep(int head_dim, const Kv4View& c, const Kv4Rows& rows, const int* path, const int* count,
                           hipStream_t s) {
  const dim3 grid(c.n_kv, rows.n_seq);
  if (head_dim == 64) hipLaunchKernelGGL(kv4_keep<64>, grid, dim3(256), 0, s, c, rows, path, count);
  else if (head_dim == 128) hipLaunchKernelGGL(kv4_keep<128>, grid, dim3(256), 0, s, c, rows, path, count);
  else hipLaunchKernelGGL(kv4_keep<256>, grid, dim3(256), 0, s, c, rows, path, count);
  return hipGetLastError();
}

}  // namespace kq
