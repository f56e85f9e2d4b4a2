// tree.hip -- trees of drafted tokens: masks and positions from parents, and
// the greedy choice along a tree (contracts: include/aspidagpu.h).
//
// tree_accept: says(r) = the largest logit of row r, the lowest index among
// equals (NaN never is one).  From row 0 on, the next row is the first child
// whose token is what its parent says; where there is none, that is the next
// token.  tree_says finds each row's largest in pieces (memory bound: all
// logits are read once; 254 rows of 151936, bf16, 77 MB in 17 us, 4.5 TB/s),
// tree_walk joins the pieces of a sequence's rows and walks in LDS (2 to 4 us
// behind a launch: bound by waiting).
#include <algorithm>

#include "kq_common.h"
#include "kv4.h"
#include "tree.h"

namespace kq {

// A parent that is not an earlier row counts as none.
__device__ __forceinline__ int tree_parent(const int* parent, int i) {
  const int p = parent[i];
  return p >= 0 && p < i ? p : -1;
}

// A workgroup per sequence: parents in LDS, then a thread for each word of
// each row's mask climbs from the row until it is below the word's bits.
__global__ __launch_bounds__(256) void tree_masks(TreeRows t, int* pos, uint32_t* mask, int words) {
  __shared__ int16_t up[TREE_MAX_ROWS];
  const int b = blockIdx.x, tid = threadIdx.x;
  const Kv4Span sp = kv4_span({t.row_start, t.kv_len, t.n_rows, t.n_seq}, b);
  const int n = sp.r1 - sp.r0, m = min(n, TREE_MAX_ROWS);
  for (int i = tid; i < m; i += 256) up[i] = (int16_t)tree_parent(t.parent + sp.r0, i);
  __syncthreads();
  if (mask)
    for (long long x = tid; x < (long long)n * words; x += 256) {
      const int i = (int)(x / words), w = (int)(x % words);
      uint32_t bits = 0;
      for (int j = i < m ? i : -1; j >= 32 * w; j = up[j])
        if (j < 32 * w + 32) bits |= 1u << (j & 31);
      mask[(size_t)sp.r0 * words + x] = bits;
    }
  if (pos)
    for (int i = tid; i < n; i += 256) {
      int depth = 0;
      if (i < m)
        for (int j = up[i]; j >= 0; j = up[j]) ++depth;
      pos[sp.r0 + i] = sp.len - n + depth;
    }
}

hipError_t launch_tree(const TreeRows& t, int* pos, uint32_t* mask, int words, hipStream_t s) {
  hipLaunchKernelGGL(tree_masks, dim3(t.n_seq), dim3(256), 0, s, t, pos, mask, words);
  return hipGetLastError();
}

struct Said { float v; int i; };  // a piece's largest logit and its index; INT_MAX: none

__device__ __forceinline__ void say(Said& s, float v, int i) {
  if (v > s.v || (v == s.v && i < s.i)) s = {v, i};
}

// 256 threads take elements [piece, piece + 1) * len of a row, eight
// consecutive ones each in turn.
template <class T>
__global__ __launch_bounds__(256) void tree_says(const T* logits, long long stride, int vocab, int pieces, int len,
                                                 Said* out) {
  __shared__ Said part[4];
  const int row = blockIdx.x / pieces, piece = blockIdx.x % pieces, tid = threadIdx.x;
  const T* const x = logits + (long long)row * stride;
  const int i0 = piece * len, i1 = (int)min((long long)vocab, (long long)i0 + len);
  Said s = {-INFINITY, 0x7FFFFFFF};
#pragma unroll 4
  for (int i = i0 + 8 * tid; i + 8 <= i1; i += 8 * 256) {
    struct { T t[8]; } r;
    __builtin_memcpy(&r, x + i, sizeof(r));
#pragma unroll
    for (int j = 0; j < 8; ++j) say(s, (float)r.t[j], i + j);
  }
  const int rest = i0 + (i1 - i0) / 8 * 8 + tid;
  if (rest < i1) say(s, (float)x[rest], rest);
  wave_argmax(s.v, s.i);
  if ((tid & 63) == 0) part[tid >> 6] = s;
  __syncthreads();
  if (tid) return;
  for (int w = 1; w < 4; ++w) say(s, part[w].v, part[w].i);
  out[(size_t)row * pieces + piece] = s;
}

// What a row says as a number that is larger for a larger logit, then for a
// lower index; 0: nothing.
__device__ __forceinline__ unsigned long long said_key(const Said& s) {
  if (s.i == 0x7FFFFFFF) return 0;
  const uint32_t u = __float_as_uint(s.v + 0.f);  // (-0 is 0)
  return (unsigned long long)(u >> 31 ? ~u : u | 0x80000000u) << 32 | (uint32_t)~s.i;
}
__device__ __forceinline__ int said_token(unsigned long long key) { return key ? ~(int)(uint32_t)key : -1; }

// A workgroup per sequence: every piece's key to its row's, every row that its
// parent says to the parent's next, and a thread follows those.  (Atomics on
// LDS whose result does not depend on their order.)
__global__ __launch_bounds__(256) void tree_walk(TreeRows t, TreeAccept a, int pieces, int cap) {
  extern __shared__ unsigned long long lds[];  // key and next row of up to cap rows
  __shared__ int ends[2];                      // rows of the path, what the last one says
  unsigned long long* const says = lds;
  int* const next = (int*)(lds + cap);
  const int b = blockIdx.x, tid = threadIdx.x;
  const Kv4Span sp = kv4_span({t.row_start, t.kv_len, t.n_rows, t.n_seq}, b);
  const int n = sp.r1 - sp.r0, m = min(n, cap);
  const Said* const in = (const Said*)a.work + (size_t)sp.r0 * pieces;
  const int total = m * pieces;  // at most 4096
  Said u = {0.f, 0x7FFFFFFF};
  int up = -1, token = -1;
  if (tid < total) u = in[tid];
  if (tid < m) {
    up = tree_parent(t.parent + sp.r0, tid);
    token = a.token[sp.r0 + tid];
  }
  for (int i = tid; i < m; i += 256) {
    says[i] = 0;
    next[i] = m;
  }
  __syncthreads();
  for (int x = tid; x < total;) {
    atomicMax(&says[x / pieces], said_key(u));
    x += 256;
    if (x < total) u = in[x];
  }
  __syncthreads();
  for (int i = tid; i < m;) {
    if (up >= 0 && token >= 0 && token == said_token(says[up])) atomicMin(&next[up], i);
    i += 256;
    if (i < m) {
      up = tree_parent(t.parent + sp.r0, i);
      token = a.token[sp.r0 + i];
    }
  }
  __syncthreads();
  if (tid == 0) {
    int count = 0, last = 0;
    for (int at = 0; at < m; at = next[at]) {
      a.path[sp.r0 + count++] = at;
      last = at;
    }
    ends[0] = count;
    ends[1] = m > 0 ? said_token(says[last]) : -1;
  }
  __syncthreads();
  const int count = ends[0];
  for (int i = count + tid; i < n; i += 256) a.path[sp.r0 + i] = -1;
  if (tid == 0) {
    a.count[b] = count;
    a.next[b] = ends[1];
    a.new_len[b] = max(sp.len - n + count, 0);
  }
}

// Pieces of a row, of 4096 elements at least: 2048 workgroups in all at most,
// which is what fits at once (254 rows of 151936, bf16: in 9 pieces 21.1 us, in 8 19.8).
static int says_pieces(int n_rows, int vocab) {
  return (int)std::max<long long>(1, std::min<long long>(2048 / n_rows, (vocab + 4095) / 4096));
}

size_t tree_accept_work_bytes(int n_rows, int vocab) {
  return ((size_t)n_rows * says_pieces(n_rows, vocab) * sizeof(Said) + 255) / 256 * 256;
}

template <class T>
static void says_go(const TreeRows& t, const TreeAccept& a, int pieces, int len, hipStream_t s) {
  hipLaunchKernelGGL(tree_says<T>, dim3((unsigned)(t.n_rows * pieces)), dim3(256), 0, s, (const T*)a.logits, a.stride,
                     a.vocab, pieces, len, (Said*)a.work);
}

hipError_t launch_tree_accept(int type, const TreeRows& t, const TreeAccept& a, hipStream_t s) {
  const int pieces = says_pieces(t.n_rows, a.vocab);
  const int len = (a.vocab / 8 + pieces) / pieces * 8;  // whole runs of eight; pieces * len >= vocab
  if (type == ACT_F32) says_go<float>(t, a, pieces, len, s);
  else if (type == ACT_F16) says_go<_Float16>(t, a, pieces, len, s);
  else says_go<bf16_t>(t, a, pieces, len, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int cap = std::min(t.n_rows, TREE_MAX_ROWS);
  hipLaunchKernelGGL(tree_walk, dim3(t.n_seq), dim3(256), 12 * cap, s, t, a, pieces, cap);
  return hipGetLastError();
}

}  // namespace kq
