// kv4.h -- the paged 4-bit key/value cache: layout and launchers.
//
// A page holds KV4_PAGE = 64 slots; per kv head it is a block of 80 D bytes
// (D = head_dim, 64, 128 or 256; NG = D / 32 groups):
//   key codes    32 D  [tile of 16 tokens][group quad][lane 64][group of quad]
//                      dwords; lane = 16 kg + token, dims 32 group + 8 kg + j
//   value codes  32 D  [block of 32 tokens][64 dims][lane 64][dim / 16 % 4]
//                      dwords; lane = 16 rg + dim % 16, code j = token
//                      16 (j / 4) + 4 rg + j % 4
//   key scales    8 D  [token][d of NG groups, m of NG groups] f16
//   value scales  8 D  [block of 32][d, then m][group][rg][j] f16
// (a head of 64 has one "quad" of two groups).  A code q stands for d q + m.
//
// Why this form:
//   * the dwords lie as the 16x16x32 matrix instructions take their operands
//     (8 consecutive k values per lane), so a wave's loads are whole lines of
//     16 bytes per lane with nothing to transpose: keys run over dims, values
//     over tokens;
//   * code j sits at bit kv4_bit(j) of its dword: with the bits of 16.0 or
//     256.0 or'ed in, two codes become the f16 pair 16 + q (or 256 + q) after
//     a mask alone (a rotation by 8 once per dword for the other four);
//   * d has 7 significant bits, so d q (11 bits) is exact in f16: one f16
//     operand carries the code part of a key or value without loss, and the
//     m part goes through the matrix cores as one more operand.  255.875 d
//     must stay finite: d <= 254.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "rope.h"

namespace kq {

constexpr int KV4_PAGE = 64;
constexpr float KV4_D_MAX = 254.f;

__host__ __device__ constexpr int kv4_head_bytes(int head_dim) { return 80 * head_dim; }
__host__ __device__ constexpr int kv4_bit(int j) {
  return (((j & 1) << 4) + ((j >> 1) == 0 ? 6 : (j >> 1) == 1 ? 2 : (j >> 1) == 2 ? 14 : 10)) & 31;
}

// A cache as the kernels see it.
struct Kv4View {
  uint8_t* pages;
  const int* table;  // [n_seq][max_pages]
  int n_kv, n_pages, max_pages;
};

// Rows of new tokens (queries, or keys and values): sequence b's rows are
// row_start[b] .. row_start[b + 1] - 1, or row b alone where row_start is
// null; its last row is the token at slot kv_len[b] - 1.
struct Kv4Rows {
  const int* row_start;
  const int* kv_len;
  int n_rows, n_seq;
};

hipError_t launch_kv4_append(int head_dim, const Kv4View& c, int type, const void* k, long long k_stride,
                             const void* v, long long v_stride, const Kv4Rows& rows, const RopeTable* rope,
                             const int* pos, hipStream_t s);
hipError_t launch_kv4_read(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, void* k, long long k_stride,
                           void* v, long long v_stride, hipStream_t s);

struct Kv4Attn {
  const void* q;
  long long q_stride;
  void* out;
  long long out_stride;
  float* lse;  // [n_rows][n_heads] or null
  void* work;
  int n_heads, max_rows, window;
  float scale;
};
size_t kv4_attn_work_bytes(int head_dim);
hipError_t launch_kv4_attn(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Attn& a,
                           hipStream_t s);

// Attention of many rows (kv4_prefill.hip), without a workspace.
bool kv4_prefill_takes(const Kv4View& c, const Kv4Rows& rows, const Kv4Attn& a);
hipError_t launch_kv4_prefill(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Attn& a,
                              hipStream_t s);

struct Kv4Weigh {
  const void* q;
  long long q_stride;
  const float* lse;      // [n_rows][n_heads]
  const float* acc_in;   // [n_seq][n_kv][acc_stride], null = zeros
  float* acc_out;
  long long acc_stride;
  int n_heads, max_rows, window;
  float scale;
};
hipError_t launch_kv4_weigh(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Weigh& w,
                            hipStream_t s);

struct Kv4Evict {
  const int* kv_len;
  const float* acc;  // [n_seq][n_kv][acc_stride]
  long long acc_stride;
  int n_seq, keep, first, recent;
  int* new_len;    // [n_seq]
  int* idx;        // [n_seq][n_kv][keep]
  float* acc_out;  // [n_seq][n_kv][keep]
};
hipError_t launch_kv4_evict(int head_dim, const Kv4View& src, const Kv4View& dst, const Kv4Evict& e, hipStream_t s);

#ifdef __HIPCC__
typedef _Float16 kvh2 __attribute__((ext_vector_type(2)));
typedef _Float16 kvh4 __attribute__((ext_vector_type(4)));
typedef _Float16 kvh8 __attribute__((ext_vector_type(8)));
typedef float kvf4 __attribute__((ext_vector_type(4)));
typedef float kvf16 __attribute__((ext_vector_type(16)));
typedef uint32_t kvu2 __attribute__((ext_vector_type(2)));
typedef uint32_t kvu4 __attribute__((ext_vector_type(4)));

// The layout of one kv head's block of a page.
template <int D> struct Kv4L {
  static constexpr int NG = D / 32;
  static constexpr int QG = NG < 4 ? NG : 4;   // groups per quad
  static constexpr int KT = 8 * D;             // bytes of a 16-token key tile
  static constexpr int V0 = 32 * D;            // value codes
  static constexpr int VB = 16 * D;            // bytes of a 32-token value block
  static constexpr int KS0 = 64 * D, VS0 = 72 * D;
  static constexpr int VSB = 4 * D;            // value scales of a 32-token block
  static constexpr int BYTES = 80 * D;
  // Byte offset of the key dword of token t (of the page), group g, lane group kg.
  __host__ __device__ static constexpr int key_word(int t, int g, int kg) {
    return (t >> 4) * KT + (g / QG) * (256 * QG) + ((16 * kg + (t & 15)) * QG + g % QG) * 4;
  }
  // Byte offset of the value dword of token t and dim; t's code is value_j(t).
  __host__ __device__ static constexpr int value_word(int t, int dim) {
    return V0 + (t >> 5) * VB + (dim >> 6) * 1024 + (16 * ((t & 15) >> 2) + (dim & 15)) * 16 + ((dim >> 4) & 3) * 4;
  }
  __host__ __device__ static constexpr int value_j(int t) { return ((t >> 4) & 1) * 4 + (t & 3); }
  __host__ __device__ static constexpr int key_d(int t, int g) { return KS0 + (t * 2 * NG + g) * 2; }
  __host__ __device__ static constexpr int key_m(int t, int g) { return key_d(t, g) + 2 * NG; }
  __host__ __device__ static constexpr int value_d(int t, int g) {
    return VS0 + (t >> 5) * VSB + (g * 32 + ((t & 15) >> 2) * 8 + value_j(t)) * 2;
  }
  __host__ __device__ static constexpr int value_m(int t, int g) { return value_d(t, g) + 64 * NG; }
};

// The block of kv head hk of sequence b's page p, or null where the table has
// no such page or names one outside the pool.
__device__ __forceinline__ uint8_t* kv4_block(const Kv4View& c, int b, int p, int hk, int head_bytes) {
  if (p < 0 || p >= c.max_pages) return nullptr;
  const int id = c.table[(size_t)b * c.max_pages + p];
  if (id < 0 || id >= c.n_pages) return nullptr;
  return c.pages + ((size_t)id * c.n_kv + hk) * head_bytes;
}

// Sequence b's rows [r0, r1) and length; row_start entries outside [0, n_rows]
// and ends before their start read as empty.
struct Kv4Span { int r0, r1, len; };
__device__ __forceinline__ Kv4Span kv4_span(const Kv4Rows& r, int b) {
  Kv4Span s;
  if (r.row_start) {
    s.r0 = min(max(r.row_start[b], 0), r.n_rows);
    s.r1 = min(max(r.row_start[b + 1], s.r0), r.n_rows);
  } else {
    s.r0 = min(b, r.n_rows);
    s.r1 = min(b + 1, r.n_rows);
  }
  s.len = max(r.kv_len[b], 0);
  return s;
}

// The lowest slot that the row at slot `pos` sees, where `reach` slots before
// its own are in the window (kv4_reach).  Rows below 0 see none; windows may
// be up to INT_MAX.
__device__ __forceinline__ int kv4_reach(int window) { return window > 0 ? window - 1 : 0x7FFFFFFF; }
__device__ __forceinline__ int kv4_lowest(int pos, int reach) { return max(0, max(pos, 0) - reach); }

__device__ __forceinline__ uint32_t kv4_code(uint32_t w, int j) {
  return __builtin_amdgcn_alignbit(w, w, (uint32_t)kv4_bit(j)) & 15u;
}
__device__ __forceinline__ float kv4_f16(const uint8_t* p) {
  return (float)*reinterpret_cast<const _Float16*>(p);
}
#endif

}  // namespace kq
