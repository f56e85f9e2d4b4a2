// w8_pack.hip -- 8-bit integer weights laid out, made from other kinds, and
// read back (done once, when a model is loaded).  A workgroup takes a row and
// zeroes what the layout has past in_dim; the last one also zeroes the rows
// that its tile has past out_dim.  Bound by memory, and in conversion by the
// element decoder, which runs twice: once for the largest magnitude, once for
// the codes.
#include "kq_elem.h"
#include "w8.h"

namespace kq {

// Row `row` of the layout: 16 codes per thread and turn, from get(k).
template <class G>
__device__ __forceinline__ void w8_write_row(uint8_t* packed, int row, int in_dim, G get) {
  const int blocks = w8_blocks(in_dim);
  for (int k = 16 * threadIdx.x; k < 64 * blocks; k += 16 * blockDim.x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = w8_four(get(k + 4 * i), get(k + 4 * i + 1), get(k + 4 * i + 2), get(k + 4 * i + 3));
    *reinterpret_cast<uint4*>(packed + w8_place(row, k, blocks)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Rows past out_dim, by the last row's workgroup.
__device__ __forceinline__ void w8_end_tile(uint8_t* packed, int in_dim, int out_dim) {
  float* const s = w8_scales(packed, in_dim, out_dim);
  for (int r = out_dim; r < 16 * w8_tiles(out_dim); ++r) {
    w8_write_row(packed, r, in_dim, [](int) { return 0; });
    if (threadIdx.x == 0) s[r] = 0.f;
  }
}

__global__ __launch_bounds__(256) void w8_pack(const int8_t* codes, long long stride, const float* scale, int in_dim,
                                               int out_dim, uint8_t* packed) {
  const int row = blockIdx.x;
  const int8_t* c = codes + (long long)row * stride;
  w8_write_row(packed, row, in_dim, [&](int k) { return k < in_dim ? (int)c[k] : 0; });
  if (threadIdx.x == 0) w8_scales(packed, in_dim, out_dim)[row] = scale[row];
  if (row == out_dim - 1) w8_end_tile(packed, in_dim, out_dim);
}

// KIND: a quantised kind, or -1 for f32.
template <int KIND>
__global__ __launch_bounds__(256) void w8_convert(const uint8_t* w, int in_dim, int out_dim, uint8_t* packed) {
  __shared__ float part[4];
  const int row = blockIdx.x;
  auto at = [&](int k) {
    if (k >= in_dim) return 0.f;
    if constexpr (KIND < 0) return reinterpret_cast<const float*>(w)[(size_t)row * in_dim + k];
    else return dequant_elem<KIND>(RowMajorBytes{w + ((size_t)row * (in_dim / 256) + k / 256) * block_bytes(KIND)}, k % 256);
  };
  float top = 0.f;
  for (int k = threadIdx.x; k < in_dim; k += 256) top = w8_top(top, at(k));
  const W8Scale s(w8_group_max<4>(top, part));
  w8_write_row(packed, row, in_dim, [&](int k) { return s.code(at(k)); });
  if (threadIdx.x == 0) w8_scales(packed, in_dim, out_dim)[row] = s.s;
  if (row == out_dim - 1) w8_end_tile(packed, in_dim, out_dim);
}

__global__ __launch_bounds__(256) void w8_unpack(const uint8_t* packed, int in_dim, int out_dim, float* w) {
  const int row = blockIdx.x, blocks = w8_blocks(in_dim);
  const float s = w8_scales(packed, in_dim, out_dim)[row];
  for (int k = threadIdx.x; k < in_dim; k += 256)
    w[(size_t)row * in_dim + k] = s * (float)(int8_t)packed[w8_place(row, k & ~15, blocks) + (k & 15)];
}

hipError_t launch_w8_pack(const int8_t* codes, long long stride, const float* scale, int in_dim, int out_dim,
                          uint8_t* packed, hipStream_t s) {
  hipLaunchKernelGGL(w8_pack, dim3(out_dim), dim3(256), 0, s, codes, stride, scale, in_dim, out_dim, packed);
  return hipGetLastError();
}

hipError_t launch_w8_convert(int kind, const void* w, int in_dim, int out_dim, uint8_t* packed, hipStream_t s) {
  const uint8_t* p = (const uint8_t*)w;
#define W8_CONVERT(K) \
  case K: hipLaunchKernelGGL(w8_convert<K>, dim3(out_dim), dim3(256), 0, s, p, in_dim, out_dim, packed); break;
  switch (kind) {
    W8_CONVERT(-1) W8_CONVERT(Q4_K) W8_CONVERT(Q6_K) W8_CONVERT(Q5_K) W8_CONVERT(Q3_K) W8_CONVERT(Q2_K) W8_CONVERT(Q8_0)
    default: return hipErrorInvalidValue;
  }
#undef W8_CONVERT
  return hipGetLastError();
}

hipError_t launch_w8_unpack(const uint8_t* packed, int in_dim, int out_dim, float* w, hipStream_t s) {
  hipLaunchKernelGGL(w8_unpack, dim3(out_dim), dim3(256), 0, s, packed, in_dim, out_dim, w);
  return hipGetLastError();
}

}  // namespace kq
