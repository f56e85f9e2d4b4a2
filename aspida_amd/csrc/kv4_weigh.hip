// kv4_weigh.hip -- the attention weight each cached slot received:
//   acc_out[b][hk][j] = acc_in[b][hk][j]
//                     + sum over rows and the query heads of hk of exp(scale q . k_j - lse)
// for the slots j a row sees (acc_out = acc_in for the others).  A slot belongs to one workgroup, which adds
// its terms in a fixed order: no atomics, the same bits every time.
#include "kv4.h"

namespace kq {

template <class T, int D>
__global__ __launch_bounds__(256) void kv4_weigh_simple(Kv4View c, Kv4Rows rows, Kv4Weigh a) {
  using L = Kv4L<D>;
  __shared__ float kf[64][D + 1];
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const Kv4Span sp = kv4_span(rows, b);
  const int n = min((long long)sp.len, a.acc_stride), G = a.n_heads / c.n_kv;
  const long long all = a.acc_stride;
  for (long long p = blockIdx.x; p * 64 < all; p += gridDim.x) {
    if (p * 64 >= n) {
      const long long slot = p * 64 + tid;
      const size_t o = ((size_t)b * c.n_kv + hk) * a.acc_stride + slot;
      if (tid < 64 && slot < all) a.acc_out[o] = a.acc_in ? a.acc_in[o] : 0.f;
      continue;
    }
    const uint8_t* blk = kv4_block(c, b, (int)p, hk, L::BYTES);
    __syncthreads();
    for (int i = tid; i < 64 * (D / 8); i += 256) {
      const int t = i / (D / 8), d0 = i % (D / 8) * 8, g = d0 >> 5;
      const uint32_t wd = blk ? *reinterpret_cast<const uint32_t*>(blk + L::key_word(t, g, (d0 >> 3) & 3)) : 0;
      const float d = blk ? kv4_f16(blk + L::key_d(t, g)) : __builtin_nanf(""), m = blk ? kv4_f16(blk + L::key_m(t, g)) : 0.f;
      for (int j = 0; j < 8; ++j) kf[t][d0 + j] = __builtin_fmaf(d, (float)kv4_code(wd, j), m);
    }
    __syncthreads();
    const int t = tid >> 2, part = tid & 3, slot = (int)p * 64 + t;
    float sum = 0.f;
    for (int r = sp.r0; r < sp.r1; ++r) {
      const int pos = sp.len - (sp.r1 - r);
      for (int h = hk * G; h < (hk + 1) * G; ++h) {
        const T* q = (const T*)a.q + (size_t)r * a.q_stride + (size_t)h * D;
        float dot = 0.f;
        for (int i = part; i < D; i += 4) dot += (float)q[i] * kf[t][i];
        dot += __shfl_xor(dot, 1, 64);
        dot += __shfl_xor(dot, 2, 64);
        const float lse = a.lse[(size_t)r * a.n_heads + h];
        if (slot <= pos && (a.window <= 0 || slot > pos - a.window) && lse != -INFINITY)
          sum += expf(dot * a.scale - lse);
      }
    }
    if (part == 0 && slot < all) {
      const size_t o = ((size_t)b * c.n_kv + hk) * a.acc_stride + slot;
      a.acc_out[o] = (a.acc_in ? a.acc_in[o] : 0.f) + (slot < n ? sum : 0.f);
    }
  }
}

template <class T>
static void weigh_typed(int head_dim, const Kv4View& c, const Kv4Rows& rows, const Kv4Weigh& a, hipStream_t s) {
  const dim3 grid(c.max_pages < 1024 ? c.max_pages : 1024, c.n_kv, rows.n_seq);
  if (head_dim == 64) hipLaunchKernelGGL((kv4_weigh_simple<T, 64>), grid, dim3(256), 0, s, c, rows, a);
  else if (head_dim == 128) hipLaunchKernelGGL((kv4_weigh_simple<T, 128>), grid, dim3(256), 0, s, c, rows, a);
  else hipLaunchKernelGGL((kv4_weigh_simple<T, 256>), grid, dim3(256), 0, s, c, rows, a);
}

hipError_t launch_kv4_weigh(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Weigh& w,
                            hipStream_t s) {
  if (type == ACT_F32) weigh_typed<float>(head_dim, c, rows, w, s);
  else if (type == ACT_F16) weigh_typed<_Float16>(head_dim, c, rows, w, s);
  else weigh_typed<bf16_t>(head_dim, c, rows, w, s);
  return hipGetLastError();
}

}  // namespace kq
