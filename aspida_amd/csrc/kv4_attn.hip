// kv4_attn.hip -- attention over the paged 4-bit cache.
//
// Row i of a sequence's n new rows sits at slot p = kv_len - n + i and sees
// the slots j <= p (and j > p - window):
//   o = sum_j softmax_j(scale q . k_j) v_j,   lse = log sum_j exp(scale q . k_j).
// A row that sees nothing gets o = 0 and lse = -inf.
#include "kv4.h"

namespace kq {

template <class T, int D>
__global__ __launch_bounds__(256) void kv4_attn_simple(Kv4View c, Kv4Rows rows, Kv4Attn a) {
  using L = Kv4L<D>;
  __shared__ float q[D], s[64];
  const int h = blockIdx.x, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
  const Kv4Span sp = kv4_span(rows, b);
  const int hk = h / (a.n_heads / c.n_kv);
  for (int r = sp.r0 + blockIdx.y; r < sp.r1; r += gridDim.y) {
    __syncthreads();
    for (int i = tid; i < D; i += 256) q[i] = (float)((const T*)a.q)[(size_t)r * a.q_stride + (size_t)h * D + i] * a.scale;
    for (int i = tid; i < D; i += 256) q[i] = __builtin_isfinite(q[i]) ? q[i] : __builtin_nanf("");
    const int pos = sp.len - (sp.r1 - r);
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    float m = -1e30f, l = 0.f, o = 0.f;
    for (int p = lo / 64; p <= (pos >= 0 ? pos / 64 : -1); ++p) {
      const uint8_t* blk = kv4_block(c, b, p, hk, L::BYTES);
      __syncthreads();
      const int t = tid >> 2, part = tid & 3;
      float dot = 0.f;
      for (int g = 0; g < L::NG; ++g) {
        const uint32_t wd = blk ? *reinterpret_cast<const uint32_t*>(blk + L::key_word(t, g, part)) : 0;
        const float d = blk ? kv4_f16(blk + L::key_d(t, g)) : __builtin_nanf(""), mm = blk ? kv4_f16(blk + L::key_m(t, g)) : 0.f;
        for (int j = 0; j < 8; ++j) dot += q[32 * g + 8 * part + j] * __builtin_fmaf(d, (float)kv4_code(wd, j), mm);
      }
      dot += __shfl_xor(dot, 1, 64);
      dot += __shfl_xor(dot, 2, 64);
      if (part == 0) s[t] = (p * 64 + t <= pos && p * 64 + t >= lo) ? dot : -INFINITY;
      __syncthreads();
      float mx = s[lane];
      for (int k = 32; k; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k, 64));
      const float mn = fmaxf(m, mx), f = expf(m - mn);
      float pr = expf(s[lane] - mn), ps = pr;
      for (int k = 32; k; k >>= 1) ps += __shfl_xor(ps, k, 64);
      l = l * f + ps;
      o *= f;
      m = mn;
      if (tid < D)
        for (int t2 = 0; t2 < 64; ++t2) {
          if (!(p * 64 + t2 <= pos && p * 64 + t2 >= lo)) continue;
          const uint32_t wd = blk ? *reinterpret_cast<const uint32_t*>(blk + L::value_word(t2, tid)) : 0;
          const float d = blk ? kv4_f16(blk + L::value_d(t2, tid >> 5)) : __builtin_nanf(""), mm = blk ? kv4_f16(blk + L::value_m(t2, tid >> 5)) : 0.f;
          o += expf(s[t2] - mn) * __builtin_fmaf(d, (float)kv4_code(wd, L::value_j(t2)), mm);
        }
    }
    if (tid < D) ((T*)a.out)[(size_t)r * a.out_stride + (size_t)h * D + tid] = (T)(l != 0.f ? o / l : 0.f);
    if (tid == 0 && a.lse) a.lse[(size_t)r * a.n_heads + h] = l != 0.f ? m + logf(l) : -INFINITY;
  }
}

size_t kv4_attn_work_bytes(int head_dim, int n_kv, int n_heads, int n_rows, int n_seq, int max_rows, int max_pages) {
  return 256;
}

template <class T>
static void attn_typed(int head_dim, const Kv4View& c, const Kv4Rows& rows, const Kv4Attn& a, hipStream_t s) {
  const dim3 grid(a.n_heads, a.max_rows < 4096 ? a.max_rows : 4096, rows.n_seq);
  if (head_dim == 64) hipLaunchKernelGGL((kv4_attn_simple<T, 64>), grid, dim3(256), 0, s, c, rows, a);
  else if (head_dim == 128) hipLaunchKernelGGL((kv4_attn_simple<T, 128>), grid, dim3(256), 0, s, c, rows, a);
  else hipLaunchKernelGGL((kv4_attn_simple<T, 256>), grid, dim3(256), 0, s, c, rows, a);
}

hipError_t launch_kv4_attn(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, const Kv4Attn& a,
                           hipStream_t s) {
  if (type == ACT_F32) attn_typed<float>(head_dim, c, rows, a, s);
  else if (type == ACT_F16) attn_typed<_Float16>(head_dim, c, rows, a, s);
  else attn_typed<bf16_t>(head_dim, c, rows, a, s);
  return hipGetLastError();
}

}  // namespace kq
