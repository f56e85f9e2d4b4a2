// kv4_cache.hip -- writing, reading back and shrinking the 4-bit cache.
//
// A group of 32 values x of a token's head is stored as
//   m = f16(min x), r = (max x - m) / 15,
//   d = r rounded up to 7 significant bits (a multiple of 2^-24 at least),
//   q = the nearest integer to (x - m) / d, ties to even, within 0 .. 15,
// d = 0 and q = 0 where r <= 0.  A group with a value that is not finite, or
// a minimum or step beyond the format, has d = m = 0, and its token's key in
// that head gets d = NaN in every group: key and value read back as NaN, and
// scores of the slot are NaN, while value scales are always finite (a weight
// of 0 times them is 0).
// The arithmetic is exact (f64 differences, remainders by fma): a code never
// depends on how a quotient was rounded.
#include <algorithm>

#include "kv4.h"

namespace kq {

struct AppendArgs {
  Kv4View c;
  Kv4Rows rows;
  const void *k, *v;
  long long ks, vs;
  const int* pos;
  RopeTable t;
};

struct Kv4Group { float d, m; int q[4]; bool bad; };

// The spacing of 7-bit steps at d >= 0, a multiple of 2^-24.
__device__ __forceinline__ float kv4_step_ulp(float d) {
  const int e = (__builtin_bit_cast(int, d) & 0x7F800000) - (6 << 23);
  return __builtin_bit_cast(float, max(e, (127 - 24) << 23));
}

// Quantises a group from four values in each of eight neighbouring lanes.
// Step and codes come from f32 quotients where those leave no doubt and are
// settled by exact f64 remainders where they might (in f64 throughout, with
// its divisions, 4097 + 1013 + 2 rows of 8 heads of 128 took 66 us for 18).
__device__ __forceinline__ Kv4Group kv4_quantise(const float (&x)[4]) {
  float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  int bad = !(__builtin_isfinite(x[0]) && __builtin_isfinite(x[1]) && __builtin_isfinite(x[2]) &&
              __builtin_isfinite(x[3]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, o, 64));
    hi = fmaxf(hi, __shfl_xor(hi, o, 64));
    bad |= __shfl_xor(bad, o, 64);
  }
  Kv4Group g;
  g.m = (float)(_Float16)lo;
  const double m = (double)g.m, z = (double)hi - m;
  // A step at or below z / 15, then up while 15 d < z: twice at most, since
  // the quotient is off by less than half a spacing.
  float d = 0.f;
  if (z > 0.0) {
    const float r = (float)z * ((1.f - 0x1p-21f) / 15.f);
    const float u = kv4_step_ulp(r);
    // 1 / u, a power of two, by its exponent.
    d = floorf(r * __builtin_bit_cast(float, (254 << 23) - __builtin_bit_cast(int, u))) * u;
    if (15.0 * (double)d < z) d += u;
    if (15.0 * (double)d < z) d += kv4_step_ulp(d);
  }
  if (bad || !__builtin_isfinite(g.m) || !(d <= KV4_D_MAX)) {
    g.bad = true;
    g.d = g.m = 0.f;
    g.q[0] = g.q[1] = g.q[2] = g.q[3] = 0;
    return g;
  }
  g.bad = false;
  g.d = d;
  // t is off by less than 16 * 2^-21 where it matters (0 <= t < 16).
  const float inv = d > 0.f ? __builtin_amdgcn_rcpf(d) : 0.f;
  float n[4];
  bool close = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = (x[i] - g.m) * inv;
    n[i] = __builtin_rintf(t);
    close |= __builtin_fabsf(t - n[i]) > 0.5f - 0x1p-16f;
  }
  if (close) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double rem = __builtin_fma(-(double)n[i], (double)d, (double)x[i] - m), h = 0.5 * (double)d;
      const bool odd = (int)n[i] & 1;
      if (rem > h || (rem == h && odd)) n[i] += 1.f;
      else if (rem < -h || (rem == -h && odd)) n[i] -= 1.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) g.q[i] = (int)fminf(fmaxf(n[i], 0.f), 15.f);
  return g;
}

template <class T>
__device__ __forceinline__ void load4(const T* p, float (&x)[4]) {
  struct { T v[4]; } r;
  __builtin_memcpy(&r, p, sizeof(r));
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = (float)r.v[i];
}

// One workgroup per (32 slots, kv head, sequence): a block of slots belongs
// to one workgroup, so the codes of a value dword that this call does not
// write are kept by a plain read and write of it.  Keys go straight from
// registers (eight lanes hold a group, two of them a dword); values pass
// through LDS, since a dword there holds eight tokens.  Every load is issued
// before the first sum: a decode step, one row a sequence, is one trip to
// memory behind its lengths and pages (32 sequences 14 -> 9 us).
template <int D, class T, bool ROPE>
__global__ __launch_bounds__(256) void kv4_append(AppendArgs a) {
  using L = Kv4L<D>;
  constexpr int NG = L::NG;
  __shared__ double2 cs[ROPE ? 16 * D / 2 : 1];  // cos, sin [token of the tile][pair]
  __shared__ uint8_t vq[32][D];
  __shared__ int bad[32];  // the token's key or value holds a group that the format does not
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const Kv4Span sp = kv4_span(a.rows, b);
  const int n = sp.r1 - sp.r0, slot0 = sp.len - n;  // the first row's slot, below 0 where kv_len < n
  const int lo = max(slot0, 0), hi = min((long long)sp.len, (long long)a.c.max_pages * KV4_PAGE);
  if (n <= 0 || lo >= hi) return;
  const int half = a.t.rot_dim >> 1;
  const int c8 = tid & 7;
  for (int blk = (lo >> 5) + blockIdx.x; blk <= (hi - 1) >> 5; blk += gridDim.x) {
    uint8_t* base = kv4_block(a.c, b, blk >> 1, hk, L::BYTES);
    if (!base) continue;
    const int s0 = blk << 5, p0 = (blk & 1) * 32;  // first slot, and its token of the page
    const bool whole = s0 >= lo && s0 + 32 <= hi;
    // The nearest row of this call: what a slot of another has is not stored.
    auto row = [&](int slot) { return (size_t)(sp.r0 + (min(max(slot, lo), hi - 1) - slot0)); };
    float xv[NG][4], xk[2][NG / 2][4], xo[2][NG / 2][4];
    int ps[2] = {0, 0};
    uint32_t old[D / 64];
    if constexpr (ROPE) {
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) ps[tile] = a.pos[row(s0 + 16 * tile + (tid >> 4))];
    }
    {
      const T* v = (const T*)a.v + row(s0 + (tid >> 3)) * a.vs + (size_t)hk * D + 4 * c8;
#pragma unroll
      for (int g = 0; g < NG; ++g) load4(v + 32 * g, xv[g]);
    }
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      const T* k = (const T*)a.k + row(s0 + 16 * tile + ((tid >> 3) & 15)) * a.ks + (size_t)hk * D;
#pragma unroll
      for (int it = 0; it < NG / 2; ++it) {
        const int d0 = 32 * (2 * it + (tid >> 7)) + 4 * c8;
        load4(k + d0, xk[tile][it]);
        if constexpr (ROPE) {
          // The other halves of the four pairs.
          auto other = [&](int d) { return d < half ? d + half : d < a.t.rot_dim ? d - half : d; };
          if (a.t.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; ++e) xo[tile][it][e] = xk[tile][it][e ^ 1];
          } else if (!(half & 3)) {
            load4(k + other(d0), xo[tile][it]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) xo[tile][it][e] = (float)k[other(d0 + e)];
          }
        }
      }
    }
    uint32_t* vw[D / 64];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const int i = tid + 256 * c, rg = i / D, d = i - rg * D;
      vw[c] = reinterpret_cast<uint32_t*>(base + L::value_word(p0 + 4 * rg, d));
      old[c] = 0;
      if (!whole) old[c] = *vw[c];
    }
    if (tid < 32) bad[tid] = 0;
    __syncthreads();
    {
      const int t = tid >> 3, slot = s0 + t;
      const bool in = slot >= lo && slot < hi;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const Kv4Group q = kv4_quantise(xv[g]);
        *reinterpret_cast<uint32_t*>(&vq[t][32 * g + 4 * c8]) =
            (uint32_t)q.q[0] | (uint32_t)q.q[1] << 8 | (uint32_t)q.q[2] << 16 | (uint32_t)q.q[3] << 24;
        if (in && c8 == 0) {
          if (q.bad) bad[t] = 1;
          *reinterpret_cast<_Float16*>(base + L::value_d(p0 + t, g)) = (_Float16)q.d;
          *reinterpret_cast<_Float16*>(base + L::value_m(p0 + t, g)) = (_Float16)q.m;
        }
      }
    }
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      const int f = s0 + 16 * tile;
      if (f >= hi || f + 16 <= lo) continue;
      if constexpr (ROPE) {
        __syncthreads();
        if (f + (tid >> 4) >= lo && f + (tid >> 4) < hi) {
          for (int p = tid & 15; p < half; p += 16) {
            double s, c;
            sincos_f64((double)ps[tile] * a.t.freq[p], s, c);
            cs[(tid >> 4) * half + p] = make_double2(c * a.t.mag, s * a.t.mag);
          }
        }
        __syncthreads();
      }
      const int t = (tid >> 3) & 15, slot = f + t, tok = p0 + 16 * tile + t;
      const bool in = slot >= lo && slot < hi;
#pragma unroll
      for (int it = 0; it < NG / 2; ++it) {
        const int g = 2 * it + (tid >> 7), d0 = 32 * g + 4 * c8;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = xk[tile][it][e];
        if constexpr (ROPE) {
          if (in) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = d0 + e;
              if (d < a.t.rot_dim) {
                const bool second = a.t.interleaved ? (d & 1) : d >= half;
                const int p = a.t.interleaved ? d >> 1 : second ? d - half : d;
                const double2 w = cs[t * half + p];
                const double me = xk[tile][it][e], o = xo[tile][it][e];
                // (a c - b s, a s + b c), rounded to f32 once.
                x[e] = (float)(second ? __builtin_fma(o, w.y, me * w.x) : __builtin_fma(me, w.x, -(o * w.y)));
              }
            }
          }
        }
        const Kv4Group q = kv4_quantise(x);
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t left = (c8 & 1) ? kv4_bit(4 + e) : kv4_bit(e);
          w |= __builtin_amdgcn_alignbit((uint32_t)q.q[e], (uint32_t)q.q[e], 32 - left);
        }
        w |= (uint32_t)__shfl_xor((int)w, 1, 64);
        if (in && !(c8 & 1)) *reinterpret_cast<uint32_t*>(base + L::key_word(tok, g, c8 >> 1)) = w;
        if (in && c8 == 0) {
          if (q.bad) bad[16 * tile + t] = 1;
          *reinterpret_cast<_Float16*>(base + L::key_d(tok, g)) = (_Float16)q.d;
          *reinterpret_cast<_Float16*>(base + L::key_m(tok, g)) = (_Float16)q.m;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const int i = tid + 256 * c, rg = i / D, d = i - rg * D;
      uint32_t w = 0, mine = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = 16 * (j >> 2) + 4 * rg + (j & 3), slot = s0 + t;
        if (slot >= lo && slot < hi) {
          const uint32_t code = vq[t][d];
          w |= __builtin_amdgcn_alignbit(code, code, (uint32_t)((32 - kv4_bit(j)) & 31));
          mine |= __builtin_amdgcn_alignbit(15u, 15u, (uint32_t)((32 - kv4_bit(j)) & 31));
        }
      }
      if (mine) *vw[c] = (old[c] & ~mine) | w;
    }
    // (A slot that is not this call's has no flag.)
    if (tid < 32 && bad[tid]) {
#pragma unroll
      for (int g = 0; g < NG; ++g) *reinterpret_cast<uint16_t*>(base + L::key_d(p0 + tid, g)) = 0x7E00;
    }
    __syncthreads();
  }
}

struct ReadArgs {
  Kv4View c;
  Kv4Rows rows;
  void *k, *v;
  long long ks, vs;
};

// One workgroup per (32 slots, kv head, sequence), a thread per dword: a key
// dword's eight values are 16 or 32 bytes of a row, a value dword's belong to
// eight rows, where neighbouring lanes write neighbouring values.
template <int D, class T>
__global__ __launch_bounds__(256) void kv4_read(ReadArgs a) {
  using L = Kv4L<D>;
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const Kv4Span sp = kv4_span(a.rows, b);
  const int n = sp.r1 - sp.r0, slot0 = sp.len - n;
  const int lo = max(slot0, 0), hi = sp.len;
  if (n <= 0 || lo >= hi) return;
  for (int blk = (lo >> 5) + blockIdx.x; blk <= (hi - 1) >> 5; blk += gridDim.x) {
    const uint8_t* base = kv4_block(a.c, b, blk >> 1, hk, L::BYTES);
    const int s0 = blk << 5, p0 = (blk & 1) * 32;
    auto in = [&](int t) { return s0 + t >= lo && s0 + t < hi; };
    auto row = [&](int t) { return (size_t)(sp.r0 + (s0 + t - slot0)); };
    if (!base) {
      for (int i = tid; i < 32 * D; i += 256) {
        const int t = i / D, d = i % D;
        if (!in(t)) continue;
        ((T*)a.k)[row(t) * a.ks + (size_t)hk * D + d] = (T)__builtin_nanf("");
        ((T*)a.v)[row(t) * a.vs + (size_t)hk * D + d] = (T)__builtin_nanf("");
      }
      continue;
    }
    uint32_t kw[D / 64], vw[D / 64];
    _Float16 kd[D / 64], km[D / 64];
    kvh8 vd[D / 64], vm[D / 64];
    const float mark = kv4_f16(base + L::key_d(p0 + (tid & 31), 0));  // NaN: the slot holds no value
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const int i = tid + 256 * c, t = i / (D / 8), oct = i % (D / 8), rg = i / D, d = i % D;
      kw[c] = *reinterpret_cast<const uint32_t*>(base + L::key_word(p0 + t, oct >> 2, oct & 3));
      kd[c] = *reinterpret_cast<const _Float16*>(base + L::key_d(p0 + t, oct >> 2));
      km[c] = *reinterpret_cast<const _Float16*>(base + L::key_m(p0 + t, oct >> 2));
      vw[c] = *reinterpret_cast<const uint32_t*>(base + L::value_word(p0 + 4 * rg, d));
      vd[c] = *reinterpret_cast<const kvh8*>(base + L::value_d(p0 + 4 * rg, d >> 5));
      vm[c] = *reinterpret_cast<const kvh8*>(base + L::value_m(p0 + 4 * rg, d >> 5));
    }
    const uint32_t none = (uint32_t)__ballot(!(mark >= 0.f));  // bit t: token t of the block
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const int i = tid + 256 * c, t = i / (D / 8), oct = i % (D / 8), rg = i / D, d = i % D;
      if (in(t)) {
        struct { T v[8]; } o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o.v[j] = (T)__builtin_fmaf((float)kd[c], (float)kv4_code(kw[c], j), (float)km[c]);
        __builtin_memcpy((T*)a.k + row(t) * a.ks + (size_t)hk * D + 8 * oct, &o, sizeof(o));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int u = 16 * (j >> 2) + 4 * rg + (j & 3);
        if (!in(u)) continue;
        float x = __builtin_fmaf((float)vd[c][j], (float)kv4_code(vw[c], j), (float)vm[c][j]);
        if (none >> u & 1) x = __builtin_nanf("");
        ((T*)a.v)[row(u) * a.vs + (size_t)hk * D + d] = (T)x;
      }
    }
  }
}

// Workgroups per (kv head, sequence): one for every 32-slot block of an
// average sequence; longer ones take theirs in turns.
static unsigned blocks_of(const Kv4Rows& r) {
  return (unsigned)std::min<long long>(65535, ((long long)r.n_rows + r.n_seq - 1) / r.n_seq / 32 + 2);
}

template <int D, class T>
static void append_go(const AppendArgs& a, bool rope, hipStream_t s) {
  const dim3 grid(blocks_of(a.rows), a.c.n_kv, a.rows.n_seq);
  if (rope) hipLaunchKernelGGL((kv4_append<D, T, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((kv4_append<D, T, false>), grid, dim3(256), 0, s, a);
}
template <int D>
static void append_typed(const AppendArgs& a, int type, bool rope, hipStream_t s) {
  if (type == ACT_F32) append_go<D, float>(a, rope, s);
  else if (type == ACT_F16) append_go<D, _Float16>(a, rope, s);
  else append_go<D, bf16_t>(a, rope, s);
}

hipError_t launch_kv4_append(int head_dim, const Kv4View& c, int type, const void* k, long long k_stride,
                             const void* v, long long v_stride, const Kv4Rows& rows, const RopeTable* rope,
                             const int* pos, hipStream_t s) {
  AppendArgs a{};
  a.c = c;
  a.rows = rows;
  a.k = k;
  a.v = v;
  a.ks = k_stride;
  a.vs = v_stride;
  a.pos = pos;
  if (rope) a.t = *rope;
  if (head_dim == 64) append_typed<64>(a, type, rope != nullptr, s);
  else if (head_dim == 128) append_typed<128>(a, type, rope != nullptr, s);
  else append_typed<256>(a, type, rope != nullptr, s);
  return hipGetLastError();
}

template <int D>
static void read_typed(const ReadArgs& a, int type, hipStream_t s) {
  const dim3 grid(blocks_of(a.rows), a.c.n_kv, a.rows.n_seq);
  if (type == ACT_F32) hipLaunchKernelGGL((kv4_read<D, float>), grid, dim3(256), 0, s, a);
  else if (type == ACT_F16) hipLaunchKernelGGL((kv4_read<D, _Float16>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((kv4_read<D, bf16_t>), grid, dim3(256), 0, s, a);
}

hipError_t launch_kv4_read(int head_dim, const Kv4View& c, int type, const Kv4Rows& rows, void* k, long long k_stride,
                           void* v, long long v_stride, hipStream_t s) {
  const ReadArgs a{c, rows, k, v, k_stride, v_stride};
  if (head_dim == 64) read_typed<64>(a, type, s);
  else if (head_dim == 128) read_typed<128>(a, type, s);
  else read_typed<256>(a, type, s);
  return hipGetLastError();
}

// ---- eviction -----------------------------------------------------------------

// A weight's rank: NaN and what is not above zero rank lowest, alike.
__device__ __forceinline__ uint32_t evict_key(float v) { return v > 0.f ? __builtin_bit_cast(uint32_t, v) : 0u; }

// Sums over all 1024 threads, and over those before the caller's (waves in
// order, lanes in order).  part: 16 words that the previous call of the same
// `part` is done with.
__device__ __forceinline__ int wg_before(int v, int* part, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(sum, o, 64);
    if (lane >= o) sum += u;
  }
  if (lane == 63) part[w] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int p = part[i];
    if (i < w) before += p;
    all += p;
  }
  *total = all;
  return sum - v + before;
}

// One workgroup per (kv head, sequence): the rank of the lightest slot kept,
// by the 31 bits of a weight from the top (a histogram of the slots still in
// question per 11, 10 and 10 of them), then the kept slots in order.  Among
// slots of that rank the lowest stay.  new_len is the same for every head;
// head 0 writes it.  Bound by latencies, the weights being in cache after the
// first pass: eight are in flight per thread, bins are summed by all threads
// (by one thread, 256 bins: 56 us at 16 x 8 rows of 8193, now 12), and the
// ranks of 8192 slots come from ballots and one barrier.
__global__ __launch_bounds__(1024) void kv4_select(Kv4Evict e, int n_kv) {
  constexpr int PER = 8;
  __shared__ int hist[2048];
  __shared__ int part[2][16];
  __shared__ int pick[2];
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = max(e.kv_len[b], 0), kept = min(n, e.keep);
  const float* acc = e.acc + ((size_t)b * n_kv + hk) * e.acc_stride;
  int* idx = e.idx + ((size_t)b * n_kv + hk) * e.keep;
  float* out = e.acc_out + ((size_t)b * n_kv + hk) * e.keep;
  const unsigned have = (unsigned)min((long long)n, e.acc_stride);  // slots with a weight
  // The weights of slots i0 + 512 wave + 64 j + lane, 0 for those without one.
  auto weights = [&](unsigned i0, float (&v)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const unsigned i = i0 + 64 * (PER * wave + j) + lane;
      v[j] = have ? acc[min(i, have - 1)] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (i0 + 64 * (PER * wave + j) + lane >= have) v[j] = 0.f;
  };
  if (hk == 0 && tid == 0) e.new_len[b] = kept;
  for (int i = kept + tid; i < e.keep; i += 1024) {
    idx[i] = -1;
    out[i] = 0.f;
  }
  if (n <= e.keep) {
    for (int i = tid; i < n; i += 1024) {
      idx[i] = i;
      out[i] = (unsigned)i < have ? acc[i] : 0.f;
    }
    return;
  }
  const unsigned m0 = e.first, m1 = n - e.recent;  // the slots in question
  int need = e.keep - e.first - e.recent;
  uint32_t top = 0, mask = 0;
  if (need > 0) {
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 20 : pass == 1 ? 10 : 0, bins = pass == 0 ? 2048 : 1024;
      hist[tid] = 0;
      hist[tid + 1024] = 0;
      __syncthreads();
      for (unsigned i0 = 0; i0 < m1; i0 += 1024 * PER) {
        float v[PER];
        weights(i0, v);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const unsigned i = i0 + 64 * (PER * wave + j) + lane;
          const uint32_t k = evict_key(v[j]);
          if (i >= m0 && i < m1 && (k & mask) == top) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
        }
      }
      __syncthreads();
      // Thread t has the t-th bins from the top; the bin where the sum reaches
      // `need` is the one.
      const int per = bins >> 10, bin = bins - per * (tid + 1);
      const int upper = hist[bin + per - 1], lower = per == 2 ? hist[bin] : 0;
      int all, before = wg_before(upper + lower, part[pass & 1], &all);
      if (before < need && before + upper >= need) {
        pick[0] = bin + per - 1;
        pick[1] = need - before;
      } else if (before + upper < need && before + upper + lower >= need) {
        pick[0] = bin;
        pick[1] = need - before - upper;
      }
      __syncthreads();
      top |= (uint32_t)pick[0] << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      need = pick[1];
    }
  }
  // Slots above `top` stay, and the first `need` of those equal to it.
  int at = 0, ties = 0, turn = 0;
  __syncthreads();
  for (unsigned i0 = 0; i0 < (unsigned)n; i0 += 1024 * PER, turn ^= 1) {
    float v[PER];
    weights(i0, v);
    uint64_t sure[PER], tie[PER];
    uint32_t count = 0;  // of the wave: sure ones, and ties << 16
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const unsigned i = i0 + 64 * (PER * wave + j) + lane;
      const uint32_t k = evict_key(v[j]);
      const bool edge = i < m0 || i >= m1;
      sure[j] = __ballot(i < (unsigned)n && (edge || (mask && k > top)));
      tie[j] = __ballot(i < (unsigned)n && !edge && mask && k == top);
      count += (uint32_t)__popcll(sure[j]) + ((uint32_t)__popcll(tie[j]) << 16);
    }
    if (lane == 0) part[turn][wave] = (int)count;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t p = (uint32_t)part[turn][i];
      if (i < wave) before += p;
      all += p;
    }
    int s = at + (int)(before & 0xFFFF), t = ties + (int)(before >> 16);
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int sb = s + __popcll(sure[j] & below), tb = t + __popcll(tie[j] & below);
      const bool is_tie = tie[j] >> lane & 1;
      if ((sure[j] >> lane & 1) || (is_tie && tb < need)) {
        const int place = sb + min(tb, need);
        idx[place] = (int)(i0 + 64 * (PER * wave + j) + lane);
        out[place] = v[j];
      }
      s += __popcll(sure[j]);
      t += __popcll(tie[j]);
    }
    at += (int)(all & 0xFFFF);
    ties += (int)(all >> 16);
  }
}

// One workgroup per (page of 64 new slots, kv head, sequence).  The key codes
// of a token are 16 bytes per lane group and quad and its key scales lie
// together; a value dword, and the 16 bytes of its scales, collect one entry
// from each of eight old tokens.  Slots of a page that the source's table does
// not have read as NaN: key steps of NaN, all else 0.  What stands in new
// slots past the last one is 0 where a word shares it.
template <int D>
__global__ __launch_bounds__(256) void kv4_gather(Kv4View src, Kv4View dst, Kv4Evict e) {
  using L = Kv4L<D>;
  constexpr int NG = L::NG;
  __shared__ const uint8_t* from[KV4_PAGE];  // the old block (or any memory of ours, unused)
  __shared__ int slot[KV4_PAGE];             // the old token in it, -1: none, -2: page missing
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int kept = min(max(e.kv_len[b], 0), e.keep);
  const int s0 = blockIdx.x * KV4_PAGE;
  if (s0 >= kept) return;
  uint8_t* to = kv4_block(dst, b, blockIdx.x, hk, L::BYTES);
  if (!to) return;
  if (tid < KV4_PAGE) {
    const int f = s0 + tid < kept ? e.idx[((size_t)b * src.n_kv + hk) * e.keep + s0 + tid] : -1;
    const uint8_t* s = f < 0 ? nullptr : kv4_block(src, b, f / KV4_PAGE, hk, L::BYTES);
    from[tid] = s ? s : to;
    slot[tid] = f < 0 ? -1 : s ? f % KV4_PAGE : -2;
  }
  __syncthreads();
  typedef uint32_t Quad __attribute__((ext_vector_type(L::QG)));
  // Key codes: token, lane group, quad.
#pragma unroll
  for (int i = tid; i < KV4_PAGE * 4 * (NG / L::QG); i += 256) {
    const int t = i & 63, kg = (i >> 6) & 3, g = (i >> 8) * L::QG, ft = slot[t];
    Quad w = *reinterpret_cast<const Quad*>(from[t] + L::key_word(max(ft, 0), g, kg));
    if (ft < 0) w = 0;
    if (ft != -1) *reinterpret_cast<Quad*>(to + L::key_word(t, g, kg)) = w;
  }
  // Value dwords, four dims (16 apart) of a thread together.
#pragma unroll
  for (int i = tid; i < 2 * D; i += 256) {
    const int l = i & 63, ch = (i >> 6) % (D / 64), blk = i / D, rg = l >> 4, dim = 64 * ch + (l & 15);
    kvu4 o[8], w = {0, 0, 0, 0};
    int ft[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = 32 * blk + 16 * (j >> 2) + 4 * rg + (j & 3);
      ft[j] = slot[t];
      o[j] = *reinterpret_cast<const kvu4*>(from[t] + L::value_word(max(ft[j], 0), dim));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t fj = (uint32_t)L::value_j(max(ft[j], 0)), four = ft[j] < 0 ? 0u : 15u;
      // kv4_bit of a run-time j: 6, 22, 2, 18, 14, 30, 10, 26.
      const uint32_t bit = ((fj & 1) << 4) + ((0xAE26u >> ((fj >> 1) << 2)) & 15u);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t word = o[j][k], c = __builtin_amdgcn_alignbit(word, word, bit) & four;
        w[k] |= __builtin_amdgcn_alignbit(c, c, (uint32_t)((32 - kv4_bit(j)) & 31));
      }
    }
    *reinterpret_cast<kvu4*>(to + L::value_word(32 * blk + 4 * rg, dim)) = w;
  }
  // Key scales of a token: NG dwords.
  for (int i = tid; i < KV4_PAGE * (NG / L::QG); i += 256) {
    const int t = i & 63, c = i >> 6, ft = slot[t];
    constexpr int STEPS = NG / 2;  // dwords of steps, then as many of minima
    Quad w = *reinterpret_cast<const Quad*>(from[t] + L::key_d(max(ft, 0), 0) + 4 * L::QG * c);
    if (ft < 0) {
#pragma unroll
      for (int k = 0; k < L::QG; ++k) w[k] = L::QG * c + k < STEPS ? 0x7E007E00u : 0u;
    }
    if (ft != -1) *reinterpret_cast<Quad*>(to + L::key_d(t, 0) + 4 * L::QG * c) = w;
  }
  // Value scales: block, step or minimum, group, lane group.
  for (int i = 255 - tid; i < 16 * NG; i += 256) {
    const int rg = i & 3, g = (i >> 2) % NG, m = (i / (4 * NG)) & 1, blk = i / (8 * NG);
    uint16_t o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = 32 * blk + 16 * (j >> 2) + 4 * rg + (j & 3), ft = slot[t];
      o[j] = *reinterpret_cast<const uint16_t*>(from[t] + L::value_d(max(ft, 0), g) + 64 * NG * m);
      if (ft < 0) o[j] = 0;
    }
    kvu4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = o[2 * k] | (uint32_t)o[2 * k + 1] << 16;
    *reinterpret_cast<kvu4*>(to + L::value_d(32 * blk + 4 * rg, g) + 64 * NG * m) = w;
  }
}

hipError_t launch_kv4_evict(int head_dim, const Kv4View& src, const Kv4View& dst, const Kv4Evict& e, hipStream_t s) {
  hipLaunchKernelGGL(kv4_select, dim3(src.n_kv, e.n_seq), dim3(1024), 0, s, e, src.n_kv);
  const dim3 grid((e.keep + KV4_PAGE - 1) / KV4_PAGE, src.n_kv, e.n_seq);
  if (head_dim == 64) hipLaunchKernelGGL((kv4_gather<64>), grid, dim3(256), 0, s, src, dst, e);
  else if (head_dim == 128) hipLaunchKernelGGL((kv4_gather<128>), grid, dim3(256), 0, s, src, dst, e);
  else hipLaunchKernelGGL((kv4_gather<256>), grid, dim3(256), 0, s, src, dst, e);
  return hipGetLastError();
}

}  // namespace kq
