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

// Quantises a group from four values in each of eight neighbouring lanes.
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
  const _Float16 mh = (_Float16)lo;
  g.m = (float)mh;
  const double m = (double)g.m, r = ((double)hi - m) / 15.0;
  double d = 0.0;
  if (r > 0.0) {
    int e;
    (void)frexp(r, &e);  // r in [2^(e-1), 2^e)
    const int step = max(e - 7, -24);
    d = ldexp(ceil(ldexp(r, -step)), step);
  }
  if (bad || !__builtin_isfinite(g.m) || d > (double)KV4_D_MAX) {
    g.bad = true;
    g.d = g.m = 0.f;
    g.q[0] = g.q[1] = g.q[2] = g.q[3] = 0;
    return g;
  }
  g.bad = false;
  g.d = (float)d;
  const double inv = d > 0.0 ? 1.0 / d : 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double z = (double)x[i] - m;
    double n = rint(z * inv);
    // z * inv may be an ulp off: the remainder decides, exactly.
    const double rem = __builtin_fma(-n, d, z), h = 0.5 * d;
    const bool odd = (int)n & 1;
    if (rem > h || (rem == h && odd && d > 0.0)) n += 1.0;
    if (rem < -h || (rem == -h && odd && d > 0.0)) n -= 1.0;
    g.q[i] = d > 0.0 ? (int)fmin(fmax(n, 0.0), 15.0) : 0;
  }
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
// through LDS, since a dword there holds eight tokens.
template <int D, class T, bool ROPE>
__global__ __launch_bounds__(256) void kv4_append(AppendArgs a) {
  using L = Kv4L<D>;
  __shared__ double2 cs[ROPE ? 16 * D / 2 : 1];  // cos, sin [token of the tile][pair]
  __shared__ uint8_t vq[32][D];
  __shared__ int bad[32];  // the token's key or value holds a group that the format does not
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const Kv4Span sp = kv4_span(a.rows, b);
  const int n = sp.r1 - sp.r0, slot0 = sp.len - n;  // the first row's slot, below 0 where kv_len < n
  const int lo = max(slot0, 0), hi = min((long long)sp.len, (long long)a.c.max_pages * KV4_PAGE);
  if (n <= 0 || lo >= hi) return;
  const int half = a.t.rot_dim >> 1;
  for (int blk = (lo >> 5) + blockIdx.x; blk <= (hi - 1) >> 5; blk += gridDim.x) {
    uint8_t* base = kv4_block(a.c, b, blk >> 1, hk, L::BYTES);
    if (!base) continue;
    const int s0 = blk << 5, p0 = (blk & 1) * 32;  // first slot, and its token of the page
    const int c8 = tid & 7;
    if (tid < 32) bad[tid] = 0;
    __syncthreads();
#pragma unroll 2
    for (int it = 0; it < L::NG; ++it) {
      const int t = tid >> 3, g = it, slot = s0 + t;
      const bool in = slot >= lo && slot < hi;
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (in) load4((const T*)a.v + (size_t)(sp.r0 + (slot - slot0)) * a.vs + (size_t)hk * D + 32 * g + 4 * c8, x);
      const Kv4Group q = kv4_quantise(x);
      *reinterpret_cast<uint32_t*>(&vq[t][32 * g + 4 * c8]) =
          (uint32_t)q.q[0] | (uint32_t)q.q[1] << 8 | (uint32_t)q.q[2] << 16 | (uint32_t)q.q[3] << 24;
      if (in && c8 == 0) {
        if (q.bad) bad[t] = 1;
        *reinterpret_cast<_Float16*>(base + L::value_d(p0 + t, g)) = (_Float16)q.d;
        *reinterpret_cast<_Float16*>(base + L::value_m(p0 + t, g)) = (_Float16)q.m;
      }
    }
    __syncthreads();
    for (int tile = 0; tile < 2; ++tile) {
      const int f = s0 + 16 * tile;
      if (f >= hi || f + 16 <= lo) continue;
      if constexpr (ROPE) {
        __syncthreads();
        for (int i = tid; i < 16 * half; i += 256) {
          const int t = i / half, p = i - t * half;
          if (f + t >= lo && f + t < hi) {
            double s, c;
            sincos_f64((double)a.pos[sp.r0 + (f + t - slot0)] * a.t.freq[p], s, c);
            cs[i] = make_double2(c * a.t.mag, s * a.t.mag);
          }
        }
        __syncthreads();
      }
#pragma unroll
      for (int it = 0; it < L::NG / 2; ++it) {
        const int t = (tid >> 3) & 15, g = 2 * it + (tid >> 7), d0 = 32 * g + 4 * c8;
        const int slot = f + t;
        const bool in = slot >= lo && slot < hi;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (in) {
          const T* row = (const T*)a.k + (size_t)(sp.r0 + (slot - slot0)) * a.ks + (size_t)hk * D;
          load4(row + d0, x);
          if constexpr (ROPE) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = d0 + e;
              y[e] = x[e];
              if (d < a.t.rot_dim) {
                const bool second = a.t.interleaved ? (d & 1) : d >= half;
                const int p = a.t.interleaved ? d >> 1 : second ? d - half : d;
                const float o = a.t.interleaved ? x[e ^ 1] : (float)row[second ? d - half : d + half];
                const double2 w = cs[t * half + p];
                // (a c - b s, a s + b c), rounded to f32 once.
                y[e] = (float)(second ? __builtin_fma((double)o, w.y, (double)x[e] * w.x)
                                      : __builtin_fma((double)x[e], w.x, -((double)o * w.y)));
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = y[e];
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
        const int tok = p0 + 16 * tile + t;
        if (in && !(c8 & 1)) *reinterpret_cast<uint32_t*>(base + L::key_word(tok, g, c8 >> 1)) = w;
        if (in && c8 == 0) {
          if (q.bad) bad[16 * tile + t] = 1;
          *reinterpret_cast<_Float16*>(base + L::key_d(tok, g)) = (_Float16)q.d;
          *reinterpret_cast<_Float16*>(base + L::key_m(tok, g)) = (_Float16)q.m;
        }
      }
    }
    const bool whole = s0 >= lo && s0 + 32 <= hi;
    for (int i = tid; i < 4 * D; i += 256) {
      const int rg = i / D, d = i - rg * D;
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
      uint32_t* p = reinterpret_cast<uint32_t*>(base + L::value_word(p0 + 4 * rg, d));
      if (whole) *p = w;
      else if (mine) *p = (*p & ~mine) | w;
    }
    __syncthreads();
    // (A slot that is not this call's has no flag.)
    if (tid < 32 && bad[tid]) {
#pragma unroll
      for (int g = 0; g < L::NG; ++g) *reinterpret_cast<uint16_t*>(base + L::key_d(p0 + tid, g)) = 0x7E00;
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

// One workgroup per (32 slots, kv head, sequence), a thread per dword.
template <int D, class T>
__global__ __launch_bounds__(256) void kv4_read(ReadArgs a) {
  using L = Kv4L<D>;
  const int hk = blockIdx.y, b = blockIdx.z;
  const Kv4Span sp = kv4_span(a.rows, b);
  const int n = sp.r1 - sp.r0, slot0 = sp.len - n;
  const int lo = max(slot0, 0), hi = sp.len;
  if (n <= 0 || lo >= hi) return;
  for (int blk = (lo >> 5) + blockIdx.x; blk <= (hi - 1) >> 5; blk += gridDim.x) {
    const uint8_t* base = kv4_block(a.c, b, blk >> 1, hk, L::BYTES);
    const int s0 = blk << 5, p0 = (blk & 1) * 32;
    for (int i = threadIdx.x; i < 4 * D; i += 256) {
      {  // key dword: token i / (D / 8), dims 8 (i % (D / 8)) ..
        const int t = i / (D / 8), d0 = (i % (D / 8)) * 8, slot = s0 + t;
        if (slot >= lo && slot < hi) {
          struct { T v[8]; } o;
          uint32_t w = 0;
          float d = __builtin_nanf(""), m = 0.f;
          if (base) {
            w = *reinterpret_cast<const uint32_t*>(base + L::key_word(p0 + t, d0 >> 5, (d0 >> 3) & 3));
            d = kv4_f16(base + L::key_d(p0 + t, d0 >> 5));
            m = kv4_f16(base + L::key_m(p0 + t, d0 >> 5));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) o.v[j] = (T)__builtin_fmaf(d, (float)kv4_code(w, j), m);
          __builtin_memcpy((T*)a.k + (size_t)(sp.r0 + (slot - slot0)) * a.ks + (size_t)hk * D + d0, &o, sizeof(o));
        }
      }
      const int rg = i / D, d = i - rg * D;
      uint32_t w = 0;
      if (base) w = *reinterpret_cast<const uint32_t*>(base + L::value_word(p0 + 4 * rg, d));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = 16 * (j >> 2) + 4 * rg + (j & 3), slot = s0 + t;
        if (slot >= lo && slot < hi) {
          float dd = __builtin_nanf(""), m = 0.f;
          if (base && kv4_f16(base + L::key_d(p0 + t, 0)) >= 0.f) {
            dd = kv4_f16(base + L::value_d(p0 + t, d >> 5));
            m = kv4_f16(base + L::value_m(p0 + t, d >> 5));
          }
          ((T*)a.v)[(size_t)(sp.r0 + (slot - slot0)) * a.vs + (size_t)hk * D + d] =
              (T)__builtin_fmaf(dd, (float)kv4_code(w, j), m);
        }
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

// Inclusive sum over the workgroup's 1024 threads; *total gets the whole.
__device__ __forceinline__ int wg_scan(int v, int* part, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 63) part[w] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int p = part[i];
    if (i < w) before += p;
    all += p;
  }
  *total = all;
  return v + before;
}

// One workgroup per (kv head, sequence): the rank of the lightest slot kept,
// by its four bytes from the top (a histogram of those still in question per
// byte), then the kept slots in order.  Among slots of that rank the lowest
// stay.  new_len is the same for every head; head 0 writes it.
__global__ __launch_bounds__(1024) void kv4_select(Kv4Evict e, int n_kv) {
  __shared__ int hist[256];
  __shared__ int part[16];
  __shared__ int pick[2];
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int n = max(e.kv_len[b], 0), kept = min(n, e.keep);
  const float* acc = e.acc + ((size_t)b * n_kv + hk) * e.acc_stride;
  int* idx = e.idx + ((size_t)b * n_kv + hk) * e.keep;
  float* out = e.acc_out + ((size_t)b * n_kv + hk) * e.keep;
  auto weight = [&](int i) { return i < e.acc_stride ? acc[i] : 0.f; };
  if (hk == 0 && tid == 0) e.new_len[b] = kept;
  for (int i = kept + tid; i < e.keep; i += 1024) {
    idx[i] = -1;
    out[i] = 0.f;
  }
  if (n <= e.keep) {
    for (int i = tid; i < n; i += 1024) {
      idx[i] = i;
      out[i] = weight(i);
    }
    return;
  }
  const int m0 = e.first, m1 = n - e.recent;  // the slots in question
  int need = e.keep - e.first - e.recent;
  uint32_t top = 0, mask = 0;
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = m0 + tid; i < m1; i += 1024) {
        const uint32_t k = evict_key(weight(i));
        if ((k & mask) == top) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int v = 255, left = need;
        while (v > 0 && hist[v] < left) left -= hist[v--];
        pick[0] = v;
        pick[1] = left;
      }
      __syncthreads();
      top |= (uint32_t)pick[0] << shift;
      mask |= 255u << shift;
      need = pick[1];
      __syncthreads();
    }
  }
  // Slots above `top` stay, and the first `need` of those equal to it.
  int at = 0, ties = 0;
  for (int i0 = 0; i0 < n; i0 += 1024) {
    const int i = i0 + tid;
    float v = 0.f;
    bool keep = false, tie = false;
    if (i < n) {
      v = weight(i);
      const uint32_t k = evict_key(v);
      if (i < m0 || i >= m1) keep = true;
      else if (mask) {
        keep = k > top;
        tie = k == top;
      }
    }
    int total;
    const int rank = wg_scan(tie, part, &total);
    if (tie && ties + rank <= need) keep = true;
    ties += total;
    const int place = wg_scan(keep, part, &total);
    if (keep) {
      idx[at + place - 1] = i;
      out[at + place - 1] = v;
    }
    at += total;
  }
}

// One workgroup per (32 new slots, kv head, sequence): keys and scales of a
// token are whole words; a value dword collects one code from each of eight
// old ones.  Slots of a page that the source's table does not have read as
// NaN.
template <int D>
__global__ __launch_bounds__(256) void kv4_gather(Kv4View src, Kv4View dst, Kv4Evict e) {
  using L = Kv4L<D>;
  __shared__ int from[32];
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int kept = min(max(e.kv_len[b], 0), e.keep);
  const int s0 = blockIdx.x * 32;
  if (s0 >= kept) return;
  uint8_t* to = kv4_block(dst, b, s0 / KV4_PAGE, hk, L::BYTES);
  if (!to) return;
  const int p0 = s0 & 32;
  if (tid < 32) from[tid] = s0 + tid < kept ? e.idx[((size_t)b * src.n_kv + hk) * e.keep + s0 + tid] : -1;
  __syncthreads();
  // Keys and all scales: (token, 32-bit word).
  constexpr int KW = D / 8, SW = L::NG;  // code words, and words of (d, m) pairs per side
  for (int i = tid; i < 32 * (KW + 2 * SW); i += 256) {
    const int t = i / (KW + 2 * SW), w = i % (KW + 2 * SW);
    const int f = from[t];
    if (f < 0) continue;
    const uint8_t* s = kv4_block(src, b, f / KV4_PAGE, hk, L::BYTES);
    const int ft = f % KV4_PAGE, tt = p0 + t;
    if (w < KW) {
      uint32_t c = 0;
      if (s) c = *reinterpret_cast<const uint32_t*>(s + L::key_word(ft, w >> 2, w & 3));
      *reinterpret_cast<uint32_t*>(to + L::key_word(tt, w >> 2, w & 3)) = c;
    } else {
      const int g = (w - KW) % SW;
      const bool val = w - KW >= SW;
      const int sd = val ? L::value_d(ft, g) : L::key_d(ft, g), sm = val ? L::value_m(ft, g) : L::key_m(ft, g);
      const int td = val ? L::value_d(tt, g) : L::key_d(tt, g), tm = val ? L::value_m(tt, g) : L::key_m(tt, g);
      *reinterpret_cast<uint16_t*>(to + td) = s ? *reinterpret_cast<const uint16_t*>(s + sd) : (uint16_t)0x7E00;
      *reinterpret_cast<uint16_t*>(to + tm) = s ? *reinterpret_cast<const uint16_t*>(s + sm) : (uint16_t)0;
    }
  }
  // Value dwords, four dims (16 apart) of a thread together.
  for (int i = tid; i < D; i += 256) {
    const int l = i & 63, ch = i >> 6, rg = l >> 4, dim = 64 * ch + (l & 15);
    kvu4 w = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int f = from[16 * (j >> 2) + 4 * rg + (j & 3)];
      if (f < 0) continue;
      const uint8_t* s = kv4_block(src, b, f / KV4_PAGE, hk, L::BYTES);
      if (!s) continue;
      const int ft = f % KV4_PAGE;
      const kvu4 o = *reinterpret_cast<const kvu4*>(s + L::value_word(ft, dim));
      const uint32_t fj = (uint32_t)L::value_j(ft);
      // kv4_bit of a run-time j: 6, 22, 2, 18, 14, 30, 10, 26.
      const uint32_t bit = ((fj & 1) << 4) + ((0xAE26u >> ((fj >> 1) << 2)) & 15u);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t c = __builtin_amdgcn_alignbit(o[k], o[k], bit) & 15u;
        w[k] |= __builtin_amdgcn_alignbit(c, c, (uint32_t)((32 - kv4_bit(j)) & 31));
      }
    }
    *reinterpret_cast<kvu4*>(to + L::value_word(p0 + 4 * rg, dim)) = w;
  }
}

hipError_t launch_kv4_evict(int head_dim, const Kv4View& src, const Kv4View& dst, const Kv4Evict& e, hipStream_t s) {
  hipLaunchKernelGGL(kv4_select, dim3(src.n_kv, e.n_seq), dim3(1024), 0, s, e, src.n_kv);
  const dim3 grid((e.keep + 31) / 32, src.n_kv, e.n_seq);
  if (head_dim == 64) hipLaunchKernelGGL((kv4_gather<64>), grid, dim3(256), 0, s, src, dst, e);
  else if (head_dim == 128) hipLaunchKernelGGL((kv4_gather<128>), grid, dim3(256), 0, s, src, dst, e);
  else hipLaunchKernelGGL((kv4_gather<256>), grid, dim3(256), 0, s, src, dst, e);
  return hipGetLastError();
}

}  // namespace kq
