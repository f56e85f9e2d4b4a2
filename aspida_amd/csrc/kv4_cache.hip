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
// The arithmetic is exact: a code never depends on how a quotient was rounded.
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

struct Kv4Group { float d, m; int q[8]; bool bad; };

// The spacing of 7-bit steps at d >= 0, a multiple of 2^-24.
__device__ __forceinline__ float kv4_step_ulp(float d) {
  const int e = (__builtin_bit_cast(int, d) & 0x7F800000) - (6 << 23);
  return __builtin_bit_cast(float, max(e, (127 - 24) << 23));
}

// The value of the lane that a row-wise pattern names.
template <int CTRL> __device__ __forceinline__ float kv4_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// Quantises a group from eight values in each of four neighbouring lanes.
// All in f32 but for the step, and exact all the same.  z = x - m rounded is
// a multiple of its ulp with an error e of half an ulp at most, and so are
// the ties (n + 1/2) d (d has 7 bits, 16 d > z): where z is no tie, x - m is
// on the same side of every tie as z.  The quotient t = z / d, corrected once
// by its exact remainder, is within 2^-45 before its last rounding: that gives
// a tie where z is one, and none where z is not, for then z is off by an ulp
// or more, which is more than half an ulp of t.  So rint(t) is the code, ties
// to even, unless z is a tie and e decides.
__device__ __forceinline__ Kv4Group kv4_quantise(const float (&x)[8]) {
  float lo = x[0], hi = x[0], odd = x[0] * 0.f;  // NaN where a value is not finite
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    odd = __builtin_fmaf(x[i], 0.f, odd);
  }
  lo = fminf(lo, kv4_dpp<0xB1>(lo));  // lanes 1 0 3 2
  hi = fmaxf(hi, kv4_dpp<0xB1>(hi));
  odd += kv4_dpp<0xB1>(odd);
  lo = fminf(lo, kv4_dpp<0x4E>(lo));  // 2 3 0 1
  hi = fmaxf(hi, kv4_dpp<0x4E>(hi));
  odd += kv4_dpp<0x4E>(odd);
  Kv4Group g;
  g.m = (float)(_Float16)lo;
  const double z = (double)hi - (double)g.m;
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
  if (odd != 0.f || !__builtin_isfinite(g.m) || !(d <= KV4_D_MAX)) {
    g.bad = true;
    g.d = g.m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) g.q[i] = 0;
    return g;
  }
  g.bad = false;
  g.d = d;
  const float inv = d > 0.f ? __builtin_amdgcn_rcpf(d) : 0.f;
  float z8[8], t[8], n[8];
  bool tie = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    z8[i] = x[i] - g.m;
    const float t0 = z8[i] * inv;
    t[i] = __builtin_fmaf(__builtin_fmaf(-t0, d, z8[i]), inv, t0);
    n[i] = __builtin_rintf(t[i]);
    tie |= __builtin_fabsf(t[i] - n[i]) == 0.5f;
  }
  if (tie) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // x - m = z + e; a tie moves to the side of e.
      const float back = z8[i] + g.m, e = (x[i] - back) - (g.m - (back - z8[i]));
      const float to = t[i] + (e > 0.f ? 0.5f : -0.5f);
      n[i] = e != 0.f && __builtin_fabsf(t[i] - n[i]) == 0.5f ? to : n[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) g.q[i] = (int)__builtin_amdgcn_fmed3f(n[i], 0.f, 15.f);
  return g;
}

// w with 4-bit code q, not yet in it, at its place j.
__device__ __forceinline__ uint32_t kv4_put(uint32_t w, uint32_t q, int j) {
  const int bit = kv4_bit(j);
  return w | (bit > 28 ? q << bit | q >> (32 - bit) : q << bit);
}

// One workgroup per (32 slots, sequence) and kv head, or several heads in
// turn for which the angles are formed once: a block of slots belongs to one
// workgroup, so the codes of a value dword that this call does not write are
// kept by a plain read and write of it.  Four lanes hold a group of a token,
// one key dword each; values pass through LDS, since a dword there holds
// eight tokens.
// One loop body serves values and keys, the next group's loads ahead of it
// (unrolled, 20 KB of code for a few rounds).  Frequencies go through LDS:
// arguments are far memory, and prompts of 7352 rows in all of 8 heads of 128
// (bf16) took 57 us with each pair's read from there, 34 now.  Bound by the
// vector units (77% of a busy unit's issue slots; without the angles, which
// each of the four workgroups of two heads forms anew, 24 us), copies of the
// same bytes take 8.  A single row passes through the body made for 32.
// How keys are rotated: not; values 8 i .. 8 i + 7 with others of that kind
// (half layout, rot_dim a multiple of 16); in any other way.
enum : int { ROPE_NONE, ROPE_EIGHTS, ROPE_ANY };

template <int D, class T, int ROPE>
__global__ __launch_bounds__(256) void kv4_append(AppendArgs a) {
  using L = Kv4L<D>;
  constexpr int NG = L::NG;
  // cos, sin of (pair p, token): 512 bytes a pair, and 64 more every eight
  // pairs, so that the four lanes of a group read from four parts of the banks.
  __shared__ double2 cs[ROPE ? 32 * D / 2 + D / 4 : 1];
  __shared__ double freq[ROPE ? D / 2 : 1];
  __shared__ uint8_t vq[32][D];
  __shared__ int bad[32];  // the token's key or value holds a group that the format does not
  const int b = blockIdx.y, tid = threadIdx.x;
  const Kv4Span sp = kv4_span(a.rows, b);
  const int n = sp.r1 - sp.r0, slot0 = sp.len - n;  // the first row's slot, below 0 where kv_len < n
  const int lo = max(slot0, 0), hi = min((long long)sp.len, (long long)a.c.max_pages * KV4_PAGE);
  if (n <= 0 || lo >= hi) return;
  const int half = a.t.rot_dim >> 1;
  const int kg = tid & 3, t = (tid >> 2) & 31, g0 = tid >> 7;  // groups g0, g0 + 2, ..
  auto angle = [](int p, int tok) { return 32 * p + 4 * (p >> 3) + tok; };
  if (ROPE && tid < half) freq[tid] = a.t.freq[tid];
  __syncthreads();
  for (int blk = (lo >> 5) + blockIdx.z; blk <= (hi - 1) >> 5; blk += gridDim.z) {
    uint8_t* page = kv4_block(a.c, b, blk >> 1, 0, L::BYTES);
    if (!page) continue;
    const int s0 = blk << 5, p0 = (blk & 1) * 32;  // first slot, and its token of the page
    const int t0 = max(lo - s0, 0), t1 = min(hi - s0, 32);  // the block's tokens of this call
    const bool whole = t1 - t0 == 32, in = t >= t0 && t < t1;
    // The nearest row of this call: what a slot of another has is not stored.
    const size_t row = (size_t)(sp.r0 + (s0 + min(max(t, t0), t1 - 1) - slot0));
    if constexpr (ROPE) {
      // As many threads a pair as the tokens need, in powers of two.
      const int sh = t1 - t0 > 1 ? 32 - __clz(t1 - t0 - 1) : 0, tok = t0 + (tid & ((1 << sh) - 1));
      if (tok < t1) {
        const double at = a.pos[sp.r0 + (s0 + tok - slot0)];
#pragma unroll 1
        for (int p = tid >> sh; p < half; p += 256 >> sh) {
          double s, c;
          sincos_f64(at * freq[p], s, c);
          cs[angle(p, tok)] = make_double2(c * a.t.mag, s * a.t.mag);
        }
      }
    }
    for (int hk = blockIdx.x; hk < a.c.n_kv; hk += gridDim.x) {
      uint8_t* base = page + (size_t)hk * L::BYTES;
      const T* k = (const T*)a.k + row * a.ks + (size_t)hk * D;
      const T* v = (const T*)a.v + row * a.vs + (size_t)hk * D;
      struct Values { T x[8]; };
      // A group's values, and those that its pairs have besides.
      auto load = [&](int it, Values& x, Values& o) {
        const bool key = it >= NG / 2;
        const int d0 = 32 * (g0 + 2 * (key ? it - NG / 2 : it)) + 8 * kg;
        const T* p = key ? k : v;
        __builtin_memcpy(&x, p + d0, sizeof(x));
        if constexpr (ROPE == ROPE_EIGHTS)
          __builtin_memcpy(&o, p + (d0 < half ? d0 + half : d0 < a.t.rot_dim ? d0 - half : d0), sizeof(o));
      };
      uint32_t old[D / 64];
      uint32_t* word[D / 64];
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {  // value dword (lane group rg, dim d)
        const int i = tid + 256 * c, rg = i / D, d = i % D;
        word[c] = reinterpret_cast<uint32_t*>(base + L::value_word(p0 + 4 * rg, d));
        old[c] = *word[c];
      }
      Values x, o;
      load(0, x, o);
      if (tid < 32) bad[tid] = 0;
      __syncthreads();
#pragma unroll 1
      for (int it = 0; it < NG; ++it) {
        Values nx, no;
        load(min(it + 1, NG - 1), nx, no);
        const bool key = it >= NG / 2;
        const int g = g0 + 2 * (key ? it - NG / 2 : it), d0 = 32 * g + 8 * kg;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (float)x.x[e];
        // (a c - b s, a s + b c), rounded to f32 once.
        if constexpr (ROPE == ROPE_EIGHTS) {
          if (key && d0 < a.t.rot_dim) {
            const bool second = d0 >= half;
            const double2* w = cs + angle(second ? d0 - half : d0, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float ot = o.x[e];
              y[e] = (float)__builtin_fma((double)(second ? ot : -ot), w[32 * e].y, (double)y[e] * w[32 * e].x);
            }
          }
        } else if constexpr (ROPE == ROPE_ANY) {
          if (key) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int d = d0 + e;
              if (d >= a.t.rot_dim) continue;
              const bool second = a.t.interleaved ? (d & 1) : d >= half;
              const double2 w = cs[angle(a.t.interleaved ? d >> 1 : second ? d - half : d, t)];
              const float ot = a.t.interleaved ? (float)x.x[e ^ 1] : (float)k[second ? d - half : d + half];
              y[e] = (float)__builtin_fma((double)(second ? ot : -ot), w.y, (double)y[e] * w.x);
            }
          }
        }
        const Kv4Group q = kv4_quantise(y);
        if (key) {
          uint32_t w = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) w = kv4_put(w, (uint32_t)q.q[e], e);
          if (in) *reinterpret_cast<uint32_t*>(base + L::key_word(p0 + t, g, kg)) = w;
        } else {
          kvu2 w = {0, 0};
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e >> 2] |= (uint32_t)q.q[e] << (8 * (e & 3));
          *reinterpret_cast<kvu2*>(&vq[t][32 * g + 8 * kg]) = w;
        }
        if (in && kg == 0) {
          if (q.bad) bad[t] = 1;
          const int d = key ? L::key_d(p0 + t, g) : L::value_d(p0 + t, g);
          *reinterpret_cast<_Float16*>(base + d) = (_Float16)q.d;
          *reinterpret_cast<_Float16*>(base + d + (key ? 2 * NG : 64 * NG)) = (_Float16)q.m;
        }
        x = nx;
        o = no;
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const int i = tid + 256 * c, rg = i / D, d = i % D;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w = kv4_put(w, vq[16 * (j >> 2) + 4 * rg + (j & 3)][d], j);
        if (!whole) {
          uint32_t mine = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int u = 16 * (j >> 2) + 4 * rg + (j & 3);
            if (u >= t0 && u < t1) mine = kv4_put(mine, 15u, j);
          }
          w = (w & mine) | (old[c] & ~mine);
        }
        *word[c] = w;
      }
      // (A slot that is not this call's has no flag.)
      if (tid < 32 && bad[tid]) {
        for (int g = 0; g < NG; ++g) *reinterpret_cast<uint16_t*>(base + L::key_d(p0 + tid, g)) = 0x7E00;
      }
      __syncthreads();
    }
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
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const Kv4Span sp = kv4_span(a.rows, b);
  const int n = sp.r1 - sp.r0, slot0 = sp.len - n;
  const int lo = max(slot0, 0), hi = sp.len;
  if (n <= 0 || lo >= hi) return;
  for (int blk = (lo >> 5) + blockIdx.z; blk <= (hi - 1) >> 5; blk += gridDim.z) {
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
// average sequence, and up to 4096 in all for longer ones, which otherwise take
// theirs in turns (prompts of 4097, 1013 and 2 rows: 57 us with 55 of 128
// blocks at a time).  They are the launch's last dimension: as its first, the
// few that short sequences use fell on two of the XCDs (32 lanes of 5 to 26 rows,
// 8 heads of 128, bf16, written and read back: 36 us, 11 now).
static unsigned blocks_of(const Kv4Rows& r, int n_kv) {
  const long long most = r.n_rows / 32 + 2, mean = ((long long)r.n_rows + r.n_seq - 1) / r.n_seq / 32 + 2;
  const long long room = 4096 / ((long long)n_kv * r.n_seq);
  return (unsigned)std::min<long long>(65535, std::min(most, std::max(mean, room)));
}

template <int D, class T>
static void append_go(const AppendArgs& a, bool rope, hipStream_t s) {
  const unsigned blocks = blocks_of(a.rows, a.c.n_kv);
  // Heads a workgroup takes in turn, as far as that leaves three workgroups a
  // compute unit (7352 rows of 8 heads: one 34.7 us, two 33.8).
  const long long all = ((long long)a.rows.n_rows / 32 + a.rows.n_seq) * a.c.n_kv;
  const int turns = rope ? (int)std::min<long long>(std::max<long long>(all / 768, 1), a.c.n_kv) : 1;
  const dim3 grid((a.c.n_kv + turns - 1) / turns, a.rows.n_seq, blocks);
  if (!rope) hipLaunchKernelGGL((kv4_append<D, T, ROPE_NONE>), grid, dim3(256), 0, s, a);
  else if (a.t.interleaved || a.t.rot_dim % 16) hipLaunchKernelGGL((kv4_append<D, T, ROPE_ANY>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((kv4_append<D, T, ROPE_EIGHTS>), grid, dim3(256), 0, s, a);
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
  const dim3 grid(a.c.n_kv, a.rows.n_seq, blocks_of(a.rows, a.c.n_kv));
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
// slots of that rank the lowest stay.  Bound by latencies, the weights being in
// cache after the first pass: eight are in flight per thread, bins are summed
// by all threads (by one thread, 256 bins: 56 us at 16 x 8 rows of 8193, now
// 12), and the ranks of 8192 slots come from ballots and one barrier.
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

// One workgroup per (page of 64 new slots, kv head, sequence).  Bound by the
// lines that it touches: slots kept here and there leave few lines of the old
// pages unread, whose pieces are 16 bytes a token (35 us of an eviction that
// writes 42 MB).  The key codes
// of a token are 16 bytes per lane group and quad and its key scales lie
// together; a value dword, and the 16 bytes of its scales, collect one entry
// from each of eight old tokens.  Slots of a page that the source's table does
// not have read as NaN: key steps of NaN, all else 0.  What stands in new
// slots past the last one is 0 where a word shares it.  The first page's
// workgroup of head 0 writes new_len: it may be kv_len, for here, unlike in
// the selection, both its values give the same slots.
template <int D>
__global__ __launch_bounds__(256) void kv4_gather(Kv4View src, Kv4View dst, Kv4Evict e) {
  using L = Kv4L<D>;
  constexpr int NG = L::NG;
  __shared__ const uint8_t* from[KV4_PAGE];  // the old block (or any memory of ours, unused)
  __shared__ int slot[KV4_PAGE];             // the old token in it, -1: none, -2: page missing
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int kept = min(max(e.kv_len[b], 0), e.keep);
  const int s0 = blockIdx.x * KV4_PAGE;
  if (s0 == 0 && hk == 0 && tid == 0) e.new_len[b] = kept;
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
