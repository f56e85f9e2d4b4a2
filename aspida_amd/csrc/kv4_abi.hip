// kv4_abi.hip -- C entry points of the rotary positions, the 4-bit key/value
// cache and trees of drafted tokens (contracts: include/aspidagpu.h).  Arguments that the host
// can see are checked here; lengths, row starts and page ids live on the
// device and are bounded by the kernels.
#include <cerrno>
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>

#include "../../include/aspidagpu.h"
#include "kv4.h"
#include "tree.h"

namespace kq {
void abi_report(int code, const char* what);  // aspidagpu.hip: the calling thread's aspida_gpu_last_error
}

namespace {

int done(hipError_t e, const char* what) {
  if (e == hipSuccess) return 0;
  kq::abi_report((int)e, what);
  return (int)e;
}

int type_bytes(int type) { return type == 0 ? 4 : type == 1 || type == 2 ? 2 : 0; }
bool aligned(const void* p, size_t n) { return p && ((uintptr_t)p & (n - 1)) == 0; }

bool valid_cache(const aspida_kv4* c) {
  return c && (c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256) && c->n_kv >= 1 && c->n_kv <= 65535 &&
         c->n_pages >= 1 && c->max_pages >= 1 && c->max_pages <= (1 << 24) && aligned(c->pages, 16) &&
         aligned(c->table, 4);
}

kq::Kv4View view(const aspida_kv4* c) {
  return {(uint8_t*)c->pages, c->table, c->n_kv, c->n_pages, c->max_pages};
}

// Rows of n_seq sequences; -EINVAL, or 1 where there is nothing to do.
int rows_of(int n_rows, int n_seq, const int* row_start, const int* kv_len, kq::Kv4Rows& r) {
  if (n_rows < 0 || n_seq < 0 || n_seq > 65535) return -EINVAL;
  if (n_rows == 0 || n_seq == 0) return 1;
  if (!aligned(kv_len, 4) || (row_start ? !aligned(row_start, 4) : n_rows != n_seq)) return -EINVAL;
  r = {row_start, kv_len, n_rows, n_seq};
  return 0;
}

// A [rows][heads][head_dim] operand of `type`, rows `stride` elements apart.
bool valid_rows(const void* p, int type, long long stride, int heads, int head_dim) {
  return type_bytes(type) && aligned(p, (size_t)type_bytes(type)) && stride >= (long long)heads * head_dim;
}

// The bound on a sequence's rows that grids are cut for: never above all rows.
int longest(int max_rows, int n_rows) { return std::min(max_rows, std::max(n_rows, 1)); }

bool valid_heads(const aspida_kv4* c, int n_heads) {
  return n_heads >= 1 && n_heads <= 65535 && n_heads % c->n_kv == 0;
}

}  // namespace

extern "C" void* aspida_rope_create(const aspida_rope_params* p) {
  auto bad = [](const char* why) -> void* {
    kq::abi_report(-EINVAL, why);
    return nullptr;
  };
  if (!p || p->rot_dim < 2 || p->rot_dim > kq::ROPE_MAX_ROT || p->rot_dim % 2)
    return bad("aspida_rope_create: rot_dim must be even, 2 to 256");
  if (!(p->base > 1.0) || !std::isfinite(p->base)) return bad("aspida_rope_create: base must be above 1");
  if (p->scaling < 0 || p->scaling > 3) return bad("aspida_rope_create: unknown scaling");
  if (p->scaling != 0 && !(p->factor > 0.0 && std::isfinite(p->factor)))
    return bad("aspida_rope_create: factor must be positive");
  if (p->scaling >= 2 && !(p->low > 0.0 && p->high > p->low && std::isfinite(p->high) && p->context > 0.0 &&
                           std::isfinite(p->context)))
    return bad("aspida_rope_create: bands need 0 < low < high and a context");
  if (!(p->magnitude >= 0.0) || !std::isfinite(p->magnitude))
    return bad("aspida_rope_create: magnitude must be finite and not negative");
  kq::RopeTable* t = new (std::nothrow) kq::RopeTable();
  if (!t) {
    kq::abi_report(-ENOMEM, "aspida_rope_create");
    return nullptr;
  }
  const double pi = 3.14159265358979323846;
  const int half = p->rot_dim / 2;
  double lo = 0.0, hi = 0.0;
  if (p->scaling == 3) {
    // The pair whose angle turns `turns` times over the context.
    auto at = [&](double turns) {
      return p->rot_dim * std::log(p->context / (turns * 2.0 * pi)) / (2.0 * std::log(p->base));
    };
    lo = std::fmax(std::floor(at(p->high)), 0.0);
    hi = std::fmin(std::ceil(at(p->low)), (double)(p->rot_dim - 1));
  }
  for (int i = 0; i < half; ++i) {
    double f = std::pow(p->base, -2.0 * i / p->rot_dim);
    if (p->freq_factors) {
      const double ff = (double)p->freq_factors[i];
      if (!(ff > 0.0) || !std::isfinite(ff)) {
        delete t;
        return bad("aspida_rope_create: freq_factors must be positive");
      }
      f /= ff;
    }
    if (p->scaling == 1) {
      f /= p->factor;
    } else if (p->scaling == 2) {
      const double turns = p->context * f / (2.0 * pi);
      const double s = std::fmin(1.0, std::fmax(0.0, (turns - p->low) / (p->high - p->low)));
      f = (1.0 - s) * f / p->factor + s * f;
    } else if (p->scaling == 3) {
      const double ramp = std::fmin(1.0, std::fmax(0.0, (i - lo) / std::fmax(hi - lo, 0.001)));
      f = f / p->factor * ramp + f * (1.0 - ramp);
    }
    if (!(f <= kq::ROPE_MAX_FREQ)) {
      delete t;
      return bad("aspida_rope_create: a pair turns by more than 2^19 a position");
    }
    t->freq[i] = f;
  }
  t->mag = p->magnitude > 0.0 ? p->magnitude : p->scaling == 3 ? 0.1 * std::log(p->factor) + 1.0 : 1.0;
  t->rot_dim = p->rot_dim;
  t->interleaved = p->interleaved ? 1 : 0;
  return t;
}

extern "C" void aspida_rope_destroy(void* rope) { delete (kq::RopeTable*)rope; }

extern "C" int aspida_rope_table(const void* rope, double* freq, double* magnitude) {
  if (!rope || !freq || !magnitude) return -EINVAL;
  const kq::RopeTable* t = (const kq::RopeTable*)rope;
  for (int i = 0; i < t->rot_dim / 2; ++i) freq[i] = t->freq[i];
  *magnitude = t->mag;
  return 0;
}

extern "C" int aspida_rope_dev(const void* rope, int type, const void* x, long long x_stride, int n_tok, int n_heads,
                               int head_dim, const int* pos, int inverse, void* y, long long y_stride, void* stream) {
  const kq::RopeTable* t = (const kq::RopeTable*)rope;
  if (!t || n_tok < 0 || n_heads < 1 || n_heads > 65535 || head_dim < t->rot_dim || head_dim > 65536) return -EINVAL;
  if (n_tok == 0) return 0;
  if (!valid_rows(x, type, x_stride, n_heads, head_dim) || !valid_rows(y, type, y_stride, n_heads, head_dim) ||
      !aligned(pos, 4) || (x == y && x_stride != y_stride))
    return -EINVAL;
  if (!kq::rope_takes(*t, type, head_dim)) return -ENOTSUP;
  return done(kq::launch_rope(*t, type, x, x_stride, n_tok, n_heads, head_dim, pos, inverse != 0, y, y_stride,
                              (hipStream_t)stream),
              "aspida_rope_dev");
}

extern "C" long long aspida_kv4_page_bytes(int head_dim, int n_kv) {
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || n_kv < 1 || n_kv > 65535) return 0;
  return (long long)kq::kv4_head_bytes(head_dim) * n_kv;
}

extern "C" int aspida_kv4_append_dev(const aspida_kv4* cache, int type, const void* k, long long k_stride,
                                     const void* v, long long v_stride, int n_rows, int n_seq, const int* row_start,
                                     const int* kv_len, const void* rope, const int* pos, void* stream) {
  if (!valid_cache(cache)) return -EINVAL;
  kq::Kv4Rows r;
  if (const int rc = rows_of(n_rows, n_seq, row_start, kv_len, r)) return rc < 0 ? rc : 0;
  const kq::RopeTable* t = (const kq::RopeTable*)rope;
  if (!valid_rows(k, type, k_stride, cache->n_kv, cache->head_dim) ||
      !valid_rows(v, type, v_stride, cache->n_kv, cache->head_dim) ||
      (t && (t->rot_dim > cache->head_dim || !aligned(pos, 4))))
    return -EINVAL;
  return done(kq::launch_kv4_append(cache->head_dim, view(cache), type, k, k_stride, v, v_stride, r, t, pos,
                                    (hipStream_t)stream),
              "aspida_kv4_append_dev");
}

extern "C" int aspida_kv4_read_dev(const aspida_kv4* cache, int type, int n_rows, int n_seq, const int* row_start,
                                   const int* kv_len, void* k, long long k_stride, void* v, long long v_stride,
                                   void* stream) {
  if (!valid_cache(cache)) return -EINVAL;
  kq::Kv4Rows r;
  if (const int rc = rows_of(n_rows, n_seq, row_start, kv_len, r)) return rc < 0 ? rc : 0;
  if (!valid_rows(k, type, k_stride, cache->n_kv, cache->head_dim) ||
      !valid_rows(v, type, v_stride, cache->n_kv, cache->head_dim))
    return -EINVAL;
  return done(kq::launch_kv4_read(cache->head_dim, view(cache), type, r, k, k_stride, v, v_stride,
                                  (hipStream_t)stream),
              "aspida_kv4_read_dev");
}

extern "C" long long aspida_kv4_attn_work_bytes(const aspida_kv4* cache, int n_heads, int n_rows, int n_seq,
                                                int max_rows) {
  if (!valid_cache(cache) || !valid_heads(cache, n_heads) || n_rows < 0 || n_seq < 0 || n_seq > 65535 || max_rows < 1)
    return -EINVAL;
  return (long long)kq::kv4_attn_work_bytes(cache->head_dim);
}

extern "C" int aspida_kv4_attn_dev(const aspida_kv4* cache, int type, const void* q, long long q_stride, int n_heads,
                                   int n_rows, int n_seq, const int* row_start, int max_rows, const int* kv_len,
                                   float scale, int window, void* out, long long out_stride, float* lse, void* work,
                                   void* stream) {
  if (!valid_cache(cache) || !valid_heads(cache, n_heads) || max_rows < 1 || window < 0 || !std::isfinite(scale))
    return -EINVAL;
  kq::Kv4Rows r;
  if (const int rc = rows_of(n_rows, n_seq, row_start, kv_len, r)) return rc < 0 ? rc : 0;
  if (!valid_rows(q, type, q_stride, n_heads, cache->head_dim) ||
      !valid_rows(out, type, out_stride, n_heads, cache->head_dim) || (lse && !aligned(lse, 4)) ||
      !aligned(work, 256))
    return -EINVAL;
  kq::Kv4Attn a{q, q_stride, out, out_stride, lse, work, n_heads, longest(max_rows, n_rows), window, scale, nullptr, 0};
  return done(kq::launch_kv4_attn(cache->head_dim, view(cache), type, r, a, (hipStream_t)stream),
              "aspida_kv4_attn_dev");
}

extern "C" int aspida_kv4_weigh_dev(const aspida_kv4* cache, int type, const void* q, long long q_stride, int n_heads,
                                    int n_rows, int n_seq, const int* row_start, int max_rows, const int* kv_len,
                                    float scale, int window, const float* lse, const float* acc_in, float* acc_out,
                                    long long acc_stride, void* stream) {
  if (!valid_cache(cache) || !valid_heads(cache, n_heads) || max_rows < 1 || window < 0 || !std::isfinite(scale))
    return -EINVAL;
  kq::Kv4Rows r;
  if (const int rc = rows_of(n_rows, n_seq, row_start, kv_len, r)) return rc < 0 ? rc : 0;
  if (!valid_rows(q, type, q_stride, n_heads, cache->head_dim) || !aligned(lse, 4) ||
      (acc_in && !aligned(acc_in, 4)) || !aligned(acc_out, 4) || acc_stride < 1)
    return -EINVAL;
  kq::Kv4Weigh w{q, q_stride, lse, acc_in, acc_out, acc_stride, n_heads, longest(max_rows, n_rows), window, scale};
  return done(kq::launch_kv4_weigh(cache->head_dim, view(cache), type, r, w, (hipStream_t)stream),
              "aspida_kv4_weigh_dev");
}

extern "C" int aspida_kv4_evict_dev(const aspida_kv4* src, int n_seq, const int* kv_len, const float* acc,
                                    long long acc_stride, int keep, int first, int recent, const aspida_kv4* dst,
                                    int* new_len, int* idx, float* acc_out, void* stream) {
  if (!valid_cache(src) || !valid_cache(dst) || src->head_dim != dst->head_dim || src->n_kv != dst->n_kv ||
      n_seq < 0 || n_seq > 65535 || keep < 1 || first < 0 || recent < 0 || first > keep - recent || acc_stride < 1 ||
      keep > (long long)dst->max_pages * kq::KV4_PAGE)
    return -EINVAL;
  if (n_seq == 0) return 0;
  if (!aligned(kv_len, 4) || !aligned(acc, 4) || !aligned(new_len, 4) || !aligned(idx, 4) || !aligned(acc_out, 4))
    return -EINVAL;
  kq::Kv4Evict e{kv_len, acc, acc_stride, n_seq, keep, first, recent, new_len, idx, acc_out};
  return done(kq::launch_kv4_evict(src->head_dim, view(src), view(dst), e, (hipStream_t)stream),
              "aspida_kv4_evict_dev");
}

extern "C" int aspida_tree_dev(const int* parent, int n_rows, int n_seq, const int* row_start, const int* kv_len,
                               int* pos, unsigned* mask, int mask_words, void* stream) {
  kq::Kv4Rows r;
  if (mask && (mask_words < 1 || mask_words > kq::TREE_MAX_WORDS)) return -EINVAL;
  if (const int rc = rows_of(n_rows, n_seq, row_start, kv_len, r)) return rc < 0 ? rc : 0;
  if (!aligned(parent, 4) || (pos && !aligned(pos, 4)) || (mask && !aligned(mask, 4))) return -EINVAL;
  return done(kq::launch_tree({parent, r.row_start, r.kv_len, n_rows, n_seq}, pos, mask, mask_words,
                              (hipStream_t)stream),
              "aspida_tree_dev");
}

extern "C" long long aspida_kv4_tree_attn_work_bytes(const aspida_kv4* cache, int n_heads, int n_rows, int n_seq,
                                                     int max_rows) {
  if (!valid_cache(cache) || !valid_heads(cache, n_heads) || n_rows < 0 || n_seq < 0 || n_seq > 65535 || max_rows < 1 ||
      max_rows > kq::TREE_MAX_ROWS)
    return -EINVAL;
  return (long long)kq::kv4_tree_work_bytes(cache->head_dim, longest(max_rows, n_rows), n_heads / cache->n_kv);
}

extern "C" int aspida_kv4_tree_attn_dev(const aspida_kv4* cache, int type, const void* q, long long q_stride,
                                        int n_heads, int n_rows, int n_seq, const int* row_start, int max_rows,
                                        const int* kv_len, const unsigned* mask, int mask_words, float scale,
                                        int window, void* out, long long out_stride, float* lse, void* work,
                                        void* stream) {
  if (!valid_cache(cache) || !valid_heads(cache, n_heads) || max_rows < 1 || max_rows > kq::TREE_MAX_ROWS ||
      mask_words < 1 || mask_words > kq::TREE_MAX_WORDS || window < 0 || !std::isfinite(scale))
    return -EINVAL;
  kq::Kv4Rows r;
  if (const int rc = rows_of(n_rows, n_seq, row_start, kv_len, r)) return rc < 0 ? rc : 0;
  if (!valid_rows(q, type, q_stride, n_heads, cache->head_dim) ||
      !valid_rows(out, type, out_stride, n_heads, cache->head_dim) || !aligned(mask, 4) || (lse && !aligned(lse, 4)) ||
      !aligned(work, 256))
    return -EINVAL;
  const int rows = longest(max_rows, n_rows);
  // Column tiles of all kv heads are a dimension of the launch.
  if (((long long)rows * (n_heads / cache->n_kv) + 15) / 16 * cache->n_kv > 65535) return -ENOTSUP;
  kq::Kv4Attn a{q, q_stride, out, out_stride, lse, work, n_heads, rows, window, scale, mask, mask_words};
  return done(kq::launch_kv4_tree(cache->head_dim, view(cache), type, r, a, (hipStream_t)stream),
              "aspida_kv4_tree_attn_dev");
}

extern "C" int aspida_kv4_keep_dev(const aspida_kv4* cache, int n_rows, int n_seq, const int* row_start,
                                   const int* kv_len, const int* path, const int* count, void* stream) {
  if (!valid_cache(cache)) return -EINVAL;
  kq::Kv4Rows r;
  if (const int rc = rows_of(n_rows, n_seq, row_start, kv_len, r)) return rc < 0 ? rc : 0;
  if (!aligned(path, 4) || !aligned(count, 4)) return -EINVAL;
  return done(kq::launch_kv4_keep(cache->head_dim, view(cache), r, path, count, (hipStream_t)stream),
              "aspida_kv4_keep_dev");
}

extern "C" long long aspida_tree_accept_work_bytes(int n_rows, int vocab) {
  if (n_rows < 0 || n_rows > (1 << 22) || vocab < 1 || vocab > (1 << 30)) return -EINVAL;
  return (long long)kq::tree_accept_work_bytes(n_rows > 0 ? n_rows : 1, vocab);
}

extern "C" int aspida_tree_accept_dev(int type, const void* logits, long long stride, int vocab, int n_rows, int n_seq,
                                      const int* row_start, const int* kv_len, const int* parent, const int* token,
                                      int* path, int* count, int* next, int* new_len, void* work, void* stream) {
  if (!type_bytes(type) || vocab < 1 || vocab > (1 << 30) || stride < vocab || n_rows > (1 << 22)) return -EINVAL;
  kq::Kv4Rows r;
  if (const int rc = rows_of(n_rows, n_seq, row_start, kv_len, r)) return rc < 0 ? rc : 0;
  if (!aligned(logits, (size_t)type_bytes(type)) || !aligned(parent, 4) || !aligned(token, 4) || !aligned(path, 4) ||
      !aligned(count, 4) || !aligned(next, 4) || !aligned(new_len, 4) || !aligned(work, 8))
    return -EINVAL;
  kq::TreeAccept a{logits, stride, vocab, token, path, count, next, new_len, work};
  return done(kq::launch_tree_accept(type, {parent, r.row_start, r.kv_len, n_rows, n_seq}, a, (hipStream_t)stream),
              "aspida_tree_accept_dev");
}
