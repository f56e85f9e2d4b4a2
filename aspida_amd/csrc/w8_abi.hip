// w8_abi.hip -- C entry points of the products with 8-bit integer weights
// (contracts: include/aspidagpu.h).  Everything that a kernel assumes of sizes
// and addresses is checked here.
#include <cerrno>
#include <cstdint>

#include "../../include/aspidagpu.h"
#include "w8.h"

namespace kq {
void abi_report(int code, const char* what);  // aspidagpu.hip: the calling thread's aspida_gpu_last_error
}

namespace {

constexpr int MAX_ROWS = 1 << 22;  // of weights, and of tokens

int done(hipError_t e, const char* what) {
  if (e == hipSuccess) return 0;
  kq::abi_report((int)e, what);
  return (int)e;
}

bool aligned(const void* p, size_t n) { return p && ((uintptr_t)p & (n - 1)) == 0; }
bool valid_dims(int in_dim, int out_dim) {
  return in_dim >= 1 && in_dim <= kq::W8_MAX_IN && out_dim >= 1 && out_dim <= MAX_ROWS;
}

int product(const char* what, const void* w, const void* up, bool gated, int in_dim, int out_dim, int act, int type,
            const void* x, long long x_stride, int n_rows, void* y, long long y_stride, void* work, void* stream) {
  const size_t size = type == 0 ? 4 : type == 1 || type == 2 ? 2 : 0;
  if (!valid_dims(in_dim, out_dim) || !size || n_rows < 0 || n_rows > MAX_ROWS ||
      (long long)n_rows * out_dim > (1ll << 38) || (gated && (act < 0 || act > 1)))
    return -EINVAL;
  if (n_rows == 0) return 0;
  if (!aligned(w, 16) || (gated && !aligned(up, 16)) || !aligned(x, size) || !aligned(y, size) || x == y ||
      x_stride < in_dim || y_stride < out_dim || !aligned(work, 256))
    return -EINVAL;
  const kq::W8Args a{(const uint8_t*)w, gated ? (const uint8_t*)up : nullptr, in_dim, out_dim, n_rows, x, x_stride, y,
                     y_stride, (uint8_t*)work, act};
  return done(kq::launch_w8(type, a, (hipStream_t)stream), what);
}

}  // namespace

extern "C" long long aspida_w8_bytes(int in_dim, int out_dim) {
  return valid_dims(in_dim, out_dim) ? (long long)kq::w8_bytes(in_dim, out_dim) : -EINVAL;
}

extern "C" int aspida_w8_pack_dev(const signed char* codes, long long stride, const float* scale, int in_dim,
                                  int out_dim, void* packed, void* stream) {
  if (!valid_dims(in_dim, out_dim) || !codes || stride < in_dim || !aligned(scale, 4) || !aligned(packed, 16))
    return -EINVAL;
  return done(kq::launch_w8_pack((const int8_t*)codes, stride, scale, in_dim, out_dim, (uint8_t*)packed,
                                 (hipStream_t)stream),
              "aspida_w8_pack_dev");
}

extern "C" int aspida_w8_convert_dev(int kind, const void* w, int in_dim, int out_dim, void* packed, void* stream) {
  if (kind < -1 || kind > 5 || !valid_dims(in_dim, out_dim) || (kind >= 0 && in_dim % 256) ||
      !aligned(w, kind < 0 ? 4 : 1) || !aligned(packed, 16))
    return -EINVAL;
  return done(kq::launch_w8_convert(kind, w, in_dim, out_dim, (uint8_t*)packed, (hipStream_t)stream),
              "aspida_w8_convert_dev");
}

extern "C" int aspida_w8_unpack_dev(const void* packed, int in_dim, int out_dim, float* w, void* stream) {
  if (!valid_dims(in_dim, out_dim) || !aligned(packed, 16) || !aligned(w, 4)) return -EINVAL;
  return done(kq::launch_w8_unpack((const uint8_t*)packed, in_dim, out_dim, w, (hipStream_t)stream),
              "aspida_w8_unpack_dev");
}

extern "C" long long aspida_w8_work_bytes(int n_rows, int in_dim) {
  if (n_rows < 0 || n_rows > MAX_ROWS || in_dim < 1 || in_dim > kq::W8_MAX_IN) return -EINVAL;
  return (long long)kq::w8_bytes(in_dim, n_rows > 0 ? n_rows : 1);
}

extern "C" int aspida_w8_matmul_dev(const void* packed, int in_dim, int out_dim, int type, const void* x,
                                    long long x_stride, int n_rows, void* y, long long y_stride, void* work,
                                    void* stream) {
  return product("aspida_w8_matmul_dev", packed, nullptr, false, in_dim, out_dim, 0, type, x, x_stride, n_rows, y,
                 y_stride, work, stream);
}

extern "C" int aspida_w8_gated_dev(const void* gate, const void* up, int in_dim, int out_dim, int act, int type,
                                   const void* x, long long x_stride, int n_rows, void* y, long long y_stride,
                                   void* work, void* stream) {
  return product("aspida_w8_gated_dev", gate, up, true, in_dim, out_dim, act, type, x, x_stride, n_rows, y, y_stride,
                 work, stream);
}
