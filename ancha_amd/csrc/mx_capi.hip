// C ABI entry points of the microscaled operators (include/ancha_hip.h): argument checks and dispatch.
#include <cstring>
#include <string>

#include "../../include/ancha_hip.h"
#include "mx.hpp"
#include "status.hpp"

namespace {

using ancha::fail;
using ancha::hip_fail;
using ancha::sticky;
namespace mx = ancha::mx;

constexpr size_t kIntMax = 0x7fffffff;

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
bool is_type(int t) { return t == ANCHA_HIP_F32 || t == ANCHA_HIP_F16 || t == ANCHA_HIP_BF16; }
bool is_format(int f) { return f == ANCHA_HIP_MX_FP8 || f == ANCHA_HIP_MX_FP4; }

// rows x dim values as fewer than 2^27 stored groups, so that sixteen or 32 threads a group (a row's in the norm)
// stay below HIP's 2^32, in rows of at most 2^26 values.
bool units_fit(size_t rows, size_t dim) {
  return rows <= kIntMax && dim <= size_t(1) << 26 &&
         rows <= ((size_t(1) << 27) - 1024) / static_cast<size_t>(mx::groups(static_cast<long>(dim)));
}

// On the bits: the library is compiled without NaN semantics.
bool finite(double x) {
  volatile uint64_t bits;
  uint64_t b;
  std::memcpy(&b, &x, sizeof(b));
  bits = b;
  return (bits >> 52 & 0x7ff) != 0x7ff;
}

int check_codes(const std::string& who, const void* codes, const void* scales) {
  if (!codes || !scales) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if (!aligned(codes, 16) || !aligned(scales, 4))
    return fail(ANCHA_HIP_INVALID, who + ": codes must be 16-byte and scales 4-byte aligned");
  return 0;
}

int not_here(const std::string& who) {
  return fail(ANCHA_HIP_UNSUPPORTED, who + ": not a gfx950 device");
}

int run_rows(const char* name, const void* x, int type, size_t rows, size_t dim, size_t ldx,
             const void* residual, size_t ldr, const float* scale, double eps, bool norm, int format,
             void* sum, void* codes, void* scales, hipStream_t stream) {
  if (const int s = sticky()) return s;
  const std::string who(name);
  if (!is_type(type) || !is_format(format))
    return fail(ANCHA_HIP_INVALID, who + ": unknown type or format");
  if (ldx < dim || (residual && ldr < dim))
    return fail(ANCHA_HIP_INVALID, who + ": a row stride is smaller than dim");
  if (!finite(eps) || eps < 0.0) return fail(ANCHA_HIP_INVALID, who + ": eps is not a number >= 0");
  if (rows == 0 || dim == 0) return ANCHA_HIP_OK;
  if (!x || (residual && !sum)) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if ((residual && sum == x && ldx != dim) || (residual && sum == residual && ldr != dim))
    return fail(ANCHA_HIP_INVALID, who + ": the sum may replace contiguous rows only");
  if (const int e = check_codes(who, codes, scales)) return e;
  if (!units_fit(rows, dim)) return fail(ANCHA_HIP_UNSUPPORTED, who + ": too many rows or columns");
  if (!ancha_hip_available()) return not_here(who);
  mx::RowParams p{};
  p.x = x;
  p.residual = residual;
  p.scale = scale;
  p.sum = sum;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint8_t*>(scales);
  p.ldx = static_cast<long>(ldx);
  p.ldr = static_cast<long>(ldr);
  p.rows = static_cast<int>(rows);
  p.dim = static_cast<int>(dim);
  p.type = type;
  p.format = format;
  p.eps = eps;
  const hipError_t e = norm ? mx::launch_norm(p, stream) : mx::launch_quantize(p, stream);
  return e == hipSuccess ? ANCHA_HIP_OK : hip_fail(e, name);
}

// Strips and groups of a weight, one workgroup each; at most 2^23 k and 2^24 columns, so that a tile's 128
// rows of codes lie within 32 bits of its first, read and written.
bool weight_fits(size_t k, size_t m) {
  return k <= size_t(1) << 23 && m <= size_t(1) << 24 &&
         static_cast<size_t>(mx::strips(static_cast<long>(m))) *
                 static_cast<size_t>(mx::groups(static_cast<long>(k))) <
             (size_t(1) << 24);
}

}  // namespace

extern "C" {

size_t ancha_mx_pitch(size_t dim, int format) {
  return is_format(format) && dim <= kIntMax / 2 ? static_cast<size_t>(mx::pitch(static_cast<long>(dim), format)) : 0;
}

size_t ancha_mx_scales(size_t dim) {
  return dim <= kIntMax / 2 ? 4 * static_cast<size_t>(mx::groups(static_cast<long>(dim))) : 0;
}

int ancha_mx_quantize(const void* x, int type, size_t rows, size_t dim, size_t ldx, int format,
                      void* codes, void* scales, hipStream_t stream) {
  return run_rows("ancha_mx_quantize", x, type, rows, dim, ldx, nullptr, 0, nullptr, 0.0, false,
                  format, nullptr, codes, scales, stream);
}

int ancha_mx_norm(const void* x, int type, size_t rows, size_t dim, size_t ldx,
                  const void* residual, size_t ldr, const float* scale, double eps, int format,
                  void* sum, void* codes, void* scales, hipStream_t stream) {
  return run_rows("ancha_mx_norm", x, type, rows, dim, ldx, residual, ldr, scale, eps, true, format,
                  sum, codes, scales, stream);
}

int ancha_mx_values(const void* codes, const void* scales, size_t rows, size_t dim, int format,
                    int type, void* out, hipStream_t stream) {
  if (const int s = sticky()) return s;
  const std::string who("ancha_mx_values");
  if (!is_type(type) || !is_format(format))
    return fail(ANCHA_HIP_INVALID, who + ": unknown type or format");
  if (rows == 0 || dim == 0) return ANCHA_HIP_OK;
  if (!out) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if (const int e = check_codes(who, codes, scales)) return e;
  if (!units_fit(rows, dim)) return fail(ANCHA_HIP_UNSUPPORTED, who + ": too many rows or columns");
  if (!ancha_hip_available()) return not_here(who);
  mx::ValueParams p{};
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = static_cast<const uint8_t*>(scales);
  p.out = out;
  p.rows = static_cast<int>(rows);
  p.dim = static_cast<int>(dim);
  p.type = type;
  p.format = format;
  const hipError_t e = mx::launch_values(p, stream);
  return e == hipSuccess ? ANCHA_HIP_OK : hip_fail(e, who);
}

size_t ancha_mx_weight_bytes(size_t k, size_t m) {
  return k && m && weight_fits(k, m)
             ? static_cast<size_t>(mx::weight_bytes(static_cast<long>(k), static_cast<long>(m)))
             : 0;
}

int ancha_mx_weight(const void* w, int type, size_t k, size_t m, size_t ldk, size_t ldm,
                    void* weight, hipStream_t stream) {
  if (const int s = sticky()) return s;
  const std::string who("ancha_mx_weight");
  if (!is_type(type)) return fail(ANCHA_HIP_INVALID, who + ": unknown type");
  if (k == 0 || m == 0 || !weight_fits(k, m))
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": empty or too large a weight");
  if (!w || !weight) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if (!aligned(weight, 16)) return fail(ANCHA_HIP_INVALID, who + ": weight must be 16-byte aligned");
  if (!ancha_hip_available()) return not_here(who);
  mx::WeightParams p{};
  p.x = w;
  p.weight = static_cast<uint8_t*>(weight);
  p.ldk = static_cast<long>(ldk);
  p.ldm = static_cast<long>(ldm);
  p.k = static_cast<int>(k);
  p.m = static_cast<int>(m);
  p.type = type;
  const hipError_t e = mx::launch_weight(p, stream);
  return e == hipSuccess ? ANCHA_HIP_OK : hip_fail(e, who);
}

int ancha_mx_weight_values(const void* weight, size_t k, size_t m, int type, void* out,
                           hipStream_t stream) {
  if (const int s = sticky()) return s;
  const std::string who("ancha_mx_weight_values");
  if (!is_type(type)) return fail(ANCHA_HIP_INVALID, who + ": unknown type");
  if (k == 0 || m == 0 || !weight_fits(k, m))
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": empty or too large a weight");
  if (!weight || !out) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if (!aligned(weight, 16)) return fail(ANCHA_HIP_INVALID, who + ": weight must be 16-byte aligned");
  if (!ancha_hip_available()) return not_here(who);
  mx::WeightValueParams p{};
  p.weight = static_cast<const uint8_t*>(weight);
  p.out = out;
  p.k = static_cast<int>(k);
  p.m = static_cast<int>(m);
  p.type = type;
  const hipError_t e = mx::launch_weight_values(p, stream);
  return e == hipSuccess ? ANCHA_HIP_OK : hip_fail(e, who);
}

int ancha_mx_linear(const void* codes, const void* scales, size_t n, size_t k, int format,
                    const void* weight, size_t m, const float* bias, int gelu, const float* rope,
                    size_t tokens, size_t width, const void* residual, int type, int out_format,
                    void* out, void* out_scales, hipStream_t stream) {
  if (const int s = sticky()) return s;
  const std::string who("ancha_mx_linear");
  if (!is_type(type) || !is_format(format) || (out_format && !is_format(out_format)))
    return fail(ANCHA_HIP_INVALID, who + ": unknown type or format");
  if (out_format && type != ANCHA_HIP_F32)
    return fail(ANCHA_HIP_INVALID, who + ": an output in codes takes an fp32 residual");
  if (k == 0 || m == 0 || !weight_fits(k, m))
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": empty or too large a weight");
  if (rope && (tokens == 0 || n % tokens != 0 || width % 64 != 0 || width > m / 2))
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": rotary shape (tokens, width) does not fit");
  if (n == 0) return ANCHA_HIP_OK;
  if (!weight || !out) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if (const int e = check_codes(who, codes, scales)) return e;
  if (!aligned(weight, 16)) return fail(ANCHA_HIP_INVALID, who + ": weight must be 16-byte aligned");
  if (out_format)
    if (const int e = check_codes(who, out, out_scales)) return e;
  if (!units_fit(n, k) || !units_fit(n, m) ||
      static_cast<size_t>(mx::strips(static_cast<long>(m))) * ((n + 15) / 16) >= (size_t(1) << 26))
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": too many rows or columns");
  if (!ancha_hip_available()) return not_here(who);
  mx::LinearParams p{};
  p.x = static_cast<const uint8_t*>(codes);
  p.x_scales = static_cast<const uint8_t*>(scales);
  p.weight = static_cast<const uint8_t*>(weight);
  p.bias = bias;
  p.rope = rope;
  p.residual = residual;
  p.out = out;
  p.out_scales = static_cast<uint8_t*>(out_scales);
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.m = static_cast<int>(m);
  p.format = format;
  p.tokens = rope ? static_cast<int>(tokens) : 1;
  p.width = rope ? static_cast<int>(width) : 0;
  p.gelu = gelu ? 1 : 0;
  p.type = type;
  p.out_format = out_format;
  const hipError_t e = mx::launch_linear(p, stream);
  return e == hipSuccess ? ANCHA_HIP_OK : hip_fail(e, who);
}

// For the tests: the kernel that a product of n rows takes (mx::LinearForm).
int ancha_amd_mx_linear_form(size_t n, size_t k, size_t m) {
  return mx::linear_form(static_cast<long>(n), static_cast<long>(k), static_cast<long>(m));
}

// For the tests: the kernel that a norm takes, 8 x threads a row + pieces (0: rows read twice).
int ancha_amd_mx_norm_form(size_t rows, size_t dim) {
  return mx::norm_form(static_cast<long>(rows), static_cast<long>(dim));
}

}  // extern "C"
