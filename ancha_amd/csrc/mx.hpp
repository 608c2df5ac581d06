// Microscaled (MX) operands of the gfx950 kernels: values in blocks of 32 along a row that share a
// power of two. A block with largest magnitude a > 0 has the scale byte
//   s = max(0, floor(log2 a) + 127 - E),   E = 8 for e4m3 ("fp8"), 2 for e2m1 ("fp4"),
// and each value v the code of v / 2^(s - 127), rounded to nearest even and saturated at 448 / 6. The
// division is exact, so the code is the only rounding. A block without a non-zero value has s = 0; one
// with a NaN or an infinity has s = 255 and codes 0: the matrix cores and the decoder make every value
// of it NaN.
//
// A row of dim values is stored as whole groups of 128: 128 (fp8) or 64 (fp4, two values to a byte,
// the first in the low half) code bytes and 4 scale bytes each; what lies behind dim is zero.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ancha_hip.h"
#include "common.hpp"

namespace ancha {
namespace mx {

constexpr int kBlock = 32, kGroup = 128;
constexpr int kFp8 = ANCHA_HIP_MX_FP8, kFp4 = ANCHA_HIP_MX_FP4;
constexpr int kF32 = ANCHA_HIP_F32, kF16 = ANCHA_HIP_F16, kBf16 = ANCHA_HIP_BF16;

__host__ __device__ constexpr long groups(long dim) { return (dim + kGroup - 1) / kGroup; }
__host__ __device__ constexpr long pitch(long dim, int format) {
  return groups(dim) * (format == kFp8 ? 128 : 64);
}

typedef int i32x8 __attribute__((ext_vector_type(8)));

template <int TYPE>
struct Stored {
  typedef float type;
};
template <>
struct Stored<kF16> {
  typedef _Float16 type;
};
template <>
struct Stored<kBf16> {
  typedef __bf16 type;
};

// N consecutive values at element `at`, of which the first `valid` exist (the others read as 0; with
// valid <= 0 nothing is read). Any alignment of whole elements: gfx950 reads wide words from any address.
// The values behind the last one are read in its place, so a row's end costs no branch per value.
template <int TYPE, int N>
__device__ __forceinline__ void load_stored(const void* base, long at, int valid,
                                            typename Stored<TYPE>::type* t) {
  typedef typename Stored<TYPE>::type T;
  const T* p = static_cast<const T*>(base) + at;
  if (valid >= N) {
    __builtin_memcpy(t, p, N * sizeof(T));
  } else if (valid > 0) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = p[i < valid ? i : valid - 1];
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = i < valid ? e[i] : (T)0.f;
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = (T)0.f;
  }
}

template <int TYPE, int N>
__device__ __forceinline__ void load_row(const void* base, long at, int valid, float* v) {
  typename Stored<TYPE>::type t[N];
  load_stored<TYPE, N>(base, at, valid, t);
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = (float)t[i];
}

// Non-temporal, like every large result here: past the caches, 16384 x 8192 values leave in 50 us instead
// of 97, codes in 55 instead of 63, and no size measured is slower.
template <int TYPE, int N>
__device__ __forceinline__ void store_row(void* base, long at, int valid, const float* v) {
  typedef typename Stored<TYPE>::type T;
  T* p = static_cast<T*>(base) + at;
  if (valid >= N) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = (T)v[i];
    if constexpr (N * sizeof(T) % 16 == 0) {
      typedef unsigned vec __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
      for (int i = 0; i < (int)(N * sizeof(T) / 16); i++) {
        vec w;
        __builtin_memcpy(&w, t + i * (16 / sizeof(T)), 16);
        __builtin_nontemporal_store(w, reinterpret_cast<vec*>(p) + i);
      }
    } else {
      __builtin_memcpy(p, t, sizeof(t));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < valid) p[i] = (T)v[i];
  }
}

// The exponent bits of the largest of |v[0]| .. |v[N - 1]|, 255 where one is infinite or a NaN: the
// instruction hands a NaN on (the library is compiled without NaN semantics, so no comparison would).
__device__ __forceinline__ float largest(float a, float b, float c) {
  float m;
  asm("v_maximum3_f32 %0, |%1|, |%2|, |%3|" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}
template <int N>
__device__ __forceinline__ unsigned top_exponent(const float* v) {
  float m = largest(v[0], v[1], v[2]);
#pragma unroll
  for (int i = 3; i < N; i += 2) m = largest(m, v[i], v[i + 1 < N ? i + 1 : i]);
  return __builtin_bit_cast(unsigned, m) >> 23 & 255u;
}

// Lane exchanges within 16 lanes (DPP, no LDS): the neighbour, the other pair of four lanes, the other
// four of eight and the other eight of sixteen (the last two reversed: for values equal within a quad).
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned x) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;

// Scale byte of a block whose largest magnitude has the exponent bits e.
__device__ __forceinline__ unsigned scale_byte(unsigned e, int format) {
  return e == 255u ? 255u : (unsigned)max((int)e - (format == kFp8 ? 8 : 2), 0);
}

// 2^(s - 127), by which the conversions divide (not for s = 255).
__device__ __forceinline__ float divisor(unsigned s) {
  return __builtin_bit_cast(float, s == 0u ? 0x00400000u : s << 23);
}

// 2^(s - 127), NaN for s = 255.
__device__ __forceinline__ float scale_value(unsigned s) {
  return __builtin_bit_cast(float, s == 255u ? 0x7fc00000u : s == 0u ? 0x00400000u : s << 23);
}

// Sets MODE.FP16_OVFL: conversions to e4m3 stop at 448 instead of turning into a NaN. Conversions to fp16 stop
// at 65504 then, and matrix instructions no longer give a NaN for the scale byte 255: only behind both.
__device__ __forceinline__ void saturate() { __builtin_amdgcn_s_setreg(1 | 23 << 6 | 0 << 11, 1); }

// e4m3 codes of four values, divided by f, with saturate() in effect.
__device__ __forceinline__ unsigned codes_fp8(const float* v, float f) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  s16x2 w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[0], v[1], f, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[2], v[3], f, true);
  return __builtin_bit_cast(unsigned, w);
}

// e2m1 codes of eight (four) values, divided by f (the conversion saturates by itself).
__device__ __forceinline__ unsigned codes_fp4(const float* v, float f) {
  unsigned r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], f, 3);
}
__device__ __forceinline__ unsigned codes_fp4x4(const float* v, float f) {
  const unsigned r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], f, 0);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], f, 1);
}

// Eight consecutive values of a row held by one lane, a block by four neighbouring lanes, all of which take
// part with saturate() in effect: rounds them, writes their codes to `codes` and, from a block's first lane,
// its scale byte to `scale`.
__device__ __forceinline__ void store_codes(const float* v, int format, bool store, uint8_t* codes,
                                            uint8_t* scale) {
  unsigned top = top_exponent<8>(v);
  top = max(top, dpp<kSwap1>(top));
  top = max(top, dpp<kSwap2>(top));
  const unsigned s = scale_byte(top, format);
  const float f = divisor(s);
  const bool none = s == 255u;
  if (!store) return;
  if (format == kFp8) {
    const u32x2 c = {none ? 0u : codes_fp8(v, f), none ? 0u : codes_fp8(v + 4, f)};
    __builtin_nontemporal_store(c, reinterpret_cast<u32x2*>(codes));
  } else {
    __builtin_nontemporal_store(none ? 0u : codes_fp4(v, f), reinterpret_cast<unsigned*>(codes));
  }
  if (threadIdx.x % 4 == 0) *scale = (uint8_t)s;
}

// ---- parameter blocks and launchers (arguments checked by the entry points)

struct RowParams {
  const void* x;         // [rows][dim], row stride ldx
  const void* residual;  // the same shape, row stride ldr, or null
  const float* scale;    // [dim] or null
  void* sum;             // [rows][dim] contiguous, with a residual (may be x or residual)
  uint8_t* codes;
  uint8_t* scales;
  long ldx, ldr;
  int rows, dim, type, format;
  double eps;
};
hipError_t launch_quantize(const RowParams& p, hipStream_t stream);
hipError_t launch_norm(const RowParams& p, hipStream_t stream);

// The form of the norm's kernel: threads a row and their pieces of eight values each, or 0 where rows are read
// twice.
constexpr int norm_code(int threads, int pieces) { return 8 * threads + pieces; }
int norm_form(long rows, long dim);

struct ValueParams {
  const uint8_t* codes;
  const uint8_t* scales;
  void* out;  // [rows][dim] contiguous
  int rows, dim, type, format;
};
hipError_t launch_values(const ValueParams& p, hipStream_t stream);

// A weight [k][m] in e2m1 along k, as the matrix cores read it: for each strip of 64 columns and each
// group of 128 k, four fragments of 1 KiB (16 columns: lane l has column l % 16, k 32 (l / 16) .. + 31
// in 16 bytes); then, behind all of them, a dword per lane with the scale bytes of its four fragments.
// m is filled up to whole 128 with zero columns, k to whole 128 with zeros.
constexpr long kStripCodes = 4096, kStripScales = 256;  // bytes per strip and group
__host__ __device__ constexpr long strips(long m) { return (m + 127) / 128 * 2; }
__host__ __device__ constexpr long weight_bytes(long k, long m) {
  return strips(m) * groups(k) * (kStripCodes + kStripScales);
}

struct WeightParams {
  const void* x;  // element (k, m) at k * ldk + m * ldm
  uint8_t* weight;
  long ldk, ldm;
  int k, m, type;
};
hipError_t launch_weight(const WeightParams& p, hipStream_t stream);

struct WeightValueParams {
  const uint8_t* weight;
  void* out;  // [k][m] contiguous
  int k, m, type;
};
hipError_t launch_weight_values(const WeightValueParams& p, hipStream_t stream);

struct LinearParams {
  const uint8_t* x;         // codes [n][pitch(k)]
  const uint8_t* x_scales;  // [n][4 groups(k)]
  const uint8_t* weight;
  const float* bias;     // [m] or null
  const float* rope;     // [4][tokens][64] or null
  const void* residual;  // [n][m] contiguous, of `type`, or null
  void* out;             // [n][m] contiguous, of `type`; with out_format the codes
  uint8_t* out_scales;   // with out_format
  int n, k, m, format;
  int tokens, width, gelu;
  int type, out_format;  // out_format 0: values of `type`
};
hipError_t launch_linear(const LinearParams& p, hipStream_t stream);

// The kernel that a product takes: few rows (16 or 32 a workgroup), tiles of 64 x 64 (the steps of k in one chain
// or four), 128 x 128 and 128 rows x 256 columns.
enum LinearForm { kFew16, kFew32, kTiles64, kTiles64Chains, kTiles128, kTiles256 };
LinearForm linear_form(long n, long k, long m);

}  // namespace mx
}  // namespace ancha
