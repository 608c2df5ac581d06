// Rows to microscaled codes and back (gfx950): quantisation, the row norm with the residual's addition
// in front of it, and the decoder. Formats and rounding: mx.hpp.
#include "mx.hpp"

namespace ancha {
namespace mx {
namespace {

constexpr int kThreads = 256;

template <int TYPE>
__global__ __launch_bounds__(kThreads) void quantize_kernel(RowParams p) {
  const unsigned per_row = 16u * (unsigned)groups(p.dim);
  const unsigned unit = blockIdx.x * (unsigned)kThreads + threadIdx.x;
  const unsigned row = unit / per_row;
  const int col = 8 * (int)(unit - row * per_row);
  const bool here = row < (unsigned)p.rows;
  float v[8];
  load_row<TYPE, 8>(p.x, here ? (long)row * p.ldx + col : 0, here ? p.dim - col : 0, v);
  store_codes(v, p.format, here, unit, p.codes, p.scales);
}

// Sum over L lanes (a power of two up to 64) in 64 bits.
template <int L>
__device__ __forceinline__ double sum_lanes(double s) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) s += __shfl_xor(s, o);
  return s;
}

// The double d with its last 32 bits folded into the one above them, as a float: truncated, with the
// last bit set if anything was lost (rounding to odd). Rounding the result to 4 or fewer bits then
// gives what rounding d itself does.
__device__ __forceinline__ float to_odd(double d) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, d);
  const unsigned hi = (unsigned)(bits >> 32) | ((unsigned)bits != 0u ? 1u : 0u);
  return (float)__builtin_bit_cast(double, (unsigned long long)hi << 32);
}

// 1 / max(sqrt(s), 1e-12) for a sum of squares s, following the division where s is not finite
// (0 for an infinity, NaN for a NaN; on the bits, as the library is compiled without NaN semantics).
__device__ __forceinline__ double inverse_length(double s) {
  unsigned hi = (unsigned)(__builtin_bit_cast(unsigned long long, s) >> 32);
  asm("" : "+v"(hi));
  if ((hi & 0x7ff00000u) == 0x7ff00000u) return (hi & 0xfffffu) ? s : 0.0;
  return 1.0 / fmax(sqrt(s), 1e-12);
}

template <int TYPE>
__device__ __forceinline__ float rounded(float x) {
  return (float)(typename Stored<TYPE>::type)x;
}

// One row by L threads, eight neighbouring values each, V times; a workgroup of 256 threads.
template <int TYPE, int L, int V>
__global__ __launch_bounds__(kThreads) void norm_kernel(RowParams p) {
  const int at = threadIdx.x % L;
  const unsigned row = blockIdx.x * (unsigned)(kThreads / L) + threadIdx.x / L;
  const bool here = row < (unsigned)p.rows;
  const int padded = kGroup * (int)groups(p.dim);
  float h[V][8];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int col = 8 * (at + L * i), valid = here ? p.dim - col : 0;
    load_row<TYPE, 8>(p.x, valid > 0 ? (long)row * p.ldx + col : 0, valid, h[i]);
    if (p.residual) {
      float r[8];
      load_row<TYPE, 8>(p.residual, valid > 0 ? (long)row * p.ldr + col : 0, valid, r);
#pragma unroll
      for (int j = 0; j < 8; j++) h[i][j] = rounded<TYPE>(h[i][j] + r[j]);
      store_row<TYPE, 8>(p.sum, valid > 0 ? (long)row * p.dim + col : 0, valid, h[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) ss = __builtin_fma((double)h[i][j], (double)h[i][j], ss);
  }
  ss = sum_lanes<(L < 64 ? L : 64)>(ss);
  if constexpr (L > 64) {
    __shared__ double part[kThreads / 64];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) ss += part[w];
  }
  const double inv = inverse_length(ss + (double)p.dim * p.eps);
  const long first = (long)row * (padded / 8);
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int col = 8 * (at + L * i);
    float s[8], y[8];
    if (p.scale) load_row<kF32, 8>(p.scale, col < p.dim ? col : 0, p.dim - col, s);
#pragma unroll
    for (int j = 0; j < 8; j++)
      y[j] = col + j < p.dim ? to_odd((double)h[i][j] * inv * (p.scale ? (double)s[j] : 1.0)) : 0.f;
    store_codes(y, p.format, here && col < padded, first + at + L * i, p.codes, p.scales);
  }
}

// Rows longer than the registers hold: read twice.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void norm_long_kernel(RowParams p) {
  const unsigned row = blockIdx.x;
  const int padded = kGroup * (int)groups(p.dim);
  double ss = 0.0;
  for (int col = 8 * threadIdx.x; col < p.dim; col += 8 * kThreads) {
    float h[8];
    load_row<TYPE, 8>(p.x, (long)row * p.ldx + col, p.dim - col, h);
    if (p.residual) {
      float r[8];
      load_row<TYPE, 8>(p.residual, (long)row * p.ldr + col, p.dim - col, r);
#pragma unroll
      for (int j = 0; j < 8; j++) h[j] = rounded<TYPE>(h[j] + r[j]);
      store_row<TYPE, 8>(p.sum, (long)row * p.dim + col, p.dim - col, h);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) ss = __builtin_fma((double)h[j], (double)h[j], ss);
  }
  __shared__ double part[kThreads / 64];
  ss = sum_lanes<64>(ss);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
  __syncthreads();
  ss = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; w++) ss += part[w];
  const double inv = inverse_length(ss + (double)p.dim * p.eps);
  const long first = (long)row * (padded / 8);
  // The sum is read back by the thread that wrote it.
  const void* from = p.residual ? p.sum : p.x;
  const long ld = p.residual ? p.dim : p.ldx;
  for (int col = 8 * threadIdx.x; col < padded; col += 8 * kThreads) {
    float h[8], s[8], y[8];
    load_row<TYPE, 8>(from, col < p.dim ? (long)row * ld + col : 0, p.dim - col, h);
    if (p.scale) load_row<kF32, 8>(p.scale, col < p.dim ? col : 0, p.dim - col, s);
#pragma unroll
    for (int j = 0; j < 8; j++)
      y[j] = col + j < p.dim ? to_odd((double)h[j] * inv * (p.scale ? (double)s[j] : 1.0)) : 0.f;
    store_codes(y, p.format, true, first + col / 8, p.codes, p.scales);
  }
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void values_kernel(ValueParams p) {
  const unsigned per_row = 16u * (unsigned)groups(p.dim);
  const unsigned unit = blockIdx.x * (unsigned)kThreads + threadIdx.x;
  const unsigned row = unit / per_row;
  const int col = 8 * (int)(unit - row * per_row);
  if (row >= (unsigned)p.rows || col >= p.dim) return;
  const float f = scale_value(p.scales[unit >> 2]);
  float v[8];
  if (p.format == kFp8) {
    const u32x2 c = *reinterpret_cast<const u32x2*>(p.codes + (long)unit * 8);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], false);
      const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], true);
      v[4 * i] = a[0], v[4 * i + 1] = a[1], v[4 * i + 2] = b[0], v[4 * i + 3] = b[1];
    }
  } else {
    const unsigned c = *reinterpret_cast<const unsigned*>(p.codes + (long)unit * 4);
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2);
    const auto e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
    v[4] = d[0], v[5] = d[1], v[6] = e[0], v[7] = e[1];
  }
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] *= f;
  store_row<TYPE, 8>(p.out, (long)row * p.dim + col, p.dim - col, v);
}

template <int TYPE, int L, int V>
void start_norm(const RowParams& p, hipStream_t stream) {
  constexpr int kRows = kThreads / L;
  hipLaunchKernelGGL((norm_kernel<TYPE, L, V>), dim3((p.rows + (long)kRows - 1) / kRows),
                     dim3(kThreads), 0, stream, p);
}

template <int TYPE>
void norm_of_type(const RowParams& p, hipStream_t stream) {
  const long g = groups(p.dim);
  if (g <= 1) return start_norm<TYPE, 16, 1>(p, stream);
  if (g <= 2) return start_norm<TYPE, 16, 2>(p, stream);
  if (g <= 3) return start_norm<TYPE, 16, 3>(p, stream);
  if (g <= 4) return start_norm<TYPE, 16, 4>(p, stream);
  if (g <= 8) return start_norm<TYPE, 64, 2>(p, stream);
  if (g <= 16) return start_norm<TYPE, 64, 4>(p, stream);
  if (g <= 32) return start_norm<TYPE, 256, 2>(p, stream);
  if (g <= 64) return start_norm<TYPE, 256, 4>(p, stream);
  hipLaunchKernelGGL(norm_long_kernel<TYPE>, dim3(p.rows), dim3(kThreads), 0, stream, p);
}

dim3 unit_grid(long rows, long dim) {
  return dim3((unsigned)((rows * 16 * groups(dim) + kThreads - 1) / kThreads));
}

}  // namespace

hipError_t launch_quantize(const RowParams& p, hipStream_t stream) {
  const dim3 grid = unit_grid(p.rows, p.dim);
  if (p.type == kF32)
    hipLaunchKernelGGL(quantize_kernel<kF32>, grid, dim3(kThreads), 0, stream, p);
  else if (p.type == kF16)
    hipLaunchKernelGGL(quantize_kernel<kF16>, grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(quantize_kernel<kBf16>, grid, dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_norm(const RowParams& p, hipStream_t stream) {
  if (p.type == kF32)
    norm_of_type<kF32>(p, stream);
  else if (p.type == kF16)
    norm_of_type<kF16>(p, stream);
  else
    norm_of_type<kBf16>(p, stream);
  return hipGetLastError();
}

hipError_t launch_values(const ValueParams& p, hipStream_t stream) {
  const dim3 grid = unit_grid(p.rows, p.dim);
  if (p.type == kF32)
    hipLaunchKernelGGL(values_kernel<kF32>, grid, dim3(kThreads), 0, stream, p);
  else if (p.type == kF16)
    hipLaunchKernelGGL(values_kernel<kF16>, grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(values_kernel<kBf16>, grid, dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mx
}  // namespace ancha
