// Rows to microscaled codes and back (gfx950): quantisation, the row norm with the residual's addition
// in front of it, and the decoder. Formats and rounding: mx.hpp.
#include "mx.hpp"

namespace ancha {
namespace mx {
namespace {

constexpr int kThreads = 256;

// The unit of eight neighbouring values that a thread has: L threads side by side in a row, 256 / L rows a
// workgroup, column pieces of 8 L along the grid's second axis.
struct Unit {
  unsigned row;
  int col;
  long at;  // among the units of the codes
};
template <int L>
__device__ __forceinline__ Unit my_unit(int dim) {
  Unit u;
  u.row = blockIdx.x * (unsigned)(kThreads / L) + threadIdx.x / L;
  const int c = (int)blockIdx.y * L + (int)threadIdx.x % L;
  u.col = 8 * c;
  u.at = (long)u.row * (16 * groups(dim)) + c;
  return u;
}

template <int TYPE, int FORMAT, int L>
__global__ __launch_bounds__(kThreads) void quantize_kernel(RowParams p) {
  const Unit u = my_unit<L>(p.dim);
  const bool here = u.row < (unsigned)p.rows && u.col < kGroup * (int)groups(p.dim);
  const int valid = here ? p.dim - u.col : 0;
  float v[8];
  load_row<TYPE, 8>(p.x, valid > 0 ? (long)u.row * p.ldx + u.col : 0, valid, v);
  saturate();
  store_codes(v, FORMAT, here, u.at, p.codes, p.scales);
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
  unsigned lost;  // one instruction where the compiler takes two
  asm("v_min_u32 %0, 1, %1" : "=v"(lost) : "v"((unsigned)bits));
  const unsigned hi = (unsigned)(bits >> 32) | lost;
  return (float)__builtin_bit_cast(double, (unsigned long long)hi << 32);
}

// 1 / max(sqrt(s), 1e-12) for a sum of squares s, following the division where s is not finite
// (0 for an infinity, NaN for a NaN; on the bits, as the library is compiled without NaN semantics).
// The hardware's estimate (about 26 bits) and two Newton steps.
__device__ __forceinline__ double inverse_length(double s) {
  unsigned hi = (unsigned)(__builtin_bit_cast(unsigned long long, s) >> 32);
  asm("" : "+v"(hi));
  if ((hi & 0x7ff00000u) == 0x7ff00000u) return (hi & 0xfffffu) ? s : 0.0;
  if (s <= 1e-24) return 1e12;
  double y = __builtin_amdgcn_rsq(s);
#pragma unroll
  for (int i = 0; i < 2; i++) y = __builtin_fma(0.5 * y, __builtin_fma(-s * y, y, 1.0), y);
  return y;
}

// saturate() between the sums' rounding to fp16, on which inv depends, and the codes, which depend on inv.
__device__ __forceinline__ void saturate_before(double& inv) {
  asm volatile("" : "+v"(inv));
  saturate();
  asm volatile("" : "+v"(inv));
}

template <int TYPE>
__device__ __forceinline__ float rounded(float x) {
  return (float)(typename Stored<TYPE>::type)x;
}

// Eight values h of a row from column col on through the norm, rounded to odd; whole: all exist.
__device__ __forceinline__ void normed(const RowParams& p, const float* h, double inv, int col, bool whole,
                                       float* y) {
  if (p.scale) {
    float s[8];
    load_row<kF32, 8>(p.scale, whole || col < p.dim ? col : 0, whole ? 8 : p.dim - col, s);
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = to_odd((double)h[j] * inv * (double)s[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = to_odd((double)h[j] * inv);
  }
  // Behind the last value: zeros, also where inv is not finite.
  if (!whole)
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = col + j < p.dim ? y[j] : 0.f;
}

// One row by L threads, eight neighbouring values each, V times; a workgroup of 256 threads. A piece of 8 L
// columns that all exist is read and written without a mask (threads behind the last row read that one).
template <int TYPE, int L, int V>
__global__ __launch_bounds__(kThreads) void norm_kernel(RowParams p) {
  const int at = threadIdx.x % L;
  const unsigned mine = blockIdx.x * (unsigned)(kThreads / L) + threadIdx.x / L;
  const bool here = mine < (unsigned)p.rows;
  const long row = here ? mine : p.rows - 1;
  const int padded = kGroup * (int)groups(p.dim);
  typedef typename Stored<TYPE>::type T;
  T x[V][8], r[V][8];  // all of the row's loads in flight before the first use
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int col = 8 * (at + L * i);
    if (8 * L * (i + 1) <= p.dim) {
      load_stored<TYPE, 8>(p.x, row * p.ldx + col, 8, x[i]);
      if (p.residual) load_stored<TYPE, 8>(p.residual, row * p.ldr + col, 8, r[i]);
    } else {
      const int valid = p.dim - col;
      load_stored<TYPE, 8>(p.x, row * p.ldx + (valid > 0 ? col : 0), valid, x[i]);
      if (p.residual) load_stored<TYPE, 8>(p.residual, row * p.ldr + (valid > 0 ? col : 0), valid, r[i]);
    }
  }
  float h[V][8];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int col = 8 * (at + L * i);
#pragma unroll
    for (int j = 0; j < 8; j++) h[i][j] = (float)x[i][j];
    if (p.residual) {
#pragma unroll
      for (int j = 0; j < 8; j++) h[i][j] = rounded<TYPE>(h[i][j] + (float)r[i][j]);
      const int valid = here ? p.dim - col : 0;
      if (8 * L * (i + 1) <= p.dim) {
        if (here) store_row<TYPE, 8>(p.sum, row * p.dim + col, 8, h[i]);
      } else {
        store_row<TYPE, 8>(p.sum, row * p.dim + (valid > 0 ? col : 0), valid, h[i]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) ss = __builtin_fma((double)h[i][j], (double)h[i][j], ss);
  }
  ss = sum_lanes<(L < 64 ? L : 64)>(ss);
  if constexpr (L > 64) {
    constexpr int kWaves = L / 64;  // of a row
    __shared__ double part[kThreads / 64];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) part[wave] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) ss += part[wave / kWaves * kWaves + w];
  }
  double inv = inverse_length(ss + (double)p.dim * p.eps);
  saturate_before(inv);
  const long first = row * (padded / 8);
#pragma unroll
  for (int i = 0; i < V; i++) {
    if (8 * L * i >= padded) break;
    const int col = 8 * (at + L * i);
    float y[8];
    normed(p, h[i], inv, col, 8 * L * (i + 1) <= p.dim, y);
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
  double inv = inverse_length(ss + (double)p.dim * p.eps);
  saturate_before(inv);
  const long first = (long)row * (padded / 8);
  // The sum is read back by the thread that wrote it.
  const void* from = p.residual ? p.sum : p.x;
  const long ld = p.residual ? p.dim : p.ldx;
  for (int col = 8 * threadIdx.x; col < padded; col += 8 * kThreads) {
    float h[8], y[8];
    load_row<TYPE, 8>(from, col < p.dim ? (long)row * ld + col : 0, p.dim - col, h);
    normed(p, h, inv, col, col + 8 <= p.dim, y);
    store_codes(y, p.format, true, first + col / 8, p.codes, p.scales);
  }
}

template <int TYPE, int FORMAT, int L>
__global__ __launch_bounds__(kThreads) void values_kernel(ValueParams p) {
  const Unit u = my_unit<L>(p.dim);
  if (u.row >= (unsigned)p.rows || u.col >= p.dim) return;
  const float f = scale_value(p.scales[u.at >> 2]);
  float v[8];
  if constexpr (FORMAT == kFp8) {
    const u32x2 c = *reinterpret_cast<const u32x2*>(p.codes + u.at * 8);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], false);
      const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], true);
      v[4 * i] = a[0], v[4 * i + 1] = a[1], v[4 * i + 2] = b[0], v[4 * i + 3] = b[1];
    }
  } else {
    const unsigned c = *reinterpret_cast<const unsigned*>(p.codes + u.at * 4);
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2);
    const auto e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
    v[4] = d[0], v[5] = d[1], v[6] = e[0], v[7] = e[1];
  }
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] *= f;
  store_row<TYPE, 8>(p.out, (long)u.row * p.dim + u.col, p.dim - u.col, v);
}

template <int TYPE, int L, int V>
void start_norm(const RowParams& p, hipStream_t stream) {
  constexpr int kRows = kThreads / L;
  hipLaunchKernelGGL((norm_kernel<TYPE, L, V>), dim3((p.rows + (long)kRows - 1) / kRows),
                     dim3(kThreads), 0, stream, p);
}

// Rows in registers, L threads a row and V pieces of 8 L values. Measured with each form forced (us, with
// the addition / without):
//   96 120 x 384 fp32     16 threads  80 / 37, 64  79 / 47, 32  107 / 54
//   30 000 x 700 bf16     32 threads  36 / 25, 64  38 / 28, 128  51 / 37
//   30 000 x 1024 bf16    64 threads  37 / 25, 32  38 / 26, 128  43 / 31
//   20 000 x 1800 fp32   128 threads  85 / 37, 64  87 / 40, 256  83 / 40, 32  106 / 53
//   30 000 x 4096 bf16   256 threads 156 / 92, 128 172 / 91, 64  208 / 112
// and, with few rows, the more threads a row the shorter the way through it: 200 x 1500 fp16 256 threads
// 5.0 / 4.4, 64 7.1 / 5.8, 32 10.3 / 8.1; 300 x 384 fp16 64 threads 4.4 / 4.7, 16 6.1 / 5.2.
template <int TYPE>
void norm_of_type(const RowParams& p, hipStream_t stream) {
  const long g = groups(p.dim);
  const bool few = p.rows < 1024;
  if (g > 64)
    hipLaunchKernelGGL(norm_long_kernel<TYPE>, dim3(p.rows), dim3(kThreads), 0, stream, p);
  else if (g > 32)
    start_norm<TYPE, 256, 4>(p, stream);
  else if (g > 16)
    start_norm<TYPE, 256, 2>(p, stream);
  else if (g > 4 && few)
    start_norm<TYPE, 256, 1>(p, stream);
  else if (g > 8)
    start_norm<TYPE, 128, 2>(p, stream);
  else if (g > 6)
    start_norm<TYPE, 64, 2>(p, stream);
  else if (g > 4)
    start_norm<TYPE, 32, 3>(p, stream);
  else if (few)
    start_norm<TYPE, 64, 1>(p, stream);
  else if (g > 2)
    g > 3 ? start_norm<TYPE, 16, 4>(p, stream) : start_norm<TYPE, 16, 3>(p, stream);
  else
    g > 1 ? start_norm<TYPE, 16, 2>(p, stream) : start_norm<TYPE, 16, 1>(p, stream);
}

template <int L>
dim3 unit_grid(long rows, long dim) {
  constexpr long kRows = kThreads / L;
  return dim3((unsigned)((rows + kRows - 1) / kRows), (unsigned)((16 * groups(dim) + L - 1) / L));
}

// Rows of up to 512 values by 16 threads a piece, up to 2048 by 64: full lines, and few idle threads.
template <int TYPE, int FORMAT>
void quantize_to(const RowParams& p, hipStream_t stream) {
  if (p.dim <= 512)
    hipLaunchKernelGGL((quantize_kernel<TYPE, FORMAT, 16>), unit_grid<16>(p.rows, p.dim), dim3(kThreads), 0,
                       stream, p);
  else if (p.dim <= 2048)
    hipLaunchKernelGGL((quantize_kernel<TYPE, FORMAT, 64>), unit_grid<64>(p.rows, p.dim), dim3(kThreads), 0,
                       stream, p);
  else
    hipLaunchKernelGGL((quantize_kernel<TYPE, FORMAT, 256>), unit_grid<256>(p.rows, p.dim), dim3(kThreads),
                       0, stream, p);
}

template <int TYPE, int FORMAT>
void values_of(const ValueParams& p, hipStream_t stream) {
  if (p.dim <= 512)
    hipLaunchKernelGGL((values_kernel<TYPE, FORMAT, 16>), unit_grid<16>(p.rows, p.dim), dim3(kThreads), 0,
                       stream, p);
  else if (p.dim <= 2048)
    hipLaunchKernelGGL((values_kernel<TYPE, FORMAT, 64>), unit_grid<64>(p.rows, p.dim), dim3(kThreads), 0,
                       stream, p);
  else
    hipLaunchKernelGGL((values_kernel<TYPE, FORMAT, 256>), unit_grid<256>(p.rows, p.dim), dim3(kThreads), 0,
                       stream, p);
}

}  // namespace

template <int TYPE>
static void start_quantize(const RowParams& p, hipStream_t stream) {
  if (p.format == kFp8)
    quantize_to<TYPE, kFp8>(p, stream);
  else
    quantize_to<TYPE, kFp4>(p, stream);
}

hipError_t launch_quantize(const RowParams& p, hipStream_t stream) {
  if (p.type == kF32)
    start_quantize<kF32>(p, stream);
  else if (p.type == kF16)
    start_quantize<kF16>(p, stream);
  else
    start_quantize<kBf16>(p, stream);
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

template <int TYPE>
static void start_values(const ValueParams& p, hipStream_t stream) {
  if (p.format == kFp8)
    values_of<TYPE, kFp8>(p, stream);
  else
    values_of<TYPE, kFp4>(p, stream);
}

hipError_t launch_values(const ValueParams& p, hipStream_t stream) {
  if (p.type == kF32)
    start_values<kF32>(p, stream);
  else if (p.type == kF16)
    start_values<kF16>(p, stream);
  else
    start_values<kBf16>(p, stream);
  return hipGetLastError();
}

}  // namespace mx
}  // namespace ancha
