// Rows to microscaled codes and back (gfx950): quantisation, the row norm with the residual's addition
// in front of it, and the decoder. Formats and rounding: mx.hpp.
#include "mx.hpp"

namespace ancha {
namespace mx {
namespace {

constexpr int kThreads = 256;

// Division by a row's groups d: n / d = n * factor >> shift for every n < 2^28, with factor = 2^shift / d + 1 and
// 2^shift = 2^31 times the largest power of two up to d (the product is off by n d / 2^shift < 1/4 of a whole).
struct Divide {
  unsigned factor;
  int shift;
};
Divide divide_by(long d) {
  int shift = 31;
  while (2l << (shift - 31) <= d) shift++;
  return {(unsigned)((1ul << shift) / (unsigned long)d + 1), shift};
}

// The unit of N neighbouring values that a thread has: 128 / N threads a group, groups in the order in which
// they are stored, so a workgroup reads and writes whole rows beside each other whatever their length.
struct Unit {
  unsigned row;
  int col;
  long at;  // among the units of the codes
};
template <int N>
__device__ __forceinline__ Unit my_unit(int dim, Divide d) {
  constexpr unsigned kLanes = kGroup / N;
  Unit u;
  const unsigned lane = threadIdx.x % kLanes, group = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  u.row = (unsigned)((unsigned long)group * d.factor >> d.shift);
  u.col = N * (int)(kLanes * (group - u.row * (unsigned)groups(dim)) + lane);
  u.at = kLanes * (long)group + lane;
  return u;
}
template <int N>
unsigned unit_blocks(long rows, long dim) {
  constexpr long kGroups = kThreads * N / kGroup;
  return (unsigned)((rows * groups(dim) + kGroups - 1) / kGroups);
}

// One pass, a unit a thread. Bound by memory: 16 384 x 8192 bf16 to e2m1 55 us (339 MB, 6.2 TB/s).
template <int TYPE, int FORMAT>
__global__ __launch_bounds__(kThreads) void quantize_kernel(RowParams p, Divide d) {
  const Unit u = my_unit<8>(p.dim, d);
  const bool here = u.row < (unsigned)p.rows;
  const int valid = here ? p.dim - u.col : 0;
  float v[8];
  load_row<TYPE, 8>(p.x, valid > 0 ? (long)u.row * p.ldx + u.col : 0, valid, v);
  saturate();
  store_codes(v, FORMAT, here, p.codes + u.at * (FORMAT == kFp8 ? 8 : 4), p.scales + (u.at >> 2));
}

// Sum over L = 16, 32 or 64 lanes in 64 bits, by lane exchanges without LDS.
template <int CTRL>
__device__ __forceinline__ double add_lane(double s) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, s);
  const unsigned long long hi = dpp<CTRL>((unsigned)(b >> 32)), lo = dpp<CTRL>((unsigned)b);
  return s + __builtin_bit_cast(double, hi << 32 | lo);
}
template <int L>
__device__ __forceinline__ double sum_lanes(double s) {
  s = add_lane<kSwap1>(s);
  s = add_lane<kSwap2>(s);
  s = add_lane<kMirror8>(s);
  s = add_lane<kMirror16>(s);
#pragma unroll
  for (int o = 16; o < L; o <<= 1) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, s);
    const unsigned h = (unsigned)(b >> 32), l = (unsigned)b;
    const auto hi = o == 16 ? __builtin_amdgcn_permlane16_swap(h, h, false, false)
                            : __builtin_amdgcn_permlane32_swap(h, h, false, false);
    const auto lo = o == 16 ? __builtin_amdgcn_permlane16_swap(l, l, false, false)
                            : __builtin_amdgcn_permlane32_swap(l, l, false, false);
    s = __builtin_bit_cast(double, (unsigned long long)(unsigned)hi[0] << 32 | (unsigned)lo[0]) +
        __builtin_bit_cast(double, (unsigned long long)(unsigned)hi[1] << 32 | (unsigned)lo[1]);
  }
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

// One row by L threads, eight neighbouring values each, V times; a workgroup of 256 threads or L. A piece of 8 L
// columns that all exist is read and written without a mask (threads behind the last row read that one).
// The row stays in registers, so memory is passed once. With the addition it is what bounds: 96 120 x 384 fp32
// 80 us (481 MB, 6.0 TB/s). Without it, on 16-bit rows, the vector ALU does (91 % busy), with about 20
// instructions a value, seven of them in 64 bits: 30 000 x 1024 bf16 22 us (4.3 TB/s).
template <int TYPE, int L, int V>
__global__ __launch_bounds__(L > kThreads ? L : kThreads) void norm_kernel(RowParams p) {
  constexpr int kAll = L > kThreads ? L : kThreads;
  const int at = threadIdx.x % L;
  const unsigned mine = blockIdx.x * (unsigned)(kAll / L) + threadIdx.x / L;
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
    __shared__ double part[kAll / 64];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) part[wave] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) ss += part[wave / kWaves * kWaves + w];
  }
  double inv = inverse_length(ss + (double)p.dim * p.eps);
  saturate_before(inv);
  const long first = row * (padded / 8) + at;
  const int bytes = p.format == kFp8 ? 8 : 4;  // of a unit
  uint8_t* const codes = p.codes + first * bytes;
  uint8_t* const scales = p.scales + (first >> 2);
#pragma unroll
  for (int i = 0; i < V; i++) {
    if (8 * L * i >= padded) break;
    const int col = 8 * (at + L * i);
    float y[8];
    normed(p, h[i], inv, col, 8 * L * (i + 1) <= p.dim, y);
    store_codes(y, p.format, here && col < padded, codes + L * i * bytes, scales + L * i / 4);
  }
}

// Rows longer than the registers hold (more than 16 384 values): read twice, the second time mostly from the
// caches. 2000 x 20 000 bf16 with the addition 76 us (3.7 TB/s of what has to be moved; 92 with the sum left in
// the caches for it).
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
  const int bytes = p.format == kFp8 ? 8 : 4;  // of a unit
  // The sum is read back by the thread that wrote it.
  const void* from = p.residual ? p.sum : p.x;
  const long ld = p.residual ? p.dim : p.ldx;
  for (int col = 8 * threadIdx.x; col < padded; col += 8 * kThreads) {
    float h[8], y[8];
    load_row<TYPE, 8>(from, col < p.dim ? (long)row * ld + col : 0, p.dim - col, h);
    normed(p, h, inv, col, col + 8 <= p.dim, y);
    store_codes(y, p.format, true, p.codes + (first + col / 8) * bytes, p.scales + (first + col / 8) / 4);
  }
}

// A unit of 16 bytes of TYPE a thread, so that a wave's store instruction writes one piece of memory: code times
// 2^(s - 127), exact but for the rounding to TYPE. Bound by memory: 16 384 x 8192 e2m1 to bf16 48 us (7.1 TB/s),
// 96 120 x 384 e4m3 to fp32 27 (6.9; 53 with eight values a thread).
template <int TYPE>
constexpr int kDecoded = TYPE == kF32 ? 4 : 8;
template <int TYPE, int FORMAT>
__global__ __launch_bounds__(kThreads) void values_kernel(ValueParams p, Divide d) {
  constexpr int N = kDecoded<TYPE>;
  const Unit u = my_unit<N>(p.dim, d);
  if (u.row >= (unsigned)p.rows || u.col >= p.dim) return;
  const float f = scale_value(p.scales[u.at / (kBlock / N)]);
  float v[N];
  if constexpr (FORMAT == kFp8) {
    unsigned c[N / 4];
    __builtin_memcpy(c, p.codes + u.at * N, N);
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], false);
      const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], true);
      v[4 * i] = a[0], v[4 * i + 1] = a[1], v[4 * i + 2] = b[0], v[4 * i + 3] = b[1];
    }
  } else {
    unsigned c = 0;
    __builtin_memcpy(&c, p.codes + u.at * (N / 2), N / 2);
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
    if constexpr (N == 8) {
      const auto e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2);
      const auto g = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3);
      v[4] = e[0], v[5] = e[1], v[6] = g[0], v[7] = g[1];
    }
  }
#pragma unroll
  for (int i = 0; i < N; i++) v[i] *= f;
  store_row<TYPE, N>(p.out, (long)u.row * p.dim + u.col, p.dim - u.col, v);
}

template <int TYPE, int L, int V>
void start_norm(const RowParams& p, hipStream_t stream) {
  constexpr int kAll = L > kThreads ? L : kThreads, kRows = kAll / L;
  hipLaunchKernelGGL((norm_kernel<TYPE, L, V>), dim3((p.rows + (long)kRows - 1) / kRows),
                     dim3(kAll), 0, stream, p);
}

template <int TYPE>
void norm_of_type(const RowParams& p, hipStream_t stream) {
  switch (norm_form(p.rows, p.dim)) {
    case norm_code(16, 1): return start_norm<TYPE, 16, 1>(p, stream);
    case norm_code(16, 2): return start_norm<TYPE, 16, 2>(p, stream);
    case norm_code(16, 3): return start_norm<TYPE, 16, 3>(p, stream);
    case norm_code(16, 4): return start_norm<TYPE, 16, 4>(p, stream);
    case norm_code(32, 3): return start_norm<TYPE, 32, 3>(p, stream);
    case norm_code(64, 1): return start_norm<TYPE, 64, 1>(p, stream);
    case norm_code(64, 2): return start_norm<TYPE, 64, 2>(p, stream);
    case norm_code(128, 2): return start_norm<TYPE, 128, 2>(p, stream);
    case norm_code(256, 1): return start_norm<TYPE, 256, 1>(p, stream);
    case norm_code(256, 2): return start_norm<TYPE, 256, 2>(p, stream);
    case norm_code(256, 4): return start_norm<TYPE, 256, 4>(p, stream);
    case norm_code(512, 4): return start_norm<TYPE, 512, 4>(p, stream);
    default: hipLaunchKernelGGL(norm_long_kernel<TYPE>, dim3(p.rows), dim3(kThreads), 0, stream, p);
  }
}

template <int TYPE, int FORMAT>
void quantize_to(const RowParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((quantize_kernel<TYPE, FORMAT>), dim3(unit_blocks<8>(p.rows, p.dim)), dim3(kThreads), 0,
                     stream, p, divide_by(groups(p.dim)));
}

template <int TYPE, int FORMAT>
void values_of(const ValueParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((values_kernel<TYPE, FORMAT>), dim3(unit_blocks<kDecoded<TYPE>>(p.rows, p.dim)),
                     dim3(kThreads), 0, stream, p, divide_by(groups(p.dim)));
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

// Rows in registers, L threads a row and V pieces of 8 L values. Measured with each form forced (us, with
// the addition / without; the forms taken are up to 15 % faster since, by lighter codes):
//   96 120 x 384 fp32     16 threads  80 / 37, 64  79 / 47, 32  107 / 54
//   30 000 x 700 bf16     32 threads  36 / 25, 64  38 / 28, 128  51 / 37
//   30 000 x 1024 bf16    64 threads  37 / 25, 32  38 / 26, 128  43 / 31
//   20 000 x 1800 fp32   128 threads  85 / 37, 64  87 / 40, 256  83 / 40, 32  106 / 53
//   30 000 x 4096 bf16   256 threads 156 / 92, 128 172 / 91, 64  208 / 112
// and, with few rows, the more threads a row the shorter the way through it: 200 x 1500 fp16 256 threads
// 5.0 / 4.4, 64 7.1 / 5.8, 32 10.3 / 8.1; 300 x 384 fp16 64 threads 4.4 / 4.7, 16 6.1 / 5.2.
// Past 8192 values 512 threads, with the addition: 2000 x 12 000 bf16 36 (read twice 47), 2000 x 16 000 fp32 74
// (118). Four fp32 values side by side a thread in place of eight were slower: 96 120 x 384 84 / 38 (80 / 31).
int norm_form(long rows, long dim) {
  const long g = groups(dim);
  const bool few = rows < 1024;
  if (g > 128) return 0;
  if (g > 64) return norm_code(512, 4);
  if (g > 32) return norm_code(256, 4);
  if (g > 16) return norm_code(256, 2);
  if (few) return g > 4 ? norm_code(256, 1) : norm_code(64, 1);
  if (g > 8) return norm_code(128, 2);
  if (g > 6) return norm_code(64, 2);
  if (g > 4) return norm_code(32, 3);
  return norm_code(16, static_cast<int>(g));
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
