// Weights in microscaled e2m1, laid out for the matrix cores (layout: mx.hpp), and back (gfx950).
#include "mx.hpp"

namespace ancha {
namespace mx {
namespace {

// Column and k block of value (c, k) in a strip and group; 16 bytes of codes per column and block.
__device__ __forceinline__ long code_place(long piece, int c, int block) {
  return piece * kStripCodes + (c >> 4) * 1024 + ((c & 15) + 16 * block) * 16;
}
__device__ __forceinline__ long scale_place(long pieces, long piece, int c, int block) {
  return pieces * kStripCodes + piece * kStripScales + ((c & 15) + 16 * block) * 4 + (c >> 4);
}

// A strip (64 columns) and group (128 k) per workgroup, any layout: lane l of wave b has column l, k block
// b. Neighbouring lanes read neighbouring columns, so [in, out] weights are read in whole lines.
// Both kernels run once per weight and are bound by memory: 8192 x 8192 [in, out] fp32 48 us (6.4 TB/s), bf16 33.
template <int TYPE>
__global__ __launch_bounds__(256) void weight_columns_kernel(WeightParams p) {
  typedef typename Stored<TYPE>::type T;
  const int c = threadIdx.x & 63, block = threadIdx.x >> 6;
  const unsigned steps = (unsigned)groups(p.k);
  const unsigned strip = blockIdx.x / steps, step = blockIdx.x - strip * steps;
  const int col = (int)strip * 64 + c, k0 = (int)step * kGroup + 32 * block;
  const T* x = static_cast<const T*>(p.x) + (long)min(col, p.m - 1) * p.ldm;
  T t[32];
#pragma unroll
  for (int i = 0; i < 32; i++) t[i] = x[(long)min(k0 + i, p.k - 1) * p.ldk];
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; i++) v[i] = col < p.m && k0 + i < p.k ? (float)t[i] : 0.f;
  const unsigned s = scale_byte(top_exponent<32>(v), kFp4);
  const float f = divisor(s);
  u32x4 q;
#pragma unroll
  for (int i = 0; i < 4; i++) q[i] = s == 255u ? 0u : codes_fp4(v + 8 * i, f);
  *reinterpret_cast<u32x4*>(p.weight + code_place(blockIdx.x, c, block)) = q;
  p.weight[scale_place(gridDim.x, blockIdx.x, c, block)] = (uint8_t)s;
}

// The same for a weight whose columns are contiguous along k ([out, in] storage): sixteen lanes have the
// 128 k of a column, eight neighbouring values each, a wave four columns at a time: 8192 x 8192 fp32 51 us (5.9
// TB/s), 811 by a lane a column.
template <int TYPE>
__global__ __launch_bounds__(256) void weight_rows_kernel(WeightParams p) {
  typedef typename Stored<TYPE>::type T;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15;
  const unsigned steps = (unsigned)groups(p.k);
  const unsigned strip = blockIdx.x / steps, step = blockIdx.x - strip * steps;
  const int k = (int)step * kGroup + 8 * j;
  T t[4][8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int col = (int)strip * 64 + 16 * wave + 4 * i + (lane >> 4);
    const int valid = col < p.m ? p.k - k : 0;
    load_stored<TYPE, 8>(p.x, valid > 0 ? (long)col * p.ldm + k : 0, valid, t[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int c = 16 * wave + 4 * i + (lane >> 4);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)t[i][e];
    unsigned top = top_exponent<8>(v);
    top = max(top, dpp<kSwap1>(top));
    top = max(top, dpp<kSwap2>(top));
    const unsigned s = scale_byte(top, kFp4);
    *reinterpret_cast<unsigned*>(p.weight + code_place(blockIdx.x, c, j >> 2) + 4 * (j & 3)) =
        s == 255u ? 0u : codes_fp4(v, divisor(s));
    if ((j & 3) == 0) p.weight[scale_place(gridDim.x, blockIdx.x, c, j >> 2)] = (uint8_t)s;
  }
}

// A strip and group per workgroup: lane l of wave `tile` decodes its 32 values.
template <int TYPE>
__global__ __launch_bounds__(256) void weight_values_kernel(WeightValueParams p) {
  typedef typename Stored<TYPE>::type T;
  const int lane = threadIdx.x & 63, tile = threadIdx.x >> 6;
  const unsigned steps = (unsigned)groups(p.k);
  const unsigned strip = blockIdx.x / steps, step = blockIdx.x - strip * steps;
  const int col = (int)strip * 64 + 16 * tile + (lane & 15);
  const int k0 = (int)step * kGroup + 32 * (lane >> 4);
  const long piece = (long)blockIdx.x;
  const u32x4 c = *reinterpret_cast<const u32x4*>(p.weight + piece * kStripCodes + tile * 1024 + lane * 16);
  const float f =
      scale_value(p.weight[(long)gridDim.x * kStripCodes + piece * kStripScales + lane * 4 + tile]);
  if (col >= p.m) return;
  T* out = static_cast<T*>(p.out) + (long)k0 * p.m + col;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], 1.f, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], 1.f, 1);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], 1.f, 2);
    const auto e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], 1.f, 3);
    const float v[8] = {a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (k0 + 8 * i + j < p.k) out[(long)(8 * i + j) * p.m] = (T)(v[j] * f);
  }
}

}  // namespace

template <int TYPE>
static void start_weight(const WeightParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)(strips(p.m) * groups(p.k)));
  if (p.ldk == 1)
    hipLaunchKernelGGL(weight_rows_kernel<TYPE>, grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL(weight_columns_kernel<TYPE>, grid, dim3(256), 0, stream, p);
}

hipError_t launch_weight(const WeightParams& p, hipStream_t stream) {
  if (p.type == kF32)
    start_weight<kF32>(p, stream);
  else if (p.type == kF16)
    start_weight<kF16>(p, stream);
  else
    start_weight<kBf16>(p, stream);
  return hipGetLastError();
}

hipError_t launch_weight_values(const WeightValueParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)(strips(p.m) * groups(p.k)));
  if (p.type == kF32)
    hipLaunchKernelGGL(weight_values_kernel<kF32>, grid, dim3(256), 0, stream, p);
  else if (p.type == kF16)
    hipLaunchKernelGGL(weight_values_kernel<kF16>, grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL(weight_values_kernel<kBf16>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mx
}  // namespace ancha
