// Weights in microscaled e2m1, laid out for the matrix cores (layout: mx.hpp), and back (gfx950).
#include "mx.hpp"

namespace ancha {
namespace mx {
namespace {

// One fragment (16 columns x 128 k) per wave: lane l quantises column l % 16, k 32 (l / 16) .. + 31.
// The four waves of a workgroup have the four fragments of a strip and group.
template <int TYPE>
__global__ __launch_bounds__(256) void weight_kernel(WeightParams p) {
  typedef typename Stored<TYPE>::type T;
  const int lane = threadIdx.x & 63, tile = threadIdx.x >> 6;
  const unsigned steps = (unsigned)groups(p.k);
  const unsigned strip = blockIdx.x / steps, step = blockIdx.x - strip * steps;
  const int col = (int)strip * 64 + 16 * tile + (lane & 15);
  const int k0 = (int)step * kGroup + 32 * (lane >> 4);
  const T* x = static_cast<const T*>(p.x) + (long)col * p.ldm;
  float v[32];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 32; i++) {
    v[i] = col < p.m && k0 + i < p.k ? (float)x[(long)(k0 + i) * p.ldk] : 0.f;
    top = max(top, magnitude(v[i]));
  }
  const unsigned s = scale_byte(top, kFp4);
  const float f = unscale(s);
#pragma unroll
  for (int i = 0; i < 32; i++) v[i] *= f;
  u32x4 c;
#pragma unroll
  for (int i = 0; i < 4; i++) c[i] = s == 255u ? 0u : codes_fp4(v + 8 * i);
  const long piece = (long)blockIdx.x;
  *reinterpret_cast<u32x4*>(p.weight + piece * kStripCodes + tile * 1024 + lane * 16) = c;
  p.weight[(long)gridDim.x * kStripCodes + piece * kStripScales + lane * 4 + tile] = (uint8_t)s;
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

hipError_t launch_weight(const WeightParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)(strips(p.m) * groups(p.k)));
  if (p.type == kF32)
    hipLaunchKernelGGL(weight_kernel<kF32>, grid, dim3(256), 0, stream, p);
  else if (p.type == kF16)
    hipLaunchKernelGGL(weight_kernel<kF16>, grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL(weight_kernel<kBf16>, grid, dim3(256), 0, stream, p);
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
