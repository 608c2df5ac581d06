// Products of microscaled rows (e4m3 or e2m1) with a microscaled e2m1 weight on the scaled matrix
// cores (gfx950): out = epilogue(sum_k x[r][k] w[k][c]). Operands and layouts: mx.hpp.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 with the weight as the first operand: D[column][row], so a lane has
// four neighbouring columns of one row of the output. Its e2m1 operand has k 32 (l / 16) .. + 31 in lane
// l, its e4m3 operand k 16 (l / 16) .. + 15 and 64 more; the scale byte of lane l counts for k block
// l / 16 of row l % 16 in both.
//
// The hardware sums products of eight neighbouring k with 13 bits below the largest of them, then goes
// on in fp32. e2m1 products always fit, e4m3 rows do not: on normal data the result is 4e-6 (rms) off.
// Where the result keeps more than that (fp32, and codes, which flip at a border), an e4m3 operand is
// split into its values of at least 2 and those below (in units of the block's scale), each of which
// fits, and multiplied in two passes: 7e-9.
#include "gemm.hpp"
#include "mx.hpp"

namespace ancha {
namespace mx {
namespace {

typedef unsigned u32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 zero4() {
  f32x4 z = {0.f, 0.f, 0.f, 0.f};
  asm volatile("" : "+v"(z));
  return z;
}

// acc += w . x over 128 k; byte B of ws and byte 0 of xs are the lane's scales.
template <int FORMAT, int B>
__device__ __forceinline__ f32x4 mfma(u32x4 w, unsigned ws, u32x8 x, unsigned xs, f32x4 acc) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      a, __builtin_bit_cast(i32x8, x), acc, 4, FORMAT == kFp8 ? 0 : 4, B, (int)ws, 0, (int)xs);
}

// The e4m3 codes with the top exponent bit set (magnitude 2 or more, and NaN), or those without;
// zeros (of either sign) in place of the others.
__device__ __forceinline__ unsigned large_part(unsigned c) {
  const unsigned t = c & 0x40404040u;
  return c & (((t << 1) - (t >> 6)) | 0x80808080u);
}
__device__ __forceinline__ unsigned small_part(unsigned c) {
  const unsigned t = c & 0x40404040u;
  return c & ~((t << 1) - (t >> 6));
}

constexpr bool kCodes(int out) { return out == kFp8 || out == kFp4; }

// Four neighbouring columns c .. c + 3 of row r of the product through the epilogue; OUT is the type of
// the result (and of the residual), or the format of its codes (fp32 residual). Columns of the filling
// become 0, also in a NaN row.
template <int OUT>
__device__ __forceinline__ void finish(const LinearParams& p, long r, int c, float* v) {
  constexpr int TYPE = kCodes(OUT) ? kF32 : OUT;
  if (p.bias) {
    float b[4];
    load_row<kF32, 4>(p.bias, c < p.m ? c : 0, p.m - c, b);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] += b[i];
  }
  if (p.gelu)
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = OUT == kF32 ? gemm::gelu_erf(v[i]) : gemm::gelu_fast(v[i]);
  if (p.rope && c < 2 * p.width) {
    const long t = (long)(r % p.tokens) * 64 + (c & 63);
    const float* table = p.rope + (c < p.width ? 0 : 2) * (long)p.tokens * 64 + t;
    float cs[4], sn[4];
    __builtin_memcpy(cs, table, 16);
    __builtin_memcpy(sn, table + (long)p.tokens * 64, 16);
    const float4 y = rotate4(make_float4(v[0], v[1], v[2], v[3]), make_float4(cs[0], cs[1], cs[2], cs[3]),
                             make_float4(sn[0], sn[1], sn[2], sn[3]));
    v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
  }
  if (p.residual) {
    float x[4];
    load_row<TYPE, 4>(p.residual, c < p.m ? r * p.m + c : 0, p.m - c, x);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] += x[i];
  }
  if (kCodes(OUT) && c + 3 >= p.m)
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = c + i < p.m ? v[i] : 0.f;
}

// The epilogue of a strip of 64 columns of one row: lane l has columns c0 + 16 t + 4 (l / 16) .. + 3 in
// acc[t]. `here`: the row exists (the lanes of a row agree).
template <int OUT>
__device__ __forceinline__ void finish_strip(const LinearParams& p, long r, bool here, int c0,
                                             const f32x4* acc) {
  const int g = (threadIdx.x & 63) >> 4;
  const long rr = here ? r : 0;
  float v[4][4];
#pragma unroll
  for (int t = 0; t < 4; t++) {
    const int c = c0 + 16 * t + 4 * g;
#pragma unroll
    for (int i = 0; i < 4; i++) v[t][i] = acc[t][i];
    finish<OUT>(p, rr, c, v[t]);
    if constexpr (!kCodes(OUT))
      if (here && c < p.m) store_row<OUT, 4>(p.out, r * p.m + c, p.m - c, v[t]);
  }
  if constexpr (kCodes(OUT)) {
    // A block of 32 columns: two tiles, in lanes l % 16 + {0, 16, 32, 48}.
#pragma unroll
    for (int h = 0; h < 2; h++) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) top = max(top, magnitude(v[2 * h + i / 4][i % 4]));
      top = max(top, (unsigned)__shfl_xor((int)top, 16));
      top = max(top, (unsigned)__shfl_xor((int)top, 32));
      const unsigned s = scale_byte(top, OUT);
      const float f = unscale(s);
      const long block = rr * 4 * groups(p.m) + (c0 >> 5) + h;
      if (here && g == 0) p.out_scales[block] = (uint8_t)s;
#pragma unroll
      for (int t = 0; t < 2; t++) {
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = i < 4 ? v[2 * h + t][i] * f : 0.f;
        if (!here) continue;
        if constexpr (OUT == kFp8)
          *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(p.out) + block * 32 + 16 * t + 4 * g) =
              s == 255u ? 0u : codes_fp8(q[0], q[1], q[2], q[3]);
        else
          *reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(p.out) + block * 16 + 8 * t + 2 * g) =
              s == 255u ? (uint16_t)0 : (uint16_t)codes_fp4(q);
      }
    }
  }
}

// acc[t] += (fragment t of the strip) . x for the four fragments of a strip, in two passes where the
// e4m3 operand is split.
template <int FORMAT, bool SPLIT>
__device__ __forceinline__ void multiply(const u32x4* a, unsigned sa, u32x8 b, u32x8 small, unsigned sb,
                                         f32x4* acc) {
  acc[0] = mfma<FORMAT, 0>(a[0], sa, b, sb, acc[0]);
  acc[1] = mfma<FORMAT, 1>(a[1], sa, b, sb, acc[1]);
  acc[2] = mfma<FORMAT, 2>(a[2], sa, b, sb, acc[2]);
  acc[3] = mfma<FORMAT, 3>(a[3], sa, b, sb, acc[3]);
  if constexpr (SPLIT) {
    acc[0] = mfma<FORMAT, 0>(a[0], sa, small, sb, acc[0]);
    acc[1] = mfma<FORMAT, 1>(a[1], sa, small, sb, acc[1]);
    acc[2] = mfma<FORMAT, 2>(a[2], sa, small, sb, acc[2]);
    acc[3] = mfma<FORMAT, 3>(a[3], sa, small, sb, acc[3]);
  }
}

template <int FORMAT>
__device__ __forceinline__ u32x8 operand(u32x4 lo, u32x4 hi) {
  return FORMAT == kFp8 ? u32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}
                        : u32x8{lo[0], lo[1], lo[2], lo[3], 0, 0, 0, 0};
}

// 16 (or 4) bytes a lane from base + off straight to LDS at `to` + 16 (4) * lane.
template <int BYTES>
__device__ __forceinline__ void to_lds(const uint8_t* base, unsigned off, uint8_t* to) {
  const auto* from = (const __attribute__((address_space(1))) void*)(base + off);
  auto* lds = (__attribute__((address_space(3))) void*)to;
  if constexpr (BYTES == 16)
    __builtin_amdgcn_global_load_lds(from, lds, 16, 0, 0);
  else
    __builtin_amdgcn_global_load_lds(from, lds, 4, 0, 0);
}

// Waits until at most N vector memory operations of this wave are in flight, and for all of its LDS
// reads (gfx9 encoding).
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x70);
}

// A workgroup barrier without the wait for this wave's loads to LDS that __syncthreads() would make; no
// memory access moves across it.
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A workgroup of WM x WN waves has 64 SM WM columns and 16 TN WN rows; a wave SM strips of 64 columns
// and TN tiles of 16 rows, its accumulators in registers. Per step of 128 k both operands and their
// scales go straight from memory to LDS, two steps ahead, in three buffers: one barrier per step, behind
// which the buffer of the step before is free.
//
// A row's 16-byte chunks lie in LDS at chunk ^ (row & 7) (e4m3: 128 bytes a row; e2m1: 64 bytes, chunk ^
// (row / 2 & 3)), so that the eight lanes that are served together hit different banks; the loads to LDS
// write in lane order, so the lanes choose their chunk in memory instead. Weight fragments are in lane
// order already.
template <int FORMAT, bool SPLIT, int OUT, int WM, int WN, int SM, int TN>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(LinearParams p, unsigned mtiles,
                                                            unsigned ntiles) {
  constexpr int W = WM * WN, STRIPS = WM * SM, ROWS = 16 * TN * WN;
  constexpr int kRow = FORMAT == kFp8 ? 128 : 64;           // bytes of a row and step
  constexpr int kX = ROWS * kRow, kW = STRIPS * (int)kStripCodes;
  constexpr int kXS = kX + kW, kWS = kXS + ROWS * 4, kStage = kWS + STRIPS * (int)kStripScales;
  constexpr int PX = kX / 1024 / W, PW = kW / 1024 / W;     // 1 KiB pieces per wave
  constexpr int QX = ROWS / 64, Q = (QX + STRIPS + W - 1) / W;  // 256-byte pieces of scales
  static_assert(PX * W * 1024 == kX && PW * W * 1024 == kW && QX * 64 == ROWS, "whole pieces");
  constexpr int kLoads = PX + PW + Q;
  __shared__ __attribute__((aligned(16))) uint8_t lds[3][kStage];
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;

  // Workgroups that run at the same time on an XCD share its L2: four row tiles by neighbouring column
  // tiles.
  const unsigned id = (unsigned)xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const unsigned band = id / (4 * mtiles), rest = id - band * 4 * mtiles;
  const unsigned high = min(4u, ntiles - 4 * band);
  const unsigned mt = rest / high, nt = 4 * band + (rest - mt * high);
  const long row0 = (long)nt * ROWS;
  const int strip0 = (int)mt * STRIPS, nstrips = (int)strips(p.m);
  const int steps = (int)groups(p.k);

  const uint8_t* x = p.x + row0 * steps * kRow;
  const uint8_t* xs = p.x_scales + row0 * steps * 4;
  const uint8_t* w = p.weight + (long)strip0 * steps * kStripCodes;
  const uint8_t* ws = p.weight + (long)nstrips * steps * kStripCodes + (long)strip0 * steps * kStripScales;
  const int last_row = (int)min((long)ROWS - 1, p.n - 1 - row0);  // rows behind the last repeat it
  const int last_strip = min(STRIPS - 1, nstrips - 1 - strip0);
  unsigned xo[PX], wo[PW], qo[Q];
#pragma unroll
  for (int i = 0; i < PX; i++) {
    const int piece = wave * PX + i;
    int r, c;
    if constexpr (FORMAT == kFp8) {
      r = 8 * piece + (lane >> 3);
      c = (lane & 7) ^ (r & 7);
    } else {
      r = 16 * piece + 2 * (lane >> 3) + ((lane >> 2) & 1);
      c = (lane & 3) ^ ((r >> 1) & 3);
    }
    xo[i] = (unsigned)min(r, last_row) * (unsigned)(steps * kRow) + 16 * c;
  }
#pragma unroll
  for (int i = 0; i < PW; i++) {
    const int piece = wave * PW + i;
    wo[i] = (unsigned)min(piece >> 2, last_strip) * (unsigned)(steps * kStripCodes) +
            (piece & 3) * 1024 + lane * 16;
  }
#pragma unroll
  for (int i = 0; i < Q; i++) {
    const int piece = min(wave * Q + i, QX + STRIPS - 1);
    qo[i] = piece < QX ? (unsigned)min(64 * piece + lane, last_row) * (unsigned)(steps * 4)
                       : (unsigned)min(piece - QX, last_strip) * (unsigned)(steps * kStripScales) + lane * 4;
  }
  auto load = [&](int s, uint8_t* to) {
#pragma unroll
    for (int i = 0; i < PX; i++) to_lds<16>(x + (long)s * kRow, xo[i], to + (wave * PX + i) * 1024);
#pragma unroll
    for (int i = 0; i < PW; i++)
      to_lds<16>(w + (long)s * kStripCodes, wo[i], to + kX + (wave * PW + i) * 1024);
#pragma unroll
    for (int i = 0; i < Q; i++) {
      const int piece = min(wave * Q + i, QX + STRIPS - 1);
      to_lds<4>(piece < QX ? xs + (long)s * 4 : ws + (long)s * kStripScales, qo[i], to + kXS + piece * 256);
    }
  };

  f32x4 acc[TN][SM][4];
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int a = 0; a < SM; a++)
#pragma unroll
      for (int t = 0; t < 4; t++) acc[j][a][t] = zero4();

  // This lane's places in a row tile and in the weight.
  int xa[2];
  const int r = lane & 15;
  if constexpr (FORMAT == kFp8) {
    xa[0] = r * 128 + ((g ^ (r & 7)) << 4);
    xa[1] = r * 128 + (((4 + g) ^ (r & 7)) << 4);
  } else {
    xa[0] = xa[1] = r * 64 + ((g ^ ((r >> 1) & 3)) << 4);
  }

  load(0, lds[0]);
  if (steps > 1) load(1, lds[1]);
  int b = 0;
  for (int s = 0; s < steps; s++) {
    if (s + 1 < steps)
      wait_loads<kLoads>();
    else
      wait_loads<0>();
    barrier();
    if (s + 2 < steps) load(s + 2, lds[b == 0 ? 2 : b - 1]);
    const uint8_t* from = lds[b];
    u32x4 a[SM][4];
    unsigned sa[SM];
#pragma unroll
    for (int i = 0; i < SM; i++) {
      const int strip = wm * SM + i;
#pragma unroll
      for (int t = 0; t < 4; t++)
        a[i][t] = *reinterpret_cast<const u32x4*>(from + kX + strip * kStripCodes + t * 1024 + lane * 16);
      sa[i] = *reinterpret_cast<const unsigned*>(from + kWS + strip * kStripScales + lane * 4);
    }
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int tile = wn * TN + j;
      const uint8_t* at = from + tile * 16 * kRow;
      const u32x4 lo = *reinterpret_cast<const u32x4*>(at + xa[0]);
      const u32x4 hi = FORMAT == kFp8 ? *reinterpret_cast<const u32x4*>(at + xa[1]) : lo;
      const unsigned sb = from[kXS + (tile * 16 + r) * 4 + g];
      u32x8 large = operand<FORMAT>(lo, hi), small = large;
      if constexpr (SPLIT)
#pragma unroll
        for (int i = 0; i < 8; i++) small[i] = small_part(large[i]), large[i] = large_part(large[i]);
#pragma unroll
      for (int i = 0; i < SM; i++) multiply<FORMAT, SPLIT>(a[i], sa[i], large, small, sb, acc[j][i]);
    }
    b = b == 2 ? 0 : b + 1;
  }
#pragma unroll
  for (int j = 0; j < TN; j++) {
    const long row = row0 + (wn * TN + j) * 16 + r;
#pragma unroll
    for (int i = 0; i < SM; i++) {
      const int strip = strip0 + wm * SM + i;
      if (strip < nstrips) finish_strip<OUT>(p, row, row < p.n, strip * 64, acc[j][i]);
    }
  }
}

template <int FORMAT, bool SPLIT, int OUT, int WM, int WN, int SM, int TN>
void start_tiles(const LinearParams& p, hipStream_t stream) {
  const unsigned mtiles = (unsigned)((strips(p.m) + WM * SM - 1) / (WM * SM));
  const unsigned ntiles = (unsigned)(((long)p.n + 16 * TN * WN - 1) / (16 * TN * WN));
  hipLaunchKernelGGL((tile_kernel<FORMAT, SPLIT, OUT, WM, WN, SM, TN>), dim3(mtiles * ntiles),
                     dim3(64 * WM * WN), 0, stream, p, mtiles, ntiles);
}

// The result's type or format picks the kernel: e4m3 rows are split for fp32 and for codes.
template <int OUT>
hipError_t linear_to(const LinearParams& p, hipStream_t stream) {
  constexpr bool kSplit = OUT == kF32 || kCodes(OUT);
  const bool wide = (long)((p.n + 255) / 256) * ((p.m + 255) / 256) >= 256;
  if (p.format == kFp4) {
    if (wide)
      start_tiles<kFp4, false, OUT, 2, 4, 2, 4>(p, stream);
    else
      start_tiles<kFp4, false, OUT, 2, 2, 1, 4>(p, stream);
  } else {
    if (wide)
      start_tiles<kFp8, kSplit, OUT, 2, 4, 2, 4>(p, stream);
    else
      start_tiles<kFp8, kSplit, OUT, 2, 2, 1, 4>(p, stream);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_linear(const LinearParams& p, hipStream_t stream) {
  switch (p.out_format ? p.out_format : p.type) {
    case kF32: return linear_to<kF32>(p, stream);
    case kF16: return linear_to<kF16>(p, stream);
    case kBf16: return linear_to<kBf16>(p, stream);
    case kFp8: return linear_to<kFp8>(p, stream);
    default: return linear_to<kFp4>(p, stream);
  }
}

}  // namespace mx
}  // namespace ancha
