// Products of microscaled rows (e4m3 or e2m1) with a microscaled e2m1 weight on the scaled matrix
// cores (gfx950): out = epilogue(sum_k x[r][k] w[k][c]). Operands and layouts: mx.hpp.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 with the weight as the first operand: D[column][row], so a lane has
// four neighbouring columns of one row of the output. Its e2m1 operand has k 32 (l / 16) .. + 31 in lane
// l, its e4m3 operand k 16 (l / 16) .. + 15 and 64 more; the scale byte of lane l counts for k block
// l / 16 of row l % 16 in both.
//
// The hardware sums products of eight neighbouring k with 13 bits below the largest of them, then goes
// on in fp32. e2m1 products always fit, e4m3 rows do not: a product 2^-13 of one beside it is lost, which is
// all of the result where the large ones cancel. So an e4m3 operand is split into its values of at least 2
// and those below (in units of the block's scale), each of which fits, and multiplied in two passes: 7e-9
// (rms, of the result on normal data; 4e-6 in one pass, which would save the matrix cores half their time).
#include <algorithm>

#include "buffer.hpp"
#include "mx.hpp"

namespace ancha {

int device_cus();

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

// Four e4m3 codes, those with the top exponent bit set (magnitude 2 or more, and NaN) apart from the
// others; zeros in place of those that went the other way. v_perm_b32's selectors 8 .. 11 spread the
// sign of a byte over eight bits: of S1's bytes 1 and 3 (the codes shifted up by one), then of S0's.
__device__ __forceinline__ void split(unsigned c, unsigned& large, unsigned& small) {
  const unsigned mask = __builtin_amdgcn_perm(c << 9, c << 1, 0x090b080au);
  large = c & mask;
  small = c & ~mask;
}

// Whether OUT names a format of codes (or a type of values).
constexpr bool kCodes(int out) { return out == kFp8 || out == kFp4; }

// erf-GELU: x Phi(x) = max(x, 0) - |x| 2^Q(|x|) with Q a polynomial for log2 Phi(-a) on [0, 13.2], beyond which
// the product is below fp32's normal range (Q goes on falling). Degree 12 for fp32 results, 10 for others. Its
// error relative to the value, fitted to least weighted maxima (tests hold it to somewhat larger ones):
//   x                       above -2   -4 .. -2   -6 .. -4   -8 .. -6   below
//   fp32                    7e-7       3e-6       6e-5       8e-4       2e-3
//   16 bits and codes       2e-6       2e-5       8e-4       9e-4       2.3e-3
// so rows of nothing but small results have right codes and 16-bit values as well. One exp2 and the polynomial, as
// the vector ALU bounds these epilogues: 96 120 x 384 -> 1536 with bias and GELU to codes 152 us (as long with
// erf's rational form, which has no small results right), to fp32 173 (229 with erff).
template <int OUT>
__device__ __forceinline__ float gelu(float x) {
  constexpr bool WIDE = OUT == kF32;
  const float a = fabsf(x);
  float q;
  if constexpr (WIDE) {
    q = fmaf(a, -2.891597725e-11f, 1.983803566e-9f);
    q = fmaf(a, q, -5.875872588e-8f);
    q = fmaf(a, q, 9.840832718e-7f);
    q = fmaf(a, q, -1.020369382e-5f);
    q = fmaf(a, q, 6.611218123e-5f);
    q = fmaf(a, q, -2.319509658e-4f);
    q = fmaf(a, q, -1.162716435e-4f);
    q = fmaf(a, q, 7.105765864e-3f);
    q = fmaf(a, q, -5.255914479e-2f);
    q = fmaf(a, q, -4.591782987e-1f);
    q = fmaf(a, q, -1.151109934f);
    q = fmaf(a, q, -9.999998808e-1f);
  } else {
    q = fmaf(a, -9.846427007e-10f, 5.148060822e-8f);
    q = fmaf(a, q, -1.048340096e-6f);
    q = fmaf(a, q, 9.514340491e-6f);
    q = fmaf(a, q, -1.032696582e-5f);
    q = fmaf(a, q, -6.584623479e-4f);
    q = fmaf(a, q, 7.906456478e-3f);
    q = fmaf(a, q, -5.322779343e-2f);
    q = fmaf(a, q, -4.588992e-1f);
    q = fmaf(a, q, -1.151154518f);
    q = fmaf(a, q, -9.999986887e-1f);
  }
  // An infinity times 0 would be NaN.
  return fmaf(-fminf(a, 1e30f), __builtin_amdgcn_exp2f(q), fmaxf(x, 0.f));
}

constexpr int kOutStage = 4096;  // LDS bytes per wave for one 16 x 64 tile on its way out

// Where a workgroup's rows lie: buffers over them, so that rows behind the last one read as 0 and are
// not written, or plain pointers (DIRECT) where a row is not whole groups of four columns or the rows
// reach past 32-bit offsets.
template <int OUT>
struct Rows {
  static constexpr int kType = kCodes(OUT) ? kF32 : OUT;
  static constexpr int kSize = kType == kF32 ? 4 : 2;  // of the residual and of uncoded results
  rsrc_t out, residual;
  long row0;
  int rows;
};

template <int OUT>
__device__ __forceinline__ Rows<OUT> rows_of(const LinearParams& p, long row0, int rows) {
  Rows<OUT> d;
  d.row0 = row0;
  d.rows = rows;
  const long row = kCodes(OUT) ? pitch(p.m, OUT) : (long)p.m * d.kSize;
  d.out = make_rsrc(static_cast<uint8_t*>(p.out) + row0 * row, (unsigned)(rows * row));
  const long span = (long)p.m * d.kSize;
  d.residual = make_rsrc(p.residual ? static_cast<const uint8_t*>(p.residual) + row0 * span : p.out,
                         p.residual ? (unsigned)(rows * span) : 0u);
  return d;
}

__device__ __forceinline__ void unpack(u32x2 w, bool half, float* v) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const unsigned short h = (unsigned short)(w[i / 2] >> (16 * (i & 1)));
    v[i] = half ? (float)__builtin_bit_cast(_Float16, h) : (float)__builtin_bit_cast(__bf16, h);
  }
}

// The residual of four neighbouring columns c .. of row r of the workgroup.
template <int OUT, bool DIRECT>
__device__ __forceinline__ void load_residual(const LinearParams& p, const Rows<OUT>& d, int r, int c,
                                              float* v) {
  constexpr int TYPE = Rows<OUT>::kType;
  if constexpr (DIRECT) {
    const bool here = r < d.rows && c < p.m;
    load_row<TYPE, 4>(p.residual, here ? (d.row0 + r) * p.m + c : 0, here ? p.m - c : 0, v);
  } else {
    const unsigned off = c < p.m ? ((unsigned)r * (unsigned)p.m + c) * d.kSize : 0x80000000u;
    if constexpr (TYPE == kF32) {
      const float4 x = bload4<true>(d.residual, off);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      unpack(__builtin_amdgcn_raw_buffer_load_b64(d.residual, off, 0, 0), TYPE == kF16, v);
    }
  }
}

template <int OUT, bool DIRECT>
__device__ __forceinline__ void store_values(const LinearParams& p, const Rows<OUT>& d, int r, int c,
                                             const float* v) {
  if constexpr (DIRECT) {
    if (r < d.rows && c < p.m) store_row<OUT, 4>(p.out, (d.row0 + r) * p.m + c, p.m - c, v);
  } else {
    const unsigned off = c < p.m ? ((unsigned)r * (unsigned)p.m + c) * d.kSize : 0x80000000u;
    if constexpr (OUT == kF32) {
      bstore4<true, kStream>(d.out, off, make_float4(v[0], v[1], v[2], v[3]));
    } else {
      typename Stored<OUT>::type t[4];
#pragma unroll
      for (int i = 0; i < 4; i++) t[i] = (typename Stored<OUT>::type)v[i];
      u32x2 w;
      __builtin_memcpy(&w, t, 8);
      __builtin_amdgcn_raw_buffer_store_b64(w, d.out, off, 0, kStream);
    }
  }
}

// Sixteen neighbouring values a lane, a block of 32 by lanes l and l ^ 16, to codes and the scale byte,
// with saturate() in effect.
template <int OUT>
__device__ __forceinline__ unsigned encode16(const float* v, unsigned* codes) {
  unsigned top = top_exponent<16>(v);
  const auto both = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = max((unsigned)both[0], (unsigned)both[1]);
  const unsigned s = scale_byte(top, OUT);
  const float f = divisor(s);
#pragma unroll
  for (int i = 0; i < (OUT == kFp8 ? 4 : 2); i++) {
    const unsigned c = OUT == kFp8 ? codes_fp8(v + 4 * i, f) : codes_fp4(v + 8 * i, f);
    codes[i] = s == 255u ? 0u : c;
  }
  return s;
}

// Turns acc[t] of a 16 x 64 tile as the MFMAs leave it (lane l: row l % 16, columns 16 t + 4 (l / 16) ..
// + 3) into sixteen neighbouring columns of the same row: lane l has columns 16 (l / 16) + 4 t .. + 3 in
// v[4 t] .. (a transposition of four lane groups and four registers, by exchanges of half and quarter
// waves).
__device__ __forceinline__ void gather16(const f32x4* acc, float* v) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    unsigned x[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const float y = acc[t][e];  // a bit cast of the vector's element itself takes element 0
      x[t] = __builtin_bit_cast(unsigned, y);
    }
    const auto a = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    v[e] = __builtin_bit_cast(float, (unsigned)c[0]);
    v[4 + e] = __builtin_bit_cast(float, (unsigned)c[1]);
    v[8 + e] = __builtin_bit_cast(float, (unsigned)d[0]);
    v[12 + e] = __builtin_bit_cast(float, (unsigned)d[1]);
  }
}

// The epilogue of 16 rows r0 .. and a strip of 64 columns c0 .. to codes; bias[i]: column c0 + 16 (l / 16)
// + i. Columns of the filling become 0, also in a NaN row.
template <int OUT, bool DIRECT>
__device__ __forceinline__ void finish_codes(const LinearParams& p, const Rows<OUT>& d, int r0, int c0,
                                             const float* bias, const f32x4* acc) {
  const int lane = threadIdx.x & 63, r = r0 + (lane & 15), c = c0 + 16 * (lane >> 4);
  float v[16];
  gather16(acc, v);
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] += bias[i];
  if (p.gelu)
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = gelu<OUT>(v[i]);
  if (p.rope && c < 2 * p.width) {
    const unsigned token = (unsigned)(d.row0 + r) % (unsigned)p.tokens;
    const float* table = p.rope + (c < p.width ? 0 : 2) * (long)p.tokens * 64 + token * 64ul + (c & 63);
#pragma unroll
    for (int t = 0; t < 4; t++) {
      float cs[4], sn[4];
      __builtin_memcpy(cs, table + 4 * t, 16);
      __builtin_memcpy(sn, table + (long)p.tokens * 64 + 4 * t, 16);
      float* y = v + 4 * t;
      const float4 z = rotate4(make_float4(y[0], y[1], y[2], y[3]), make_float4(cs[0], cs[1], cs[2], cs[3]),
                               make_float4(sn[0], sn[1], sn[2], sn[3]));
      y[0] = z.x, y[1] = z.y, y[2] = z.z, y[3] = z.w;
    }
  }
  if (p.residual)
#pragma unroll
    for (int t = 0; t < 4; t++) {
      float x[4];
      load_residual<OUT, DIRECT>(p, d, r, c + 4 * t, x);
#pragma unroll
      for (int i = 0; i < 4; i++) v[4 * t + i] += x[i];
    }
  if (c0 + 64 > p.m)
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = c + i < p.m ? v[i] : 0.f;
  unsigned codes[4];
  const unsigned s = encode16<OUT>(v, codes);
  const unsigned width = 128u * (unsigned)groups(p.m);  // values of a stored row
  const unsigned at = (unsigned)r * width + c;
  if constexpr (OUT == kFp8)
    __builtin_amdgcn_raw_buffer_store_b128(u32x4{codes[0], codes[1], codes[2], codes[3]}, d.out, at, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{codes[0], codes[1]}, d.out, at >> 1, 0, 0);
  if ((lane & 16) == 0 && r < d.rows)
    p.out_scales[(d.row0 + r) * (long)(width >> 5) + (c >> 5)] = (uint8_t)s;
}

// The epilogue of 16 rows r0 .. of the workgroup and a strip of 64 columns c0 ..; acc[t] as the MFMAs
// leave it: lane l has row l % 16, columns 16 t + 4 (l / 16) .. + 3. The tile passes through `st` (row of
// 256 bytes, 16-byte chunk c of row r at c ^ r), so that sixteen lanes have a row's 64 neighbouring
// columns: whole rows of the strip are read and written, past the caches: 96 120 x 384 -> 1536 to fp32 122 us
// (5.2 TB/s), 297 in pieces of 64 bytes through them.
template <int OUT, bool DIRECT>
__device__ __forceinline__ void finish_tile(const LinearParams& p, const Rows<OUT>& d, int r0, int c0,
                                            const float* bias, const f32x4* acc, const int* tokens,
                                            uint8_t* st) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int c = c0 + 4 * r;
  float x[4][4], v[4][4];
  if (p.residual)
#pragma unroll
    for (int q = 0; q < 4; q++) load_residual<OUT, DIRECT>(p, d, r0 + 4 * q + g, c, x[q]);
#pragma unroll
  for (int t = 0; t < 4; t++) *reinterpret_cast<f32x4*>(st + r * 256 + (((4 * t + g) ^ r) << 4)) = acc[t];
#pragma unroll
  for (int q = 0; q < 4; q++) {
    const int tr = 4 * q + g;
    const f32x4 y = *reinterpret_cast<const f32x4*>(st + tr * 256 + ((r ^ tr) << 4));
#pragma unroll
    for (int i = 0; i < 4; i++) v[q][i] = y[i] + bias[i];
  }
  if (p.gelu)
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        v[q][i] = gelu<OUT>(v[q][i]);
  if (p.rope && c < 2 * p.width) {
    const float* table = p.rope + (c < p.width ? 0 : 2) * (long)p.tokens * 64 + (c & 63);
#pragma unroll
    for (int q = 0; q < 4; q++) {
      float cs[4], sn[4];
      const float* at = table + tokens[r0 + 4 * q + g] * 64l;
      __builtin_memcpy(cs, at, 16);
      __builtin_memcpy(sn, at + (long)p.tokens * 64, 16);
      const float4 y = rotate4(make_float4(v[q][0], v[q][1], v[q][2], v[q][3]),
                               make_float4(cs[0], cs[1], cs[2], cs[3]),
                               make_float4(sn[0], sn[1], sn[2], sn[3]));
      v[q][0] = y.x, v[q][1] = y.y, v[q][2] = y.z, v[q][3] = y.w;
    }
  }
  if (p.residual)
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
      for (int i = 0; i < 4; i++) v[q][i] += x[q][i];
#pragma unroll
  for (int q = 0; q < 4; q++) store_values<OUT, DIRECT>(p, d, r0 + 4 * q + g, c, v[q]);
}

// The epilogue of a wave: SM strips from column c0 on, TN tiles of 16 rows from r0 on.
template <int OUT, bool DIRECT, int SM, int TN>
__device__ __forceinline__ void finish_wave(const LinearParams& p, const Rows<OUT>& d, int r0, int c0,
                                            const f32x4 (*acc)[SM][4], const int* tokens, uint8_t* st) {
  constexpr int N = kCodes(OUT) ? 16 : 4;  // neighbouring columns of a lane
  const int c = c0 + (kCodes(OUT) ? 16 * ((threadIdx.x & 63) >> 4) : 4 * (threadIdx.x & 15));
#pragma unroll
  for (int i = 0; i < SM; i++) {
    if (c0 + 64 * i >= 64 * (int)strips(p.m)) break;
    float bias[N] = {};
    if (p.bias) load_row<kF32, N>(p.bias, c + 64 * i < p.m ? c + 64 * i : 0, p.m - c - 64 * i, bias);
#pragma unroll
    for (int j = 0; j < TN; j++) {
      if constexpr (kCodes(OUT))
        finish_codes<OUT, DIRECT>(p, d, r0 + 16 * j, c0 + 64 * i, bias, acc[j][i]);
      else
        finish_tile<OUT, DIRECT>(p, d, r0 + 16 * j, c0 + 64 * i, bias, acc[j][i], tokens, st);
    }
  }
}

// acc[t] += (fragment t of the strip) . x for the four fragments of a strip, an e4m3 operand in its two
// parts.
template <int FORMAT>
__device__ __forceinline__ void multiply(const u32x4* a, unsigned sa, u32x8 b, u32x8 small, unsigned sb,
                                         f32x4* acc) {
  acc[0] = mfma<FORMAT, 0>(a[0], sa, b, sb, acc[0]);
  acc[1] = mfma<FORMAT, 1>(a[1], sa, b, sb, acc[1]);
  acc[2] = mfma<FORMAT, 2>(a[2], sa, b, sb, acc[2]);
  acc[3] = mfma<FORMAT, 3>(a[3], sa, b, sb, acc[3]);
  if constexpr (FORMAT == kFp8) {
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
// scales go straight from memory to LDS, ST - 1 steps ahead, in ST buffers: one barrier per step, behind
// which the buffer of the step before is free. OCC: waves per SIMD that the registers leave room for.
//
// KG > 1: that many such groups of waves take the steps in turn, for few tiles with a long k, where the
// time is the chain of steps; the first adds up the sums of all.
//
// A row's 16-byte chunks lie in LDS at chunk ^ (row & 7) (e4m3: 128 bytes a row; e2m1: 64 bytes, chunk ^
// (row / 2 & 3)), so that the eight lanes that are served together hit different banks; the loads to LDS
// write in lane order, so the lanes choose their chunk in memory instead. Weight fragments are in lane
// order already.
//
// Long k: bound by the matrix cores, 8192 x 8192 x 8192 e2m1 to bf16 289 us (3.8 PFLOP/s; 4.5 in a bare loop of
// the instruction), e4m3, twice the products, 620 us (3.5 PFLOP/s of them; 4.2 in a bare loop). Short k: by the epilogue's vector instructions and the results, 96 120 x 384 ->
// 1536 with bias and GELU to e4m3 152 us.
template <int FORMAT, int OUT, int WM, int WN, int SM, int TN, int ST, int OCC, int KG = 1>
__global__ __launch_bounds__(64 * WM * WN * KG, OCC) void tile_kernel(LinearParams p, unsigned mtiles,
                                                            unsigned ntiles, int direct) {
  constexpr int W = WM * WN, STRIPS = WM * SM, ROWS = 16 * TN * WN;
  constexpr int kRow = FORMAT == kFp8 ? 128 : 64;           // bytes of a row and step
  constexpr int kX = ROWS * kRow, kW = STRIPS * (int)kStripCodes;
  constexpr int kXS = kX + kW, kWS = kXS + ROWS * 4, kStageBytes = kWS + STRIPS * (int)kStripScales;
  constexpr int PX = kX / 1024 / W, PW = kW / 1024 / W;     // 1 KiB pieces per wave
  constexpr int QX = ROWS / 64, Q = (QX + STRIPS + W - 1) / W;  // 256-byte pieces of scales
  static_assert(PX * W * 1024 == kX && PW * W * 1024 == kW && QX * 64 == ROWS, "whole pieces");
  constexpr int kLoads = PX + PW + Q;
  __shared__ __attribute__((aligned(16))) uint8_t lds[ST][KG][kStageBytes];
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int any = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = any % W, kg = any / W;
  const int wm = wave % WM, wn = wave / WM;

  // Workgroups that run at the same time on an XCD share its L2: four row tiles by neighbouring column
  // tiles.
  const unsigned id = (unsigned)xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const unsigned band = id / (4 * mtiles), rest = id - band * 4 * mtiles;
  const unsigned high = min(4u, ntiles - 4 * band);
  const unsigned mt = rest / high, nt = 4 * band + (rest - mt * high);
  const long row0 = (long)nt * ROWS;
  const int strip0 = (int)mt * STRIPS, nstrips = (int)strips(p.m);
  const int steps = (int)groups(p.k), chunks = (steps + KG - 1) / KG;

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
  // Chunk c: this group's step of it (the last step again behind the end, not multiplied).
  auto load = [&](int c, uint8_t* to) {
    const int s = KG == 1 ? c : min(c * KG + kg, steps - 1);
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

#pragma unroll
  for (int c = 0; c < ST - 1; c++)
    if (c < chunks) load(c, lds[c][kg]);
  int b = 0;
  for (int c = 0; c < chunks; c++) {
    if (c + ST - 2 < chunks)
      wait_loads<(ST - 2) * kLoads>();
    else
      wait_loads<0>();
    barrier();
    if (c + ST - 1 < chunks) load(c + ST - 1, lds[b == 0 ? ST - 1 : b - 1][kg]);
    const uint8_t* from = lds[b][kg];
    b = b == ST - 1 ? 0 : b + 1;
    if (KG > 1 && c * KG + kg >= steps) break;  // the last chunk: no barrier follows in the loop
    // A strip's fragments are read from LDS while the strip before it is multiplied (left to the compiler,
    // all of a step's reads come first and the matrix cores wait for the last).
    const uint8_t* wl = from + kX + wm * SM * kStripCodes + lane * 16;
    u32x4 a[2][4];
    auto fetch = [&](int i) {
#pragma unroll
      for (int t = 0; t < 4; t++)
        a[i & 1][t] = *reinterpret_cast<const u32x4*>(wl + i * kStripCodes + t * 1024);
    };
    u32x8 large[TN], small[TN];
    unsigned sa[SM], sb[TN];
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int tile = wn * TN + j;
      const uint8_t* at = from + tile * 16 * kRow;
      const u32x4 lo = *reinterpret_cast<const u32x4*>(at + xa[0]);
      const u32x4 hi = FORMAT == kFp8 ? *reinterpret_cast<const u32x4*>(at + xa[1]) : lo;
      sb[j] = from[kXS + (tile * 16 + r) * 4 + g];
      large[j] = operand<FORMAT>(lo, hi);
    }
#pragma unroll
    for (int i = 0; i < SM; i++)
      sa[i] = *reinterpret_cast<const unsigned*>(from + kWS + (wm * SM + i) * kStripScales + lane * 4);
    fetch(0);
#pragma unroll
    for (int i = 0; i < SM; i++) {
      if (i + 1 < SM) fetch(i + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < TN; j++) {
        if (i == 0) {
          small[j] = large[j];
          if constexpr (FORMAT == kFp8)
#pragma unroll
            for (int e = 0; e < 8; e++) {
              unsigned u, v;
              split(large[j][e], u, v);
              large[j][e] = u, small[j][e] = v;
            }
        }
        multiply<FORMAT>(a[i & 1], sa[i], large[j], small[j], sb[j], acc[j][i]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  constexpr int kSums = W * TN * SM * 4 * 1024;  // bytes of a group's sums
  static_assert((KG - 1) * kSums + W * kOutStage + ROWS * 4 <= ST * KG * kStageBytes,
                "sums and results on their way out fit the operands' buffers");
  uint8_t* free = &lds[0][0][0];
  int* tokens = reinterpret_cast<int*>(free + (KG - 1) * kSums + W * kOutStage);
  const int rows = (int)min((long)ROWS, p.n - row0);
  if (KG > 1 || !kCodes(OUT)) {
    // Every wave is done with the operands before something else takes their place.
    wait_loads<0>();
    barrier();
  }
  if (!kCodes(OUT) && p.rope && (int)threadIdx.x < ROWS)
    tokens[threadIdx.x] = (int)((unsigned)(row0 + threadIdx.x) % (unsigned)p.tokens);
  if constexpr (KG > 1) {
    if (kg)
#pragma unroll
      for (int q = 0; q < TN * SM * 4; q++)
        reinterpret_cast<f32x4*>(free + (kg - 1) * kSums)[(wave * TN * SM * 4 + q) * 64 + lane] =
            acc[q / (SM * 4)][q / 4 % SM][q % 4];
  }
  if (KG > 1 || (!kCodes(OUT) && p.rope)) __syncthreads();
  if constexpr (KG > 1) {
    if (kg) return;
#pragma unroll
    for (int o = 0; o < KG - 1; o++)
#pragma unroll
      for (int q = 0; q < TN * SM * 4; q++)
        acc[q / (SM * 4)][q / 4 % SM][q % 4] +=
            reinterpret_cast<const f32x4*>(free + o * kSums)[(wave * TN * SM * 4 + q) * 64 + lane];
  }
  if (kCodes(OUT)) saturate();  // behind the last product
  const Rows<OUT> d = rows_of<OUT>(p, row0, rows);
  const int c0 = (strip0 + wm * SM) * 64;
  if (direct)
    finish_wave<OUT, true, SM, TN>(p, d, wn * TN * 16, c0, acc, tokens,
                                      free + (KG - 1) * kSums + wave * kOutStage);
  else
    finish_wave<OUT, false, SM, TN>(p, d, wn * TN * 16, c0, acc, tokens,
                                      free + (KG - 1) * kSums + wave * kOutStage);
}

// Whether the rows of a workgroup are written (and the residual read) through plain pointers.
int direct_rows(const LinearParams& p, long rows) {
  return p.m % 4 != 0 || rows * (p.m + 128l) * 4 >= 1l << 31 ||
         (reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.residual)) % 4 != 0;
}

template <int FORMAT, int OUT, int WM, int WN, int SM, int TN, int ST, int OCC, int KG = 1>
void start_tiles(const LinearParams& p, hipStream_t stream) {
  const unsigned mtiles = (unsigned)((strips(p.m) + WM * SM - 1) / (WM * SM));
  const unsigned ntiles = (unsigned)(((long)p.n + 16 * TN * WN - 1) / (16 * TN * WN));
  hipLaunchKernelGGL((tile_kernel<FORMAT, OUT, WM, WN, SM, TN, ST, OCC, KG>), dim3(mtiles * ntiles),
                     dim3(64 * WM * WN * KG), 0, stream, p, mtiles, ntiles, direct_rows(p, 16 * TN * WN));
}

// Few rows: the weight is what has to be read. A workgroup has 32 columns and 16 TN rows; its waves (one
// to sixteen) take the steps of 128 k in turn, straight from memory, and add up their sums in LDS. Then
// eight threads have a row, four neighbouring columns each. Small weights are bound by the way to memory and the sum
// over the waves, large ones by memory; the weight from memory: 1 x 4096 x 4096 5.3 us, 1 x 4096 x 28 672 17 us (3.7
// TB/s), 1 x 4096 x 128 256 56 us (5.0 TB/s).
constexpr int kFewColumns = 32, kFewWaves = 16;

template <int FORMAT, int OUT, int TN>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(LinearParams p) {
  constexpr int kRow = FORMAT == kFp8 ? 128 : 64;
  constexpr int kPart = 16 * TN * kFewColumns * 4;  // bytes of one wave's sums
  extern __shared__ __attribute__((aligned(16))) uint8_t part[];
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int steps = (int)groups(p.k), nstrips = (int)strips(p.m);
  const int strip = (int)blockIdx.x >> 1, half = (int)blockIdx.x & 1;
  const long row0 = (long)blockIdx.y * (16 * TN);
  const uint8_t* w = p.weight + (long)strip * steps * kStripCodes + half * 2048 + lane * 16;
  const uint8_t* ws = p.weight + (long)nstrips * steps * kStripCodes +
                      (long)strip * steps * kStripScales + lane * 4 + half * 2;
  const uint8_t *x[TN], *xs[TN];
#pragma unroll
  for (int j = 0; j < TN; j++) {
    const long row = min(row0 + 16 * j + r, (long)p.n - 1);
    x[j] = p.x + row * steps * kRow + 16 * g;
    xs[j] = p.x_scales + row * steps * 4 + g;
  }
  f32x4 acc[TN][2];
#pragma unroll
  for (int j = 0; j < TN; j++) acc[j][0] = zero4(), acc[j][1] = zero4();
  // A step's loads are in flight together, one step's at a time: with up to 32 waves on a CU, two or four steps' of
  // a wave at once (all loads before the first product) gain nothing and cost registers, so workgroups: 1 x 4096 x
  // 14 336 9.4 us (two steps 10.8, four 10.9), 16 x 14 336 x 4096 14.9 (14.9, 15.0), 1 x 4096 x 4096 4.4 (4.4, 4.4).
  for (int s = wave; s < steps; s += waves) {
    const u32x4 a0 = *reinterpret_cast<const u32x4*>(w + (long)s * kStripCodes);
    const u32x4 a1 = *reinterpret_cast<const u32x4*>(w + (long)s * kStripCodes + 1024);
    const unsigned sa = *reinterpret_cast<const uint16_t*>(ws + (long)s * kStripScales);
    u32x4 lo[TN], hi[TN];
    unsigned sb[TN];
#pragma unroll
    for (int j = 0; j < TN; j++) {
      lo[j] = *reinterpret_cast<const u32x4*>(x[j] + (long)s * kRow);
      hi[j] = FORMAT == kFp8 ? *reinterpret_cast<const u32x4*>(x[j] + (long)s * kRow + 64) : lo[j];
      sb[j] = xs[j][s * 4l];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < TN; j++) {
      u32x8 large = operand<FORMAT>(lo[j], hi[j]), small = large;
      if constexpr (FORMAT == kFp8)
#pragma unroll
        for (int i = 0; i < 8; i++) {
          unsigned y, z;
          split(large[i], y, z);
          large[i] = y, small[i] = z;
        }
      acc[j][0] = mfma<FORMAT, 0>(a0, sa, large, sb[j], acc[j][0]);
      acc[j][1] = mfma<FORMAT, 1>(a1, sa, large, sb[j], acc[j][1]);
      if constexpr (FORMAT == kFp8) {
        acc[j][0] = mfma<FORMAT, 0>(a0, sa, small, sb[j], acc[j][0]);
        acc[j][1] = mfma<FORMAT, 1>(a1, sa, small, sb[j], acc[j][1]);
      }
    }
  }
  // Row of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7).
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int t = 0; t < 2; t++)
      *reinterpret_cast<f32x4*>(part + wave * kPart + (16 * j + r) * 128 + (((4 * t + g) ^ (r & 7)) << 4)) =
          acc[j][t];
  __syncthreads();
  if (kCodes(OUT)) saturate();  // behind the last product
  for (int i = (int)threadIdx.x; i < 16 * TN * 8; i += (int)blockDim.x) {
    const int tr = i >> 3, c = (int)blockIdx.x * kFewColumns + 4 * (i & 7);
    const long row = row0 + tr;
    const bool here = row < p.n;
    const uint8_t* at = part + tr * 128 + (((i & 7) ^ (tr & 7)) << 4);
    f32x4 y = *reinterpret_cast<const f32x4*>(at);
    for (int q = 1; q < waves; q++) y += *reinterpret_cast<const f32x4*>(at + q * kPart);
    float v[4] = {y[0], y[1], y[2], y[3]}, b[4];
    const int valid = here ? p.m - c : 0;
    const long to = valid > 0 ? row * p.m + c : 0;
    if (p.bias) {
      load_row<kF32, 4>(p.bias, valid > 0 ? c : 0, valid, b);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] += b[e];
    }
    if (p.gelu)
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = gelu<OUT>(v[e]);
    if (p.rope && here && c < 2 * p.width) {
      const float* table = p.rope + (c < p.width ? 0 : 2) * (long)p.tokens * 64 +
                           (unsigned)row % (unsigned)p.tokens * 64ul + (c & 63);
      float cs[4], sn[4];
      __builtin_memcpy(cs, table, 16);
      __builtin_memcpy(sn, table + (long)p.tokens * 64, 16);
      const float4 z = rotate4(make_float4(v[0], v[1], v[2], v[3]), make_float4(cs[0], cs[1], cs[2], cs[3]),
                               make_float4(sn[0], sn[1], sn[2], sn[3]));
      v[0] = z.x, v[1] = z.y, v[2] = z.z, v[3] = z.w;
    }
    if (p.residual) {
      load_row<Rows<OUT>::kType, 4>(p.residual, to, valid, b);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] += b[e];
    }
    if constexpr (!kCodes(OUT)) {
      if (valid > 0) store_row<OUT, 4>(p.out, to, valid, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = e < valid ? v[e] : 0.f;
      unsigned top = top_exponent<4>(v);
      top = max(top, dpp<kSwap1>(top));
      top = max(top, dpp<kSwap2>(top));
      top = max(top, dpp<kMirror8>(top));
      const unsigned s = scale_byte(top, OUT);
      const float f = divisor(s);
      if (!here) continue;
      const long unit = row * 32 * groups(p.m) + (c >> 2);  // four values
      if ((i & 7) == 0) p.out_scales[unit >> 3] = (uint8_t)s;
      uint8_t* out = static_cast<uint8_t*>(p.out);
      if constexpr (OUT == kFp8)
        *reinterpret_cast<unsigned*>(out + unit * 4) =
            s == 255u ? 0u : codes_fp8(v, f);
      else
        *reinterpret_cast<uint16_t*>(out + unit * 2) =
            s == 255u ? (uint16_t)0 : (uint16_t)codes_fp4x4(v, f);
    }
  }
}

template <int FORMAT, int OUT, int TN>
void start_few(const LinearParams& p, hipStream_t stream) {
  const int waves = (int)std::min<long>(kFewWaves, groups(p.k));
  // Codes have their filling written too.
  const unsigned columns = kCodes(OUT) ? (unsigned)strips(p.m) * 2 : (unsigned)((p.m + 31l) / 32);
  hipLaunchKernelGGL((few_kernel<FORMAT, OUT, TN>),
                     dim3(columns, (unsigned)((p.n + 16l * TN - 1) / (16 * TN))), dim3(64 * waves),
                     (size_t)waves * 16 * TN * kFewColumns * 4, stream, p);
}

template <int FORMAT, int OUT>
void start(const LinearParams& p, hipStream_t stream) {
  switch (linear_form(p.n, p.k, p.m)) {
    case kFew16: return start_few<FORMAT, OUT, 1>(p, stream);
    case kFew32: return start_few<FORMAT, OUT, 2>(p, stream);
    case kTiles64: return start_tiles<FORMAT, OUT, 1, 4, 1, 1, 3, 4>(p, stream);
    case kTiles64Chains: return start_tiles<FORMAT, OUT, 1, 4, 1, 1, 3, 4, 4>(p, stream);
    case kTiles128: return start_tiles<FORMAT, OUT, 1, 4, 2, 2, 2, 3>(p, stream);
    case kTiles256: break;
  }
  // 32 x 256 a wave where rows are split (twice the registers for a row tile), 64 x 128 otherwise (fewer
  // LDS reads): 8192 x 8192 x 8192 e4m3 629 / 709, in one pass 400 / 375.
  if constexpr (FORMAT == kFp8)
    start_tiles<FORMAT, OUT, 1, 4, 4, 2, 2, 2>(p, stream);
  else
    start_tiles<FORMAT, OUT, 2, 2, 2, 4, 2, 2>(p, stream);
}

// The formats of the rows and of the result pick the kernel.
template <int OUT>
hipError_t linear_to(const LinearParams& p, hipStream_t stream) {
  if (p.format == kFp4)
    start<kFp4, OUT>(p, stream);
  else
    start<kFp8, OUT>(p, stream);
  return hipGetLastError();
}

}  // namespace

// Measured with each form forced, to bf16, the weights from memory, us, e4m3 / e2m1 rows (n x k x m):
//                       16 rows      32 rows      64 x 64      in four chains
//   1 x 4096 x 14 336   10.2 /  9.3  13.8 /  9.8  16.2 / 13.5  12.8 /  9.3
//   16 x 4096 x 28 672  18.7 / 17.5  28.2 / 18.3  21.7 / 16.1  25.4 / 19.4
//   1 x 4096 x 128 256  55.7 / 55.0  91.7 / 57.2  72.4 / 51.6  93.8 / 65.6
//   24 x 4096 x 4096     6.8 /  5.8   8.5 /  7.4  15.7 / 12.7  11.5 /  8.5
//   128 x 2048 x 512     4.5 /  4.0   5.9 /  5.0   8.9 /  6.3   7.5 /  5.8
//   24 x 4096 x 7168     9.5 /  9.1   8.7 /  7.8  15.9 / 13.1  11.8 /  8.8
//   64 x 4096 x 4096    10.1 /  8.4   9.5 /  7.6  15.7 / 13.2  13.5 / 11.7
//   24 x 8192 x 8192    17.3 / 16.4  15.3 / 12.5  28.5 / 23.2  19.6 / 14.1
//   64 x 2048 x 4096     6.8 /  5.7   6.5 /  5.5   9.4 /  8.0   8.8 /  7.4
//   64 x 1024 x 4096     4.7 /  4.2   4.7 /  4.1   6.1 /  5.2   6.3 /  5.4
//   128 x 384 x 1536     3.1 /  2.8   3.4 /  3.0   3.9 /  3.4   4.7 /  4.2
//   48 x 4096 x 4128    10.1 /  8.8  13.1 / 10.2  15.7 / 12.9  12.6 / 10.0
//   24 x 8192 x 8224    20.8 / 18.8  26.2 / 18.4  28.6 / 23.3  19.6 / 14.1
//   24 x 4096 x 14 336  15.9 / 14.9  16.2 / 11.5  16.4 / 13.8  12.8 /  9.8
//   64 x 4096 x 7168    17.1 / 14.9  17.3 / 12.2  16.0 / 13.5  14.0 / 12.1
//                                                 64 x 64      in four chains  128 x 128
//   128 x 4096 x 4096                             15.9 / 13.1  13.4 / 11.2     33.1 / 27.0
//   512 x 2048 x 2048                              9.9 /  7.6   8.7 /  6.8     18.5 / 13.9
//   512 x 1024 x 1024                              6.0 /  4.6   5.9 /  5.0     11.0 /  7.6
//   128 x 4096 x 14 336                           21.9 / 18.3  25.6 / 21.5     33.4 / 27.6
//   512 x 4096 x 4096                             22.8 / 15.9  24.7 / 19.3     33.3 / 26.2
//   64 x 4096 x 28 672                            24.2 / 21.1  27.6 / 24.5     34.9 / 28.1
//   64 x 4096 x 128 256                           89.1 / 82.5   109 / 92.8     99.2 / 81.3
//   128 x 4096 x 28 672                           39.0 / 35.8  49.9 / 40.9     34.4 / 29.5
//   1024 x 4096 x 4096                            38.2 / 28.6                  34.2 / 25.9
//                                                              128 x 128       128 x 256
//   2048 x 4096 x 4096                                         48.4 / 37.4     52.3 / 30.8
//   4096 x 4096 x 4096                                         92.5 / 63.4     85.4 / 46.6
//   8192 x 8192 x 8192                                          664 / 396       616 / 300
//   96 120 x 384 x 1536                                         107 / 70.5      100 / 69.3
//   96 120 x 1536 x 384 (the second tile half empty)           79.7 / 46.2     96.0 / 51.3
LinearForm linear_form(long n, long k, long m) {
  const long cus = device_cus();
  const long columns = (m + 31) / 32, narrow = (m + 127) / 128, wide = (m + 255) / 256;
  const long high = (n + 127) / 128, blocks16 = (n + 15) / 16 * columns, blocks32 = (n + 31) / 32 * columns;
  // One tile of rows, whatever the width: the weight is read once. Also where the workgroups fit one to a CU.
  if (n <= 16 || blocks16 <= cus) return kFew16;
  // Twice the rows where that is what makes them fit and there is a chain of steps to save.
  if (blocks32 <= cus && k >= 2048) return kFew32;
  if (blocks16 <= 2 * cus) return kFew16;
  // A tile of 128 rows half empty at best, or fewer of them than three for four CUs.
  if (n <= 64 || narrow * high * 4 < 3 * cus)
    return (n + 63) / 64 * ((m + 63) / 64) <= cus && k >= 2048 ? kTiles64Chains : kTiles64;
  // 256 columns unless they leave a tile mostly empty or less than two tiles to a CU.
  return wide * 32 <= narrow * 17 && wide * high >= 2 * cus ? kTiles256 : kTiles128;
}

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
