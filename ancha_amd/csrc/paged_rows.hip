// Rows of the paged operators (gfx950): rotary positions, keys and values into the pages of a cache, and back.
// Contracts: include/ancha_hip.h; the cache's layout: paged.hpp.
#include "paged.hpp"

namespace ancha {
namespace paged {
namespace {

using namespace mx;

constexpr int kThreads = 256;
constexpr int kTrig = 1024;  // angles of a workgroup's rows

// cos and sin of angle a to fp32: the multiple of a right angle is taken off in 64 bits, so far positions lose nothing.
__device__ __forceinline__ float2 cos_sin(double a) {
  const double quarters = a * 0.6366197723675813430755;
  const double whole = __builtin_rint(quarters);
  float s, c;
  sincospif(0.5f * (float)(quarters - whole), &s, &c);
  const int turn = (int)(whole - 4.0 * __builtin_floor(0.25 * whole));
  const float x = turn & 1 ? s : c, y = turn & 1 ? c : s;
  return make_float2(turn == 1 || turn == 2 ? -x : x, turn & 2 ? -y : y);
}

// Rows of heads at their positions. A workgroup has `rows` rows: their cosines and sines once, into LDS, then all of
// the heads' pairs, as many a thread as 16 bytes hold (HALF: from two places of the head, otherwise neighbours);
// columns behind the rotated ones are copied as they are. Bound by memory.
template <int TYPE, bool HALF>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryParams p, int rows, Divide by_row, Divide by_head) {
  constexpr int V = 16 / (int)sizeof(typename Stored<TYPE>::type);
  __shared__ float2 trig[kTrig];
  __shared__ int of_none[kThreads];
  const int pairs = p.plan.width / 2;
  const long first = (long)blockIdx.x * rows;
  const int mine = (int)min((long)rows, p.rows - first);
  for (int i = threadIdx.x; i < mine * pairs; i += kThreads) {
    const int r = i / pairs, j = i - r * pairs;
    long at;
    bool there = true;
    if (p.positions) {
      at = p.wide ? static_cast<const long*>(p.positions)[first + r] : static_cast<const int*>(p.positions)[first + r];
    } else {
      int s, position = 0;
      there = place(p.batch, (int)first + r, s, position);
      at = position;
    }
    const float2 t = cos_sin((double)at * p.plan.freqs[j]);
    const float m = (float)p.plan.magnitude;
    trig[i] = make_float2(m * t.x, m * t.y);
    if (j == 0) of_none[r] = !there;
  }
  __syncthreads();
  const int turned = (pairs + V - 1) / V, rest = p.dim - p.plan.width;
  const int units = turned + (rest + 2 * V - 1) / (2 * V);  // of a head
  const int total = mine * p.heads * units;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int r = (int)divided(i, by_row), in_row = i - r * p.heads * units;
    const int head = (int)divided(in_row, by_head), u = in_row - head * units;
    const long from = (first + r) * p.ld + head * p.ldh, to = ((first + r) * p.heads + head) * p.dim;
    float a[V], b[V];
    int col_a, col_b, valid_a, valid_b;
    if (u >= turned) {
      const int at = (u - turned) * 2 * V;
      col_a = p.plan.width + at, valid_a = rest - at;
      col_b = col_a + V, valid_b = valid_a - V;
    } else if (HALF) {
      col_a = u * V, col_b = pairs + col_a;
      valid_a = valid_b = pairs - col_a;
    } else {
      col_a = 2 * V * u, col_b = col_a + V;
      valid_a = p.plan.width - col_a, valid_b = valid_a - V;
    }
    if (valid_b <= 0) col_b = col_a;  // nothing is read or written there
    load_row<TYPE, V>(p.x, from + col_a, valid_a, a);
    load_row<TYPE, V>(p.x, from + col_b, valid_b, b);
    if (u < turned) {
      const float2* t = trig + r * pairs + u * V;
#pragma unroll
      for (int j = 0; j < V; j++) {
        if (u * V + j >= pairs) break;
        const float2 cs = t[j];
        float& x = HALF ? a[j] : j < V / 2 ? a[2 * j] : b[2 * j - V];
        float& y = HALF ? b[j] : j < V / 2 ? a[2 * j + 1] : b[2 * j + 1 - V];
        const float x0 = x;
        x = __builtin_fmaf(x0, cs.x, -(y * cs.y));
        y = __builtin_fmaf(y, cs.x, x0 * cs.y);
      }
    }
    if (of_none[r])
#pragma unroll
      for (int j = 0; j < V; j++) a[j] = b[j] = 0.f;
    store_row<TYPE, V>(p.out, to + col_a, valid_a, a);
    store_row<TYPE, V>(p.out, to + col_b, valid_b, b);
  }
}

// Eight columns from col on of a key, rotated in 64 bits: the rounding to the codes is the only one. x: the columns
// themselves, `row` the key's first value, trig those of the row's pairs.
template <int TYPE>
__device__ __forceinline__ void turn_key(const Plan& plan, const typename Stored<TYPE>::type* row, int col,
                                         const double2* trig, float* x) {
  const int pairs = plan.width / 2;
  if (plan.interleaved) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if (col + j >= plan.width) break;
      const double2 t = trig[(col + j) / 2];
      const double a = x[j], b = x[j + 1];
      x[j] = to_odd(a * t.x - b * t.y);
      x[j + 1] = to_odd(b * t.x + a * t.y);
    }
    return;
  }
  // The other value of each pair: eight neighbours, unless the eight cross from one half to the other.
  float other[8];
  const bool low = col < pairs;
  if (pairs % 8 == 0) {
    load_row<TYPE, 8>(row, low ? col + pairs : col - pairs, 8, other);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int d = col + j;
      other[j] = d < plan.width ? (float)row[d < pairs ? d + pairs : d - pairs] : 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int d = col + j;
    if (d >= plan.width) break;
    const double2 t = trig[d < pairs ? d : d - pairs];
    const double a = x[j], b = other[j];
    x[j] = d < pairs ? to_odd(a * t.x - b * t.y) : to_odd(a * t.x + b * t.y);
  }
}

// New keys and values into their pages. A workgroup has `rows` rows: their places and their pairs' cosines and sines
// once (in 64 bits), then eight columns a thread, four threads a block of codes. Rows without a place are left out.
template <int TYPE, int FORMAT>
__global__ __launch_bounds__(kThreads) void write_kernel(WriteParams p, int rows, Divide by_row) {
  __shared__ double2 trig[kTrig];
  __shared__ int2 places[kThreads];  // page (or -1) and slot
  const int pairs = p.plan.freqs ? p.plan.width / 2 : 0;
  const long first = (long)blockIdx.x * rows;
  const int mine = (int)min((long)rows, p.rows - first);
  for (int r = threadIdx.x; r < mine; r += kThreads) {
    int s = 0, position = 0, page = -1;
    if (place(p.batch, (int)first + r, s, position) && position >= 0) page = page_of(p.batch, p.cache, s, position);
    places[r] = make_int2(page, position & ((1 << p.cache.shift) - 1));
  }
  for (int i = threadIdx.x; i < mine * pairs; i += kThreads) {
    const int r = i / pairs;
    int s = 0, position = 0;
    place(p.batch, (int)first + r, s, position);
    double sine, cosine;
    sincos((double)position * p.plan.freqs[i - r * pairs], &sine, &cosine);
    trig[i] = make_double2(p.plan.magnitude * cosine, p.plan.magnitude * sine);
  }
  __syncthreads();
  saturate();
  const int dim = p.cache.dim, heads = p.cache.heads;
  const int units = dim / 8;  // of a head; a multiple of 4, so a block's threads stay together
  const int total = mine * 2 * heads * units;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int r = (int)divided(i, by_row), in_row = i - r * 2 * heads * units;
    const int both = in_row / units, col = 8 * (in_row - both * units);
    const int which = both >= heads, head = both - which * heads;
    const int2 to = places[r];
    if (to.x < 0) continue;
    typedef typename Stored<TYPE>::type T;
    const T* row = which ? static_cast<const T*>(p.v) + (first + r) * p.ldv + head * p.ldvh
                         : static_cast<const T*>(p.k) + (first + r) * p.ldk + head * p.ldkh;
    float x[8];
    load_row<TYPE, 8>(row, col, 8, x);
    if (!which && col < 2 * pairs) turn_key<TYPE>(p.plan, row, col, trig + r * pairs, x);
    const long slot = slot_of(p.cache, which, to.x, head, to.y);
    store_codes(x, FORMAT, true, p.cache.codes + slot * row_bytes(dim, FORMAT) + (FORMAT == kFp8 ? col : col / 2),
                p.cache.scales + slot * (dim / kBlock) + col / kBlock);
  }
}

// Sequences as values, 16 bytes of the result a thread; zeros where there is no token.
template <int TYPE, int FORMAT>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadParams p, int tokens, Divide by_token) {
  constexpr int N = 16 / (int)sizeof(typename Stored<TYPE>::type);
  __shared__ int2 places[kThreads];
  const int blocks = (p.size + tokens - 1) / tokens;
  const int s = blockIdx.x / blocks, first = (int)(blockIdx.x - (unsigned)s * blocks) * tokens;
  const int mine = min(tokens, p.size - first);
  for (int t = threadIdx.x; t < mine; t += kThreads) {
    const int at = first + t;
    const int page = at < p.batch.lengths[s] ? page_of(p.batch, p.cache, s, at) : -1;
    places[t] = make_int2(page, at & ((1 << p.cache.shift) - 1));
  }
  __syncthreads();
  const int dim = p.cache.dim, heads = p.cache.heads, units = dim / N;
  const int total = mine * 2 * heads * units;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int t = (int)divided(i, by_token), in_token = i - t * 2 * heads * units;
    const int both = in_token / units, col = N * (in_token - both * units);
    const int which = both >= heads, head = both - which * heads;
    const int2 from = places[t];
    float v[N];
    if (from.x >= 0) {
      const long slot = slot_of(p.cache, which, from.x, head, from.y);
      const float f = scale_value(p.cache.scales[slot * (dim / kBlock) + col / kBlock]);
      const uint8_t* codes = p.cache.codes + slot * row_bytes(dim, FORMAT) + (FORMAT == kFp8 ? col : col / 2);
      if constexpr (FORMAT == kFp8) {
        unsigned c[N / 4];
        __builtin_memcpy(c, codes, N);
#pragma unroll
        for (int j = 0; j < N / 4; j++) {
          const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(c[j], false);
          const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(c[j], true);
          v[4 * j] = a[0], v[4 * j + 1] = a[1], v[4 * j + 2] = b[0], v[4 * j + 3] = b[1];
        }
      } else {
        unsigned c = 0;
        __builtin_memcpy(&c, codes, N / 2);
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
      for (int j = 0; j < N; j++) v[j] *= f;
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) v[j] = 0.f;
    }
    store_row<TYPE, N>(which ? p.v : p.k, (((long)s * p.size + first + t) * heads + head) * dim + col, N, v);
  }
}

template <int TYPE>
void start_rotary(const RotaryParams& p, hipStream_t stream) {
  constexpr int V = 16 / (int)sizeof(typename Stored<TYPE>::type);
  const int pairs = p.plan.width / 2;
  // As many rows as fill the workgroup with angles, but two workgroups a CU first.
  const int rows = max(1, min(min(kThreads / pairs, 32), p.rows / 512));
  const int units = (pairs + V - 1) / V + (p.dim - p.plan.width + 2 * V - 1) / (2 * V);
  const dim3 grid((unsigned)((p.rows + (long)rows - 1) / rows));
  const Divide by_row = divide_by((long)p.heads * units), by_head = divide_by(units);
  if (p.plan.interleaved)
    hipLaunchKernelGGL((rotary_kernel<TYPE, false>), grid, dim3(kThreads), 0, stream, p, rows, by_row, by_head);
  else
    hipLaunchKernelGGL((rotary_kernel<TYPE, true>), grid, dim3(kThreads), 0, stream, p, rows, by_row, by_head);
}

template <int TYPE>
void start_write(const WriteParams& p, hipStream_t stream) {
  const int units = 2 * p.cache.heads * p.cache.dim / 8;
  const int rows = max(1, min(min(4, 4096 / units), p.rows / 512));
  const dim3 grid((unsigned)((p.rows + (long)rows - 1) / rows));
  if (p.cache.format == kFp8)
    hipLaunchKernelGGL((write_kernel<TYPE, kFp8>), grid, dim3(kThreads), 0, stream, p, rows, divide_by(units));
  else
    hipLaunchKernelGGL((write_kernel<TYPE, kFp4>), grid, dim3(kThreads), 0, stream, p, rows, divide_by(units));
}

template <int TYPE>
void start_read(const ReadParams& p, hipStream_t stream) {
  constexpr int N = 16 / (int)sizeof(typename Stored<TYPE>::type);
  const int units = 2 * p.cache.heads * p.cache.dim / N;
  const int tokens = max(1, min(2048 / units, 64));
  const dim3 grid((unsigned)(((p.size + (long)tokens - 1) / tokens) * p.batch.sequences));
  if (p.cache.format == kFp8)
    hipLaunchKernelGGL((read_kernel<TYPE, kFp8>), grid, dim3(kThreads), 0, stream, p, tokens, divide_by(units));
  else
    hipLaunchKernelGGL((read_kernel<TYPE, kFp4>), grid, dim3(kThreads), 0, stream, p, tokens, divide_by(units));
}

}  // namespace

hipError_t launch_rotary(const RotaryParams& p, hipStream_t stream) {
  if (p.type == kF32)
    start_rotary<kF32>(p, stream);
  else if (p.type == kF16)
    start_rotary<kF16>(p, stream);
  else
    start_rotary<kBf16>(p, stream);
  return hipGetLastError();
}

hipError_t launch_write(const WriteParams& p, hipStream_t stream) {
  if (p.type == kF32)
    start_write<kF32>(p, stream);
  else if (p.type == kF16)
    start_write<kF16>(p, stream);
  else
    start_write<kBf16>(p, stream);
  return hipGetLastError();
}

hipError_t launch_read(const ReadParams& p, hipStream_t stream) {
  if (p.type == kF32)
    start_read<kF32>(p, stream);
  else if (p.type == kF16)
    start_read<kF16>(p, stream);
  else
    start_read<kBf16>(p, stream);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace ancha
