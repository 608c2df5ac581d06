// Rows of the paged operators (gfx950): rotary positions, keys and values into the pages of a cache, and back.
// Contracts: include/ancha_hip.h; the cache's layout: paged.hpp.
#include "paged.hpp"

namespace ancha {
namespace paged {
namespace {

using namespace mx;

constexpr int kThreads = 256;
constexpr int kTrig = 1024;     // angles of a workgroup's rows
constexpr int kMostRows = 64;   // of a workgroup

// cos and sin of angle a to fp32: the multiple of a right angle is taken off in 64 bits, which is off by less than
// 2^-27 below 2^26 and by as much as the angle itself is rounded beyond.
__device__ __forceinline__ float2 cos_sin(double a) {
  const double quarters = a * 0.6366197723675813430755;
  const double whole = __builtin_rint(quarters);
  float s, c;
  sincospif(0.5f * (float)(quarters - whole), &s, &c);
  const int turn = (int)(whole - 4.0 * __builtin_floor(0.25 * whole));
  const float x = turn & 1 ? s : c, y = turn & 1 ? c : s;
  return make_float2(turn == 1 || turn == 2 ? -x : x, turn & 2 ? -y : y);
}

// The same for keys that are written: half pi is taken off in two parts by fused multiply-adds, the rest, about pi /
// 4 at most, goes through the Taylor series to its 15th and 16th power. Within 2^-52 for angles below 2^48. Beyond, a
// * 2 / pi is itself rounded by up to an eighth of a quarter turn and more, so the rest leaves the series' range:
// within 2^-49 below 2^50 and 2^-45 below 2^51, which positions and frequencies up to 2^20 do not pass; a code has 4
// bits. (Largest of 200 000 angles of each octave against 113-bit ones, in the same steps on the CPU: 0.87, 1.5, 5.5
// and 85 times 2^-52 up to 2^48, 2^49, 2^50 and 2^51.) With the library's function, which reduces any angle, 16 384
// keys of 8 x 128 are written in 35 us instead of 30.
__device__ __forceinline__ double2 cos_sin_64(double a) {
  const double whole = __builtin_rint(a * 0.6366197723675813430755);
  double r = __builtin_fma(-whole, 1.5707963267948965579990, a);
  r = __builtin_fma(-whole, 6.1232339957367660358688e-17, r);
  const double z = r * r;
  double s = -1.0 / 1307674368000, c = 1.0 / 20922789888000;
  s = __builtin_fma(s, z, 1.0 / 6227020800);
  s = __builtin_fma(s, z, -1.0 / 39916800);
  s = __builtin_fma(s, z, 1.0 / 362880);
  s = __builtin_fma(s, z, -1.0 / 5040);
  s = __builtin_fma(s, z, 1.0 / 120);
  s = __builtin_fma(s, z, -1.0 / 6);
  s = __builtin_fma(s * z, r, r);
  c = __builtin_fma(c, z, -1.0 / 87178291200);
  c = __builtin_fma(c, z, 1.0 / 479001600);
  c = __builtin_fma(c, z, -1.0 / 3628800);
  c = __builtin_fma(c, z, 1.0 / 40320);
  c = __builtin_fma(c, z, -1.0 / 720);
  c = __builtin_fma(c, z, 1.0 / 24);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int turn = (int)(whole - 4.0 * __builtin_floor(0.25 * whole));
  const double x = turn & 1 ? s : c, y = turn & 1 ? c : s;
  return make_double2(turn == 1 || turn == 2 ? -x : x, turn & 2 ? -y : y);
}

// Threads for the rotated columns of a head, V values at a time.
template <bool HALF>
__host__ __device__ constexpr int turned_units(int pairs, int V) {
  return ((HALF ? pairs : 2 * pairs) + V - 1) / V;
}

// Rows of heads at their positions. A workgroup has `rows` rows: their cosines and sines once, into LDS, then all of
// the heads' columns, 16 bytes a thread (HALF: of both halves), so that an instruction of a wave writes one piece of
// memory; columns behind the rotated ones are copied as they are. The first values are on their way while the angles
// are taken. Bound by memory: 16 384 rows of 40 heads of 128 in bf16, 336 MB, take 65 us, 5.1 TB/s, as fast as a copy;
// 6007 of 5 of 96 in fp32 (48 interleaved) 7.7 us, of which 4.5 are the memory's, and 10.0 with both values of a pair
// read by themselves; one row 3.5 us.
template <int TYPE, bool HALF>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryParams p, int rows, Divide by_row, Divide by_head) {
  constexpr int V = 16 / (int)sizeof(typename Stored<TYPE>::type);
  __shared__ float2 trig[kTrig];
  __shared__ long at_row[kMostRows];
  __shared__ bool of_none[kMostRows];
  const int pairs = p.plan.width / 2;
  const long first = (long)blockIdx.x * rows;
  const int mine = (int)min((long)rows, p.rows - first);
  const int turned = turned_units<HALF>(pairs, V), units = turned + (p.dim - p.plan.width + V - 1) / V;  // of a head
  const int total = mine * p.heads * units;
  struct Unit {
    int row, u, col_a, col_b, valid_a, valid_b;
    long from, to;
    float a[V], b[V];
  };
  const auto load = [&](int i, Unit& x) {
    x.row = (int)divided(i, by_row);
    const int in_row = i - x.row * p.heads * units;
    const int head = (int)divided(in_row, by_head);
    x.u = in_row - head * units;
    x.from = (first + x.row) * p.ld + head * p.ldh, x.to = ((first + x.row) * p.heads + head) * p.dim;
    const bool copied = x.u >= turned;
    x.col_a = copied ? p.plan.width + (x.u - turned) * V : x.u * V;
    x.valid_a = (copied ? p.dim : HALF ? pairs : p.plan.width) - x.col_a;
    x.col_b = HALF && !copied ? pairs + x.col_a : x.col_a;
    x.valid_b = HALF && !copied ? x.valid_a : 0;  // 0: nothing is read or written there
    load_row<TYPE, V>(p.x, x.from + x.col_a, x.valid_a, x.a);
    load_row<TYPE, V>(p.x, x.from + x.col_b, x.valid_b, x.b);
  };
  Unit x;
  if ((int)threadIdx.x < total) load(threadIdx.x, x);
  if (p.positions) {
    if ((int)threadIdx.x < mine) {
      const long r = first + threadIdx.x;
      at_row[threadIdx.x] = p.wide ? static_cast<const long*>(p.positions)[r] : static_cast<const int*>(p.positions)[r];
      of_none[threadIdx.x] = false;
    }
  } else {
    for (int r = threadIdx.x / 64; r < mine; r += kThreads / 64) {
      int s, position = 0;
      const bool there = place(p.batch, (int)first + r, s, position);
      at_row[r] = position;
      of_none[r] = !there;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < mine * pairs; i += kThreads) {
    const int r = i / pairs;
    const float2 t = cos_sin((double)at_row[r] * p.plan.freqs[i - r * pairs]);
    const float m = (float)p.plan.magnitude;
    trig[i] = make_float2(m * t.x, m * t.y);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < total;) {
    if (x.u < turned) {
      constexpr int kPairs = HALF ? V : V / 2;
      const float2* t = trig + x.row * pairs + x.u * kPairs;
#pragma unroll
      for (int j = 0; j < kPairs; j++) {
        if (x.u * kPairs + j >= pairs) break;
        const float2 cs = t[j];
        float& y0 = HALF ? x.a[j] : x.a[2 * j];
        float& y1 = HALF ? x.b[j] : x.a[2 * j + 1];
        const float y = y0;
        y0 = __builtin_fmaf(y, cs.x, -(y1 * cs.y));
        y1 = __builtin_fmaf(y1, cs.x, y * cs.y);
      }
    }
    if (of_none[x.row])
#pragma unroll
      for (int j = 0; j < V; j++) x.a[j] = x.b[j] = 0.f;
    store_row<TYPE, V>(p.out, x.to + x.col_a, x.valid_a, x.a);
    store_row<TYPE, V>(p.out, x.to + x.col_b, x.valid_b, x.b);
    i += kThreads;
    if (i < total) load(i, x);
  }
}

// Place of a pair's cosine and sine in LDS: one free behind every eight, so that lanes eight pairs apart meet different
// banks.
__host__ __device__ constexpr int trig_at(int pair) { return pair + pair / 8; }

// Eight columns from col on of a key, rotated in 64 bits: the rounding to the codes is the only one. x: the columns
// themselves, other: for HALF the other values of their pairs; trig the pairs of the key's row. Where the eight are all
// rotated, and for HALF of one half, which is so for most widths, no column is looked at by itself.
template <bool HALF>
__device__ __forceinline__ void turn_key(const Plan& plan, int col, const double2* trig, const float* other, float* x) {
  const int pairs = plan.width / 2;
  if (HALF && pairs % 8 == 0) {
    const bool second = col >= pairs;
    const double2* t = trig + trig_at(second ? col - pairs : col);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double s = second ? t[j].y : -t[j].y;
      x[j] = to_odd(__builtin_fma((double)x[j], t[j].x, (double)other[j] * s));
    }
  } else if (!HALF && pairs % 4 == 0) {
    const double2* t = trig + trig_at(col / 2);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const double a = x[2 * j], b = x[2 * j + 1];
      x[2 * j] = to_odd(__builtin_fma(a, t[j].x, -(b * t[j].y)));
      x[2 * j + 1] = to_odd(__builtin_fma(b, t[j].x, a * t[j].y));
    }
  } else if (HALF) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int d = col + j;
      if (d >= plan.width) break;
      const double2 t = trig[trig_at(d < pairs ? d : d - pairs)];
      const double a = x[j], b = other[j];
      x[j] = d < pairs ? to_odd(a * t.x - b * t.y) : to_odd(a * t.x + b * t.y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if (col + j >= plan.width) break;
      const double2 t = trig[trig_at((col + j) / 2)];
      const double a = x[j], b = x[j + 1];
      x[j] = to_odd(a * t.x - b * t.y);
      x[j + 1] = to_odd(b * t.x + a * t.y);
    }
  }
}

// New keys and values into their pages. A workgroup has `rows` rows: their places and their pairs' cosines and sines
// once (in 64 bits), then eight columns a thread, four threads a block of codes. Rows without a place are left out.
// The first values are on their way while the places are found and the angles taken. 16 384 tokens of 8 heads of 128
// in bf16, 101 MB, take 30 us, of which 20 are the memory's; the vector instructions bound it, 84 % busy. About one
// in seven of them is of the 64 bits of the sines and the turn; the rest are loads' conversions, blocks' largest
// values, codes and addresses. (With a decision for every column and sines side by side in LDS it was 35 us, 90 %
// busy.) One, two or eight rows a workgroup, rows dealt by XCD, or the next values fetched ahead changed nothing. 32
// tokens take 5 us.
template <int TYPE, int FORMAT, bool HALF>
__global__ __launch_bounds__(kThreads) void write_kernel(WriteParams p, int rows, Divide by_row, Divide by_pair) {
  typedef typename Stored<TYPE>::type T;
  __shared__ double2 trig[trig_at(kTrig / 2)];
  __shared__ int2 places[kMostRows];  // page (or -1) and position
  const int pairs = p.plan.freqs ? p.plan.width / 2 : 0;
  const long first = (long)blockIdx.x * rows;
  const int mine = (int)min((long)rows, p.rows - first);
  const int dim = p.cache.dim, heads = p.cache.heads;
  const int units = dim / 8;  // of a head; 8, 16 or 32, so a block's threads stay together
  const int shift = __builtin_ctz(units);
  const int total = mine * 2 * heads * units;
  struct Unit {
    int row, which, head, col;
    float x[8], other[8];
  };
  const auto eight = [](const T* from, float* x) {
    T t[8];
    __builtin_memcpy(t, from, sizeof(t));
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = (float)t[j];
  };
  const auto load = [&](int i, Unit& u) {
    u.row = (int)divided(i, by_row);
    const int in_row = i - u.row * 2 * heads * units, both = in_row >> shift;
    u.col = 8 * (in_row & (units - 1));
    u.which = both >= heads, u.head = both - u.which * heads;
    const T* row = u.which ? static_cast<const T*>(p.v) + (first + u.row) * p.ldv + u.head * p.ldvh
                           : static_cast<const T*>(p.k) + (first + u.row) * p.ldk + u.head * p.ldkh;
    eight(row + u.col, u.x);
    if (!HALF || u.which || u.col >= 2 * pairs) return;
    // Eight neighbours, unless the eight cross from one half to the other.
    if (pairs % 8 == 0) {
      eight(row + (u.col < pairs ? u.col + pairs : u.col - pairs), u.other);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int d = u.col + j;
        u.other[j] = d < 2 * pairs ? (float)row[d < pairs ? d + pairs : d - pairs] : 0.f;
      }
    }
  };
  Unit u;
  if ((int)threadIdx.x < total) load(threadIdx.x, u);
  for (int r = threadIdx.x / 64; r < mine; r += kThreads / 64) {
    int s = 0, position = 0, page = -1;
    if (place(p.batch, (int)first + r, s, position) && position >= 0) page = page_of(p.batch, p.cache, s, position);
    places[r] = make_int2(page, position);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < mine * pairs; i += kThreads) {
    const int r = (int)divided(i, by_pair), pair = i - r * pairs;
    const double2 t = cos_sin_64((double)places[r].y * p.plan.freqs[pair]);
    trig[r * trig_at(pairs) + trig_at(pair)] = make_double2(p.plan.magnitude * t.x, p.plan.magnitude * t.y);
  }
  __syncthreads();
  saturate();
  for (int i = threadIdx.x; i < total;) {
    const int2 to = places[u.row];
    if (to.x >= 0) {
      if (!u.which && u.col < 2 * pairs) turn_key<HALF>(p.plan, u.col, trig + u.row * trig_at(pairs), u.other, u.x);
      const long slot = slot_of(p.cache, u.which, to.x, u.head, to.y & ((1 << p.cache.shift) - 1));
      uint8_t* const codes = p.cache.codes + slot * row_bytes(dim, FORMAT);
      store_codes(u.x, FORMAT, true, codes + (FORMAT == kFp8 ? u.col : u.col / 2),
                  p.cache.scales + slot * (dim / kBlock) + u.col / kBlock);
    }
    i += kThreads;
    if (i < total) load(i, u);
  }
}

// Sequences as values, 16 bytes of the result a thread; zeros where there is no token. Bound by memory once there are
// enough tokens: 16 384 of 8 heads of 128 in bf16, 102 MB, take 24 us, 4.2 TB/s. A short read is latency, so the
// workgroups are as small as it takes to have 2048: 6.2 us, not 9.7, for 10 843 of 3 heads of 64.
template <int TYPE, int FORMAT>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadParams p, int tokens, Divide by_token) {
  constexpr int N = 16 / (int)sizeof(typename Stored<TYPE>::type);
  __shared__ int2 places[kMostRows];
  const int blocks = (p.size + tokens - 1) / tokens;
  const int s = blockIdx.x / blocks, first = (int)(blockIdx.x - (unsigned)s * blocks) * tokens;
  const int mine = min(tokens, p.size - first);
  for (int t = threadIdx.x; t < mine; t += kThreads) {
    const int at = first + t;
    const int page = at < p.batch.lengths[s] ? page_of(p.batch, p.cache, s, at) : -1;
    places[t] = make_int2(page, at & ((1 << p.cache.shift) - 1));
  }
  __syncthreads();
  const int dim = p.cache.dim, heads = p.cache.heads, units = dim / N, shift = __builtin_ctz(units);
  const int total = mine * 2 * heads * units;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int t = (int)divided(i, by_token), in_token = i - t * 2 * heads * units;
    const int both = in_token >> shift, col = N * (in_token & (units - 1));
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
  const int turned = p.plan.interleaved ? turned_units<false>(pairs, V) : turned_units<true>(pairs, V);
  const int units = turned + (p.dim - p.plan.width + V - 1) / V;
  const dim3 grid((unsigned)((p.rows + (long)rows - 1) / rows));
  const Divide by_row = divide_by((long)p.heads * units), by_head = divide_by(units);
  if (p.plan.interleaved)
    hipLaunchKernelGGL((rotary_kernel<TYPE, false>), grid, dim3(kThreads), 0, stream, p, rows, by_row, by_head);
  else
    hipLaunchKernelGGL((rotary_kernel<TYPE, true>), grid, dim3(kThreads), 0, stream, p, rows, by_row, by_head);
}

template <int TYPE, int FORMAT>
void start_write(const WriteParams& p, hipStream_t stream) {
  const int units = 2 * p.cache.heads * p.cache.dim / 8;
  const int rows = max(1, min(min(4, 4096 / units), p.rows / 512));
  const dim3 grid((unsigned)((p.rows + (long)rows - 1) / rows));
  const Divide by_row = divide_by(units), by_pair = divide_by(max(p.plan.freqs ? p.plan.width / 2 : 1, 1));
  if (p.plan.interleaved)
    hipLaunchKernelGGL((write_kernel<TYPE, FORMAT, false>), grid, dim3(kThreads), 0, stream, p, rows, by_row, by_pair);
  else
    hipLaunchKernelGGL((write_kernel<TYPE, FORMAT, true>), grid, dim3(kThreads), 0, stream, p, rows, by_row, by_pair);
}

template <int TYPE, int FORMAT>
void start_read(const ReadParams& p, hipStream_t stream) {
  constexpr int N = 16 / (int)sizeof(typename Stored<TYPE>::type);
  const int units = 2 * p.cache.heads * p.cache.dim / N;
  // Up to eight units a thread, but eight workgroups a CU first.
  const long all = (long)p.size * p.batch.sequences;
  const int tokens = (int)max(1l, min(min(2048 / units, kMostRows) + 0l, all / 2048));
  const dim3 grid((unsigned)(((p.size + (long)tokens - 1) / tokens) * p.batch.sequences));
  hipLaunchKernelGGL((read_kernel<TYPE, FORMAT>), grid, dim3(kThreads), 0, stream, p, tokens, divide_by(units));
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
  const bool fp8 = p.cache.format == kFp8;
  if (p.type == kF32)
    fp8 ? start_write<kF32, kFp8>(p, stream) : start_write<kF32, kFp4>(p, stream);
  else if (p.type == kF16)
    fp8 ? start_write<kF16, kFp8>(p, stream) : start_write<kF16, kFp4>(p, stream);
  else
    fp8 ? start_write<kBf16, kFp8>(p, stream) : start_write<kBf16, kFp4>(p, stream);
  return hipGetLastError();
}

hipError_t launch_read(const ReadParams& p, hipStream_t stream) {
  const bool fp8 = p.cache.format == kFp8;
  if (p.type == kF32)
    fp8 ? start_read<kF32, kFp8>(p, stream) : start_read<kF32, kFp4>(p, stream);
  else if (p.type == kF16)
    fp8 ? start_read<kF16, kFp8>(p, stream) : start_read<kF16, kFp4>(p, stream);
  else
    fp8 ? start_read<kBf16, kFp8>(p, stream) : start_read<kBf16, kFp4>(p, stream);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace ancha
