// Device helpers of the attention kernels over a paged cache: codes to matrix operands, the mask, and the query tiles
// that a batch has.
#pragma once
#include "paged.hpp"

namespace ancha {
namespace paged {

using namespace mx;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

// Two codes (number `pair` of those in w) as bf16 / fp16 times 2^(s - 127), f having the exponent bits s.
template <int FORMAT>
__device__ __forceinline__ unsigned two_bf16(unsigned w, float f, int pair) {
  bf16x2 r;
  if constexpr (FORMAT == kFp8)
    r = pair ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, f, true)
             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, f, false);
  else
    r = pair == 0   ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0)
        : pair == 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1)
        : pair == 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2)
                    : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3);
  return __builtin_bit_cast(unsigned, r);
}
template <int FORMAT>
__device__ __forceinline__ unsigned two_f16(unsigned w, float f, int pair) {
  h16x2 r;
  if constexpr (FORMAT == kFp8)
    r = pair ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, f, true)
             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, f, false);
  else
    r = pair == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 0)
        : pair == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 1)
        : pair == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 2)
                    : __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 3);
  return __builtin_bit_cast(unsigned, r);
}

__device__ __forceinline__ float power(int e) { return __builtin_bit_cast(float, (unsigned)(e + 127) << 23); }

// A NaN that the compiler, which assumes there is none, cannot see.
__device__ __forceinline__ float hidden_nan() {
  unsigned bits = 0x7fc00000u;
  asm volatile("" : "+v"(bits));
  return __builtin_bit_cast(float, bits);
}

// The upper 8 bits of eight values as bf16, which are taken off them: three times leaves nothing of 24 bits. Cut off,
// not rounded, so that the largest number does not become an infinity, and the parts of one value have its sign, so
// that products beyond fp32 are infinities of one sign too.
__device__ __forceinline__ u32x4 upper_bits(float* v) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const unsigned a = __builtin_bit_cast(unsigned, v[2 * j]), b = __builtin_bit_cast(unsigned, v[2 * j + 1]);
    r[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    v[2 * j] -= __builtin_bit_cast(float, a & 0xffff0000u);
    v[2 * j + 1] -= __builtin_bit_cast(float, b & 0xffff0000u);
  }
  return r;
}

// The exponent of a weight, up + scale x - m for a row's maximum m, is one fused multiply-add: scale x + base. Its
// product is exact and the one that m was taken from is rounded, which up to 2^22 leaves at most 1/4 between them.
// Beyond, that would be up to half of the score's last place, 2^7 at 2^31, and the largest weight no number of fp16:
// there scores are first replaced by what their own rounded products leave of m, over scale, and base is `up`.
__device__ __forceinline__ bool is_far(float m) { return __builtin_fabsf(m) >= 4194304.f && m != -__builtin_inff(); }
__device__ __forceinline__ float base_of(float m, float up) {
  return m == -__builtin_inff() ? 0.f : is_far(m) ? up : up - m;
}
__device__ __forceinline__ float behind(const AttentionParams& p, float x, float m) {
#pragma clang fp contract(off)
  const float t = x * p.scale;
  return (t - m) * p.unscale;
}

// Zeros for a first product, in registers: as the instruction's constant they leave its result free to lie over its
// operands.
__device__ __forceinline__ f32x4 zeros() {
  f32x4 z = {0.f, 0.f, 0.f, 0.f};
  asm volatile("" : "+v"(z));
  return z;
}

// In place of a part's sum: the row has met keys there, all with scores of minus infinity. They weigh nothing beside
// others; where a row has no others its result is 0 / 0, a NaN, while a row that sees no key at all is 0.
constexpr float kLost = -1.f;
__device__ __forceinline__ bool is_zero(float x) {  // on the bits: a NaN is none
  unsigned bits = __builtin_bit_cast(unsigned, x);
  asm volatile("" : "+v"(bits));
  return (bits & 0x7fffffffu) == 0;
}

// Keys [low, high) that row r of a sequence sees, r = token * group + head.
struct Range {
  int low, high;
};
__device__ __forceinline__ Range visible(const AttentionParams& p, const Sequence& s, int token) {
  // Some steps below 2^31, so that a step ahead of the last one is still a number.
  const int capacity = (int)min((long)p.batch.columns << p.cache.shift, 0x7fff0000l);
  const long at = (long)s.at + token;
  const long high = p.causal ? at + 1 : s.length, low = p.window ? at - p.window + 1 : 0;
  const int h = (int)min(max(high, 0l), (long)capacity);
  return {(int)min(max(low, 0l), (long)h), h};
}

// Tile `id` of `rows` rows: its sequence and first row (of count * group), false behind the last one, when `id` is left
// with its number among those.
__device__ __forceinline__ bool find_tile(const AttentionParams& p, int group, int rows, int& id, int& i, Sequence& s,
                                          int& row) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < p.batch.sequences; base += 64) {
    Sequence mine = {0, 0, 0, 0};
    if (base + lane < p.batch.sequences) mine = sequence(p.batch, base + lane, p.rows);
    // At most 2^24 (a call has fewer): starts that do not ascend cannot make the sums overflow.
    const int tiles = (int)min(((long)mine.count * group + rows - 1) / rows, 1l << 24);
    int sum;  // of the tiles up to this lane's
    if (!__any(tiles > 1)) {
      const unsigned long long some = __ballot(tiles != 0);
      const unsigned low = __builtin_amdgcn_mbcnt_lo((unsigned)some, 0u);
      sum = tiles + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(some >> 32), low);
    } else {
      sum = tiles;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int below = __shfl_up(sum, o);
        if (lane >= o) sum += below;
      }
    }
    const int all = __builtin_amdgcn_readlane(sum, 63);
    if (id < all) {
      const unsigned long long past = __ballot(sum > id);
      const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
      i = base + at;
      s.first = __builtin_amdgcn_readlane(mine.first, at);
      s.count = __builtin_amdgcn_readlane(mine.count, at);
      s.length = __builtin_amdgcn_readlane(mine.length, at);
      s.at = __builtin_amdgcn_readlane(mine.at, at);
      row = (id - (__builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(tiles, at))) * rows;
      return true;
    }
    id -= all;
  }
  return false;
}

// Rows of the call that are of no sequence: zeros, by the workgroups behind the last tile (`which` of `count`).
template <typename T>
__device__ void clear_rows(const AttentionParams& p, int which, int count) {
  const int n = p.batch.sequences;
  const int from = n ? min(max(p.batch.starts[0], 0), p.rows) : 0;
  const int to = n ? min(max(p.batch.starts[n], from), p.rows) : 0;
  const long wide = (long)p.heads * p.cache.dim;
  T* out = static_cast<T*>(p.out);
  count = max(count, 1);
  for (long at = (long)which * blockDim.x + threadIdx.x; at < (p.rows - (to - from)) * wide;
       at += (long)count * blockDim.x)
    out[at < from * wide ? at : at + (to - from) * wide] = (T)0.f;
}

// Steps of `keys` keys that the rows of a tile see, and how many of the p.splits workgroups share them.
constexpr int kLeastKeys = 256;  // that a workgroup of a split has at least
struct Walk {
  int first, high, low;  // keys [first, high); the steps begin at low, a multiple of `keys`
  int steps, each, splits;
};
__device__ __forceinline__ Walk walk_of(const AttentionParams& p, const Sequence& s, int group, int row, int rows,
                                        int keys) {
  const int last = min(row + rows, s.count * group) - 1;
  const Range a = visible(p, s, row / group), b = visible(p, s, last / group);
  Walk w;
  w.first = a.low;
  w.low = a.low & ~(keys - 1);
  w.high = b.high;
  w.steps = w.high > w.low ? (w.high - w.low - 1) / keys + 1 : 0;
  w.each = max((w.steps + p.splits - 1) / p.splits, kLeastKeys / keys);
  w.splits = max((w.steps + w.each - 1) / w.each, 1);
  return w;
}

// Workspace of a split: per (tile, head of the cache) what the parts are of, then per (tile, head, split) the rows'
// maxima and sums and their results.
struct Joined {
  int splits, first, row, rows;  // parts; the sequence's first row of the call; the tile's first and its number of rows
};
__host__ __device__ constexpr long part_floats(int rows, int dim) { return (long)rows * (dim + 2); }
__host__ __device__ constexpr long joined_floats(long tiles, int heads) { return tiles * heads * 4; }
__device__ __forceinline__ float* part_of(const AttentionParams& p, int tile, int head, int split, int rows, int dim) {
  const long at = ((long)tile * p.cache.heads + head) * p.splits + split;
  return p.parts + joined_floats(p.tiles, p.cache.heads) + at * part_floats(rows, dim);
}
// By the first workgroup of every (tile, head), also where there is no tile (rows 0).
__device__ __forceinline__ void note_tile(const AttentionParams& p, int tile, int head, int split, Joined j) {
  if (p.splits > 1 && split == 0 && threadIdx.x == 0)
    reinterpret_cast<Joined*>(p.parts)[(long)tile * p.cache.heads + head] = j;
}

}  // namespace paged
}  // namespace ancha
