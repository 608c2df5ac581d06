// Attention of new tokens over a paged, microscaled cache (gfx950). Contract: include/ancha_hip.h; layout: paged.hpp.
//
// For a query row r (a token and a head; the heads that share a head of the cache are rows beside each other) and the
// keys j that it sees:  o = sum_j e^(c q.k_j) v_j / sum_j e^(c q.k_j), in one pass with a running maximum.
//
// Operands. A key's codes times their power of two are bf16 values without loss (of scale bytes below 3 to within
// 2^-134), so products with a bf16 query are exact; a query of 16 or 32 bits that bf16 does not hold is the sum of
// two or three bf16 parts, a product each. The weights e^.. are the sum of two fp16 parts, 22 bits, for results of
// every type and in both kernels: with one part the distance of fp16 results from the exact ones was 1.4 times that
// of their own rounding (2.9e-4 instead of 2.1e-4 of their size), and of bf16 ones 1.006 times. The second part costs
// 1 to 5 % where the cache bounds a call and 30 to 35 % where the products do (see chunk_kernel). So values have to
// be fp16 too: each block of 32 columns has a reference power `ref` that all of its values are taken relative to, so
// that the largest fits; what lies 2^-32 below it, where fp16 ends, is far below the result's own rounding. When a
// larger one comes, the sums so far are scaled down, like those of the running maximum.
#include "paged_attention.hpp"

namespace ancha {
namespace paged {
namespace {

constexpr int kTile = 16;  // query rows
constexpr int kStep = 32;  // keys

// One tile of 16 query rows over some of its keys: every WAVES-th step of 32 keys a wave. Lane l = 16 g + c has
//   scores   keys 4 g + i of both 16-key halves for row c (K . Q^T), and so the weights as P . V's operand,
//   K        key c of each half: 16 (fp8) or up to 32 (fp4) neighbouring columns at a time,
//   V        the same eight keys as its weights, columns D / 16 * c on, transposed in registers two by two.
// Nothing passes through LDS before the waves' sums are joined. Bound by the reading of the cache while there are few
// rows: with 8 heads of 128 for 32 of q, 64 sequences of up to 8192 tokens in e4m3 (558 MB) take 122 us, 4.6 TB/s,
// one of 131 072 in e2m1 (143 MB) 35 us and 6 to join its parts, one of 2048 tokens 12 us with the join, which is the
// latency of a few dependent reads. A page's number is read two steps ahead and codes one: in the first build, of
// four waves and weights of one part, both one step ahead made the first 183 us, not 142, and the second 77, not 57;
// codes two steps ahead changed nothing. Eight waves, twice the reads in flight, then brought them to 137 and 43 us,
// and 32 sequences of 8192 with heads of 64 in fp32 from 77 to 51.
template <int D, int FORMAT, int TYPE, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attention_kernel(AttentionParams p) {
  typedef typename Stored<TYPE>::type T;
  constexpr int kWaves = WAVES;
  constexpr int kQ = TYPE == kBf16 ? 1 : TYPE == kF16 ? 2 : 3;  // parts of a query
  constexpr int kP = 2;                                          // of a weight
  constexpr int kRow = row_bytes(D, FORMAT), kBlocks = D / kBlock;
  constexpr int kChunk = FORMAT == kFp4 && D >= 128 ? 32 : 16;  // columns of a key that a lane has beside each other
  constexpr int kChunks = D / (4 * kChunk);
  constexpr int kChunkWords = kChunk * (FORMAT == kFp8 ? 8 : 4) / 32;
  constexpr int kCols = D / 16;                                    // columns of V a lane
  constexpr int kColBytes = FORMAT == kFp8 ? kCols : kCols / 2;    // 2 to 16
  constexpr int kColWords = kColBytes < 4 ? 1 : kColBytes / 4;
  constexpr int kScaleWords = (kBlocks + 3) / 4;
  // Powers of two of a block's scale byte over its reference: as many as fp16 holds, and when the reference is taken a
  // few less, so a block may grow by 8 (fp8) or 16 times before the sums are scaled.
  constexpr int kMost = FORMAT == kFp8 ? 7 : 13, kTaken = FORMAT == kFp8 ? 4 : 9;
  constexpr int kNoRef = -1000;
  // Weights are e^.. 2^kUp: a maximum may lag 2^2 behind before the sums are scaled. The row's largest is 2^12 or
  // more and fp16's second part ends at 2^-25, so a weight is off by 2^-37 of it where that is more than its own 22
  // bits. With 2^7 and a lag of 2^8 it was 2^-31, and a first token that took the scores but had no value left 250
  // others e^-23 of it with none; a prompt of 8192 tokens took 814 us then and 818 so, with a lag of 2^1 826.
  constexpr float kUp = 13.f, kLag = 2.f;

  const int group = p.heads / p.cache.heads;
  int id = blockIdx.x / (p.splits * p.cache.heads), i, row;
  const int in_tile = blockIdx.x - id * (p.splits * p.cache.heads);
  const int head = in_tile / p.splits, split = in_tile - head * p.splits;
  const int tile = id;
  Sequence s;
  if (!find_tile(p, group, kTile, id, i, s, row)) {
    // id tiles are behind the last one, of which p.tiles - (tile - id) there are.
    note_tile(p, tile, head, split, {0, 0, 0, 0});
    clear_rows<T>(p, id * p.splits * p.cache.heads + in_tile, (p.tiles - (tile - id)) * p.splits * p.cache.heads);
    return;
  }
  const Walk w = walk_of(p, s, group, row, kTile, kStep);
  note_tile(p, tile, head, split, {w.splits, s.first, row, min(kTile, s.count * group - row)});
  if (split >= w.splits) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, c = lane & 15;

  // The row of this lane and what it sees.
  const int rows = s.count * group;
  const int my_row = row + c, token = min(my_row, rows - 1) / group;
  const int my_head = head * group + min(my_row, rows - 1) - token * group;
  Range seen = visible(p, s, token);
  if (my_row >= rows) seen = {0, 0};
  // What all rows of the tile see: no masks there.
  const Range first_sees = visible(p, s, row / group), last_sees = visible(p, s, (min(row + kTile, rows) - 1) / group);
  const int all_low = last_sees.low, all_high = first_sees.high;

  u32x4 q[kQ][D / 32];
  {
    const T* from = static_cast<const T*>(p.q) + (s.first + token) * p.ldq + my_head * p.ldqh;
#pragma unroll
    for (int k = 0; k < D / 32; k++) {
      constexpr int kPer = kChunk / 8;  // of 32 columns in a chunk
      T t[8];
      __builtin_memcpy(t, from + k / kPer * 4 * kChunk + g * kChunk + k % kPer * 8, sizeof(t));
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = (float)t[j];
#pragma unroll
      for (int part = 0; part < kQ; part++) q[part][k] = upper_bits(v);
    }
  }

  const int shift = p.cache.shift, slots = 1 << shift;
  const int* const table = p.batch.table + (long)i * p.batch.columns;
  const long values = (long)p.cache.pages * p.cache.heads << shift;  // slots between a key and its value
  // The pages of both half steps of 16 keys from `key` on, and the slot of a half's first key, or -1 where there are
  // none.
  struct Pages {
    int of[2];
  };
  const auto pages_at = [&](int key) {
    Pages g;
#pragma unroll
    for (int h = 0; h < 2; h++) g.of[h] = table[min(key + 16 * h, w.high - 1) >> shift];
    return g;
  };
  const auto half_at = [&](int key, int of) -> long {
    const int page = __builtin_amdgcn_readfirstlane(of);
    if (key >= w.high || (unsigned)page >= (unsigned)p.cache.pages) return -1;
    return slot_of(p.cache, 0, page, head, key & (slots - 1));
  };

  struct Raw {
    unsigned k[2][kChunks][kChunkWords], v[2][4][kColWords], ks[2][kScaleWords], vs[2][kBlocks];
    bool there[2];
  };
  const auto fetch = [&](int key, const Pages& pages, Raw& r) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      long slot = half_at(key + 16 * h, pages.of[h]);
      r.there[h] = slot >= 0;
      if (slot < 0) slot = 0;
      const uint8_t* kc = p.cache.codes + slot * kRow + c * kRow + g * (4 * kChunkWords);
      const uint8_t* vc = p.cache.codes + (slot + values) * kRow + 4 * g * kRow + c * kColBytes;
#pragma unroll
      for (int n = 0; n < kChunks; n++) __builtin_memcpy(r.k[h][n], kc + n * 16 * kChunkWords, 4 * kChunkWords);
      r.ks[h][0] = 0;
      __builtin_memcpy(r.ks[h], p.cache.scales + (slot + c) * kBlocks, kBlocks);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        r.v[h][j][0] = 0;
        __builtin_memcpy(r.v[h][j], vc + j * kRow, kColBytes);
      }
      __builtin_memcpy(r.vs[h], p.cache.scales + (slot + values + 4 * g) * kBlocks, 4 * kBlocks);
    }
  };

  float m = -__builtin_inff(), l = 0.f;  // of row c: a whole number near its maximum, and this lane's share of the sum
  float base = 0.f;                      // what its scores get to be the exponents of its weights
  bool far = false;                      // whether any row's maximum is, see is_far
  bool any = false;                      // whether this lane has met a key that the row sees
  unsigned none = 0;                     // a bit for each element of its sums in which the row sees a NaN
  int ref = kNoRef;                      // of the block that this lane has columns of
  f32x4 acc[kCols];                      // element i of number t: column kCols * (4 g + i) + t of row c
#pragma unroll
  for (int t = 0; t < kCols; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Lane whose ref is that of element i of this lane's sums.
  const auto of_sums = [&](int i) {
    return D == 64 ? 8 * (g >> 1) : D == 128 ? 4 * g : 4 * g + (i & 2);
  };

  const int end = w.low + kStep * min(w.steps, (split + 1) * w.each);
  int key = w.low + kStep * (split * w.each + wave);
  // Codes one step ahead, page numbers two.
  constexpr int kStride = kStep * kWaves;
  Raw raw, next;
  Pages pages;
  if (key < end) {
    pages = pages_at(key);
    fetch(key, pages, next);
    pages = pages_at(key + kStride);
  }
  for (; key < end; key += kStride) {
    raw = next;
    if (key + kStride < end) {
      const Pages now = pages;
      pages = pages_at(key + 2 * kStride);
      fetch(key + kStride, now, next);
    }

    float x[8];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      f32x4 sum = zeros();
#pragma unroll
      for (int n = 0; n < kChunks; n++) {
        // The chunk lies in block (4 n + g) kChunk / 32.
        const unsigned scale = kChunk == 32 ? raw.ks[h][n] >> 8 * g : raw.ks[h][n / 2] >> (16 * (n & 1) + 8 * (g >> 1));
        const float f = __builtin_bit_cast(float, (scale & 255u) << 23);
#pragma unroll
        for (int e = 0; e < kChunk / 8; e++) {
          u32x4 a;
#pragma unroll
          for (int j = 0; j < 4; j++)
            a[j] = FORMAT == kFp8 ? two_bf16<FORMAT>(raw.k[h][n][2 * e + j / 2], f, j & 1)
                                  : two_bf16<FORMAT>(raw.k[h][n][e], f, j);
#pragma unroll
          for (int part = kQ - 1; part >= 0; part--) sum = mfma_bf16(a, q[part][n * (kChunk / 8) + e], sum);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; j++) x[4 * h + j] = sum[j];
    }

    // Scale bytes of V's blocks; keys that no row sees and pages that are not there count as zeros.
    int sv[8];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int block = c * kCols / kBlock;
        unsigned word;
        if constexpr (D == 64)
          word = raw.vs[h][j / 2] >> (16 * (j & 1) + 8 * block);
        else if constexpr (D == 128)
          word = raw.vs[h][j] >> 8 * block;
        else
          word = (block & 4 ? raw.vs[h][2 * j + 1] : raw.vs[h][2 * j]) >> 8 * (block & 3);
        sv[4 * h + j] = word & 255u;
      }
    const bool whole = key >= w.first && key + kStep <= w.high && raw.there[0] && raw.there[1];
    unsigned sees = 255u;  // a bit for each of the eight keys
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int at = key + 16 * (j / 4) + 4 * g + j % 4;
        if (raw.there[j / 4] && at >= w.first && at < w.high) continue;
        sv[j] = 0;
#pragma unroll
        for (int n = 0; n < kColWords; n++) raw.v[j / 4][j % 4][n] = 0;
      }
    }
    if (!whole || key < all_low || key + kStep > all_high) {
      sees = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int at = key + 16 * (j / 4) + 4 * g + j % 4;
        const bool yes = raw.there[j / 4] && at >= seen.low && at < seen.high;
        sees |= (unsigned)yes << j;
        x[j] = yes ? x[j] : -__builtin_inff();
      }
    }
    any |= sees != 0;

    float top = fmaxf(x[0], x[1]);
#pragma unroll
    for (int j = 2; j < 8; j++) top = fmaxf(top, x[j]);
    top *= p.scale;
    if (__any(top > m + kLag) || far) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float to = fmaxf(m, __builtin_ceilf(top));
      const float f = m == -__builtin_inff() ? 0.f : fast_exp2(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int t = 0; t < kCols; t++) acc[t] *= f;
      base = base_of(m, kUp);
      far = __any(is_far(m));
      if (far)
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = is_far(m) ? behind(p, x[j], m) : x[j];
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      x[j] = fast_exp2(__builtin_fmaf(x[j], p.scale, base));
      l += x[j];
    }
    u32x4 weight[kP];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const unsigned two = pack_h2(x[2 * j], x[2 * j + 1]);
      weight[0][j] = two;
      const h16x2 high = __builtin_bit_cast(h16x2, two);
      weight[1][j] = pack_h2(x[2 * j] - (float)high[0], x[2 * j + 1] - (float)high[1]);
    }

    // Blocks that hold a NaN (scale byte 255): NaN in those columns of the rows that see the key, in no other.
    int largest = 0;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      bad |= sv[j] == 255;
      largest = max(largest, sv[j] == 255 ? 0 : sv[j]);
    }
    if (__any(bad)) {
      u32x4 nan, see;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        nan[j] = (sv[2 * j] == 255 ? 0x3c00u : 0u) | (sv[2 * j + 1] == 255 ? 0x3c000000u : 0u);
        see[j] = (sees >> 2 * j & 1u ? 0x3c00u : 0u) | (sees >> (2 * j + 1) & 1u ? 0x3c000000u : 0u);
      }
      const f32x4 met = mfma16x16x32(nan, see, zeros());
#pragma unroll
      for (int j = 0; j < 4; j++) none |= (unsigned)(met[j] > 0.5f) << j;
#pragma unroll
      for (int j = 0; j < 8; j++) sv[j] = sv[j] == 255 ? 0 : sv[j];
    }
    if (__any(largest > ref + kMost)) {
      largest = max(largest, __shfl_xor(largest, 16));
      largest = max(largest, __shfl_xor(largest, 32));
      const int to = largest > ref + kMost ? largest - kTaken : ref, down = ref - to;
      ref = to;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int d = __shfl(down, of_sums(j));
        const float f = d < -126 ? 0.f : power(d);
#pragma unroll
        for (int t = 0; t < kCols; t++) acc[t][j] *= f;
      }
    }
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = __builtin_bit_cast(float, (unsigned)max(sv[j] - ref + 127, 0) << 23);
#pragma unroll
    for (int u = 0; u < kCols / 2; u++) {
      unsigned two[8];
#pragma unroll
      for (int j = 0; j < 8; j++)
        two[j] = FORMAT == kFp8 ? two_f16<FORMAT>(raw.v[j / 4][j % 4][u / 2], f[j], u & 1)
                                : two_f16<FORMAT>(raw.v[j / 4][j % 4][u / 4], f[j], u & 3);
      u32x4 even, odd;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        even[j] = __builtin_amdgcn_perm(two[2 * j + 1], two[2 * j], 0x05040100u);
        odd[j] = __builtin_amdgcn_perm(two[2 * j + 1], two[2 * j], 0x07060302u);
      }
#pragma unroll
      for (int part = kP - 1; part >= 0; part--) {
        acc[2 * u] = mfma16x16x32(even, weight[part], acc[2 * u]);
        acc[2 * u + 1] = mfma16x16x32(odd, weight[part], acc[2 * u + 1]);
      }
    }
  }

  // The waves' sums joined: rows' maxima and sums, and the values, into LDS.
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  int met = any;
  met |= __shfl_xor(met, 16);
  met |= __shfl_xor(met, 32);
  const float nan = hidden_nan();
  // Divided before the power of two comes back: the mean of values is in their range, their sum may not be.
  const float mean = l == 0.f ? 0.f : 1.f / l;
  if (met && is_zero(l)) l = kLost;
  __shared__ float tops[kWaves][kTile], sums[kWaves][kTile];
  __shared__ __attribute__((aligned(16))) float outs[kWaves][kTile][D + 4];
  if (g == 0) {
    tops[wave][c] = m;
    sums[wave][c] = l;
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int e = __shfl(ref, of_sums(j)) - 127;
#pragma unroll
    for (int t = 0; t < kCols; t++)
      outs[wave][c][kCols * (4 * g + j) + t] = none >> j & 1u ? nan : __builtin_ldexpf(acc[t][j] * mean, e);
  }
  __syncthreads();
  if (WAVES > 4 && threadIdx.x >= 256) return;
  const int r = threadIdx.x / 16, part = threadIdx.x % 16;  // columns kCols * part on of row r
  float top = tops[0][r];
#pragma unroll
  for (int v = 1; v < kWaves; v++) top = fmaxf(top, tops[v][r]);
  float sum = 0.f, share[kWaves], o[kCols];
  bool lost = false;
#pragma unroll
  for (int t = 0; t < kCols; t++) o[t] = 0.f;
#pragma unroll
  for (int v = 0; v < kWaves; v++) {
    share[v] = (tops[v][r] == -__builtin_inff() ? 0.f : fast_exp2(tops[v][r] - top)) * sums[v][r];
    sum += share[v];
    lost |= sums[v][r] == kLost;
  }
  lost &= is_zero(sum);
  const float over = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int v = 0; v < kWaves; v++)
#pragma unroll
    for (int t = 0; t < kCols; t++) o[t] = __builtin_fmaf(share[v] * over, outs[v][r][kCols * part + t], o[t]);
  if (w.splits > 1) {
    float* to = part_of(p, tile, head, split, kTile, D);
    if (part == 0) {
      to[r] = top;
      to[kTile + r] = lost ? kLost : sum;
    }
    __builtin_memcpy(to + 2 * kTile + r * D + kCols * part, o, sizeof(o));
  } else if (row + r < rows) {
    if (lost)
#pragma unroll
      for (int t = 0; t < kCols; t++) o[t] = nan;
    const int token = (row + r) / group, at_head = head * group + row + r - token * group;
    store_row<TYPE, kCols>(p.out, ((long)(s.first + token) * p.heads + at_head) * D + kCols * part, kCols, o);
  }
}

// The parts of split tiles of `rows` rows joined: D / 4 lanes a row, four columns each, which also share the parts'
// maxima and sums. A tile's workgroups have left a note of its rows and parts, so no workgroup looks for its sequence:
// with a search in each, one workgroup a row, the parts of 4 times 801 rows of 8 heads of 64 took 20.7 us, now 5.7.
template <int D, int TYPE>
__global__ __launch_bounds__(256) void join_kernel(AttentionParams p, int rows) {
  constexpr int kLanes = D / 4, kRows = 256 / kLanes;  // of a workgroup, all in one tile
  const long kPart = part_floats(rows, D);
  const int lane = threadIdx.x % kLanes;
  const int at = blockIdx.x * kRows / rows, r = blockIdx.x * kRows % rows + threadIdx.x / kLanes;
  const int head = at % p.cache.heads;
  const Joined w = reinterpret_cast<const Joined*>(p.parts)[at];
  if (r >= w.rows || w.splits == 1) return;
  const float* parts = part_of(p, at / p.cache.heads, head, 0, rows, D);
  float top = -__builtin_inff();
  for (int j = lane; j < w.splits; j += kLanes) top = fmaxf(top, parts[j * kPart + r]);
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  const auto share = [&](int j) {
    const float m = parts[j * kPart + r];
    return (m == -__builtin_inff() ? 0.f : fast_exp2(m - top)) * parts[j * kPart + rows + r];
  };
  float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  int lost = 0;
  for (int j = lane; j < w.splits; j += kLanes) {
    sum += share(j);
    lost |= parts[j * kPart + rows + r] == kLost;
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) {
    sum += __shfl_xor(sum, o);
    lost |= __shfl_xor(lost, o);
  }
  const float over = sum == 0.f ? 0.f : 1.f / sum;
  for (int base = 0; base < w.splits; base += kLanes) {
    const float weight = base + lane < w.splits ? share(base + lane) * over : 0.f;
    const int count = min(kLanes, w.splits - base);
    for (int j = 0; j < count; j += 8) {  // eight reads in flight; behind the last part its own again, without weight
      float o[8][4];
#pragma unroll
      for (int k = 0; k < 8; k++)
        __builtin_memcpy(o[k], parts + (base + min(j + k, count - 1)) * kPart + 2 * rows + r * D + lane * 4, 16);
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float f = __shfl(weight, min(j + k, kLanes - 1), kLanes);
        if (j + k < count)
#pragma unroll
          for (int n = 0; n < 4; n++) v[n] = __builtin_fmaf(f, o[k][n], v[n]);
      }
    }
  }
  if (lost && is_zero(sum)) v[0] = v[1] = v[2] = v[3] = hidden_nan();
  const int group = p.heads / p.cache.heads, token = (w.row + r) / group;
  const int at_head = head * group + w.row + r - token * group;
  store_row<TYPE, 4>(p.out, ((long)(w.first + token) * p.heads + at_head) * D + lane * 4, 4, v);
}

template <int D, int FORMAT, int WAVES>
void start_tiles(const AttentionParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((long)p.tiles * p.cache.heads * p.splits)), block(64 * WAVES);
  if (p.type == kF32)
    hipLaunchKernelGGL((attention_kernel<D, FORMAT, kF32, WAVES>), grid, block, 0, stream, p);
  else if (p.type == kF16)
    hipLaunchKernelGGL((attention_kernel<D, FORMAT, kF16, WAVES>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((attention_kernel<D, FORMAT, kBf16, WAVES>), grid, block, 0, stream, p);
}

template <int D, int FORMAT>
void start_format(const AttentionParams& p, hipStream_t stream) {
  if constexpr (D < 256)
    if (p.form == kTiles8) return start_tiles<D, FORMAT, 8>(p, stream);
  start_tiles<D, FORMAT, 4>(p, stream);
}

template <int D>
void start(const AttentionParams& p, hipStream_t stream) {
  if (p.form == kChunk)
    launch_chunk(p, stream);
  else if (p.cache.format == kFp8)
    start_format<D, kFp8>(p, stream);
  else
    start_format<D, kFp4>(p, stream);
  if (p.splits == 1) return;
  const int rows = p.form == kChunk ? chunk_rows(D, p.type) : kTile;
  const dim3 grid((unsigned)((long)p.tiles * p.cache.heads * rows * (D / 4) / 256)), block(256);
  if (p.type == kF32)
    hipLaunchKernelGGL((join_kernel<D, kF32>), grid, block, 0, stream, p, rows);
  else if (p.type == kF16)
    hipLaunchKernelGGL((join_kernel<D, kF16>), grid, block, 0, stream, p, rows);
  else
    hipLaunchKernelGGL((join_kernel<D, kBf16>), grid, block, 0, stream, p, rows);
}

}  // namespace

AttentionForm attention_form(const AttentionParams& p) {
  AttentionForm f{};
  const long group = p.heads / p.cache.heads, rows = p.rows * group, some = min(p.batch.sequences, p.rows);
  const long keys = (long)p.batch.columns << p.cache.shift;
  // Chunks are for sequences that fill three quarters of one, where the rows read enough to pay for its longer start.
  // Both measured, 32 heads over 8 of 128 in bf16 (tiles / chunks): 8 sequences of 64 rows over 8192 keys 274 / 141
  // us, of 16 rows 74 / 85, 8 of 128 rows over 1024 85 / 56, of 64 46 / 41, of 32 30 / 33; one of 64 over 8192 43 /
  // 41, of 128 over 1024 16 / 32. In fp32, 8 heads of 64, 8 sequences: 128 rows over 8192 98 / 71, 64 rows 52 / 59.
  // Between, 32 rows over 8192 in bf16, half a chunk, would be faster in chunks, 131 / 97, where half a chunk of fp32
  // is not. `keys` is what the table has room for: 128 rows over 1024 keys take 17 us, but 34 with a table for 2^17.
  // Heads of 256 columns have no chunks: three buffers of 64 of their keys and values are 192 KiB of LDS.
  const int high = p.cache.dim < 256 ? chunk_rows(p.cache.dim, p.type) : 0;
  const bool chunk = high && 4 * rows >= 3 * high * some && rows * p.cache.heads >= (1l << 24) / max(keys, 1l);
  const int of = chunk ? high : kTile;
  // Sequences fill their last tiles in part; one tile more for rows of no sequence.
  f.tiles = (rows + some * (of - 1)) / of + 1;
  const long groups = f.tiles * p.cache.heads;
  // Eight waves a tile read more at once, but have twice the sums to join: with 1024 workgroups the CUs are full either
  // way, and 256 sequences of 1024 keys take 81 us with four and 96 with eight. Heads of 256 would spill.
  f.form = chunk ? kChunk : p.cache.dim < 256 && groups < 1024 ? kTiles8 : kTiles4;
  // Workgroups share a tile's keys as long as all of them run at once: one of eight waves a CU, two of four. Rows are
  // taken to be spread evenly over the sequences. 8 sequences of 128 rows over 8192 keys take 375 us with one workgroup
  // a tile, 240 so; one of 512 over 16 384 725 and 225. Twice as many shares of chunks gain up to 18 % where sequences
  // differ in length (the same 8, ragged: 204 and 167) and lose as much as 28 % where they do not (16 of 100 over 2048:
  // 117 and 150). One long sequence among many short ones is not shared at all: 131 072 keys and 31 times 500 take 880
  // us, the long one alone 70.
  const long slots = (chunk ? chunk_waves(p.cache.dim, p.type) == 8 : f.form == kTiles8) ? 256 : 512;
  const long full = some ? some * ((rows + some * of - 1) / (some * of)) : 1;
  f.splits = (int)min(max(slots / (full * p.cache.heads), 1l), min(keys / kLeastKeys + 1, 256l));
  // Sharing saves a tile's waves these keys and costs a second launch. Both measured (shared / not), one row a head,
  // calls in a stream with their launches: 400 keys 11.7 / 9.5 us, 801 11.4 / 11.7 (heads of 64 in fp32 11.4 / 9.4),
  // 1100 11.4 / 13.6; kernels alone, 16 sequences of 801 keys 16.9 / 13.5, of 2048 21.9 / 22.2.
  if (!chunk && keys * (f.splits - 1) < (f.form == kTiles8 ? 640 : 320) * f.splits) f.splits = 1;
  if (f.splits > 1)
    f.bytes = 4 * (size_t)(joined_floats(f.tiles, p.cache.heads) + groups * f.splits * part_floats(of, p.cache.dim));
  return f;
}

hipError_t launch_attention(AttentionParams p, const AttentionForm& f, hipStream_t stream) {
  p.tiles = (int)f.tiles;
  p.splits = f.splits;
  p.form = f.form;
  if (p.cache.dim == 64)
    start<64>(p, stream);
  else if (p.cache.dim == 128)
    start<128>(p, stream);
  else
    start<256>(p, stream);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace ancha
