// Attention of many new tokens over a paged, microscaled cache (gfx950): chunks and whole prompts. The operation and
// its operands are those of paged_attention.hip; here 128 or 256 query rows share the keys that a workgroup reads.
// Heads of 64 or 128 columns.
#include "paged_attention.hpp"

namespace ancha {
namespace paged {
namespace {

constexpr int kBuffers = 3;         // steps of keys and values in LDS
constexpr int kKeys = kChunkKeys;  // of a step

__device__ __forceinline__ f32x16 mfma32_bf16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

// Orders what this wave's lanes write to LDS before what they read from it (LDS serves a wave in order).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int D, int FORMAT, int TYPE>
struct Shape {
  static constexpr int kQ = TYPE == kBf16 ? 1 : TYPE == kF16 ? 2 : 3;  // bf16 parts of a query
  static constexpr int kP = 2;                                         // fp16 parts of a weight
  static constexpr int kWaves = chunk_waves(D, TYPE), kThreads = 64 * kWaves, kRows = 32 * kWaves;
  static constexpr int kScales = D / kBlock;            // scale bytes a token
  static constexpr int kBuffer = 2 * kKeys * D * 2;     // LDS bytes of a step's keys and values
  // A wave's own: the powers of two of a step's values, and for every buffer which blocks of a token are NaN.
  static constexpr int kPowers = kKeys * kScales * 4, kPrivate = kPowers + kBuffers * kKeys;
  static constexpr int kLds = kBuffers * kBuffer + kWaves * kPrivate;
};

// A workgroup has 32 query rows a wave and walks over the keys in steps of 64: its threads bring a step's codes to
// bf16 (keys) and fp16 (values) once and leave them in LDS in the order in which the matrix instructions take them, two
// steps ahead. With l = 32 h + r, a lane has
//   scores   element 4 q + e: key 8 q + 4 h + e of 32 for row r (K . Q^T), so the weights are the operand of V^T . P
//            as they are, if V's keys come in the same order: 16 s + 4 h + (0..3) and 8 further on,
//   sums     element 4 q + e of block b: column 32 b + 8 q + 4 h + e of row r.
// A block of 32 columns is one of the cache's own, so its reference power is one number a workgroup.
//
// Bound by the matrix units and what runs beside them: a prompt of 8192 tokens, 32 heads over 8 of 128 in bf16, is
// 0.55 TFLOP and takes 793 to 878 us replayed on one card and another, 0.63 to 0.69 PFLOP/s; with the weights' second
// part it is 0.82 TFLOP of products, 0.94 to 1.04 PFLOP/s, where a library product of 8192^3 reaches 1.3. 4 times 801
// rows of 8 heads of 64 over 4096 keys, in fp32, take 69 us and 6 to join. With weights of one part, 11 bits, the
// prompt took 615 to 653 us on the same cards; of that build: with the products alone 389 us, without bringing the
// codes 513, without the exponentials 611. What did not help an earlier one of 655 us: 64 rows a wave with one wave a
// SIMD 946; four reads ahead of the products 698; groups given to the scheduler 700; wave priorities 690; sums by
// adds 675 or by a product with ones 655; the next half's scores ahead of these weights, codes two steps ahead: no
// change. Both halves of a step at once made that one 3 % faster, 636, and have not been tried on this one.
template <int D, int FORMAT, int TYPE>
__global__ __launch_bounds__(64 * chunk_waves(D, TYPE), D == 64 ? 2 : 1) void chunk_kernel(AttentionParams p) {
  typedef typename Stored<TYPE>::type T;
  typedef Shape<D, FORMAT, TYPE> S;
  constexpr int kQ = S::kQ, kP = S::kP, kScales = S::kScales, kRow = row_bytes(D, FORMAT);
  constexpr int kWaves = S::kWaves, kThreads = S::kThreads;
  // As many blocks of keys as groups of eight values x four columns: one of each a thread, or half the waves have
  // either.
  constexpr int kUnits = kKeys * kScales;
  static_assert(kUnits == kThreads || 2 * kUnits == kThreads, "a unit a thread");
  constexpr bool kApart = kUnits < kThreads;
  constexpr int kBlockWords = FORMAT == kFp8 ? 8 : 4;
  constexpr int kTurn = 8 / kScales;                                             // see slot_of_key
  constexpr int kMost = FORMAT == kFp8 ? 7 : 13, kTaken = FORMAT == kFp8 ? 4 : 9;  // see paged_attention.hip
  constexpr int kNoRef = -1000;
  constexpr float kUp = 13.f, kLag = 2.f;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];

  const int group = p.heads / p.cache.heads;
  // Workgroups beside each other on an XCD share a head. Tiles go from the last to the first, so that of one sequence
  // those that see the most keys begin first (of several, the last sequence's, however long it is).
  const int place = xcd_remap(blockIdx.x, p.tiles * p.cache.heads * p.splits);
  const int head = place / (p.tiles * p.splits), in_head = place - head * (p.tiles * p.splits);
  int id = p.tiles - 1 - in_head / p.splits, i, row;
  const int tile = id, split = in_head % p.splits;
  Sequence s;
  if (!find_tile(p, group, S::kRows, id, i, s, row)) {
    note_tile(p, tile, head, split, {0, 0, 0, 0});
    clear_rows<T>(p, (id * p.cache.heads + head) * p.splits + split,
                  (p.tiles - (tile - id)) * p.cache.heads * p.splits);
    return;
  }
  const Walk w = walk_of(p, s, group, row, S::kRows, kKeys);
  note_tile(p, tile, head, split, {w.splits, s.first, row, min(S::kRows, s.count * group - row)});
  if (split >= w.splits) return;
  const int begin = split * w.each, end = min(w.steps, begin + w.each);  // steps of this workgroup
  const int thread = threadIdx.x, lane = thread & 63, h = lane >> 5, r = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
  const int rows = s.count * group;

  // The row of this lane and what it sees, and the steps that this wave's rows see.
  const int my_rows = row + 32 * wave, my_row = my_rows + r, token = min(my_row, rows - 1) / group;
  const int my_head = head * group + min(my_row, rows - 1) - token * group;
  Range seen = visible(p, s, token);
  if (my_row >= rows) seen = {0, 0};
  const Range wave_first = visible(p, s, min(my_rows, rows - 1) / group);
  const Range wave_last = visible(p, s, (min(my_rows + 32, rows) - 1) / group);
  const int wave_begin = max(begin, (wave_first.low - w.low) / kKeys);
  const int wave_end = my_rows < rows ? min(end, (wave_last.high - w.low + kKeys - 1) / kKeys) : 0;
  u32x4 q[kQ][D / 16];
  {
    const T* from = static_cast<const T*>(p.q) + (s.first + token) * p.ldq + my_head * p.ldqh;
#pragma unroll
    for (int k = 0; k < D / 16; k++) {
      T t[8];
      __builtin_memcpy(t, from + 16 * k + 8 * h, sizeof(t));
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = (float)t[j];
#pragma unroll
      for (int part = 0; part < kQ; part++) q[part][k] = upper_bits(v);
    }
  }

  const int shift = p.cache.shift;
  const int* const table = p.batch.table + (long)i * p.batch.columns;
  const long values = (long)p.cache.pages * p.cache.heads << shift;
  const auto page_at = [&](int key) -> int {
    const int column = key >> shift;
    return key < w.high ? table[column] : -1;
  };
  const auto slot_at = [&](int page, int key) -> long {
    const bool there = (unsigned)page < (unsigned)p.cache.pages;
    return slot_of(p.cache, 0, there ? page : 0, head, there ? key & ((1 << shift) - 1) : key & 15);
  };
  // What this thread brings: the scale bytes of key `lane` (every wave for itself), a block of a key, a group of
  // values.
  const bool has_key = !kApart || wave < kWaves / 2, has_value = !kApart || wave >= kWaves / 2;
  const int unit = thread % kUnits;
  const int my_key = unit / kScales, key_block = unit % kScales;
  const int half = unit / (D / 4), col = unit % (D / 4), value_block = col / 8;  // half: 2 s + h; col: of four
  const auto value_of = [&](int j) { return 16 * (half / 2) + 4 * (half & 1) + j / 4 * 8 + j % 4; };
  // LDS order of an operand: 64 pieces of 16 bytes, lane l's at l with a few low bits turned, so that threads beside
  // each other, which write to several operands or every fourth piece, meet different banks.
  const auto slot_of_key = [&](int l, int block) { return l ^ (block * kTurn & 7); };
  const auto slot_of_value = [&](int l) { return l ^ (l >> 3 & 3); };

  struct Pages {
    int scale, key, value;
  };
  struct Raw {
    unsigned codes[kApart ? 8 : 16], vs, ks;  // of a key (block by block), of eight values; the same place where apart
    int page;                                 // of key `lane`
  };
  constexpr int kValues = kApart ? 0 : 8;  // where the values' are
  const auto fetch_pages = [&](int key, Pages& g) {
    g.scale = page_at(key + lane);
    if (has_key) g.key = page_at(key + my_key);
    if (has_value) g.value = page_at(key + 16 * (half / 2));
  };
  const auto fetch = [&](int key, const Pages& g, Raw& w) {
    w.vs = 0;
    __builtin_memcpy(&w.vs, p.cache.scales + (slot_at(g.scale, key + lane) + values) * kScales, kScales);
    w.page = g.scale;
    if (has_key) {
      const long at = slot_at(g.key, key + my_key);
      w.ks = p.cache.scales[at * kScales + key_block];
      __builtin_memcpy(w.codes, p.cache.codes + at * kRow + key_block * 4 * kBlockWords, 4 * kBlockWords);
    }
    if (has_value) {
      const uint8_t* from = p.cache.codes + (slot_at(g.value, key + 16 * (half / 2)) + values) * kRow +
                            col * (FORMAT == kFp8 ? 4 : 2);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        w.codes[kValues + j] = 0;
        __builtin_memcpy(&w.codes[kValues + j], from + (value_of(j) & 15) * kRow, FORMAT == kFp8 ? 4 : 2);
      }
    }
  };

  float m = -__builtin_inff(), l = 0.f;  // of row r: a whole number near its maximum; this lane's share of its sum
  float base = 0.f;                      // what its scores get to be the exponents of its weights
  bool far = false;                      // whether any row's maximum is, see is_far
  bool any = false;                      // whether this lane has met a key that the row sees
  unsigned none = 0;                     // a bit for each block of columns in which the row sees a NaN
  f32x16 acc[kScales];
#pragma unroll
  for (int c = 0; c < kScales; c++) acc[c] = mfma32_zero();
  // References: of the sums, of the next step's values in LDS, of the ones behind them.
  int sum_ref[kScales], next_ref[kScales], ref[kScales];
#pragma unroll
  for (int c = 0; c < kScales; c++) sum_ref[c] = next_ref[c] = ref[c] = kNoRef;
  // Tokens that are there and whether any of them has a NaN among its values, in the same order.
  constexpr unsigned long long kAll = ~0ull;
  unsigned long long there = 0, next_there = 0, last_there = 0;
  bool bad = false, next_bad = false, last_bad = false;

  uint8_t* const mine = lds + kBuffers * S::kBuffer + wave * S::kPrivate;
  float* const powers = reinterpret_cast<float*>(mine);  // [block][value]
  // Brings the codes of the step from `key` on into buffer `to`.
  const auto bring = [&](int key, Raw& w_, int to) {
    uint8_t* const keys = lds + to * S::kBuffer;
    uint8_t* const vals = keys + kKeys * D * 2;
    const int at_key = key + lane;
    const bool here = (unsigned)w_.page < (unsigned)p.cache.pages && at_key >= w.first && at_key < w.high;
    last_there = __ballot(here);
    int e[kScales];
    bool over = false;  // a block that is larger than its reference allows, or NaN (255)
#pragma unroll
    for (int c = 0; c < kScales; c++) {
      e[c] = here ? (int)(w_.vs >> 8 * c & 255u) : 0;
      over |= e[c] > ref[c] + kMost;
    }
    last_bad = false;
    if (__any(over)) {
      unsigned nan = 0;
#pragma unroll
      for (int c = 0; c < kScales; c++) {
        nan |= (unsigned)(e[c] == 255) << c;
        if (e[c] == 255) e[c] = 0;
        int x = e[c];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) x = max(x, __shfl_xor(x, o));
        x = __builtin_amdgcn_readfirstlane(x);
        // At most 254 - kMost, which has room for the largest byte of a number and leaves 255 above it.
        ref[c] = x > ref[c] + kMost ? min(x - kTaken, 254 - kMost) : ref[c];
      }
      last_bad = __any(nan != 0);
      mine[S::kPowers + to * kKeys + lane] = nan;
    }
    if (has_value) {
#pragma unroll
      for (int c = 0; c < kScales; c++)
        powers[c * kKeys + lane] = __builtin_bit_cast(float, (unsigned)max(e[c] - ref[c] + 127, 0) << 23);
    }
    wave_sync();
    if (has_key) {
      const float f = __builtin_bit_cast(float, w_.ks << 23);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        u32x4 x;
#pragma unroll
        for (int n = 0; n < 4; n++)
          x[n] = FORMAT == kFp8 ? two_bf16<FORMAT>(w_.codes[2 * j + n / 2], f, n & 1)
                                : two_bf16<FORMAT>(w_.codes[j], f, n);
        const int at = (my_key / 32 * (D / 16) + 2 * key_block + j / 2) * 64;
        *reinterpret_cast<u32x4*>(keys + (at + slot_of_key(32 * (j & 1) + my_key % 32, key_block)) * 16) = x;
      }
    }
    if (has_value) {
      if (last_there != kAll) {
        asm volatile("");  // a branch, not eight selections every time
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (!(last_there >> value_of(j) & 1)) w_.codes[kValues + j] = 0;
      }
      float f[8];
      __builtin_memcpy(f, powers + value_block * kKeys + value_of(0), 16);
      __builtin_memcpy(f + 4, powers + value_block * kKeys + value_of(4), 16);
      unsigned two[2][8];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int j = 0; j < 8; j++) two[u][j] = two_f16<FORMAT>(w_.codes[kValues + j], f[j], u);
#pragma unroll
      for (int d = 0; d < 4; d++) {
        u32x4 x;
#pragma unroll
        for (int j = 0; j < 4; j++)
          x[j] = __builtin_amdgcn_perm(two[d / 2][2 * j + 1], two[d / 2][2 * j], d & 1 ? 0x07060302u : 0x05040100u);
        const int at = slot_of_value(32 * (half & 1) + col % 8 * 4 + d);  // the lane that takes it
        *reinterpret_cast<u32x4*>(vals + ((value_block * (kKeys / 16) + half / 2) * 64 + at) * 16) = x;
      }
    }
    wave_sync();
  };
  const f32x16 zero = mfma32_zero();
  // Scores of half u of the step in buffer `from`.
  const auto scores = [&](int from, int u) {
    const uint8_t* const keys = lds + from * S::kBuffer + u * (D / 16) * 1024;
    f32x16 x = zero;
#pragma unroll
    for (int k = 0; k < D / 16; k++) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(keys + k * 1024 + slot_of_key(lane, k / 2) * 16);
#pragma unroll
      for (int part = kQ - 1; part >= 0; part--) x = mfma32_bf16(a, q[part][k], x);
    }
    return x;
  };

  const auto key_at = [&](int step) { return w.low + step * kKeys; };
  Pages pages;
  Raw raw;
  if (begin < end) {
    fetch_pages(key_at(begin), pages);
    fetch(key_at(begin), pages, raw);
    if (begin + 1 < end) fetch_pages(key_at(begin + 1), pages);
    bring(key_at(begin), raw, 0);
    if (begin + 1 < end) {
      next_there = last_there, next_bad = last_bad;
#pragma unroll
      for (int c = 0; c < kScales; c++) next_ref[c] = ref[c];
      fetch(key_at(begin + 1), pages, raw);
      if (begin + 2 < end) fetch_pages(key_at(begin + 2), pages);
      bring(key_at(begin + 1), raw, 1);
      if (begin + 2 < end) fetch(key_at(begin + 2), pages, raw);
      if (begin + 3 < end) fetch_pages(key_at(begin + 3), pages);
    } else {
      next_there = last_there, next_bad = last_bad;
#pragma unroll
      for (int c = 0; c < kScales; c++) next_ref[c] = ref[c];
    }
  }
  __syncthreads();
  for (int step = begin, from = 0; step < end; step++) {
    const int key = key_at(step), after = from == 2 ? 0 : from + 1, last = after == 2 ? 0 : after + 1;
    there = next_there, bad = next_bad;
    next_there = last_there, next_bad = last_bad;
    bool scaled = false;
#pragma unroll
    for (int c = 0; c < kScales; c++) scaled |= next_ref[c] != sum_ref[c];
    if (scaled) {
#pragma unroll
      for (int c = 0; c < kScales; c++) {
        const int d = sum_ref[c] - next_ref[c];
        acc[c] *= d < -126 ? 0.f : power(d);
        sum_ref[c] = next_ref[c];
      }
    }
#pragma unroll
    for (int c = 0; c < kScales; c++) next_ref[c] = ref[c];
    const uint8_t* const vals = lds + from * S::kBuffer + kKeys * D * 2 + slot_of_value(lane) * 16;
    const bool active = step >= wave_begin && step < wave_end;
    const bool plain = there == kAll && key >= wave_last.low && key + kKeys <= wave_first.high;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      if (active) {
        f32x16 x = scores(from, u);
        unsigned sees = 0x0f0f0f0fu;  // bit 8 q + e: whether the row sees the key of element 4 q + e
        if (!plain) {
          asm volatile("");
          const int at = key + 32 * u + 4 * h;
          const unsigned below = ~0u >> (32 - min(max(seen.high - at, 0), 31)) % 32;
          sees = (seen.high > at ? below : 0u) & ~0u << min(max(seen.low - at, 0), 31);
          sees &= (unsigned)(there >> 32 * u) >> 4 * h & 0x0f0f0f0fu;
#pragma unroll
          for (int j = 0; j < 16; j++) x[j] = sees >> (j / 4 * 8 + j % 4) & 1u ? x[j] : -__builtin_inff();
        }
        any |= sees != 0;
        if (bad) {
#pragma unroll
          for (int j = 0; j < 16; j++) {
            const unsigned nan = mine[S::kPowers + from * kKeys + 32 * u + j / 4 * 8 + 4 * h + j % 4];
            none |= sees >> (j / 4 * 8 + j % 4) & 1u ? nan : 0u;
          }
        }
        float top = fmaxf(x[0], x[1]);
#pragma unroll
        for (int j = 2; j < 16; j++) top = fmaxf(top, x[j]);
        top *= p.scale;
        if (__any(top > m + kLag) || far) {
          top = fmaxf(top, __shfl_xor(top, 32));
          const float to = fmaxf(m, __builtin_ceilf(top));
          const float f = m == -__builtin_inff() ? 0.f : fast_exp2(m - to);
          m = to;
          l *= f;
#pragma unroll
          for (int c = 0; c < kScales; c++) acc[c] *= f;
          base = base_of(m, kUp);
          far = __any(is_far(m));
          if (far)
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = is_far(m) ? behind(p, x[j], m) : x[j];
        }
        u32x4 weight[kP][2];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float a = fast_exp2(__builtin_fmaf(x[2 * j], p.scale, base));
          const float b = fast_exp2(__builtin_fmaf(x[2 * j + 1], p.scale, base));
          const unsigned two = pack_h2(a, b);
          weight[0][j / 4][j % 4] = two;
          const h16x2 high = __builtin_bit_cast(h16x2, two);
          weight[1][j / 4][j % 4] = pack_h2(a - (float)high[0], b - (float)high[1]);
          l += a;
          l += b;
        }
#pragma unroll
        for (int v = 0; v < 2; v++)
#pragma unroll
          for (int c = 0; c < kScales; c++) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(vals + (c * (kKeys / 16) + 2 * u + v) * 1024);
#pragma unroll
            for (int part = kP - 1; part >= 0; part--) acc[c] = mfma32(a, weight[part][v], acc[c]);
          }
      }
      if (u == 0 && step + 2 < end) {
        bring(key_at(step + 2), raw, last);
        if (step + 3 < end) fetch(key_at(step + 3), pages, raw);
        if (step + 4 < end) fetch_pages(key_at(step + 4), pages);
      }
    }
    from = after;
    __syncthreads();
  }

  const float sum = l + __shfl_xor(l, 32);
  int met = any;
  met |= __shfl_xor(met, 32);
  none |= __shfl_xor(none, 32);
  const float nan = hidden_nan();
  const float over = sum == 0.f ? 0.f : 1.f / sum;
  const bool lost = met && is_zero(sum);
  if (lost && w.splits == 1) none = ~0u;
  float* const part = part_of(p, tile, head, split, S::kRows, D);
  if (w.splits > 1 && h == 0) {
    part[32 * wave + r] = m;
    part[S::kRows + 32 * wave + r] = lost ? kLost : sum;
  }
  if (my_row >= rows) return;
  const long to = ((long)(s.first + token) * p.heads + my_head) * D;
#pragma unroll
  for (int c = 0; c < kScales; c++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; e++)
        v[e] = none >> c & 1u ? nan : __builtin_ldexpf(acc[c][4 * j + e] * over, sum_ref[c] - 127);
      const int at = 32 * c + 8 * j + 4 * h;
      if (w.splits > 1)
        __builtin_memcpy(part + 2 * S::kRows + (32 * wave + r) * D + at, v, sizeof(v));
      else
        store_row<TYPE, 4>(p.out, to + at, 4, v);
    }
}

template <int D, int FORMAT, int TYPE>
void start(const AttentionParams& p, hipStream_t stream) {
  typedef Shape<D, FORMAT, TYPE> S;
  hipLaunchKernelGGL((chunk_kernel<D, FORMAT, TYPE>), dim3((unsigned)((long)p.tiles * p.cache.heads * p.splits)),
                     dim3(S::kThreads), S::kLds, stream, p);
}

template <int D, int FORMAT>
void start_type(const AttentionParams& p, hipStream_t stream) {
  if (p.type == kF32) return start<D, FORMAT, kF32>(p, stream);
  if (p.type == kF16) return start<D, FORMAT, kF16>(p, stream);
  start<D, FORMAT, kBf16>(p, stream);
}

template <int D>
void start_format(const AttentionParams& p, hipStream_t stream) {
  if (p.cache.format == kFp8)
    start_type<D, kFp8>(p, stream);
  else
    start_type<D, kFp4>(p, stream);
}

}  // namespace

void launch_chunk(const AttentionParams& p, hipStream_t stream) {
  if (p.cache.dim == 64)
    start_format<64>(p, stream);
  else
    start_format<128>(p, stream);
}

}  // namespace paged
}  // namespace ancha
