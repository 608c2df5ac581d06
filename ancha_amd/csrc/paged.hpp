// Paged operators of the gfx950 library: rotary positions, a cache of keys and values in pages of microscaled codes
// (mx.hpp) and attention of new tokens over it. Entry points and their contracts: include/ancha_hip.h.
//
// A cache [2][pages][heads][page][dim] holds keys, then values: codes of dim / 32 blocks a token beside each other and
// their scale bytes in a second array of the same order, so what one head has in one page is one piece of memory of
// each. The tokens of sequence b lie in the pages table[b][0], table[b][1], ...; a number outside [0, pages) is a page
// that is not there.
#pragma once
#include "mx.hpp"

namespace ancha {
namespace paged {

using mx::kBf16;
using mx::kF16;
using mx::kF32;
using mx::kFp4;
using mx::kFp8;
using mx::Stored;

// Sequences of a call, in device memory that the kernels do not trust: every row and page number that they take from
// it is compared with its range first.
struct Batch {
  const int* starts;   // [sequences + 1]
  const int* lengths;  // [sequences]
  const int* table;    // [sequences][columns]
  int sequences, columns;
};

struct Cache {
  uint8_t* codes;
  uint8_t* scales;
  int pages, heads, shift, dim, format;  // 2^shift tokens a page
};
__host__ __device__ constexpr int row_bytes(int dim, int format) { return format == kFp8 ? dim : dim / 2; }

struct Plan {
  const double* freqs;  // [width / 2], or null: nothing is rotated
  int width, interleaved;
  double magnitude;
};

// New tokens [first, first + count) of the rows, the first at position `at`; the sequence has `length` with them.
struct Sequence {
  int first, count, length, at;
};
__device__ __forceinline__ Sequence sequence(const Batch& b, int i, int rows) {
  const int from = min(max(b.starts[i], 0), rows), end = max(b.starts[i + 1], from), length = max(b.lengths[i], 0);
  return {from, min(end, rows) - from, length, length - (end - from)};
}

// The sequence that row r is of, and its position (false: of none); a wave's lanes look together, r is the same in all.
__device__ __forceinline__ bool place(const Batch& b, int r, int& i, int& position) {
  const int lane = threadIdx.x & 63;
  i = 0;  // starts[i] <= r < starts[i + 1], if r is of a sequence: as many ends as are not behind r
  for (int base = 0; base < b.sequences; base += 64) {
    const int more = __popcll(__ballot(base + lane < b.sequences && b.starts[base + lane + 1] <= r));
    i += more;
    if (more < 64) break;
  }
  if (i >= b.sequences) return false;
  const int from = b.starts[i], to = b.starts[i + 1];
  position = max(b.lengths[i], 0) - (to - r);
  return r >= from && r < to;
}

// The page that holds the token at `position` >= 0 of sequence i, or -1.
__device__ __forceinline__ int page_of(const Batch& b, const Cache& c, int i, int position) {
  const int column = position >> c.shift;
  if (column >= b.columns) return -1;
  const int page = b.table[(long)i * b.columns + column];
  return (unsigned)page < (unsigned)c.pages ? page : -1;
}

// Token slot of a head in a page, counted over the whole array of keys (values: pages further on).
__device__ __forceinline__ long slot_of(const Cache& c, int which, int page, int head, int slot) {
  return ((((long)which * c.pages + page) * c.heads + head) << c.shift) + slot;
}

// ---- parameter blocks and launchers (arguments checked by the entry points)

struct RotaryParams {
  const void* x;          // element (row, head, d) at row * ld + head * ldh + d
  const void* positions;  // [rows] of 32 or 64 bits, or null: the batch's
  void* out;              // [rows][heads][dim]
  Batch batch;
  Plan plan;
  long ld, ldh;
  int rows, heads, dim, type, wide;
};
hipError_t launch_rotary(const RotaryParams& p, hipStream_t stream);

struct WriteParams {
  const void* k;
  const void* v;
  Batch batch;
  Plan plan;
  Cache cache;
  long ldk, ldkh, ldv, ldvh;
  int rows, type;
};
hipError_t launch_write(const WriteParams& p, hipStream_t stream);

struct ReadParams {
  Batch batch;
  Cache cache;
  void* k;  // [sequences][size][heads][dim]
  void* v;
  int size, type;
};
hipError_t launch_read(const ReadParams& p, hipStream_t stream);

struct AttentionParams {
  const void* q;  // element (row, head, d) at row * ldq + head * ldqh + d
  void* out;      // [rows][heads][dim]
  Batch batch;
  Cache cache;
  float* parts;  // workspace of a split, see attention_form
  long ldq, ldqh;
  int rows, heads, type, causal, window;  // window 0: none
  float scale, unscale;                   // of the scores, times log2(e), and its inverse
  int tiles, splits, form;                // of its AttentionForm
};

// How a call is laid out: tiles of 16 query rows by four or eight waves, or the chunk kernel's; tiles (an upper bound,
// the kernels count the real ones); the workgroups that share the keys of a tile; bytes of workspace.
enum { kTiles4, kTiles8, kChunk };
struct AttentionForm {
  int form;
  long tiles;
  int splits;
  size_t bytes;
};
AttentionForm attention_form(const AttentionParams& p);  // of the type, the sizes and the batch's
hipError_t launch_attention(AttentionParams p, const AttentionForm& form, hipStream_t stream);
void launch_chunk(const AttentionParams& p, hipStream_t stream);

// The chunk kernel takes heads of 64 or 128 columns; its waves have 32 query rows each and walk in steps of kChunkKeys.
// (fp32 queries of 128 columns are 96 registers in three parts, which leaves room for one wave a SIMD.)
constexpr int kChunkKeys = 64;
constexpr int chunk_waves(int dim, int type) { return dim == 128 && type != kF32 ? 8 : 4; }
constexpr int chunk_rows(int dim, int type) { return 32 * chunk_waves(dim, type); }

}  // namespace paged
}  // namespace ancha
