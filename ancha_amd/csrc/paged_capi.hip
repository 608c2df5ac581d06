// C ABI entry points of the paged operators (include/ancha_hip.h): argument checks and dispatch.
#include <cmath>
#include <string>

#include "paged.hpp"
#include "status.hpp"

namespace {

using ancha::fail;
using ancha::hip_fail;
using ancha::sticky;
namespace paged = ancha::paged;

constexpr size_t kIntMax = 0x7fffffff;
constexpr size_t kRows = (1 << 24) - 1;  // a workgroup of 256 threads each: below HIP's 2^32 of them

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
bool is_type(int t) { return t == ANCHA_HIP_F32 || t == ANCHA_HIP_F16 || t == ANCHA_HIP_BF16; }

// A finite number above `least`; on the bits, as the library is compiled without NaN semantics.
bool above(double x, double least) {
  volatile uint64_t bits;
  bits = __builtin_bit_cast(uint64_t, x);
  return (bits >> 52 & 0x7ff) != 0x7ff && x > least;
}

int not_here(const std::string& who) { return fail(ANCHA_HIP_UNSUPPORTED, who + ": not a gfx950 device"); }

// 0, or what is wrong with a batch, which goes to `to`.
int check_batch(const std::string& who, const ancha_paged_batch* b, bool starts, bool table, paged::Batch& to) {
  if (!b) return fail(ANCHA_HIP_INVALID, who + ": null batch");
  if (b->sequences && ((starts && !b->starts) || !b->lengths || (table && b->columns && !b->table)))
    return fail(ANCHA_HIP_INVALID, who + ": null tensor in the batch");
  if (!aligned(b->starts, 4) || !aligned(b->lengths, 4) || !aligned(b->table, 4))
    return fail(ANCHA_HIP_INVALID, who + ": the batch must be 4-byte aligned");
  if (b->sequences >= kIntMax || b->columns > kIntMax)
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": too many sequences or pages of one");
  to = {b->starts, b->lengths, b->table, static_cast<int>(b->sequences), static_cast<int>(b->columns)};
  return 0;
}

int check_cache(const std::string& who, const ancha_paged_cache* c, paged::Cache& to) {
  if (!c) return fail(ANCHA_HIP_INVALID, who + ": null cache");
  if (c->format != ANCHA_HIP_MX_FP8 && c->format != ANCHA_HIP_MX_FP4)
    return fail(ANCHA_HIP_INVALID, who + ": unknown format");
  if (!c->codes || !c->scales || c->pages == 0 || c->heads == 0)
    return fail(ANCHA_HIP_INVALID, who + ": an empty cache");
  if (!aligned(c->codes, 16) || !aligned(c->scales, 16))
    return fail(ANCHA_HIP_INVALID, who + ": the cache must be 16-byte aligned");
  if (c->page < 16 || c->page > 65536 || (c->page & (c->page - 1)))
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": pages hold a power of two of tokens, from 16 to 65536");
  if (c->dim != 64 && c->dim != 128 && c->dim != 256)
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": the head width is 64, 128 or 256");
  // A token's heads in a 28-bit count of 4-value units; slots in 48 bits, so their bytes stay in 63.
  if (c->pages > kIntMax || c->heads > 65536 || c->pages * c->heads > (size_t(1) << 47) / c->page)
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": too large a cache");
  to = {static_cast<uint8_t*>(c->codes), static_cast<uint8_t*>(c->scales), static_cast<int>(c->pages),
        static_cast<int>(c->heads), __builtin_ctzll(c->page), static_cast<int>(c->dim), c->format};
  return 0;
}

int check_plan(const std::string& who, const ancha_paged_plan* p, size_t dim, paged::Plan& to) {
  if (!p->freqs || !aligned(p->freqs, 8)) return fail(ANCHA_HIP_INVALID, who + ": freqs is null or not 8-byte aligned");
  if (p->width == 0 || p->width % 2 || p->width > dim)
    return fail(ANCHA_HIP_INVALID, who + ": the rotated width is even, above 0 and at most the head's");
  if (!above(p->magnitude, 0.0) || p->magnitude > 3.4e38)
    return fail(ANCHA_HIP_INVALID, who + ": magnitude is not an fp32 number > 0");
  to = {p->freqs, static_cast<int>(p->width), p->interleaved ? 1 : 0, p->magnitude};
  return 0;
}

// Strides of [rows][heads][dim]: neighbouring heads and rows may lie anywhere (broadcast ones at one place).
bool strides_fit(size_t rows, size_t ld, size_t heads, size_t ldh) {
  constexpr size_t kMost = size_t(1) << 59;
  return (rows < 2 || ld <= kMost / rows) && (heads < 2 || ldh <= kMost / heads);
}

}  // namespace

extern "C" {

int ancha_paged_rotary(const void* x, int type, size_t rows, size_t heads, size_t dim, size_t ldx, size_t ldh,
                       const void* positions, int position_bytes, const ancha_paged_batch* batch,
                       const ancha_paged_plan* plan, void* out, hipStream_t stream) {
  if (const int s = sticky()) return s;
  const std::string who("ancha_paged_rotary");
  if (!is_type(type)) return fail(ANCHA_HIP_INVALID, who + ": unknown type");
  if (!plan) return fail(ANCHA_HIP_INVALID, who + ": null plan");
  paged::RotaryParams p{};
  if (const int e = check_plan(who, plan, dim, p.plan)) return e;
  if (positions) {
    if ((position_bytes != 4 && position_bytes != 8) || !aligned(positions, static_cast<size_t>(position_bytes)))
      return fail(ANCHA_HIP_INVALID, who + ": positions have 4 or 8 bytes and are aligned to them");
  } else if (const int e = check_batch(who, batch, true, false, p.batch)) {
    return e;
  }
  if (rows == 0 || heads == 0) return ANCHA_HIP_OK;
  if (!x || !out) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if (plan->width > 2048 || rows > kRows || heads > (size_t(1) << 21) || dim > (size_t(1) << 21) ||
      heads * dim > (size_t(1) << 21) || !strides_fit(rows, ldx, heads, ldh))
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": too many rows, heads or columns");
  if (!ancha_hip_available()) return not_here(who);
  p.x = x;
  p.positions = positions;
  p.out = out;
  p.ld = static_cast<long>(ldx);
  p.ldh = static_cast<long>(ldh);
  p.rows = static_cast<int>(rows);
  p.heads = static_cast<int>(heads);
  p.dim = static_cast<int>(dim);
  p.type = type;
  p.wide = position_bytes == 8;
  const hipError_t e = paged::launch_rotary(p, stream);
  return e == hipSuccess ? ANCHA_HIP_OK : hip_fail(e, who);
}

int ancha_paged_write(const void* k, const void* v, int type, size_t rows, size_t ldk, size_t ldkh, size_t ldv,
                      size_t ldvh, const ancha_paged_batch* batch, const ancha_paged_plan* plan,
                      const ancha_paged_cache* cache, hipStream_t stream) {
  if (const int s = sticky()) return s;
  const std::string who("ancha_paged_write");
  if (!is_type(type)) return fail(ANCHA_HIP_INVALID, who + ": unknown type");
  paged::WriteParams p{};
  if (const int e = check_cache(who, cache, p.cache)) return e;
  if (plan)
    if (const int e = check_plan(who, plan, cache->dim, p.plan)) return e;
  if (const int e = check_batch(who, batch, true, true, p.batch)) return e;
  if (rows == 0) return ANCHA_HIP_OK;
  if (!k || !v) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if (rows > kRows || !strides_fit(rows, ldk, cache->heads, ldkh) || !strides_fit(rows, ldv, cache->heads, ldvh))
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": too many rows");
  if (!ancha_hip_available()) return not_here(who);
  p.k = k;
  p.v = v;
  p.ldk = static_cast<long>(ldk);
  p.ldkh = static_cast<long>(ldkh);
  p.ldv = static_cast<long>(ldv);
  p.ldvh = static_cast<long>(ldvh);
  p.rows = static_cast<int>(rows);
  p.type = type;
  const hipError_t e = paged::launch_write(p, stream);
  return e == hipSuccess ? ANCHA_HIP_OK : hip_fail(e, who);
}

int ancha_paged_read(const ancha_paged_cache* cache, const ancha_paged_batch* batch, size_t size, int type, void* k,
                     void* v, hipStream_t stream) {
  if (const int s = sticky()) return s;
  const std::string who("ancha_paged_read");
  if (!is_type(type)) return fail(ANCHA_HIP_INVALID, who + ": unknown type");
  paged::ReadParams p{};
  if (const int e = check_cache(who, cache, p.cache)) return e;
  if (const int e = check_batch(who, batch, false, true, p.batch)) return e;
  if (size == 0 || batch->sequences == 0) return ANCHA_HIP_OK;
  if (!k || !v) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(ANCHA_HIP_INVALID, who + ": k and v must be 16-byte aligned");
  // At most one workgroup a token, of 256 threads: below HIP's 2^32 of them.
  if (size > kIntMax - 65536 || size > ((size_t(1) << 24) - 1) / batch->sequences)
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": too many tokens");
  if (!ancha_hip_available()) return not_here(who);
  p.k = k;
  p.v = v;
  p.size = static_cast<int>(size);
  p.type = type;
  const hipError_t e = paged::launch_read(p, stream);
  return e == hipSuccess ? ANCHA_HIP_OK : hip_fail(e, who);
}

size_t ancha_paged_attention_workspace(int type, size_t rows, size_t heads, const ancha_paged_cache* cache,
                                       const ancha_paged_batch* batch) {
  paged::AttentionParams p{};
  if (!is_type(type) || !cache || !batch || !cache->heads || !heads || heads % cache->heads || rows == 0 ||
      rows > kIntMax || heads > kIntMax || rows * heads > kIntMax || cache->page < 16 || cache->page > 65536 ||
      batch->sequences >= kIntMax || batch->columns > kIntMax)
    return 0;
  p.type = type;
  p.rows = static_cast<int>(rows);
  p.heads = static_cast<int>(heads);
  p.cache.heads = static_cast<int>(cache->heads);
  p.cache.shift = __builtin_ctzll(cache->page);
  p.cache.dim = static_cast<int>(cache->dim);
  p.batch.sequences = static_cast<int>(batch->sequences);
  p.batch.columns = static_cast<int>(batch->columns);
  return paged::attention_form(p).bytes;
}

int ancha_paged_attention(const void* q, int type, size_t rows, size_t heads, size_t ldq, size_t ldqh,
                          const ancha_paged_cache* cache, const ancha_paged_batch* batch, double scale, int causal,
                          size_t window, void* workspace, size_t workspace_bytes, void* out, hipStream_t stream) {
  if (const int s = sticky()) return s;
  const std::string who("ancha_paged_attention");
  if (!is_type(type)) return fail(ANCHA_HIP_INVALID, who + ": unknown type");
  paged::AttentionParams p{};
  if (const int e = check_cache(who, cache, p.cache)) return e;
  if (const int e = check_batch(who, batch, true, true, p.batch)) return e;
  if (heads == 0 || heads % cache->heads)
    return fail(ANCHA_HIP_INVALID, who + ": the heads of q are not a multiple of the cache's");
  // 2^-100 .. 2^100: times log2(e) a normal fp32 number.
  if (!above(scale, 7.9e-31) || scale > 1.2e30)
    return fail(ANCHA_HIP_INVALID, who + ": scale is not a number between 2^-100 and 2^100");
  if (rows == 0) return ANCHA_HIP_OK;
  if (!q || !out) return fail(ANCHA_HIP_INVALID, who + ": null tensor");
  if (rows > kIntMax || heads > 65536 || rows * heads > kIntMax || !strides_fit(rows, ldq, heads, ldqh))
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": too many rows or heads");
  p.type = type;
  p.rows = static_cast<int>(rows);
  p.heads = static_cast<int>(heads);
  const paged::AttentionForm form = paged::attention_form(p);
  // Below HIP's 2^32 threads, up to 512 a workgroup (and few tiles where there are several workgroups a tile).
  if (form.tiles * static_cast<long>(cache->heads) * form.splits >= 1l << 23)
    return fail(ANCHA_HIP_UNSUPPORTED, who + ": too many rows and heads");
  if (workspace_bytes < form.bytes || (form.bytes && (!workspace || !aligned(workspace, 16))))
    return fail(ANCHA_HIP_INVALID, who + ": the workspace is null, too small or not 16-byte aligned");
  if (!ancha_hip_available()) return not_here(who);
  p.q = q;
  p.out = out;
  p.parts = static_cast<float*>(workspace);
  p.ldq = static_cast<long>(ldq);
  p.ldqh = static_cast<long>(ldqh);
  p.causal = causal ? 1 : 0;
  p.window = static_cast<int>(window < kIntMax ? window : 0);
  p.scale = static_cast<float>(scale * 1.4426950408889634);
  p.unscale = 1.f / p.scale;
  const hipError_t e = paged::launch_attention(p, form, stream);
  return e == hipSuccess ? ANCHA_HIP_OK : hip_fail(e, who);
}

// For the tests: how a call is laid out, 3 x splits + its kernel (paged::AttentionForm).
int ancha_amd_paged_form(int type, size_t rows, size_t heads, size_t cache_heads, size_t dim, size_t sequences,
                         size_t keys) {
  paged::AttentionParams p{};
  p.type = type;
  p.rows = static_cast<int>(rows);
  p.heads = static_cast<int>(heads);
  p.cache.heads = static_cast<int>(cache_heads);
  p.cache.dim = static_cast<int>(dim);
  p.batch.sequences = static_cast<int>(sequences);
  p.batch.columns = static_cast<int>((keys + 15) / 16);
  p.cache.shift = 4;
  const paged::AttentionForm f = paged::attention_form(p);
  return 3 * f.splits + f.form;
}

}  // extern "C"
