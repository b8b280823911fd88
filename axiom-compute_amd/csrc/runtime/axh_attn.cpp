// Rotary positions and the paged 4-bit cache over resident device buffers: checks of
// arguments, choice of kernel, grid and launch of the kernels in kv_cache.hip and
// kv_attention.hip.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "axh_attn.h"
#include "axh_internal.h"

using namespace axh;

namespace {

constexpr uint32_t kMaxHeadDim = 256, kMaxRopeDim = 1024;
constexpr uint64_t kMaxStride = 1ull << 31; // elements between tokens
constexpr uint64_t kMaxPage = 1ull << 31;   // bytes of a page of keys
constexpr float kLog2E = 1.44269504088896340736f;
constexpr uint32_t kMaxSplits = 256;        // 64 of a wave of the kernel that joins them

axh_status bad(const char *msg) { return fail(AXH_ERR_INVALID_ARGUMENT, msg); }
bool aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1u)) == 0; }
void *mut(const void *p) { return const_cast<void *>(p); }
uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1u) / b; }

const char *type_name(uint32_t t) {
  switch (t) {
  case AXH_GGML_F32: return "f32";
  case AXH_GGML_F16: return "f16";
  case AXH_GGML_BF16: return "bf16";
  default: return nullptr;
  }
}
uint32_t type_size(uint32_t t) { return t == AXH_GGML_F32 ? 4u : 2u; }

// Rows of `row` elements `stride` apart (0: row), 16-byte aligned.
axh_status check_rows(const char *name, const void *p, uint64_t *stride, uint64_t row,
                      uint32_t n_rows, uint32_t size) {
  if (*stride == 0) *stride = row;
  if (*stride < row || *stride >= kMaxStride)
    return bad((std::string(name) + ": the stride must be at least a row and below 2^31").c_str());
  if (!p) return bad("NULL device pointer");
  if (!aligned(p, 16) || (n_rows > 1 && (*stride * size) % 16u))
    return bad((std::string(name) + ": rows must be 16-byte aligned").c_str());
  return AXH_OK;
}

axh_status check_rope(const axh_rope *r, uint32_t head_dim) {
  if (r->dim < 2u || r->dim % 2u || r->dim > head_dim)
    return bad("a rotation's dim must be even, 2 to head_dim");
  if (r->layout > AXH_ROPE_HALVES) return bad("unknown rotation layout");
  if (!r->table || !aligned(r->table, 8)) return bad("a rotation's table must be 8-byte aligned");
  return AXH_OK;
}

bool cache_sizes(uint32_t page_size, uint32_t kv_heads, uint32_t head_dim) {
  return page_size >= 16u && page_size <= 4096u && (page_size & (page_size - 1u)) == 0 &&
         kv_heads >= 1u && kv_heads <= 65536u && head_dim >= 32u && head_dim <= kMaxHeadDim &&
         head_dim % 32u == 0 &&
         (uint64_t)page_size * kv_heads * (head_dim / 32u) * 17u < kMaxPage;
}

// Sizes only: what a workspace depends on.
axh_status check_sizes(const axh_kv_cache *c, const axh_kv_batch *b) {
  if (!c || !b) return bad("cache or batch is NULL");
  if (!cache_sizes(c->page_size, c->kv_heads, c->head_dim))
    return bad("a cache has pages of 16 to 4096 tokens (a power of two), 1 to 65536 heads, and a "
               "head_dim that is a multiple of 32 up to 256; a page is below 2^31 bytes");
  if (c->n_pages == 0 || c->n_pages >= 1u << 31) return bad("n_pages must be 1 to 2^31 - 1");
  if (b->max_pages == 0 || (uint64_t)b->max_pages * c->page_size >= 1ull << 31)
    return bad("max_pages must be at least 1, and max_pages * page_size below 2^31");
  if (b->n_tokens >= 1u << 31 || b->n_seqs >= 1u << 31) return bad("too many tokens");
  if (!b->starts && b->n_tokens != b->n_seqs)
    return bad("without starts a batch has one token of each sequence");
  return AXH_OK;
}

bool nothing(const axh_kv_batch *b) { return b->n_tokens == 0 || b->n_seqs == 0; }

axh_status check_pointers(const axh_kv_cache *c, const axh_kv_batch *b) {
  if (!c->k || !c->v || !b->lengths || !b->table) return bad("NULL device pointer");
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return bad("a cache must be 16-byte aligned");
  if (!aligned(b->starts, 4) || !aligned(b->lengths, 4) || !aligned(b->table, 4))
    return bad("starts, lengths and table must be 4-byte aligned");
  return AXH_OK;
}

uint32_t log2_of(uint32_t n) {
  uint32_t s = 0;
  while ((1u << s) < n) ++s;
  return s;
}

// Heads that a lane goes through with its token's place and angles: as many as leave 2^least
// lanes.  Rotations 2^18 (4096 x 40 x 128 in bf16 14.4 us, with 2^16 20.5), rows in and out of the
// cache 2^16 (9001 x 4 x 96 in f16, turned, in and out again 13.9 us, with 2^18 19.2: an angle
// takes the time of a head's elements).
uint32_t heads_of_lane(uint64_t units, uint32_t n_heads, uint32_t least) {
  const uint64_t per = std::max<uint64_t>(1u, std::min<uint64_t>(n_heads, units >> least));
  return (uint32_t)div_up(n_heads, div_up(n_heads, per));
}

// ---- attention: the kernel and the split of the keys ----------------------------
// Keep in sync with kv_attention.hip.
struct AttentionPlan {
  const char *kind;
  uint32_t rows;   // query rows of a workgroup
  uint64_t groups; // of them, at most
  uint32_t chunk, splits;
};

AttentionPlan plan_attention(const axh_kv_cache *c, const axh_kv_batch *b,
                             const axh_attention_options *o, uint32_t type) {
  AttentionPlan p{};
  const uint32_t per = o->n_heads / c->kv_heads, dims = (uint32_t)div_up(c->head_dim, 64u);
  const bool f32 = type == AXH_GGML_F32;
  const uint64_t rows = (uint64_t)b->n_tokens * per, seqs = std::max(1u, b->n_seqs);
  const uint64_t mean = div_up(rows, seqs); // of a sequence
  auto most = [&](uint32_t n) { // groups of n rows where each sequence's last one is not full
    return b->starts ? (rows + seqs * (n - 1u)) / n : seqs * div_up(per, n);
  };
  auto expected = [&](uint32_t n) { // workgroups where sequences are equally long
    return std::max<uint64_t>(1u, std::min(most(n), seqs * div_up(mean, n)) * c->kv_heads);
  };
  // 128 rows (which convert a key or a value once for 128 rows, not for 16 or 32, but go through
  // all keys one after the other) where they are full and make 1024 workgroups; 32 rows (heads up
  // to 128 in 16 bits: others have no registers for them) where they make 256.  Times (us) with
  // 32 query and 8 key heads of 128 in bf16, queries to keys, 16 / 32 / 128 rows: 4096 to 4096
  // 210 / 180 / 157; 3000 to 3000 (752 workgroups of 128 rows, three a CU at once, the longest as
  // long as without the others) 127 / 116 / 165; 1024 to 6000 134 / 109 / 146; 256 to 6000 47 /
  // 42 / 143; 128 to 6000 34 / 43 / 142.  4096 to 4096 in f32 440 / - / 470, heads of 256 in bf16
  // 452 / - / 438, in f32 1197 / - / 768.
  if (mean >= 128u && expected(128u) >= 1024u) {
    p.kind = "many";
    p.rows = 128u;
  } else if (!f32 && dims <= 2u && mean > 16u && expected(32u) >= 256u) {
    p.kind = "more";
    p.rows = 32u;
  } else {
    p.kind = "few";
    p.rows = 16u;
  }
  p.groups = most(p.rows);
  const uint64_t capacity = (uint64_t)b->max_pages * c->page_size;
  uint64_t keys = o->max_length ? std::min<uint64_t>(o->max_length, capacity) : capacity;
  if (o->window) keys = std::min<uint64_t>(keys, (uint64_t)o->window + 32u + div_up(p.rows, per));
  // A split's parts are written and read once more, and joined by another launch: nothing is
  // split below 1024 keys (333 keys 6.9 us, in two 10.0; 1000 keys 9.3, in two 10.4), and beyond
  // that into as many as make a workgroup a CU, two where that leaves them over 1024 keys each
  // and three over 2048, as far as registers let a CU have them.  32 sequences of 8192 keys (256
  // workgroups unsplit): 66 us, in two 48, three 44, four 46, eight 47.  One of 131072, 16 heads,
  // f32: in 16 61, in 32 44, in 48 43, in 96 45.  One of 6000, 8 heads, 4 rows: in 8 11.1, in 32
  // 9.7, in 48 10.6; 64 rows: in 4 15.2, in 8 12.6, in 12 14.6.
  uint64_t splits = 1u;
  if (p.rows == 16u && keys >= 1024u) {
    const uint64_t wgs = expected(p.rows), each = keys * wgs / 256u;
    const uint64_t room = f32 ? (dims == 1u ? 3u : dims == 4u ? 1u : 2u) : dims <= 2u ? 3u : 2u;
    const uint64_t a_cu = std::min<uint64_t>(room, each > 2048u ? 3u : each > 1024u ? 2u : 1u);
    splits = std::max<uint64_t>(1u, std::min<uint64_t>(kMaxSplits, 256u * a_cu / wgs));
  }
  p.chunk = (uint32_t)(div_up(div_up(keys, splits), 128u) * 128u);
  p.splits = (uint32_t)div_up(keys, p.chunk);
  return p;
}

axh_status check_attention(const axh_kv_cache *c, const axh_kv_batch *b,
                           const axh_attention_options *o, uint32_t type) {
  axh_status s = check_sizes(c, b);
  if (s != AXH_OK) return s;
  if (!o) return bad("options is NULL");
  if (!type_name(type)) return bad("x_type must be f32, f16 or bf16");
  if (o->n_heads == 0 || o->n_heads % c->kv_heads || o->n_heads > 65536u)
    return bad("n_heads must be a multiple of kv_heads, at most 65536");
  if (!(o->scale > 0.0f) || !std::isfinite(o->scale * kLog2E))
    return bad("scale must be positive, and finite in base 2");
  if ((uint64_t)b->n_tokens * o->n_heads >= 1ull << 31) return bad("too many rows for one call");
  return AXH_OK;
}

uint64_t workspace_bytes_of(const axh_kv_cache *c, const axh_kv_batch *b,
                            const axh_attention_options *o, const AttentionPlan &p) {
  if (p.splits <= 1u || nothing(b)) return 0;
  const uint64_t parts = (uint64_t)b->n_tokens * o->n_heads * p.splits;
  return 4u * ((parts + 1u) / 2u * 4u + parts * c->head_dim);
}

} // namespace

extern "C" {

uint64_t axh_rope_table_bytes(uint32_t dim) {
  if (dim < 2u || dim % 2u || dim > kMaxRopeDim) return 0;
  return (uint64_t)dim / 2u * 8u + 8u;
}

axh_status axh_rope_table(axh_context *ctx, const axh_rope_options *o, const float *factors,
                          void *table) {
  if (!ctx || !o || !table) return bad("NULL argument");
  if (axh_rope_table_bytes(o->dim) == 0) return bad("dim must be even, 2 to 1024");
  if (o->layout > AXH_ROPE_HALVES) return bad("unknown rotation layout");
  if (!aligned(table, 8)) return bad("table must be 8-byte aligned");
  if (!(o->base > 1.0) || !std::isfinite(o->base)) return bad("base must be above 1 and finite");
  if (!(o->scale > 0.0) || !std::isfinite(o->scale)) return bad("scale must be positive and finite");
  if (!(o->extrapolate >= 0.0 && o->extrapolate <= 1.0)) return bad("extrapolate must be 0 to 1");
  if (!std::isfinite(o->magnitude)) return bad("magnitude must be finite");
  const long double two_pi = 6.283185307179586476925286766559L;
  const uint32_t pairs = o->dim / 2u;
  long double low = 0, high = 0;
  if (o->extrapolate > 0.0) {
    if (!(o->beta_fast > 0.0) || !(o->beta_slow > 0.0) || !std::isfinite(o->beta_fast) ||
        !std::isfinite(o->beta_slow) || o->original == 0)
      return bad("extrapolate needs beta_fast, beta_slow and original");
    auto pair_of = [&](double turns) { // the pair that turns so often in the original context
      return o->dim * std::log((long double)o->original / (turns * two_pi)) /
             (2.0L * std::log((long double)o->base));
    };
    low = std::max(0.0L, std::floor(pair_of(o->beta_fast)));
    high = std::min((long double)o->dim - 1.0L, std::ceil(pair_of(o->beta_slow)));
  }
  uint8_t host[kMaxRopeDim / 2u * 8u + 8u] = {};
  for (uint32_t i = 0; i < pairs; ++i) {
    long double f = std::pow((long double)o->base, -2.0L * i / o->dim);
    if (factors) {
      if (!(factors[i] > 0.0f) || !std::isfinite(factors[i]))
        return bad("factors must be positive and finite");
      f /= factors[i];
    }
    long double w = 0.0L;
    if (o->extrapolate > 0.0) {
      const long double r = (i - low) / std::max(0.001L, high - low);
      w = o->extrapolate * (1.0L - std::min(1.0L, std::max(0.0L, r)));
    }
    f *= o->scale * (1.0L - w) + w;
    const long double turns = f / two_pi;
    // the fraction of a turn in 64 bits (a whole turn is none)
    const long double bits = std::round((turns - std::floor(turns)) * 18446744073709551616.0L);
    const uint64_t u = bits >= 18446744073709551616.0L ? 0u : (uint64_t)bits;
    std::memcpy(host + 8u * i, &u, 8);
  }
  std::memcpy(host + 8u * pairs, &o->magnitude, 4);
  return axh_upload(ctx, table, host, axh_rope_table_bytes(o->dim));
}

axh_status axh_rope_apply(axh_context *ctx, uint32_t x_type, const void *x, uint64_t x_stride,
                          void *y, uint64_t y_stride, const int32_t *positions, uint32_t n_tokens,
                          uint32_t n_heads, uint32_t head_dim, const axh_rope *rope, void *stream) {
  if (!ctx) return bad("ctx is NULL");
  const char *type = type_name(x_type);
  if (!type) return bad("x_type must be f32, f16 or bf16");
  if (head_dim < 2u || head_dim > kMaxRopeDim) return bad("head_dim must be 2 to 1024");
  if (n_heads > 65536u) return bad("n_heads must be at most 65536");
  if (!rope) return bad("rope is NULL");
  axh_status s = check_rope(rope, head_dim);
  if (s != AXH_OK) return s;
  const uint64_t row = (uint64_t)n_heads * head_dim;
  if (x_stride == 0) x_stride = row;
  if (y_stride == 0) y_stride = row;
  if (x_stride < row || y_stride < row || x_stride >= kMaxStride || y_stride >= kMaxStride)
    return bad("strides must be at least a row and below 2^31");
  if (n_tokens == 0 || n_heads == 0) return ok();
  if (!x || !y || !positions) return bad("NULL device pointer");
  const uint32_t size = type_size(x_type);
  if (!aligned(x, size) || !aligned(y, size) || !aligned(positions, 4))
    return bad("operands must be aligned to their elements");
  if (x == y && x_stride != y_stride) return bad("in place, the strides must be equal");
  // Whole 16-byte pieces, or one pair at a time where rows or the rotated part are not of
  // them.
  const bool wide = aligned(x, 16) && aligned(y, 16) && head_dim % 8u == 0 && rope->dim % 16u == 0 &&
                    (n_tokens == 1u || ((x_stride * size) % 16u == 0 && (y_stride * size) % 16u == 0));
  const uint32_t turned = rope->layout == AXH_ROPE_HALVES
                              ? rope->dim / (wide ? 16u : 2u)
                              : rope->dim / (wide ? 8u : 2u);
  const uint32_t rest = x == y ? 0u : (head_dim - rope->dim) / (wide ? 8u : 1u);
  const uint32_t units = turned + rest;
  const uint32_t per = heads_of_lane((uint64_t)n_tokens * units * n_heads, n_heads, 18u);
  const uint64_t groups = div_up(n_heads, per);
  const uint32_t words[] = {n_tokens, n_heads,   head_dim, (uint32_t)x_stride, (uint32_t)y_stride,
                            rope->dim, rope->layout, units, per, (uint32_t)groups};
  void *bufs[] = {mut(x), y, mut(positions), mut(rope->table)};
  return mx_launch(ctx, kKvCache, std::string("axh_rope_") + (wide ? "wide_" : "single_") + type,
                   div_up((uint64_t)n_tokens * groups * units, 256u), 1, 256, 0, bufs, 4, words, 10,
                   stream);
}

uint64_t axh_kv_page_bytes(uint32_t page_size, uint32_t kv_heads, uint32_t head_dim) {
  if (!cache_sizes(page_size, kv_heads, head_dim)) return 0;
  return (uint64_t)page_size * kv_heads * (head_dim / 32u) * 17u;
}

axh_status axh_kv_append(axh_context *ctx, uint32_t x_type, const void *k, uint64_t k_stride,
                         const void *v, uint64_t v_stride, const axh_kv_cache *cache,
                         const axh_kv_batch *batch, const axh_rope *rope, void *stream) {
  if (!ctx) return bad("ctx is NULL");
  const char *type = type_name(x_type);
  if (!type) return bad("x_type must be f32, f16 or bf16");
  axh_status s = check_sizes(cache, batch);
  if (s == AXH_OK && rope) s = check_rope(rope, cache->head_dim);
  if (s != AXH_OK) return s;
  if (nothing(batch)) return ok();
  const uint64_t row = (uint64_t)cache->kv_heads * cache->head_dim;
  s = check_rows("k", k, &k_stride, row, batch->n_tokens, type_size(x_type));
  if (s == AXH_OK) s = check_rows("v", v, &v_stride, row, batch->n_tokens, type_size(x_type));
  if (s == AXH_OK) s = check_pointers(cache, batch);
  if (s != AXH_OK) return s;
  const uint32_t units = cache->head_dim / 8u;
  const uint32_t per =
      heads_of_lane((uint64_t)batch->n_tokens * units * cache->kv_heads, cache->kv_heads, 16u);
  const uint64_t groups = div_up(cache->kv_heads, per);
  const uint32_t words[] = {batch->n_tokens, batch->n_seqs, batch->max_pages, cache->n_pages,
                            log2_of(cache->page_size), cache->kv_heads, cache->head_dim,
                            (uint32_t)k_stride, (uint32_t)v_stride, rope ? rope->dim : 0u,
                            rope ? rope->layout : 0u, per, (uint32_t)groups};
  void *bufs[] = {mut(k), mut(v), cache->k, cache->v, mut(batch->starts), mut(batch->lengths),
                  mut(batch->table), rope ? mut(rope->table) : nullptr};
  return mx_launch(ctx, kKvCache, std::string("axh_kv_append_") + type,
                   div_up((uint64_t)batch->n_tokens * groups * units, 256u), 2, 256, 0, bufs, 8,
                   words, 13, stream);
}

axh_status axh_kv_read(axh_context *ctx, const axh_kv_cache *cache, const axh_kv_batch *batch,
                       uint32_t y_type, void *k, uint64_t k_stride, void *v, uint64_t v_stride,
                       void *stream) {
  if (!ctx) return bad("ctx is NULL");
  const char *type = type_name(y_type);
  if (!type) return bad("y_type must be f32, f16 or bf16");
  axh_status s = check_sizes(cache, batch);
  if (s != AXH_OK) return s;
  if (nothing(batch)) return ok();
  const uint64_t row = (uint64_t)cache->kv_heads * cache->head_dim;
  s = check_rows("k", k, &k_stride, row, batch->n_tokens, type_size(y_type));
  if (s == AXH_OK) s = check_rows("v", v, &v_stride, row, batch->n_tokens, type_size(y_type));
  if (s == AXH_OK) s = check_pointers(cache, batch);
  if (s != AXH_OK) return s;
  const uint32_t units = cache->head_dim / 8u;
  const uint32_t per =
      heads_of_lane((uint64_t)batch->n_tokens * units * cache->kv_heads, cache->kv_heads, 16u);
  const uint64_t groups = div_up(cache->kv_heads, per);
  const uint32_t words[] = {batch->n_tokens, batch->n_seqs, batch->max_pages, cache->n_pages,
                            log2_of(cache->page_size), cache->kv_heads, cache->head_dim,
                            (uint32_t)k_stride, (uint32_t)v_stride, per, (uint32_t)groups};
  void *bufs[] = {cache->k, cache->v, mut(batch->starts), mut(batch->lengths), mut(batch->table),
                  k, v};
  return mx_launch(ctx, kKvCache, std::string("axh_kv_read_") + type,
                   div_up((uint64_t)batch->n_tokens * groups * units, 256u), 2, 256, 0, bufs, 7,
                   words, 11, stream);
}

uint64_t axh_kv_attention_bytes(const axh_kv_cache *cache, const axh_kv_batch *batch,
                                const axh_attention_options *options, uint32_t x_type) {
  if (check_attention(cache, batch, options, x_type) != AXH_OK) return 0;
  return workspace_bytes_of(cache, batch, options, plan_attention(cache, batch, options, x_type));
}

axh_status axh_kv_attention(axh_context *ctx, uint32_t x_type, const void *q, uint64_t q_stride,
                            void *y, uint64_t y_stride, const axh_kv_cache *cache,
                            const axh_kv_batch *batch, const axh_attention_options *options,
                            void *workspace, uint64_t workspace_bytes, void *stream) {
  if (!ctx) return bad("ctx is NULL");
  axh_status s = check_attention(cache, batch, options, x_type);
  if (s != AXH_OK) return s;
  if (nothing(batch)) return ok();
  const uint64_t row = (uint64_t)options->n_heads * cache->head_dim;
  s = check_rows("q", q, &q_stride, row, batch->n_tokens, type_size(x_type));
  if (s == AXH_OK) s = check_rows("y", y, &y_stride, row, batch->n_tokens, type_size(x_type));
  if (s == AXH_OK) s = check_pointers(cache, batch);
  if (s != AXH_OK) return s;
  const AttentionPlan p = plan_attention(cache, batch, options, x_type);
  const uint64_t need = workspace_bytes_of(cache, batch, options, p);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return bad("the workspace must be 16-byte aligned and axh_kv_attention_bytes() long");
  const std::string type = type_name(x_type);
  const float c = options->scale * kLog2E;
  uint32_t c_bits;
  std::memcpy(&c_bits, &c, 4);
  // (positions are below 2^31)
  const uint32_t window = options->window >= 1u << 31 ? 0u : options->window;
  const uint32_t words[] = {batch->n_seqs, batch->n_tokens, batch->max_pages, cache->n_pages,
                            log2_of(cache->page_size), cache->kv_heads, cache->head_dim,
                            options->n_heads / cache->kv_heads, (uint32_t)q_stride,
                            (uint32_t)y_stride, c_bits, window, p.chunk, p.splits,
                            (uint32_t)axh_kv_page_bytes(cache->page_size, cache->kv_heads,
                                                        cache->head_dim)};
  void *bufs[] = {mut(q), cache->k, cache->v, mut(batch->starts), mut(batch->lengths),
                  mut(batch->table), y, workspace};
  s = mx_launch(ctx, kKvAttention,
                std::string("axh_kv_attention_") + p.kind + "_d" +
                    std::to_string(div_up(cache->head_dim, 64u) * 64u) + "_" + type,
                p.groups * p.splits * cache->kv_heads, 1, 256, 0, bufs, 8, words, 15, stream);
  if (s != AXH_OK || p.splits <= 1u) return s;
  const uint32_t join[] = {batch->n_tokens, batch->n_seqs, options->n_heads, cache->head_dim,
                           (uint32_t)y_stride, p.splits};
  void *joined[] = {workspace, mut(batch->starts), y};
  // Four waves a row where its parts are more than a wave reads at once.
  const uint64_t all = (uint64_t)batch->n_tokens * options->n_heads;
  const uint32_t per = p.splits > 8u ? 4u : 1u;
  const uint32_t across = cache->head_dim > 128u ? 256u : cache->head_dim > 64u ? 128u : 64u;
  return mx_launch(ctx, kKvAttention,
                   "axh_kv_combine_w" + std::to_string(per) + "_d" + std::to_string(across) + "_" +
                       type,
                   div_up(all * per, 4u), 1, 256, 0, joined, 3, join, 6, stream);
}

} // extern "C"
