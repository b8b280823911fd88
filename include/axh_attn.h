/*
 * axh: rotary positions and attention over a paged 4-bit cache on MI355X (gfx950).
 *
 * Same conventions as axh_mx.h: plain device pointers and sizes, an axh_status
 * and axh_last_error(), `stream` NULL for the context's own stream, asynchronous
 * launches, no allocation in any call (axh_rope_table, a set-up call, copies and
 * waits).  Calls with nothing to do return AXH_OK and launch nothing.  Element
 * types are ggml type ids: AXH_GGML_F32, AXH_GGML_F16 or AXH_GGML_BF16.  Strides
 * are in elements, 0 for rows that follow one another, below 2^31; rows that a
 * call takes 16 bytes at a time are 16-byte aligned.  No counterpart in the
 * reference, which has no step that uses a position or a cache.
 */
#ifndef AXH_ATTN_H
#define AXH_ATTN_H

#include "axh_mx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rotary positions --------------------------------------------------------
 * The first `dim` elements of a head are pairs, (2i, 2i + 1) or (i, i + dim / 2);
 * pair i of a token at position p is turned by the angle p * f_i and multiplied by
 * `magnitude`: (a, b) -> (a cos - b sin, a sin + b cos) * magnitude.
 *   f_i = base^(-2i / dim) / factors[i] * (scale * (1 - w_i) + w_i),
 * w_i = extrapolate * (1 - ramp_i): with extrapolate 0 every frequency is scaled
 * (linear interpolation; scale 1: none), with 1 those that turn more than
 * beta_fast times within `original` positions are kept, those that turn less than
 * beta_slow times are scaled, and between them (YaRN)
 *   ramp_i = clamp((i - low) / max(high - low, 0.001), 0, 1),
 *   low, high = floor, ceil of dim ln(original / (2 pi beta)) / (2 ln base) at
 * beta_fast and beta_slow, low at least 0 and high at most dim - 1.
 *   Angles are exact to 2^-32 turns at any position: they are counted in integers,
 * as 64-bit fractions of a turn. */
enum { AXH_ROPE_PAIRS = 0, AXH_ROPE_HALVES = 1 };
typedef struct axh_rope_options {
    uint32_t dim;       /* even, 2 to 1024 */
    uint32_t layout;    /* AXH_ROPE_* */
    double base;        /* above 1 */
    double scale;       /* above 0 */
    double extrapolate; /* 0 to 1 */
    double beta_fast;   /* these three with extrapolate > 0 only */
    double beta_slow;
    uint32_t original;
    float magnitude;
} axh_rope_options;
/* A rotation as the calls take it: its table on the device, dim and layout. */
typedef struct axh_rope {
    const void *table;
    uint32_t dim;
    uint32_t layout;
} axh_rope;
/* Bytes of a table (0 for a dim that is not even, 2 to 1024), and the table of
 * these options (factors: dim / 2 divisors on the host, or NULL), copied to
 * `table` (8-byte aligned) before the call returns. */
uint64_t axh_rope_table_bytes(uint32_t dim);
axh_status axh_rope_table(axh_context *ctx, const axh_rope_options *options, const float *factors,
                          void *table);
/* y = x, n_tokens x n_heads x head_dim of one type, turned by positions[token] (int32,
 * also negative); strides between tokens; elements from dim on are copied.  In place (y
 * == x, equal strides) or apart.  In f32, rounded once.  head_dim at most 1024.  The gradient
 * of x is that of y turned by the negated positions, with the same table. */
axh_status axh_rope_apply(axh_context *ctx, uint32_t x_type, const void *x, uint64_t x_stride,
                          void *y, uint64_t y_stride, const int32_t *positions, uint32_t n_tokens,
                          uint32_t n_heads, uint32_t head_dim, const axh_rope *rope, void *stream);

/* ---- the cache ----------------------------------------------------------------
 * One layer's keys and values in MXFP4 (blocks of 32 along a head), in pages of
 * page_size tokens (a power of two, 16 to 4096), n_pages of them for the keys at k
 * and for the values at v (16-byte aligned), axh_kv_page_bytes() each.  head_dim is
 * a multiple of 32, 32 to 256, and a page of the keys is below 2^31 bytes.  It has, for
 * each head in turn,
 *   keys:    page_size rows of head_dim / 2 bytes of codes, then page_size rows
 *            of head_dim / 32 scale bytes;
 *   values:  for each four tokens, 4 bytes of codes (8 elements) of each of them,
 *            then the next 8 elements, to head_dim; then for each four tokens
 *            their scale bytes of the first block, of the second, and so on.
 * What it holds before it is written does not matter: no row is read beyond a
 * sequence's length.
 *
 * A batch is n_tokens new tokens of n_seqs sequences: sequence s has tokens
 * starts[s] .. starts[s + 1] - 1 (starts NULL: one token each, n_tokens ==
 * n_seqs) and lengths[s] cached tokens with these included, the last of which
 * they are: token j is at position lengths[s] - starts[s + 1] + j.  Position p is
 * row p % page_size of page table[s * max_pages + p / page_size].  All three are
 * int32 on the device, read when the kernels run, so that a graph's replays see
 * what they hold then.  Pages outside 0 .. n_pages - 1 are not there: what would
 * be written to them is left out, and so is what would be read; the same goes for
 * positions below 0 (more tokens than the length) and from max_pages * page_size
 * (below 2^31) on.  Tokens before starts[0] or from starts[n_seqs] on belong to no
 * sequence, and no call touches their rows.  starts must not decrease, from 0 on and up
 * to n_tokens.  A length below 0 is one of 0. */
typedef struct axh_kv_cache {
    void *k;
    void *v;
    uint32_t n_pages;
    uint32_t page_size;
    uint32_t kv_heads;
    uint32_t head_dim;
} axh_kv_cache;
typedef struct axh_kv_batch {
    uint32_t n_seqs;
    uint32_t n_tokens;
    uint32_t max_pages;
    const int32_t *starts;
    const int32_t *lengths;
    const int32_t *table;
} axh_kv_batch;
/* Bytes of a page of keys (of values: the same); 0 for sizes outside the limits. */
uint64_t axh_kv_page_bytes(uint32_t page_size, uint32_t kv_heads, uint32_t head_dim);
/* Writes the batch's rows, k and v (n_tokens x kv_heads x head_dim, strides
 * between tokens), quantised as axh_mxfp4_quantize does; with rope, the keys are
 * turned by their position first, in f32.  Two tokens at one place (a page that two
 * sequences write to) are not ordered. */
axh_status axh_kv_append(axh_context *ctx, uint32_t x_type, const void *k, uint64_t k_stride,
                         const void *v, uint64_t v_stride, const axh_kv_cache *cache,
                         const axh_kv_batch *batch, const axh_rope *rope, void *stream);
/* k and v = the batch's rows as the cache holds them (f32, f16 or bf16, which f32
 * and bf16 hold exactly); 0 for tokens whose page is not there. */
axh_status axh_kv_read(axh_context *ctx, const axh_kv_cache *cache, const axh_kv_batch *batch,
                       uint32_t y_type, void *k, uint64_t k_stride, void *v, uint64_t v_stride,
                       void *stream);

/* ---- attention ------------------------------------------------------------------
 * y[t][h] = sum over keys j of softmax_j(scale * q[t][h] . K[j][g]) V[j][g], g = h /
 * (n_heads / kv_heads), over the cached tokens j of t's sequence with j <= p, t's
 * position, and with window > 0 also j > p - window.  q and y are n_tokens x n_heads x
 * head_dim of one type, strides between tokens; y apart from q.  A row that sees no key, or none
 * whose score is above -inf, is 0.  Keys that a row does not see have no part in
 * it, whatever their bytes; NaN blocks of those that it sees make it NaN.
 *   Scores, maxima and sums are f32 and the output is rounded once.  Scores (scaled) are meant to
 * be below 2^23 ln 2 = 5.8e6 in magnitude, where f32 still tells halves apart in base 2: a
 * row with larger ones may be 0 or NaN.  The matrix instructions
 * multiply bf16 for bf16 and f32 operands, f16 for f16: a cached value is exact in bf16, a
 * q in its own type, an f32 q as three bf16 terms that add up to it.  The softmax's weights
 * are rounded once to bf16 (2^-8) or f16 (2^-11), or are three bf16 terms (2^-24), and the
 * sums are of the rounded weights.  For f16 operands cached values count as f16: those
 * below 2^-14 are rounded to multiples of 2^-24, and a block with values of 2^16 and more
 * (scale bytes above 140) makes the rows that see it infinite or NaN; weights below 2^-32
 * of a row's largest may count as 0.
 *   max_length bounds the lengths as far as the caller knows (0: max_pages *
 * page_size).  With it the keys are split among workgroups; sequences beyond it are
 * computed all the same.  workspace: axh_kv_attention_bytes() for the same cache
 * sizes, batch sizes, options and type, 16-byte aligned (NULL where that is 0), the call's own until it is
 * done: calls that may overlap need one each, and so do graphs that do. */
typedef struct axh_attention_options {
    uint32_t n_heads;    /* a multiple of kv_heads */
    float scale;         /* above 0, below 2.3e38 */
    uint32_t window;     /* 0: none, and so is 2^31 and more */
    uint32_t max_length;
} axh_attention_options;
uint64_t axh_kv_attention_bytes(const axh_kv_cache *cache, const axh_kv_batch *batch,
                                const axh_attention_options *options, uint32_t x_type);
axh_status axh_kv_attention(axh_context *ctx, uint32_t x_type, const void *q, uint64_t q_stride,
                            void *y, uint64_t y_stride, const axh_kv_cache *cache,
                            const axh_kv_batch *batch, const axh_attention_options *options,
                            void *workspace, uint64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* AXH_ATTN_H */
