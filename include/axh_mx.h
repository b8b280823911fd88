/*
 * axh: microscaled 4-bit floats (MXFP4) and expert layers on MI355X (gfx950).
 *
 * Same conventions as axh.h: plain device pointers and sizes, an axh_status and
 * axh_last_error(), `stream` NULL for the context's own stream, asynchronous
 * launches, no allocation in any call.  Calls with nothing to do (no rows, no
 * tokens) return AXH_OK and launch nothing.  No counterpart in the reference,
 * whose formats are Q4_0 and Q4_K.
 *
 * MXFP4 (OCP Microscaling Formats v1.0): 32 consecutive elements of a row share
 * an E8M0 scale byte e, the factor 2^(e - 127) (255: the block is NaN); an
 * element is an E2M1 code, in order of code 0, 0.5, 1, 1.5, 2, 3, 4, 6 and the
 * same with the sign bit (8) set.  A rows x cols matrix (cols a multiple of 32,
 * at most 2^22) is two arrays: codes, rows x cols / 2 bytes, the even element in
 * the low nibble, 16-byte aligned; and scales, rows x cols / 32 bytes, of any
 * alignment.  A call quantises, decodes or unpacks at most 2^30 - 64 blocks of 32,
 * and sums up the choices of at most 2^24 - 1 tokens.  Element types of other
 * operands are ggml type ids: AXH_GGML_F32, AXH_GGML_F16 or AXH_GGML_BF16, and
 * AXH_GGML_MXFP4 where it is said.
 */
#ifndef AXH_MX_H
#define AXH_MX_H

#include "axh.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ggml's id of MXFP4 tensors: 17-byte blocks of 32 elements (the scale byte,
 * then 16 bytes with elements 0-15 in the low and 16-31 in the high nibbles). */
enum { AXH_GGML_MXFP4 = 39 };

/* ---- quantisation -----------------------------------------------------------
 * codes / scales = MXFP4 of x (f32, f16 or bf16; rows x cols, x_stride elements
 * between rows, 0 for cols; rows 16-byte aligned).  The scale of a block is
 * 2^(floor(log2 m) - 2), m its largest magnitude, no less than 2^-127; elements
 * are rounded to nearest, ties to even, and magnitudes above 6 become 6.  A
 * block with an infinity or a NaN gets scale byte 255 and codes 0; one of zeros
 * gets scale byte 0, its codes keep the signs. */
axh_status axh_mxfp4_quantize(axh_context *ctx, uint32_t x_type, const void *x, uint64_t x_stride,
                              void *codes, void *scales, uint32_t rows, uint32_t cols,
                              void *stream);
/* w = the 32 * n_blocks values that codes / scales stand for, as f32, f16 or
 * bf16 (exact in f32 and bf16 up to the largest value; f16 rounds what is
 * outside its range).  codes 4-byte and w 16-byte aligned. */
axh_status axh_mxfp4_dequant(axh_context *ctx, const void *codes, const void *scales,
                             uint32_t w_type, void *w, uint64_t n_blocks, void *stream);
/* codes / scales of n_blocks ggml MXFP4 blocks (a tensor of a GGUF file, see
 * axh_gguf_upload_tensor), which a program does once when it loads a model. */
axh_status axh_mxfp4_unpack_ggml(axh_context *ctx, const void *q, void *codes, void *scales,
                                 uint64_t n_blocks, void *stream);

/* ---- products ---------------------------------------------------------------
 * Single token: y[r] = sum_k W[r][k] * x[k] with f32 x (16-byte aligned), y. */
axh_status axh_mxfp4_matvec(axh_context *ctx, const void *codes, const void *scales,
                            const float *x, float *y, uint32_t n_rows, uint32_t cols,
                            void *stream);
/* Batches and prompts: y[b * n_rows + r] = sum_k W[r][k] * X[b][k], both in
 * MXFP4 (X batch x cols, from axh_mxfp4_quantize), accumulated in f32 on the
 * scaled matrix instructions; y f32, f16 or bf16, rounded once. */
axh_status axh_mxfp4_matmul(axh_context *ctx, const void *w_codes, const void *w_scales,
                            const void *x_codes, const void *x_scales, uint32_t y_type, void *y,
                            uint32_t n_rows, uint32_t cols, uint32_t batch, void *stream);
/* Name of the kernel that axh_mxfp4_matmul launches (no device work). */
axh_status axh_mxfp4_matmul_kernel_name(uint32_t n_rows, uint32_t cols, uint32_t batch,
                                        uint32_t y_type, char *buf, size_t cap);

/* ---- routing ---------------------------------------------------------------- */
/* The router's product: logits[t * n_experts + e] = sum_k W[e][k] * x[t][k], W (n_experts x
 * cols) f32, f16 or bf16, x (n_tokens x cols) and logits f32, products and sums in f32 for
 * any number of tokens (their order depends on it).  w and x 16-byte aligned, cols a
 * multiple of 32, n_experts <= 1024. */
axh_status axh_expert_logits(axh_context *ctx, uint32_t w_type, const void *w, const float *x,
                             float *logits, uint32_t n_experts, uint32_t cols, uint32_t n_tokens,
                             void *stream);
/* Choices and weights of n_tokens tokens from their router logits (f32, f16 or
 * bf16, n_tokens x n_experts).  The score of an expert is the softmax over the
 * token's logits or the sigmoid of its logit; the order is by key, the score
 * plus the expert's bias (f32, NULL for none), the lowest expert first among
 * equals.  With groups (n_groups > 1, dividing n_experts, at most 64), a
 * group's key is its best key or the sum of its two best (group_best 1, or 2 in
 * groups of at least two experts), the groups_kept best groups are kept, and
 * choices come from them only.  The weight of a choice is its score, without the
 * bias, divided by the sum over the token's choices where normalize is set, times
 * scale.
 *   Scores are f32 (a sigmoid below its range is 0; choices whose scores add up
 * to 0 have weight 0).  Keys are compared as f32; where only the order of single scores counts (no
 * bias, and one group or group_best 1) the logits themselves are compared.
 *   Logits of -inf (masked experts) and NaN are never chosen: a token with
 * fewer candidates than top_k ends in experts of -1 with weight 0.  A group
 * with fewer than group_best candidates has key -inf.  Logits of +inf share a
 * softmax's weight.
 * experts: n_tokens x top_k int32, weights: n_tokens x top_k f32, both in
 * descending order of key.  Limits: n_experts <= 1024, top_k <= 64. */
enum { AXH_SCORE_SOFTMAX = 0, AXH_SCORE_SIGMOID = 1 };
typedef struct axh_route_options {
    uint32_t n_experts;
    uint32_t top_k;
    uint32_t score;       /* AXH_SCORE_* */
    uint32_t n_groups;    /* 0 or 1: none */
    uint32_t groups_kept;
    uint32_t group_best;  /* 1 or 2 */
    uint32_t normalize;
    float scale;
} axh_route_options;
axh_status axh_expert_route(axh_context *ctx, uint32_t logits_type, const void *logits,
                            const float *bias, int32_t *experts, float *weights,
                            uint32_t n_tokens, const axh_route_options *options, void *stream);

/* ---- expert layers ------------------------------------------------------------
 * experts: n_tokens x top_k int32 as from axh_expert_route; choice k of token t
 * is slot t * top_k + k.  Choices outside 0 .. n_experts - 1 are left out.  The
 * experts' matrices follow one another (n_experts x n_rows x cols), each below
 * 2 GiB of codes.  silu(g) * u is within 3 ulp, 0 from g = -88.72 down, for few
 * tokens, and within 5 ulp, 0 from g = -87.3 down, for prompts.
 *
 * Few tokens, f32 activations, every chosen expert's weights read once a slot:
 *   gate_up: h[slot] = silu(Wg[e] x[t]) * (Wu[e] x[t]), slots x n_rows f32 (0
 *            for choices left out);
 *   down:    y[t] = sum over choices of weight * (Wd[e] h[slot]), n_tokens x
 *            n_rows f32.  x and h 16-byte aligned.  n_tokens * top_k <= 65535. */
axh_status axh_mxfp4_expert_gate_up(axh_context *ctx, const void *gate_codes,
                                    const void *gate_scales, const void *up_codes,
                                    const void *up_scales, const float *x, const int32_t *experts,
                                    float *h, uint32_t n_rows, uint32_t cols, uint32_t n_tokens,
                                    uint32_t top_k, uint32_t n_experts, void *stream);
axh_status axh_mxfp4_expert_down(axh_context *ctx, const void *codes, const void *scales,
                                 const float *h, const int32_t *experts, const float *weights,
                                 float *y, uint32_t n_rows, uint32_t cols, uint32_t n_tokens,
                                 uint32_t top_k, uint32_t n_experts, void *stream);
/* Prompts.  The plan is the slots in order of their experts, made on the device
 * for one set of choices and used by the products below: offsets[n_experts + 1]
 * (u32; padded to a multiple of 16 words), then the slots (u32), expert e's
 * from offsets[e] to offsets[e + 1], ascending.  plan: 4-byte aligned,
 * axh_expert_plan_bytes() long.  n_experts <= 1024. */
uint64_t axh_expert_plan_bytes(uint32_t n_tokens, uint32_t top_k, uint32_t n_experts);
axh_status axh_expert_plan(axh_context *ctx, const int32_t *experts, void *plan, uint32_t n_tokens,
                           uint32_t top_k, uint32_t n_experts, void *stream);
/* h[slot] = silu(Wg[e] x[t]) * (Wu[e] x[t]) with MXFP4 x (n_tokens x cols).
 * h: slots x n_rows of f32, f16 or bf16 (h_scales unused), or AXH_GGML_MXFP4:
 * codes in h and scales in h_scales, quantised as axh_mxfp4_quantize does from
 * the f32 results (n_rows a multiple of 32).  Slots left out are not written. */
axh_status axh_mxfp4_expert_gate_up_matmul(axh_context *ctx, const void *gate_codes,
                                           const void *gate_scales, const void *up_codes,
                                           const void *up_scales, const void *x_codes,
                                           const void *x_scales, const void *plan, uint32_t h_type,
                                           void *h, void *h_scales, uint32_t n_rows, uint32_t cols,
                                           uint32_t n_tokens, uint32_t top_k, uint32_t n_experts,
                                           void *stream);
/* y[slot] = W[e] h[slot] with MXFP4 h (slots x cols); y slots x n_rows of f32,
 * f16 or bf16.  Slots left out are not written. */
axh_status axh_mxfp4_expert_matmul(axh_context *ctx, const void *codes, const void *scales,
                                   const void *h_codes, const void *h_scales, const void *plan,
                                   uint32_t y_type, void *y, uint32_t n_rows, uint32_t cols,
                                   uint32_t n_tokens, uint32_t top_k, uint32_t n_experts,
                                   void *stream);
/* y[t] = sum over choices of weight * slots[slot], in f32 in the choices'
 * order, rounded once; slots and y of one type (f32, f16 or bf16), both 16-byte
 * aligned.  Slots of 16 bits were rounded once more when they were written: in
 * bf16 the error of y is 0.0024 by norm, 0.0017 for f32 slots whose sum is then
 * rounded.  n_experts 0 leaves out negative choices only. */
axh_status axh_expert_combine(axh_context *ctx, uint32_t y_type, const void *slots,
                              const int32_t *experts, const float *weights, void *y,
                              uint32_t n_rows, uint32_t n_tokens, uint32_t top_k,
                              uint32_t n_experts, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* AXH_MX_H */
