// MXFP4 operations and expert layers over resident device buffers: checks of
// arguments, choice of kernel, grid and launch of the kernels in mx_elem.hip,
// mx_matvec.hip and mx_matmul.hip.
#include <algorithm>
#include <cstdio>
#include <cstring>
#include <string>
#include <utility>

#include "axh_internal.h"
#include "axh_mx.h"

extern "C" const unsigned char axh_mx_elem_co_begin[], axh_mx_elem_co_end[];
extern "C" const unsigned char axh_mx_matvec_co_begin[], axh_mx_matvec_co_end[];
extern "C" const unsigned char axh_mx_matmul_co_begin[], axh_mx_matmul_co_end[];
extern "C" const unsigned char axh_kv_cache_co_begin[], axh_kv_cache_co_end[];
extern "C" const unsigned char axh_kv_attention_co_begin[], axh_kv_attention_co_end[];

namespace axh {

bool mx_code_object(uint32_t i, const void **co, size_t *bytes) {
  const unsigned char *objs[kMxObjects][2] = {
      {axh_mx_elem_co_begin, axh_mx_elem_co_end},
      {axh_mx_matvec_co_begin, axh_mx_matvec_co_end},
      {axh_mx_matmul_co_begin, axh_mx_matmul_co_end},
      {axh_kv_cache_co_begin, axh_kv_cache_co_end},
      {axh_kv_attention_co_begin, axh_kv_attention_co_end}};
  if (i >= kMxObjects) return false;
  *co = objs[i][0];
  *bytes = (size_t)(objs[i][1] - objs[i][0]);
  return true;
}

namespace {

constexpr MxObject kElem = kMxElem, kMatvec = kMxMatvec, kMatmul = kMxMatmul;

constexpr uint32_t kMaxCols = 1u << 22;    // the tiles' row offsets stay below 1 GiB
constexpr uint64_t kMaxBuffer = 1ull << 31; // bytes of a buffer of the products' kernels
constexpr uint32_t kMaxExperts = 1024, kMaxTopK = 64, kMaxGroups = 64;

axh_status bad(const char *msg) { return fail(AXH_ERR_INVALID_ARGUMENT, msg); }

bool aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1u)) == 0; }

const char *type_name(uint32_t t) {
  switch (t) {
  case AXH_GGML_F32: return "f32";
  case AXH_GGML_F16: return "f16";
  case AXH_GGML_BF16: return "bf16";
  default: return nullptr;
  }
}

axh_status check_cols(uint32_t cols) {
  if (cols == 0 || cols % 32u || cols > kMaxCols)
    return bad("cols must be a multiple of 32, from 32 to 2^22");
  return AXH_OK;
}

// (the launches of this file)
template <class... A> axh_status launch(A &&...args) { return mx_launch(std::forward<A>(args)...); }

uint32_t div_up(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1u) / b); }

void *mut(const void *p) { return const_cast<void *>(p); }

// ---- single-token products ----------------------------------------------------
// Lanes of a row (see mx_matvec.hip), waves of a group, groups and batches.
struct MatvecPlan {
  uint32_t lanes, uw, groups, batches, group_rows, lds;
  uint64_t wgs;
};

// `picks`: units of the summed axis beside the row's own (down: choices);
// `loads`: load instructions of a batch, shared by `mats` matrices; `items`:
// workgroups along y.
//   A workgroup has 4 waves (or a wave for each unit, up to 8) where that makes
// 256 workgroups of two batches, else one group.  Four batches where they make
// one round of workgroups: 14336 x 4096 8.86 us against 9.07 with two, 8192 x
// 8192 9.94 / 10.29, but 128256 x 4096 49.3 / 46.7 (fewer, and 4096 x 14336
// 11.98 / 9.44).
MatvecPlan plan_matvec(uint32_t n_rows, uint32_t nblk, uint32_t picks, uint32_t loads,
                       uint32_t mats, uint32_t items) {
  MatvecPlan p{};
  p.lanes = nblk <= 16u ? 16u : nblk <= 32u ? 32u : 64u;
  const uint64_t units = (uint64_t)picks * (p.lanes == 64u ? div_up(nblk, 64u) : 1u);
  p.uw = (uint32_t)std::min<uint64_t>(units, 8u);
  const uint32_t batch_rows = loads * (64u / p.lanes) / mats;
  const uint64_t batches = (uint64_t)div_up(n_rows, batch_rows) * items;
  p.groups = (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>(4u / p.uw, batches / 512u));
  auto grid = [&](uint32_t b) {
    return (uint64_t)div_up(n_rows, (uint64_t)p.groups * b * batch_rows) * items;
  };
  p.batches = grid(4) >= 200u && grid(4) <= 512u ? 4u : 2u;
  p.group_rows = p.batches * batch_rows;
  p.wgs = div_up(n_rows, (uint64_t)p.groups * p.group_rows);
  p.lds = p.groups * p.uw * (p.lanes * 128u + p.group_rows * mats * 4u);
  return p;
}

// ---- matmul kernels -----------------------------------------------------------
// A kind's tile and launch; keep in sync with mx_matmul.hip.
struct MatmulKind {
  const char *name;
  uint32_t rows, cols; // a workgroup's outputs (gate/up: half of the rows)
  uint32_t threads, lds;
};
constexpr MatmulKind k256x256 = {"t256x256", 256, 256, 512, 147456};
constexpr MatmulKind k128x128 = {"t128x128", 128, 128, 256, 73728};
constexpr MatmulKind k128x128Short = {"t128x128n", 128, 128, 256, 73728};
constexpr MatmulKind k128x64 = {"t128x64", 128, 64, 256, 81920};
constexpr MatmulKind k64x128 = {"t64x128", 64, 128, 256, 81920};
constexpr MatmulKind k64x64 = {"t64x64", 64, 64, 128, 53248};
constexpr MatmulKind k64x64s2 = {"t64x64s2", 64, 64, 256, 106496};
constexpr MatmulKind kSplit32 = {"k32", 32, 32, 512, 131072};
constexpr MatmulKind kSplit32GateUp = {"k32", 64, 32, 256, 147456};
constexpr MatmulKind kSplit16 = {"k16", 16, 32, 512, 147456};
constexpr uint32_t kTileMinBlocks = 16; // the tiles read 16 scales of a row at once

// The largest tile that gives most of the 256 CUs one (and is not mostly empty): a
// larger one reads less, but what has no tile waits.  14336 x 4096, us: 1024 columns
// 256x256 45.2, 128x128 58.6; 512 columns 34.3 (112 tiles), 31.9; 256 columns 128x128
// 20.9, 64x128 22.3, 64x64 28.3.  64x128 where 64x64 would give more than one round:
// 5001 x 5408, 256 columns, 15.5 against 17.8; 8192 x 8192, 128 columns (128 tiles), 21.6
// against 16.1.  A round of 64x64 has its K axis shared by two groups of waves, more
// rounds not: 14336 x 4096, 32 columns, 10.2 against 11.2; 28672 x 8192, 32 columns, 32.0
// against 30.0.  The K-split kernel where its tiles are one round too: 4096 x 4096, 64
// columns, 6.6 against 7.1; 128 columns (512 tiles) 12.3 against 7.7; with half the rows
// if K is long and those fit as well: 4096 x 14336, 32 columns, 13.9 against 16.3; 4096 x
// 4096 7.6 against 6.6.
// Rows of fewer than 16 blocks: the K-split kernel where its tiles are one round, else 128x128.
// bf16 y, us, K-split / 128x128: 1536 x 256, 128 columns (192 tiles) 3.5 / 4.2, 256 columns
// (384) 5.7 / 4.3, 2000 columns 27.9 / 5.1; 8192 x 480, 32 columns (256) 3.7 / 4.0, 64 columns
// (512) 6.1 / 4.4; 16384 x 32, 16 columns (512) 4.4 / 4.1; 32 x 480, 4096 columns (128) 3.6 /
// 4.2; 2880 x 32, 128 columns (360) 4.5 / 4.3.
const MatmulKind &dense_kind(uint32_t n_rows, uint32_t nblk, uint32_t batch) {
  auto grid = [&](const MatmulKind &k) {
    return (uint64_t)div_up(n_rows, k.rows) * div_up(batch, k.cols);
  };
  if (nblk < kTileMinBlocks) // (a load of 16 scales has to stay inside both arrays)
    return batch >= 16u && n_rows >= 16u && grid(kSplit32) > 256u ? k128x128Short : kSplit32;
  if (batch > 128u && grid(k256x256) >= 200u) return k256x256;
  if (batch > 64u && grid(k128x128) >= 200u) return k128x128;
  if (batch > 64u && grid(k64x64) > 256u) return k64x128;
  if (grid(kSplit32) <= 256u) return nblk >= 320u && grid(kSplit16) <= 256u ? kSplit16 : kSplit32;
  return grid(k64x64) <= 256u ? k64x64s2 : k64x64;
}

// By the mean number of columns of an expert: tiles of 64 columns while most experts
// have one of them, of 256 where an expert's outputs are many, so that such tiles are
// mostly full and still many.  Gate and up / down, us.  40 experts, 1312 x 736, mean 50:
// 128x64 15.7 / 10.4, 128x128 18.8 / 12.4.  64 experts, 2048 x 1408: mean 32: 46.5 / 27.1,
// 55.9 / 29.5; mean 64: 58.7 / 38.1, 57.5 / 33.3.  128x128 and 256x256: 64 experts, 2048 x
// 1408, mean 256: down 70.3, 63.0; mean 512: 188 / 115, 165 / 105; 32 experts, 2048 x
// 1024, mean 256: 47.8 / 32.5, 53 / 33.2; mean 512: 77 / 49.5, 71 / 48; 2880 x 2880, mean
// 256: 190 / 90, 167 / 95; 8 experts, 4096 x 14336, mean 75: 124 / 65, 167 / 97; mean 175:
// 234 / 89, 174 / 92.
// Rows of fewer than 16 blocks, through 128x128 against the K-split kernel, a layer of us:
// 2894 tokens, 6 of 34 experts, 1536 x 352: 75.5 / 416; 3639 tokens, 7 of 72, 2048 x 256:
// 110 / 838; 30 experts, 2048 x 480, mean 4: 24 / 41, mean 60: 32 / 88; 64, 1536 x 256,
// mean 4: 26 / 52, mean 60: 38 / 122.
const MatmulKind &expert_kind(uint32_t n_rows, uint32_t nblk, uint64_t slots, uint32_t n_experts,
                              uint32_t n_x, bool gate_up) {
  const uint64_t mean = slots / n_experts;
  if (nblk < kTileMinBlocks) { // (a load of 16 scales has to stay inside both arrays)
    if (n_rows >= 16u && n_x >= 16u) return k128x128Short;
    return gate_up ? kSplit32GateUp : kSplit32;
  }
  if (mean <= 52u) return k128x64;
  return mean >= 160u && mean * n_rows >= 1u << 19 ? k256x256 : k128x128;
}

// The router's product: a wave a logit up to 6144 logits (256 experts, 7168 columns, us: 16
// tokens 9.3 against 13.6 with tiles of 16 x 16, 32 tokens 17.2 against 14.0; 4096 columns
// 5.2 / 8.1 and 9.0 / 8.4), then the largest tile that most of the CUs get one of: 7168
// columns, 333 tokens, 16 x 16 25.6 and 32 x 32 43.9 (88 tiles), 1024 tokens 54.9 / 48.2;
// 2048 tokens, 32 x 32 86.9 and 64 x 64 126.7 (128 tiles), 4096 tokens 170.9 / 135.9.
constexpr uint32_t kFewLogits = 6144, kLogitTiles = 200;

// Shared checks of the expert products for prompts.
axh_status check_experts(axh_context *ctx, uint32_t n_rows, uint32_t cols, uint32_t n_tokens,
                         uint32_t top_k, uint32_t n_experts) {
  if (!ctx) return bad("ctx is NULL");
  axh_status s = check_cols(cols);
  if (s != AXH_OK) return s;
  if (n_experts == 0 || n_experts > kMaxExperts) return bad("n_experts must be 1 to 1024");
  if (top_k == 0 || top_k > kMaxTopK) return bad("top_k must be 1 to 64");
  if ((uint64_t)n_tokens * top_k >= kMaxBuffer) return bad("too many slots");
  if ((uint64_t)n_rows * (cols / 2u) >= kMaxBuffer) return bad("an expert's matrix must be below 2 GiB");
  return AXH_OK;
}

axh_status expert_launch(axh_context *ctx, const char *op, const char *type, bool gate_up,
                         void *const *bufs, uint32_t n_rows, uint32_t cols, uint32_t n_x,
                         uint32_t x_div, uint64_t slots, uint32_t n_experts, void *stream) {
  if ((uint64_t)n_x * (cols / 2u) >= kMaxBuffer)
    return bad("the activations' codes must be below 2 GiB");
  const MatmulKind &k = expert_kind(n_rows, cols / 32u, slots, n_experts, n_x, gate_up);
  // the experts' last tiles are partial: at most so many tiles in all
  const uint64_t active = std::min<uint64_t>(n_experts, slots);
  const uint64_t tiles = active + (slots - active) / k.cols;
  const uint32_t row_tiles = div_up(n_rows, gate_up ? k.rows / 2u : k.rows);
  const uint32_t words[] = {n_rows, cols / 32u, n_x, x_div, n_experts, row_tiles};
  return launch(ctx, kMatmul, std::string("axh_mxfp4_") + op + "_" + k.name + "_" + type,
                tiles * row_tiles, 1, k.threads, k.lds, bufs, 9, words, 6, stream);
}

} // namespace

axh_status mx_launch(axh_context *ctx, MxObject obj, const std::string &name, uint64_t gx, uint64_t gy,
                  uint32_t threads, uint32_t lds, void *const *bufs, uint32_t n_bufs,
                  const uint32_t *words, uint32_t n_words, void *stream) {
  // (a dimension's work-items are counted in 32 bits)
  if (gx > ctx->core->max_wg[0] || gy > ctx->core->max_wg[1] || gx * threads > UINT32_MAX)
    return fail(AXH_ERR_WORKGROUP_COUNT_EXCEEDS_LIMIT, name + ": grid exceeds the device limit");
  hipSetDevice(ctx->core->device);
  axh_kernel *k = nullptr;
  axh_status s = mx_kernel(ctx, obj, name.c_str(), n_bufs, n_words * 4u, threads, &k);
  if (s != AXH_OK) return s;
  const uint32_t grid[3] = {(uint32_t)gx, (uint32_t)gy, 1};
  s = launch_raw(k, grid, bufs, n_bufs, words, n_words * 4u, lds, pick_stream(ctx, stream));
  return s == AXH_OK ? ok() : s;
}

// Kernel `entry` of one of the code objects above, prepared once per context.
axh_status mx_kernel(axh_context *ctx, uint32_t object, const char *entry, uint32_t n_buffers,
                     uint32_t pc_bytes, uint32_t wg_x, axh_kernel **out) {
  std::lock_guard<std::mutex> lk(ctx->ops_mu);
  std::string key = std::string(entry) + "@" + std::to_string(wg_x);
  auto it = ctx->ops.find(key);
  if (it != ctx->ops.end()) {
    *out = it->second;
    return AXH_OK;
  }
  uint8_t access[16];
  if (n_buffers == 0 || n_buffers > sizeof(access)) return bad("bad binding count");
  std::memset(access, AXH_ACCESS_READ_WRITE, sizeof(access));
  axh_binding_plan plan{};
  plan.n_buffers = n_buffers;
  plan.access = access;
  plan.push_constant_total_bytes = pc_bytes;
  plan.workgroup_size[0] = wg_x;
  plan.workgroup_size[1] = 1;
  plan.workgroup_size[2] = 1;
  const void *co = nullptr;
  size_t n = 0;
  if (!mx_code_object(object, &co, &n)) return bad("no such code object");
  axh_kernel *k = nullptr;
  axh_status s = axh_prepare_kernel(ctx, co, n, &plan, pc_bytes, entry, &k);
  if (s != AXH_OK) return s;
  ctx->ops.emplace(std::move(key), k);
  *out = k;
  return AXH_OK;
}

} // namespace axh

using namespace axh;

extern "C" {

axh_status axh_mxfp4_quantize(axh_context *ctx, uint32_t x_type, const void *x, uint64_t x_stride,
                              void *codes, void *scales, uint32_t rows, uint32_t cols,
                              void *stream) {
  if (!ctx) return bad("ctx is NULL");
  const char *type = type_name(x_type);
  if (!type) return bad("x_type must be f32, f16 or bf16");
  axh_status s = check_cols(cols);
  if (s != AXH_OK || rows == 0) return s == AXH_OK ? ok() : s;
  const uint64_t stride = x_stride ? x_stride : cols;
  const uint64_t size = x_type == AXH_GGML_F32 ? 4u : 2u;
  if (stride < cols) return bad("x_stride must be at least cols");
  if (!x || !codes || !scales) return bad("NULL device pointer");
  if (!aligned(x, 16) || (rows > 1 && (stride * size) % 16u))
    return bad("the rows of x must be 16-byte aligned");
  if (!aligned(codes, 16)) return bad("codes must be 16-byte aligned");
  const uint64_t blocks = (uint64_t)rows * (cols / 32u);
  if (blocks >= (1ull << 30)) return bad("too many blocks for one call");
  // Four loads of a lane at once where there are enough, of 16 bits: 8192 x 4096 15.3 us
  // against 17.2, 2048 x 4096 5.0 against 4.7; f32 8192 x 4096 27.2 against 25.1.
  const uint32_t per = size == 2u && blocks >= 1u << 19 ? 4u : 1u;
  const uint32_t words[] = {(uint32_t)blocks, stride == cols ? 0u : cols / 32u, (uint32_t)stride,
                            (uint32_t)(stride >> 32), per};
  void *bufs[] = {mut(x), codes, scales};
  return launch(ctx, kElem, std::string("axh_mxfp4_quantize_") + type, div_up(blocks, 64u * per), 1,
                256, 0, bufs, 3, words, 5, stream);
}

axh_status axh_mxfp4_dequant(axh_context *ctx, const void *codes, const void *scales,
                             uint32_t w_type, void *w, uint64_t n_blocks, void *stream) {
  if (!ctx) return bad("ctx is NULL");
  const char *type = type_name(w_type);
  if (!type) return bad("w_type must be f32, f16 or bf16");
  if (n_blocks == 0) return ok();
  if (!codes || !scales || !w) return bad("NULL device pointer");
  if (!aligned(codes, 4) || !aligned(w, 16))
    return bad("codes must be 4-byte and w 16-byte aligned");
  if (n_blocks >= (1ull << 30)) return bad("too many blocks for one call");
  const uint32_t words[] = {(uint32_t)n_blocks};
  void *bufs[] = {mut(codes), mut(scales), w};
  return launch(ctx, kElem, std::string("axh_mxfp4_dequant_") + type, div_up(n_blocks, 64u), 1,
                256, 0, bufs, 3, words, 1, stream);
}

axh_status axh_mxfp4_unpack_ggml(axh_context *ctx, const void *q, void *codes, void *scales,
                                 uint64_t n_blocks, void *stream) {
  if (!ctx) return bad("ctx is NULL");
  if (n_blocks == 0) return ok();
  if (!q || !codes || !scales) return bad("NULL device pointer");
  if (!aligned(codes, 4)) return bad("codes must be 4-byte aligned");
  if (n_blocks >= (1ull << 30)) return bad("too many blocks for one call");
  const uint32_t words[] = {(uint32_t)n_blocks};
  void *bufs[] = {mut(q), codes, scales};
  return launch(ctx, kElem, "axh_mxfp4_unpack_ggml", div_up(n_blocks, 64u), 1, 256, 0, bufs, 3,
                words, 1, stream);
}

axh_status axh_mxfp4_matvec(axh_context *ctx, const void *codes, const void *scales,
                            const float *x, float *y, uint32_t n_rows, uint32_t cols,
                            void *stream) {
  if (!ctx) return bad("ctx is NULL");
  axh_status s = check_cols(cols);
  if (s != AXH_OK || n_rows == 0) return s == AXH_OK ? ok() : s;
  if (!codes || !scales || !x || !y) return bad("NULL device pointer");
  if (!aligned(codes, 16) || !aligned(x, 16) || !aligned(y, 4))
    return bad("codes and x must be 16-byte and y 4-byte aligned");
  const uint32_t nblk = cols / 32u;
  const MatvecPlan p = plan_matvec(n_rows, nblk, 1, 8, 1, 1);
  const uint32_t words[] = {n_rows, nblk, p.uw, p.batches};
  void *bufs[] = {mut(codes), mut(scales), mut(x), y};
  return launch(ctx, kMatvec, "axh_mxfp4_matvec_l" + std::to_string(p.lanes), p.wgs, 1,
                64u * p.uw * p.groups, p.lds, bufs, 4, words, 4, stream);
}

axh_status axh_mxfp4_matmul_kernel_name(uint32_t n_rows, uint32_t cols, uint32_t batch,
                                        uint32_t y_type, char *buf, size_t cap) {
  if (!buf || cap == 0) return bad("buf is NULL");
  axh_status s = check_cols(cols);
  if (s != AXH_OK) return s;
  const char *type = type_name(y_type);
  if (!type) return bad("y_type must be f32, f16 or bf16");
  const int n = std::snprintf(buf, cap, "axh_mxfp4_matmul_%s_%s",
                              dense_kind(n_rows, cols / 32u, batch).name, type);
  return n > 0 && (size_t)n < cap ? ok() : bad("buffer too small");
}

axh_status axh_mxfp4_matmul(axh_context *ctx, const void *w_codes, const void *w_scales,
                            const void *x_codes, const void *x_scales, uint32_t y_type, void *y,
                            uint32_t n_rows, uint32_t cols, uint32_t batch, void *stream) {
  if (!ctx) return bad("ctx is NULL");
  const char *type = type_name(y_type);
  if (!type) return bad("y_type must be f32, f16 or bf16");
  axh_status s = check_cols(cols);
  if (s != AXH_OK || n_rows == 0 || batch == 0) return s == AXH_OK ? ok() : s;
  if (!w_codes || !w_scales || !x_codes || !x_scales || !y) return bad("NULL device pointer");
  if (!aligned(w_codes, 16) || !aligned(x_codes, 16)) return bad("codes must be 16-byte aligned");
  if (!aligned(y, y_type == AXH_GGML_F32 ? 4 : 2)) return bad("y must be aligned to its elements");
  const MatmulKind &k = dense_kind(n_rows, cols / 32u, batch);
  const uint32_t row_tiles = div_up(n_rows, k.rows);
  const uint32_t words[] = {n_rows, cols / 32u, batch, row_tiles};
  void *bufs[] = {mut(w_codes), mut(w_scales), mut(x_codes), mut(x_scales), y};
  return launch(ctx, kMatmul, std::string("axh_mxfp4_matmul_") + k.name + "_" + type,
                (uint64_t)row_tiles * div_up(batch, k.cols), 1, k.threads, k.lds, bufs, 5, words, 4,
                stream);
}

axh_status axh_expert_logits(axh_context *ctx, uint32_t w_type, const void *w, const float *x,
                             float *logits, uint32_t n_experts, uint32_t cols, uint32_t n_tokens,
                             void *stream) {
  if (!ctx) return bad("ctx is NULL");
  const char *type = type_name(w_type);
  if (!type) return bad("w_type must be f32, f16 or bf16");
  axh_status s = check_cols(cols);
  if (s != AXH_OK) return s;
  if (n_experts == 0 || n_experts > kMaxExperts) return bad("n_experts must be 1 to 1024");
  if (n_tokens >= kMaxBuffer) return bad("too many tokens");
  if (n_tokens == 0) return ok();
  if (!w || !x || !logits) return bad("NULL device pointer");
  if (!aligned(w, 16) || !aligned(x, 16) || !aligned(logits, 4))
    return bad("w and x must be 16-byte and logits 4-byte aligned");
  void *bufs[] = {const_cast<float *>(x), mut(w), logits};
  const std::string name = "axh_expert_logits_";
  if ((uint64_t)n_tokens * n_experts <= kFewLogits) {
    const uint32_t words[] = {n_tokens, n_experts, cols};
    return launch(ctx, kElem, name + "row_" + type, div_up(n_experts, 4u), n_tokens, 256, 0, bufs,
                  3, words, 3, stream);
  }
  auto grid = [&](uint32_t side) {
    return (uint64_t)div_up(n_tokens, side) * div_up(n_experts, side);
  };
  const uint32_t side = grid(64) >= kLogitTiles ? 64u : grid(32) >= kLogitTiles ? 32u : 16u;
  const uint64_t tiles = grid(side);
  const uint32_t words[] = {n_tokens, n_experts, cols, (uint32_t)tiles};
  return launch(ctx, kElem, name + "t" + std::to_string(side) + "_" + type,
                8u * div_up(tiles, 8u), 1, side == 64u ? 512 : 1024, side == 16u ? 65536 : 131072,
                bufs, 3, words, 4, stream);
}

axh_status axh_expert_route(axh_context *ctx, uint32_t logits_type, const void *logits,
                            const float *bias, int32_t *experts, float *weights,
                            uint32_t n_tokens, const axh_route_options *o, void *stream) {
  if (!ctx) return bad("ctx is NULL");
  if (!o) return bad("options is NULL");
  const char *type = type_name(logits_type);
  if (!type) return bad("logits_type must be f32, f16 or bf16");
  if (o->n_experts == 0 || o->n_experts > kMaxExperts) return bad("n_experts must be 1 to 1024");
  if (o->top_k == 0 || o->top_k > kMaxTopK || o->top_k > o->n_experts)
    return bad("top_k must be 1 to 64 and at most n_experts");
  if (o->score > AXH_SCORE_SIGMOID) return bad("unknown score");
  const uint32_t groups = o->n_groups > 1u ? o->n_groups : 1u;
  if (groups > 1u) {
    if (groups > kMaxGroups || o->n_experts % groups)
      return bad("n_groups must divide n_experts and be at most 64");
    if (o->groups_kept == 0 || o->groups_kept > groups)
      return bad("groups_kept must be 1 to n_groups");
    if (o->group_best != 1u && o->group_best != 2u) return bad("group_best must be 1 or 2");
    if (o->group_best > o->n_experts / groups)
      return bad("groups of one expert have no two best: group_best must be 1");
    if ((uint64_t)o->groups_kept * (o->n_experts / groups) < o->top_k)
      return bad("the kept groups hold fewer experts than top_k");
  }
  if (!(o->scale - o->scale == 0.0f)) return bad("scale must be finite");
  if (n_tokens == 0) return ok();
  if (!logits || !experts || !weights) return bad("NULL device pointer");
  if (!aligned(logits, logits_type == AXH_GGML_F32 ? 4 : 2) || !aligned(bias, 4) ||
      !aligned(experts, 4) || !aligned(weights, 4))
    return bad("operands must be aligned to their elements");
  const uint32_t best = groups > 1u ? o->group_best : 1u;
  const bool by_logit = !bias && best == 1u;
  const uint32_t flags = (o->score == AXH_SCORE_SIGMOID ? 1u : 0u) | (o->normalize ? 2u : 0u) |
                         (by_logit ? 4u : 0u);
  uint32_t npl = 1;
  while (npl * 64u < o->n_experts) npl *= 2u;
  uint32_t scale = 0;
  std::memcpy(&scale, &o->scale, 4);
  const uint32_t words[] = {n_tokens, o->n_experts, o->top_k,       flags,
                            groups,   groups > 1u ? o->groups_kept : 1u, best, scale};
  void *bufs[] = {mut(logits), const_cast<float *>(bias), experts, weights};
  return launch(ctx, kElem,
                std::string("axh_expert_route_") + type + "_n" + std::to_string(npl),
                div_up(n_tokens, 4u), 1, 256, 0, bufs, 4, words, 8, stream);
}

axh_status axh_mxfp4_expert_gate_up(axh_context *ctx, const void *gate_codes,
                                    const void *gate_scales, const void *up_codes,
                                    const void *up_scales, const float *x, const int32_t *experts,
                                    float *h, uint32_t n_rows, uint32_t cols, uint32_t n_tokens,
                                    uint32_t top_k, uint32_t n_experts, void *stream) {
  axh_status s = check_experts(ctx, n_rows, cols, n_tokens, top_k, n_experts);
  if (s != AXH_OK || n_rows == 0 || n_tokens == 0) return s == AXH_OK ? ok() : s;
  if (!gate_codes || !gate_scales || !up_codes || !up_scales || !x || !experts || !h)
    return bad("NULL device pointer");
  if (!aligned(gate_codes, 16) || !aligned(up_codes, 16) || !aligned(x, 16) ||
      !aligned(experts, 4) || !aligned(h, 4))
    return bad("codes and x must be 16-byte, experts and h 4-byte aligned");
  const uint64_t slots = (uint64_t)n_tokens * top_k;
  if (slots > 65535u) return bad("at most 65535 slots: prompts take the matmul form");
  const uint32_t nblk = cols / 32u;
  const MatvecPlan p = plan_matvec(n_rows, nblk, 1, 8, 2, (uint32_t)slots);
  const uint32_t words[] = {n_rows, nblk, p.uw, p.batches, top_k, n_experts};
  void *bufs[] = {mut(gate_codes), mut(gate_scales), mut(up_codes), mut(up_scales),
                  mut(x),          mut(experts),     h};
  return launch(ctx, kMatvec, "axh_mxfp4_expert_gate_up_l" + std::to_string(p.lanes), p.wgs, slots,
                64u * p.uw * p.groups, p.lds, bufs, 7, words, 6, stream);
}

axh_status axh_mxfp4_expert_down(axh_context *ctx, const void *codes, const void *scales,
                                 const float *h, const int32_t *experts, const float *weights,
                                 float *y, uint32_t n_rows, uint32_t cols, uint32_t n_tokens,
                                 uint32_t top_k, uint32_t n_experts, void *stream) {
  axh_status s = check_experts(ctx, n_rows, cols, n_tokens, top_k, n_experts);
  if (s != AXH_OK || n_rows == 0 || n_tokens == 0) return s == AXH_OK ? ok() : s;
  if (!codes || !scales || !h || !experts || !weights || !y) return bad("NULL device pointer");
  if (!aligned(codes, 16) || !aligned(h, 16) || !aligned(experts, 4) || !aligned(weights, 4) ||
      !aligned(y, 4))
    return bad("codes and h must be 16-byte, experts, weights and y 4-byte aligned");
  if ((uint64_t)n_tokens * top_k > 65535u)
    return bad("at most 65535 slots: prompts take the matmul form");
  const uint32_t nblk = cols / 32u;
  const MatvecPlan p = plan_matvec(n_rows, nblk, top_k, 4, 1, n_tokens);
  const uint32_t words[] = {n_rows, nblk, p.uw, p.batches, top_k, n_experts};
  void *bufs[] = {mut(codes), mut(scales), mut(h), mut(experts), mut(weights), y};
  return launch(ctx, kMatvec, "axh_mxfp4_expert_down_l" + std::to_string(p.lanes), p.wgs, n_tokens,
                64u * p.uw * p.groups, p.lds, bufs, 6, words, 6, stream);
}

uint64_t axh_expert_plan_bytes(uint32_t n_tokens, uint32_t top_k, uint32_t n_experts) {
  return 4ull * (((uint64_t)n_experts + 1u + 15u) / 16u * 16u + (uint64_t)n_tokens * top_k);
}

axh_status axh_expert_plan(axh_context *ctx, const int32_t *experts, void *plan, uint32_t n_tokens,
                           uint32_t top_k, uint32_t n_experts, void *stream) {
  axh_status s = check_experts(ctx, 1, 32, n_tokens, top_k, n_experts);
  if (s != AXH_OK || n_tokens == 0) return s == AXH_OK ? ok() : s;
  if (!experts || !plan) return bad("NULL device pointer");
  if (!aligned(experts, 4) || !aligned(plan, 4)) return bad("experts and plan must be 4-byte aligned");
  uint32_t bits = 0;
  while ((1u << bits) < n_experts) ++bits;
  const uint32_t slots = n_tokens * top_k;
  // a chunk of 2048 slots each, or more, so that there are at most 128
  uint32_t part_bits = 7;
  while ((uint64_t)slots >> part_bits > 16u * 128u) ++part_bits;
  const uint32_t words[] = {slots, n_experts, bits, part_bits};
  void *bufs[] = {mut(experts), plan};
  return launch(ctx, kElem, "axh_expert_plan", div_up(slots, 16ull << part_bits), 1, 1024,
                (18u * n_experts + 16u) * 4u, bufs, 2, words, 4, stream);
}

axh_status axh_mxfp4_expert_gate_up_matmul(axh_context *ctx, const void *gate_codes,
                                           const void *gate_scales, const void *up_codes,
                                           const void *up_scales, const void *x_codes,
                                           const void *x_scales, const void *plan, uint32_t h_type,
                                           void *h, void *h_scales, uint32_t n_rows, uint32_t cols,
                                           uint32_t n_tokens, uint32_t top_k, uint32_t n_experts,
                                           void *stream) {
  axh_status s = check_experts(ctx, n_rows, cols, n_tokens, top_k, n_experts);
  if (s != AXH_OK) return s;
  const bool packed = h_type == AXH_GGML_MXFP4;
  const char *type = packed ? "mxfp4" : type_name(h_type);
  if (!type) return bad("h_type must be f32, f16, bf16 or mxfp4");
  if (packed && n_rows % 32u) return bad("MXFP4 h needs n_rows to be a multiple of 32");
  if (n_rows == 0 || n_tokens == 0) return ok();
  if (!gate_codes || !gate_scales || !up_codes || !up_scales || !x_codes || !x_scales || !plan ||
      !h || (packed && !h_scales))
    return bad("NULL device pointer");
  if (!aligned(gate_codes, 16) || !aligned(up_codes, 16) || !aligned(x_codes, 16))
    return bad("codes must be 16-byte aligned");
  if (!aligned(h, packed ? 16 : h_type == AXH_GGML_F32 ? 4 : 2) || !aligned(plan, 4))
    return bad("h must be aligned to its elements (MXFP4: 16 bytes) and plan to 4 bytes");
  void *bufs[] = {mut(gate_codes), mut(gate_scales), mut(up_codes), mut(up_scales), mut(x_codes),
                  mut(x_scales),   mut(plan),        h,             packed ? h_scales : h};
  return expert_launch(ctx, "expert_gate_up", type, true, bufs, n_rows, cols, n_tokens, top_k,
                       (uint64_t)n_tokens * top_k, n_experts, stream);
}

axh_status axh_mxfp4_expert_matmul(axh_context *ctx, const void *codes, const void *scales,
                                   const void *h_codes, const void *h_scales, const void *plan,
                                   uint32_t y_type, void *y, uint32_t n_rows, uint32_t cols,
                                   uint32_t n_tokens, uint32_t top_k, uint32_t n_experts,
                                   void *stream) {
  axh_status s = check_experts(ctx, n_rows, cols, n_tokens, top_k, n_experts);
  if (s != AXH_OK) return s;
  const char *type = type_name(y_type);
  if (!type) return bad("y_type must be f32, f16 or bf16");
  if (n_rows == 0 || n_tokens == 0) return ok();
  if (!codes || !scales || !h_codes || !h_scales || !plan || !y) return bad("NULL device pointer");
  if (!aligned(codes, 16) || !aligned(h_codes, 16)) return bad("codes must be 16-byte aligned");
  if (!aligned(y, y_type == AXH_GGML_F32 ? 4 : 2) || !aligned(plan, 4))
    return bad("y must be aligned to its elements and plan to 4 bytes");
  const uint32_t slots = n_tokens * top_k;
  void *bufs[] = {mut(codes),    mut(scales), mut(codes), mut(scales), mut(h_codes),
                  mut(h_scales), mut(plan),   y,          y};
  return expert_launch(ctx, "expert_matmul", type, false, bufs, n_rows, cols, slots, 1u, slots,
                       n_experts, stream);
}

axh_status axh_expert_combine(axh_context *ctx, uint32_t y_type, const void *slots,
                              const int32_t *experts, const float *weights, void *y,
                              uint32_t n_rows, uint32_t n_tokens, uint32_t top_k,
                              uint32_t n_experts, void *stream) {
  if (!ctx) return bad("ctx is NULL");
  const char *type = type_name(y_type);
  if (!type) return bad("y_type must be f32, f16 or bf16");
  if (top_k == 0 || top_k > kMaxTopK) return bad("top_k must be 1 to 64");
  if (n_rows > (1u << 26)) return bad("n_rows must be at most 2^26");
  if (n_rows == 0 || n_tokens == 0) return ok();
  if (!slots || !experts || !weights || !y) return bad("NULL device pointer");
  if (!aligned(slots, 16) || !aligned(y, 16) || !aligned(experts, 4) || !aligned(weights, 4))
    return bad("slots and y must be 16-byte, experts and weights 4-byte aligned");
  const uint32_t words[] = {n_rows, top_k, n_experts ? n_experts : 0x80000000u};
  void *bufs[] = {mut(slots), mut(experts), mut(weights), y};
  return launch(ctx, kElem, std::string("axh_expert_combine_") + type, n_tokens,
                div_up(n_rows, 2048u), 256, 0, bufs, 4, words, 3, stream);
}

} // extern "C"
