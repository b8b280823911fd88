// Attention over the paged 4-bit cache (gfx950): softmax(scale q K^T) V with one pass
// over the keys, the running maximum and sum of each row's softmax in f32.
//
// A wave multiplies 16 kRows query rows (of one key/value head: the heads of its group,
// token after token) with 32 keys a step.  Both products run on v_mfma_f32_16x16x32_bf16,
// transposed, so that no operand changes lanes:
//   S^T (16 keys x 16 rows) = K (keys x dims) Q^T: lane (m, g), m = lane % 16, g = lane /
//     16, has 32 elements of key m of a tile, 16 bytes of codes, their one scale, and the
//     same elements of query row m;
//   S^T leaves a lane with row m and keys 4 g + i of the step's two tiles.  The keys of
//     the second product's sum may come in any order, so these eight are what the lane
//     holds of P^T (keys x rows), and
//   O^T (16 x 16 rows) = V^T P^T: of V the lane has elements 8 m .. 8 m + 7 of the same
//     keys 4 g + i, one 16-byte load and one dword of scales a tile (the layout of a
//     page is made for this), and product t of 8 is elements 8 m + t;
//   so O^T leaves the lane with elements 32 g .. 32 g + 31 of row m.
// Heads of up to 64 elements, and what is left behind 128 of them, have half of that: a lane
// takes 16 elements of a key, and 4 of a value for product t of 4.
//
// Codes become bf16 (f16 where q is), by the converting instruction, which takes the scale:
// exactly, but for f16's range.  An f32 q is three bf16 terms that add up to it, and so are
// its softmax's weights, within 2^-24; bf16 and f16 weights are rounded once (2^-8, 2^-11).
// f16 weights are kept between 2^7, for the largest, and 2^15, so that what falls below f16's
// smallest, 2^-25, is 2^-32 of the largest, and 2^-15 of a row's sum at 2^17 keys.
//
// The running maximum of a row moves only when a score passes it by 2^8: the sums need no
// rescaling in almost all steps, nor the four lanes of a row an exchange of their maxima.
#include "kv_common.h"

using namespace axh;

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(4))) int32_t *const_i32; // read by the scalar unit
typedef const __attribute__((address_space(4))) uint8_t *const_u8;

// 16-bit halves of two dwords: {low a, low b} and {high a, high b}.
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
// Byte i of a dword of scales where an f32 has its exponent field.
__device__ __forceinline__ float scale_of(uint32_t scales, int i) {
  return __builtin_bit_cast(float, i == 3 ? scales >> 1 : scales << (23 - 8 * i));
}
__device__ __forceinline__ f32x4_t mfma_bf16(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x16_t mfma32_bf16(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// Eight bits as eight bf16 of 1 or 0.
__device__ __forceinline__ u32x4_t flags(uint32_t bits) {
  u32x4_t w;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w[j] = (bits >> (2 * j) & 1u ? 0x3F80u : 0u) | (bits >> (2 * j + 1) & 1u ? 0x3F800000u : 0u);
  return w;
}

constexpr float kLowest = -0x1.fffffep127f; // no finite score is below it, and no -inf less -inf
constexpr float kSlack = 8.0f;    // how far (log2) a score may pass its row's maximum

// What the products are made of for each type of q: terms of an operand, the two codes of a
// byte times 2^(e - 127) (e the exponent field of `scale`, whose other bits do not count;
// 255: NaN), two weights, the weight (log2) of a new maximum, the largest scale byte of
// blocks that are finite in that type.
template <class T> struct Mul { // bf16, and f32 as three terms of it
  static constexpr int kN = T::kBytes == 4u ? 3 : 1;
  static constexpr uint32_t kOnes = 0x3F803F80u, kLastScale = 254u;
  static constexpr float kBias = 0.0f;
  template <int kByte> static __device__ __forceinline__ uint32_t codes(uint32_t c, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, kByte));
  }
  static __device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return mfma_bf16(a, b, c);
  }
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    return mfma32_bf16(a, b, c);
  }
  // two weights, as they are multiplied, and a sum
  static __device__ __forceinline__ float add2(uint32_t w, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w),
                                           __builtin_bit_cast(bf16x2_t, kOnes), sum, false);
  }
  // each term the rest of those before it, rounded
  static __device__ __forceinline__ void weights(float a, float b, uint32_t *w) {
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      w[j] = pack2<TBF16>(a, b);
      if (j + 1 < kN) {
        float x, y;
        unpack2<TBF16>(w[j], x, y);
        a -= x;
        b -= y;
      }
    }
  }
};
template <> struct Mul<TF16> {
  static constexpr int kN = 1;
  static constexpr uint32_t kOnes = 0x3C003C00u, kLastScale = 140u; // 6 * 2^13
  static constexpr float kBias = 7.0f;
  template <int kByte> static __device__ __forceinline__ uint32_t codes(uint32_t c, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, kByte));
  }
  static __device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a),
                                                  __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a),
                                                  __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(uint32_t w, float sum) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, w),
                                  __builtin_bit_cast(half2_t, kOnes), sum, false);
  }
  static __device__ __forceinline__ void weights(float a, float b, uint32_t *w) {
    w[0] = pack2<TF16>(a, b);
  }
};

// Two elements of an f32 q as kN dwords of bf16 terms, cut off, so that they add up exactly;
// an infinity or a NaN is its own first term, and the others are 0.
template <int kN> __device__ __forceinline__ void split_query(float a, float b, uint32_t *w) {
  const bool fa = a - a == 0.0f, fb = b - b == 0.0f;
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    if (a != a) x = 0x7FC00000u; // whose bits may all be cut off
    if (b != b) y = 0x7FC00000u;
    w[j] = highs(x, y);
    a = fa ? a - __builtin_bit_cast(float, x & 0xFFFF0000u) : 0.0f;
    b = fb ? b - __builtin_bit_cast(float, y & 0xFFFF0000u) : 0.0f;
  }
}

// Two elements, byte kByte of each dword of codes, of eight keys: pairs of keys, as the matrix
// instruction wants them, from pairs of elements, as the codes are.
template <class T, int kByte = 0>
__device__ __forceinline__ void pair(const u32x4_t (&codes)[2], const uint32_t (&scales)[2],
                                     u32x4_t &even, u32x4_t &odd) {
  using M = Mul<T>;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int x = j >> 1, e = 2 * (j & 1);
    const uint32_t p = M::template codes<kByte>(codes[x][e], scale_of(scales[x], e));
    const uint32_t q = M::template codes<kByte>(codes[x][e + 1], scale_of(scales[x], e + 1));
    even[j] = lows(p, q);
    odd[j] = highs(p, q);
  }
}

// A workspace: the maximum and the sum of each split's part of each row, then the parts.
__device__ __forceinline__ uint64_t parts_at(uint64_t rows, uint32_t splits) {
  return (rows * splits + 1u) / 2u * 4u; // 16-byte aligned
}

struct Args {
  const uint8_t *q, *k, *v;
  const int32_t *starts, *lengths, *table;
  uint8_t *y;
  float *ws;
  uint32_t n_seqs, n_tokens, max_pages;
  Geometry g;
  uint32_t per;   // query heads of a key/value head
  uint32_t q_stride, y_stride;
  float c;        // scale * log2 e
  uint32_t window;
  uint32_t chunk, splits; // keys of a split (the last takes what is left), and how many
  uint32_t page_bytes;    // of all heads
};

// The sequence, first token, tokens and tile of a group of `rows` query rows.
struct Group {
  int32_t seq, first, tokens;
  uint32_t tile;
};
__device__ __forceinline__ Group locate(const Args &a, uint32_t group, uint32_t rows) {
  if (!a.starts) {
    const uint32_t tiles = (a.per + rows - 1u) / rows;
    const uint32_t seq = group / tiles;
    return {(int32_t)seq, (int32_t)seq, 1, group - seq * tiles};
  }
  // 64 sequences at a time: how many groups they and those before them have
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t before = 0;
  for (uint32_t s0 = 0; s0 < a.n_seqs; s0 += 64u) {
    const uint32_t s = s0 + lane;
    int32_t first = 0, n = 0;
    if (s < a.n_seqs) {
      first = a.starts[s];
      n = a.starts[s + 1u] - first;
      // (what lies outside the batch is left out)
      if (first < 0 || n < 0 || (uint32_t)first + (uint32_t)n > a.n_tokens) n = 0;
    }
    const uint32_t mine = ((uint32_t)n * a.per + rows - 1u) / rows;
    uint32_t sum = mine;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
      const uint32_t o = (uint32_t)__shfl_up((int)sum, d);
      sum += lane >= d ? o : 0u;
    }
    const uint64_t past = __ballot(before + sum > group);
    if (past) {
      const int who = __builtin_ctzll(past);
      Group r;
      r.seq = (int32_t)(s0 + (uint32_t)who);
      r.first = __builtin_amdgcn_readlane(first, who);
      r.tokens = __builtin_amdgcn_readlane(n, who);
      r.tile = group - before - (uint32_t)__builtin_amdgcn_readlane((int)(sum - mine), who);
      return r;
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  }
  return {-1, 0, 0, 0};
}

// Eight elements of a row from e0 on: the output, or a part with its maximum and sum.  Rows of
// the output, or of a split's part, go by (token, head).
template <class T>
__device__ __forceinline__ void store_row(const Args &a, const Group &at, uint32_t head,
                                          uint32_t split, uint32_t row, uint32_t e0, float *x,
                                          float maximum, float total, bool lead) {
  const uint32_t n = row / a.per, token = (uint32_t)at.first + n;
  const uint32_t h = head * a.per + row - n * a.per;
  if (a.splits == 1u) {
    const float f = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = total == 0.0f ? 0.0f : x[j] * f;
    store8<T>(a.y + ((uint64_t)token * a.y_stride + (uint64_t)h * a.g.dim + e0) * T::kBytes, x);
    return;
  }
  const uint64_t all = (uint64_t)a.n_tokens * a.g.kv_heads * a.per;
  const uint64_t part = (uint64_t)split * all + (uint64_t)token * (a.g.kv_heads * a.per) + h;
  if (lead) {
    float *ms = a.ws + 2u * part;
    ms[0] = maximum;
    ms[1] = total;
  }
  if (total != 0.0f) // (or NaN; an empty part's elements are not read)
    store8<TF32>(reinterpret_cast<uint8_t *>(a.ws + parts_at(all, a.splits) + part * a.g.dim + e0), x);
}

// Keys that a row at a position sees: from the first to before the end.
__device__ __forceinline__ int32_t first_key(const Args &a, int32_t pos) {
  return a.window && pos >= (int32_t)a.window ? pos - (int32_t)a.window + 1 : 0;
}
__device__ __forceinline__ int32_t end_key(const Args &a, int32_t pos) {
  const int32_t capacity = (int32_t)(a.max_pages << a.g.page_shift);
  return pos < capacity ? pos + 1 : capacity;
}
// A sequence's row's position (row: of its tokens' query heads in the group).
__device__ __forceinline__ int32_t position(const Args &a, const Group &at, uint32_t row,
                                            int32_t length) {
  return length - at.tokens + (int32_t)(row / a.per);
}
// The keys of a workgroup whose rows are those from `first` to `end`: what some row sees,
// from a whole step on, and its split of them.
__device__ __forceinline__ void keys_of(const Args &a, const Group &at, uint32_t split,
                                        uint32_t first, uint32_t end, int32_t length, uint32_t &lo,
                                        uint32_t &hi) {
  const uint32_t rows = (uint32_t)at.tokens * a.per;
  end = end < rows ? end : rows;
  lo = hi = 0;
  if (first >= end) return;
  const int32_t stop_key = end_key(a, position(a, at, end - 1u, length));
  if (stop_key <= 0) return;
  const uint32_t begin = (uint32_t)first_key(a, position(a, at, first, length)) & ~31u;
  const uint64_t mine = (uint64_t)begin + (uint64_t)split * a.chunk;
  uint64_t stop = (uint32_t)stop_key;
  if (split + 1u < a.splits && mine + a.chunk < stop) stop = mine + a.chunk;
  if (mine < stop) {
    lo = (uint32_t)mine;
    hi = (uint32_t)stop;
  }
}
// The page of a key in a sequence's row of the table (beyond the table, where no row sees a
// key: its last page); outside 0 .. n_pages - 1 it is not there.
__device__ __forceinline__ uint32_t page_id(const Args &a, const int32_t *pages, uint32_t key) {
  const uint32_t slot = key >> a.g.page_shift, last = a.max_pages - 1u;
  return (uint32_t)*(const_i32)((const_u8)pages + (slot < last ? slot : last) * 4u);
}

// The codes and scales of a step's two tiles of 16 keys, as a lane has them.
template <int kChunks> struct Raw {
  u32x4_t k[2][kChunks], v[2][kChunks];
  uint32_t ks[2][kChunks], vs[2][kChunks];
};
// A step's pages (of its two tiles of 16 keys, one page in pages of 32 tokens or more): their
// numbers in the table, and where the cache has them.
struct Ids {
  uint32_t id[2];
};
struct Pages {
  uint64_t at[2];
  bool there[2];
  __device__ __forceinline__ bool both() const { return there[0] && there[1]; }
};

// A wave's 16 kRows rows and its part of their sums, and the steps of 32 keys.  kDim: 64,
// 128, 192 or 256, the head's elements to the next multiple of 64.
template <class T, int kDim, int kRows> struct Rows {
  using M = Mul<T>;
  static constexpr int kN = M::kN, kChunks = (kDim + 127) / 128;
  // Elements of a value that a lane has of chunk c, and so its products.
  static constexpr int width(int c) { return kDim - 128 * c >= 128 ? 8 : 4; }

  const Args &a;
  const uint32_t lane = threadIdx.x & 63u, m = lane & 15u, grp = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t head, split;
  Group at;
  uint32_t rows, row0;           // of the sequence; the wave's first
  int32_t all_from, all_to;      // keys that all rows of the wave see
  // Where a lane's codes and scales are in a page, of its first tile.
  uint32_t kc[kChunks], ks[kChunks], vc[kChunks], vs[kChunks];
  const uint8_t *kh, *vh;        // the head's part of page 0
  const int32_t *pages_of;       // the sequence's row of the table

  u32x4_t q[kRows][kChunks][4][kN];
  f32x4_t o[kRows][kChunks][8];
  f32x4_t sum[kRows]; // of the weights as they were multiplied; four times the same
  float top[kRows];   // what a score (log2) is a weight of 1 at
  uint32_t wild[kRows]; // bit 4 c + j: elements j of chunk c's products are NaN
  int32_t from[kRows], to[kRows]; // keys that the lane's row sees: from <= key < to

  __device__ __forceinline__ Rows(const Args &args, uint32_t h, uint32_t s)
      : a(args), head(h), split(s) {}

  // The rows from row0 on: the keys that they see, and their queries.
  __device__ __forceinline__ void start(uint32_t first_row, int32_t length) {
    row0 = first_row;
    rows = (uint32_t)at.tokens * a.per;
    all_from = all_to = 0;
    if (row0 < rows) {
      const uint32_t last = row0 + 16u * kRows < rows ? row0 + 16u * kRows : rows;
      all_from = first_key(a, position(a, at, last - 1u, length));
      all_to = end_key(a, position(a, at, row0, length));
    }
    const uint32_t dim = a.g.dim;
    const uint64_t head_at = (uint64_t)head * a.g.head_bytes();
    pages_of = a.table + (uint64_t)(uint32_t)at.seq * a.max_pages;
    kh = a.k + head_at;
    vh = a.v + head_at;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      // elements from dim on: others in their place, times a q of 0, or never stored
      const uint32_t w = (uint32_t)width(c);
      uint32_t kd = 16u * c + grp * (w / 2u), vd = 16u * c + (w == 8u ? m : m / 2u); // dwords
      if (8u * kd >= dim) kd = 0;
      if (8u * vd >= dim) vd = 0;
      kc[c] = a.g.key_code(m, kd);
      ks[c] = a.g.key_scale(m, kd >> 2);
      vc[c] = a.g.value_code(4u * grp, vd);
      vs[c] = a.g.value_scale(4u * grp, vd >> 2);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const uint32_t row = row0 + 16u * i + m;
      const bool real = row < rows;
      from[i] = to[i] = 0;
      if (real) {
        from[i] = first_key(a, position(a, at, row, length));
        to[i] = end_key(a, position(a, at, row, length));
      }
      const uint32_t token = real ? row / a.per : 0u, h = real ? row - token * a.per : 0u;
      const uint8_t *qr = a.q + ((uint64_t)((uint32_t)at.first + token) * a.q_stride +
                                 (uint64_t)(head * a.per + h) * dim) * T::kBytes;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int b = 0; b < width(c) / 2; ++b) {
          const uint32_t e = 128u * c + grp * (uint32_t)(4 * width(c)) + 8u * b;
          const bool on = real && e < dim;
          if constexpr (kN == 1) {
            u32x4_t w = {0, 0, 0, 0};
            if (on) w = *reinterpret_cast<const u32x4_t *>(qr + e * 2u);
            q[i][c][b][0] = w;
          } else {
            float x[8] = {};
            if (on) load8<T>(qr + e * T::kBytes, x);
            uint32_t w[4][kN];
#pragma unroll
            for (int j = 0; j < 4; ++j) split_query<kN>(x[2 * j], x[2 * j + 1], w[j]);
#pragma unroll
            for (int j = 0; j < kN; ++j)
              q[i][c][b][j] = (u32x4_t){w[0][j], w[1][j], w[2][j], w[3][j]};
          }
        }
    }
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int e = 0; e < width(c); ++e) o[i][c][e] = (f32x4_t){0, 0, 0, 0};
      sum[i] = (f32x4_t){0, 0, 0, 0};
      wild[i] = 0;
      top[i] = kLowest;
    }
  }

  __device__ __forceinline__ Ids ids(uint32_t t) const {
    return {{page_id(a, pages_of, t), page_id(a, pages_of, t + 16u)}};
  }
  // (page 0 in the place of one that is not there: memory that is)
  __device__ __forceinline__ Pages pages(const Ids &p) const {
    auto at = [&](uint32_t id) { return (uint64_t)(id < a.g.n_pages ? id : 0u) * a.page_bytes; };
    return {{at(p.id[0]), at(p.id[1])}, {p.id[0] < a.g.n_pages, p.id[1] < a.g.n_pages}};
  }
  // A tile's page; codes and scales of the tile so much further on, of keys as of values.
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile(const uint8_t *base, const Pages &p,
                                                         int T16, uint32_t t, uint32_t &codes,
                                                         uint32_t &scales) const {
    const uint32_t row = (t + 16u * T16) & (a.g.page_rows() - 1u);
    codes = a.g.key_code(row, 0u);
    scales = row * (a.g.dim / 32u);
    return rsrc(base + p.at[T16], a.g.head_bytes());
  }
  __device__ __forceinline__ void load_keys(Raw<kChunks> &r, const Pages &p, uint32_t t) const {
#pragma unroll
    for (int T16 = 0; T16 < 2; ++T16) {
      uint32_t codes, scales;
      const auto page = tile(kh, p, T16, t, codes, scales);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if (width(c) == 8) {
          r.k[T16][c] = __builtin_amdgcn_raw_buffer_load_b128(page, (int)kc[c], (int)codes, 0);
        } else {
          const u32x2_t w = __builtin_amdgcn_raw_buffer_load_b64(page, (int)kc[c], (int)codes, 0);
          r.k[T16][c] = (u32x4_t){w.x, w.y, 0, 0};
        }
        r.ks[T16][c] = __builtin_amdgcn_raw_buffer_load_b8(page, (int)ks[c], (int)scales, 0);
      }
    }
  }
  __device__ __forceinline__ void load_values(Raw<kChunks> &r, const Pages &p, uint32_t t) const {
#pragma unroll
    for (int T16 = 0; T16 < 2; ++T16) {
      uint32_t codes, scales;
      const auto page = tile(vh, p, T16, t, codes, scales);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        r.v[T16][c] = __builtin_amdgcn_raw_buffer_load_b128(page, (int)vc[c], (int)codes, 0);
        r.vs[T16][c] = __builtin_amdgcn_raw_buffer_load_b32(page, (int)vs[c], (int)scales, 0);
      }
    }
  }

  __device__ __forceinline__ void scores(const Raw<kChunks> &r, f32x4_t (&s)[kRows][2]) const {
#pragma unroll
    for (int T16 = 0; T16 < 2; ++T16) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) s[i][T16] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const float scale = scale_of(r.ks[T16][c], 0);
#pragma unroll
        for (int b = 0; b < width(c) / 2; ++b) {
          const uint32_t w = r.k[T16][c][b];
          const u32x4_t key = {M::template codes<0>(w, scale), M::template codes<1>(w, scale),
                               M::template codes<2>(w, scale), M::template codes<3>(w, scale)};
#pragma unroll
          for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int j = 0; j < kN; ++j) s[i][T16] = M::mfma(key, q[i][c][b][j], s[i][T16]);
        }
      }
    }
  }

  // Whether every row of the wave sees all keys of a step.
  __device__ __forceinline__ bool whole(const Pages &p, uint32_t t) const {
    return p.both() && (int32_t)t >= all_from && (int32_t)(t + 32u) <= all_to;
  }
  // Scores of keys that a row does not see: -inf.  Bit 4 T16 + j of seen[i]: it sees that one.
  __device__ __forceinline__ void mask(const Pages &p, uint32_t t, f32x4_t (&s)[kRows][2],
                                       uint32_t (&seen)[kRows]) const {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      seen[i] = 0;
#pragma unroll
      for (int T16 = 0; T16 < 2; ++T16) {
        f32x4_t x = s[i][T16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int32_t key = (int32_t)(t + 16u * T16 + 4u * grp + j);
          const bool on = p.there[T16] && key >= from[i] && key < to[i];
          seen[i] |= (on ? 1u : 0u) << (4 * T16 + j);
          x[j] = on ? x[j] : -__builtin_inff();
        }
        s[i][T16] = x;
      }
    }
  }

  // Whether a score is above what its row's weights go to: the maximum's, and the slack.
  __device__ __forceinline__ bool over(const f32x4_t (&s)[kRows][2]) const {
    bool is = false;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      is |= __builtin_fmaf(highest(s[i]), a.c, -top[i]) > kSlack + M::kBias;
    return __ballot(is) != 0u;
  }
  static __device__ __forceinline__ float highest(const f32x4_t (&s)[2]) {
    float most = s[0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) most = __builtin_fmaxf(most, s[j >> 2][j & 3]);
    return most;
  }
  // Then its row has a new maximum, the same in the row's four lanes.
  __device__ __forceinline__ void raise(const f32x4_t (&s)[kRows][2]) {
    if (!over(s)) return;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float x = highest(s[i]);
      x = __builtin_fmaxf(x, __shfl_xor(x, 16));
      x = __builtin_fmaxf(x, __shfl_xor(x, 32)) * a.c - M::kBias;
      const float now = x - top[i] > kSlack ? x : top[i];
      const float f = __builtin_amdgcn_exp2f(top[i] - now);
      top[i] = now;
      sum[i] *= f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int e = 0; e < width(c); ++e) o[i][c][e] *= f;
    }
  }

  // The weights of a step, and their sums: a product with ones, over the weights as the
  // values are multiplied by them.
  __device__ __forceinline__ void weights(const f32x4_t (&s)[kRows][2],
                                          u32x4_t (&weight)[kRows][kN]) {
    const u32x4_t ones = {M::kOnes, M::kOnes, M::kOnes, M::kOnes};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      uint32_t p[4][kN];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int T16 = j >> 1, e = 2 * (j & 1);
        M::weights(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i][T16][e], a.c, -top[i])),
                   __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][T16][e + 1], a.c, -top[i])), p[j]);
      }
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        weight[i][j] = (u32x4_t){p[0][j], p[1][j], p[2][j], p[3][j]};
        sum[i] = M::mfma(ones, weight[i][j], sum[i]);
      }
    }
  }

  __device__ __forceinline__ void add(int c, int tile, u32x4_t values,
                                      const u32x4_t (&weight)[kRows][kN]) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j) o[i][c][tile] = M::mfma(values, weight[i][j], o[i][c][tile]);
  }

  // Values of the lane's eight keys that are 0 from here on whatever bytes they have:
  // those whose bit in `keep` is not set (beyond the length, or of a page that is not there),
  // and, as a weight of 0 times a NaN is no 0, with `careful` blocks that are not finite.
  __device__ __forceinline__ void hide(Raw<kChunks> &r, uint32_t keep, bool careful) const {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      u32x4_t codes[2];
      uint32_t scales[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int T16 = j >> 2, e = j & 3;
        const bool wide = careful && (r.vs[T16][c] >> (8 * e) & 255u) > M::kLastScale;
        const uint32_t part = !(keep >> j & 1u) || wide ? 0u : ~0u;
        codes[T16][e] = r.v[T16][c][e] & part;
        scales[T16] |= (r.vs[T16][c] & part & 255u << (8 * e)) | (~part & 127u << (8 * e));
      }
#pragma unroll
      for (int T16 = 0; T16 < 2; ++T16) {
        r.v[T16][c] = codes[T16];
        r.vs[T16][c] = scales[T16];
      }
    }
  }
  // The blocks of the lane's eight keys that are not finite, of those whose bit is in `keep`.
  __device__ __forceinline__ bool not_finite(const Raw<kChunks> &r, uint32_t keep,
                                             uint32_t (&bad)[kChunks]) const {
    uint32_t any = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      bad[c] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((r.vs[j >> 2][c] >> (8 * (j & 3)) & 255u) > M::kLastScale) bad[c] |= 1u << j;
      bad[c] &= keep;
      any |= bad[c];
    }
    return __ballot(any != 0u) != 0u;
  }
  // NaN for the rows that see one of them: a product of the blocks' and the keys' flags
  // finds them.
  __device__ __forceinline__ void poison(const uint32_t (&bad)[kChunks],
                                         const uint32_t (&seen)[kRows]) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const f32x4_t nan = mfma_bf16(flags(bad[c]), flags(seen[i]), (f32x4_t){0, 0, 0, 0});
#pragma unroll
        for (int j = 0; j < 4; ++j) wild[i] |= (nan[j] > 0.0f ? 1u : 0u) << (4 * c + j);
      }
  }

  // Eight consecutive elements of the lane's row i: group j of those that it has of chunk c.
  static constexpr int groups(int c) { return width(c) / 2; }
  __device__ __forceinline__ uint32_t eight(int i, int c, int j, float *x) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int tile = width(c) == 8 ? e : e & 3, k = width(c) == 8 ? j : 2 * j + (e >> 2);
      x[e] = wild[i] >> (4 * c + k) & 1u ? __builtin_nanf("") : o[i][c][tile][k];
    }
    return 128u * c + grp * (uint32_t)(4 * width(c)) + 8u * j;
  }
};

// ---------------------------------------------------------------------------
// Few rows: the four waves of a workgroup have the same rows and every fourth step of 32
// keys, and add their sums in LDS at the end.  The keys, and then the values, of a wave's
// next step are requested as soon as the registers of this one's are free.
//   Few rows read each key once and are bound by memory where there are many of them: 32
// sequences of 8192 keys, 8 heads of 128 in bf16, 36.5 to 40 us for 178 MB (a copy of as many
// bytes takes 36).  In f32 three products a term cost the vector and matrix units more than that:
// 131072 keys, 16 heads of 64, 37.5 us for 143 MB.  8 sequences of 6000, 32 rows of 256 each:
// 18.5 us for 36 MB, six steps a wave between a chain of reads (start, length, page, key) and the
// sum.  32 rows a wave convert a key or value once for both halves of them: prompts in between,
// 1501 queries to 6007 keys in f16, 7 heads a key's, 125 us, 730 TFLOP/s (16 rows 146); vector
// units 66 % busy, matrix units 37 %.
// ---------------------------------------------------------------------------
template <class T, int kDim, int kRows> struct Few : Rows<T, kDim, kRows> {
  using R = Rows<T, kDim, kRows>;
  using R::a, R::at, R::grp, R::m, R::sum, R::top, R::wave, R::row0, R::rows;
  static constexpr int kN = R::kN, kChunks = R::kChunks;
  static constexpr uint32_t kWaves = 4u, kGroupRows = 16u * kRows, kStep = 32u * kWaves;
  static constexpr uint32_t kPitch = kDim + 4u; // floats of a row in LDS
  static constexpr uint32_t kLds = kWaves * 16u * (kPitch + 2u);

  __device__ __forceinline__ Few(const Args &args, uint32_t h, uint32_t s) : R(args, h, s) {}

  // What a step needs where not all of its keys are seen by all rows, or one is a new maximum.
  __device__ __forceinline__ void look(Raw<kChunks> &r, f32x4_t (&s)[kRows][2], const Pages &p,
                                       uint32_t t) {
    if (!R::whole(p, t)) {
      uint32_t seen[kRows], some = 0, bad[kChunks];
      R::mask(p, t, s, seen);
      // a key that one of the wave's rows sees (four lanes hold four keys of all rows each)
#pragma unroll
      for (int i = 0; i < kRows; ++i) some |= seen[i];
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) some |= (uint32_t)__shfl_xor((int)some, d);
      if (R::not_finite(r, some, bad)) R::poison(bad, seen);
      R::hide(r, some, true);
    }
    R::raise(s);
  }

  __device__ __forceinline__ void values(const Raw<kChunks> &r,
                                         const u32x4_t (&weight)[kRows][kN]) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      u32x4_t even, odd, codes[2] = {r.v[0][c], r.v[1][c]};
      if (R::width(c) == 4) { // the lane's half of the dword
        codes[0] >>= 16u * (m & 1u);
        codes[1] >>= 16u * (m & 1u);
      }
      pair<T, 0>(codes, {r.vs[0][c], r.vs[1][c]}, even, odd);
      R::add(c, 0, even, weight);
      R::add(c, 1, odd, weight);
      pair<T, 1>(codes, {r.vs[0][c], r.vs[1][c]}, even, odd);
      R::add(c, 2, even, weight);
      R::add(c, 3, odd, weight);
      if (R::width(c) == 8) {
        pair<T, 2>(codes, {r.vs[0][c], r.vs[1][c]}, even, odd);
        R::add(c, 4, even, weight);
        R::add(c, 5, odd, weight);
        pair<T, 3>(codes, {r.vs[0][c], r.vs[1][c]}, even, odd);
        R::add(c, 6, even, weight);
        R::add(c, 7, odd, weight);
      }
    }
  }

  __device__ __forceinline__ void run(uint32_t group, float *lds) {
    at = locate(a, group, kGroupRows);
    if (at.seq < 0) return; // the whole workgroup
    at.seq = __builtin_amdgcn_readfirstlane(at.seq);
    const int32_t length = max(((const_i32)a.lengths)[at.seq], 0);
    R::start(at.tile * kGroupRows, length);
    R::clear();
    uint32_t t, end;
    keys_of(a, at, R::split, row0, row0 + kGroupRows, length, t, end);
    t += 32u * wave;
    if (t < end) {
      Raw<kChunks> r;
      // the steps at t, t + kStep and t + 2 kStep
      Pages p0 = R::pages(R::ids(t)), p1 = R::pages(R::ids(t + kStep));
      Ids i2 = R::ids(t + 2u * kStep);
      R::load_keys(r, p0, t);
      R::load_values(r, p0, t);
      f32x4_t s[kRows][2];
      R::scores(r, s);
      if (t + kStep < end) R::load_keys(r, p1, t + kStep);
      bool plain;
      do {
        look(r, s, p0, t);
        do { // a loop of its own where only the products change the sums: they stay in place
          const Pages p2 = R::pages(i2);
          i2 = R::ids(t + 3u * kStep);
          u32x4_t weight[kRows][kN];
          R::weights(s, weight);
          values(r, weight);
          if (t + kStep < end) R::load_values(r, p1, t + kStep);
          R::scores(r, s);
          if (t + 2u * kStep < end) R::load_keys(r, p2, t + 2u * kStep);
          t += kStep;
          p0 = p1;
          p1 = p2;
          plain = t < end && R::whole(p0, t) && !R::over(s);
        } while (plain);
      } while (t < end);
    }
    join(lds);
  }

  // Sixteen rows at a time: the waves' sums, then 8 elements of a row a lane, added in the
  // waves' order.
  __device__ __forceinline__ void join(float *lds) const {
    float *tops = lds + kWaves * 16u * kPitch, *sums = tops + kWaves * 16u;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (i) __syncthreads();
      if (row0 + 16u * i + m < rows) {
        if (grp == 0u) {
          tops[16u * wave + m] = top[i];
          sums[16u * wave + m] = sum[i][0];
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int j = 0; j < R::groups(c); ++j) {
            float x[8];
            const uint32_t e0 = R::eight(i, c, j, x);
            store8<TF32>(reinterpret_cast<uint8_t *>(lds + (16u * wave + m) * kPitch + e0), x);
            __builtin_amdgcn_sched_barrier(0); // (one after another: they take registers to gather)
          }
      }
      __syncthreads();
      constexpr uint32_t kAcross = kDim / 8u;
      for (uint32_t at0 = threadIdx.x; at0 < 16u * kAcross; at0 += 64u * kWaves) {
        const uint32_t r = at0 / kAcross, e0 = at0 % kAcross * 8u, row = row0 + 16u * i + r;
        if (row >= rows || e0 >= a.g.dim) continue;
        float most = tops[r], total = 0.0f, x[8] = {};
#pragma unroll
        for (uint32_t w = 1; w < kWaves; ++w) most = __builtin_fmaxf(most, tops[16u * w + r]);
#pragma unroll 4
        for (uint32_t w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f(tops[16u * w + r] - most);
          total += sums[16u * w + r] * f;
          float y[8];
          load8<TF32>(reinterpret_cast<const uint8_t *>(lds + (16u * w + r) * kPitch + e0), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(y[e], f, x[e]);
        }
        store_row<T>(a, at, R::head, R::split, row, e0, x, most, total, e0 == 0u);
      }
    }
  }
};

// ---------------------------------------------------------------------------
// Many rows: the four waves of a workgroup have 32 rows each and go through the same keys,
// 32 a step, on v_mfma_f32_32x32x16 (which leaves the other instructions three quarters of
// the time, where 16x16x32 leaves half).  Lane (m, h), m = lane % 32, h = lane / 32:
//   of a key it has elements 64 h .. 64 h + 63, of the scores row m's with keys 8 a + 4 h + b
//   (a, b = 0 .. 3), which are what it holds of the weights in the second product; of a value
//   elements 4 m .. 4 m + 3 of the same keys; and of the output 16 elements from 32 a + 16 h on.
// (Of the last 64 elements of a head half of each.)
//   Codes and scales go to a ring of kRing steps in LDS, loaded straight there, a quarter a
// wave, three steps before they are used: the latency of a line that no cache has is two
// steps long.  The values' fragments are made from them once for the four waves, one step
// ahead; keys, which need no exchange of elements, each wave converts for itself, one step
// ahead as well, so that the next scores run beside the exponentials of these.
//   Values are multiplied as they are, in steps that some rows see in part too; if an
// output turns out not to be finite, the workgroup starts over, carefully: blocks that are
// not become 0, and the rows that see them NaN.
//   4096 queries to as many keys, 32 query and 8 key heads of 128 in bf16: 157 to 163 us, 840 to
// 870 TFLOP/s, where a product of 8192^3 reaches 1319.  A step has 133 vector instructions, 18 of
// LDS and 16 products a wave; matrix units are 46 % busy and vector units 67 %, at a clock that
// falls to 1.8 GHz (149 us in place of 178 with zeros for data, on a slower card).  Not faster
// were, in turn on one card: keys' fragments through LDS too (106 vector instructions, 27 of LDS),
// +9 %; all of a step's reads at once and products and exponentials one by one in turn, two waves
// a SIMD, +20 %; 64 rows a wave, one wave a SIMD, +47 %; fragments read one product ahead, the
// same.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void lds_void_t;

template <class T, int kDim> struct Many {
  using M = Mul<T>;
  static constexpr int kN = M::kN, kChunks = (kDim + 127) / 128;
  static constexpr int pieces(int c) { return kDim - 128 * c >= 128 ? 2 : 1; } // of 16 bytes a key
  static constexpr uint32_t kGroupRows = 128, kRing = 4;
  static constexpr uint32_t kTiles = kDim / 16u;  // fragments of a step: kDim / 32 of 16 keys each
  // LDS, in bytes: of a step a chunk's codes and scales of keys and values; then the fragments
  // of two steps.
  static constexpr uint32_t kPart = 2u * (2048u + 512u), kStage = kChunks * kPart;
  static constexpr uint32_t kFrags = kRing * kStage, kHalf = kTiles * 1024u;
  static constexpr uint32_t kLds = (kFrags + 2u * kHalf) / 4u; // floats
  static constexpr int kLoads = 2 * kChunks; // of a wave and step

  const Args &a;
  const uint32_t lane = threadIdx.x & 63u, m = lane & 31u, h = lane >> 5;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t head, split;
  uint8_t *lds;
  Group at;
  uint32_t rows, row0, begin, end; // of the sequence; the wave's first; keys of the workgroup
  uint32_t all_from, all_to;       // keys that all rows of the wave see
  int32_t from, to;                // that the lane's row sees
  uint32_t code_at[kChunks], scale_at[kChunks]; // the lane's part of a wave's loads
  uint32_t key_shift[kChunks][2];               // of the scale bytes in a dword
  const uint8_t *base;   // the head's part of page 0, of the wave's keys or values
  const int32_t *pages;  // the sequence's row of the table

  u32x4_t q[kChunks][8][kN];
  f32x16_t o[kChunks][4];
  float top, sum; // what a score (log2) is a weight of 1 at; the lane's part of the sum
  uint32_t wild; // bit 4 c + i: elements 32 i .. of chunk c are NaN

  __device__ __forceinline__ Many(const Args &args, uint32_t hd, uint32_t s)
      : a(args), head(hd), split(s) {}

  __device__ __forceinline__ void start(int32_t length) {
    const uint32_t first = at.tile * kGroupRows, dim = a.g.dim;
    rows = (uint32_t)at.tokens * a.per;
    row0 = first + 32u * wave;
    keys_of(a, at, split, first, first + kGroupRows, length, begin, end);
    all_from = all_to = 0;
    if (row0 < rows) {
      const uint32_t last = row0 + 32u < rows ? row0 + 32u : rows;
      const int32_t stop = end_key(a, position(a, at, row0, length));
      all_from = (uint32_t)first_key(a, position(a, at, last - 1u, length));
      all_to = stop > 0 ? (uint32_t)stop : 0u;
      all_to = all_to < end ? all_to : end;
    }
    pages = a.table + (uint64_t)(uint32_t)at.seq * a.max_pages;
    base = (wave < 2u ? a.k : a.v) + (uint64_t)head * a.g.head_bytes();
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      // lanes of a load: 16 keys of each piece in turn, or the dwords of four values in turn
      // (elements from dim on: others in their place, times a q of 0, or never stored)
      const bool two = pieces(c) == 2;
      const uint32_t l = two ? lane : lane & 31u;
      uint32_t piece = 4u * c + (l >> 4), dw = 16u * c + (two ? l & 15u : l & 7u);
      if (piece >= dim / 32u) piece = 0;
      if (dw >= dim / 8u) dw = 0;
      const uint32_t four = two ? l >> 4 : l >> 3;
      code_at[c] = wave < 2u ? a.g.key_code(l & 15u, 4u * piece) : a.g.value_code(4u * four, dw);
      scale_at[c] = a.g.key_scale(0u, 0u) + (wave < 2u ? ((l & 15u) * (dim / 32u) + piece) & ~3u
                                                       : four * (dim / 8u) + (dw >> 2) * 4u);
#pragma unroll
      for (uint32_t p = 0; p < 2; ++p) {
        uint32_t mine = 4u * c + (two ? 2u * h + p : h);
        if (mine >= dim / 32u) mine = 0;
        key_shift[c][p] = 8u * (((m & 15u) * (dim / 32u) + mine) & 3u);
      }
    }
    const uint32_t row = row0 + m;
    const bool real = row < rows;
    from = to = 0;
    if (real) {
      from = first_key(a, position(a, at, row, length));
      to = end_key(a, position(a, at, row, length));
    }
    const uint32_t token = real ? row / a.per : 0u, qh = real ? row - token * a.per : 0u;
    const uint8_t *qr = a.q + ((uint64_t)((uint32_t)at.first + token) * a.q_stride +
                               (uint64_t)(head * a.per + qh) * dim) * T::kBytes;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int b = 0; b < 4 * pieces(c); ++b) {
        const uint32_t e = 128u * c + 32u * (uint32_t)pieces(c) * h + 8u * b;
        const bool on = real && e < dim;
        if constexpr (kN == 1) {
          u32x4_t w = {0, 0, 0, 0};
          if (on) w = *reinterpret_cast<const u32x4_t *>(qr + e * 2u);
          q[c][b][0] = w;
        } else {
          float x[8] = {};
          if (on) load8<T>(qr + e * T::kBytes, x);
          uint32_t w[4][kN];
#pragma unroll
          for (int j = 0; j < 4; ++j) split_query<kN>(x[2 * j], x[2 * j + 1], w[j]);
#pragma unroll
          for (int j = 0; j < kN; ++j) q[c][b][j] = (u32x4_t){w[0][j], w[1][j], w[2][j], w[3][j]};
        }
      }
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 2 * pieces(c); ++e)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][e][i] = 0.0f;
    sum = 0.0f;
    wild = 0;
    top = kLowest;
  }

  // The wave's quarter of the step at t into a part of the ring: waves 0 and 1 the first and
  // second 16 keys, 2 and 3 values; `page`: own_page(t).
  __device__ __forceinline__ uint32_t own_page(uint32_t t) const {
    return page_id(a, pages, t + 16u * (wave & 1u));
  }
  __device__ __forceinline__ void request(uint32_t t, uint32_t stage, uint32_t page) const {
    const uint32_t row = (t + 16u * (wave & 1u)) & (a.g.page_rows() - 1u);
    // (page 0 in the place of one that is not there: memory that is)
    const auto r = rsrc(base + (uint64_t)(page < a.g.n_pages ? page : 0u) * a.page_bytes,
                        a.g.head_bytes());
    const uint32_t codes = a.g.key_code(row, 0u), scales = row * (a.g.dim / 32u);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      uint8_t *to = lds + stage + c * kPart;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t *)(to + wave * 1024u), 16,
                                               (int)code_at[c], (int)codes, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t *)(to + 4096u + wave * 256u), 4,
                                               (int)scale_at[c], (int)scales, 0, 0);
    }
  }

  __device__ __forceinline__ f32x16_t scores(uint32_t stage) const {
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int p = 0; p < pieces(c); ++p) {
        const uint32_t at0 = (pieces(c) == 2 ? 2u * h + p : h) * 16u + (m & 15u);
        const uint8_t *part = lds + stage + c * kPart;
        const u32x4_t w = *reinterpret_cast<const u32x4_t *>(part + (m >> 4) * 1024u + at0 * 16u);
        const uint32_t sc =
            *reinterpret_cast<const uint32_t *>(part + 4096u + (m >> 4) * 256u + at0 * 4u);
        const float scale = scale_of(sc >> key_shift[c][p], 0);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const u32x4_t key = {M::template codes<0>(w[b], scale), M::template codes<1>(w[b], scale),
                               M::template codes<2>(w[b], scale), M::template codes<3>(w[b], scale)};
#pragma unroll
          for (int j = 0; j < kN; ++j) s = M::mfma32(key, q[c][4 * p + b][j], s);
        }
      }
    return s;
  }

  // The wave's share of a step's values: 16 keys (u) and, of chunk c, two products' elements of
  // each (waves 1 and 3 have none of the last 64).
  struct Share {
    u32x4_t codes[kChunks][2];
    uint32_t scales[kChunks][2];
  };
  __device__ __forceinline__ void fetch(Share &v, uint32_t stage) const {
    const uint32_t u = wave >> 1;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const bool two = pieces(c) == 2;
      const uint32_t dw = two ? m >> 1 : m >> 2, across = two ? 16u : 8u;
      const uint8_t *part = lds + stage + c * kPart;
#pragma unroll
      for (uint32_t x = 0; x < 2; ++x) {
        const uint32_t at0 = (2u * x + h) * across + dw;
        v.codes[c][x] = *reinterpret_cast<const u32x4_t *>(part + 2048u + u * 1024u + at0 * 16u);
        v.scales[c][x] = *reinterpret_cast<const uint32_t *>(part + 4608u + u * 256u + at0 * 4u);
      }
    }
  }
  // 0, whatever bytes they have: those of the step at t beyond the last key, of a page that is not
  // there, and with `careful` blocks that are not finite.
  __device__ __forceinline__ void hide(Share &v, uint32_t t, bool careful) const {
    const uint32_t u = wave >> 1;
    const bool there = page_id(a, pages, t + 16u * u) < a.g.n_pages;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (uint32_t x = 0; x < 2; ++x) {
        u32x4_t w = v.codes[c][x];
        uint32_t sc = 0;
#pragma unroll
        for (uint32_t b = 0; b < 4; ++b) {
          bool keep = there && t + 16u * u + 8u * x + 4u * h + b < end;
          keep = keep && !(careful && (v.scales[c][x] >> (8u * b) & 255u) > M::kLastScale);
          w[b] = keep ? w[b] : 0u;
          sc |= (keep ? v.scales[c][x] & 255u << (8u * b) : 127u << (8u * b));
        }
        v.codes[c][x] = w;
        v.scales[c][x] = sc;
      }
  }
  // Their fragments.
  __device__ __forceinline__ void make(const Share &v, uint8_t *frags) const {
    const uint32_t u = wave >> 1, byte = wave & 1u;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const bool two = pieces(c) == 2;
      const uint32_t shift = two ? 8u * byte + 16u * (m & 1u) : 8u * (m & 3u);
      u32x4_t even, odd, codes[2] = {v.codes[c][0] >> shift, v.codes[c][1] >> shift};
      pair<T>(codes, v.scales[c], even, odd);
      u32x4_t *out = reinterpret_cast<u32x4_t *>(frags) +
                     (8u * c + (two ? 4u : 2u) * u + 2u * byte) * 64u + lane;
      if (two || byte == 0u) {
        out[0] = even;
        out[64] = odd;
      }
    }
  }

  __device__ __forceinline__ int32_t key_of(uint32_t t, int i) const {
    return (int32_t)(t + 8u * (i >> 2) + 4u * h + (i & 3));
  }
  // Scores of keys that the row does not see: -inf.  Bit i: it sees score i's.
  __device__ __forceinline__ uint32_t mask(uint32_t t, f32x16_t &s) const {
    const bool there[2] = {page_id(a, pages, t) < a.g.n_pages,
                           page_id(a, pages, t + 16u) < a.g.n_pages};
    uint32_t seen = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool on = there[i >> 3] && key_of(t, i) >= from && key_of(t, i) < to;
      seen |= (on ? 1u : 0u) << i;
      s[i] = on ? s[i] : -__builtin_inff();
    }
    return seen;
  }
  // NaN for the rows that see a block that is not finite: a product of the blocks' and the keys'
  // flags finds them.  (Its scales are read again: the ring may have gone on.)
  __device__ __forceinline__ void poison(uint32_t t, uint32_t seen) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const bool two = pieces(c) == 2;
      uint32_t dw = 16u * c + (two ? m >> 1 : m >> 2);
      if (dw >= a.g.dim / 8u) dw = 0;
      f32x16_t nan;
#pragma unroll
      for (int i = 0; i < 16; ++i) nan[i] = 0.0f;
#pragma unroll
      for (uint32_t u = 0; u < 2; ++u) {
        const uint32_t page = page_id(a, pages, t + 16u * u);
        const uint8_t *vh = a.v + (uint64_t)head * a.g.head_bytes() +
                            (uint64_t)(page < a.g.n_pages ? page : 0u) * a.page_bytes;
        const uint32_t row = (t + 16u * u) & (a.g.page_rows() - 1u);
        uint32_t bad = 0;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          const uint32_t sc = vh[a.g.value_scale(row + 8u * (j >> 2) + 4u * h + (j & 3u), dw >> 2)];
          bad |= (sc > M::kLastScale ? 1u : 0u) << j; // (of keys that are seen, see below)
        }
        nan = mfma32_bf16(flags(bad), flags(seen >> (8u * u)), nan);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) wild |= (nan[4 * i] > 0.0f ? 1u : 0u) << (4 * c + i);
    }
  }

  static __device__ __forceinline__ float highest(const f32x16_t &s) {
    float most = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) most = __builtin_fmaxf(most, s[i]);
    return most;
  }
  __device__ __forceinline__ bool over(const f32x16_t &s) const {
    return __ballot(__builtin_fmaf(highest(s), a.c, -top) > kSlack + M::kBias) != 0u;
  }
  __device__ __forceinline__ void raise(const f32x16_t &s) {
    if (!over(s)) return;
    float x = highest(s);
    x = __builtin_fmaxf(x, __shfl_xor(x, 32)) * a.c - M::kBias;
    const float now = x - top > kSlack ? x : top;
    const float f = __builtin_amdgcn_exp2f(top - now);
    top = now;
    sum *= f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 2 * pieces(c); ++e) o[c][e] *= f;
  }

  // The weights of 16 keys each, and the lane's sum of them as they are multiplied: above
  // kMost if a score passed its row's maximum by more than the slack.
  static constexpr float kMost = M::kBias > 0.0f ? 32768.0f : 4096.0f;
  __device__ __forceinline__ float weights(const f32x16_t &s, u32x4_t (&weight)[2][kN]) const {
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      uint32_t w[kN];
      M::weights(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.c, -top)),
                 __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + 1], a.c, -top)), w);
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        weight[i >> 3][j][i >> 1 & 3] = w[j];
        part = M::add2(w[j], part);
      }
    }
    return part;
  }

  // What a wave has asked for of the steps up to the next one has landed, all but what it asked
  // for of kBehind behind that, and so, behind the barrier, has everyone's; fragments that it
  // wrote are there, those that it read are read.
  template <int kBehind> static __device__ __forceinline__ void wait() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kBehind * kLoads) : "memory");
  }

  // Whether the pages of all keys are there.
  __device__ __forceinline__ bool dense() const {
    bool all = true;
    for (uint32_t slot = (begin >> a.g.page_shift) + lane; slot <= (end - 1u) >> a.g.page_shift;
         slot += 64u)
      all = all && (uint32_t)pages[slot] < a.g.n_pages;
    return __ballot(!all) == 0u;
  }

  // `slow`: every step is looked at (careful, or some pages are not there).
  __device__ __forceinline__ void pass(bool careful, bool slow) {
#pragma unroll
    for (uint32_t i = 0; i < kRing; ++i)
      request(begin + 32u * i, i * kStage, own_page(begin + 32u * i));
    uint32_t page = own_page(begin + 32u * kRing);
    wait<kRing - 1>();
    uint8_t *frags = lds + kFrags, *other = frags + kHalf;
    Share v;
    fetch(v, 0u);
    if (slow || begin + 32u > end) hide(v, begin, careful);
    make(v, frags);
    f32x16_t s = scores(0u);
    wait<kRing - 2>();
    uint32_t t = begin, stage = 0; // the step at t is in `stage`, its fragments in `frags`
    // steps from `all_from` on whose next one starts up to here need no look
    uint32_t plain = all_to < end ? all_to : end;
    plain = slow || end < 64u ? 0u : plain + 32u > end ? end - 32u : plain;
    do {
      if (slow || t < all_from || t + 32u > all_to) {
        const uint32_t seen = mask(t, s);
        if (careful) poison(t, seen);
      }
      raise(s);
      u32x4_t weight[2][kN];
      sum += weights(s, weight);
      bool look = slow || t + 64u > end, more;
      do { // a loop of its own where only the products change the sums: they stay in place
        request(t + 32u * kRing, stage, page);
        t += 32u;
        page = own_page(t + 32u * kRing);
        stage = stage == (kRing - 1u) * kStage ? 0u : stage + kStage;
        fetch(v, stage);
        if (look) hide(v, t, careful);
        const u32x4_t *mine = reinterpret_cast<const u32x4_t *>(frags) + lane;
        u32x4_t value[kTiles];
#pragma unroll
        for (int e = 0; e < (int)kTiles; ++e) {
          value[e] = mine[64 * e];
          const int c = e / 8, half = 2 * pieces(c), u = e % 8 / half, k = e % half;
#pragma unroll
          for (int j = 0; j < kN; ++j) o[c][k] = M::mfma32(value[e], weight[u][j], o[c][k]);
        }
        make(v, other);
        s = scores(stage);
        uint8_t *was = frags;
        frags = other;
        other = was;
        wait<kRing - 2>();
        look = false;
        more = t >= all_from && t + 32u <= plain;
        if (more) {
          const float part = weights(s, weight);
          more = __ballot(part > kMost) == 0u;
          if (more) sum += part;
        }
      } while (more);
    } while (t < end);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // nothing is on its way to LDS any more
  }

  __device__ __forceinline__ void run(uint32_t group, float *floats) {
    at = locate(a, group, kGroupRows);
    if (at.seq < 0) return; // the whole workgroup
    at.seq = __builtin_amdgcn_readfirstlane(at.seq);
    lds = reinterpret_cast<uint8_t *>(floats);
    start(max(((const_i32)a.lengths)[at.seq], 0));
    bool careful = false;
    const bool gaps = begin < end && !dense();
    for (;;) {
      clear();
      if (begin < end) pass(careful, careful || gaps);
      if (careful) break;
      // finite, or once more
      float x = 0.0f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int e = 0; e < 2 * pieces(c); ++e)
#pragma unroll
          for (int i = 0; i < 16; ++i) x = __builtin_fmaf(o[c][e][i], 0.0f, x);
      careful = __ballot(x != 0.0f) != 0u;
      __syncthreads(); // (LDS is read)
      if (threadIdx.x == 0u) floats[0] = 0.0f;
      __syncthreads();
      if (careful) floats[0] = 1.0f;
      __syncthreads();
      careful = __builtin_amdgcn_readfirstlane((int)(floats[0] != 0.0f)) != 0;
      if (!careful) break;
      __syncthreads(); // (the flag is read)
    }
    const uint32_t row = row0 + m;
    const float total = sum + __shfl_xor(sum, 32);
    if (row >= rows) return;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < pieces(c); ++j) {
          const bool two = pieces(c) == 2;
          const uint32_t e0 = 128u * c + (two ? 32u * i + 16u * h + 8u * j : 16u * i + 8u * h);
          if (e0 >= a.g.dim) continue;
          float x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float v = two ? o[c][k & 3][4 * i + 2 * j + (k >> 2)] : o[c][k & 1][4 * i + (k >> 1)];
            x[k] = wild >> (4 * c + i) & 1u ? __builtin_nanf("") : v;
          }
          store_row<T>(a, at, head, split, row, e0, x, top, total, e0 == 0u);
        }
  }
};

// ---------------------------------------------------------------------------
// The splits' parts of a row, added: kWaves waves a row, each at most 64 parts, whose maxima
// and sums are a lane's each; kAcross lanes (of 4 elements) a part, the others beside them, all
// parts of 8 rounds in flight together with the maxima.  16 rows of 47 parts, 128 elements 2.0 us
// less than with one wave that reads the maxima first; up to 8 parts of a row, one wave is as fast, and four
// rows a workgroup are fewer workgroups.
// ---------------------------------------------------------------------------
template <class T, int kWaves, int kAcross>
__device__ __forceinline__ void combine_body(const float *ws, const int32_t *starts, uint8_t *y,
                                             uint32_t n_tokens, uint32_t n_seqs, uint32_t n_heads,
                                             uint32_t dim, uint32_t y_stride, uint32_t splits,
                                             float *lds) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, part = wave % kWaves;
  const uint64_t n = (uint64_t)n_tokens * n_heads;
  const uint32_t id = blockIdx.x * (4u / kWaves) + wave / kWaves; // (below 2^31)
  const uint32_t token = id / n_heads, h = id - token * n_heads;
  bool real = id < n;
  if (real && starts) real = (int32_t)token >= starts[0] && (int32_t)token < starts[n_seqs];
  // the wave's parts
  const uint32_t each = (splits + kWaves - 1u) / kWaves, s0 = part * each;
  const uint32_t mine = s0 < splits ? (splits - s0 < each ? splits - s0 : each) : 0u;
  float top = kLowest, total = 0.0f;
  if (real && lane < mine) {
    const float *ms = ws + 2u * ((uint64_t)(s0 + lane) * n + id);
    top = ms[0];
    total = ms[1];
  }
  const uint32_t at = lane % kAcross, beside = lane / kAcross, e = 4u * at;
  constexpr uint32_t kBeside = 64u / kAcross, kRound = 8u * kBeside;
  const float *parts = ws + parts_at(n, splits);
  f32x4_t v[8];
  auto ask = [&](uint32_t s) {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t k = s + kBeside * i + beside;
      v[i] = (f32x4_t){0, 0, 0, 0};
      if (real && k < mine && e < dim)
        v[i] = *reinterpret_cast<const f32x4_t *>(parts + ((uint64_t)(s0 + k) * n + id) * dim + e);
    }
  };
  ask(0u);
  const uint64_t has = __ballot(total != 0.0f); // (or NaN; what empty parts hold is not used)
  float most = has >> lane & 1u ? top : kLowest;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) most = __builtin_fmaxf(most, __shfl_xor(most, d));
  const float f = has >> lane & 1u ? __builtin_amdgcn_exp2f(top - most) : 0.0f;
  total *= f;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
  f32x4_t x = {0, 0, 0, 0};
  for (uint32_t s = 0; s < mine; s += kRound) {
    if (s) ask(s);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t k = s + kBeside * i + beside;
      const float g = __shfl(f, (int)(k < 64u ? k : 63u));
      const bool on = k < mine && (has >> k & 1u);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(on ? v[i][j] : 0.0f, on ? g : 0.0f, x[j]);
    }
  }
#pragma unroll
  for (int d = kAcross; d < 64; d <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += __shfl_xor(x[j], d);
  if constexpr (kWaves > 1) { // the waves' sums, in their order
    if (beside == 0u) reinterpret_cast<f32x4_t *>(lds)[wave * kAcross + at] = x;
    float *tops = lds + 4u * 4u * kAcross;
    if (lane == 0u) {
      tops[wave] = most;
      tops[4u + wave] = total;
    }
    __syncthreads();
    if (part) return;
    float all = tops[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) all = __builtin_fmaxf(all, tops[w]);
    x = (f32x4_t){0, 0, 0, 0};
    total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float g = __builtin_amdgcn_exp2f(tops[w] - all);
      const f32x4_t v = reinterpret_cast<const f32x4_t *>(lds)[w * kAcross + at];
      total += tops[4 + w] * g;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(v[j], g, x[j]);
    }
  }
  if (!real || beside || e >= dim) return;
  const float g = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = total == 0.0f ? 0.0f : x[j] * g;
  uint8_t *to = y + ((uint64_t)token * y_stride + (uint64_t)h * dim + e) * T::kBytes;
  if constexpr (T::kBytes == 4u) *reinterpret_cast<f32x4_t *>(to) = x;
  else *reinterpret_cast<u32x2_t *>(to) = (u32x2_t){pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
}

} // namespace

#define AXH_ATTEND(KIND, DIM, NAME, WAVES, SPLIT, ...)                                            \
  extern "C" __global__ void __launch_bounds__(256)                                               \
      __attribute__((amdgpu_waves_per_eu(WAVES, WAVES)))                                          \
      axh_kv_attention_##KIND##_d##DIM##_##NAME(                                                  \
          const uint8_t *q, const uint8_t *k, const uint8_t *v, const int32_t *starts,            \
          const int32_t *lengths, const int32_t *table, uint8_t *y, float *ws, uint32_t n_seqs,   \
          uint32_t n_tokens, uint32_t max_pages, uint32_t n_pages, uint32_t page_shift,           \
          uint32_t kv_heads, uint32_t head_dim, uint32_t per, uint32_t q_stride,                  \
          uint32_t y_stride, uint32_t c, uint32_t window, uint32_t chunk, uint32_t n_splits,      \
          uint32_t page_bytes) {                                                                  \
    using A = __VA_ARGS__;                                                                        \
    __shared__ alignas(16) float lds[A::kLds];                                                    \
    const uint32_t splits = SPLIT ? n_splits : 1u;                                                \
    const Args args{q, k, v, starts, lengths, table, y, ws, n_seqs, n_tokens, max_pages,          \
                    Geometry{n_pages, page_shift, kv_heads, head_dim}, per, q_stride, y_stride,   \
                    __builtin_bit_cast(float, c), window, chunk, splits, page_bytes};             \
    /* workgroups of a head share an XCD and its cache where heads are as many as XCDs; the */    \
    /* last rows of a sequence, which see most keys, are begun first */                           \
    const uint32_t rest = blockIdx.x / kv_heads;                                                  \
    const uint32_t group = gridDim.x / kv_heads / splits - 1u - rest / splits;                    \
    A(args, blockIdx.x % kv_heads, rest % splits).run(group, lds);                                \
  }
#define AXH_FEW(DIM, NAME, T, WAVES) AXH_ATTEND(few, DIM, NAME, WAVES, true, Few<T, DIM, 1>)
#define AXH_MORE(DIM, NAME, T, WAVES) AXH_ATTEND(more, DIM, NAME, WAVES, false, Few<T, DIM, 2>)
#define AXH_MANY(DIM, NAME, T, WAVES) AXH_ATTEND(many, DIM, NAME, WAVES, false, Many<T, DIM>)
#define AXH_COMBINE(WAVES, DIM, NAME, T)                                                          \
  extern "C" __global__ void __launch_bounds__(256) axh_kv_combine_w##WAVES##_d##DIM##_##NAME(    \
      const float *ws, const int32_t *starts, uint8_t *y, uint32_t n_tokens, uint32_t n_seqs,     \
      uint32_t n_heads, uint32_t dim, uint32_t y_stride, uint32_t splits) {                       \
    __shared__ alignas(16) float lds[WAVES > 1 ? 4 * DIM + 8 : 4];                                \
    combine_body<T, WAVES, DIM / 4>(ws, starts, y, n_tokens, n_seqs, n_heads, dim, y_stride,      \
                                    splits, lds);                                                 \
  }
// The attention's last argument: waves a SIMD, as many as the registers of its sums and operands
// leave room for.
#define AXH_KINDS16(NAME, T)                                                                      \
  AXH_FEW(64, NAME, T, 4)                                                                         \
  AXH_FEW(128, NAME, T, 4)                                                                        \
  AXH_FEW(192, NAME, T, 2)                                                                        \
  AXH_FEW(256, NAME, T, 2)                                                                        \
  AXH_MORE(64, NAME, T, 3)                                                                        \
  AXH_MORE(128, NAME, T, 2)                                                                       \
  AXH_MANY(64, NAME, T, 3)                                                                        \
  AXH_MANY(128, NAME, T, 3)                                                                       \
  AXH_MANY(192, NAME, T, 2)                                                                       \
  AXH_MANY(256, NAME, T, 1)
#define AXH_COMBINES(NAME, T)                                                                     \
  AXH_COMBINE(1, 64, NAME, T)                                                                     \
  AXH_COMBINE(1, 128, NAME, T)                                                                    \
  AXH_COMBINE(1, 256, NAME, T)                                                                    \
  AXH_COMBINE(4, 64, NAME, T)                                                                     \
  AXH_COMBINE(4, 128, NAME, T)                                                                    \
  AXH_COMBINE(4, 256, NAME, T)
AXH_KINDS16(bf16, TBF16)
AXH_KINDS16(f16, TF16)
AXH_FEW(64, f32, TF32, 3)
AXH_FEW(128, f32, TF32, 2)
AXH_FEW(192, f32, TF32, 2)
AXH_FEW(256, f32, TF32, 1)
AXH_MANY(64, f32, TF32, 2)
AXH_MANY(128, f32, TF32, 1)
AXH_MANY(192, f32, TF32, 1)
AXH_MANY(256, f32, TF32, 1)
AXH_COMBINES(bf16, TBF16)
AXH_COMBINES(f16, TF16)
AXH_COMBINES(f32, TF32)
