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
// Codes become bf16, exactly, by the converting instruction, which takes the scale.  A q
// that is not bf16 is two (f16) or three (f32) bf16 terms that add up to it, and so are
// the softmax's weights, each term rounded: within 2^-16 and 2^-24, and 2^-8 for bf16.
//
// The running maximum of a row moves only when a score passes it by 2^8: the weights
// stay below 2^8 (f32 sums, and bf16 has f32's range), and the sums need no rescaling in
// almost all steps, nor the four lanes of a row an exchange of their maxima.
#include "kv_common.h"

using namespace axh;

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(4))) int32_t *const_i32;

// 16-bit halves of two dwords: {low a, low b} and {high a, high b}.
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
// The two codes of byte kByte times 2^(e - 127), e the exponent field of `scale`, as bf16.
template <int kByte> __device__ __forceinline__ uint32_t fp4_bf16(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, kByte));
}
__device__ __forceinline__ bf16x8_t frag(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(bf16x8_t, (u32x4_t){a, b, c, d});
}
__device__ __forceinline__ f32x4_t mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

constexpr float kLowest = -3e38f; // below every score, and finite: no -inf less -inf
constexpr float kSlack = 8.0f;    // how far (log2) a score may pass its row's maximum

// bf16 terms of an operand.
template <class T> struct Terms;
template <> struct Terms<TBF16> { static constexpr int kN = 1; };
template <> struct Terms<TF16> { static constexpr int kN = 2; };
template <> struct Terms<TF32> { static constexpr int kN = 3; };

// Two weights as kN dwords of bf16 terms, each the rest of the ones before, rounded.
template <int kN> __device__ __forceinline__ void split_pair(float a, float b, uint32_t *w) {
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
// Two elements of q as kN dwords of bf16 terms, cut off, so that they add up exactly; an
// infinity or a NaN is its own first term, and the others are 0.
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

// The codes and scales of a step's two tiles of 16 keys, as a lane has them.
template <int kChunks> struct Raw {
  u32x4_t k[2][kChunks], v[2][kChunks];
  uint32_t ks[2][kChunks], vs[2][kChunks];
};
// Pages of a step's two tiles; outside 0 .. n_pages - 1: not there.
struct Pages {
  uint32_t id[2];
};

template <class T, int kChunks, int kRows, bool kSplitKeys> struct Attend {
  static constexpr int kN = Terms<T>::kN;
  static constexpr uint32_t kGroupRows = 16u * kRows * (kSplitKeys ? 1u : 4u);
  static constexpr uint32_t kStep = kSplitKeys ? 128u : 32u; // keys of a workgroup's step

  const Args &a;
  uint32_t lane, wave, m, grp; // lane = 16 grp + m
  uint32_t kp[kChunks], vd[kChunks]; // the lane's piece of a key, dword of a value
  const uint8_t *kh, *vh; // the head's part of page 0
  int32_t seq;

  bf16x8_t q[kRows][kChunks][4][kN];
  f32x4_t o[kRows][kChunks][8];
  float top[kRows], sum[kRows]; // log2 of the running maximum's weight, the lane's sum
  int32_t pos[kRows];           // position of the lane's row, -1: no row

  __device__ __forceinline__ explicit Attend(const Args &args) : a(args) {}

  __device__ __forceinline__ Pages pages(uint32_t t) const {
    Pages p;
#pragma unroll
    for (int T16 = 0; T16 < 2; ++T16) {
      const uint32_t slot = (t + 16u * T16) >> a.g.page_shift;
      p.id[T16] = ~0u;
      if (slot < a.max_pages)
        p.id[T16] = (uint32_t)((const_i32)a.table)[(uint64_t)(uint32_t)seq * a.max_pages + slot];
    }
    return p;
  }
  __device__ __forceinline__ bool there(const Pages &p, int T16) const {
    return p.id[T16] < a.g.n_pages;
  }
  // (page 0 in the place of one that is not there: memory that is)
  __device__ __forceinline__ uint64_t offset(const Pages &p, int T16) const {
    return (uint64_t)(there(p, T16) ? p.id[T16] : 0u) * a.g.kv_heads * a.g.head_bytes();
  }
  __device__ __forceinline__ void load_keys(Raw<kChunks> &r, const Pages &p, uint32_t t) const {
#pragma unroll
    for (int T16 = 0; T16 < 2; ++T16) {
      const uint8_t *kb = kh + offset(p, T16);
      const uint32_t row = (t + 16u * T16) & (a.g.page_rows() - 1u);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        r.k[T16][c] = *reinterpret_cast<const u32x4_t *>(kb + a.g.key_code(row + m, 4u * kp[c]));
        r.ks[T16][c] = kb[a.g.key_scale(row + m, kp[c])];
      }
    }
  }
  __device__ __forceinline__ void load_values(Raw<kChunks> &r, const Pages &p, uint32_t t) const {
#pragma unroll
    for (int T16 = 0; T16 < 2; ++T16) {
      const uint8_t *vb = vh + offset(p, T16);
      const uint32_t row = (t + 16u * T16) & (a.g.page_rows() - 1u);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        r.v[T16][c] =
            *reinterpret_cast<const u32x4_t *>(vb + a.g.value_code(row + 4u * grp, vd[c]));
        r.vs[T16][c] = *reinterpret_cast<const uint32_t *>(
            vb + a.g.value_scale(row + 4u * grp, vd[c] >> 2));
      }
    }
  }

  // One step; `whole`: every row of the wave sees all of its 32 keys.  The keys, and then
  // the values, of the wave's next step (pages `ahead`) are requested as soon as the
  // registers of this one's are free.
  template <bool kWhole>
  __device__ __forceinline__ void step(Raw<kChunks> &r, const Pages &here, const Pages &ahead,
                                       uint32_t t, bool more) {
    f32x4_t s[kRows][2];
#pragma unroll
    for (int T16 = 0; T16 < 2; ++T16) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) s[i][T16] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const float scale = __builtin_bit_cast(float, r.ks[T16][c] << 23);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint32_t w = r.k[T16][c][b];
          const bf16x8_t key = frag(fp4_bf16<0>(w, scale), fp4_bf16<1>(w, scale),
                                    fp4_bf16<2>(w, scale), fp4_bf16<3>(w, scale));
#pragma unroll
          for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int j = 0; j < kN; ++j) s[i][T16] = mfma(key, q[i][c][b][j], s[i][T16]);
        }
      }
    }
    if (more) load_keys(r, ahead, t + kStep);
    uint32_t seen[kRows]; // bit 4 T16 + j: the row sees its key j of tile T16
    if constexpr (!kWhole) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        seen[i] = 0;
#pragma unroll
        for (int T16 = 0; T16 < 2; ++T16)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int32_t key = (int32_t)(t + 16u * T16 + 4u * grp + j);
            const bool on = there(here, T16) && key <= pos[i] &&
                            (a.window == 0u || (uint32_t)(pos[i] - key) < a.window);
            seen[i] |= (on ? 1u : 0u) << (4 * T16 + j);
            s[i][T16][j] = on ? s[i][T16][j] : -__builtin_inff();
          }
      }
    }
    uint32_t p[kRows][4][kN];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float most = s[i][0][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) most = __builtin_fmaxf(most, s[i][j >> 2][j & 3]);
      if (__ballot(__builtin_fmaf(most, a.c, -top[i]) > kSlack)) raise(i, most);
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][j >> 2][j & 3], a.c, -top[i]));
        sum[i] += w[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) split_pair<kN>(w[2 * j], w[2 * j + 1], p[i][j]);
    }
    bf16x8_t weight[kRows][kN];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j) weight[i][j] = frag(p[i][0][j], p[i][1][j], p[i][2][j], p[i][3][j]);
    f32x4_t nan[kRows][kChunks];
    bool any_nan = false;
    if constexpr (!kWhole) any_nan = hide(r, t, seen, nan);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      float scale[2][4];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        scale[j >> 2][j & 3] = __builtin_bit_cast(
            float, (r.vs[j >> 2][c] >> (8 * (j & 3)) & 255u) << 23);
      values<0>(r, c, scale, weight);
      values<1>(r, c, scale, weight);
      values<2>(r, c, scale, weight);
      values<3>(r, c, scale, weight);
      if (!kWhole && any_nan) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (nan[i][c][j] > 0.0f)
#pragma unroll
              for (int e = 0; e < 8; ++e) o[i][c][e][j] = __builtin_nanf("");
      }
    }
    if (more) load_values(r, ahead, t + kStep);
  }

  // Elements 8 m + 2 kB and 8 m + 2 kB + 1 of the values: pairs of keys, as the matrix
  // instruction wants them, from pairs of elements, as the codes are.
  template <int kB>
  __device__ __forceinline__ void values(const Raw<kChunks> &r, int c, const float (&scale)[2][4],
                                         const bf16x8_t (&weight)[kRows][kN]) {
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int T16 = j >> 1, e = 2 * (j & 1);
      const uint32_t x = fp4_bf16<kB>(r.v[T16][c][e], scale[T16][e]);
      const uint32_t y = fp4_bf16<kB>(r.v[T16][c][e + 1], scale[T16][e + 1]);
      lo[j] = lows(x, y);
      hi[j] = highs(x, y);
    }
    const bf16x8_t even = frag(lo[0], lo[1], lo[2], lo[3]), odd = frag(hi[0], hi[1], hi[2], hi[3]);
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        o[i][c][2 * kB] = mfma(even, weight[i][j], o[i][c][2 * kB]);
        o[i][c][2 * kB + 1] = mfma(odd, weight[i][j], o[i][c][2 * kB + 1]);
      }
  }

  // A row's maximum passed by more than the slack: a new one, the same in its four lanes.
  __device__ __forceinline__ void raise(int i, float most) {
    most = __builtin_fmaxf(most, __shfl_xor(most, 16));
    most = __builtin_fmaxf(most, __shfl_xor(most, 32));
    const float now = __builtin_fmaxf(top[i], most * a.c);
    const float f = __builtin_amdgcn_exp2f(top[i] - now);
    top[i] = now;
    sum[i] *= f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) o[i][c][e] *= f;
  }

  // Values that some row does not see.  Those of no row (beyond the length, or of a page
  // that is not there) are 0 from here on, whatever bytes they have.  A weight of 0 times a
  // NaN is no 0: NaN blocks are 0 as well, and rows that do see one are found by a
  // product of the blocks' with the keys' flags (true if there are any).
  __device__ __forceinline__ bool hide(Raw<kChunks> &r, uint32_t t, const uint32_t (&seen)[kRows],
                                       f32x4_t (&nan)[kRows][kChunks]) {
    uint32_t bad[kChunks];
    uint32_t any = 0;
    uint32_t some = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) some |= seen[i];
    // a key is a row's own: look at all sixteen rows (four lanes hold four keys each)
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) some |= (uint32_t)__shfl_xor((int)some, d);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      bad[c] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int T16 = j >> 2, e = j & 3;
        const bool drop = !(some >> j & 1u);
        const bool is_nan = !drop && (r.vs[T16][c] >> (8 * e) & 255u) == 255u;
        bad[c] |= (is_nan ? 1u : 0u) << j;
        if (drop || is_nan) {
          r.v[T16][c][e] = 0u;
          r.vs[T16][c] = (r.vs[T16][c] & ~(255u << (8 * e))) | 127u << (8 * e);
        }
      }
      any |= bad[c];
    }
    if (!__ballot(any != 0u)) return false;
    auto flags = [](uint32_t bits) { // eight bits as eight 1.0 or 0.0
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = (bits >> (2 * j) & 1u ? 0x3F80u : 0u) | (bits >> (2 * j + 1) & 1u ? 0x3F800000u : 0u);
      return frag(w[0], w[1], w[2], w[3]);
    };
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        nan[i][c] = mfma(flags(bad[c]), flags(seen[i]), (f32x4_t){0, 0, 0, 0});
    return true;
  }

  __device__ __forceinline__ void run(float *lds) {
    lane = threadIdx.x & 63u;
    wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    m = lane & 15u;
    grp = lane >> 4;
    // workgroups of a head share an XCD and its cache where heads are as many as XCDs
    const uint32_t head = blockIdx.x % a.g.kv_heads, rest = blockIdx.x / a.g.kv_heads;
    const uint32_t split = rest % a.splits;
    const Group at = locate(a, rest / a.splits, kGroupRows);
    if (at.seq < 0) return; // the whole workgroup
    seq = __builtin_amdgcn_readfirstlane(at.seq);
    const int32_t length = ((const_i32)a.lengths)[seq];
    const uint32_t rows = (uint32_t)at.tokens * a.per;
    const uint32_t row0 = at.tile * kGroupRows + (kSplitKeys ? 0u : wave * 16u * kRows);
    // positions of the wave's first and last rows (p: of the sequence's new token 0)
    const int32_t p0 = length - at.tokens;
    auto position = [&](uint32_t row) { return p0 + (int32_t)(row / a.per); };
    const uint32_t last = row0 + 16u * kRows < rows ? row0 + 16u * kRows : rows;
    const bool none = row0 >= rows;
    const int32_t pos_lo = none ? -1 : position(row0), pos_hi = none ? -1 : position(last - 1u);

    const uint32_t pieces = a.g.dim / 32u;
    const uint64_t head_at = (uint64_t)head * a.g.head_bytes();
    kh = a.k + head_at;
    vh = a.v + head_at;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      // elements from dim on: others in their place, times a q of 0, or never stored
      kp[c] = grp + 4u * c < pieces ? grp + 4u * c : 0u;
      vd[c] = m + 16u * c < 4u * pieces ? m + 16u * c : 0u;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const uint32_t row = row0 + 16u * i + m;
      const bool real = row < rows;
      pos[i] = real ? position(row) : -1;
      const uint32_t token = real ? row / a.per : 0u, h = real ? row - token * a.per : 0u;
      const uint8_t *qr = a.q + ((uint64_t)((uint32_t)at.first + token) * a.q_stride +
                                 (uint64_t)(head * a.per + h) * a.g.dim) * T::kBytes;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const bool on = real && grp + 4u * c < pieces;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if constexpr (kN == 1) {
            u32x4_t w = {0, 0, 0, 0};
            if (on) w = *reinterpret_cast<const u32x4_t *>(qr + (32u * (grp + 4u * c) + 8u * b) * 2u);
            q[i][c][b][0] = __builtin_bit_cast(bf16x8_t, w);
          } else {
            float x[8] = {};
            if (on) load8<T>(qr + (32u * (grp + 4u * c) + 8u * b) * T::kBytes, x);
            uint32_t w[4][kN];
#pragma unroll
            for (int j = 0; j < 4; ++j) split_query<kN>(x[2 * j], x[2 * j + 1], w[j]);
#pragma unroll
            for (int j = 0; j < kN; ++j)
              q[i][c][b][j] = frag(w[0][j], w[1][j], w[2][j], w[3][j]);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) o[i][c][e] = (f32x4_t){0, 0, 0, 0};
      }
      top[i] = kLowest;
      sum[i] = 0.0f;
    }

    // Keys of the workgroup: from the first that its first row sees, in whole steps, its
    // split of them; of the wave: to the last that its last row sees.
    const int32_t capacity = (int32_t)(a.max_pages << a.g.page_shift);
    const uint32_t first_row = at.tile * kGroupRows;
    int32_t begin = first_row < rows ? position(first_row) : 0;
    begin = a.window && begin >= (int32_t)a.window ? begin - (int32_t)a.window + 1 : 0;
    begin &= ~31;
    int32_t end = pos_hi + 1;
    if (end > length) end = length;
    if (end > capacity) end = capacity;
    const uint64_t from = (uint64_t)(uint32_t)begin + (uint64_t)split * a.chunk;
    uint32_t to = end > 0 ? (uint32_t)end : 0u;
    if (split + 1u < a.splits && from + a.chunk < to) to = (uint32_t)(from + a.chunk);
    uint32_t t = from < to ? (uint32_t)from + (kSplitKeys ? 32u * wave : 0u) : to;
    if (t < to) {
      Raw<kChunks> r;
      Pages here = pages(t), ahead = pages(t + kStep);
      load_keys(r, here, t);
      load_values(r, here, t);
      for (; t < to; t += kStep) {
        const Pages later = pages(t + 2u * kStep);
        const bool more = t + kStep < to;
        if (there(here, 0) && there(here, 1) && (int32_t)(t + 31u) <= pos_lo &&
            (a.window == 0u || pos_hi - (int32_t)t < (int32_t)a.window))
          step<true>(r, here, ahead, t, more);
        else
          step<false>(r, here, ahead, t, more);
        here = ahead;
        ahead = later;
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      sum[i] += __shfl_xor(sum[i], 16);
      sum[i] += __shfl_xor(sum[i], 32);
    }
    if constexpr (kSplitKeys) join(lds, at, head, split, rows, row0);
    else finish(at, head, split, rows, row0);
  }

  // Rows of the output, or of a split's part, go by (token, head).
  __device__ __forceinline__ uint64_t out_row(const Group &at, uint32_t head, uint32_t row,
                                              uint32_t &token, uint32_t &h) const {
    const uint32_t n = row / a.per;
    token = (uint32_t)at.first + n;
    h = head * a.per + row - n * a.per;
    return (uint64_t)token * (a.g.kv_heads * a.per) + h;
  }
  // Eight elements of a row from e0 on: the output, or a part with its maximum and sum.
  __device__ __forceinline__ void store(const Group &at, uint32_t head, uint32_t split,
                                        uint32_t row, uint32_t e0, float *x, float maximum,
                                        float total, bool lead) const {
    uint32_t token, h;
    const uint64_t id = out_row(at, head, row, token, h);
    if (a.splits == 1u) {
      const float f = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = total == 0.0f ? 0.0f : x[j] * f;
      store8<T>(a.y + ((uint64_t)token * a.y_stride + (uint64_t)h * a.g.dim + e0) * T::kBytes, x);
      return;
    }
    const uint64_t n = (uint64_t)a.n_tokens * a.g.kv_heads * a.per;
    const uint64_t part = (uint64_t)split * n + id;
    if (lead) {
      float *ms = a.ws + 2u * part;
      ms[0] = maximum;
      ms[1] = total;
    }
    if (total != 0.0f) // (or NaN; an empty part's elements are not read)
      store8<TF32>(reinterpret_cast<uint8_t *>(a.ws + parts_at(n, a.splits) + part * a.g.dim + e0), x);
  }

  __device__ __forceinline__ void finish(const Group &at, uint32_t head, uint32_t split,
                                         uint32_t rows, uint32_t row0) const {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const uint32_t row = row0 + 16u * i + m;
      if (row >= rows) continue;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        if (32u * (grp + 4u * c) < a.g.dim)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = o[i][c][e][j];
            store(at, head, split, row, 32u * (grp + 4u * c) + 8u * j, x, top[i], sum[i],
                  c == 0 && j == 0 && grp == 0u);
          }
    }
  }

  // The four waves' parts of the same rows, added in LDS: sixteen rows at a time.
  static constexpr uint32_t kPitch = 128u * kChunks + 4u; // floats of a row
  static constexpr uint32_t kLds = 4u * 16u * (kPitch + 2u);
  __device__ __forceinline__ void join(float *lds, const Group &at, uint32_t head, uint32_t split,
                                       uint32_t rows, uint32_t row0) const {
    float *tops = lds + 4u * 16u * kPitch, *sums = tops + 64u;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (i) __syncthreads();
      if (grp == 0u) {
        tops[16u * wave + m] = top[i];
        sums[16u * wave + m] = sum[i];
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float *to = lds + (16u * wave + m) * kPitch + 128u * c + 32u * grp + 8u * j;
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = o[i][c][e][j];
          store8<TF32>(reinterpret_cast<uint8_t *>(to), x);
        }
      __syncthreads();
      const uint32_t r = threadIdx.x >> 4, row = row0 + 16u * i + r;
      if (row >= rows) continue;
      float most = tops[r], total = 0.0f, f[4];
#pragma unroll
      for (uint32_t w = 1; w < 4; ++w) most = __builtin_fmaxf(most, tops[16u * w + r]);
#pragma unroll
      for (uint32_t w = 0; w < 4; ++w) {
        f[w] = __builtin_amdgcn_exp2f(tops[16u * w + r] - most);
        total += sums[16u * w + r] * f[w];
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const uint32_t e0 = 128u * c + 8u * (threadIdx.x & 15u);
        if (e0 >= a.g.dim) continue;
        float x[8] = {};
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
          float y[8];
          load8<TF32>(reinterpret_cast<const uint8_t *>(lds + (16u * w + r) * kPitch + e0), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(y[e], f[w], x[e]);
        }
        store(at, head, split, row, e0, x, most, total, e0 == 0u);
      }
    }
  }
};

// ---------------------------------------------------------------------------
// The splits' parts of a row, added: a workgroup a row, dim / 4 lanes a part of it, the
// others beside them, joined in LDS in the splits' order.
// ---------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ void combine_body(const float *ws, const int32_t *starts, uint8_t *y,
                                             uint32_t n_tokens, uint32_t n_seqs, uint32_t n_heads,
                                             uint32_t dim, uint32_t y_stride, uint32_t splits,
                                             float *lds) {
  const uint32_t id = blockIdx.x, token = id / n_heads, h = id - token * n_heads;
  if (starts && ((int32_t)token < starts[0] || (int32_t)token >= starts[n_seqs])) return;
  const uint64_t n = (uint64_t)n_tokens * n_heads;
  const float *parts = ws + parts_at(n, splits);
  const uint32_t across = dim / 4u, lanes = 256u / across; // parts at a time
  const uint32_t mine = threadIdx.x / across, e = threadIdx.x % across * 4u;
  float most = kLowest;
  for (uint32_t s = 0; s < splits; ++s) {
    const float *ms = ws + 2u * ((uint64_t)s * n + id);
    if (ms[1] != 0.0f) most = __builtin_fmaxf(most, ms[0]);
  }
  f32x4_t x = {0, 0, 0, 0};
  float total = 0.0f;
  if (mine < lanes)
    for (uint32_t s = mine; s < splits; s += lanes) {
      const float *ms = ws + 2u * ((uint64_t)s * n + id);
      if (ms[1] == 0.0f) continue;
      const float f = __builtin_amdgcn_exp2f(ms[0] - most);
      total += ms[1] * f;
      const f32x4_t v = *reinterpret_cast<const f32x4_t *>(parts + ((uint64_t)s * n + id) * dim + e);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(v[j], f, x[j]);
    }
  // 256 lanes of four sums and a total
  reinterpret_cast<f32x4_t *>(lds)[threadIdx.x] = x;
  lds[1024u + threadIdx.x] = total;
  __syncthreads();
  if (threadIdx.x >= across) return;
  for (uint32_t l = 1; l < lanes; ++l) {
    const f32x4_t v = reinterpret_cast<const f32x4_t *>(lds)[l * across + threadIdx.x];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += v[j];
    total += lds[1024u + l * across];
  }
  const float f = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = total == 0.0f ? 0.0f : x[j] * f;
  uint8_t *to = y + ((uint64_t)token * y_stride + (uint64_t)h * dim + e) * T::kBytes;
  if constexpr (T::kBytes == 4u) *reinterpret_cast<f32x4_t *>(to) = x;
  else *reinterpret_cast<u32x2_t *>(to) = (u32x2_t){pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
}

} // namespace

#define AXH_ATTEND(NAME, T, CHUNKS, KIND, ROWS, SPLIT, WAVES)                                      \
  extern "C" __global__ void __launch_bounds__(256)                                               \
      __attribute__((amdgpu_waves_per_eu(WAVES, WAVES)))                                          \
      axh_kv_attention_##KIND##_c##CHUNKS##_##NAME(                                               \
          const uint8_t *q, const uint8_t *k, const uint8_t *v, const int32_t *starts,            \
          const int32_t *lengths, const int32_t *table, uint8_t *y, float *ws, uint32_t n_seqs,   \
          uint32_t n_tokens, uint32_t max_pages, uint32_t n_pages, uint32_t page_shift,           \
          uint32_t kv_heads, uint32_t head_dim, uint32_t per, uint32_t q_stride,                  \
          uint32_t y_stride, uint32_t c, uint32_t window, uint32_t chunk, uint32_t splits) {      \
    using A = Attend<T, CHUNKS, ROWS, SPLIT>;                                                     \
    __shared__ alignas(16) float lds[SPLIT ? A::kLds : 4];                                        \
    const Args args{q, k, v, starts, lengths, table, y, ws, n_seqs, n_tokens, max_pages,          \
                    Geometry{n_pages, page_shift, kv_heads, head_dim}, per, q_stride, y_stride,   \
                    __builtin_bit_cast(float, c), window, chunk, splits};                         \
    A(args).run(lds);                                                                             \
  }
#define AXH_COMBINE(NAME, T)                                                                      \
  extern "C" __global__ void __launch_bounds__(256) axh_kv_combine_##NAME(                        \
      const float *ws, const int32_t *starts, uint8_t *y, uint32_t n_tokens, uint32_t n_seqs,     \
      uint32_t n_heads, uint32_t dim, uint32_t y_stride, uint32_t splits) {                       \
    __shared__ alignas(16) float lds[1280];                                                       \
    combine_body<T>(ws, starts, y, n_tokens, n_seqs, n_heads, dim, y_stride, splits, lds);        \
  }
AXH_ATTEND(bf16, TBF16, 1, r1, 1, true, 4)
AXH_ATTEND(f16, TF16, 1, r1, 1, true, 3)
AXH_ATTEND(f32, TF32, 1, r1, 1, true, 2)
AXH_ATTEND(bf16, TBF16, 2, r1, 1, true, 2)
AXH_ATTEND(f16, TF16, 2, r1, 1, true, 2)
AXH_ATTEND(f32, TF32, 2, r1, 1, true, 2)
AXH_COMBINE(bf16, TBF16)
AXH_COMBINE(f16, TF16)
AXH_COMBINE(f32, TF32)
