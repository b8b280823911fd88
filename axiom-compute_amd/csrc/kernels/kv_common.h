// Shared device helpers of the kernels of the paged 4-bit cache (gfx950).
//
// A page holds, for each head in turn, page_size rows of head_dim elements in
// MXFP4.  Keys: rows of codes (head_dim / 2 bytes), then rows of scale bytes
// (head_dim / 32).  Values: for each four tokens, a dword of codes (8 elements) of
// each of them, then the next dword; then for each four tokens their scale bytes of
// a block, then of the next.  So a lane that multiplies 8 values of four tokens
// reads 16 bytes of codes and 4 of scales at once.
#pragma once
#include "mx_common.h"

namespace axh {

struct Geometry {
  uint32_t n_pages, page_shift, kv_heads, dim; // dim: a multiple of 32 up to 256
  __device__ __forceinline__ uint32_t page_rows() const { return 1u << page_shift; }
  __device__ __forceinline__ uint32_t head_bytes() const {
    return page_rows() * (dim / 2u + dim / 32u);
  }
  __device__ __forceinline__ uint64_t head_offset(uint32_t page, uint32_t head) const {
    return ((uint64_t)page * kv_heads + head) * head_bytes();
  }
  // Offsets in a head's part of a page: dword `dw` of codes (elements 8 dw .. 8 dw + 7)
  // and the scale byte of block `blk`, of row `row`.
  __device__ __forceinline__ uint32_t key_code(uint32_t row, uint32_t dw) const {
    return row * (dim / 2u) + dw * 4u;
  }
  __device__ __forceinline__ uint32_t key_scale(uint32_t row, uint32_t blk) const {
    return page_rows() * (dim / 2u) + row * (dim / 32u) + blk;
  }
  __device__ __forceinline__ uint32_t value_code(uint32_t row, uint32_t dw) const {
    return (row >> 2) * (dim * 2u) + dw * 16u + (row & 3u) * 4u;
  }
  __device__ __forceinline__ uint32_t value_scale(uint32_t row, uint32_t blk) const {
    return page_rows() * (dim / 2u) + (row >> 2) * (dim / 8u) + blk * 4u + (row & 3u);
  }
};

// Where a token of a batch is: its sequence and position, or seq < 0.
struct Place {
  int32_t seq, pos;
};
// starts NULL: one token a sequence.  starts[] does not decrease, so the last s with
// starts[s] <= token is the one that holds it (those before it may be empty).  All lanes of
// the wave call it, also those whose token is none of the batch.  Up to 64 sequences, a lane
// reads one's start and length, and the search is among lanes: two reads in place of a chain of
// log2 n_seqs + 2.
__device__ __forceinline__ Place place_of(const int32_t *starts, const int32_t *lengths,
                                          uint32_t n_seqs, uint32_t n_tokens, uint32_t token) {
  if (!starts) return {(int32_t)token, token < n_tokens ? lengths[token] - 1 : -1};
  uint32_t lo = 0;
  int32_t first, last, len;
  if (n_seqs <= 64u) {
    const uint32_t lane = threadIdx.x & 63u;
    const int32_t start = lane < n_seqs ? starts[lane] : 0, end = starts[n_seqs];
    const int32_t mine = lane < n_seqs ? lengths[lane] : 0;
#pragma unroll
    for (uint32_t step = 32; step; step >>= 1) {
      const int32_t v = __shfl(start, (int)((lo + step) & 63u));
      if (lo + step < n_seqs && v <= (int32_t)token) lo += step;
    }
    first = __shfl(start, (int)lo);
    last = __shfl(start, (int)((lo + 1u) & 63u));
    if (lo + 1u == n_seqs) last = end;
    len = __shfl(mine, (int)lo);
  } else {
    uint32_t hi = n_seqs; // starts[lo] <= token < starts[hi], if it is in a sequence
    while (hi - lo > 1u) {
      const uint32_t mid = (lo + hi) >> 1;
      if (starts[mid] <= (int32_t)token) lo = mid;
      else hi = mid;
    }
    first = starts[lo];
    last = starts[lo + 1u];
    len = lengths[lo];
  }
  if ((int32_t)token < first || (int32_t)token >= last) return {-1, -1};
  const int32_t pos = (int32_t)((uint32_t)len - (uint32_t)last + token);
  return {(int32_t)lo, pos < len ? pos : -1};
}
// The page of a position, or -1.
__device__ __forceinline__ int32_t page_of(const int32_t *table, const Geometry &g,
                                           uint32_t max_pages, const Place &at) {
  if (at.seq < 0 || at.pos < 0) return -1;
  const uint32_t slot = (uint32_t)at.pos >> g.page_shift;
  if (slot >= max_pages) return -1;
  const int32_t page = table[(uint64_t)at.seq * max_pages + slot];
  return (uint32_t)page < g.n_pages ? page : -1;
}

// Eight consecutive elements as f32, 16-byte aligned (f32: two loads).
template <class T> __device__ __forceinline__ void load8(const uint8_t *p, float *v) {
  if constexpr (T::kBytes == 4u) {
    const f32x4_t a = reinterpret_cast<const f32x4_t *>(p)[0];
    const f32x4_t b = reinterpret_cast<const f32x4_t *>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else {
    const u32x4_t w = *reinterpret_cast<const u32x4_t *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
  }
}
template <class T> __device__ __forceinline__ void store8(uint8_t *p, const float *v) {
  if constexpr (T::kBytes == 4u) {
    reinterpret_cast<f32x4_t *>(p)[0] = (f32x4_t){v[0], v[1], v[2], v[3]};
    reinterpret_cast<f32x4_t *>(p)[1] = (f32x4_t){v[4], v[5], v[6], v[7]};
  } else {
    *reinterpret_cast<u32x4_t *>(p) = (u32x4_t){pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                                pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
  }
}
template <class T> __device__ __forceinline__ float load1(const uint8_t *p) {
  if constexpr (T::kBytes == 4u) {
    return *reinterpret_cast<const float *>(p);
  } else {
    float lo, hi;
    unpack2<T>(*reinterpret_cast<const uint16_t *>(p), lo, hi);
    return lo;
  }
}
template <class T> __device__ __forceinline__ void store1(uint8_t *p, float v) {
  if constexpr (T::kBytes == 4u) *reinterpret_cast<float *>(p) = v;
  else *reinterpret_cast<uint16_t *>(p) = (uint16_t)pack2<T>(v, v);
}

// cos and sin of pos * turns, a 64-bit fraction of a turn: the product's integer part
// falls away by itself, whatever the position, so the angle is exact to the bits that
// are kept (2^-32 turns).  The nearest quarter turn is taken off; the series of both
// functions on the rest, at most pi / 4, end at 2e-9 and 1e-10.
__device__ __forceinline__ void rotation(uint64_t turns, int32_t pos, float &c, float &s) {
  const uint32_t a = (uint32_t)(((uint64_t)(int64_t)pos * turns) >> 32);
  const uint32_t quarter = (a + 0x20000000u) >> 30;
  const float r = (float)(int32_t)(a - (quarter << 30)) * 0x1.921fb6p-30f; // 2 pi / 2^32
  const float z = r * r;
  float u = __builtin_fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
  u = __builtin_fmaf(z, u, 1.0f / 120.0f);
  u = __builtin_fmaf(z, u, -1.0f / 6.0f);
  const float sn = __builtin_fmaf(r * z, u, r);
  float w = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  w = __builtin_fmaf(z, w, -1.0f / 720.0f);
  w = __builtin_fmaf(z, w, 1.0f / 24.0f);
  w = __builtin_fmaf(z, w, -0.5f);
  const float cs = __builtin_fmaf(z, w, 1.0f);
  const float x = (quarter & 1u) ? -sn : cs, y = (quarter & 1u) ? cs : sn;
  c = (quarter & 2u) ? -x : x;
  s = (quarter & 2u) ? -y : y;
}

// A rotation's table: dim / 2 fractions of a turn for each position, then the magnitude.
struct Rope {
  const uint64_t *turns;
  uint32_t dim;
  bool halves;
  float magnitude;
  __device__ __forceinline__ Rope(const void *table, uint32_t d, uint32_t layout)
      : turns(static_cast<const uint64_t *>(table)), dim(d), halves(layout != 0u),
        magnitude(table ? *reinterpret_cast<const float *>(turns + d / 2u) : 1.0f) {}
  __device__ __forceinline__ void at(uint32_t pair, int32_t pos, float &c, float &s) const {
    of(turns[pair], pos, c, s);
  }
  __device__ __forceinline__ void of(uint64_t turn, int32_t pos, float &c, float &s) const {
    rotation(turn, pos, c, s);
    c *= magnitude;
    s *= magnitude;
  }
};

} // namespace axh
