// Rotary positions; rows written to the paged 4-bit cache and read back (gfx950).  All
// of them are bound by memory or, for few tokens, by the latency of a launch and a few reads:
// rotation of 4096 x 40 x 128 in bf16 14.4 us (84 MB, which stay in the cache: 5.8 TB/s), of one
// token of 32 heads 2.1; 40000 x 8 x 128 read as bf16 44 us (207 MB, 4.7 TB/s; a copy 4.9);
// 9001 x 4 x 96 in f16 turned and written 8 us (17.5 MB), 16 x 8 x 128 4.4 (start and length, page,
// store one after the other).
#include "kv_common.h"

using namespace axh;

namespace {

// ---------------------------------------------------------------------------
// Rotation of heads.  A lane has a unit of a token's head, kN pairs (8 elements of pairs
// that follow one another, 8 and 8 of the two halves; 1 pair where rows are not of whole
// 16-byte pieces), or of the elements behind the rotated ones, which are copied; it
// computes the unit's angles once and goes through `per` heads with them.
// ---------------------------------------------------------------------------
template <class T, bool kWide>
__device__ __forceinline__ void rope_body(const uint8_t *x, uint8_t *y, const int32_t *positions,
                                          const void *table, uint32_t n_tokens, uint32_t n_heads,
                                          uint32_t head_dim, uint32_t x_stride, uint32_t y_stride,
                                          uint32_t dim, uint32_t layout, uint32_t units,
                                          uint32_t per, uint32_t groups) {
  const Rope rope(table, dim, layout);
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  const uint32_t unit = id % units, rest = id / units;
  const uint32_t token = rest / groups, h0 = rest % groups * per;
  if (token >= n_tokens) return;
  const uint32_t h1 = h0 + per < n_heads ? h0 + per : n_heads;
  const uint8_t *xr = x + (uint64_t)token * x_stride * T::kBytes;
  uint8_t *yr = y + (uint64_t)token * y_stride * T::kBytes;
  constexpr uint32_t kStep = kWide ? 8u : 1u;
  // units of the rotated part; halves: of one half, the other being its partner
  const uint32_t turned = rope.halves ? dim / 2u / kStep : dim / (kWide ? 8u : 2u);
  if (unit >= turned) { // copied
    const uint32_t e = dim + (unit - turned) * kStep;
    for (uint32_t h = h0; h < h1; ++h) {
      const uint32_t at = (h * head_dim + e) * T::kBytes;
      if constexpr (kWide) {
        float v[8];
        load8<T>(xr + at, v);
        store8<T>(yr + at, v);
      } else {
        store1<T>(yr + at, load1<T>(xr + at));
      }
    }
    return;
  }
  const int32_t pos = positions[token];
  if (rope.halves) {
    float c[kStep], s[kStep];
#pragma unroll
    for (uint32_t i = 0; i < kStep; ++i) rope.at(unit * kStep + i, pos, c[i], s[i]);
    for (uint32_t h = h0; h < h1; ++h) {
      const uint32_t lo = (h * head_dim + unit * kStep) * T::kBytes;
      const uint32_t hi = lo + dim / 2u * T::kBytes;
      float a[kStep], b[kStep], u[kStep], v[kStep];
      if constexpr (kWide) {
        load8<T>(xr + lo, a);
        load8<T>(xr + hi, b);
      } else {
        a[0] = load1<T>(xr + lo);
        b[0] = load1<T>(xr + hi);
      }
#pragma unroll
      for (uint32_t i = 0; i < kStep; ++i) {
        u[i] = a[i] * c[i] - b[i] * s[i];
        v[i] = a[i] * s[i] + b[i] * c[i];
      }
      if constexpr (kWide) {
        store8<T>(yr + lo, u);
        store8<T>(yr + hi, v);
      } else {
        store1<T>(yr + lo, u[0]);
        store1<T>(yr + hi, v[0]);
      }
    }
  } else {
    constexpr uint32_t kPairs = kWide ? 4u : 1u;
    float c[kPairs], s[kPairs];
#pragma unroll
    for (uint32_t i = 0; i < kPairs; ++i) rope.at(unit * kPairs + i, pos, c[i], s[i]);
    for (uint32_t h = h0; h < h1; ++h) {
      const uint32_t at = (h * head_dim + unit * 2u * kPairs) * T::kBytes;
      float a[2 * kPairs], u[2 * kPairs];
      if constexpr (kWide) {
        load8<T>(xr + at, a);
      } else {
        a[0] = load1<T>(xr + at);
        a[1] = load1<T>(xr + at + T::kBytes);
      }
#pragma unroll
      for (uint32_t i = 0; i < kPairs; ++i) {
        u[2 * i] = a[2 * i] * c[i] - a[2 * i + 1] * s[i];
        u[2 * i + 1] = a[2 * i] * s[i] + a[2 * i + 1] * c[i];
      }
      if constexpr (kWide) {
        store8<T>(yr + at, u);
      } else {
        store1<T>(yr + at, u[0]);
        store1<T>(yr + at + T::kBytes, u[1]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Rows into the cache.  A lane has 8 elements of a token's heads, four lanes (a quad) a
// block of 32: its largest magnitude is two DPP steps away, and the converting
// instruction divides by the block's power of two, so an element is rounded once.
// blockIdx.y 0: keys, turned first where there is a table (angles once a lane, for `per`
// heads; the partners of the other half are read beside the lane's own), 1: values.  A head's
// elements are asked for before the one before it is written, the first's and the angles' turns
// before the token's place is known.
// ---------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ void append_body(const uint8_t *k, const uint8_t *v, uint8_t *cache_k,
                                            uint8_t *cache_v, const int32_t *starts,
                                            const int32_t *lengths, const int32_t *table,
                                            const void *turns, uint32_t n_tokens, uint32_t n_seqs,
                                            uint32_t max_pages, const Geometry &g,
                                            uint32_t k_stride, uint32_t v_stride, uint32_t dim,
                                            uint32_t layout, uint32_t per, uint32_t groups) {
  const bool values = blockIdx.y != 0u;
  const uint32_t units = g.dim / 8u;
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  const uint32_t unit = id % units, rest = id / units;
  const uint32_t token = rest / groups, h0 = rest % groups * per;
  const bool real = token < n_tokens; // (whole quads: units is a multiple of 4)
  const uint32_t h1 = h0 + per < g.kv_heads ? h0 + per : g.kv_heads;
  const uint8_t *xr = (values ? v : k) + (uint64_t)token * (values ? v_stride : k_stride) * T::kBytes;
  const uint32_t e0 = unit * 8u, half = dim / 2u;
  // element e0 + i times c[i], and its partner times s[i]
  const bool turn = !values && turns && e0 < dim;
  const bool halves = layout != 0u, wide = dim % 16u == 0u; // (of halves: partners are 8 in a row)
  const uint32_t partner = e0 < half ? e0 + half : e0 - half;
  float x[8] = {}, o[8] = {};
  auto ask = [&](uint32_t h, float *xs, float *os) {
    const uint8_t *head = xr + (uint64_t)h * g.dim * T::kBytes;
    load8<T>(head + e0 * T::kBytes, xs);
    if (!turn || !halves) return;
    if (wide) {
      load8<T>(head + partner * T::kBytes, os);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t e = e0 + i;
        if (e < dim) os[i] = load1<T>(head + (e < half ? e + half : e - half) * T::kBytes);
      }
    }
  };
  if (real) ask(h0, x, o);
  // (of the pair, where both its elements are the lane's: once)
  const Rope rope(turns, dim, layout);
  uint64_t angle[8] = {};
  if (turn) {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t e = e0 + i;
      if (e < dim && (halves || i % 2u == 0u))
        angle[i] = rope.turns[!halves ? e >> 1 : e < half ? e : e - half];
    }
  }
  const Place at = place_of(starts, lengths, n_seqs, n_tokens, token);
  if (!real) return;
  const int32_t page = page_of(table, g, max_pages, at);
  if (page < 0) return;
  const uint32_t row = (uint32_t)at.pos & (g.page_rows() - 1u);
  float c[8], s[8];
  if (turn) { // (elements behind the rotated ones are left alone below)
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      if (halves) {
        rope.of(angle[i], at.pos, c[i], s[i]);
        if (e0 + i < half) s[i] = -s[i];
      } else if (i % 2u == 0u) {
        rope.of(angle[i], at.pos, c[i], s[i]);
        c[i + 1] = c[i];
        s[i + 1] = s[i];
        s[i] = -s[i];
      }
    }
  }
  uint8_t *out = (values ? cache_v : cache_k) + g.head_offset((uint32_t)page, 0);
  const uint32_t code_at = values ? g.value_code(row, unit) : g.key_code(row, unit);
  const uint32_t scale_at = values ? g.value_scale(row, unit >> 2) : g.key_scale(row, unit >> 2);
  for (uint32_t h = h0; h < h1; ++h) {
    float next[8], other[8];
    if (h + 1u < h1) ask(h + 1u, next, other);
    if (turn) {
      if (!halves) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) o[i] = x[i ^ 1u];
      }
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (e0 + i < dim) x[i] = __builtin_fmaf(x[i], c[i], o[i] * s[i]);
    }
    uint32_t m = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t b = __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu;
      m = b > m ? b : m;
    }
    uint32_t w = dpp_u32<kXor1>(m);
    m = w > m ? w : m;
    w = dpp_u32<kXor2>(m);
    m = w > m ? w : m;
    const uint32_t e = mx_scale_byte(m);
    const uint32_t codes = e == 255u ? 0u : fp4_pack8(x, mx_divisor(e));
    uint8_t *base = out + (uint64_t)h * g.head_bytes();
    *reinterpret_cast<uint32_t *>(base + code_at) = codes;
    if ((unit & 3u) == 0u) base[scale_at] = (uint8_t)e;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      x[i] = next[i];
      o[i] = other[i];
    }
  }
}

// Rows of the cache as f32, f16 or bf16: a lane has 8 elements of a token's heads, four heads'
// codes and scales in flight; bound by the stores.
template <class T>
__device__ __forceinline__ void read_body(const uint8_t *cache_k, const uint8_t *cache_v,
                                          const int32_t *starts, const int32_t *lengths,
                                          const int32_t *table, uint8_t *k, uint8_t *v,
                                          uint32_t n_tokens, uint32_t n_seqs, uint32_t max_pages,
                                          const Geometry &g, uint32_t k_stride, uint32_t v_stride,
                                          uint32_t per, uint32_t groups) {
  const bool values = blockIdx.y != 0u;
  const uint32_t units = g.dim / 8u;
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  const uint32_t unit = id % units, rest = id / units;
  const uint32_t token = rest / groups, h0 = rest % groups * per;
  const Place at = place_of(starts, lengths, n_seqs, n_tokens, token);
  if (token >= n_tokens || at.seq < 0) return; // (of no sequence)
  const int32_t page = page_of(table, g, max_pages, at);
  const uint32_t row = (uint32_t)at.pos & (g.page_rows() - 1u);
  const uint32_t h1 = h0 + per < g.kv_heads ? h0 + per : g.kv_heads;
  uint8_t *yr = (values ? v : k) + (uint64_t)token * (values ? v_stride : k_stride) * T::kBytes;
  const uint8_t *in = (values ? cache_v : cache_k) + g.head_offset(page < 0 ? 0u : (uint32_t)page, 0);
  const uint32_t code_at = values ? g.value_code(row, unit) : g.key_code(row, unit);
  const uint32_t scale_at = values ? g.value_scale(row, unit >> 2) : g.key_scale(row, unit >> 2);
  for (uint32_t h = h0; h < h1; h += 4u) {
    uint32_t codes[4], scales[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint8_t *base = in + (uint64_t)(h + i) * g.head_bytes();
      const bool on = page >= 0 && h + i < h1;
      codes[i] = on ? *reinterpret_cast<const uint32_t *>(base + code_at) : 0u;
      scales[i] = on ? base[scale_at] : 0u;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      if (h + i >= h1) break;
      const float s = e8m0_to_f32(scales[i]);
      const f32x2_t p0 = fp4_pair<0>(codes[i]), p1 = fp4_pair<1>(codes[i]),
                    p2 = fp4_pair<2>(codes[i]), p3 = fp4_pair<3>(codes[i]);
      const float x[8] = {p0.x * s, p0.y * s, p1.x * s, p1.y * s,
                          p2.x * s, p2.y * s, p3.x * s, p3.y * s};
      store8<T>(yr + ((uint64_t)(h + i) * g.dim + unit * 8u) * T::kBytes, x);
    }
  }
}

} // namespace

#define AXH_ROPE(NAME, T, WIDTH, WIDE)                                                            \
  extern "C" __global__ void __launch_bounds__(256) axh_rope_##WIDTH##_##NAME(                    \
      const uint8_t *x, uint8_t *y, const int32_t *positions, const void *table,                  \
      uint32_t n_tokens, uint32_t n_heads, uint32_t head_dim, uint32_t x_stride,                  \
      uint32_t y_stride, uint32_t dim, uint32_t layout, uint32_t units, uint32_t per,             \
      uint32_t groups) {                                                                          \
    rope_body<T, WIDE>(x, y, positions, table, n_tokens, n_heads, head_dim, x_stride, y_stride,   \
                       dim, layout, units, per, groups);                                          \
  }
#define AXH_KV(NAME, T)                                                                           \
  AXH_ROPE(NAME, T, wide, true)                                                                   \
  AXH_ROPE(NAME, T, single, false)                                                                \
  extern "C" __global__ void __launch_bounds__(256) axh_kv_append_##NAME(                         \
      const uint8_t *k, const uint8_t *v, uint8_t *cache_k, uint8_t *cache_v,                     \
      const int32_t *starts, const int32_t *lengths, const int32_t *table, const void *turns,     \
      uint32_t n_tokens, uint32_t n_seqs, uint32_t max_pages, uint32_t n_pages,                   \
      uint32_t page_shift, uint32_t kv_heads, uint32_t head_dim, uint32_t k_stride,               \
      uint32_t v_stride, uint32_t dim, uint32_t layout, uint32_t per, uint32_t groups) {          \
    append_body<T>(k, v, cache_k, cache_v, starts, lengths, table, turns, n_tokens, n_seqs,       \
                   max_pages, Geometry{n_pages, page_shift, kv_heads, head_dim}, k_stride,        \
                   v_stride, dim, layout, per, groups);                                           \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) axh_kv_read_##NAME(                           \
      const uint8_t *cache_k, const uint8_t *cache_v, const int32_t *starts,                      \
      const int32_t *lengths, const int32_t *table, uint8_t *k, uint8_t *v, uint32_t n_tokens,    \
      uint32_t n_seqs, uint32_t max_pages, uint32_t n_pages, uint32_t page_shift,                 \
      uint32_t kv_heads, uint32_t head_dim, uint32_t k_stride, uint32_t v_stride, uint32_t per,   \
      uint32_t groups) {                                                                          \
    read_body<T>(cache_k, cache_v, starts, lengths, table, k, v, n_tokens, n_seqs, max_pages,     \
                 Geometry{n_pages, page_shift, kv_heads, head_dim}, k_stride, v_stride, per,      \
                 groups);                                                                         \
  }
AXH_KV(f32, TF32)
AXH_KV(f16, TF16)
AXH_KV(bf16, TBF16)
