// MXFP4 x MXFP4 products on scaled MFMA (gfx950):
//   y[b][r] = sum_k W[r][k] * X[b][k],  f32 accumulation,
// W n_rows x cols and X batch x cols, both rows of codes and of scales (see
// mx_common.h), y batch x n_rows; and the same product for expert layers,
// where the rows of X are grouped by expert and each group has a matrix of its
// own.  v_mfma_scale_f32_32x32x64_f8f6f4 multiplies the codes as they are
// stored: lane l holds the 32 codes (16 bytes) of block l / 32 of row l % 32
// of a 32 x 64 operand tile and that block's scale byte; products of codes and
// scales are exact in f32.
//
// Two kinds of kernel:
//   * skinny (few columns, bound by W's bytes): a workgroup has one 32-row tile
//     of W (gate/up: one of each matrix), its waves split the K axis, operands
//     go straight to registers and the waves' partial tiles meet in LDS;
//   * tile (many columns, bound by the matrix cores): a workgroup has a BM x BN
//     tile, K in steps of 256 through two LDS buffers filled by direct-to-LDS
//     loads, each wave a part of the tile.
#include "mx_common.h"

#include <type_traits>

using namespace axh;

namespace {

typedef __attribute__((address_space(3))) void lds_void_t;

// Offset of what lies past the end of an operand: with a step's offset on top
// it is still past every buffer's end and below 2^32 (the host keeps the rows
// of a buffer below 2 GiB), so such loads return zeros.
constexpr uint32_t kFar = 0x80000000u;

template <int kk>
__device__ __forceinline__ f32x16_t mfma(u32x4_t a, u32x4_t b, f32x16_t c, uint32_t sa,
                                         uint32_t sb) {
  const i32x8_t A = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8_t B = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, kk, (int)sa, kk, (int)sb);
}

// The eight scale bytes of a row's K step (blocks 8s .. 8s + 7), as loaded:
// rows of at least eight blocks are read inside the row, the bytes of a last,
// partial step shifted down at their use (scales8); the scales past the row's
// end come out 0 (2^-127, times codes that are 0).
struct ScaleStep {
  uint32_t at;    // byte offset in the row
  uint32_t shift; // bits
};
__device__ __forceinline__ ScaleStep scale_step(uint32_t s, uint32_t nblk) {
  const uint32_t want = 8u * s, last = nblk < 8u ? 0u : nblk - 8u;
  const uint32_t at = want < last ? want : last;
  return {at, nblk < 8u ? 0u : (want - at) * 8u};
}
__device__ __forceinline__ u32x2_t load_scales8(__amdgpu_buffer_rsrc_t r, uint32_t row_off,
                                                ScaleStep st, uint32_t nblk) {
  if (nblk >= 8u) return __builtin_amdgcn_raw_buffer_load_b64(r, (int)(row_off + st.at), 0, 0);
  uint32_t v[8];
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i)
    v[i] = __builtin_amdgcn_raw_buffer_load_b8(r, (int)(i < nblk ? row_off + i : kFar), 0, 0);
  return (u32x2_t){v[0] | v[1] << 8 | v[2] << 16 | v[3] << 24,
                   v[4] | v[5] << 8 | v[6] << 16 | v[7] << 24};
}
// The lane's four scale bytes of the step: those of blocks 2 kk + lane / 32.
__device__ __forceinline__ uint32_t lane_scales(u32x2_t w, ScaleStep st, uint32_t sel) {
  const uint64_t v = ((uint64_t)w.y << 32 | w.x) >> st.shift;
  return __builtin_amdgcn_perm((uint32_t)(v >> 32), (uint32_t)v, sel);
}
__device__ __forceinline__ uint32_t scale_selector(uint32_t half) {
  return half ? 0x07050301u : 0x06040200u;
}

// Four consecutive rows of one output column.
template <class T>
__device__ __forceinline__ void store4(uint8_t *col, uint32_t r, uint32_t n_rows, f32x4_t v) {
  uint8_t *p = col + (uint64_t)r * T::kBytes;
  if (r + 4u <= n_rows && ((uintptr_t)p & (4u * T::kBytes - 1u)) == 0u) {
    if constexpr (T::kBytes == 4)
      *reinterpret_cast<f32x4_t *>(p) = v;
    else
      *reinterpret_cast<u32x2_t *>(p) =
          (u32x2_t){pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (r + i < n_rows) {
        if constexpr (T::kBytes == 4)
          reinterpret_cast<float *>(p)[i] = v[i];
        else
          reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)pack2<T>(v[i], 0.0f);
      }
  }
}


// A 32-feature block of one column of h as MXFP4: lanes l and l + 32 of a wave
// hold its features 8q + 4 (lane / 32) + i in h[4q + i].  Each lane packs its
// sixteen codes, and stores eight bytes of the block: the low half its first
// two quarters', the other the last two.
__device__ __forceinline__ void store_packed(uint8_t *codes, uint8_t *scales, uint64_t blk,
                                             const float *h, uint32_t half, bool real) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, h[i]) & 0x7FFFFFFFu;
    m = b > m ? b : m;
  }
  const uint32_t o = (uint32_t)__shfl_xor((int)m, 32);
  m = o > m ? o : m;
  const uint32_t e = mx_scale_byte(m);
  const float f = mx_inverse(e);
  uint32_t q01, q23; // quarters 0 and 1, 2 and 3: four codes (16 bits) each
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = h[i] * f;
  q01 = e == 255u ? 0u : fp4_pack8(v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = h[8 + i] * f;
  q23 = e == 255u ? 0u : fp4_pack8(v);
  const uint32_t mine = half ? q23 : q01;
  const uint32_t theirs = (uint32_t)__shfl_xor((int)(half ? q01 : q23), 32);
  // the low half's features come first in every group of eight
  const uint32_t lo = half ? theirs : mine, hi = half ? mine : theirs;
  const u32x2_t out = {(lo & 0xFFFFu) | hi << 16, lo >> 16 | (hi & 0xFFFF0000u)};
  if (!real) return;
  *reinterpret_cast<u32x2_t *>(codes + blk * 16u + half * 8u) = out;
  if (half == 0u) scales[blk] = (uint8_t)e;
}

// What a workgroup multiplies and where the result goes.
enum Mode { kDense, kGrouped, kGateUp };

struct Args {
  const uint8_t *wc, *ws;   // weights (gate)
  const uint8_t *uc, *us;   // up
  const uint8_t *xc, *xs;   // activations
  const uint32_t *plan;     // expert layers: offsets, then slots by expert
  uint8_t *y, *ysc;         // output (codes), its scales where packed
  uint32_t n_rows, nblk;    // rows of a matrix, blocks of a row
  uint32_t n_cols;          // dense: batch
  uint32_t n_x;             // rows of X
  uint32_t x_div;           // expert layers: slot / x_div is the row of X
  uint32_t n_experts;
  uint32_t row_tiles;       // workgroups along the rows
};

struct Tile {
  uint32_t m, n0, count, first, expert; // first: expert layers, place of column 0 in the order
  bool real;
};

// Workgroup -> tile.  Consecutive workgroups go to the eight XCDs in turn; each
// XCD is given a contiguous part of the tiles, rows fastest for expert layers
// (the tiles of one group of columns share X), columns fastest otherwise.
template <Mode M, int BN> __device__ __forceinline__ Tile tile_of(const Args &a, uint32_t *lds) {
  const uint32_t total = gridDim.x, id = blockIdx.x;
  const uint32_t per = total / 8u, rest = total % 8u, xcd = id % 8u;
  const uint32_t t = xcd * per + (xcd < rest ? xcd : rest) + id / 8u;
  Tile r;
  if constexpr (M == kDense) {
    const uint32_t cols = (a.n_cols + BN - 1u) / BN;
    r.m = t / cols;
    r.n0 = (t - r.m * cols) * BN;
    r.count = a.n_cols - r.n0;
    r.first = 0;
    r.expert = 0;
    r.real = true;
  } else {
    const uint32_t nt = t / a.row_tiles;
    r.m = t - nt * a.row_tiles;
    // the expert whose tiles of BN columns hold number nt: every wave looks
    // through the offsets, 64 experts at a time
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t before = 0;
    r.real = false;
    r.n0 = r.count = r.first = r.expert = 0;
    for (uint32_t e0 = 0; e0 < a.n_experts; e0 += 64u) {
      const uint32_t e = e0 + lane;
      const uint32_t lo = a.plan[e < a.n_experts ? e : a.n_experts];
      const uint32_t hi = a.plan[e < a.n_experts ? e + 1u : a.n_experts];
      const uint32_t tiles = (hi - lo + BN - 1u) / BN;
      uint32_t incl = tiles;
#pragma unroll
      for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)incl, d);
        if (lane >= d) incl += o;
      }
      const uint32_t excl = before + incl - tiles;
      const uint64_t at = __ballot(nt >= excl && nt < excl + tiles);
      if (at) {
        const int who = __builtin_ctzll(at);
        const uint32_t k = (nt - (uint32_t)__builtin_amdgcn_readlane((int)excl, who)) * BN;
        const uint32_t l = (uint32_t)__builtin_amdgcn_readlane((int)lo, who);
        const uint32_t h = (uint32_t)__builtin_amdgcn_readlane((int)hi, who);
        r.expert = e0 + (uint32_t)who;
        r.first = l + k;
        r.count = h - l - k;
        r.real = true;
        break;
      }
      before += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
  }
  if (r.count > (uint32_t)BN) r.count = BN;
  (void)lds;
  return r;
}

__device__ __forceinline__ const uint32_t *plan_order(const Args &a) {
  return a.plan + ((a.n_experts + 1u + 15u) & ~15u);
}

// Finishes four rows r .. r + 3 of a column (not packed).
template <Mode M, class T>
__device__ __forceinline__ void emit4(const Args &a, uint32_t out_row, uint32_t r, f32x4_t g,
                                      f32x4_t u) {
  if constexpr (M == kGateUp) {
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = swiglu(g[i], u[i]);
  }
  if (r < a.n_rows)
    store4<T>(a.y + (uint64_t)out_row * a.n_rows * T::kBytes, r, a.n_rows, g);
}

// ---------------------------------------------------------------------------
// Skinny kind: NW waves, 32 rows (of one matrix, or of gate and up), 32 * NI
// columns.
// ---------------------------------------------------------------------------
template <Mode M, class T, bool kPacked, int NI, int NW>
__device__ __forceinline__ void skinny_body(const Args &a, f32x4_t *lds) {
  constexpr int MI = M == kGateUp ? 2 : 1;
  constexpr int BN = 32 * NI;
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t half = lane >> 5, r32 = lane & 31u;
  const Tile t = tile_of<M, BN>(a, nullptr);
  if (!t.real) return;
  const uint32_t row0 = t.m * 32u;
  const uint32_t nblk = a.nblk, row_bytes = nblk * 16u;
  const uint64_t matrix = (uint64_t)a.n_rows * nblk, wat = t.expert * matrix + (uint64_t)row0 * nblk;
  const uint32_t rows = a.n_rows - row0 < 32u ? a.n_rows - row0 : 32u;
  __amdgpu_buffer_rsrc_t wc[MI], ws[MI];
  wc[0] = rsrc(a.wc + wat * 16u, rows * row_bytes);
  ws[0] = rsrc(a.ws + wat, rows * nblk);
  if constexpr (MI == 2) {
    wc[1] = rsrc(a.uc + wat * 16u, rows * row_bytes);
    ws[1] = rsrc(a.us + wat, rows * nblk);
  }
  // columns: X's rows, and the rows of y they go to
  uint32_t xrow[NI], out[NI];
  uint64_t xbase = 0;
  uint32_t xrows = a.n_x;
  if constexpr (M == kDense) {
    xbase = t.n0;
    xrows = t.count;
  }
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const uint32_t j = 32u * n + r32;
    if constexpr (M == kDense) {
      xrow[n] = j < t.count ? j : 0xFFFFFFFFu;
      out[n] = t.n0 + j;
    } else {
      const uint32_t slot = plan_order(a)[t.first + (j < t.count ? j : 0u)];
      xrow[n] = j < t.count ? slot / a.x_div : 0xFFFFFFFFu;
      out[n] = slot;
    }
  }
  const __amdgpu_buffer_rsrc_t xc = rsrc(a.xc + xbase * row_bytes, xrows * row_bytes);
  const __amdgpu_buffer_rsrc_t xs = rsrc(a.xs + xbase * nblk, xrows * nblk);

  f32x16_t acc[MI][NI] = {};
  const uint32_t sel = scale_selector(half);
  const uint32_t steps = (nblk + 7u) / 8u;
  struct Step {
    u32x4_t a[MI][4], b[NI][4];
    u32x2_t sa[MI], sb[NI];
    ScaleStep st;
  };
  auto load = [&](uint32_t s, Step &p) {
    p.st = scale_step(s, nblk);
#pragma unroll
    for (int m = 0; m < MI; ++m) p.sa[m] = load_scales8(ws[m], r32 * nblk, p.st, nblk);
#pragma unroll
    for (int n = 0; n < NI; ++n)
      p.sb[n] = load_scales8(xs, xrow[n] == 0xFFFFFFFFu ? kFar : xrow[n] * nblk, p.st, nblk);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t blk = 8u * s + 2u * k + half;
      const bool in = blk < nblk;
#pragma unroll
      for (int m = 0; m < MI; ++m)
        p.a[m][k] = __builtin_amdgcn_raw_buffer_load_b128(
            wc[m], (int)(in ? r32 * row_bytes + blk * 16u : kFar), 0, 0);
#pragma unroll
      for (int n = 0; n < NI; ++n)
        p.b[n][k] = __builtin_amdgcn_raw_buffer_load_b128(
            xc, (int)(in && xrow[n] != 0xFFFFFFFFu ? xrow[n] * row_bytes + blk * 16u : kFar), 0,
            0);
    }
  };
  auto multiply = [&](const Step &p) {
    uint32_t sa[MI], sb[NI];
#pragma unroll
    for (int m = 0; m < MI; ++m) sa[m] = lane_scales(p.sa[m], p.st, sel);
#pragma unroll
    for (int n = 0; n < NI; ++n) sb[n] = lane_scales(p.sb[n], p.st, sel);
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        acc[m][n] = mfma<0>(p.a[m][0], p.b[n][0], acc[m][n], sa[m], sb[n]);
        acc[m][n] = mfma<1>(p.a[m][1], p.b[n][1], acc[m][n], sa[m], sb[n]);
        acc[m][n] = mfma<2>(p.a[m][2], p.b[n][2], acc[m][n], sa[m], sb[n]);
        acc[m][n] = mfma<3>(p.a[m][3], p.b[n][3], acc[m][n], sa[m], sb[n]);
      }
  };
  Step p0, p1;
  uint32_t s = wave;
  if (s < steps) load(s, p0);
  for (; s < steps; s += 2u * NW) {
    if (s + NW < steps) load(s + NW, p1);
    multiply(p0);
    if (s + 2u * NW < steps) load(s + 2u * NW, p0);
    if (s + NW < steps) multiply(p1);
  }

  // partial tiles: [wave][matrix][column group][quarter][lane]
  constexpr uint32_t kTiles = MI * NI;
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        lds[((wave * kTiles + m * NI + n) * 4u + q) * 64u + lane] =
            (f32x4_t){acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2],
                      acc[m][n][4 * q + 3]};
  __syncthreads();
  auto total = [&](uint32_t m, uint32_t n, uint32_t q) {
    f32x4_t v = lds[((m * NI + n) * 4u + q) * 64u + lane];
#pragma unroll
    for (uint32_t w = 1; w < NW; ++w) v += lds[((w * kTiles + m * NI + n) * 4u + q) * 64u + lane];
    return v;
  };
  if constexpr (kPacked) {
    for (uint32_t n = wave; n < (uint32_t)NI; n += NW) {
      float h[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4_t g = total(0, n, q), u = total(MI - 1, n, q);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[4 * q + i] = swiglu(g[i], u[i]);
      }
      uint32_t o = out[0];
#pragma unroll
      for (uint32_t k = 1; k < NI; ++k) o = n == k ? out[k] : o;
      store_packed(a.y, a.ysc, (uint64_t)o * (a.n_rows / 32u) + t.m, h, half,
                   32u * n + r32 < t.count);
    }
  } else {
    for (uint32_t i = wave; i < 4u * NI; i += NW) {
      const uint32_t n = i / 4u, q = i % 4u;
      const f32x4_t g = total(0, n, q), u = M == kGateUp ? total(MI - 1, n, q) : g;
      uint32_t o = out[0];
#pragma unroll
      for (uint32_t k = 1; k < NI; ++k) o = n == k ? out[k] : o;
      if (32u * n + r32 < t.count) emit4<M, T>(a, o, row0 + 8u * q + 4u * half, g, u);
    }
  }
}

// ---------------------------------------------------------------------------
// Tile kind: BM x BN outputs (gate/up: BM / 2 rows of each matrix, in turns of
// 32), WM x WN waves.  An LDS row is 128 bytes, the codes of one K step, with
// 16-byte piece c at place c ^ (row % 8): the 32 rows that a fragment read
// touches then meet all the banks.
// ---------------------------------------------------------------------------
template <Mode M, class T, bool kPacked, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void tile_body(const Args &a, uint8_t *lds) {
  constexpr int NW = WM * WN, MI = BM / WM / 32, NI = BN / WN / 32;
  constexpr uint32_t kBuf = (BM + BN) * 128u;
  constexpr int kLoads = (BM + BN) / 8 / NW; // per wave and step; rows of A first
  constexpr int kALoads = BM / 8 / NW;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "whole loads per wave");
  static_assert(M != kGateUp || MI % 2 == 0, "gate and up rows in one wave");
  constexpr uint32_t kRows = M == kGateUp ? BM / 2 : BM; // rows of y
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t wm = wave / WN, wn = wave % WN;
  const uint32_t half = lane >> 5, r32 = lane & 31u;
  const Tile t = tile_of<M, BN>(a, nullptr);
  if (!t.real) return;
  const uint32_t row0 = t.m * kRows;
  const uint32_t nblk = a.nblk, row_bytes = nblk * 16u;
  const uint64_t wat = (uint64_t)t.expert * a.n_rows * nblk + (uint64_t)row0 * nblk;
  const uint32_t rows = a.n_rows - row0 < kRows ? a.n_rows - row0 : kRows;
  const __amdgpu_buffer_rsrc_t wc = rsrc(a.wc + wat * 16u, rows * row_bytes);
  const __amdgpu_buffer_rsrc_t ws = rsrc(a.ws + wat, rows * nblk);
  const __amdgpu_buffer_rsrc_t uc = M == kGateUp ? rsrc(a.uc + wat * 16u, rows * row_bytes) : wc;
  const __amdgpu_buffer_rsrc_t us = M == kGateUp ? rsrc(a.us + wat, rows * nblk) : ws;
  const uint64_t xbase = M == kDense ? t.n0 : 0u;
  const uint32_t xrows = M == kDense ? t.count : a.n_x;
  const __amdgpu_buffer_rsrc_t xc = rsrc(a.xc + xbase * row_bytes, xrows * row_bytes);
  const __amdgpu_buffer_rsrc_t xs = rsrc(a.xs + xbase * nblk, xrows * nblk);
  // row of X of column j of the tile, and the row of y that it gives
  auto slot_of = [&](uint32_t j) {
    return M == kDense ? t.n0 + j : plan_order(a)[t.first + (j < t.count ? j : 0u)];
  };
  auto xrow_of = [&](uint32_t j) { return M == kDense ? j : slot_of(j) / a.x_div; };

  // this lane's part of each load: row 8 * (load * NW + wave) + lane / 8
  const uint32_t l8 = lane >> 3, piece = (lane & 7u) ^ (l8 & 7u);
  uint32_t off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    if (i < kALoads) {
      const uint32_t r = 8u * (i * NW + wave) + l8;
      const uint32_t row = M == kGateUp ? (r >> 6) * 32u + (r & 31u) : r;
      off[i] = row * row_bytes + piece * 16u;
    } else {
      const uint32_t j = 8u * ((i - kALoads) * NW + wave) + l8;
      off[i] = j < t.count ? xrow_of(j) * row_bytes + piece * 16u : kFar;
    }
  }
  const uint32_t steps = (nblk + 7u) / 8u;
  auto fill = [&](uint32_t s, uint32_t buf) {
    const bool in = 8u * s + piece < nblk; // false past the end of a last, partial step
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t load = i < kALoads ? i : i - kALoads;
      const uint32_t r8 = 8u * (load * NW + wave);
      const bool up = M == kGateUp && i < kALoads && ((r8 >> 5) & 1u);
      uint8_t *to = lds + buf * kBuf + ((i < kALoads ? 0u : (uint32_t)BM) + r8) * 128u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(i < kALoads ? (up ? uc : wc) : xc,
                                               (lds_void_t *)to, 16, (int)(in ? off[i] : kFar),
                                               (int)(s * 128u), 0, 0);
    }
  };
  // scales: the lane's row of each of the wave's 32-row operand tiles
  uint32_t arow[MI], brow[NI];
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const uint32_t tile = wm * MI + m;
    arow[m] = ((M == kGateUp ? tile >> 1 : tile) * 32u + r32) * nblk;
  }
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const uint32_t j = (wn * NI + n) * 32u + r32;
    brow[n] = j < t.count ? xrow_of(j) * nblk : kFar;
  }
  struct Scales {
    u32x2_t a[MI], b[NI];
    ScaleStep st;
  };
  auto load_scales = [&](uint32_t s, Scales &p) {
    p.st = scale_step(s, nblk);
#pragma unroll
    for (int m = 0; m < MI; ++m)
      p.a[m] = load_scales8(M == kGateUp && (m & 1) ? us : ws, arow[m], p.st, nblk);
#pragma unroll
    for (int n = 0; n < NI; ++n) p.b[n] = load_scales8(xs, brow[n], p.st, nblk);
  };

  f32x16_t acc[MI][NI] = {};
  const uint32_t sel = scale_selector(half);
  uint32_t frag[4]; // byte offset of the lane's piece of K part kk in a 32-row tile
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) frag[k] = r32 * 128u + (((2u * k + half) ^ (r32 & 7u)) * 16u);
  auto multiply = [&](const Scales &p, uint32_t buf) {
    uint32_t sa[MI], sb[NI];
#pragma unroll
    for (int m = 0; m < MI; ++m) sa[m] = lane_scales(p.a[m], p.st, sel);
#pragma unroll
    for (int n = 0; n < NI; ++n) sb[n] = lane_scales(p.b[n], p.st, sel);
    const uint8_t *la = lds + buf * kBuf + wm * (MI * 4096u);
    const uint8_t *lb = lds + buf * kBuf + BM * 128u + wn * (NI * 4096u);
    auto part = [&](auto kk) {
      constexpr int K = decltype(kk)::value;
      u32x4_t fa[MI], fb[NI];
#pragma unroll
      for (int m = 0; m < MI; ++m)
        fa[m] = *reinterpret_cast<const u32x4_t *>(la + m * 4096 + frag[K]);
#pragma unroll
      for (int n = 0; n < NI; ++n)
        fb[n] = *reinterpret_cast<const u32x4_t *>(lb + n * 4096 + frag[K]);
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n)
          acc[m][n] = mfma<K>(fa[m], fb[n], acc[m][n], sa[m], sb[n]);
    };
    part(std::integral_constant<int, 0>());
    part(std::integral_constant<int, 1>());
    part(std::integral_constant<int, 2>());
    part(std::integral_constant<int, 3>());
  };

  Scales p0, p1;
  load_scales(0, p0);
  fill(0, 0);
  for (uint32_t s = 0; s < steps; s += 2u) {
    // step s has landed everywhere, and nobody reads the other buffer any more
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + 1u < steps) {
      load_scales(s + 1u, p1);
      fill(s + 1u, 1);
    }
    multiply(p0, 0);
    if (s + 1u >= steps) break;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + 2u < steps) {
      load_scales(s + 2u, p0);
      fill(s + 2u, 0);
    }
    multiply(p1, 1);
  }

#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const uint32_t j = (wn * NI + n) * 32u + r32;
    const bool real = j < t.count;
    const uint32_t out = slot_of(j);
    constexpr int kStep = M == kGateUp ? 2 : 1;
#pragma unroll
    for (int m = 0; m < MI; m += kStep) {
      const uint32_t block = (wm * MI + m) / kStep; // 32-row block of the tile
      const f32x16_t &g = acc[m][n], &u = acc[M == kGateUp ? m + 1 : m][n];
      if constexpr (kPacked) {
        float h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = swiglu(g[i], u[i]);
        const uint32_t fb = row0 / 32u + block;
        store_packed(a.y, a.ysc, (uint64_t)out * (a.n_rows / 32u) + fb, h, half,
                     real && fb < a.n_rows / 32u);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (real)
            emit4<M, T>(a, out, row0 + block * 32u + 8u * q + 4u * half,
                        (f32x4_t){g[4 * q], g[4 * q + 1], g[4 * q + 2], g[4 * q + 3]},
                        (f32x4_t){u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]});
      }
    }
  }
}

} // namespace

#define AXH_MX_DENSE_ARGS                                                                         \
  const uint8_t *wc, const uint8_t *ws, const uint8_t *xc, const uint8_t *xs, uint8_t *y,         \
      uint32_t n_rows, uint32_t nblk, uint32_t n_cols, uint32_t row_tiles
#define AXH_MX_DENSE_UNPACK                                                                       \
  const Args a{wc, ws,     wc,   ws,     xc,     xs, nullptr, y, nullptr,                         \
               n_rows, nblk, n_cols, n_cols, 1u, 0u, row_tiles}
#define AXH_MX_EXPERT_ARGS                                                                        \
  const uint8_t *wc, const uint8_t *ws, const uint8_t *uc, const uint8_t *us, const uint8_t *xc,  \
      const uint8_t *xs, const uint32_t *plan, uint8_t *y, uint8_t *ysc, uint32_t n_rows,         \
      uint32_t nblk, uint32_t n_x, uint32_t x_div, uint32_t n_experts, uint32_t row_tiles
#define AXH_MX_EXPERT_UNPACK                                                                      \
  const Args a{wc, ws, uc, us, xc, xs, plan, y, ysc, n_rows, nblk, 0u, n_x, x_div, n_experts,     \
               row_tiles}

// Skinny kernels: NI column groups of 32, NW waves.
#define AXH_MX_SKINNY(TN, T, NI, NW)                                                              \
  extern "C" __global__ void __launch_bounds__(64 * NW)                                           \
      axh_mxfp4_matmul_s##NI##_##TN(AXH_MX_DENSE_ARGS) {                                          \
    extern __shared__ f32x4_t part[];                                                             \
    AXH_MX_DENSE_UNPACK;                                                                          \
    skinny_body<kDense, T, false, NI, NW>(a, part);                                               \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(64 * NW)                                           \
      axh_mxfp4_expert_matmul_s##NI##_##TN(AXH_MX_EXPERT_ARGS) {                                  \
    extern __shared__ f32x4_t part[];                                                             \
    AXH_MX_EXPERT_UNPACK;                                                                         \
    skinny_body<kGrouped, T, false, NI, NW>(a, part);                                             \
  }
#define AXH_MX_SKINNY_GU(TN, T, PACKED, NI, NW)                                                   \
  extern "C" __global__ void __launch_bounds__(64 * NW)                                           \
      axh_mxfp4_expert_gate_up_s##NI##_##TN(AXH_MX_EXPERT_ARGS) {                                 \
    extern __shared__ f32x4_t part[];                                                             \
    AXH_MX_EXPERT_UNPACK;                                                                         \
    skinny_body<kGateUp, T, PACKED, NI, NW>(a, part);                                             \
  }
#define AXH_MX_SKINNY_N(NI, NW, NWG)              \
  AXH_MX_SKINNY(f32, TF32, NI, NW)                \
  AXH_MX_SKINNY(f16, TF16, NI, NW)                \
  AXH_MX_SKINNY(bf16, TBF16, NI, NW)              \
  AXH_MX_SKINNY_GU(f32, TF32, false, NI, NWG)     \
  AXH_MX_SKINNY_GU(f16, TF16, false, NI, NWG)     \
  AXH_MX_SKINNY_GU(bf16, TBF16, false, NI, NWG)   \
  AXH_MX_SKINNY_GU(mxfp4, TF32, true, NI, NWG)
AXH_MX_SKINNY_N(1, 8, 8)
AXH_MX_SKINNY_N(2, 8, 4)

// Tile kernels.
#define AXH_MX_TILE(NAME, TN, T, BM, BN, WM, WN)                                                  \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN)                                      \
      axh_mxfp4_matmul_##NAME##_##TN(AXH_MX_DENSE_ARGS) {                                         \
    extern __shared__ __align__(16) uint8_t tile[];                                                       \
    AXH_MX_DENSE_UNPACK;                                                                          \
    tile_body<kDense, T, false, BM, BN, WM, WN>(a, tile);                                         \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN)                                      \
      axh_mxfp4_expert_matmul_##NAME##_##TN(AXH_MX_EXPERT_ARGS) {                                 \
    extern __shared__ __align__(16) uint8_t tile[];                                                       \
    AXH_MX_EXPERT_UNPACK;                                                                         \
    tile_body<kGrouped, T, false, BM, BN, WM, WN>(a, tile);                                       \
  }
#define AXH_MX_TILE_GU(NAME, TN, T, PACKED, BM, BN, WM, WN)                                       \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN)                                      \
      axh_mxfp4_expert_gate_up_##NAME##_##TN(AXH_MX_EXPERT_ARGS) {                                \
    extern __shared__ __align__(16) uint8_t tile[];                                                       \
    AXH_MX_EXPERT_UNPACK;                                                                         \
    tile_body<kGateUp, T, PACKED, BM, BN, WM, WN>(a, tile);                                       \
  }
#define AXH_MX_TILE_N(NAME, BM, BN, WM, WN)                        \
  AXH_MX_TILE(NAME, f32, TF32, BM, BN, WM, WN)                     \
  AXH_MX_TILE(NAME, f16, TF16, BM, BN, WM, WN)                     \
  AXH_MX_TILE(NAME, bf16, TBF16, BM, BN, WM, WN)                   \
  AXH_MX_TILE_GU(NAME, f32, TF32, false, BM, BN, WM, WN)           \
  AXH_MX_TILE_GU(NAME, f16, TF16, false, BM, BN, WM, WN)           \
  AXH_MX_TILE_GU(NAME, bf16, TBF16, false, BM, BN, WM, WN)         \
  AXH_MX_TILE_GU(NAME, mxfp4, TF32, true, BM, BN, WM, WN)
AXH_MX_TILE_N(t128x128, 128, 128, 2, 2)
