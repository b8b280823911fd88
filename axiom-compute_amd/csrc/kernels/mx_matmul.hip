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
//   * K-split (few columns and rows, bound by the time that W's bytes take to
//     come): a workgroup has 16 or 32 rows of W (gate/up: 32 of each matrix) and
//     32 columns, its waves split the K axis;
//   * tile: a workgroup has a BM x BN tile, each wave a part of it, and all its
//     waves go through K together.
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

template <int kk>
__device__ __forceinline__ f32x4_t mfma16(u32x4_t a, u32x4_t b, f32x4_t c, uint32_t sa,
                                          uint32_t sb) {
  const i32x8_t A = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8_t B = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, kk, (int)sa, kk, (int)sb);
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
template <bool kShort>
__device__ __forceinline__ u32x2_t load_scales8(__amdgpu_buffer_rsrc_t r, uint32_t row_off,
                                                ScaleStep st, uint32_t nblk) {
  if constexpr (!kShort)
    return __builtin_amdgcn_raw_buffer_load_b64(r, (int)(row_off + st.at), 0, 0);
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

// Four consecutive rows of one output column; kVec: n_rows and y allow whole
// vector stores (store_whole), so the four are all there or none.
template <class T>
__device__ __forceinline__ bool store_whole(const uint8_t *y, uint32_t n_rows) {
  return n_rows % 4u == 0u && ((uintptr_t)y & (4u * T::kBytes - 1u)) == 0u;
}
template <class T, bool kVec>
__device__ __forceinline__ void store4(uint8_t *col, uint32_t r, uint32_t n_rows, f32x4_t v) {
  uint8_t *p = col + (uint64_t)r * T::kBytes;
  if constexpr (kVec) {
    if (r >= n_rows) return;
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
  const float divisor = mx_divisor(e);
  // quarters 0 and 1, 2 and 3: four codes (16 bits) each
  const uint32_t q01 = e == 255u ? 0u : fp4_pack8(h, divisor);
  const uint32_t q23 = e == 255u ? 0u : fp4_pack8(h + 8, divisor);
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

// Number k of a contiguous part for each of the eight XCDs, to which consecutive
// workgroups go in turn: tiles that share data then share an L2.
__device__ __forceinline__ uint32_t by_xcd(uint32_t id, uint32_t total) {
  const uint32_t per = total / 8u, rest = total % 8u, xcd = id % 8u;
  return xcd * per + (xcd < rest ? xcd : rest) + id / 8u;
}

// Inclusive prefix sum over the wave.
__device__ __forceinline__ uint32_t prefix(uint32_t v, uint32_t lane) {
#pragma unroll
  for (uint32_t d = 1; d < 64u; d <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// Workgroup -> tile, columns fastest in dense products and rows fastest in expert
// layers, where the tiles of one group of columns share X.
//   How many tiles an expert layer has is in the plan only; the grid is an upper
// bound, and the XCDs share the real ones (sharing the grid's left the last XCDs
// without work: 333 tokens, 6 of 40 experts, 1312 x 736, 26.1 us in place of 15.7).  Every wave finds the expert of its tile: each lane sums up
// the tiles of its experts, and for more than 64 experts a second step looks through
// those of the lane that was found.
template <Mode M, int BN> __device__ __forceinline__ Tile tile_of(const Args &a) {
  Tile r;
  if constexpr (M == kDense) {
    const uint32_t t = by_xcd(blockIdx.x, gridDim.x);
    const uint32_t cols = (a.n_cols + BN - 1u) / BN;
    r.m = t / cols;
    r.n0 = (t - r.m * cols) * BN;
    r.count = a.n_cols - r.n0;
    r.first = 0;
    r.expert = 0;
    r.real = true;
  } else {
    const uint32_t lane = threadIdx.x & 63u, slots = a.n_x * a.x_div;
    const uint32_t per = (a.n_experts + 63u) / 64u;
    auto offset = [&](uint32_t e) { // kept in range: see slot_at
      const uint32_t o = a.plan[e < a.n_experts ? e : a.n_experts];
      return o < slots ? o : slots;
    };
    auto tiles_of = [](uint32_t lo, uint32_t hi) {
      return hi > lo ? (hi - lo + BN - 1u) / BN : 0u;
    };
    uint32_t e0 = lane * per, lo = offset(e0), hi = lo, tiles = 0;
#pragma unroll 4
    for (uint32_t j = 0; j < per; ++j) {
      const uint32_t next = offset(e0 + j + 1u);
      tiles += tiles_of(hi, next);
      hi = next;
    }
    uint32_t incl = prefix(tiles, lane);
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63) * a.row_tiles;
    r.real = blockIdx.x < total;
    r.m = r.n0 = r.count = r.first = r.expert = 0;
    if (!r.real) return r;
    const uint32_t t = by_xcd(blockIdx.x, total);
    uint32_t nt = t / a.row_tiles;
    r.m = t - nt * a.row_tiles;
    int who = __builtin_ctzll(__ballot(nt < incl));
    nt -= (uint32_t)__builtin_amdgcn_readlane((int)(incl - tiles), who);
    if (per > 1u) {
      const uint32_t of = (uint32_t)who * per;
      e0 = of + (lane < per ? lane : per);
      lo = offset(e0);
      hi = offset(e0 + (lane < per ? 1u : 0u));
      tiles = tiles_of(lo, hi);
      incl = prefix(tiles, lane);
      who = __builtin_ctzll(__ballot(nt < incl) | 1ull << 63);
      nt -= (uint32_t)__builtin_amdgcn_readlane((int)(incl - tiles), who);
    }
    r.expert = (uint32_t)__builtin_amdgcn_readlane((int)e0, who);
    r.expert = r.expert < a.n_experts ? r.expert : a.n_experts - 1u;
    const uint32_t l = (uint32_t)__builtin_amdgcn_readlane((int)lo, who) + nt * BN;
    const uint32_t h = (uint32_t)__builtin_amdgcn_readlane((int)hi, who);
    r.first = l;
    r.count = h - l;
    r.real = l < h;
  }
  if (r.count > (uint32_t)BN) r.count = BN;
  return r;
}

// The slot at place p of the plan's order.  Kept in range, as the offsets are: a plan
// that was overwritten gives wrong rows, but no access outside the buffers.
__device__ __forceinline__ uint32_t slot_at(const Args &a, uint32_t p) {
  const uint32_t slot = a.plan[((a.n_experts + 1u + 15u) & ~15u) + p];
  const uint32_t last = a.n_x * a.x_div - 1u;
  return slot < last ? slot : last;
}

// Finishes four rows r .. r + 3 of a column (not packed).
template <Mode M, class T, bool kVec>
__device__ __forceinline__ void emit4(const Args &a, uint32_t out_row, uint32_t r, f32x4_t g,
                                      f32x4_t u) {
  if constexpr (M == kGateUp) {
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = swiglu(g[i], u[i]);
  }
  store4<T, kVec>(a.y + (uint64_t)out_row * a.n_rows * T::kBytes, r, a.n_rows, g);
}

// ---------------------------------------------------------------------------
// K-split kind: 32 or 16 rows (gate/up: 32 of each matrix) by 32 columns, NW
// waves.  Steps of 256 along K go to the waves in turn; each wave fills NB
// buffers of its own in LDS by direct-to-LDS loads, so nothing but its load
// counter is waited for until the waves' partial tiles are summed in LDS, in
// the waves' order.  The LDS rows are the tile kind's.
//   Bound by the weights' bytes and, as these are few, by the latency of a launch and of
// the first loads: 4096 x 4096, 32 columns, 6.6 us (8.9 MB, 1.7 us at the rate of a
// copy); 4096 x 14336, 32 columns, 13.9 us with 16 rows (31 MB, 6.0 us), where a CU's 8
// waves ask for 128 bytes of a row at a time.
// ---------------------------------------------------------------------------
template <Mode M, class T, bool kPacked, int kRows, int NW, int NB>
__device__ __forceinline__ void ksplit_body(const Args &a, uint8_t *lds) {
  constexpr int MI = M == kGateUp ? 2 : 1;
  constexpr uint32_t kARows = MI * kRows, kBuf = (kARows + 32u) * 128u;
  constexpr int kALoads = kARows / 8, kLoads = kALoads + 4;
  static_assert(kRows == 32 || (kRows == 16 && M != kGateUp), "16 rows: one matrix");
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const Tile t = tile_of<M, 32>(a);
  if (!t.real) return;
  const uint32_t row0 = t.m * kRows;
  const uint32_t nblk = a.nblk, row_bytes = nblk * 16u;
  const uint64_t wat = ((uint64_t)t.expert * a.n_rows + row0) * nblk;
  const uint32_t rows = a.n_rows - row0 < (uint32_t)kRows ? a.n_rows - row0 : (uint32_t)kRows;
  const __amdgpu_buffer_rsrc_t wc = rsrc(a.wc + wat * 16u, rows * row_bytes);
  const __amdgpu_buffer_rsrc_t ws = rsrc(a.ws + wat, rows * nblk);
  const __amdgpu_buffer_rsrc_t uc = M == kGateUp ? rsrc(a.uc + wat * 16u, rows * row_bytes) : wc;
  const __amdgpu_buffer_rsrc_t us = M == kGateUp ? rsrc(a.us + wat, rows * nblk) : ws;
  const uint64_t xbase = M == kDense ? t.n0 : 0u;
  const uint32_t xrows = M == kDense ? t.count : a.n_x;
  const __amdgpu_buffer_rsrc_t xc = rsrc(a.xc + xbase * row_bytes, xrows * row_bytes);
  const __amdgpu_buffer_rsrc_t xs = rsrc(a.xs + xbase * nblk, xrows * nblk);
  auto slot_of = [&](uint32_t j) {
    return M == kDense ? t.n0 + j : slot_at(a, t.first + (j < t.count ? j : 0u));
  };
  auto xrow_of = [&](uint32_t j) { return M == kDense ? j : slot_of(j) / a.x_div; };

  // this lane's part of each load of codes: row 8 * load + lane / 8 of A or of B
  const uint32_t l8 = lane >> 3;
  uint32_t off[kLoads], piece[2]; // the piece depends on the row mod 16
#pragma unroll
  for (uint32_t p = 0; p < 2; ++p) piece[p] = (lane & 7u) ^ ((4u * p + (l8 >> 1)) & 7u);
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    if (i < kALoads) {
      off[i] = ((8u * i + l8) % kRows) * row_bytes + piece[i & 1] * 16u;
    } else {
      const uint32_t j = 8u * (i - kALoads) + l8;
      off[i] = j < t.count ? xrow_of(j) * row_bytes + piece[i & 1] * 16u : kFar;
    }
  }
  // the lane's rows of scales
  const uint32_t r32 = lane & 31u, group = kRows == 32 ? lane >> 5 : lane >> 4;
  const uint32_t arow = (lane & (kRows - 1u)) * nblk;
  uint32_t brow[kRows == 32 ? 1 : 2];
#pragma unroll
  for (uint32_t n = 0; n < (kRows == 32 ? 1u : 2u); ++n) {
    const uint32_t j = kRows == 32 ? r32 : 16u * n + (lane & 15u);
    brow[n] = j < t.count ? xrow_of(j) * nblk : kFar;
  }
  constexpr int NI = kRows == 32 ? 1 : 2; // operand tiles of B
  const uint32_t sel = kRows == 32 ? scale_selector(group) : group | (group + 4u) << 8;

  uint8_t *const ring = lds + wave * (NB * kBuf);
  const uint32_t steps = (nblk + 7u) / 8u;
  struct Scales {
    u32x2_t a[MI], b[NI];
  };
  auto request = [&](uint32_t s, uint32_t buf) { // steps past the end: zeros
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const bool in = 8u * s + piece[i & 1] < nblk;
      const bool up = M == kGateUp && i >= kRows / 8 && i < kALoads;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(i < kALoads ? (up ? uc : wc) : xc,
                                               (lds_void_t *)(ring + buf * kBuf + i * 1024u), 16,
                                               (int)(in ? off[i] + s * 128u : kFar), 0, 0, 0);
    }
  };
  auto load_scales = [&](uint32_t s, Scales &c, auto few) {
    constexpr bool kFew = decltype(few)::value;
    const ScaleStep st = scale_step(s < steps ? s : steps - 1u, nblk);
    c.a[0] = load_scales8<kFew>(ws, arow, st, nblk);
    if constexpr (M == kGateUp) c.a[1] = load_scales8<kFew>(us, arow, st, nblk);
#pragma unroll
    for (int n = 0; n < NI; ++n) c.b[n] = load_scales8<kFew>(xs, brow[n], st, nblk);
  };

  f32x16_t acc[MI] = {};    // 32 rows
  f32x4_t acc16[2] = {};    // 16 rows: two groups of 16 columns
  auto multiply = [&](uint32_t s, uint32_t buf, const Scales &c) {
    const ScaleStep st = scale_step(s, nblk);
    const uint8_t *p = ring + buf * kBuf;
    uint32_t sa[MI], sb[NI];
#pragma unroll
    for (int m = 0; m < MI; ++m) sa[m] = lane_scales(c.a[m], st, sel);
#pragma unroll
    for (int n = 0; n < NI; ++n) sb[n] = lane_scales(c.b[n], st, sel);
    const uint32_t row = lane & (kRows - 1u), swz = (row >> 1) & 7u;
    auto frag = [&](uint32_t first, uint32_t k) {
      constexpr uint32_t kG = kRows == 32 ? 2u : 4u;
      return *reinterpret_cast<const u32x4_t *>(p + (first + row) * 128u +
                                                (((kG * k + group) ^ swz) * 16u));
    };
    if constexpr (kRows == 32) {
      u32x4_t fa[MI][4], fb[4];
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
#pragma unroll
        for (uint32_t m = 0; m < MI; ++m) fa[m][k] = frag(32u * m, k);
        fb[k] = frag(kARows, k);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // read before the buffer is refilled
      request(s + NB * NW, buf);
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        acc[m] = mfma<0>(fa[m][0], fb[0], acc[m], sa[m], sb[0]);
        acc[m] = mfma<1>(fa[m][1], fb[1], acc[m], sa[m], sb[0]);
        acc[m] = mfma<2>(fa[m][2], fb[2], acc[m], sa[m], sb[0]);
        acc[m] = mfma<3>(fa[m][3], fb[3], acc[m], sa[m], sb[0]);
      }
    } else {
      u32x4_t fa[2], fb[2][2];
#pragma unroll
      for (uint32_t k = 0; k < 2; ++k) {
        fa[k] = frag(0, k);
#pragma unroll
        for (uint32_t n = 0; n < 2; ++n) fb[n][k] = frag(16u + 16u * n, k);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      request(s + NB * NW, buf);
#pragma unroll
      for (uint32_t n = 0; n < 2; ++n) {
        acc16[n] = mfma16<0>(fa[0], fb[n][0], acc16[n], sa[0], sb[n]);
        acc16[n] = mfma16<1>(fa[1], fb[n][1], acc16[n], sa[0], sb[n]);
      }
    }
  };

  // Everything that a step requests is requested in one go, so that the counter
  // says which steps have landed: all but the NB - 1 younger ones.
  constexpr int kStepLoads = kLoads + MI + NI;
  if (nblk >= 8u) {
    Scales c[NB];
#pragma unroll
    for (uint32_t i = 0; i < NB; ++i) {
      load_scales(wave + i * NW, c[i], std::false_type());
      request(wave + i * NW, i);
    }
    for (uint32_t s = wave; s < steps; s += NB * NW) {
#pragma unroll
      for (uint32_t i = 0; i < NB; ++i) {
        const uint32_t at = s + i * NW;
        if (at >= steps) break;
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NB - 1) * kStepLoads) : "memory");
        const Scales now = c[i];
        load_scales(at + NB * NW, c[i], std::false_type());
        multiply(at, i, now);
      }
    }
  } else if (wave == 0u) { // one step, of fewer blocks than a load of scales has
    Scales c;
    load_scales(0, c, std::true_type());
    request(0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    multiply(0, 0, c);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // loads past the last step
  __syncthreads();

  // partial tiles: [wave][matrix or column group][quarter][lane]
  f32x4_t *const part = reinterpret_cast<f32x4_t *>(lds);
  constexpr uint32_t kQuarters = kRows == 32 ? 4u * MI : 2u;
  if constexpr (kRows == 32) {
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        part[(wave * kQuarters + m * 4u + q) * 64u + lane] =
            (f32x4_t){acc[m][4 * q], acc[m][4 * q + 1], acc[m][4 * q + 2], acc[m][4 * q + 3]};
  } else {
#pragma unroll
    for (int n = 0; n < 2; ++n) part[(wave * kQuarters + n) * 64u + lane] = acc16[n];
  }
  __syncthreads();
  auto total = [&](uint32_t q) {
    f32x4_t v = part[q * 64u + lane];
#pragma unroll
    for (uint32_t w = 1; w < NW; ++w) v += part[(w * kQuarters + q) * 64u + lane];
    return v;
  };
  const bool whole = store_whole<T>(a.y, a.n_rows);
  auto emit = [&](uint32_t j, uint32_t r, f32x4_t g, f32x4_t u) {
    if (j >= t.count) return;
    if (whole)
      emit4<M, T, true>(a, slot_of(j), r, g, u);
    else
      emit4<M, T, false>(a, slot_of(j), r, g, u);
  };
  if constexpr (kPacked) {
    if (wave == 0u) {
      float h[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4_t g = total(q), u = total(4u * (MI - 1) + q);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[4 * q + i] = swiglu(g[i], u[i]);
      }
      store_packed(a.y, a.ysc, (uint64_t)slot_of(r32) * (a.n_rows / 32u) + t.m, h, group,
                   r32 < t.count);
    }
  } else if constexpr (kRows == 32) {
    if (wave < 4u) {
      const f32x4_t g = total(wave), u = M == kGateUp ? total(4u * (MI - 1) + wave) : g;
      emit(r32, row0 + 8u * wave + 4u * group, g, u);
    }
  } else if (wave < 2u) {
    const f32x4_t g = total(wave);
    emit(16u * wave + (lane & 15u), row0 + 4u * group, g, g);
  }
}

// ---------------------------------------------------------------------------
// Tile kind: BM x BN outputs (gate/up: BM / 2 rows of each matrix, in turns of
// 32), WM x WN waves, rows of at least sixteen blocks.  K goes in steps of 256
// through NBUF LDS buffers filled by direct-to-LDS loads.  An LDS row is 128
// bytes, the codes of one step (a whole line, so that eight lanes of a load are
// one request to L2), with 16-byte piece c at place c ^ (row / 2 % 8): the
// sixteen rows that a quarter of a fragment read touches (rows 0-3, 12-15, 20-23
// and 24-27, or the others, of 32) then meet all the banks.  The scales of two
// steps, 16 bytes a row, go through registers to LDS.
//
// A step is four parts of 64 columns; a part's fragments are read among the
// products of the part before it.  One barrier a step, before its last part: by
// then every wave has read its last fragments of the step, so its buffer is
// refilled during the last part and the next step's first one, and has seen its
// own loads of the next step land.
//   WK groups of such waves may share the K axis, each with buffers of its own, so
// that twice the bytes are on their way where a CU has one workgroup; the groups'
// sums meet in LDS.
//   kShort: rows of fewer than 16 blocks, two steps at most.  A row's scales come with
// the next rows' behind them, or, at the end of the array, with those before; they are
// shifted down and the others cleared, as a NaN would pass through the codes' zeros.
// ---------------------------------------------------------------------------
template <Mode M, class T, bool kPacked, int BM, int BN, int WM, int WN, int WK,
          int NBUF, bool kShort = false>
__device__ __forceinline__ void tile_body(const Args &a, uint8_t *all_lds) {
  constexpr int NW = WM * WN, MI = BM / WM / 32, NI = BN / WN / 32;
  constexpr int kSRows = (BM + BN + 64 * NW - 1) / (64 * NW); // rows of scales per lane
  constexpr uint32_t kBuf = (BM + BN) * 128u, kSBuf = kSRows * 64u * NW * 16u;
  constexpr int kLate = kShort ? 0 : kSRows; // loads of scales behind those of a step
  constexpr int kLoads = (BM + BN) / 8 / NW; // per wave and step; rows of A first
  constexpr int kALoads = BM / 8 / NW, kHalf = kLoads / 2;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "whole loads per wave");
  static_assert(NW % 2 == 0, "the rows of a lane's loads are alike mod 16");
  static_assert(M != kGateUp || MI % 2 == 0, "gate and up rows in one wave");
  constexpr uint32_t kRows = M == kGateUp ? BM / 2 : BM; // rows of y
  constexpr uint32_t kRegion = NBUF * kBuf + 2u * kSBuf;
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t any_wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t group = WK == 1 ? 0u : any_wave / NW, wave = any_wave - group * NW;
  const uint32_t thread = wave * 64u + lane; // of the group
  uint8_t *const lds = all_lds + group * kRegion, *const slds = lds + NBUF * kBuf;
  const uint32_t wm = wave / WN, wn = wave % WN;
  const uint32_t half = lane >> 5, r32 = lane & 31u;
  const Tile t = tile_of<M, BN>(a);
  if (!t.real) return;
  const uint32_t row0 = t.m * kRows;
  const uint32_t nblk = a.nblk, row_bytes = nblk * 16u;
  // the group's blocks: from kb, a multiple of 16 (two steps) but for the last group
  const uint32_t share = WK == 1 ? nblk : (nblk + 16u * WK - 1u) / (16u * WK) * 16u;
  const uint32_t kb = group * share, ke = kb + share < nblk ? kb + share : nblk;
  const uint32_t kn = kb < ke ? ke - kb : 0u;
  const uint64_t wat = (uint64_t)t.expert * a.n_rows * nblk + (uint64_t)row0 * nblk;
  const uint32_t rows = a.n_rows - row0 < kRows ? a.n_rows - row0 : kRows;
  const __amdgpu_buffer_rsrc_t wc = rsrc(a.wc + wat * 16u, rows * row_bytes);
  const __amdgpu_buffer_rsrc_t uc = M == kGateUp ? rsrc(a.uc + wat * 16u, rows * row_bytes) : wc;
  const uint64_t xbase = M == kDense ? t.n0 : 0u;
  const uint32_t xrows = M == kDense ? t.count : a.n_x;
  const __amdgpu_buffer_rsrc_t xc = rsrc(a.xc + xbase * row_bytes, xrows * row_bytes);
  // row of X of column j of the tile, and the row of y that it gives
  auto slot_of = [&](uint32_t j) {
    return M == kDense ? t.n0 + j : slot_at(a, t.first + (j < t.count ? j : 0u));
  };

  // this lane's part of each load of codes: row 8 * (load * NW + wave) + lane / 8
  const uint32_t l8 = lane >> 3, piece = (lane & 7u) ^ ((4u * wave + (l8 >> 1)) & 7u);
  // The columns' slots are requested first and used behind the requests of A below:
  // they are the end of a chain of loads, expert, slot, row of X.
  uint32_t off[kLoads], slot[kLoads - kALoads], sslot[kSRows];
#pragma unroll
  for (int i = kALoads; i < kLoads; ++i) {
    const uint32_t j = 8u * ((i - kALoads) * NW + wave) + l8;
    slot[i - kALoads] = slot_of(j);
  }
#pragma unroll
  for (int i = 0; i < kSRows; ++i) {
    const uint32_t r = 64u * NW * i + thread, j = r < (uint32_t)BM ? 0u : r - BM;
    sslot[i] = slot_of(j < t.count ? j : t.count - 1u);
  }
  auto xrow = [&](uint32_t s) { return M == kDense ? s - t.n0 : s / a.x_div; };
#pragma unroll
  for (int i = 0; i < kALoads; ++i) {
    const uint32_t r = 8u * (i * NW + wave) + l8;
    const uint32_t row = M == kGateUp ? (r >> 6) * 32u + (r & 31u) : r;
    off[i] = row * row_bytes + (kb + piece) * 16u;
  }
  const uint32_t steps = (share + 7u) / 8u;
  // load i of step s into buffer buf; steps past the end: zeros
  auto request = [&](uint32_t s, uint32_t buf, int i) {
    const bool in = 8u * s + piece < kn;
    const uint32_t r8 = 8u * ((i < kALoads ? i : i - kALoads) * NW + wave);
    const bool up = M == kGateUp && i < kALoads && ((r8 >> 5) & 1u);
    uint8_t *to = lds + buf * kBuf + ((i < kALoads ? 0u : (uint32_t)BM) + r8) * 128u;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(i < kALoads ? (up ? uc : wc) : xc, (lds_void_t *)to,
                                             16, (int)(in ? off[i] + s * 128u : kFar), 0, 0, 0);
  };

  // The first loads: A of the steps 0 .. NBUF - 2, then their X, then half of step
  // NBUF - 1's.  The waits count on every load of a step being older than all of the
  // steps from NBUF - 1 on.
  static_assert(NBUF <= 3, "else step 1's X is younger than step 2's A");
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (uint32_t st = 0; st + 1u < NBUF; ++st)
#pragma unroll
    for (int i = 0; i < kALoads; ++i) request(st, st, i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = kALoads; i < kLoads; ++i) {
    const uint32_t j = 8u * ((i - kALoads) * NW + wave) + l8;
    off[i] = j < t.count ? xrow(slot[i - kALoads]) * row_bytes + (kb + piece) * 16u : kFar;
  }

  // scales: lane (64 * NW * i + thread) takes a row of A or of B (rows that there
  // are not: the last one's, whose products are not stored)
  const uint8_t *sbase[kSRows];
#pragma unroll
  for (int i = 0; i < kSRows; ++i) {
    const uint32_t r = 64u * NW * i + thread;
    if (r < (uint32_t)BM) {
      uint32_t row = M == kGateUp ? (r >> 6) * 32u + (r & 31u) : r;
      row = row < rows ? row : rows - 1u;
      const bool up = M == kGateUp && ((r >> 5) & 1u);
      sbase[i] = (up ? a.us : a.ws) + wat + (uint64_t)row * nblk;
    } else { // (lanes past the rows of B repeat its last one)
      sbase[i] = a.xs + (xbase + xrow(sslot[i])) * nblk;
    }
  }
  // the scales of blocks 16 p .. 16 p + 15, read inside the row: at its end from
  // further back, and shifted down by put_scales
  u32x4_t sreg[kSRows];
  const uint32_t last16 = nblk - 16u;
  uint32_t back[kSRows]; // kShort: bytes from where the load begins to the row
  if constexpr (kShort) {
    const uint64_t all_a = (uint64_t)(M == kDense ? 1u : a.n_experts) * a.n_rows * nblk;
    const uint64_t all_b = (uint64_t)a.n_x * nblk; // (both 16 at least)
#pragma unroll
    for (int i = 0; i < kSRows; ++i) {
      const uint32_t r = 64u * NW * i + thread;
      const bool is_a = r < (uint32_t)BM;
      const bool up = is_a && M == kGateUp && ((r >> 5) & 1u);
      const uint8_t *end = is_a ? (up ? a.us : a.ws) + all_a : a.xs + all_b;
      const uint32_t rest = end - sbase[i] < 16 ? (uint32_t)(end - sbase[i]) : 16u;
      back[i] = 16u - rest;
      sbase[i] -= back[i];
    }
  }
  auto get_scales = [&](uint32_t p) {
    if constexpr (kShort) { // one load in all: the waits count none behind it
      if (p == 0u)
#pragma unroll
        for (int i = 0; i < kSRows; ++i) __builtin_memcpy(&sreg[i], sbase[i], 16);
      return;
    }
    const uint32_t at = kb + 16u * p < last16 ? kb + 16u * p : last16;
#pragma unroll
    for (int i = 0; i < kSRows; ++i) __builtin_memcpy(&sreg[i], sbase[i] + at, 16);
  };
  auto put_scales = [&](uint32_t p) {
    if constexpr (kShort) {
      const uint64_t all = p ? 0ull : ~0ull; // steps past the row: zeros
      const uint64_t in_lo = nblk >= 8u ? all : all & ((1ull << 8u * nblk) - 1u);
      const uint64_t in_hi = nblk > 8u ? all & ((1ull << 8u * (nblk - 8u)) - 1u) : 0u;
#pragma unroll
      for (int i = 0; i < kSRows; ++i) {
        const uint32_t shift = 8u * (back[i] & 7u);
        uint64_t lo = (uint64_t)sreg[i].y << 32 | sreg[i].x;
        uint64_t hi = (uint64_t)sreg[i].w << 32 | sreg[i].z;
        lo = back[i] & 8u ? hi : lo;
        hi = back[i] & 8u ? 0u : hi;
        lo = (lo >> shift | (hi << 1) << (63u - shift)) & in_lo;
        hi = hi >> shift & in_hi;
        *reinterpret_cast<u32x4_t *>(slds + (p & 1u) * kSBuf + (64u * NW * i + thread) * 16u) =
            (u32x4_t){(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      }
      return;
    }
    // bytes, 15 at most if there are such blocks
    const uint32_t d = kb + 16u * p < last16 ? 0u : kb + 16u * p - last16;
    const uint32_t bits = 8u * (d & 7u);
#pragma unroll
    for (int i = 0; i < kSRows; ++i) {
      uint64_t lo = (uint64_t)sreg[i].y << 32 | sreg[i].x, hi = (uint64_t)sreg[i].w << 32 | sreg[i].z;
      lo = d & 8u ? hi : lo;
      hi = d & 8u ? 0u : hi;
      lo = lo >> bits | (hi << 1) << (63u - bits);
      hi >>= bits;
      if (WK > 1 && d > 15u) lo = hi = 0u; // a group may have none: no NaN in its zeros' place
      *reinterpret_cast<u32x4_t *>(slds + (p & 1u) * kSBuf + (64u * NW * i + thread) * 16u) =
          (u32x4_t){(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
  };

  f32x16_t acc[MI][NI] = {};
  const uint32_t sel = scale_selector(half);
  uint32_t frag[4]; // byte offset of the lane's piece of part kk in a 32-row tile
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k)
    frag[k] = r32 * 128u + (((2u * k + half) ^ ((r32 >> 1) & 7u)) * 16u);
  const uint32_t abase = wm * (MI * 4096u), bbase = BM * 128u + wn * (NI * 4096u);
  struct Frags {
    u32x4_t a[MI], b[NI];
  };
  auto read_frag = [&](Frags &f, int k, uint32_t buf, int i) {
    const uint8_t *p = lds + buf * kBuf + frag[k];
    if (i < MI)
      f.a[i] = *reinterpret_cast<const u32x4_t *>(p + abase + i * 4096);
    else
      f.b[i - MI] = *reinterpret_cast<const u32x4_t *>(p + bbase + (i - MI) * 4096);
  };
  auto read_frags = [&](Frags &f, int k, uint32_t buf) {
#pragma unroll
    for (int i = 0; i < MI + NI; ++i) read_frag(f, k, buf, i);
  };
  struct Scales { // of one step, a byte a part
    uint32_t a[MI], b[NI];
  };
  auto read_scales = [&](Scales &c, uint32_t s) {
    const uint8_t *q = slds + ((s >> 1) & 1u) * kSBuf + (s & 1u) * 8u + r32 * 16u;
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      const u32x2_t v = *reinterpret_cast<const u32x2_t *>(q + (wm * MI + m) * 512u);
      c.a[m] = __builtin_amdgcn_perm(v.y, v.x, sel);
    }
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const u32x2_t v = *reinterpret_cast<const u32x2_t *>(q + BM * 16u + (wn * NI + n) * 512u);
      c.b[n] = __builtin_amdgcn_perm(v.y, v.x, sel);
    }
  };
  auto multiply = [&](const Frags &f, const Scales &c, auto kk) {
    constexpr int K = decltype(kk)::value;
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n)
        acc[m][n] = mfma<K>(f.a[m], f.b[n], acc[m][n], c.a[m], c.b[n]);
  };
  constexpr std::integral_constant<int, 0> k0;
  constexpr std::integral_constant<int, 1> k1;
  constexpr std::integral_constant<int, 2> k2;
  constexpr std::integral_constant<int, 3> k3;
  auto after = [](uint32_t b) { return b + 1u == NBUF ? 0u : b + 1u; };
  // What goes among a part's products: the next part's fragments f (part k of
  // buffer from) and the requests [begin, end) of step s into buffer `to`.  The
  // compiler keeps reads and requests in this order, both being accesses to LDS.
  constexpr int kReads = MI + NI;
  auto loads = [&](Frags &f, int k, uint32_t from, uint32_t s, uint32_t to, int begin, int end) {
    const int n = end - begin;
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      read_frag(f, k, from, i);
#pragma unroll
      for (int r = begin + i * n / kReads; r < begin + (i + 1) * n / kReads; ++r)
        request(s, to, r);
    }
  };
  auto interleave = [&](auto requests) {
    constexpr int kPer = (MI * NI + kReads - 1) / kReads, kN = decltype(requests)::value;
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);    // LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, kPer, 0); // MFMA
      if (kN > 0) __builtin_amdgcn_sched_group_barrier(0x020, (kN + kReads - 1) / kReads, 0);
    }
  };
  Frags f0, f1;
  Scales c0, c1;
  constexpr std::integral_constant<int, 0> kNone;
  constexpr std::integral_constant<int, kHalf> kFirst;
  constexpr std::integral_constant<int, kLoads - kHalf> kSecond;
  // Step s is in buffer buf, step s + 1 in buffer then; before: buffer of step
  // s - 1.  The scales of two steps come together, and early, as a load that is
  // late holds up all the counted ones behind it: those of steps s + 3 and s + 4
  // are requested in an odd step s, after the requests that its barrier waits for,
  // and put into LDS in step s + 2.
  auto step = [&](uint32_t s, auto odd, uint32_t before, uint32_t buf, uint32_t then,
                  const Scales &c, Scales &next) {
    constexpr bool kOdd = decltype(odd)::value;
    __builtin_amdgcn_sched_barrier(0);
    if (kOdd) put_scales((s >> 1) + 1u); // read after the barrier
    loads(f1, 1, buf, s + NBUF - 1u, before, kHalf, kLoads);
    multiply(f0, c, k0);
    interleave(kSecond);
    __builtin_amdgcn_sched_barrier(0);
    if (kOdd && !kShort) get_scales((s >> 1) + 2u); // behind the requests above
    read_frags(f0, 2, buf);
    multiply(f1, c, k1);
    interleave(kNone);
    __builtin_amdgcn_sched_barrier(0);
    read_frags(f1, 3, buf);
    multiply(f0, c, k2);
    interleave(kNone);
    __builtin_amdgcn_sched_barrier(0);
    // step s + 1 has landed: of the younger loads, NBUF - 2 steps' and, in an odd step
    // or with a third buffer, the scales', may be on their way
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(
                     (NBUF - 2) * kLoads + (kOdd || NBUF > 2 ? kLate : 0))
                 : "memory");
    __builtin_amdgcn_sched_barrier(0);
    loads(f0, 0, then, s + NBUF, buf, 0, kHalf);
    multiply(f1, c, k3);
    interleave(kFirst);
    read_scales(next, s + 1u);
  };

  get_scales(0);
#pragma unroll
  for (uint32_t st = 0; st + 1u < NBUF; ++st)
#pragma unroll
    for (int i = kALoads; i < kLoads; ++i) request(st, st, i);
#pragma unroll
  for (int i = 0; i < kHalf; ++i) request(NBUF - 1u, NBUF - 1u, i);
  put_scales(0);
  if (!kShort) get_scales(1);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(
                   (NBUF - 2) * (kLoads - kALoads) + kHalf + kLate) // (all younger than step 0)
               : "memory");
  read_frags(f0, 0, 0);
  read_scales(c0, 0);
  // Groups of two steps, zeros past the last one.  No branch inside: the compiler
  // moves products over one, and then past the barriers, which leaves the loads
  // nothing to hide behind.
  uint32_t b0 = 0, before = NBUF - 1u;
  for (uint32_t s = 0; s < steps; s += 2u) {
    const uint32_t b1 = after(b0), b2 = after(b1);
    step(s, std::false_type(), before, b0, b1, c0, c1);
    step(s + 1u, std::true_type(), b0, b1, b2, c1, c0);
    before = b1;
    b0 = b2;
  }

  // Loads past the last step have landed and every wave is done with LDS: it holds
  // the waves' results next.  What follows is not computed ahead of the loop, where
  // registers are few.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  uint32_t tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const uint32_t l = tid & 63u, col32 = tid & 31u, half4 = (tid >> 5 & 1u) * 4u;
  if constexpr (WK > 1) {
    // the other groups' sums, added in their order; past what the waves write below
    constexpr uint32_t kWave = MI * NI * 4096u, kAt = NW * 32u * (BM / WM * 4u + 16u);
    static_assert(kAt + (WK - 1) * NW * kWave <= WK * kRegion, "the sums fit LDS");
    uint8_t *const part = all_lds + kAt + wave * kWave + l * 16u;
    if (group != 0u) {
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4_t *>(part + (group - 1u) * (NW * kWave) +
                                         ((m * NI + n) * 4 + q) * 1024) =
                (f32x4_t){acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2],
                          acc[m][n][4 * q + 3]};
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (group != 0u) return;
#pragma unroll
    for (int g = 0; g < WK - 1; ++g)
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4_t v = *reinterpret_cast<const f32x4_t *>(
                part + g * (NW * kWave) + ((m * NI + n) * 4 + q) * 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][n][4 * q + i] += v[i];
          }
  }
  constexpr int kStep = M == kGateUp ? 2 : 1, kBlocks = MI / kStep; // 32-row blocks of a wave
  const uint32_t wrow0 = row0 + wm * (kBlocks * 32u);               // the wave's first row of y
  if constexpr (kPacked) {
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const uint32_t j = (wn * NI + n) * 32u + col32;
      const uint32_t out = slot_of(j);
#pragma unroll
      for (int m = 0; m < MI; m += kStep) {
        float h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = swiglu(acc[m][n][i], acc[m + kStep - 1][n][i]);
        const uint32_t fb = wrow0 / 32u + m / kStep;
        store_packed(a.y, a.ysc, (uint64_t)out * (a.n_rows / 32u) + fb, h, half4 / 4u,
                     j < t.count && fb < a.n_rows / 32u);
      }
    }
  } else {
    // A column of the wave's block after another in LDS (with 16 bytes between, so
    // that the columns of a write meet all the banks), and from there in whole
    // rows of 16-byte pieces: a store instruction then writes 256 to 512
    // consecutive bytes of a column of y in place of 32 bytes of 32 columns.
    constexpr uint32_t kColBytes = kBlocks * 32u * T::kBytes, kPitch = kColBytes + 16u;
    constexpr uint32_t kLanes = kColBytes / 16u, kCols = 64u / kLanes; // lanes of a column
    constexpr uint32_t kPer = 16u / T::kBytes;                         // rows of a piece
    static_assert(NW * 32u * kPitch <= NBUF * kBuf + 2u * kSBuf, "the columns fit LDS");
    uint8_t *const mine = lds + wave * (32u * kPitch);
    const uint32_t c0_ = l / kLanes, piece_row = (l % kLanes) * kPer;
    const bool whole = a.n_rows % kPer == 0u && ((uintptr_t)a.y & 15u) == 0u;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const uint32_t j0 = (wn * NI + n) * 32u;
#pragma unroll
      for (int m = 0; m < MI; m += kStep)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4_t v;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = M == kGateUp ? swiglu(acc[m][n][4 * q + i], acc[m + kStep - 1][n][4 * q + i])
                                : acc[m][n][4 * q + i];
          uint8_t *p = mine + col32 * kPitch + ((m / kStep) * 32u + 8u * q + half4) * T::kBytes;
          if constexpr (T::kBytes == 4)
            *reinterpret_cast<f32x4_t *>(p) = v;
          else
            *reinterpret_cast<u32x2_t *>(p) =
                (u32x2_t){pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the wave's own writes
#pragma unroll 4
      for (uint32_t c = 0; c < 32u; c += kCols) {
        const uint32_t j = j0 + c + c0_, r = wrow0 + piece_row;
        const u32x4_t v =
            *reinterpret_cast<const u32x4_t *>(mine + (c + c0_) * kPitch + (l % kLanes) * 16u);
        if (j < t.count && r < a.n_rows) {
          uint8_t *to = a.y + ((uint64_t)slot_of(j) * a.n_rows + r) * T::kBytes;
          if (whole) {
            *reinterpret_cast<u32x4_t *>(to) = v;
          } else {
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i)
              if (r + i < a.n_rows) {
                if constexpr (T::kBytes == 4)
                  reinterpret_cast<uint32_t *>(to)[i] = v[i];
                else
                  reinterpret_cast<uint16_t *>(to)[i] = (uint16_t)(v[i / 2u] >> (16u * (i % 2u)));
              }
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // read before the next columns come
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

#define AXH_MX_TYPES(KERNEL, ...)  \
  KERNEL(f32, TF32, __VA_ARGS__)   \
  KERNEL(f16, TF16, __VA_ARGS__)   \
  KERNEL(bf16, TBF16, __VA_ARGS__)

// K-split kernels: NAME, rows, waves, buffers of a wave.
#define AXH_MX_KSPLIT_DENSE(TN, T, NAME, ROWS, NW, NB)           \
  extern "C" __global__ void __launch_bounds__(64 * NW)          \
      axh_mxfp4_matmul_##NAME##_##TN(AXH_MX_DENSE_ARGS) {        \
    extern __shared__ __align__(16) uint8_t ring[];              \
    AXH_MX_DENSE_UNPACK;                                         \
    ksplit_body<kDense, T, false, ROWS, NW, NB>(a, ring);        \
  }
#define AXH_MX_KSPLIT_EXPERT(TN, T, NAME, ROWS, NW, NB)          \
  extern "C" __global__ void __launch_bounds__(64 * NW)          \
      axh_mxfp4_expert_matmul_##NAME##_##TN(AXH_MX_EXPERT_ARGS) {\
    extern __shared__ __align__(16) uint8_t ring[];              \
    AXH_MX_EXPERT_UNPACK;                                        \
    ksplit_body<kGrouped, T, false, ROWS, NW, NB>(a, ring);      \
  }
#define AXH_MX_KSPLIT_GATE_UP(TN, T, NAME, PACKED, NW, NB)         \
  extern "C" __global__ void __launch_bounds__(64 * NW)            \
      axh_mxfp4_expert_gate_up_##NAME##_##TN(AXH_MX_EXPERT_ARGS) { \
    extern __shared__ __align__(16) uint8_t ring[];                \
    AXH_MX_EXPERT_UNPACK;                                          \
    ksplit_body<kGateUp, T, PACKED, 32, NW, NB>(a, ring);          \
  }
AXH_MX_TYPES(AXH_MX_KSPLIT_DENSE, k16, 16, 8, 3)
AXH_MX_TYPES(AXH_MX_KSPLIT_DENSE, k32, 32, 8, 2)
AXH_MX_TYPES(AXH_MX_KSPLIT_EXPERT, k32, 32, 8, 2)
AXH_MX_TYPES(AXH_MX_KSPLIT_GATE_UP, k32, false, 4, 3)
AXH_MX_KSPLIT_GATE_UP(mxfp4, TF32, k32, true, 4, 3)

// Tile kernels: NAME, rows and columns of the tile, waves along both and groups of
// them along K, buffers of a group, waves of a SIMD (and true: short rows).
#define AXH_MX_TILE_DENSE(TN, T, NAME, BM, BN, WM, WN, WK, NBUF, WPE, ...) \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN * WK)      \
      __attribute__((amdgpu_waves_per_eu(WPE, WPE)))              \
      axh_mxfp4_matmul_##NAME##_##TN(AXH_MX_DENSE_ARGS) {         \
    extern __shared__ __align__(16) uint8_t tile[];               \
    AXH_MX_DENSE_UNPACK;                                          \
    tile_body<kDense, T, false, BM, BN, WM, WN, WK, NBUF __VA_OPT__(,) __VA_ARGS__>(a, tile);   \
  }
#define AXH_MX_TILE_EXPERT(TN, T, NAME, BM, BN, WM, WN, WK, NBUF, WPE, ...) \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN * WK)       \
      __attribute__((amdgpu_waves_per_eu(WPE, WPE)))               \
      axh_mxfp4_expert_matmul_##NAME##_##TN(AXH_MX_EXPERT_ARGS) {  \
    extern __shared__ __align__(16) uint8_t tile[];                \
    AXH_MX_EXPERT_UNPACK;                                          \
    tile_body<kGrouped, T, false, BM, BN, WM, WN, WK, NBUF __VA_OPT__(,) __VA_ARGS__>(a, tile);  \
  }
#define AXH_MX_TILE_GATE_UP(TN, T, NAME, PACKED, BM, BN, WM, WN, WK, NBUF, WPE, ...) \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN * WK)                \
      __attribute__((amdgpu_waves_per_eu(WPE, WPE)))                        \
      axh_mxfp4_expert_gate_up_##NAME##_##TN(AXH_MX_EXPERT_ARGS) {          \
    extern __shared__ __align__(16) uint8_t tile[];                         \
    AXH_MX_EXPERT_UNPACK;                                                   \
    tile_body<kGateUp, T, PACKED, BM, BN, WM, WN, WK, NBUF __VA_OPT__(,) __VA_ARGS__>(a, tile);           \
  }
#define AXH_MX_TILE_EXPERTS(NAME, ...)                        \
  AXH_MX_TYPES(AXH_MX_TILE_EXPERT, NAME, __VA_ARGS__)         \
  AXH_MX_TYPES(AXH_MX_TILE_GATE_UP, NAME, false, __VA_ARGS__) \
  AXH_MX_TILE_GATE_UP(mxfp4, TF32, NAME, true, __VA_ARGS__)
AXH_MX_TYPES(AXH_MX_TILE_DENSE, t64x64, 64, 64, 1, 2, 1, 3, 1)
AXH_MX_TYPES(AXH_MX_TILE_DENSE, t64x64s2, 64, 64, 1, 2, 2, 3, 1)
AXH_MX_TYPES(AXH_MX_TILE_DENSE, t64x128, 64, 128, 1, 4, 1, 3, 2)
AXH_MX_TYPES(AXH_MX_TILE_DENSE, t128x128, 128, 128, 2, 2, 1, 2, 2)
AXH_MX_TYPES(AXH_MX_TILE_DENSE, t256x256, 256, 256, 2, 4, 1, 2, 2)
AXH_MX_TILE_EXPERTS(t128x64, 128, 64, 2, 2, 1, 3, 2)
AXH_MX_TILE_EXPERTS(t128x128, 128, 128, 2, 2, 1, 2, 2)
AXH_MX_TILE_EXPERTS(t256x256, 256, 256, 2, 4, 1, 2, 2)
AXH_MX_TYPES(AXH_MX_TILE_DENSE, t128x128n, 128, 128, 2, 2, 1, 2, 2, true)
AXH_MX_TILE_EXPERTS(t128x128n, 128, 128, 2, 2, 1, 2, 2, true)
