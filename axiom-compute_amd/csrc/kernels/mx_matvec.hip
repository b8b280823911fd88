// MXFP4 products for single tokens (gfx950): y = W x with f32 activations, and
// the two halves of an expert layer for few tokens.  Bound by the weights'
// bytes.
//
// The axis that is summed over is cut into units of LPR blocks of 32 columns
// (LPR = 64, or 32 or 16 where a row has no more blocks than that): a lane has
// one block of a unit, its 32 activations, once staged, stay in VGPRs for every
// row that the wave takes, so neither LDS traffic nor a cross-lane step stands
// between the weight loads and the multiplications.  A load instruction of a wave reads 64
// consecutive blocks (1 KiB of codes) of 64 / LPR rows.  The waves of a group
// have a unit each and the same rows; a group's partial sums meet in LDS, in
// the units' order.
//   128256 x 4096: 46.7 us, 6.0 TB/s.  4096 x 14336 (31 MB, 6.0 us at the rate of a
// copy): 8.5 us in a loop, of which a launch and the wait for the activations and the
// first codes are about 3 (activations straight to registers would save part of that: the
// one-pass Q4_K kernel takes 7.6 us for 5 % more bytes).  8 choices of 64 experts, 2048 x 1024: gate and up 6.9 us (3.4
// for the bytes), down 5.9 (1.7); two batches of loads a wave, so that what bounds
// them is the chain of launch, expert, codes and sum.
#include "mx_common.h"

using namespace axh;

namespace {

typedef __attribute__((address_space(3))) void lds_void_t;

enum Mode { kDense, kGateUp, kDown };

// Offset of lanes past a row's last block.  The row's offset is added to it: the
// host keeps the rows of a group below 1 GiB, so the sum is past every buffer's
// end and below 2^32, and such loads return zeros.
constexpr uint32_t kFar = 0x80000000u;
// Load instructions of a batch, of 64 / LPR rows each: fewer where a group's waves
// share out the choices of a token, so that there are more groups.
template <Mode M> constexpr int kLoadsOf = M == kDown ? 4 : 8;

__device__ __forceinline__ f32x2_t swap32_f(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a),
                                                  __builtin_bit_cast(uint32_t, b), false, false);
  const uint32_t lo = r[0], hi = r[1];
  return (f32x2_t){__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}
__device__ __forceinline__ f32x2_t swap16_f(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a),
                                                  __builtin_bit_cast(uint32_t, b), false, false);
  const uint32_t lo = r[0], hi = r[1];
  return (f32x2_t){__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}

// silu(g) * u on the library's exponential and an exact quotient, as the gate/up kernels of
// the other formats have it: within 3 ulp, and 0 from g = -88.72 on, where the exponential is
// beyond f32.  One a row, after the sums, so that it costs next to nothing (1 token, 8 of 64
// experts, 2048 x 1024: 6.80 us against 6.74 with swiglu of mx_common.h, which prompts take,
// as its fewer instructions count there).
__device__ __forceinline__ float silu_mul(float g, float u) {
  return g / (1.0f + expf(-g)) * u;
}

// The sum over the 16 lanes of a DPP row, in all of them.
__device__ __forceinline__ float row_sum16(float v) {
  v += dpp_f32<kXor1>(v);
  v += dpp_f32<kXor2>(v);
  v += dpp_f32<kHalfMirror>(v);
  v += dpp_f32<kMirror>(v);
  return v;
}

// dot of 32 codes with the lane's activations, unscaled.
__device__ __forceinline__ float dot32(u32x4_t c, const f32x4_t *x) {
  float a = 0.0f, b = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const f32x2_t p0 = fp4_pair<0>(c[w]), p1 = fp4_pair<1>(c[w]);
    const f32x2_t p2 = fp4_pair<2>(c[w]), p3 = fp4_pair<3>(c[w]);
    const f32x4_t x0 = x[2 * w], x1 = x[2 * w + 1];
    a = __builtin_fmaf(p0.x, x0[0], a);
    b = __builtin_fmaf(p0.y, x0[1], b);
    a = __builtin_fmaf(p1.x, x0[2], a);
    b = __builtin_fmaf(p1.y, x0[3], b);
    a = __builtin_fmaf(p2.x, x1[0], a);
    b = __builtin_fmaf(p2.y, x1[1], b);
    a = __builtin_fmaf(p3.x, x1[2], a);
    b = __builtin_fmaf(p3.y, x1[3], b);
  }
  return a + b;
}

struct Shape {
  uint32_t n_rows;  // output rows (gate/up: of each matrix)
  uint32_t nblk;    // blocks of a row
  uint32_t uw;      // waves of a group
  uint32_t batches; // batches of a group, even
  uint32_t top_k, n_experts;
};

// The rows of one matrix that a group reads, as a buffer that ends at the
// matrix's last row.
struct Rows {
  __amdgpu_buffer_rsrc_t codes, scales;
  __device__ __forceinline__ Rows(const uint8_t *c, const uint8_t *s, uint64_t row0,
                                  uint32_t count, uint32_t nblk)
      : codes(rsrc(c + row0 * nblk * 16u, count * nblk * 16u)),
        scales(rsrc(s + row0 * nblk, count * nblk)) {}
};

template <Mode M, int LPR>
__device__ __forceinline__ void
matvec_body(const uint8_t *wc, const uint8_t *ws, const uint8_t *wc2, const uint8_t *ws2,
            const float *x, const int32_t *experts, const float *weights, float *y, Shape a,
            uint8_t *lds_bytes) {
  constexpr int kR = kLoadsOf<M>;
  constexpr uint32_t kPer = 64u / LPR;                       // rows of a load instruction
  constexpr uint32_t kMats = M == kGateUp ? 2u : 1u;
  constexpr uint32_t kBatchRows = kR * kPer / kMats;         // rows of a batch, per matrix
  struct Batch { // codes and scales
    u32x4_t c[kR];
    uint32_t s[kR];
  };
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t group = wave / a.uw, u0 = wave - group * a.uw;
  const uint32_t groups = (blockDim.x >> 6) / a.uw;
  const uint32_t group_rows = a.batches * kBatchRows;
  const uint32_t row0 = (blockIdx.x * groups + group) * group_rows;
  const uint32_t bl = lane & (LPR - 1u), sub = lane / LPR;
  const uint32_t chunks = LPR == 64 ? (a.nblk + 63u) / 64u : 1u;
  const uint32_t units = M == kDown ? a.top_k * chunks : chunks;
  const uint32_t left = row0 < a.n_rows ? a.n_rows - row0 : 0u;
  const uint32_t count = left < group_rows ? left : group_rows;
  const uint64_t matrix = (uint64_t)a.n_rows * a.nblk; // blocks of one expert
  const uint32_t item = blockIdx.y;                    // gate/up: slot; down: token
  // LDS: a unit's activations per wave, then the partial sums
  uint8_t *const stage = lds_bytes + wave * (LPR * 128u);
  float *const lds = reinterpret_cast<float *>(lds_bytes + (blockDim.x >> 6) * (LPR * 128u));
  float *mine = lds + group * (group_rows * kMats * a.uw);

  uint32_t only = 0; // gate/up: the slot's expert
  if (M == kGateUp) only = (uint32_t)experts[item];
  const bool skip = M == kGateUp && only >= a.n_experts;

  for (uint32_t b = lane; b < group_rows * kMats; b += 64u) mine[b * a.uw + u0] = 0.0f;

  for (uint32_t u = u0; u < units && !skip && count; u += a.uw) {
    const uint32_t chunk = M == kDown ? u % chunks : u;
    uint32_t e = 0;
    float weight = 1.0f;
    const float *xu = x;
    if (M == kGateUp) {
      e = only;
      xu = x + (uint64_t)(item / a.top_k) * a.nblk * 32u;
    } else if (M == kDown) {
      const uint64_t slot = (uint64_t)item * a.top_k + u / chunks;
      e = (uint32_t)experts[slot];
      if (e >= a.n_experts) continue;
      weight = weights[slot];
      xu = x + slot * a.nblk * 32u;
    }
    const uint32_t blk = chunk * 64u + bl;
    const bool in = blk < a.nblk;
    const Rows m0(wc + e * matrix * 16u, ws + e * matrix, row0, count, a.nblk);
    const Rows m1 = M == kGateUp ? Rows(wc2 + e * matrix * 16u, ws2 + e * matrix, row0, count,
                                        a.nblk)
                                 : m0;
    const uint32_t cbase = in ? (sub * a.nblk + blk) * 16u : kFar;
    const uint32_t sbase = in ? sub * a.nblk + blk : kFar;
    const uint32_t step = kPer * a.nblk; // blocks between load instructions

    auto load = [&](uint32_t batch, Batch &t) {
#pragma unroll
      for (uint32_t i = 0; i < kR; ++i) {
        const uint32_t mi = i / (kR / kMats), k = i % (kR / kMats);
        const uint32_t at = (batch * (kR / kMats) + k) * step; // uniform
        t.c[i] = __builtin_amdgcn_raw_buffer_load_b128(mi ? m1.codes : m0.codes,
                                                       (int)(cbase + at * 16u), 0, 0);
        t.s[i] = __builtin_amdgcn_raw_buffer_load_b8(mi ? m1.scales : m0.scales,
                                                     (int)(sbase + at), 0, 0);
      }
    };
    auto finish = [&](uint32_t batch, const Batch &t, const f32x4_t *xr) {
      float v[kR];
#pragma unroll
      for (int i = 0; i < kR; ++i) v[i] = dot32(t.c[i], xr) * e8m0_to_f32(t.s[i]);
      // LDS row of load i's row `sub`: matrix, then row in the group
      auto put = [&](uint32_t i, float sum) {
        const uint32_t mi = i / (kR / kMats), k = i % (kR / kMats);
        const uint32_t r = mi * group_rows + batch * kBatchRows + k * kPer + sub;
        if ((lane & 15u) == 0u) {
          if (M == kDown)
            mine[r * a.uw + u0] += weight * sum;
          else
            mine[r * a.uw + u0] += sum;
        }
      };
      // Sums over the lanes of a row: exchanges of half the values between half
      // the lanes, then DPP steps inside 16 lanes.
      if constexpr (LPR == 64) {
        float h[kR / 2];
#pragma unroll
        for (int i = 0; i < kR / 2; ++i) {
          const f32x2_t p = swap32_f(v[i], v[i + kR / 2]);
          h[i] = p.x + p.y;
        }
#pragma unroll
        for (uint32_t i = 0; i < kR / 4; ++i) {
          const f32x2_t p = swap16_f(h[i], h[i + kR / 4]);
          put(i + (kR / 4) * ((lane >> 4) & 1u) + (kR / 2) * (lane >> 5), row_sum16(p.x + p.y));
        }
      } else if constexpr (LPR == 32) {
#pragma unroll
        for (uint32_t i = 0; i < kR / 2; ++i) {
          const f32x2_t p = swap16_f(v[i], v[i + kR / 2]);
          put(i + (kR / 2) * ((lane >> 4) & 1u), row_sum16(p.x + p.y));
        }
      } else {
#pragma unroll
        for (uint32_t i = 0; i < kR; ++i) put(i, row_sum16(v[i]));
      }
    };

    // The unit's activations, 128 bytes a lane, come through LDS in whole lines
    // (loaded by the lanes themselves, an instruction would touch 64 lines for 16
    // bytes of each); 16-byte piece p of block b at place p ^ (b / 2 % 8), so that
    // the reads of 64 blocks' pieces meet all the banks.
    const __amdgpu_buffer_rsrc_t xb = rsrc(xu, a.nblk * 128u);
#pragma unroll
    for (uint32_t i = 0; i < LPR / 8; ++i) {
      const uint32_t b = 8u * i + (lane >> 3), p = (lane & 7u) ^ ((b >> 1) & 7u);
      const uint32_t at = chunk * 64u + b;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xb, (lds_void_t *)(stage + i * 1024u), 16,
                                               (int)(at < a.nblk ? at * 128u + p * 16u : kFar), 0,
                                               0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    Batch t0, t1;
    load(0, t0);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kR) : "memory"); // all but the batch
    f32x4_t xr[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
      xr[i] = *reinterpret_cast<const f32x4_t *>(stage + bl * 128u + ((i ^ ((bl >> 1) & 7u)) * 16u));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // read before another unit's come
    // An even number of batches (those past the last row read zeros), so that the
    // loop has one way through and the compiler's waits count the loads on it.
    uint32_t b = 0;
    do {
      load(b + 1u, t1);
      finish(b, t0, xr);
      load(b + 2u, t0);
      finish(b + 1u, t1, xr);
      b += 2u;
    } while (b < a.batches);
  }
  __syncthreads();
  for (uint32_t r = threadIdx.x; r < groups * group_rows; r += blockDim.x) {
    const uint32_t g = r / group_rows, k = r - g * group_rows;
    const uint32_t row = (blockIdx.x * groups + g) * group_rows + k;
    if (row >= a.n_rows) continue;
    const float *p = lds + (g * group_rows * kMats + k) * a.uw;
    float sum = 0.0f;
    for (uint32_t u = 0; u < a.uw; ++u) sum += p[u];
    if (M == kGateUp) {
      const float *q = p + group_rows * a.uw;
      float up = 0.0f;
      for (uint32_t u = 0; u < a.uw; ++u) up += q[u];
      sum = silu_mul(sum, up);
    }
    y[(uint64_t)item * a.n_rows + row] = sum;
  }
}

} // namespace

#define AXH_MX_MATVEC(LPR)                                                                        \
  extern "C" __global__ void __launch_bounds__(512) axh_mxfp4_matvec_l##LPR(                     \
      const uint8_t *wc, const uint8_t *ws, const float *x, float *y, uint32_t n_rows,            \
      uint32_t nblk, uint32_t uw, uint32_t batches) {                                             \
    extern __shared__ __align__(16) uint8_t lds[];                                                \
    matvec_body<kDense, LPR>(wc, ws, nullptr, nullptr, x, nullptr, nullptr, y,                    \
                             Shape{n_rows, nblk, uw, batches, 1, 1}, lds);                        \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(512) axh_mxfp4_expert_gate_up_l##LPR(             \
      const uint8_t *gc, const uint8_t *gs, const uint8_t *uc, const uint8_t *us, const float *x, \
      const int32_t *experts, float *h, uint32_t n_rows, uint32_t nblk, uint32_t uw,              \
      uint32_t batches, uint32_t top_k, uint32_t n_experts) {                                     \
    extern __shared__ __align__(16) uint8_t lds[];                                                \
    matvec_body<kGateUp, LPR>(gc, gs, uc, us, x, experts, nullptr, h,                             \
                              Shape{n_rows, nblk, uw, batches, top_k, n_experts}, lds);           \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(512) axh_mxfp4_expert_down_l##LPR(                \
      const uint8_t *wc, const uint8_t *ws, const float *h, const int32_t *experts,               \
      const float *weights, float *y, uint32_t n_rows, uint32_t nblk, uint32_t uw,                \
      uint32_t batches, uint32_t top_k, uint32_t n_experts) {                                     \
    extern __shared__ __align__(16) uint8_t lds[];                                                \
    matvec_body<kDown, LPR>(wc, ws, nullptr, nullptr, h, experts, weights, y,                     \
                            Shape{n_rows, nblk, uw, batches, top_k, n_experts}, lds);             \
  }
AXH_MX_MATVEC(64)
AXH_MX_MATVEC(32)
AXH_MX_MATVEC(16)
