// MXFP4 quantisation, decoding and unpacking; routing of tokens to experts,
// the slots' order by expert, and the weighted sum of the experts' outputs
// (gfx950).  All of them are bound by memory or, for few tokens, by the
// latency of a launch.
#include "mx_common.h"

using namespace axh;

namespace {

// Eight consecutive elements as f32.
template <class T> __device__ __forceinline__ void load8(const uint8_t *p, float *v);
template <> __device__ __forceinline__ void load8<TF32>(const uint8_t *p, float *v) {
  const f32x4_t a = reinterpret_cast<const f32x4_t *>(p)[0];
  const f32x4_t b = reinterpret_cast<const f32x4_t *>(p)[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = a[i];
    v[4 + i] = b[i];
  }
}
template <class T> __device__ __forceinline__ void load8h(const uint8_t *p, float *v) {
  const u32x4_t w = *reinterpret_cast<const u32x4_t *>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
}
template <> __device__ __forceinline__ void load8<TF16>(const uint8_t *p, float *v) {
  load8h<TF16>(p, v);
}
template <> __device__ __forceinline__ void load8<TBF16>(const uint8_t *p, float *v) {
  load8h<TBF16>(p, v);
}

template <class T> __device__ __forceinline__ void store8(uint8_t *p, const float *v);
template <> __device__ __forceinline__ void store8<TF32>(uint8_t *p, const float *v) {
  reinterpret_cast<f32x4_t *>(p)[0] = (f32x4_t){v[0], v[1], v[2], v[3]};
  reinterpret_cast<f32x4_t *>(p)[1] = (f32x4_t){v[4], v[5], v[6], v[7]};
}
template <class T> __device__ __forceinline__ void store8h(uint8_t *p, const float *v) {
  *reinterpret_cast<u32x4_t *>(p) = (u32x4_t){pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                              pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
}
template <> __device__ __forceinline__ void store8<TF16>(uint8_t *p, const float *v) {
  store8h<TF16>(p, v);
}
template <> __device__ __forceinline__ void store8<TBF16>(uint8_t *p, const float *v) {
  store8h<TBF16>(p, v);
}

// ---------------------------------------------------------------------------
// Quantisation.  Four lanes share a block of 32 elements, eight each (one or
// two 16-byte loads): the block's largest magnitude is a maximum over bit
// patterns (magnitudes order like integers, NaN above infinity), two DPP steps
// inside the quad.  The converting instruction divides by the block's power of two,
// which is exact, so each element is rounded once; f16 and bf16 go through it as they
// are, as the instructions, not the bytes, would else bound the kernel.  8192 x 4096 bf16: 15.3 us (20.3 through f32
// and with a division a block), 5.5 TB/s.
// ---------------------------------------------------------------------------
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

template <class T> struct Eight { // elements of 16 bits
  u32x4_t w;
  __device__ __forceinline__ void load(const uint8_t *p) {
    w = *reinterpret_cast<const u32x4_t *>(p);
  }
  // the quad's largest magnitude, as the bits of an f32
  __device__ __forceinline__ uint32_t quad_max() const {
    u16x2_t m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w[i] & 0x7FFF7FFFu));
    uint32_t b = __builtin_bit_cast(uint32_t, m);
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, dpp_u32<kXor1>(b)));
    b = __builtin_bit_cast(uint32_t, m);
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, dpp_u32<kXor2>(b)));
    const uint16_t both = m.x > m.y ? m.x : m.y;
    float lo, hi;
    unpack2<T>(both, lo, hi);
    return __builtin_bit_cast(uint32_t, lo);
  }
  __device__ __forceinline__ uint32_t codes(uint32_t e) const {
    const float scale = mx_divisor(e);
    uint32_t c = 0;
    if constexpr (__is_same(T, TF16)) {
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, pair<half2_t>(0), scale, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, pair<half2_t>(1), scale, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, pair<half2_t>(2), scale, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, pair<half2_t>(3), scale, 3);
    } else {
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair<bf16x2_t>(0), scale, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair<bf16x2_t>(1), scale, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair<bf16x2_t>(2), scale, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair<bf16x2_t>(3), scale, 3);
    }
    return c;
  }
  template <class V> __device__ __forceinline__ V pair(int i) const {
    const uint32_t v = w[i];
    return __builtin_bit_cast(V, v);
  }
};
template <> struct Eight<TF32> {
  float v[8];
  __device__ __forceinline__ void load(const uint8_t *p) { load8<TF32>(p, v); }
  __device__ __forceinline__ uint32_t quad_max() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu;
      m = b > m ? b : m;
    }
    uint32_t o = dpp_u32<kXor1>(m);
    m = o > m ? o : m;
    o = dpp_u32<kXor2>(m);
    return o > m ? o : m;
  }
  __device__ __forceinline__ uint32_t codes(uint32_t e) const {
    return fp4_pack8(v, mx_divisor(e));
  }
};

// row_blocks 0: the rows follow one another.  A workgroup takes `per` (1 or 4) times
// 64 blocks.
template <class T>
__device__ __forceinline__ void quantize_body(const uint8_t *x, uint8_t *codes, uint8_t *scales,
                                              uint32_t n_blocks, uint32_t row_blocks,
                                              uint32_t stride_lo, uint32_t stride_hi,
                                              uint32_t per) {
  const uint32_t part = threadIdx.x & 3u;
  const uint32_t blk0 = blockIdx.x * per * 64u + (threadIdx.x >> 2);
  const uint64_t stride = (uint64_t)stride_hi << 32 | stride_lo; // elements
  auto address = [&](uint32_t blk) {
    uint64_t at = blk * 32ull;
    if (row_blocks) {
      const uint32_t row = blk / row_blocks;
      at = row * stride + (uint64_t)(blk - row * row_blocks) * 32u;
    }
    return x + (at + part * 8u) * T::kBytes;
  };
  auto finish = [&](uint32_t blk, const Eight<T> &v) {
    const uint32_t e = mx_scale_byte(v.quad_max());
    const uint32_t c = e == 255u ? 0u : v.codes(e);
    reinterpret_cast<uint32_t *>(codes)[(uint64_t)blk * 4u + part] = c;
    if (part == 0u) scales[blk] = (uint8_t)e;
  };
  if (per == 1u) {
    if (blk0 >= n_blocks) return; // whole quads
    Eight<T> v;
    v.load(address(blk0));
    finish(blk0, v);
  } else {
    Eight<T> v[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t blk = blk0 + 64u * k;
      v[k].load(address(blk < n_blocks ? blk : n_blocks - 1u));
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (blk0 + 64u * k < n_blocks) finish(blk0 + 64u * k, v[k]);
  }
}

// ---------------------------------------------------------------------------
// Decoding: eight codes (one dword) a lane, 32 bytes (16) of f32 (f16, bf16) out: bound
// by the stores.  8192 x 4096 to bf16: 13.3 us, 6.4 TB/s.
// ---------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ void dequant_body(const uint8_t *codes, const uint8_t *scales,
                                             uint8_t *w, uint32_t n_blocks) {
  const uint32_t t = blockIdx.x * 256u + threadIdx.x;
  const uint32_t blk = t >> 2;
  if (blk >= n_blocks) return;
  const uint32_t c = reinterpret_cast<const uint32_t *>(codes)[t];
  const float s = e8m0_to_f32(scales[blk]);
  float v[8];
  const f32x2_t p0 = fp4_pair<0>(c), p1 = fp4_pair<1>(c), p2 = fp4_pair<2>(c), p3 = fp4_pair<3>(c);
  v[0] = p0.x * s;
  v[1] = p0.y * s;
  v[2] = p1.x * s;
  v[3] = p1.y * s;
  v[4] = p2.x * s;
  v[5] = p2.y * s;
  v[6] = p3.x * s;
  v[7] = p3.y * s;
  store8<T>(w + (uint64_t)t * 8u * T::kBytes, v);
}

} // namespace

#define AXH_MX_ELEM(NAME, T)                                                                      \
  extern "C" __global__ void __launch_bounds__(256) axh_mxfp4_quantize_##NAME(                    \
      const uint8_t *x, uint8_t *codes, uint8_t *scales, uint32_t n_blocks, uint32_t row_blocks,  \
      uint32_t stride_lo, uint32_t stride_hi, uint32_t per) {                                     \
    quantize_body<T>(x, codes, scales, n_blocks, row_blocks, stride_lo, stride_hi, per);          \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) axh_mxfp4_dequant_##NAME(                     \
      const uint8_t *codes, const uint8_t *scales, uint8_t *w, uint32_t n_blocks) {               \
    dequant_body<T>(codes, scales, w, n_blocks);                                                  \
  }
AXH_MX_ELEM(f32, TF32)
AXH_MX_ELEM(f16, TF16)
AXH_MX_ELEM(bf16, TBF16)

// ggml's MXFP4 blocks (17 bytes: the scale byte, then 16 bytes whose low
// nibbles are elements 0..15 and whose high nibbles are elements 16..31) as
// codes and scales.  One lane per output dword (elements 8p .. 8p + 7 of a
// block): the same nibble of eight consecutive bytes.  14336 x 4096: 16.7 us, 3.7 TB/s, once a
// tensor when a model is loaded.
extern "C" __global__ void __launch_bounds__(256) axh_mxfp4_unpack_ggml(const uint8_t *q,
                                                                       uint8_t *codes,
                                                                       uint8_t *scales,
                                                                       uint32_t n_blocks) {
  const uint32_t t = blockIdx.x * 256u + threadIdx.x;
  const uint32_t blk = t >> 2, part = t & 3u;
  if (blk >= n_blocks) return;
  const uint8_t *b = q + (uint64_t)blk * 17u;
  const uint32_t shift = (part >> 1) * 4u;
  uint32_t c = 0;
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) c |= ((b[1u + (part & 1u) * 8u + i] >> shift) & 15u) << (4u * i);
  reinterpret_cast<uint32_t *>(codes)[t] = c;
  if (part == 0u) scales[blk] = b[0];
}

// ---------------------------------------------------------------------------
// Routing.  One wave per token; lane l holds experts l, l + 64, ... (NPL of
// them).  Keys are order-preserving unsigned integers, 0 for experts that
// cannot be chosen, so a round of the top-k is a maximum over the wave (DPP),
// and the lowest expert among equals is the first set bit of the first
// non-empty ballot.
//   Bound by latency for few tokens (1.7 us for one of 32 experts), by the vector
// instructions for many: 4096 x 256 experts, 8 chosen from 4 of 8 groups, 7.1 us a call back
// to back (7.5 in a kernel trace), about 650 of them a token (its bytes would take 0.9).
// ---------------------------------------------------------------------------
namespace {

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  uint32_t o = dpp_u32<kXor1>(v);
  v = o > v ? o : v;
  o = dpp_u32<kXor2>(v);
  v = o > v ? o : v;
  o = dpp_u32<kHalfMirror>(v);
  v = o > v ? o : v;
  o = dpp_u32<kMirror>(v);
  v = o > v ? o : v;
  const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 0);
  const uint32_t b = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 32);
  const uint32_t d = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
  const uint32_t ab = a > b ? a : b, cd = c > d ? c : d;
  return ab > cd ? ab : cd;
}

__device__ __forceinline__ float wave_sum_f32(float v) {
  v += dpp_f32<kXor1>(v);
  v += dpp_f32<kXor2>(v);
  v += dpp_f32<kHalfMirror>(v);
  v += dpp_f32<kMirror>(v);
  const int i = __builtin_bit_cast(int, v);
  const float a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 0));
  const float b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 16));
  const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 32));
  const float d = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 48));
  return (a + b) + (c + d);
}

// f32 -> unsigned with the same order; -0 counts as +0, NaN as -inf.
__device__ __forceinline__ uint32_t order_of(float f) {
  if (f != f) f = -__builtin_inff();
  const uint32_t b = __builtin_bit_cast(uint32_t, f + 0.0f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __builtin_bit_cast(float, (o >> 31) ? o & 0x7FFFFFFFu : ~o);
}
constexpr uint32_t kOrderMinusInf = 0x007FFFFFu; // order_of(-inf)

enum : uint32_t { kSigmoid = 1u, kNormalize = 2u, kKeyIsLogit = 4u };

// Logit i of a token, whatever their type.
template <class T> __device__ __forceinline__ float logit_at(const uint8_t *row, uint32_t i);
template <> __device__ __forceinline__ float logit_at<TF32>(const uint8_t *row, uint32_t i) {
  return reinterpret_cast<const float *>(row)[i];
}
template <> __device__ __forceinline__ float logit_at<TF16>(const uint8_t *row, uint32_t i) {
  return (float)reinterpret_cast<const _Float16 *>(row)[i];
}
template <> __device__ __forceinline__ float logit_at<TBF16>(const uint8_t *row, uint32_t i) {
  return __builtin_bit_cast(float, (uint32_t)reinterpret_cast<const uint16_t *>(row)[i] << 16);
}

template <class T, int NPL>
__device__ __forceinline__ void route_body(const uint8_t *logits, const float *bias,
                                           int32_t *experts, float *weights, uint32_t n_tokens,
                                           uint32_t n_experts, uint32_t top_k, uint32_t flags,
                                           uint32_t n_groups, uint32_t groups_kept,
                                           uint32_t group_best, float scale, uint32_t *lds) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t token = blockIdx.x * 4u + wave;
  const bool real = token < n_tokens;
  const uint8_t *row = logits + (uint64_t)(real ? token : 0u) * n_experts * T::kBytes;
  const float kInf = __builtin_inff();

  float l[NPL]; // logits, -inf where masked, NaN or past the end
  float most = -kInf;
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const uint32_t e = 64u * j + lane;
    const float v = e < n_experts ? logit_at<T>(row, e) : -kInf;
    l[j] = v == v ? v : -kInf;
    most = l[j] > most ? l[j] : most;
  }
  float s[NPL]; // scores; masked experts score 0
  if (flags & kSigmoid) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) s[j] = 1.0f / (1.0f + expf(-l[j]));
  } else {
    most = value_of(wave_max_u32(order_of(most)));
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) { // +inf logits share all the weight
      s[j] = l[j] == -kInf ? 0.0f : l[j] == most ? 1.0f : expf(l[j] - most);
      sum += s[j];
    }
    sum = wave_sum_f32(sum);
#pragma unroll
    for (int j = 0; j < NPL; ++j) s[j] = sum > 0.0f ? s[j] / sum : 0.0f;
  }
  uint32_t key[NPL];
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const uint32_t e = 64u * j + lane;
    float k = (flags & kKeyIsLogit) ? l[j] : s[j];
    if (bias) k += e < n_experts ? bias[e] : 0.0f;
    const uint32_t o = order_of(k);
    key[j] = l[j] == -kInf || o <= kOrderMinusInf ? 0u : o;
  }

  if (n_groups > 1u) {
    // Every lane looks at its part of one group: 64 / G lanes (a power of two)
    // per group, then the two best of the lanes of a group are merged.
    uint32_t *mine = lds + wave * (64u * NPL);
#pragma unroll
    for (int j = 0; j < NPL; ++j) mine[64u * j + lane] = key[j];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the wave's own
    const uint32_t per = n_experts / n_groups;
    uint32_t log_lanes = 0;
    while ((n_groups << (log_lanes + 1u)) <= 64u) ++log_lanes;
    const uint32_t lanes = 1u << log_lanes, g = lane >> log_lanes, part = lane & (lanes - 1u);
    uint32_t a = 0, b = 0; // best and second best
    if (g < n_groups)
      for (uint32_t i = part; i < per; i += lanes) {
        const uint32_t k = mine[g * per + i];
        b = k > a ? a : k > b ? k : b;
        a = k > a ? k : a;
      }
    for (uint32_t m = 1; m < lanes; m <<= 1) {
      const uint32_t oa = (uint32_t)__shfl_xor((int)a, (int)m);
      const uint32_t ob = (uint32_t)__shfl_xor((int)b, (int)m);
      const uint32_t lo = a < oa ? a : oa;
      a = a < oa ? oa : a;
      b = b < ob ? ob : b;
      b = b < lo ? lo : b;
    }
    uint32_t gk = a;
    if (group_best == 2u)
      gk = order_of((a ? value_of(a) : -kInf) + (b ? value_of(b) : -kInf));
    // lane g: group g's key, and its rank: greater ones and equal ones before it
    const uint32_t at0 = (uint32_t)__shfl((int)gk, (int)(lane << log_lanes & 63u));
    const uint32_t own = lane < n_groups ? at0 : 0u;
    uint32_t rank = 0;
    for (uint32_t i = 0; i < n_groups; ++i) {
      const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)own, (int)i);
      rank += k > own || (k == own && i < lane) ? 1u : 0u;
    }
    const uint64_t kept = __ballot(lane < n_groups && rank < groups_kept);
    // e / per by a product, exact for e and per up to 1024
    const uint32_t inverse = (1u << 20) / per + 1u;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const uint32_t e = 64u * j + lane;
      if (e < n_experts && !((kept >> (e * inverse >> 20)) & 1u)) key[j] = 0u;
    }
  }

  int32_t picked = -1; // lane i holds choice i of up to 64
  float weight = 0.0f;
  for (uint32_t i = 0; i < top_k; ++i) {
    uint32_t best = 0;
#pragma unroll
    for (int j = 0; j < NPL; ++j) best = key[j] > best ? key[j] : best;
    best = wave_max_u32(best);
    if (best == 0u) break; // nothing left: -1 and weight 0
    bool found = false;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const uint64_t at = __ballot(key[j] == best);
      if (!found && at) {
        found = true;
        const int who = __builtin_ctzll(at);
        const float w = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s[j]), who));
        if (lane == i) {
          picked = 64 * j + who;
          weight = w;
        }
        if (lane == (uint32_t)who) key[j] = 0u;
      }
    }
  }
  if (flags & kNormalize) {
    const float sum = wave_sum_f32(weight);
    weight = sum > 0.0f ? weight / sum : 0.0f;
  }
  if (real && lane < top_k) {
    experts[(uint64_t)token * top_k + lane] = picked;
    weights[(uint64_t)token * top_k + lane] = weight * scale;
  }
}

} // namespace

#define AXH_ROUTE(NAME, T, NPL)                                                                   \
  extern "C" __global__ void __launch_bounds__(256) axh_expert_route_##NAME##_n##NPL(             \
      const uint8_t *logits, const float *bias, int32_t *experts, float *weights,                 \
      uint32_t n_tokens, uint32_t n_experts, uint32_t top_k, uint32_t flags, uint32_t n_groups,   \
      uint32_t groups_kept, uint32_t group_best, uint32_t scale) {                                \
    __shared__ uint32_t lds[4 * 64 * NPL];                                                 \
    route_body<T, NPL>(logits, bias, experts, weights, n_tokens, n_experts, top_k, flags,         \
                       n_groups, groups_kept, group_best, __builtin_bit_cast(float, scale), lds); \
  }
#define AXH_ROUTE_N(NPL)   \
  AXH_ROUTE(f32, TF32, NPL) \
  AXH_ROUTE(f16, TF16, NPL) \
  AXH_ROUTE(bf16, TBF16, NPL)
AXH_ROUTE_N(1)
AXH_ROUTE_N(2)
AXH_ROUTE_N(4)
AXH_ROUTE_N(8)
AXH_ROUTE_N(16)

// ---------------------------------------------------------------------------
// Router logits: logits[t][e] = sum over k of W[e][k] * x[t][k], f32 x, W of f32, f16 or
// bf16 (exact in f32), products and sums in f32, so that the choice of the experts does
// not depend on a quantisation.
//   Few logits: a wave each, eight elements a lane and step, four steps requested at once.
// 256 x 7168, one token, 3.9 us in a loop of calls (a launch).
//   More: v_mfma_f32_16x16x4_f32 over tiles of 16, 32 or 64 tokens by as many experts, K
// shared among the waves in chunks of 32 elements and joined through LDS in the waves'
// order.  A wave brings its chunk to LDS of its own by whole 128-byte lines, as f32, and
// has no one to wait for; the next chunk is on its way during the products.  (Fragments
// loaded straight from memory, a line for each lane, were bound by the cache's lookups: 256
// x 4096, 4096 tokens, 108 us.)  An instruction's k indexes are elements 8 g + j of the
// chunk, g the lane's quarter, in both operands.  Tiles of the same tokens run on one XCD.
//   Bound by the matrix units: 4096 tokens, 256 x 4096 80 us, 256 x 7168 136 us, 107 and
// 111 TFLOP/s.  For fewer tokens, the 16 waves of few workgroups: 100 tokens 9.3 and 14.7.
// ---------------------------------------------------------------------------
namespace {

template <class T>
__device__ __forceinline__ void logits_row_body(const float *x, const uint8_t *w, float *logits,
                                                uint32_t n_tokens, uint32_t n_experts,
                                                uint32_t cols) {
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t e = blockIdx.x * 4u + (threadIdx.x >> 6), t = blockIdx.y;
  if (e >= n_experts || t >= n_tokens) return;
  const uint8_t *xr = reinterpret_cast<const uint8_t *>(x + (uint64_t)t * cols);
  const uint8_t *wr = w + (uint64_t)e * cols * T::kBytes;
  const uint32_t pieces = cols / 8u;
  float acc[4] = {};
  uint32_t p = 0;
  for (; p + 256u <= pieces; p += 256u) {
    float a[4][8], b[4][8];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      load8<T>(wr + (uint64_t)(p + 64u * i + lane) * 8u * T::kBytes, a[i]);
      load8<TF32>(xr + (uint64_t)(p + 64u * i + lane) * 32u, b[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i] = __builtin_fmaf(a[i][j], b[i][j], acc[i]);
  }
  for (p += lane; p < pieces; p += 64u) {
    float a[8], b[8];
    load8<T>(wr + (uint64_t)p * 8u * T::kBytes, a);
    load8<TF32>(xr + (uint64_t)p * 32u, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j & 3] = __builtin_fmaf(a[j], b[j], acc[j & 3]);
  }
  const float sum = wave_sum_f32((acc[0] + acc[1]) + (acc[2] + acc[3]));
  if (lane == 0u) logits[(uint64_t)t * n_experts + e] = sum;
}

// A chunk of a wave's kRows rows, 32 elements of each, on its way to LDS: 16-byte loads of
// consecutive lanes along a row.
template <class T, int kRows> struct Chunk {
  static constexpr uint32_t kPer = 16u / T::kBytes;  // elements of a load
  static constexpr uint32_t kAcross = 32u / kPer, kStep = 64u / kAcross; // loads a row, rows a step
  u32x4_t v[kRows / kStep];
  __device__ __forceinline__ void load(const uint8_t *base, uint32_t first, uint32_t n,
                                       uint32_t cols, uint32_t k, uint32_t lane) {
#pragma unroll
    for (uint32_t i = 0; i < kRows / kStep; ++i) {
      // rows past the last are the last one's: their outputs are not stored
      const uint32_t r = first + kStep * i + lane / kAcross;
      v[i] = *reinterpret_cast<const u32x4_t *>(
          base + ((uint64_t)(r < n ? r : n - 1u) * cols + k + lane % kAcross * kPer) * T::kBytes);
    }
  }
  // As f32 rows of 128 bytes; 16-byte piece q of row r is at q ^ (r / 2 % 8), so that the
  // sixteen rows of a read meet all banks.
  __device__ __forceinline__ void store(float *lds, uint32_t lane) const {
#pragma unroll
    for (uint32_t i = 0; i < kRows / kStep; ++i) {
      const uint32_t r = kStep * i + lane / kAcross, q = lane % kAcross, x = r >> 1 & 7u;
      f32x4_t *row = reinterpret_cast<f32x4_t *>(lds + r * 32u);
      if constexpr (T::kBytes == 4u) {
        row[q ^ x] = __builtin_bit_cast(f32x4_t, v[i]);
      } else {
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack2<T>(v[i][j], f[2 * j], f[2 * j + 1]);
        row[(2u * q) ^ x] = (f32x4_t){f[0], f[1], f[2], f[3]};
        row[(2u * q + 1u) ^ x] = (f32x4_t){f[4], f[5], f[6], f[7]};
      }
    }
  }
};

template <class T, int kT, int kWaves>
__device__ __forceinline__ void logits_tile_body(const float *x, const uint8_t *w, float *logits,
                                                 uint32_t n_tokens, uint32_t n_experts,
                                                 uint32_t cols, uint32_t tiles, float *lds) {
  constexpr uint32_t kSide = 16u * kT, kOuts = kSide * kSide, kMine = 64u * kSide;
  static_assert(kOuts <= kMine, "a wave's outputs take the place of its chunks");
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t tile = (blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (tile >= tiles) return; // the whole workgroup
  const uint32_t across = (n_experts + kSide - 1u) / kSide;
  const uint32_t t0 = tile / across * kSide, e0 = tile % across * kSide;
  const uint32_t r = lane & 15u, quarter = lane >> 4, swizzle = r >> 1;
  float *mine = lds + wave * kMine;
  const uint8_t *xb = reinterpret_cast<const uint8_t *>(x);
  f32x4_t acc[kT][kT] = {};
  const uint32_t chunks = cols / 32u;
  if (wave < chunks) {
    Chunk<TF32, kSide> a;
    Chunk<T, kSide> b;
    a.load(xb, t0, n_tokens, cols, wave * 32u, lane);
    b.load(w, e0, n_experts, cols, wave * 32u, lane);
    for (uint32_t c = wave; c < chunks; c += kWaves) {
      a.store(mine, lane);
      b.store(mine + kSide * 32u, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the wave's own
      const uint32_t next = c + kWaves < chunks ? c + kWaves : c;
      a.load(xb, t0, n_tokens, cols, next * 32u, lane);
      b.load(w, e0, n_experts, cols, next * 32u, lane);
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        f32x4_t fa[kT], fb[kT];
        const uint32_t at = ((2u * quarter + h) ^ swizzle) * 4u;
#pragma unroll
        for (int i = 0; i < kT; ++i) {
          fa[i] = *reinterpret_cast<const f32x4_t *>(mine + (16u * i + r) * 32u + at);
          fb[i] = *reinterpret_cast<const f32x4_t *>(mine + (kSide + 16u * i + r) * 32u + at);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int m = 0; m < kT; ++m)
#pragma unroll
            for (int n = 0; n < kT; ++n)
              acc[m][n] =
                  __builtin_amdgcn_mfma_f32_16x16x4f32(fa[m][j], fb[n][j], acc[m][n], 0, 0, 0);
      }
      asm volatile("" ::: "memory"); // the reads stay before the next chunk's stores
    }
  }
  // output v of a lane: token 4 * quarter + v, expert r of its 16 x 16
#pragma unroll
  for (int m = 0; m < kT; ++m)
#pragma unroll
    for (int n = 0; n < kT; ++n)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        mine[((m * kT + n) * 4 + v) * 64u + lane] = acc[m][n][v];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < kOuts; i += 64u * kWaves) {
    float sum = lds[i];
#pragma unroll
    for (uint32_t k = 1; k < kWaves; ++k) sum += lds[k * kMine + i];
    const uint32_t v = i >> 6 & 3u, mn = i >> 8; // lane is i & 63 here too
    const uint32_t t = t0 + mn / kT * 16u + quarter * 4u + v;
    const uint32_t e = e0 + mn % kT * 16u + r;
    if (t < n_tokens && e < n_experts) logits[(uint64_t)t * n_experts + e] = sum;
  }
}

} // namespace

#define AXH_LOGITS_TILE(NAME, T, SIDE, WAVES)                                                     \
  extern "C" __global__ void __launch_bounds__(64 * WAVES) axh_expert_logits_t##SIDE##_##NAME(    \
      const float *x, const uint8_t *w, float *logits, uint32_t n_tokens, uint32_t n_experts,     \
      uint32_t cols, uint32_t tiles) {                                                            \
    extern __shared__ float sums[];                                                               \
    logits_tile_body<T, SIDE / 16, WAVES>(x, w, logits, n_tokens, n_experts, cols, tiles, sums);  \
  }
#define AXH_LOGITS(NAME, T)                                                                       \
  extern "C" __global__ void __launch_bounds__(256) axh_expert_logits_row_##NAME(                 \
      const float *x, const uint8_t *w, float *logits, uint32_t n_tokens, uint32_t n_experts,     \
      uint32_t cols) {                                                                            \
    logits_row_body<T>(x, w, logits, n_tokens, n_experts, cols);                                  \
  }                                                                                               \
  AXH_LOGITS_TILE(NAME, T, 16, 16)                                                                \
  AXH_LOGITS_TILE(NAME, T, 32, 16)                                                                \
  AXH_LOGITS_TILE(NAME, T, 64, 8)
AXH_LOGITS(f32, TF32)
AXH_LOGITS(f16, TF16)
AXH_LOGITS(bf16, TBF16)

// ---------------------------------------------------------------------------
// The order of slots by expert: a stable counting sort.  Slot i is choice
// i % top_k of token i / top_k.  A workgroup gives a contiguous chunk of the
// slots their places, a wave of it a contiguous part of the chunk; it counts the
// experts of the slots before its chunk, of each wave's part and after the chunk,
// so that no workgroup waits for another.  Within 64 slots, the lanes with the
// same expert are found by one ballot per bit of the expert's index: these are
// the most of the work, which is why the slots are shared out to workgroups.
// plan: offsets[n_experts + 1], padded to 16 words, then the slots.
//   3.9 us for 2000 slots of 40 experts, 7.0 us for 16384 of 32 (12.9 in one workgroup
// with a load at a time).
// ---------------------------------------------------------------------------
extern "C" __global__ void __launch_bounds__(1024) axh_expert_plan(const int32_t *experts,
                                                                  uint32_t *plan,
                                                                  uint32_t n_slots,
                                                                  uint32_t n_experts,
                                                                  uint32_t id_bits,
                                                                  uint32_t part_bits) {
  // [16 waves, then slots before the chunk, then after it][n_experts]: counts, then
  // the waves' places; [16] sums
  extern __shared__ uint32_t lds[];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  uint32_t *sums = lds + 18u * n_experts;
  for (uint32_t i = tid; i < 18u * n_experts; i += 1024u) lds[i] = 0u;
  __syncthreads();
  const uint32_t part = 1u << part_bits, chunk = 16u * part, from = blockIdx.x * chunk;
  for (uint32_t i0 = tid; i0 < n_slots; i0 += 8192u) {
    uint32_t e[8]; // all requested before the first is waited for
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
      const uint32_t i = i0 + 1024u * k;
      e[k] = (uint32_t)experts[i < n_slots ? i : n_slots - 1u];
    }
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
      const uint32_t i = i0 + 1024u * k;
      const uint32_t row = i < from ? 16u : i - from < chunk ? i - from >> part_bits : 17u;
      if (i < n_slots && e[k] < n_experts) atomicAdd(&lds[row * n_experts + e[k]], 1u);
    }
  }
  __syncthreads();
  // thread e: the expert's counts, and their total
  uint32_t counts[18], total = 0;
  if (tid < n_experts) {
#pragma unroll
    for (uint32_t w = 0; w < 18u; ++w) counts[w] = lds[w * n_experts + tid];
#pragma unroll
    for (uint32_t w = 0; w < 18u; ++w) total += counts[w];
  }
  uint32_t incl = total; // inclusive prefix over the experts of this wave
#pragma unroll
  for (uint32_t d = 1; d < 64u; d <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 63u) sums[wave] = incl;
  __syncthreads();
  uint32_t first = incl - total;
#pragma unroll
  for (uint32_t w = 0; w < 16u; ++w) first += w < wave ? sums[w] : 0u;
  if (tid < n_experts) {
    if (blockIdx.x == 0) {
      plan[tid] = first;
      if (tid == n_experts - 1u) plan[n_experts] = first + total;
    }
    first += counts[16];
#pragma unroll
    for (uint32_t w = 0; w < 16u; ++w) {
      lds[w * n_experts + tid] = first;
      first += counts[w];
    }
  }
  __syncthreads();
  uint32_t *order = plan + ((n_experts + 1u + 15u) & ~15u);
  uint32_t i0 = from + wave * part;
  const uint32_t to = i0 + part < n_slots ? i0 + part : n_slots;
  for (; i0 < to; i0 += 128u) { // (a part is 128 or more)
    uint32_t e[2], lo[2], hi[2]; // lo, hi: the lanes with the same expert
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
      const uint32_t i = i0 + 64u * k + lane;
      e[k] = i < to ? (uint32_t)experts[i] : n_experts;
      const uint64_t in = __ballot(e[k] < n_experts);
      lo[k] = (uint32_t)in;
      hi[k] = (uint32_t)(in >> 32);
    }
    for (uint32_t b = 0; b < id_bits; ++b)
#pragma unroll
      for (uint32_t k = 0; k < 2; ++k) {
        const uint32_t mask = 0u - (e[k] >> b & 1u);
        const uint64_t set = __ballot(mask != 0u);
        lo[k] &= ~((uint32_t)set ^ mask);
        hi[k] &= ~((uint32_t)(set >> 32) ^ mask);
      }
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k)
      if (e[k] < n_experts) {
        const uint32_t before = __builtin_amdgcn_mbcnt_hi(hi[k], __builtin_amdgcn_mbcnt_lo(lo[k], 0u));
        const uint32_t at = lds[wave * n_experts + e[k]] + before;
        if (at < n_slots) order[at] = i0 + 64u * k + lane; // (not less only if experts change meanwhile)
        // the last of the lanes moves the place on; the wave's LDS operations are in order
        if (before + 1u == (uint32_t)(__builtin_popcount(lo[k]) + __builtin_popcount(hi[k])))
          lds[wave * n_experts + e[k]] = at + 1u;
      }
  }
}

// ---------------------------------------------------------------------------
// y[t] = sum over a token's choices of weight * slot output, in f32, rounded
// once.  Choices outside 0 .. n_experts - 1 (the router's -1 among them) are left
// out: their slots hold nothing.  Eight columns a lane where n_cols is a multiple of
// eight and the rows are 16-byte aligned, else one.  Bound by memory: 4096 tokens of 4
// choices, 2048 columns, bf16, 13.3 us, 6.3 TB/s.
// ---------------------------------------------------------------------------
namespace {

template <class T> __device__ __forceinline__ void store1(uint8_t *p, float v);
template <> __device__ __forceinline__ void store1<TF32>(uint8_t *p, float v) {
  *reinterpret_cast<float *>(p) = v;
}
template <> __device__ __forceinline__ void store1<TF16>(uint8_t *p, float v) {
  *reinterpret_cast<uint16_t *>(p) = (uint16_t)pack2<TF16>(v, 0.0f);
}
template <> __device__ __forceinline__ void store1<TBF16>(uint8_t *p, float v) {
  *reinterpret_cast<uint16_t *>(p) = (uint16_t)pack2<TBF16>(v, 0.0f);
}

template <class T>
__device__ __forceinline__ void combine_body(const uint8_t *slots, const int32_t *experts,
                                             const float *weights, uint8_t *y, uint32_t n_cols,
                                             uint32_t top_k, uint32_t n_experts) {
  const uint32_t token = blockIdx.x;
  const uint64_t first = (uint64_t)token * top_k;
  if (n_cols % 8u == 0u) {
    const uint32_t c = (blockIdx.y * 256u + threadIdx.x) * 8u;
    if (c >= n_cols) return;
    float acc[8] = {};
    for (uint32_t k = 0; k < top_k; ++k) {
      if ((uint32_t)experts[first + k] >= n_experts) continue;
      const float w = weights[first + k];
      float v[8];
      load8<T>(slots + ((first + k) * n_cols + c) * T::kBytes, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(w, v[i], acc[i]);
    }
    store8<T>(y + ((uint64_t)token * n_cols + c) * T::kBytes, acc);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t c = blockIdx.y * 2048u + i * 256u + threadIdx.x;
      if (c >= n_cols) return;
      float acc = 0.0f;
      for (uint32_t k = 0; k < top_k; ++k) {
        if ((uint32_t)experts[first + k] >= n_experts) continue;
        const uint8_t *row = slots + (first + k) * n_cols * T::kBytes;
        acc = __builtin_fmaf(weights[first + k], logit_at<T>(row, c), acc);
      }
      store1<T>(y + ((uint64_t)token * n_cols + c) * T::kBytes, acc);
    }
  }
}

} // namespace

#define AXH_COMBINE(NAME, T)                                                                      \
  extern "C" __global__ void __launch_bounds__(256) axh_expert_combine_##NAME(                    \
      const uint8_t *slots, const int32_t *experts, const float *weights, uint8_t *y,             \
      uint32_t n_cols, uint32_t top_k, uint32_t n_experts) {                                      \
    combine_body<T>(slots, experts, weights, y, n_cols, top_k, n_experts);                        \
  }
AXH_COMBINE(f32, TF32)
AXH_COMBINE(f16, TF16)
AXH_COMBINE(bf16, TBF16)
