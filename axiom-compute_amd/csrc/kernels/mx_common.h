// Shared device helpers of the MXFP4 kernels (gfx950).
//
// MXFP4 (OCP Microscaling Formats v1.0): 32 consecutive elements of a row
// share one E8M0 scale byte e, the power of two 2^(e - 127) (255: NaN); an
// element is an E2M1 code (sign, two exponent bits, one mantissa bit) of
// magnitude 0, 0.5, 1, 1.5, 2, 3, 4 or 6.  In memory a row of `cols` elements
// is cols / 2 bytes of codes, the even element in the low nibble, and, in an
// array of its own, cols / 32 scale bytes; rows follow one another.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace axh {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes,
                                           0x00020000);
}

// 2^(e - 127) of a scale byte: e = 0 is the f32 subnormal 2^-127, 255 NaN.
__device__ __forceinline__ float e8m0_to_f32(uint32_t e) {
  const uint32_t b = e == 0u ? 0x00400000u : e == 255u ? 0x7FC00000u : e << 23;
  return __builtin_bit_cast(float, b);
}

// The two codes of byte kByte of a dword as f32 (v_cvt_scalef32_pk_f32_fp4
// with scale 1: exact).
template <int kByte> __device__ __forceinline__ f32x2_t fp4_pair(uint32_t codes) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, kByte);
}

// The scale byte of a block whose largest magnitude has the bits `amax`
// (0 .. 0x7FFFFFFF): floor(log2) - 2 + 127, E2M1's largest exponent being 2;
// 255 where the block holds an infinity or a NaN.  f32 subnormals and the
// smallest normals clamp to 0.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  const uint32_t e = amax >> 23;
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

// The divisor of the converting instructions for a block of scale byte e (0 .. 252,
// what mx_scale_byte gives for finite blocks): they read its exponent field only, so
// 0 stands for 2^-127.
__device__ __forceinline__ float mx_divisor(uint32_t e) {
  return __builtin_bit_cast(float, e << 23);
}

// Eight values of a block with that divisor as eight codes: round to nearest even,
// magnitudes above 6 become 6 (v_cvt_scalef32_pk_fp4_f32).
__device__ __forceinline__ uint32_t fp4_pack8(const float *v, float divisor) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], divisor, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], divisor, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], divisor, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], divisor, 3);
  return c;
}

// Element types of activations and outputs.
struct TF32 {
  static constexpr uint32_t kBytes = 4;
};
struct TF16 {
  static constexpr uint32_t kBytes = 2;
};
struct TBF16 {
  static constexpr uint32_t kBytes = 2;
};

// Two f32 as a dword of f16 or bf16, round to nearest even.
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<TF16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, half2_t));
}
template <> __device__ __forceinline__ uint32_t pack2<TBF16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, bf16x2_t));
}
template <class T> __device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b);
template <> __device__ __forceinline__ void unpack2<TF16>(uint32_t w, float &a, float &b) {
  const half2_t h = __builtin_bit_cast(half2_t, w);
  a = (float)h.x;
  b = (float)h.y;
}
template <> __device__ __forceinline__ void unpack2<TBF16>(uint32_t w, float &a, float &b) {
  a = __builtin_bit_cast(float, w << 16);
  b = __builtin_bit_cast(float, w & 0xFFFF0000u);
}

// silu(g) * u with silu(g) = g / (1 + 2^(-g log2 e)).  The exponent's rounding is
// made good by a factor (a relative error of |g| / 2^24 else), and with the 1 ulp of
// the exponential and of the reciprocal the result is within 5 ulp: the library's
// exponential and an exact division cost three times the instructions, which in the
// expert layers' epilogue counts (4096 tokens, 4 of 32 experts, 2048 x 1024: 80.6 us for
// gate and up with those, 71.0 with these).  Past +-104 the exponential is 0 or infinite
// in f32 whatever g is, and the reciprocal of infinity 0.  Below g = -87.3 the reciprocal is
// subnormal and may be 0, where silu(g) is less than 2e-36.
__device__ __forceinline__ float swiglu(float g, float u) {
  constexpr float kLog2e = 0x1.715476p+0f, kRest = 0x1.4ae0cp-26f; // their sum: log2 e
  const float n = __builtin_amdgcn_fmed3f(-g, -104.0f, 104.0f);
  const float t = n * kLog2e;
  const float rest = __builtin_fmaf(n, kRest, __builtin_fmaf(n, kLog2e, -t));
  const float e = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(rest, 0x1.62e43p-1f, 1.0f); // ln 2
  return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

template <int kCtrl> __device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, false);
}
template <int kCtrl> __device__ __forceinline__ float dpp_f32(float v) {
  return __builtin_bit_cast(float, dpp_u32<kCtrl>(__builtin_bit_cast(uint32_t, v)));
}
// Controls whose lane pairing is an exchange inside rows of 16 lanes.
constexpr int kXor1 = 0xB1;       // quad_perm [1,0,3,2]
constexpr int kXor2 = 0x4E;       // quad_perm [2,3,0,1]
constexpr int kHalfMirror = 0x141; // lane i <-> 7 - i in each 8
constexpr int kMirror = 0x140;     // lane i <-> 15 - i in each 16

} // namespace axh
