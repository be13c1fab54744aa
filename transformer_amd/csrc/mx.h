// Blocks of 32 values along a row that share a power of two 2^(b - 127), b a byte (255: not a number), the layout
// that gfx950's matrix instructions take operands in. Weights are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a
// byte with the first in the low half; rows of activations are e4m3 (largest 448).
//
// The scale of a block is the smallest power of two with which its largest magnitude is at most the format's
// largest value, so nothing is cut off; the byte does not go below 0. A block that holds an infinity or a NaN gets
// the byte 255 and stands for 32 NaN.
#pragma once
#include "common.h"

#define MX_BLOCK 32
#define MX_NAN 255u

typedef uint32_t mx_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 mx_bf16x2;
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 mx_bf16x8;

// Byte of the scale from the bits of the largest magnitude, for a largest value of (1 + top_mantissa / 2^23) 2^top_exponent.
// Bits of magnitudes order as the magnitudes do, infinities and NaN above them all.
template <uint32_t TOP_EXPONENT, uint32_t TOP_MANTISSA>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t bits) {
  if (bits >= 0x7f800000u) return MX_NAN;
  const int b = (int)(bits >> 23) - (int)TOP_EXPONENT + ((bits & 0x7fffffu) > TOP_MANTISSA ? 1 : 0);
  return b > 0 ? (uint32_t)b : 0u;
}
__device__ __forceinline__ uint32_t mx8_scale_byte(uint32_t bits) { return mx_scale_byte<8, 0x600000u>(bits); }   // 448 = 1.75 * 2^8
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t bits) { return mx_scale_byte<2, 0x400000u>(bits); }   // 6 = 1.5 * 2^2

// 2^(127 - byte), which takes a block to its codes: exact, as both formats' bytes stay below 254
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// 2^(byte - 127): 0 is a subnormal float32, 255 a NaN
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte == MX_NAN ? 0x7fc00000u : byte ? byte << 23 : 0x00400000u);
}

__device__ __forceinline__ uint32_t mx_max(uint32_t a, uint32_t b) { return a > b ? a : b; }

// the largest of 8 magnitudes' bits
__device__ __forceinline__ uint32_t mx_top8(const float* v) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = mx_max(t, __float_as_uint(v[i]) & 0x7fffffffu);
  return t;
}

// the largest over the four lanes of a quad, which hold a block, 8 values each
__device__ __forceinline__ uint32_t mx_top_quad(uint32_t t) {
  t = mx_max(t, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)t, 0xB1, 0xf, 0xf, true));
  return mx_max(t, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)t, 0x4E, 0xf, 0xf, true));
}

// 8 values to e4m3, each rounded to nearest even once: the multiplication by a power of two is exact, but for values below
// 2^-126 of a block far below what e4m3 holds
__device__ __forceinline__ mx_u32x2 mx8_codes(const float* v, uint32_t byte) {
  if (byte == MX_NAN) return mx_u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
  const float s = mx_inverse(byte);
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * s, v[1] * s, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * s, v[3] * s, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * s, v[5] * s, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * s, v[7] * s, hi, true);
  return mx_u32x2{(uint32_t)lo, (uint32_t)hi};
}

// Stores a lane's 8 values of a row whose block the quad shares: codes at `codes`, the byte at `scale` by the quad's first lane.
__device__ __forceinline__ void mx8_store(const float* v, uint8_t* codes, uint8_t* scale) {
  const uint32_t byte = mx8_scale_byte(mx_top_quad(mx_top8(v)));
  *reinterpret_cast<mx_u32x2*>(codes) = mx8_codes(v, byte);
  if (threadIdx.x % 4 == 0) *scale = (uint8_t)byte;
}

// e2m1 of a magnitude over its scale, to nearest, ties to the code with an even last bit
__device__ __forceinline__ uint32_t mx4_code(float v) {
  const float a = fabsf(v);
  uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  return c | (__float_as_uint(v) >> 31) << 3;
}

// 8 values from 16 (bfloat16) or 32 bytes
__device__ __forceinline__ void mx_load8(const bf16_t* p, float* v) {
  const mx_u32x4 q = *reinterpret_cast<const mx_u32x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(q[i] << 16);
    v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void mx_load8(const float* p, float* v) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
