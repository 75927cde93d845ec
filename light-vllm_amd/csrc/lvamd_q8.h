// Device helpers of the 8-bit paged cache (e4m3 codes, one scale per block and
// kv head) on gfx950.
//
// A row of a block stands for code * scale with scale = 2^e.  Powers of two
// make every conversion exact where a general factor would round: a code has
// four significant bits, so code * scale is a bf16 value (fp16: exact from
// 2^-21 on, below that the nearest fp16 value), and moving a row to a larger
// scale only lowers its exponent (it rounds where the code becomes subnormal).
// The format loses nothing by it: an e4m3 value's relative step does not
// depend on the scale.
#pragma once

#include "lvamd_common.h"

namespace lvamd {

constexpr int kQ8MinExponent = -100;  // of a block that holds zeros only

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Smallest e >= kQ8MinExponent with amax <= 448 * 2^e, as the fp32 2^e
// (448 = 1.75 * 2^8; amax finite and not negative, so e <= 120).
__device__ __forceinline__ float q8_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)((e < kQ8MinExponent ? kQ8MinExponent : e) + 127) << 23);
}
// 1 / scale of a power of two from 2^-126 to 2^126.
__device__ __forceinline__ float q8_inverse(float scale) { return __uint_as_float(0x7f000000u - __float_as_uint(scale)); }

// Largest magnitude that is stored: the largest value of T with four
// significant bits, so that no code's value overflows T.
template <typename T>
__device__ __forceinline__ float q8_largest() {
  return std::is_same<T, __bf16>::value ? __uint_as_float(0x7f700000u) : 61440.f;
}

// Code input of one element: x / scale, NaN where x is not finite (e4m3 has
// no infinity).  Rounded once, to the nearest code (ties to even), by the
// conversion instruction.
template <typename T>
__device__ __forceinline__ float q8_scaled(float x, float inverse) {
  const float big = q8_largest<T>();
  return __builtin_fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -big, big) * inverse : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d) {
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Four codes times ratio (a power of two, at most 1) as codes.
__device__ __forceinline__ uint32_t q8_rescale4(uint32_t w, float ratio) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return q8_pack4(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
}

// Four codes times scale as four elements of T.
template <typename T>
__device__ __forceinline__ uint2 q8_values4(uint32_t w, float scale) {
  if constexpr (std::is_same<T, __bf16>::value) {
    return make_uint2(bitcast<uint32_t>((bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
                      bitcast<uint32_t>((bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)));
  } else {
    return make_uint2(bitcast<uint32_t>((f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false)),
                      bitcast<uint32_t>((f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true)));
  }
}
// Sixteen codes times scale as two 16-byte chunks of T.
template <typename T>
__device__ __forceinline__ void q8_values16(uint4 codes, float scale, uint4& lo, uint4& hi) {
  const uint2 a = q8_values4<T>(codes.x, scale), b = q8_values4<T>(codes.y, scale);
  const uint2 c = q8_values4<T>(codes.z, scale), d = q8_values4<T>(codes.w, scale);
  lo = make_uint4(a.x, a.y, b.x, b.y);
  hi = make_uint4(c.x, c.y, d.x, d.y);
}

// Whether one of four codes is NaN (0x7f or 0xff), as a mask of the codes'
// sign bits: the low seven bits plus one carry into bit 7.
__device__ __forceinline__ uint32_t q8_nan4(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ bool q8_has_nan(uint4 c) {
  return (q8_nan4(c.x) | q8_nan4(c.y) | q8_nan4(c.z) | q8_nan4(c.w)) != 0;
}
// The codes with every NaN replaced by zero.
__device__ __forceinline__ uint32_t q8_without_nan4(uint32_t w) {
  const uint32_t n = q8_nan4(w) >> 7;  // 1 per NaN byte
  return w & ~(n * 255u);
}

// Row stride, in 16-byte chunks, of a tile of dequantised rows of `chunks`
// chunks in LDS: 2 modulo 4, so the 16 rows of an operand read (32 lanes: 16
// rows at two chunks) and the 8 rows of a transpose read (32 bytes each)
// cover all 64 banks evenly.
constexpr int q8_row_stride(int chunks) { return chunks + (chunks % 4 == 0 ? 2 : 0); }

}  // namespace lvamd
