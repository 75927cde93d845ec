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
// Sixteen elements (two 16-byte chunks of T): the largest finite magnitude, as
// its fp32 bits (which order as the magnitudes do), and their codes.
template <typename T>
__device__ __forceinline__ uint32_t q8_largest16(uint4 lo, uint4 hi) {
  T e[16];
  __builtin_memcpy(e, &lo, 16);
  __builtin_memcpy(e + 8, &hi, 16);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float f = __builtin_fabsf(to_f32(e[i]));
    m = fmaxf(m, f < INFINITY ? f : 0.f);  // (NaN compares false)
  }
  return __float_as_uint(m);
}
template <typename T>
__device__ __forceinline__ uint4 q8_codes16(uint4 lo, uint4 hi, float scale) {
  T e[16];
  __builtin_memcpy(e, &lo, 16);
  __builtin_memcpy(e + 8, &hi, 16);
  const float inverse = q8_inverse(scale);
  float f[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = q8_scaled<T>(to_f32(e[i]), inverse);
  return make_uint4(q8_pack4(f[0], f[1], f[2], f[3]), q8_pack4(f[4], f[5], f[6], f[7]),
                    q8_pack4(f[8], f[9], f[10], f[11]), q8_pack4(f[12], f[13], f[14], f[15]));
}
// Sixteen codes times ratio, as q8_rescale4.
__device__ __forceinline__ uint4 q8_rescale16(uint4 c, float ratio) {
  return make_uint4(q8_rescale4(c.x, ratio), q8_rescale4(c.y, ratio), q8_rescale4(c.z, ratio), q8_rescale4(c.w, ratio));
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
// The same mask for four elements of T that are about to be stored: NaN codes
// are what its values that are not finite become.
template <typename T>
__device__ __forceinline__ uint32_t q8_nan4_of(uint2 x) {
  constexpr uint32_t e = std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
  auto bit = [&](uint32_t w, int from, int to) { return ((w >> from) & e) == e ? 0x80u << to : 0u; };
  return bit(x.x, 0, 0) | bit(x.x, 16, 8) | bit(x.y, 0, 16) | bit(x.y, 16, 24);
}
// The codes with every NaN replaced by zero.
__device__ __forceinline__ uint32_t q8_without_nan4(uint32_t w) {
  const uint32_t n = q8_nan4(w) >> 7;  // 1 per NaN byte
  return w & ~(n * 255u);
}
__device__ __forceinline__ uint4 q8_without_nan16(uint4 c) {
  return make_uint4(q8_without_nan4(c.x), q8_without_nan4(c.y), q8_without_nan4(c.z), q8_without_nan4(c.w));
}

// Row stride, in 16-byte chunks, of a tile of dequantised rows of `chunks`
// chunks in LDS: 2 modulo 4, so the 16 rows of an operand read (32 lanes: 16
// rows at two chunks) and the 8 rows of a transpose read (32 bytes each)
// cover all 64 banks evenly.
constexpr int q8_row_stride(int chunks) { return chunks + (chunks % 4 == 0 ? 2 : 0); }

// ---- host: the types and head sizes that the attention kernels are built for
inline bool q8_head_size(int d) { return d >= 32 && d <= 256 && d % 16 == 0; }

template <typename T, typename F>
int q8_with_head_size(int head_size, F& f) {
  switch (head_size) {
    case 32: return f.template operator()<T, 32>();
    case 48: return f.template operator()<T, 48>();
    case 64: return f.template operator()<T, 64>();
    case 80: return f.template operator()<T, 80>();
    case 96: return f.template operator()<T, 96>();
    case 112: return f.template operator()<T, 112>();
    case 128: return f.template operator()<T, 128>();
    case 144: return f.template operator()<T, 144>();
    case 160: return f.template operator()<T, 160>();
    case 176: return f.template operator()<T, 176>();
    case 192: return f.template operator()<T, 192>();
    case 208: return f.template operator()<T, 208>();
    case 224: return f.template operator()<T, 224>();
    case 240: return f.template operator()<T, 240>();
    case 256: return f.template operator()<T, 256>();
    default: return LVAMD_ERR_UNSUPPORTED;
  }
}
template <typename F>
int q8_dispatch(int dtype, int head_size, F f) {
  if (!q8_head_size(head_size)) return LVAMD_ERR_UNSUPPORTED;
  switch (dtype) {
    case LVAMD_BF16: return q8_with_head_size<__bf16>(head_size, f);
    case LVAMD_F16: return q8_with_head_size<_Float16>(head_size, f);
    default: return LVAMD_ERR_UNSUPPORTED;
  }
}

}  // namespace lvamd
