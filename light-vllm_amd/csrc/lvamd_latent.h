// Sizes and dispatch of the kernels over a paged cache of latent vectors on
// gfx950.
//
// A layer's pool holds one row per token, [latent | rotated key]: L latent
// values that every head shares, then P values of one rotated key.
#pragma once

#include <initializer_list>

#include "lvamd_common.h"

namespace lvamd {

inline bool latent_sizes(int latent, int rope) {
  return latent >= 128 && latent <= 512 && latent % 128 == 0 && (rope == 32 || rope == 64);
}
inline bool latent_dtype(int dtype) { return dtype == LVAMD_BF16 || dtype == LVAMD_F16; }

template <typename T, int L, typename F>
int latent_with_rope(int rope, F& f) {
  switch (rope) {
    case 32: return f.template operator()<T, L, 32>();
    case 64: return f.template operator()<T, L, 64>();
    default: return LVAMD_ERR_UNSUPPORTED;
  }
}
template <typename T, typename F>
int latent_with_size(int latent, int rope, F& f) {
  switch (latent) {
    case 128: return latent_with_rope<T, 128>(rope, f);
    case 256: return latent_with_rope<T, 256>(rope, f);
    case 384: return latent_with_rope<T, 384>(rope, f);
    case 512: return latent_with_rope<T, 512>(rope, f);
    default: return LVAMD_ERR_UNSUPPORTED;
  }
}
template <typename F>
int latent_dispatch(int dtype, int latent, int rope, F f) {
  switch (dtype) {
    case LVAMD_BF16: return latent_with_size<__bf16>(latent, rope, f);
    case LVAMD_F16: return latent_with_size<_Float16>(latent, rope, f);
    default: return LVAMD_ERR_UNSUPPORTED;
  }
}

// Softmax weights are rounded to T as 2^kWeightLift times themselves (their sum counts
// them so too).  fp16 has a fixed step of 2^-24 below 2^-14: unlifted, a weight less than
// 2^-25 of the largest would count as nothing, and thousands of such keys with it;
// lifted that is 2^-32.  The largest weight stays below fp16's largest: 2^7 times the
// 2^8 by which a running maximum may lag.
template <typename T>
inline constexpr float kWeightLift = std::is_same<T, _Float16>::value ? 7.f : 0.f;

// A pair turned by an angle of cosine c and sine s.  (Written as these products,
// so that every kernel rounds alike.)
__device__ __forceinline__ void turn_pair(float x, float y, float c, float s, float& a, float& b) {
  a = __builtin_fmaf(x, c, -(y * s));
  b = __builtin_fmaf(y, c, x * s);
}
// Eight values, four pairs (2i, 2i + 1); c and s are four floats each, 16-byte aligned.
template <typename T>
__device__ __forceinline__ uint4 turn_chunk(uint4 x, f32x4 cv, f32x4 sv) {
  T e[8];
  __builtin_memcpy(e, &x, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    turn_pair(to_f32(e[2 * i]), to_f32(e[2 * i + 1]), cv[i], sv[i], a, b);
    e[2 * i] = from_f32<T>(a);
    e[2 * i + 1] = from_f32<T>(b);
  }
  __builtin_memcpy(&x, e, 16);
  return x;
}
template <typename T>
__device__ __forceinline__ uint4 turn_chunk(uint4 x, const float* c, const float* s) {
  return turn_chunk<T>(x, *reinterpret_cast<const f32x4*>(c), *reinterpret_cast<const f32x4*>(s));
}
// Sixteen values, eight pairs (lo i, hi i).
template <typename T>
__device__ __forceinline__ void turn_chunks(uint4& lo, uint4& hi, const f32x4 (&c)[2], const f32x4 (&s)[2]) {
  T x[8], y[8];
  __builtin_memcpy(x, &lo, 16);
  __builtin_memcpy(y, &hi, 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a, b;
    turn_pair(to_f32(x[i]), to_f32(y[i]), c[i / 4][i % 4], s[i / 4][i % 4], a, b);
    x[i] = from_f32<T>(a);
    y[i] = from_f32<T>(b);
  }
  __builtin_memcpy(&lo, x, 16);
  __builtin_memcpy(&hi, y, 16);
}
template <typename T>
__device__ __forceinline__ void turn_chunks(uint4& lo, uint4& hi, const float* c, const float* s) {
  const f32x4 cv[2] = {reinterpret_cast<const f32x4*>(c)[0], reinterpret_cast<const f32x4*>(c)[1]};
  const f32x4 sv[2] = {reinterpret_cast<const f32x4*>(s)[0], reinterpret_cast<const f32x4*>(s)[1]};
  turn_chunks<T>(lo, hi, cv, sv);
}

// Whether rows at p, of these element strides, are made of whole 16-byte chunks.
inline bool rows16(const void* p, std::initializer_list<int64_t> strides) {
  if (((uintptr_t)p & 15u) != 0) return false;
  for (int64_t s : strides)
    if (s % 8 != 0) return false;
  return true;
}

}  // namespace lvamd
