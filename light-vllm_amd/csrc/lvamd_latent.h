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

// Whether rows at p, of these element strides, are made of whole 16-byte chunks.
inline bool rows16(const void* p, std::initializer_list<int64_t> strides) {
  if (((uintptr_t)p & 15u) != 0) return false;
  for (int64_t s : strides)
    if (s % 8 != 0) return false;
  return true;
}

}  // namespace lvamd
