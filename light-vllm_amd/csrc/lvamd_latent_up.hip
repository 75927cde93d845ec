// The heads' weights of attention over latent vectors, on gfx950: products of
// every head's rows with that head's weights, y[t][h] = W[h] x[t][h].
//   * lvamd_latent_heads: queries times key_up^T (into latent space) and results
//     times value_up (out of it), for the steps' short requests.
//   * lvamd_latent_expand: a request's rows times key_up and value_up, into
//     per-head keys and values in a workspace, for its long prompt chunk.
// Products are MFMA 16x16x32 with fp32 sums, rounded once to T.

#include "lvamd_latent.h"

namespace lvamd {

namespace {

typedef const __attribute__((address_space(1))) void* lds_gptr;
typedef __attribute__((address_space(3))) void* lds_lptr;

__device__ __forceinline__ constexpr int swizzle(int row) {
  return (((row >> 2) & 1) << 1) | ((((row >> 3) ^ (row >> 1)) & 1) << 2);
}

struct HeadsArgs {
  const void* x;
  int64_t x_tok_stride, x_head_stride;
  const void* w;  // [heads][n][k]
  void* y;
  int64_t y_tok_stride, y_head_stride;
  const int32_t* rows;  // token of row i, or null: token i
  int32_t num_rows, k, n;
};

}  // namespace

// A wave: 16 values of n for 16 MT rows.  Weights and rows go from global memory
// to operands as they lie (each lane 16 bytes of a row): a step's few tokens
// leave nothing to reuse that the caches do not hold.
template <typename T, int MT>
__global__ __launch_bounds__(256) void latent_heads_kernel(const HeadsArgs a, const int32_t blocks_n) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int l16 = lane & 15, g = lane >> 4;
  const int h = blockIdx.x / blocks_n;
  const int n0 = (blockIdx.x - h * blocks_n) * 64 + 16 * wave;
  const int m0 = blockIdx.y * 16 * MT;
  const T* w = static_cast<const T*>(a.w) + ((int64_t)h * a.n + n0 + l16) * a.k + 8 * g;
  const T* x[MT];
  int64_t tok[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = min(m0 + 16 * m + l16, a.num_rows - 1);
    tok[m] = a.rows ? a.rows[r] : r;
    x[m] = static_cast<const T*>(a.x) + tok[m] * a.x_tok_stride + (int64_t)h * a.x_head_stride + 8 * g;
    acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int k = 0; k < a.k; k += 64) {
#pragma unroll
    for (int kk = 0; kk < 64; kk += 32) {
      const uint4 wf = load16(w + k + kk);
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] = Mma<T>::qk(wf, load16(x[m] + k + kk), acc[m]);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m0 + 16 * m + l16 >= a.num_rows) continue;
    T* y = static_cast<T*>(a.y) + tok[m] * a.y_tok_stride + (int64_t)h * a.y_head_stride + n0 + 4 * g;
    store_partial4<false, T>(y, acc[m], 1.f);
  }
}

// ---------------------------------------------------------------------------
// Expand.  A workgroup of four waves: 128 rows of the cache by NW values of one
// head's keys or values; steps of 64 latent values through LDS (both operands
// loaded straight into it, double-buffered).
// ---------------------------------------------------------------------------
namespace {

constexpr int kBlockRows = 64;  // rows per block record
constexpr int kTileRows = 128;

struct ExpandArgs {
  const void* pool;          // [slots][row]
  const int32_t* blocks;     // [n][4]: table offset, first position, positions of the request, 0
  const int32_t* tables;
  const void* w;             // [heads][NW][latent]
  void* out;                 // [heads][keys][NW]
  void* rope;                // [keys][rope], or null
  int64_t keys;              // rows of the workspace, a multiple of 128
  int32_t heads, tiles, block_size, latent, row;
  FastDiv by_block, by_heads;
};

// The largest value of T holds what is beyond it (a masked row's infinity would
// not stay where it is); NaN for sums that are not finite.
template <typename T>
__device__ __forceinline__ float held(float x) {
  if constexpr (std::is_same<T, _Float16>::value) {
    return __builtin_fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f) : __uint_as_float(0x7fc00000u);
  }
  return x;
}

}  // namespace

template <typename T, int NW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void latent_expand_kernel(const ExpandArgs a) {
  constexpr int A_BYTES = kTileRows * 128, B_BYTES = NW * 128;
  __shared__ __attribute__((aligned(1024))) char a0[A_BYTES];
  __shared__ __attribute__((aligned(1024))) char a1[A_BYTES];
  __shared__ __attribute__((aligned(1024))) char b0[B_BYTES];
  __shared__ __attribute__((aligned(1024))) char b1[B_BYTES];
  const int tid = threadIdx.x & 255;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int l16 = lane & 15, g = lane >> 4;
  // Eight tiles of rows at a time, one per XCD, each for all heads: an XCD's L2
  // holds the rows it works on.
  const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
  const int tg = fast_div(i, a.by_heads);
  const int h = i - tg * a.heads, tile = tg * 8 + xcd;
  if (tile >= a.tiles) return;
  // Loads: instruction j of a wave fills rows 8 (4 j + wave) .. + 7, lane l row
  // l / 8 of them, chunk slot l % 8.
  constexpr int LA = kTileRows / 32, LB = NW / 32;
  gptr<const T> arow[LA];
  gptr<const T> brow[LB];
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = 8 * (4 * j + wave) + (lane >> 3);
    const int32_t* b = a.blocks + 4 * (2 * tile + (r >= kBlockRows ? 1 : 0));
    const int pos = min(b[1] + (r & (kBlockRows - 1)), b[2] - 1);
    const int lb = fast_div(pos, a.by_block);
    const int64_t slot = (int64_t)a.tables[b[0] + lb] * a.block_size + (pos - lb * a.block_size);
    arow[j] = (gptr<const T>)(a.pool) + slot * a.row + 8 * ((lane & 7) ^ swizzle(r));
    if (a.rope && h == 0) {
      const int chunks = (a.row - a.latent) / 8;
      if ((lane & 7) < chunks) {
        gptr<const T> const from = (gptr<const T>)(a.pool) + slot * a.row + a.latent + 8 * (lane & 7);
        store16((gptr<T>)(a.rope) + ((int64_t)tile * kTileRows + r) * (a.row - a.latent) + 8 * (lane & 7), load16(from));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < LB; ++j) {
    const int r = 8 * (4 * j + wave) + (lane >> 3);
    brow[j] = (gptr<const T>)(a.w) + ((int64_t)h * NW + r) * a.latent + 8 * ((lane & 7) ^ swizzle(r));
  }
  auto issue = [&](int k, char* ta, char* tb) {
#pragma unroll
    for (int j = 0; j < LA; ++j)
      __builtin_amdgcn_global_load_lds((lds_gptr)(arow[j] + k), (lds_lptr)(ta + (4 * j + wave) * 1024), 16, 0, 0);
#pragma unroll
    for (int j = 0; j < LB; ++j)
      __builtin_amdgcn_global_load_lds((lds_gptr)(brow[j] + k), (lds_lptr)(tb + (4 * j + wave) * 1024), 16, 0, 0);
  };
  // Wave tile: 64 rows (wave / 2) by NW / 2 values (wave % 2).
  constexpr int RT = 4, NT = NW / 32;
  const int r0 = 64 * (wave >> 1), n0 = NW / 2 * (wave & 1);
  f32x4 acc[NT][RT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[n][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const char* ta, const char* tb) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int slot = 16 * ((4 * kk + g) ^ swizzle(l16));
      uint4 wf[NT], xf[RT];
#pragma unroll
      for (int n = 0; n < NT; ++n) wf[n] = *reinterpret_cast<const uint4*>(tb + (n0 + 16 * n + l16) * 128 + slot);
#pragma unroll
      for (int r = 0; r < RT; ++r) xf[r] = *reinterpret_cast<const uint4*>(ta + (r0 + 16 * r + l16) * 128 + slot);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[n][r] = Mma<T>::qk(wf[n], xf[r], acc[n][r]);
    }
  };
  auto done = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __builtin_amdgcn_s_barrier();
  };
  issue(0, a0, b0);
  done();
  // (latent is a multiple of 128: an even number of steps.)
  for (int k = 0; k < a.latent; k += 128) {
    issue(k + 64, a1, b1);
    compute(a0, b0);
    done();
    if (k + 128 < a.latent) issue(k + 128, a0, b0);
    compute(a1, b1);
    done();
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int64_t key = (int64_t)tile * kTileRows + r0 + 16 * r + l16;
    T* const to = static_cast<T*>(a.out) + ((int64_t)h * a.keys + key) * NW + n0 + 4 * g;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 v = acc[n][r];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = held<T>(v[e]);
      store_partial4<false, T>(to + 16 * n, v, 1.f);
    }
  }
}

}  // namespace lvamd

using namespace lvamd;

extern "C" int lvamd_latent_heads(const void* x, int64_t x_token_stride, int64_t x_head_stride, const void* weights, void* y,
                                  int64_t y_token_stride, int64_t y_head_stride, const int32_t* rows, int64_t num_rows,
                                  int32_t num_heads, int32_t k, int32_t n, int32_t dtype, lvamd_stream_t stream) {
  if (!latent_dtype(dtype) || k <= 0 || k % 64 != 0 || n <= 0 || n % 64 != 0) return LVAMD_ERR_UNSUPPORTED;
  if (num_rows < 0 || num_rows > 65535 * 16LL || num_heads <= 0) return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return LVAMD_OK;
  if (!x || !weights || !y || !rows16(x, {x_token_stride, x_head_stride}) || !rows16(weights, {}) || ((uintptr_t)y & 7u) ||
      y_token_stride % 4 != 0 || y_head_stride % 4 != 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  HeadsArgs a{x, x_token_stride, x_head_stride, weights, y, y_token_stride, y_head_stride, rows, (int32_t)num_rows, k, n};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int blocks_n = n / 64;
  auto launch = [&]<typename T>() -> int {
    // 64 rows per wave where that leaves the GPU enough workgroups.
    if (num_rows > 64 && (int64_t)num_heads * blocks_n * ((num_rows + 63) / 64) >= 512) {
      hipLaunchKernelGGL((latent_heads_kernel<T, 4>), dim3(num_heads * blocks_n, (unsigned)((num_rows + 63) / 64)), dim3(256),
                         0, s, a, blocks_n);
    } else {
      hipLaunchKernelGGL((latent_heads_kernel<T, 1>), dim3(num_heads * blocks_n, (unsigned)((num_rows + 15) / 16)), dim3(256),
                         0, s, a, blocks_n);
    }
    return launch_status();
  };
  return dtype == LVAMD_BF16 ? launch.operator()<__bf16>() : launch.operator()<_Float16>();
}

extern "C" int lvamd_latent_expand(const void* pool, const int32_t* blocks, int32_t num_blocks, const int32_t* tables,
                                   const void* key_up, const void* value_up, void* keys, void* values, void* rope_keys,
                                   int32_t num_heads, int32_t latent_size, int32_t rope_size, int32_t nope_size,
                                   int32_t value_size, int32_t block_size, int32_t dtype, lvamd_stream_t stream) {
  if (!latent_sizes(latent_size, rope_size) || !latent_dtype(dtype) || (nope_size != 64 && nope_size != 128) ||
      (value_size != 64 && value_size != 128))
    return LVAMD_ERR_UNSUPPORTED;
  if (num_blocks < 0 || num_blocks % 2 != 0 || num_heads <= 0 || block_size <= 0) return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_blocks == 0) return LVAMD_OK;
  if (!pool || !blocks || !tables || !key_up || !value_up || !keys || !values || !rope_keys || !rows16(pool, {}) ||
      !rows16(key_up, {}) || !rows16(value_up, {}) || !rows16(keys, {}) || !rows16(values, {}) || !rows16(rope_keys, {}))
    return LVAMD_ERR_INVALID_ARGUMENT;
  const int tiles = num_blocks / 2;
  const int64_t grid = (int64_t)(tiles + 7) / 8 * 8 * num_heads;
  if (grid > 0x7fffffffLL) return LVAMD_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&]<typename T>(const void* w, void* out, void* rope, int width) -> int {
    ExpandArgs a{.by_block = FastDiv(block_size), .by_heads = FastDiv(num_heads)};
    a.pool = pool;
    a.blocks = blocks;
    a.tables = tables;
    a.w = w;
    a.out = out;
    a.rope = rope;
    a.keys = (int64_t)tiles * kTileRows;
    a.heads = num_heads;
    a.tiles = tiles;
    a.block_size = block_size;
    a.latent = latent_size;
    a.row = latent_size + rope_size;
    if (width == 64) {
      hipLaunchKernelGGL((latent_expand_kernel<T, 64>), dim3((unsigned)grid), dim3(256), 0, s, a);
    } else {
      hipLaunchKernelGGL((latent_expand_kernel<T, 128>), dim3((unsigned)grid), dim3(256), 0, s, a);
    }
    return launch_status();
  };
  auto both = [&]<typename T>() -> int {
    const int status = launch.operator()<T>(key_up, keys, rope_keys, nope_size);
    return status != LVAMD_OK ? status : launch.operator()<T>(value_up, values, nullptr, value_size);
  };
  return dtype == LVAMD_BF16 ? both.operator()<__bf16>() : both.operator()<_Float16>();
}
