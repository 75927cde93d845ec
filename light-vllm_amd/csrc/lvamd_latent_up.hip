// The heads' weights of attention over latent vectors, on gfx950: products of
// every head's rows with that head's weights, y[t][h] = W[h] x[t][h].
//   * lvamd_latent_heads: queries times key_up^T (into latent space) and results
//     times value_up (out of it), for the steps' short requests.
//   * lvamd_latent_expand: a request's rows times key_up and value_up, into
//     per-head keys and values in a workspace, for its long prompt chunk.
// Products are MFMA 16x16x32 with fp32 sums, rounded once to T: what they make
// is an operand of the next matrix instructions, which take one type.  (Keeping the
// attended latents in two halves, 16 bits each, moved a decode layer's error from
// 0.0034 to 0.0030 of its norm, for 10 % of its time; what stays is the rounding of
// the queries in latent space, whose second half no instance has registers for.)

#include "lvamd_latent.h"

namespace lvamd {

namespace {

typedef const __attribute__((address_space(1))) void* lds_gptr;
typedef __attribute__((address_space(3))) void* lds_lptr;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct HeadsArgs {
  const void* x;
  int64_t x_tok_stride, x_head_stride;
  const void* w;  // [heads][n][k]
  void* y;
  int64_t y_tok_stride, y_head_stride;
  const int32_t *x_rows, *y_rows;  // where row i lies in x and y, or null: i
  int32_t num_rows, k, n;
};

}  // namespace

// A wave: 16 NT values of n for 16 MT rows.  Weights and rows go from global memory
// to operands as they lie (each lane 16 bytes of a row): a step's few tokens
// leave nothing to reuse that the caches do not hold.  With two of NT the rows of
// the weights are dealt so that a lane's results of both lie side by side.
template <typename T, int MT, int NT>
__global__ __launch_bounds__(256) void latent_heads_kernel(const HeadsArgs a, const int32_t waves, const FastDiv by_blocks) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int l16 = lane & 15, g = lane >> 4;
  const int i = blockIdx.x * 4 + wave;
  if (i >= waves) return;
  const int h = fast_div(i, by_blocks);
  const int n0 = 16 * NT * (i - h * (a.n / (16 * NT)));
  const int m0 = blockIdx.y * 16 * MT;
  const int wrow = NT == 1 ? l16 : 8 * (l16 >> 2) + (l16 & 3);
  const T* w = static_cast<const T*>(a.w) + ((int64_t)h * a.n + n0 + wrow) * a.k + 8 * g;
  const T* x[MT];
  int to[MT];
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = min(m0 + 16 * m + l16, a.num_rows - 1);
    to[m] = a.y_rows ? a.y_rows[r] : r;
    const int64_t at = a.x_rows ? a.x_rows[r] : r;
    x[m] = static_cast<const T*>(a.x) + at * a.x_tok_stride + (int64_t)h * a.x_head_stride + 8 * g;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int k = 0; k < a.k; k += 64) {
#pragma unroll
    for (int kk = 0; kk < 64; kk += 32) {
      uint4 wf[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) wf[n] = load16(w + (int64_t)4 * n * a.k + k + kk);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4 xf = load16(x[m] + k + kk);
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = Mma<T>::qk(wf[n], xf, acc[m][n]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m0 + 16 * m + l16 >= a.num_rows) continue;
    T* y = static_cast<T*>(a.y) + to[m] * a.y_tok_stride + (int64_t)h * a.y_head_stride + n0 + 4 * NT * g;
#pragma unroll
    for (int n = 0; n < NT; ++n) store_partial4<false, T>(y + 4 * n, acc[m][n], 1.f);
  }
}

// ---------------------------------------------------------------------------
// Expand.  A workgroup of four waves: 128 rows of the cache by one head's keys and
// values, steps of 32 latent values through LDS (both operands loaded straight
// into it), three steps in LDS: two are on their way while one is multiplied.
// A wave's tile is 64 rows by the head's keys or by its values.
//
// LDS layout of a step: rows of 64 bytes, chunk slots permuted by row bits (reads
// of 16 rows by 4 chunks then cover every bank evenly).  The weights' rows are
// dealt to the matrix instructions so that a lane's results of two of them lie
// side by side: 16-byte stores.
//
// 16,384 rows for 16 heads (512 to 128 + 128, 69 GFLOP, 134 MB out): 97 us,
// 0.71 PFLOP/s; 125 in two launches of 64-value steps two deep, 113 with 8-byte
// stores.  LDS reads (12 for 32 matrix instructions) and the stores bound it.
// ---------------------------------------------------------------------------
namespace {

constexpr int kBlockRows = 64;  // rows per block record
constexpr int kTileRows = 128;
constexpr int kStep = 32;

__device__ __forceinline__ constexpr int swz(int row) {
  return ((row >> 2) & 1) | ((((row >> 2) ^ (row >> 3)) & 1) << 1);
}

// The same for the weights, read in fours of rows, eight rows apart.
__device__ __forceinline__ constexpr int swz_weights(int row) { return (row >> 3) & 3; }

struct ExpandArgs {
  const void* pool;          // [slots][row]
  const int32_t* blocks;     // [n][4]: table offset, first position, positions of the request, 0
  const int32_t* tables;
  const void* key_up;        // [heads][NK][latent]
  const void* value_up;      // [heads][NV][latent]
  void* key_out;             // [heads][keys][NK]
  void* value_out;           // [heads][keys][NV]
  void* rope;                // [keys][rope]
  int64_t keys;              // rows of the workspace, a multiple of 128
  int32_t heads, tiles, block_size, rope_size;
  FastDiv by_block, by_heads;
};

// The larger of each half's magnitude, as bits: what is not a number of T is at
// least its infinity's.
__device__ __forceinline__ uint32_t larger_bits(uint32_t most, uint32_t x) {
  return bitcast<uint32_t>(__builtin_elementwise_max(bitcast<u16x2>(most), bitcast<u16x2>(x & 0x7fff7fffu)));
}
template <typename T>
__device__ __forceinline__ bool all_numbers(uint32_t most) {
  constexpr uint32_t infinity = std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
  return max(most & 0xffffu, most >> 16) < infinity;
}

}  // namespace

template <typename T, int L, int NK, int NV>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void latent_expand_kernel(const ExpandArgs a) {
  const int ROW = L + a.rope_size;
  constexpr int A_BYTES = kTileRows * 64, B_BYTES = (NK + NV) * 64;
  __shared__ __attribute__((aligned(1024))) char a0[A_BYTES];
  __shared__ __attribute__((aligned(1024))) char a1[A_BYTES];
  __shared__ __attribute__((aligned(1024))) char a2[A_BYTES];
  __shared__ __attribute__((aligned(1024))) char b0[B_BYTES];
  __shared__ __attribute__((aligned(1024))) char b1[B_BYTES];
  __shared__ __attribute__((aligned(1024))) char b2[B_BYTES];
  __shared__ uint32_t lost[kTileRows];
  const int tid = threadIdx.x & 255;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int l16 = lane & 15, g = lane >> 4;
  // Eight tiles of rows at a time, one per XCD, each for all heads: an XCD's L2
  // holds the rows it works on.
  const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
  const int tg = fast_div(i, a.by_heads);
  const int h = i - tg * a.heads, tile = tg * 8 + xcd;
  if (tile >= a.tiles) return;
  // Loads: instruction j of a wave fills rows 16 (4 j + wave) .. + 15, lane l row
  // l / 4 of them, chunk slot l % 4.
  constexpr int LA = kTileRows / 64, LB = (NK + NV) / 64;
  gptr<const T> arow[LA];
  gptr<const T> brow[LB];
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = 16 * (4 * j + wave) + (lane >> 2);
    const int32_t* b = a.blocks + 4 * (2 * tile + j);
    const int pos = min(b[1] + (r & (kBlockRows - 1)), b[2] - 1);
    const int lb = fast_div(pos, a.by_block);
    const int64_t slot = (int64_t)a.tables[b[0] + lb] * a.block_size + (pos - lb * a.block_size);
    arow[j] = (gptr<const T>)(a.pool) + slot * ROW + 8 * ((lane & 3) ^ swz(r));
    if (h == 0) {
      gptr<const T> const from = (gptr<const T>)(a.pool) + slot * ROW + L;
      gptr<T> const to = (gptr<T>)(a.rope) + ((int64_t)tile * kTileRows + r) * a.rope_size;
      for (int c = 8 * (lane & 3); c < a.rope_size; c += 32) store16(to + c, load16(from + c));
    }
  }
#pragma unroll
  for (int j = 0; j < LB; ++j) {
    const int r = 16 * (4 * j + wave) + (lane >> 2);
    gptr<const T> const w = 64 * j < NK ? (gptr<const T>)(a.key_up) + ((int64_t)h * NK + r) * L
                                        : (gptr<const T>)(a.value_up) + ((int64_t)h * NV + r - NK) * L;
    brow[j] = w + 8 * ((lane & 3) ^ swz_weights(r));
  }
  auto issue = [&](int k, char* ta, char* tb) {
#pragma unroll
    for (int j = 0; j < LA; ++j)
      __builtin_amdgcn_global_load_lds((lds_gptr)(arow[j] + k), (lds_lptr)(ta + (4 * j + wave) * 1024), 16, 0, 0);
#pragma unroll
    for (int j = 0; j < LB; ++j)
      __builtin_amdgcn_global_load_lds((lds_gptr)(brow[j] + k), (lds_lptr)(tb + (4 * j + wave) * 1024), 16, 0, 0);
  };
  const bool values = wave & 1;
  const int r0 = 64 * (wave >> 1);
  if (tid < kTileRows) lost[tid] = 0;  // (the steps' barriers come before its first use)
  // (Its own loop for each width: the barriers are the same.)
  auto run = [&]<int WIDTH>(int n0, void* out) __attribute__((always_inline)) {
    constexpr int RT = 4, NT = WIDTH / 16;
    f32x4 acc[NT][RT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[n][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int x_at = (r0 + l16) * 64 + 16 * (g ^ swz(l16));
    // (Row 4 i + e of instruction n is value 32 (n / 2) + 8 i + 4 (n % 2) + e.)
    const int wrow = 8 * (l16 >> 2) + (l16 & 3);
    const int w_at = (n0 + wrow) * 64 + 16 * (g ^ swz_weights(wrow));
    auto compute = [&](const char* ta, const char* tb) __attribute__((always_inline)) {
      uint4 xf[RT], wf[NT];
#pragma unroll
      for (int r = 0; r < RT; ++r) xf[r] = *reinterpret_cast<const uint4*>(ta + (1024 * r + x_at));
#pragma unroll
      for (int n = 0; n < NT; ++n) wf[n] = *reinterpret_cast<const uint4*>(tb + (2048 * (n / 2) + 256 * (n % 2) + w_at));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[n][r] = Mma<T>::qk(wf[n], xf[r], acc[n][r]);
    };
    char *const as[3] = {a0, a1, a2}, *const bs[3] = {b0, b1, b2};
    constexpr int STEPS = L / kStep;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      // The step's loads have landed (the next one's may be on their way), and every
      // wave has read the step before, whose place the step after the next takes.
      if (i + 1 < STEPS) {
        __builtin_amdgcn_s_waitcnt(0x0F70 | (LA + LB));
      } else {
        __builtin_amdgcn_s_waitcnt(0x0F70);
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (i + 2 < STEPS) issue((i + 2) * kStep, as[(i + 2) % 3], bs[(i + 2) % 3]);
      __builtin_amdgcn_sched_barrier(0);  // (or the loads would be put off to the step's end)
      compute(as[i % 3], bs[i % 3]);
    }
    auto place = [&](int r) -> gptr<T> {
      const int64_t key = (int64_t)tile * kTileRows + r0 + 16 * r + l16;
      return (gptr<T>)(out) + ((int64_t)h * a.keys + key) * WIDTH + 8 * g;
    };
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      uint32_t most = 0;
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = from_f32<T>(acc[n + e / 4][r][e % 4]);
        uint4 x;
        __builtin_memcpy(&x, v, 16);
        store16(place(r) + 16 * n, x);
        most = larger_bits(larger_bits(larger_bits(larger_bits(most, x.x), x.y), x.z), x.w);
      }
      if (!all_numbers<T>(most)) lost[r0 + 16 * r + l16] = 1;
    }
    // A row whose key or value T does not hold gets a key of NaN (by the threads that
    // wrote it): every score of it shows that it is not finite, so it reaches all queries
    // that see it and, its values taken out, no others (a zero weight would not hide an
    // infinite value).
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (values) return;
#pragma unroll 1
    for (int r = 0; r < RT; ++r) {
      if (!lost[r0 + 16 * r + l16]) continue;
#pragma unroll
      for (int n = 0; n < NT; n += 2) store16(place(r) + 16 * n, make_uint4(~0u, ~0u, ~0u, ~0u));
    }
  };
  __builtin_amdgcn_s_waitcnt(0x0F70);  // (the copies of the rotated keys: a step counts its own loads)
  issue(0, a0, b0);
  issue(kStep, a1, b1);
  if constexpr (NK == NV) {
    run.template operator()<NK>(values ? NK : 0, values ? a.value_out : a.key_out);
  } else if (values) {
    run.template operator()<NV>(NK, a.value_out);
  } else {
    run.template operator()<NK>(0, a.key_out);
  }
}

}  // namespace lvamd

using namespace lvamd;

extern "C" int lvamd_latent_heads(const void* x, int64_t x_token_stride, int64_t x_head_stride, const void* weights, void* y,
                                  int64_t y_token_stride, int64_t y_head_stride, const int32_t* x_rows, const int32_t* y_rows,
                                  int64_t num_rows, int32_t num_heads, int32_t k, int32_t n, int32_t dtype, lvamd_stream_t stream) {
  if (!latent_dtype(dtype) || k <= 0 || k % 64 != 0 || n <= 0 || n % 64 != 0) return LVAMD_ERR_UNSUPPORTED;
  if (num_rows < 0 || num_rows > 65535 * 16LL || num_heads <= 0) return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return LVAMD_OK;
  if (!x || !weights || !y || !rows16(x, {x_token_stride, x_head_stride}) || !rows16(weights, {}) || ((uintptr_t)y & 7u) ||
      y_token_stride % 4 != 0 || y_head_stride % 4 != 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  HeadsArgs a{x, x_token_stride, x_head_stride, weights, y, y_token_stride, y_head_stride, x_rows, y_rows,
              (int32_t)num_rows, k, n};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&]<typename T, int MT, int NT>() -> int {
    const int blocks = n / (16 * NT), waves = num_heads * blocks;
    hipLaunchKernelGGL((latent_heads_kernel<T, MT, NT>), dim3((unsigned)(waves + 3) / 4, (unsigned)((num_rows + 16 * MT - 1) / (16 * MT))), dim3(256), 0, s, a,
                       waves, FastDiv(blocks));
    return launch_status();
  };
  // 64 rows by 32 values a wave where enough waves are left (us, 16 x 16 against
  // 64 x 32): 16 heads, 128 to 512 values, 96 rows 4.9 / 5.4, 192 rows 8.4 / 5.7, 1536
  // rows 47 / 24; back to 128, 192 rows 9.6 / 13.4, 384 rows 13.3 / 16.7, 768 rows 24.4 /
  // 19.2; 128 heads, 96 rows 25.7 / 16.0 and 24.0 / 18.0.
  auto typed = [&]<typename T>() -> int {
    const bool wide = num_rows > 32 && (int64_t)num_heads * (n / 64) * ((num_rows + 63) / 64) >= 320;
    return wide ? launch.template operator()<T, 4, 2>() : launch.template operator()<T, 1, 1>();
  };
  return dtype == LVAMD_BF16 ? typed.operator()<__bf16>() : typed.operator()<_Float16>();
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
  auto launch = [&]<typename T, int L>() -> int {
    ExpandArgs a{.by_block = FastDiv(block_size), .by_heads = FastDiv(num_heads)};
    a.pool = pool;
    a.blocks = blocks;
    a.tables = tables;
    a.key_up = key_up;
    a.value_up = value_up;
    a.key_out = keys;
    a.value_out = values;
    a.rope = rope_keys;
    a.keys = (int64_t)tiles * kTileRows;
    a.heads = num_heads;
    a.tiles = tiles;
    a.block_size = block_size;
    a.rope_size = rope_size;
    auto with = [&]<int NK, int NV>() {
      hipLaunchKernelGGL((latent_expand_kernel<T, L, NK, NV>), dim3((unsigned)grid), dim3(256), 0, s, a);
    };
    if (nope_size == 64) {
      value_size == 64 ? with.template operator()<64, 64>() : with.template operator()<64, 128>();
    } else {
      value_size == 64 ? with.template operator()<128, 64>() : with.template operator()<128, 128>();
    }
    return launch_status();
  };
  auto sized = [&]<typename T>() -> int {
    switch (latent_size) {
      case 128: return launch.template operator()<T, 128>();
      case 256: return launch.template operator()<T, 256>();
      case 384: return launch.template operator()<T, 384>();
      default: return launch.template operator()<T, 512>();
    }
  };
  return dtype == LVAMD_BF16 ? sized.operator()<__bf16>() : sized.operator()<_Float16>();
}
