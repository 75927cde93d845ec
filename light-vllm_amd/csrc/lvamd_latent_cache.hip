// Rotary angles, and the movement of rows in a paged cache of latent vectors,
// on gfx950: append (with the rotation of the step's keys and queries),
// compact and block copy.  All are bound by HBM in long steps, by one launch
// in short ones.

#include "lvamd_latent.h"

namespace lvamd {

// ---------------------------------------------------------------------------
// Angles.  Pair i of a position p turns by p * f_i; the host gives f_i in turns
// (fp64).  p * f_i is formed and reduced to an eighth of a turn in fp64, where
// it is off by less than 2^-51 of its turns, the frequency's own roundings included
// (2^-31 of a turn at a million turns); the reduced angle r, |r| <= pi / 4, is an fp32 value (off by 2^-25 r)
// and sine and cosine are its Taylor sums to r^9 and r^10, whose next terms are
// below 2^-29 and 2^-33.  A thread per pair; 32760 tokens of 64 values take 4.6
// us, 64 of them 2.3; the host's call and its two allocations take 7.0 for either.
// ---------------------------------------------------------------------------
struct AnglesArgs {
  const void* positions;
  const double* turns;
  void* cosines;
  void* sines;
  int64_t count;  // tokens * half
  int32_t half;
  int32_t repeat;  // values per row: half, or twice half (each twice, as the half layout pairs them)
  FastDiv by_half;
  float magnitude;
};

template <typename T, typename I>
__global__ __launch_bounds__(256) void rotary_angles_kernel(const AnglesArgs a) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= a.count) return;
  const int t = fast_div((int)n, a.by_half), i = (int)n - t * a.half;
  const double x = (double)static_cast<const I*>(a.positions)[t] * a.turns[i];
  const double octs = __builtin_rint(4.0 * x);
  const float r = (float)((x - 0.25 * octs) * 6.283185307179586);
  // The quarter of a turn: octs modulo 4, exact in fp64.
  const int q = (int)(octs - 4.0 * __builtin_floor(0.25 * octs));
  const float z = r * r;
  const float s = r + r * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
  const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
  const float cq = q & 1 ? s : c, sq = q & 1 ? c : s;
  const T co = from_f32<T>((q == 1 || q == 2 ? -cq : cq) * a.magnitude);
  const T si = from_f32<T>((q >= 2 ? -sq : sq) * a.magnitude);
  const int64_t at = (int64_t)t * a.repeat + i;
  static_cast<T*>(a.cosines)[at] = co;
  static_cast<T*>(a.sines)[at] = si;
  if (a.repeat > a.half) {
    static_cast<T*>(a.cosines)[at + a.half] = co;
    static_cast<T*>(a.sines)[at + a.half] = si;
  }
}

// ---------------------------------------------------------------------------
// Append.  One thread per 16-byte chunk of a row's latent part, and per chunk
// (interleaved pairs), pair of chunks (half layout) or chunk (no rotation) of
// its key; then the same of every query head's rotated part.  The rotation is
// fp32, rounded once to T.  Entries whose slot or token is out of range are passed
// over.  A thread per chunk, for reads and writes of whole lines: 8190 tokens of
// 256 + 32 (10.5 MB in and out) take 4.2 us, 64 of 512 + 64 2.5; the host's call takes
// 5.5 for either.
// ---------------------------------------------------------------------------
struct LatentAppendArgs {
  const void* latent;
  const void* rope;
  int64_t latent_stride, rope_stride;
  void* pool;
  const int64_t* slots;
  const int64_t* sources;  // null: entry i is token i
  const float* cosines;    // [tokens][P / 2], or null
  const float* sines;
  int64_t angle_stride;
  const void* query;  // [tokens][heads][P], or null
  int64_t q_tok_stride, q_head_stride;
  void* rotated;  // [tokens][heads][P]
  int64_t entries, tokens, query_items;
  int32_t chunks;     // 16-byte chunks of the latent part
  int32_t rope_work;  // work items of a key or query
  int32_t heads, num_slots;
  FastDiv by_row, by_token, by_rope;  // / (chunks + rope_work), / (heads * rope_work), / rope_work
  int32_t row;                        // elements
};

enum class Layout { kNone, kInterleaved, kHalf };

// Work item w of a P-value vector: copied or turned by the token's angles.
template <typename T, Layout K>
__device__ __forceinline__ void turn(const T* src, T* dst, int w, int pairs, const float* cs, const float* sn) {
  if constexpr (K == Layout::kNone) {
    store16((gptr<T>)(dst + 8 * w), load16(src + 8 * w));
  } else if constexpr (K == Layout::kInterleaved) {
    store16((gptr<T>)(dst + 8 * w), turn_chunk<T>(load16(src + 8 * w), cs + 4 * w, sn + 4 * w));
  } else {
    uint4 lo = load16(src + 8 * w), hi = load16(src + 8 * w + pairs);
    turn_chunks<T>(lo, hi, cs + 8 * w, sn + 8 * w);
    store16((gptr<T>)(dst + 8 * w), lo);
    store16((gptr<T>)(dst + 8 * w + pairs), hi);
  }
}

template <typename T, Layout K>
__global__ __launch_bounds__(256) void latent_append_kernel(const LatentAppendArgs a, const int32_t pairs) {
  const int64_t row_items = a.entries * (a.chunks + a.rope_work);
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n < row_items) {
    const int e = fast_div((int)n, a.by_row), i = (int)n - e * (a.chunks + a.rope_work);
    const int64_t slot = a.slots[e];
    if (slot < 0 || slot >= a.num_slots) return;
    const int64_t t = a.sources ? a.sources[e] : e;
    if (t < 0 || t >= a.tokens) return;
    T* const row = static_cast<T*>(a.pool) + slot * a.row;
    if (i < a.chunks) {
      store16((gptr<T>)(row + 8 * i), load16(static_cast<const T*>(a.latent) + t * a.latent_stride + 8 * i));
    } else {
      turn<T, K>(static_cast<const T*>(a.rope) + t * a.rope_stride, row + 8 * a.chunks, i - a.chunks, pairs,
                 a.cosines + t * a.angle_stride, a.sines + t * a.angle_stride);
    }
  } else if (n - row_items < a.query_items) {
    const int m = (int)(n - row_items);
    const int t = fast_div(m, a.by_token), j = m - t * a.heads * a.rope_work;
    const int h = fast_div(j, a.by_rope), i = j - h * a.rope_work;
    turn<T, K>(static_cast<const T*>(a.query) + t * a.q_tok_stride + h * a.q_head_stride,
               static_cast<T*>(a.rotated) + ((int64_t)t * a.heads + h) * 2 * pairs, i, pairs,
               a.cosines + (int64_t)t * a.angle_stride, a.sines + (int64_t)t * a.angle_stride);
  }
}

// ---------------------------------------------------------------------------
// Rows (or whole blocks) of every layer's pool from places to places.
// ---------------------------------------------------------------------------
constexpr int kFewMoves = 32;
struct Moves {  // in the kernel arguments
  int64_t src[kFewMoves], dst[kFewMoves];
};
struct MoveArgs {
  const uint64_t* pools;
  int32_t num_layers;
  int64_t chunks;  // 16-byte chunks of a row
  const int64_t* src;
  const int64_t* dst;
  int64_t pairs;
  uint4* staged;  // [layer][pair][chunk]
};

// At most kFewMoves pairs: a thread reads its chunk of every source before it
// writes one, so sources may be destinations of other pairs.
template <int N>
__global__ __launch_bounds__(256) void latent_move_few_kernel(const uint64_t* __restrict__ pools, const int64_t items,
                                                              const int64_t chunks, const int32_t pairs, const Moves m) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= items) return;
  const int64_t layer = n / chunks, c = n - layer * chunks;
  gptr<uint4> const base = (gptr<uint4>)pools[layer] + c;
  uint4 held[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < pairs) held[i] = load16((gptr<const uint4>)(base + m.src[i] * chunks));
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < pairs) store16(base + m.dst[i] * chunks, held[i]);
}

// kGather: pool rows to the workspace; kScatter: from it; kCopy: straight (no
// source is a destination).
enum class Move { kGather, kScatter, kCopy };
template <Move K>
__global__ __launch_bounds__(256) void latent_move_kernel(const MoveArgs a) {
  const int64_t total = a.num_layers * a.pairs * a.chunks;
  for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < total; n += (int64_t)gridDim.x * 256) {
    const int64_t row = n / a.chunks, c = n - row * a.chunks;
    const int64_t layer = row / a.pairs, p = row - layer * a.pairs;
    gptr<uint4> const base = (gptr<uint4>)a.pools[layer] + c;
    const uint4 v = K == Move::kScatter ? load16((gptr<const uint4>)(a.staged + n))
                                        : load16((gptr<const uint4>)(base + a.src[p] * a.chunks));
    if constexpr (K == Move::kGather) {
      store16((gptr<uint4>)(a.staged + n), v);
    } else {
      store16(base + a.dst[p] * a.chunks, v);
    }
  }
}

}  // namespace lvamd

using namespace lvamd;

extern "C" {

int lvamd_rotary_angles(const void* positions, int32_t position_bytes, int64_t num_tokens, const double* turns,
                        int32_t half, float magnitude, void* cosines, void* sines, int32_t repeat, int32_t dtype,
                        lvamd_stream_t stream) {
  if ((position_bytes != 4 && position_bytes != 8) || num_tokens < 0 || half <= 0 || (repeat != 1 && repeat != 2) ||
      dtype_size(dtype) == 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return LVAMD_OK;
  if (!positions || !turns || !cosines || !sines) return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_tokens > 0x7fffffffLL / half) return LVAMD_ERR_INVALID_ARGUMENT;
  AnglesArgs a{positions, turns, cosines, sines, num_tokens * half, half, repeat * half, FastDiv(half), magnitude};
  const dim3 grid((unsigned)((a.count + 255) / 256));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&]<typename T>() -> int {
    if (position_bytes == 8) {
      hipLaunchKernelGGL((rotary_angles_kernel<T, int64_t>), grid, dim3(256), 0, s, a);
    } else {
      hipLaunchKernelGGL((rotary_angles_kernel<T, int32_t>), grid, dim3(256), 0, s, a);
    }
    return launch_status();
  };
  switch (dtype) {
    case LVAMD_F32: return launch.operator()<float>();
    case LVAMD_F16: return launch.operator()<_Float16>();
    default: return launch.operator()<__bf16>();
  }
}

int lvamd_latent_append(const void* latent, int64_t latent_token_stride, const void* rope_key,
                        int64_t rope_key_token_stride, void* pool, int64_t num_slots, const int64_t* slots,
                        const int64_t* sources, int64_t num_entries, const float* cosines, const float* sines,
                        int64_t angle_token_stride, int32_t interleaved, const void* query_rope,
                        int64_t query_token_stride, int64_t query_head_stride, void* rotated, int64_t num_tokens,
                        int32_t num_heads, int32_t latent_size, int32_t rope_size, int32_t dtype,
                        lvamd_stream_t stream) {
  if (!latent_sizes(latent_size, rope_size) || !latent_dtype(dtype)) return LVAMD_ERR_UNSUPPORTED;
  if (num_entries < 0 || num_tokens < 0 || num_slots <= 0 || num_slots > 0x7fffffffLL ||
      (cosines == nullptr) != (sines == nullptr) ||
      (query_rope && (!rotated || !cosines || num_heads <= 0)))
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_entries > 0 && (!latent || !rope_key || !pool || !slots || !rows16(pool, {}) ||
                          !rows16(latent, {latent_token_stride}) || !rows16(rope_key, {rope_key_token_stride})))
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (query_rope && (!rows16(query_rope, {query_token_stride, query_head_stride}) || !rows16(rotated, {})))
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (cosines && (((uintptr_t)cosines & 15u) || ((uintptr_t)sines & 15u) || angle_token_stride % 4 != 0))
    return LVAMD_ERR_INVALID_ARGUMENT;
  const Layout layout = !cosines ? Layout::kNone : interleaved ? Layout::kInterleaved : Layout::kHalf;
  const int work = layout == Layout::kHalf ? rope_size / 16 : rope_size / 8;
  const int heads = query_rope ? num_heads : 1;
  if (num_entries > 0x3fffffffLL / (latent_size / 8 + work) || num_tokens > 0x3fffffffLL / ((int64_t)heads * work))
    return LVAMD_ERR_INVALID_ARGUMENT;
  LatentAppendArgs a{.by_row = FastDiv(latent_size / 8 + work), .by_token = FastDiv(heads * work), .by_rope = FastDiv(work)};
  a.latent = latent;
  a.rope = rope_key;
  a.latent_stride = latent_token_stride;
  a.rope_stride = rope_key_token_stride;
  a.pool = pool;
  a.slots = slots;
  a.sources = sources;
  a.cosines = cosines;
  a.sines = sines;
  a.angle_stride = angle_token_stride;
  a.query = query_rope;
  a.q_tok_stride = query_token_stride;
  a.q_head_stride = query_head_stride;
  a.rotated = rotated;
  a.entries = num_entries;
  a.tokens = num_tokens;
  a.query_items = query_rope ? num_tokens * heads * work : 0;
  a.chunks = latent_size / 8;
  a.rope_work = work;
  a.heads = heads;
  a.num_slots = (int32_t)num_slots;
  a.row = latent_size + rope_size;
  const int64_t items = num_entries * (a.chunks + work) + a.query_items;
  if (items == 0) return LVAMD_OK;
  const dim3 grid((unsigned)((items + 255) / 256));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&]<typename T>() -> int {
    switch (layout) {
      case Layout::kNone: hipLaunchKernelGGL((latent_append_kernel<T, Layout::kNone>), grid, dim3(256), 0, s, a, rope_size / 2); break;
      case Layout::kInterleaved:
        hipLaunchKernelGGL((latent_append_kernel<T, Layout::kInterleaved>), grid, dim3(256), 0, s, a, rope_size / 2);
        break;
      default: hipLaunchKernelGGL((latent_append_kernel<T, Layout::kHalf>), grid, dim3(256), 0, s, a, rope_size / 2);
    }
    return launch_status();
  };
  return dtype == LVAMD_BF16 ? launch.operator()<__bf16>() : launch.operator()<_Float16>();
}

int64_t lvamd_latent_move_few_pairs(void) { return kFewMoves; }

int lvamd_latent_move_few(const uint64_t* pools, int32_t num_layers, int64_t row_bytes, const int64_t* src,
                          const int64_t* dst, int64_t num_pairs, lvamd_stream_t stream) {
  if (num_layers <= 0 || row_bytes <= 0 || row_bytes % 16 != 0 || num_pairs < 0 || num_pairs > kFewMoves)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_pairs == 0) return LVAMD_OK;
  if (!pools || !src || !dst) return LVAMD_ERR_INVALID_ARGUMENT;
  Moves m{};
  for (int64_t i = 0; i < num_pairs; ++i) {
    m.src[i] = src[i];
    m.dst[i] = dst[i];
  }
  const int64_t chunks = row_bytes / 16, items = num_layers * chunks;
  if (items > 0x7fffffffLL) return LVAMD_ERR_INVALID_ARGUMENT;
  const dim3 grid((unsigned)((items + 255) / 256));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (num_pairs <= 8) {
    hipLaunchKernelGGL(latent_move_few_kernel<8>, grid, dim3(256), 0, s, pools, items, chunks, (int32_t)num_pairs, m);
  } else {
    hipLaunchKernelGGL(latent_move_few_kernel<32>, grid, dim3(256), 0, s, pools, items, chunks, (int32_t)num_pairs, m);
  }
  return launch_status();
}

int64_t lvamd_latent_move_workspace_size(int64_t num_pairs, int32_t num_layers, int64_t row_bytes) {
  return num_pairs <= 0 || num_layers <= 0 || row_bytes <= 0 ? 0 : num_pairs * num_layers * row_bytes;
}

int lvamd_latent_move(const uint64_t* pools, int32_t num_layers, int64_t row_bytes, const int64_t* src,
                      const int64_t* dst, int64_t num_pairs, void* workspace, int64_t workspace_bytes,
                      lvamd_stream_t stream) {
  if (num_layers <= 0 || row_bytes <= 0 || row_bytes % 16 != 0 || num_pairs < 0) return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_pairs == 0) return LVAMD_OK;
  if (!pools || !src || !dst) return LVAMD_ERR_INVALID_ARGUMENT;
  if (workspace && (((uintptr_t)workspace & 15u) ||
                    workspace_bytes < lvamd_latent_move_workspace_size(num_pairs, num_layers, row_bytes)))
    return LVAMD_ERR_WORKSPACE;
  MoveArgs a{pools, num_layers, row_bytes / 16, src, dst, num_pairs, static_cast<uint4*>(workspace)};
  const int64_t blocks = (num_layers * num_pairs * a.chunks + 255) / 256;
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!workspace) {
    hipLaunchKernelGGL(latent_move_kernel<Move::kCopy>, grid, dim3(256), 0, s, a);
    return launch_status();
  }
  hipLaunchKernelGGL(latent_move_kernel<Move::kGather>, grid, dim3(256), 0, s, a);
  if (const int status = launch_status(); status != LVAMD_OK) return status;
  hipLaunchKernelGGL(latent_move_kernel<Move::kScatter>, grid, dim3(256), 0, s, a);
  return launch_status();
}

}  // extern "C"
