// Writing the 8-bit paged cache on gfx950: the quantising append and the
// compact of accepted rows.
//
// Codes are e4m3, [block][offset][kv head][D] as in the 16-bit cache; a block
// holds one scale per kv head, 2^e with e the smallest exponent that brings
// the largest magnitude of its rows within 448 (lvamd_q8.h).

#include <algorithm>
#include <cmath>

#include "lvamd_q8.h"

namespace lvamd {

// Largest of a wave's 64 values (not negative).
__device__ __forceinline__ float wave_max(float v) {
  v = row_max4(v);  // across the four 16-lane rows
#pragma unroll
  for (int d = 8; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// Every store that this wave has issued is done (same-wave stores to one
// address then land in program order).
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---------------------------------------------------------------------------
// Append.  A run is the tokens of one call that go to one block; they are
// consecutive in the slot list.  One wave per (run, K or V, kv head):
//   amax over the run's rows, then scale = 2^e(amax) for a block that starts
//   anew (its offset 0 is in the run), else max(old, 2^e(amax)); if that is
//   above the old scale, the block's rows are re-scaled by old / new; then the
//   run's codes and the scale.
//
// The waves find the runs themselves: a workgroup looks at a window of 64
// entries of the list, one per lane, and a ballot marks those whose
// predecessor is in another block.  The window's (run, unit) tasks go round
// robin over the waves of gridDim.y workgroups, enough of them that a window
// of single tokens (64 runs) has few tasks per wave; a prompt's window has few
// runs and most of its workgroups exit at once.  (With a workgroup per entry,
// the runs of a prompt's blocks of 16 all began on workgroups of one XCD: 2,048
// tokens 17 us against 7 for the same tokens in 128 requests.)
//
// HBM-bound for prompts (each row read once and held in registers, up to
// kHeld passes of 64 lanes; longer runs read their later rows again), a chain
// of three round trips (slots, rows and old scale, stores) for single tokens.
// 4 kv heads, D = 128, bf16, blocks of 16: 64 tokens of 64 requests 4.7 us, 8,190
// of 16 prompts 8.5 us (25 MB, 3.0 TB/s).
// ---------------------------------------------------------------------------
struct Q8AppendArgs {
  const char* key;
  const char* value;
  int64_t key_tok_bytes, key_head_bytes;
  int64_t value_tok_bytes, value_head_bytes;
  uint8_t* key_pool;
  uint8_t* value_pool;
  float* key_scales;
  float* value_scales;
  const int64_t* sources;  // token of each slot, or null: token i
  int64_t num_slots;
  int32_t num_kv_heads;
  int32_t head_size;
  int32_t block_size;
  FastDiv by_block, by_lanes, by_units;  // / block_size, / lanes per row, / (K and V, kv heads)
};

constexpr int kHeld = 4;  // passes of rows that stay in registers
constexpr int kAppendWaves = 4;

template <typename T>
__device__ __forceinline__ void append_run(const Q8AppendArgs& a, const int64_t* __restrict__ slots, int lane,
                                           int64_t base, uint64_t leads, uint64_t ends, uint64_t zeros, int my_block,
                                           int task) {
  const int bs = a.block_size;
  const int run = fast_div(task, a.by_units);
  const int unit = task - run * 2 * a.num_kv_heads;
  // The run's first entry, the run-th of the window's.
  for (int i = 0; i < run; ++i) leads &= leads - 1;
  const int l = __builtin_ctzll(leads);
  const int64_t i0 = base + l;
  const int block = __builtin_amdgcn_readlane(my_block, l);
  // Its length, and whether it holds the block's offset 0.
  const uint64_t after = l < 63 ? ends >> (l + 1) : 0;
  int n = after ? __builtin_ctzll(after) + 1 : 64 - l;
  bool fresh = ((zeros >> l) & (n < 64 ? ((uint64_t)1 << n) - 1 : ~(uint64_t)0)) != 0;
  if (l + n == 64) {
    // On into the next windows.
    for (;; n += 64) {
      const int64_t i = i0 + n + lane;
      const int64_t s = i < a.num_slots ? slots[i] : -1;
      const bool in = s >= 0 && fast_div((int)s, a.by_block) == block;
      const uint64_t out = ~__ballot(in);
      const int len = out == 0 ? 64 : __builtin_ctzll(out);
      fresh |= __any(in && lane < len && (int)s == block * bs);
      if (len < 64) {
        n += len;
        break;
      }
    }
  }
  const bool is_v = unit >= a.num_kv_heads;
  const int h = is_v ? unit - a.num_kv_heads : unit;
  const char* src = (is_v ? a.value + h * a.value_head_bytes : a.key + h * a.key_head_bytes);
  const int64_t tok_bytes = is_v ? a.value_tok_bytes : a.key_tok_bytes;
  float* const scale_at = (is_v ? a.value_scales : a.key_scales) + (int64_t)block * a.num_kv_heads + h;
  const int64_t row_bytes = (int64_t)a.num_kv_heads * a.head_size;
  uint8_t* const pool = (is_v ? a.value_pool : a.key_pool) + (int64_t)h * a.head_size;
  const float old = fresh ? 0.f : *scale_at;

  // Eight elements per lane, lanes-per-row lanes to a row, R rows a pass.
  const int lpr = a.head_size / 8;
  const int R = fast_div(64, a.by_lanes);
  const int r0 = fast_div(lane, a.by_lanes);
  const int c = lane - r0 * lpr;
  auto load = [&](int r) -> uint4 {
    const int64_t i = i0 + r;
    const int64_t t = a.sources ? a.sources[i] : i;
    return load16(reinterpret_cast<const T*>(src + t * tok_bytes) + 8 * c);
  };
  auto row_of = [&](int pass) -> int { return r0 < R ? pass * R + r0 : n; };  // n: none
  uint4 held[kHeld];
  int64_t to[kHeld];
  float amax = 0.f;
  auto largest = [&](uint4 v) {
    T x[8];
    __builtin_memcpy(x, &v, 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m = __builtin_fabsf(to_f32(x[e]));
      amax = fmaxf(amax, m < INFINITY ? m : 0.f);  // (NaN compares false)
    }
  };
#pragma unroll
  for (int p = 0; p < kHeld; ++p) {
    held[p] = row_of(p) < n ? load(row_of(p)) : zero_u4();
    to[p] = row_of(p) < n ? slots[i0 + row_of(p)] : 0;
  }
#pragma unroll
  for (int p = 0; p < kHeld; ++p) largest(held[p]);
  for (int p = kHeld; p * R < n; ++p)
    if (row_of(p) < n) largest(load(row_of(p)));
  amax = wave_max(amax);
  const float scale = fmaxf(old, q8_scale(amax));
  const float inverse = q8_inverse(scale);

  if (!fresh && scale > old) {
    // The rows that the block holds, at the new scale.
    const float ratio = old * inverse;
    for (int r = r0; r < bs; r += R) {
      if (r0 >= R) break;
      uint2* const at = reinterpret_cast<uint2*>(pool + ((int64_t)block * bs + r) * row_bytes + 8 * c);
      const uint2 w = *at;
      *at = make_uint2(q8_rescale4(w.x, ratio), q8_rescale4(w.y, ratio));
    }
    stores_done();
  }
  auto store = [&](int64_t s, uint4 v) {
    T x[8];
    __builtin_memcpy(x, &v, 16);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = q8_scaled<T>(to_f32(x[e]), inverse);
    *reinterpret_cast<uint2*>(pool + s * row_bytes + 8 * c) =
        make_uint2(q8_pack4(f[0], f[1], f[2], f[3]), q8_pack4(f[4], f[5], f[6], f[7]));
  };
#pragma unroll
  for (int p = 0; p < kHeld; ++p)
    if (row_of(p) < n) store(to[p], held[p]);
  for (int p = kHeld; p * R < n; ++p)
    if (row_of(p) < n) store(slots[i0 + row_of(p)], load(row_of(p)));
  if (lane == 0) *scale_at = scale;
}

template <typename T>
__global__ __launch_bounds__(64 * kAppendWaves) void q8_append_kernel(const int64_t* __restrict__ slots,
                                                                      const Q8AppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int bs = a.block_size;
  const int units = 2 * a.num_kv_heads;
  const int64_t base = (int64_t)blockIdx.x * 64;
  auto block_of = [&](int64_t s) -> int { return s < 0 ? -1 : fast_div((int)s, a.by_block); };
  // The window: this lane's entry, which entries begin a run, which end one.
  const int64_t mine = base + lane < a.num_slots ? slots[base + lane] : -1;
  const int64_t before = base + lane > 0 && base + lane <= a.num_slots ? slots[base + lane - 1] : -1;
  const int my_block = block_of(mine);
  const uint64_t leads = __ballot(mine >= 0 && block_of(before) != my_block);
  const uint64_t ends = leads | __ballot(mine < 0);
  const uint64_t zeros = __ballot(mine >= 0 && (int)mine == my_block * bs);  // offset 0 of a block
  const int tasks = __popcll(leads) * units;
  for (int task = blockIdx.y * kAppendWaves + wave; task < tasks; task += gridDim.y * kAppendWaves)
    append_run<T>(a, slots, lane, base, leads, ends, zeros, my_block, task);
}

// ---------------------------------------------------------------------------
// Compact of accepted rows that the kernel after this one does not take (more
// pairs, a request of more than 32, tables that share blocks), two launches: the
// first copies every pair's row (codes and its block's scale, for every layer, K
// and V) to the workspace, the second writes them.  Pairs come grouped by destination block; one wave
// per (destination block, layer, K or V, kv head) takes the larger of the
// block's scale and those its rows come with, re-scales the block's rows if
// that is above its own, then writes the moved rows at it.  (Every source is
// read before any block changes: a source's block may be another's
// destination.)  Latency-bound: 145 rows of 128 requests, 12 layers, 2 kv heads,
// D = 128 (1.8 MB read and written) take 3.1 + 4.4 us.
// ---------------------------------------------------------------------------
struct Q8CompactArgs {
  const uint64_t* layer_keys;
  const uint64_t* layer_values;
  int64_t scale_offset;  // bytes from a pool's base to its scales
  const int64_t* src;
  const int64_t* dst;
  uint8_t* rows;         // workspace: [pairs][layers * 2][kv heads][D]
  float* row_scales;     // workspace: [pairs][layers * 2][kv heads]
  int32_t num_layers, num_kv_heads, head_size, block_size;
  FastDiv by_block, by_heads, by_chunks, by_sides;
};

constexpr int kCompactThreads = 256;

// One thread per (pair, layer side, kv head, 16-byte chunk).
__global__ __launch_bounds__(kCompactThreads) void q8_gather_kernel(const int64_t total, const Q8CompactArgs a) {
  const int64_t id = (int64_t)blockIdx.x * kCompactThreads + threadIdx.x;
  if (id >= total) return;
  const int chunks = a.head_size / 16;
  const int row = fast_div((int)id, a.by_chunks);  // (pair, layer side, kv head)
  const int c = (int)id - row * chunks;
  const int ps = fast_div(row, a.by_heads);
  const int h = row - ps * a.num_kv_heads;
  const int sides = 2 * a.num_layers;
  const int pair = fast_div(ps, a.by_sides);
  const int side = ps - pair * sides;
  const char* base = reinterpret_cast<const char*>(side & 1 ? a.layer_values[side >> 1] : a.layer_keys[side >> 1]);
  const int64_t s = a.src[pair];
  const uint4 v = load16(reinterpret_cast<const uint8_t*>(base) + (s * a.num_kv_heads + h) * a.head_size + 16 * c);
  *reinterpret_cast<uint4*>(a.rows + (int64_t)row * a.head_size + 16 * c) = v;
  if (c == 0) {
    const float* scales = reinterpret_cast<const float*>(base + a.scale_offset);
    a.row_scales[row] = scales[(int64_t)fast_div((int)s, a.by_block) * a.num_kv_heads + h];
  }
}

// Grid: (destination groups, kv heads x layer sides / waves).
__global__ __launch_bounds__(64 * kAppendWaves) void q8_scatter_kernel(const int64_t* __restrict__ starts,
                                                                       const Q8CompactArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int unit = blockIdx.y * kAppendWaves + wave;  // (layer side, kv head)
  const int sides = 2 * a.num_layers;
  if (unit >= sides * a.num_kv_heads) return;
  const int side = fast_div(unit, a.by_heads);
  const int h = unit - side * a.num_kv_heads;
  const int64_t first = starts[blockIdx.x], last = starts[blockIdx.x + 1];
  char* base = reinterpret_cast<char*>(side & 1 ? a.layer_values[side >> 1] : a.layer_keys[side >> 1]);
  const int block = fast_div((int)a.dst[first], a.by_block);
  float* const scale_at = reinterpret_cast<float*>(base + a.scale_offset) + (int64_t)block * a.num_kv_heads + h;
  auto row = [&](int64_t pair) { return (pair * sides + side) * a.num_kv_heads + h; };
  const float old = *scale_at;
  float most = 0.f;
  for (int64_t p = first + lane; p < last; p += 64) most = fmaxf(most, a.row_scales[row(p)]);
  const float scale = fmaxf(old, wave_max(most));
  const int chunks = a.head_size / 16;
  const int R = fast_div(64, a.by_chunks);
  const int r0 = fast_div(lane, a.by_chunks);
  const int c = lane - r0 * chunks;
  if (r0 >= R) return;
  const int64_t row_bytes = (int64_t)a.num_kv_heads * a.head_size;
  uint8_t* const pool = reinterpret_cast<uint8_t*>(base) + (int64_t)h * a.head_size + 16 * c;
  const float inverse = q8_inverse(scale);
  if (scale > old) {
    const float ratio = old * inverse;
    for (int r = r0; r < a.block_size; r += R) {
      uint4* const at = reinterpret_cast<uint4*>(pool + ((int64_t)block * a.block_size + r) * row_bytes);
      *at = q8_rescale16(*at, ratio);
    }
    stores_done();
    if (lane == 0) *scale_at = scale;
  }
  for (int64_t p = first + r0; p < last; p += R) {
    const float from = a.row_scales[row(p)];
    uint4 w = load16(a.rows + row(p) * a.head_size + 16 * c);
    if (from < scale) w = q8_rescale16(w, from * inverse);
    *reinterpret_cast<uint4*>(pool + a.dst[p] * row_bytes) = w;
  }
}

// ---------------------------------------------------------------------------
// Compact of a step's accepted drafts: one launch, no workspace, the pairs in the
// kernel's arguments, cut into chunks of at most kFewPairs that do not touch each
// other's blocks.  A wave owns one kv head of one layer's K or V and one chunk, so
// it can hold all the chunk's rows of it in registers (kFewPairs rows of D bytes,
// 16 per lane and pass) before it writes any.  Lane i has pair i's slots and
// scales; a segmented scan gives each destination block's new scale.  A chain of
// three round trips (scales and rows, re-scaled rows, stores): 3.4 us for one
// row of 12 layers, 4.2 for 145 of 128 requests, against 7.5 in two launches
// behind an upload (a call of 128 requests 28.5 us against 41).
// ---------------------------------------------------------------------------
constexpr int kFewPairs = 32;     // of a chunk
constexpr int kCallPairs = 384;   // of a call (3 KB of arguments)
constexpr int kCallChunks = 32;
// (A single chunk travels in arguments of its own size: the larger ones cost the
// launch 1.2 us of host time, 7.7 us against 6.9 a call of one request.)
template <int PAIRS, int CHUNKS>
struct Q8FewArgs {
  const uint64_t* layer_keys;
  const uint64_t* layer_values;
  int64_t scale_offset;
  int32_t num_kv_heads, head_size, block_size;
  FastDiv by_block, by_heads, by_chunks;
  int32_t starts[CHUNKS + 1];  // each chunk's first pair
  int32_t src[PAIRS], dst[PAIRS];
};

// Grid: (layer sides x kv heads, chunks).

template <int PAIRS, int CHUNKS>
__global__ __launch_bounds__(64) void q8_compact_few_kernel(const Q8FewArgs<PAIRS, CHUNKS> a) {
  constexpr int kPasses = kFewPairs * 16 / 64;  // head size 256
  const int lane = threadIdx.x & 63;
  const int side = fast_div((int)blockIdx.x, a.by_heads);
  const int h = (int)blockIdx.x - side * a.num_kv_heads;
  const int first = a.starts[blockIdx.y], n = a.starts[blockIdx.y + 1] - first;
  char* base = reinterpret_cast<char*>(side & 1 ? a.layer_values[side >> 1] : a.layer_keys[side >> 1]);
  float* const scales = reinterpret_cast<float*>(base + a.scale_offset) + h;
  const int64_t row_bytes = (int64_t)a.num_kv_heads * a.head_size;
  uint8_t* const pool = reinterpret_cast<uint8_t*>(base) + (int64_t)h * a.head_size;
  const int pair = lane < n ? lane : n - 1;  // (lanes past the pairs repeat the last)
  const int from = a.src[first + pair], to = a.dst[first + pair];
  const int to_block = fast_div(to, a.by_block);
  const float from_scale = scales[(int64_t)fast_div(from, a.by_block) * a.num_kv_heads];
  const float old = scales[(int64_t)to_block * a.num_kv_heads];
  const int chunks = a.head_size / 16;
  uint4 rows[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = fast_div(lane + 64 * p, a.by_chunks);
    const int c = lane + 64 * p - row * chunks;
    const int slot = __shfl(from, row & 31);
    rows[p] = row < n ? load16(pool + slot * row_bytes + 16 * c) : zero_u4();
  }
  // Groups of one destination block; the largest scale of a group is at its
  // last lane.
  const int before = __shfl_up(to_block, 1);
  const uint64_t leads = __ballot(lane < n && (lane == 0 || before != to_block));
  const int group = __popcll(leads & ((2ull << lane) - 1));
  float most = fmaxf(from_scale, old);
#pragma unroll
  for (int d = 1; d < kFewPairs; d <<= 1) {
    const float other = __shfl_up(most, d);
    const int other_group = __shfl_up(group, d);
    if (lane >= d && other_group == group) most = fmaxf(most, other);
  }
  const uint64_t after = lane < 63 ? leads >> (lane + 1) : 0;
  const int last = after ? lane + __builtin_ctzll(after) : n - 1;
  const float scale = __shfl(most, last);
  const bool grew = ((leads >> lane) & 1) && scale > old;
  stores_done();  // (every row is loaded before any is written)
  for (uint64_t todo = __ballot(grew); todo; todo &= todo - 1) {
    const int l = __builtin_ctzll(todo);
    const int64_t block = __builtin_amdgcn_readlane(to_block, l);
    const float ratio = __shfl(old, l) * q8_inverse(__shfl(scale, l));
    for (int i = lane; i < a.block_size * chunks; i += 64) {
      const int r = fast_div(i, a.by_chunks);
      uint4* const at = reinterpret_cast<uint4*>(pool + (block * a.block_size + r) * row_bytes + 16 * (i - r * chunks));
      *at = q8_rescale16(*at, ratio);
    }
  }
  stores_done();
  if (grew) scales[(int64_t)to_block * a.num_kv_heads] = scale;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = fast_div(lane + 64 * p, a.by_chunks);
    const int c = lane + 64 * p - row * chunks;
    const int slot = __shfl(to, row & 31);
    const float ratio = __shfl(from_scale, row & 31) * q8_inverse(__shfl(scale, row & 31));
    if (row < n) {
      uint4 w = rows[p];
      if (ratio < 1.f) w = q8_rescale16(w, ratio);
      *reinterpret_cast<uint4*>(pool + slot * row_bytes + 16 * c) = w;
    }
  }
}

static bool aligned_to(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace lvamd

using namespace lvamd;

extern "C" int lvamd_kv_append_q8(const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                                  int64_t value_token_stride, int64_t value_head_stride, void* key_pool,
                                  float* key_scales, void* value_pool, float* value_scales, const int64_t* slots,
                                  const int64_t* sources, int64_t num_slots, int32_t num_kv_heads, int32_t head_size,
                                  int32_t block_size, int32_t dtype, lvamd_stream_t stream) {
  if ((dtype != LVAMD_BF16 && dtype != LVAMD_F16) || !q8_head_size(head_size)) return LVAMD_ERR_UNSUPPORTED;
  if (num_slots < 0 || num_kv_heads <= 0 || num_kv_heads > 32768 || block_size <= 0) return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_slots == 0) return LVAMD_OK;
  if (!key || !value || !key_pool || !key_scales || !value_pool || !value_scales || !slots || num_slots > 0x7fffffffLL)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (!aligned_to(key, 16) || !aligned_to(value, 16) || !aligned_to(key_pool, 16) || !aligned_to(value_pool, 16) ||
      !aligned_to(key_scales, 4) || !aligned_to(value_scales, 4) || key_token_stride % 8 != 0 ||
      key_head_stride % 8 != 0 || value_token_stride % 8 != 0 || value_head_stride % 8 != 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  Q8AppendArgs a{.by_block = FastDiv(block_size), .by_lanes = FastDiv(head_size / 8),
                 .by_units = FastDiv(2 * num_kv_heads)};
  a.key = static_cast<const char*>(key);
  a.value = static_cast<const char*>(value);
  a.key_tok_bytes = key_token_stride * 2;
  a.key_head_bytes = key_head_stride * 2;
  a.value_tok_bytes = value_token_stride * 2;
  a.value_head_bytes = value_head_stride * 2;
  a.key_pool = static_cast<uint8_t*>(key_pool);
  a.value_pool = static_cast<uint8_t*>(value_pool);
  a.key_scales = key_scales;
  a.value_scales = value_scales;
  a.sources = sources;
  a.num_slots = num_slots;
  a.num_kv_heads = num_kv_heads;
  a.head_size = head_size;
  a.block_size = block_size;
  // Workgroups per window: about 4,096 in all, at most one wave per task of a
  // window of 64 runs.
  const int64_t windows = (num_slots + 63) / 64;
  const int64_t most = (64 * 2 * (int64_t)num_kv_heads + kAppendWaves - 1) / kAppendWaves;
  const int64_t share = std::max<int64_t>(1, std::min<int64_t>(4096 / windows, most));
  const dim3 grid((unsigned)windows, (unsigned)share);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == LVAMD_BF16)
    hipLaunchKernelGGL((q8_append_kernel<__bf16>), grid, dim3(64 * kAppendWaves), 0, s, slots, a);
  else
    hipLaunchKernelGGL((q8_append_kernel<_Float16>), grid, dim3(64 * kAppendWaves), 0, s, slots, a);
  return launch_status();
}

extern "C" int64_t lvamd_kv_compact_q8_workspace_size(int64_t num_pairs, int32_t num_layers, int32_t num_kv_heads,
                                                      int32_t head_size) {
  if (num_pairs <= 0 || num_layers <= 0 || num_kv_heads <= 0 || head_size <= 0) return 0;
  return num_pairs * num_layers * 2 * num_kv_heads * ((int64_t)head_size + 4);
}

extern "C" int lvamd_kv_compact_q8(const uint64_t* layer_key_ptrs, const uint64_t* layer_value_ptrs, int32_t num_layers,
                                   int32_t num_kv_heads, int32_t head_size, int32_t block_size, int64_t scale_offset,
                                   const int64_t* src_slots, const int64_t* dst_slots, int64_t num_pairs,
                                   const int64_t* block_starts, int64_t num_dst_blocks, void* workspace,
                                   int64_t workspace_bytes, lvamd_stream_t stream) {
  if (!q8_head_size(head_size)) return LVAMD_ERR_UNSUPPORTED;
  if (num_pairs < 0 || num_layers <= 0 || num_kv_heads <= 0 || block_size <= 0 || num_dst_blocks < 0 ||
      num_dst_blocks > num_pairs || (num_pairs > 0) != (num_dst_blocks > 0) || scale_offset < 0 || scale_offset % 4 != 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_pairs == 0) return LVAMD_OK;
  if (!layer_key_ptrs || !layer_value_ptrs || !src_slots || !dst_slots || !block_starts) return LVAMD_ERR_INVALID_ARGUMENT;
  const int64_t units = (int64_t)num_layers * 2 * num_kv_heads;
  const int64_t chunks = num_pairs * units * (head_size / 16);
  const int64_t groups_y = (units + kAppendWaves - 1) / kAppendWaves;
  // 32-bit indexes in the kernels, and the grid's limits.
  if (units > 0x7fffffffLL / 64 || num_pairs > 0x7fffffffLL || chunks > 0x7fffffffLL || groups_y > 65535)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (!workspace || !aligned_to(workspace, 16) ||
      workspace_bytes < lvamd_kv_compact_q8_workspace_size(num_pairs, num_layers, num_kv_heads, head_size))
    return LVAMD_ERR_WORKSPACE;
  Q8CompactArgs a{.by_block = FastDiv(block_size), .by_heads = FastDiv(num_kv_heads), .by_chunks = FastDiv(head_size / 16),
                  .by_sides = FastDiv(2 * num_layers)};
  a.layer_keys = layer_key_ptrs;
  a.layer_values = layer_value_ptrs;
  a.scale_offset = scale_offset;
  a.src = src_slots;
  a.dst = dst_slots;
  a.rows = static_cast<uint8_t*>(workspace);
  a.row_scales = reinterpret_cast<float*>(a.rows + num_pairs * units * head_size);
  a.num_layers = num_layers;
  a.num_kv_heads = num_kv_heads;
  a.head_size = head_size;
  a.block_size = block_size;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(q8_gather_kernel, dim3((unsigned)((chunks + kCompactThreads - 1) / kCompactThreads)),
                     dim3(kCompactThreads), 0, s, chunks, a);
  const int status = launch_status();
  if (status != LVAMD_OK) return status;
  hipLaunchKernelGGL(q8_scatter_kernel, dim3((unsigned)num_dst_blocks, (unsigned)groups_y), dim3(64 * kAppendWaves), 0, s,
                     block_starts, a);
  return launch_status();
}

extern "C" int64_t lvamd_kv_compact_q8_few_pairs(void) { return kFewPairs; }
extern "C" int64_t lvamd_kv_compact_q8_few_call_pairs(void) { return kCallPairs; }

extern "C" int lvamd_kv_compact_q8_few(const uint64_t* layer_key_ptrs, const uint64_t* layer_value_ptrs,
                                       int32_t num_layers, int32_t num_kv_heads, int32_t head_size, int32_t block_size,
                                       int64_t scale_offset, const int64_t* src_slots, const int64_t* dst_slots,
                                       int64_t num_pairs, const int32_t* chunk_starts, int32_t num_chunks,
                                       lvamd_stream_t stream) {
  if (!q8_head_size(head_size)) return LVAMD_ERR_UNSUPPORTED;
  if (num_pairs < 0 || num_pairs > kCallPairs || num_chunks < 0 || num_chunks > kCallChunks || num_layers <= 0 ||
      num_kv_heads <= 0 || block_size <= 0 || scale_offset < 0 || scale_offset % 4 != 0 ||
      (int64_t)block_size * (head_size / 16) > 0x7fffffffLL || (int64_t)num_layers * 2 * num_kv_heads > 0x7fffffffLL)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_pairs == 0) return LVAMD_OK;
  if (!layer_key_ptrs || !layer_value_ptrs || !src_slots || !dst_slots || !chunk_starts || num_chunks == 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  for (int c = 0; c < num_chunks; ++c) {
    const int64_t pairs = (int64_t)chunk_starts[c + 1] - chunk_starts[c];
    if (pairs < 1 || pairs > kFewPairs) return LVAMD_ERR_INVALID_ARGUMENT;
  }
  if (chunk_starts[0] != 0 || chunk_starts[num_chunks] != num_pairs) return LVAMD_ERR_INVALID_ARGUMENT;
  for (int64_t i = 0; i < num_pairs; ++i)
    if (src_slots[i] < 0 || src_slots[i] > 0x7fffffffLL || dst_slots[i] < 0 || dst_slots[i] > 0x7fffffffLL)
      return LVAMD_ERR_INVALID_ARGUMENT;
  auto launch = [&]<int PAIRS, int CHUNKS>() -> int {
    Q8FewArgs<PAIRS, CHUNKS> a{
        .by_block = FastDiv(block_size), .by_heads = FastDiv(num_kv_heads), .by_chunks = FastDiv(head_size / 16)};
    for (int c = 0; c <= num_chunks; ++c) a.starts[c] = chunk_starts[c];
    for (int64_t i = 0; i < num_pairs; ++i) {
      a.src[i] = (int32_t)src_slots[i];
      a.dst[i] = (int32_t)dst_slots[i];
    }
    a.layer_keys = layer_key_ptrs;
    a.layer_values = layer_value_ptrs;
    a.scale_offset = scale_offset;
    a.num_kv_heads = num_kv_heads;
    a.head_size = head_size;
    a.block_size = block_size;
    hipLaunchKernelGGL((q8_compact_few_kernel<PAIRS, CHUNKS>),
                       dim3((unsigned)(num_layers * 2 * num_kv_heads), (unsigned)num_chunks), dim3(64), 0,
                       static_cast<hipStream_t>(stream), a);
    return launch_status();
  };
  return num_chunks == 1 ? launch.template operator()<kFewPairs, 1>()
                         : launch.template operator()<kCallPairs, kCallChunks>();
}
