// Attention of prompt chunks over latent vectors on gfx950, with per-head keys
// and values (the expanded form): lvamd_latent_expand has written, per head, the
// request's keys [key][N] and values [key][V], and the shared rotated keys
// [key][P] once.  Linear requests: query j of a request with c computed tokens
// sees positions [0, c + j].
//
// A (query, key) pair costs N + P + V products here against 2 L + P in latent
// space, which a long chunk earns back over the expansion of its keys.
//
// Mapping onto CDNA4: the 16-bit prefill kernel's (lvamd_prefill.hip), with one
// head per kv head, keys and values of different widths, and no block tables:
//   * a unit is up to 128 queries of one head: four waves of two 16-query column
//     tiles; keys in tiles of 64, loaded straight into LDS, double-buffered, one
//     barrier per tile;
//   * S^T = K Q^T and O^T = V^T P^T on MFMA 16x16x32, the online softmax in the
//     log2 domain with lazy rescaling, the sums on the matrix cores;
//   * a later token's row may hold what is not finite: where a score of a tile is not
//     finite, the tile's values that are not become zeros on their way to the products.
//     Queries that see such a row get NaN through its score: lvamd_latent_expand makes a
//     key NaN wherever its value is not finite;
//   * units over a key range write fp32 partials, merged by
//     lvamd_paged_attention_merge_q8's kernel.
//
// 2,048 queries behind 14,336 tokens, 16 heads, 128 + 64 and 128 (322 GFLOP): 370 to
// 400 us, 0.80 to 0.87 PFLOP/s, as far as the 16-bit prefill kernel: softmax and LDS
// reads share the issue with the matrix units.

#include <cmath>

#include "lvamd_latent.h"

namespace lvamd {

namespace {

constexpr float kSlack = 8.0f;  // log2 units
constexpr int KT = 64;          // keys per tile
constexpr int kUnitColumns = 128;

typedef const __attribute__((address_space(1))) void* lds_gptr;
typedef __attribute__((address_space(3))) void* lds_lptr;

// LDS tile layout as the 16-bit prefill kernel's: groups of 64 bytes of every
// row, group-major, chunk slots permuted by row bits.
__device__ __forceinline__ constexpr int swz(int row) {
  return ((row >> 2) & 1) | ((((row >> 2) ^ (row >> 3)) & 1) << 1);
}

struct LatentPrefillArgs {
  const void* q;  // [tokens][heads][N ...]
  int64_t q_tok_stride, q_head_stride;
  const void* qr;  // [tokens][heads][P]
  int64_t qr_tok_stride, qr_head_stride;
  const void* keys;    // [heads][keys][N]
  const void* values;  // [heads][keys][V]
  const void* rope;    // [keys][P]
  int64_t num_keys;
  void* out;
  int64_t out_tok_stride, out_head_stride;
  float* part_acc;  // [slots][heads][128][V]
  float* part_ml;
  int32_t heads;
  FastDiv by_heads;
  float scale_log2;
};

// Eight 16-bit values with those that are not finite replaced by zero.
template <typename T>
__device__ __forceinline__ uint4 finite_only(uint4 v) {
  constexpr uint32_t e = std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
  auto word = [](uint32_t w) {
    const uint32_t lo = (w & e) == e ? 0u : w & 0xffffu;
    const uint32_t hi = ((w >> 16) & e) == e ? 0u : w & 0xffff0000u;
    return lo | hi;
  };
  return make_uint4(word(v.x), word(v.y), word(v.z), word(v.w));
}

}  // namespace

template <typename T, int N, int P, int V>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void latent_prefill_kernel(
    const int32_t* __restrict__ units, const LatentPrefillArgs a) {
  constexpr int GK = (N + P) / 32, GV = V / 32;  // 64-byte groups of a row
  constexpr int GB = KT * 64;
  constexpr int KS = KT / 16, NCH = (N + P) / 32, NT = V / 16, CT = 2;
  constexpr int LOADS = GK + GV;
  using V8 = typename std::conditional<std::is_same<T, __bf16>::value, bf16x8, f16x8>::type;
  __shared__ __attribute__((aligned(1024))) char klds0[GK * GB];
  __shared__ __attribute__((aligned(1024))) char klds1[GK * GB];
  __shared__ __attribute__((aligned(1024))) char vlds0[GV * GB];
  __shared__ __attribute__((aligned(1024))) char vlds1[GV * GB];

  const int tid = threadIdx.x & 255;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int l16 = lane & 15;
  const int g = lane >> 4;
  const int unit = fast_div((int)blockIdx.x, a.by_heads);
  const int h = (int)blockIdx.x - unit * a.heads;
  const int32_t* u = units + (int64_t)unit * LVAMD_PREFILL_FIELDS;
  const int col0 = u[1], ncols = u[2], key_begin = u[3], key_end = u[4], slot = u[5];
  const int64_t key0 = (int64_t)u[6] * KT;  // the request's first row of the workspace
  const int q_start = u[7], computed = u[8];
  if (ncols <= 0) return;  // a padding record
  const int col_end = col0 + ncols;
  const int kneed = computed + col_end;
  const int kmax = key_end > 0 && key_end < kneed ? key_end : kneed;
  const int tile0 = key_begin / KT;
  const int ntiles = (kmax + KT - 1) / KT - tile0;

  // ---- tile loads: wave w loads rows 16 w .. 16 w + 15, lane l row l / 4 of
  // them into chunk slot l % 4 of every group.  (Rows past the request's keys are
  // its last key again, or another's; they are masked.)
  const int lrow = 16 * wave + (lane >> 2);
  const int lchunk = (lane & 3) ^ swz(lrow);
  const int64_t first = key0 + (int64_t)tile0 * KT + lrow;
  gptr<const T> ksrc = (gptr<const T>)(a.keys) + ((int64_t)h * a.num_keys + first) * N + 8 * lchunk;
  gptr<const T> vsrc = (gptr<const T>)(a.values) + ((int64_t)h * a.num_keys + first) * V + 8 * lchunk;
  gptr<const T> rsrc = (gptr<const T>)(a.rope) + first * P + 8 * lchunk;
  auto issue_load = [&](int i, char* kdst, char* vdst) {
    if (i < GK) {
      gptr<const T> const from = i < N / 32 ? ksrc + 32 * i : rsrc + 32 * (i - N / 32);
      __builtin_amdgcn_global_load_lds((lds_gptr)from, (lds_lptr)(kdst + i * GB + wave * 1024), 16, 0, 0);
    } else {
      __builtin_amdgcn_global_load_lds((lds_gptr)(vsrc + 32 * (i - GK)), (lds_lptr)(vdst + (i - GK) * GB + wave * 1024), 16,
                                       0, 0);
    }
  };
  auto next_tile = [&]() {
    ksrc += (int64_t)KT * N;
    vsrc += (int64_t)KT * V;
    rsrc += (int64_t)KT * P;
  };

  // ---- this wave's queries
  int qi[CT];
  bool ok[CT];
  uint4 qf[CT][NCH];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = col0 + 16 * (CT * wave + ct) + l16;
    ok[ct] = col < col_end;
    qi[ct] = ok[ct] ? col : col_end - 1;
    const T* q = static_cast<const T*>(a.q) + (int64_t)(q_start + qi[ct]) * a.q_tok_stride + (int64_t)h * a.q_head_stride;
    const T* qr = static_cast<const T*>(a.qr) + (int64_t)(q_start + qi[ct]) * a.qr_tok_stride + (int64_t)h * a.qr_head_stride;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
      qf[ct][k] = ok[ct] ? load16(32 * k < N ? q + 32 * k + 8 * g : qr + 32 * k - N + 8 * g) : zero_u4();
  }
  const int wave_first = col0 + 16 * CT * wave;
  const bool wave_active = wave_first < col_end;
  const int wave_kmax = computed + min(wave_first + 16 * CT, col_end);
  const int full_tiles = (computed + col0 + 1) / KT;  // visible to every query of the unit

  float m_run[CT];
  f32x4 l_run[CT];
  f32x4 acc[CT][NT];
  V8 ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = from_f32<T>(1.f);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m_run[ct] = -INFINITY;
    l_run[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[ct][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int q4 = l16 & 3;
  const int k_off = l16 * 64 + 16 * (g ^ swz(l16));
  const int v_row = 4 * g + (l16 >> 2);
  const int v_off0 = v_row * 64 + 16 * ((q4 >> 1) ^ swz(v_row)) + 8 * (q4 & 1);
  const int v_off1 = v_row * 64 + 16 * ((2 + (q4 >> 1)) ^ swz(v_row)) + 8 * (q4 & 1);

  // MASKED: the tile may reach past what every query sees.  The unmasked copy
  // issues the next tile's loads between its matrix instructions.
  auto compute_tile = [&]<bool MASKED>(int tr, const char* kt, const char* vt, char* kn, char* vn)
      __attribute__((always_inline)) {
    const int t = tile0 + tr;
    if (!wave_active || (MASKED && t * KT >= wave_kmax)) return;
    __builtin_amdgcn_s_setprio(1);
    f32x4 st[CT][KS];
    {
      constexpr int TOT = KS * NCH, LEAD = 3;
      static_assert(TOT >= LOADS, "every load of the next tile has a place");
      constexpr int LSTEP = TOT / LOADS;
      auto rd = [&](int i) -> uint4 {
        return *reinterpret_cast<const uint4*>(kt + (i % NCH) * GB + (i / NCH) * 1024 + k_off);
      };
      uint4 kf[LEAD];
#pragma unroll
      for (int i = 0; i < LEAD; ++i) kf[i] = rd(i);
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < TOT; ++i) {
        const int s = i / NCH, k = i % NCH;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) st[ct][s] = Mma<T>::qk(kf[i % LEAD], qf[ct][k], k == 0 ? z : st[ct][s]);
        if (i + LEAD < TOT) kf[i % LEAD] = rd(i + LEAD);
        if (!MASKED && i % LSTEP == 0 && i / LSTEP < LOADS) issue_load(i / LSTEP, kn, vn);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    bool odd = false;
    if (MASKED && t >= full_tiles) {
      // A later token's row may hold what is not finite; its scores are not
      // finite either, and its zero probability would not hide its values.
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int last = computed + qi[ct] - t * KT - 4 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            odd |= !(__builtin_fabsf(st[ct][s][r]) < INFINITY);
            st[ct][s][r] = 16 * s + r > last ? -INFINITY : st[ct][s][r] * a.scale_log2;
          }
      }
      odd = __any(odd);
    } else {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int s = 0; s < KS; ++s) st[ct][s] *= a.scale_log2;
    }
    V8 pb[CT][KS / 2];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float mt = -INFINITY;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) mt = fmaxf(mt, st[ct][s][r]);
      mt = row_max4(mt);
      if (__any(mt > m_run[ct] + kSlack)) {
        const float m_new = fmaxf(m_run[ct], mt);
        const float alpha = (m_new == -INFINITY) ? 1.f : fast_exp2(m_run[ct] - m_new);
        l_run[ct] *= alpha;
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[ct][n] *= alpha;
        m_run[ct] = m_new;
      }
      const float nbase = (m_run[ct] == -INFINITY) ? 0.f : kWeightLift<T> - m_run[ct];
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) pb[ct][s >> 1][(s & 1) * 4 + r] = from_f32<T>(fast_exp2(st[ct][s][r] + nbase));
    }
    __builtin_amdgcn_s_setprio(1);
    {
      constexpr int TOT = KS / 2 * NT, LEAD = 2;
      auto rd = [&](int i) -> V8 {
        const int hh = i / NT, n = i % NT;
        const int lo = (n & 1 ? v_off1 : v_off0) + (n >> 1) * GB + hh * 32 * 64;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vt + lo));
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vt + lo + 16 * 64));
        const s16x4 both[2] = {v0, v1};
        return bitcast<V8>(both);
      };
      auto mm = [&](V8 x, V8 y, f32x4 c) -> f32x4 {
        if constexpr (std::is_same<T, __bf16>::value) {
          return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
        } else {
          return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
        }
      };
      V8 vf[LEAD];
#pragma unroll
      for (int i = 0; i < LEAD; ++i) vf[i] = rd(i);
#pragma unroll
      for (int hh = 0; hh < KS / 2; ++hh)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) l_run[ct] = mm(ones, pb[ct][hh], l_run[ct]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TOT; ++i) {
        const int hh = i / NT, n = i % NT;
        V8 v = vf[i % LEAD];
        if (MASKED && odd) v = bitcast<V8>(finite_only<T>(bitcast<uint4>(v)));
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) acc[ct][n] = mm(v, pb[ct][hh], acc[ct][n]);
        if (i + LEAD < TOT) vf[i % LEAD] = rd(i + LEAD);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };

  auto tile_done = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __builtin_amdgcn_s_barrier();
  };
#pragma unroll
  for (int i = 0; i < LOADS; ++i) issue_load(i, klds0, vlds0);
  next_tile();
  tile_done();
  auto step = [&]<bool MASKED>(int t, const char* kc, const char* vc, char* kn, char* vn) __attribute__((always_inline)) {
    const bool more = !MASKED || t + 1 < ntiles;
    if ((MASKED || !wave_active) && more) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) issue_load(i, kn, vn);
    }
    compute_tile.template operator()<MASKED>(t, kc, vc, kn, vn);
    next_tile();
    tile_done();
  };
  int t = 0;
  const int nfull = min((computed + col0) / KT - tile0, ntiles - 1) - 1;
  for (; t < nfull; t += 2) {
    step.template operator()<false>(t, klds0, vlds0, klds1, vlds1);
    step.template operator()<false>(t + 1, klds1, vlds1, klds0, vlds0);
  }
  for (; t < ntiles; t += 2) {
    step.template operator()<true>(t, klds0, vlds0, klds1, vlds1);
    if (t + 1 < ntiles) step.template operator()<true>(t + 1, klds1, vlds1, klds0, vlds0);
  }

  if (!wave_active) return;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (!ok[ct]) continue;
    const float l_tot = l_run[ct][0];
    // (A unit over a key range may hold no key that a query sees, and weighs nothing
    // then; a whole softmax without a finite score is NaN.)
    const float inv = l_tot > 0.f ? 1.f / l_tot : slot < 0 ? NAN : l_tot == l_tot ? 0.f : l_tot;
    if (slot >= 0) {
      const int64_t cs = ((int64_t)slot * a.heads + h) * kUnitColumns + 16 * (CT * wave + ct) + l16;
#pragma unroll
      for (int n = 0; n < NT; ++n) store_partial4<true, float>(a.part_acc + cs * V + 16 * n + 4 * g, acc[ct][n], inv);
      const float m = l_tot == l_tot || m_run[ct] != -INFINITY ? m_run[ct] : 0.f;
      if (g == 0) __builtin_nontemporal_store(f32x2{m, l_tot}, reinterpret_cast<f32x2*>(a.part_ml + cs * 2));
      continue;
    }
    T* to = static_cast<T*>(a.out) + (int64_t)(q_start + qi[ct]) * a.out_tok_stride + (int64_t)h * a.out_head_stride;
#pragma unroll
    for (int n = 0; n < NT; ++n) store_partial4<false, T>(to + 16 * n + 4 * g, acc[ct][n], inv);
  }
}

template <typename T, int N, int P, typename F>
static int with_value(int value, F& f) {
  return value == 64 ? f.template operator()<T, N, P, 64>() : f.template operator()<T, N, P, 128>();
}
template <typename T, int N, typename F>
static int with_rope(int rope, int value, F& f) {
  return rope == 32 ? with_value<T, N, 32>(value, f) : with_value<T, N, 64>(value, f);
}
template <typename T, typename F>
static int with_nope(int nope, int rope, int value, F& f) {
  return nope == 64 ? with_rope<T, 64>(rope, value, f) : with_rope<T, 128>(rope, value, f);
}
template <typename F>
static int prefill_dispatch(int dtype, int nope, int rope, int value, F f) {
  if (!latent_dtype(dtype) || (nope != 64 && nope != 128) || (rope != 32 && rope != 64) || (value != 64 && value != 128))
    return LVAMD_ERR_UNSUPPORTED;
  return dtype == LVAMD_BF16 ? with_nope<__bf16>(nope, rope, value, f) : with_nope<_Float16>(nope, rope, value, f);
}

}  // namespace lvamd

using namespace lvamd;

extern "C" int lvamd_latent_prefill_resident_units(int32_t dtype, int32_t nope_size, int32_t rope_size, int32_t value_size) {
  return prefill_dispatch(dtype, nope_size, rope_size, value_size, [&]<typename T, int N, int P, int V>() -> int {
    int device = 0, cus = 0, per_cu = 0;
    if (hipGetDevice(&device) != hipSuccess) return LVAMD_ERR_LAUNCH;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess) return LVAMD_ERR_LAUNCH;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, (const void*)&latent_prefill_kernel<T, N, P, V>, 256, 0) !=
        hipSuccess)
      return LVAMD_ERR_LAUNCH;
    return per_cu * cus;
  });
}

extern "C" int lvamd_latent_prefill(const void* query, int64_t query_token_stride, int64_t query_head_stride,
                                    const void* query_rope, int64_t rope_token_stride, int64_t rope_head_stride,
                                    const void* keys, const void* values, const void* rope_keys, int64_t num_keys, void* out,
                                    int64_t out_token_stride, int64_t out_head_stride, const int32_t* units,
                                    int32_t num_units, const int32_t* jobs, int32_t num_jobs, int32_t merge_columns,
                                    float* part_acc, float* part_ml, int64_t num_partial_slots, int32_t num_heads,
                                    int32_t nope_size, int32_t rope_size, int32_t value_size, float scale, int32_t dtype,
                                    lvamd_stream_t stream) {
  if (num_units < 0 || num_jobs < 0 || num_heads <= 0 || num_keys < 0 || num_partial_slots < 0 || merge_columns < 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_units > 0) {
    if (!query || !query_rope || !keys || !values || !rope_keys || !out || !units || (num_jobs > 0 && !jobs) ||
        !rows16(query, {query_token_stride, query_head_stride}) || !rows16(query_rope, {rope_token_stride, rope_head_stride}) ||
        !rows16(keys, {}) || !rows16(values, {}) || !rows16(rope_keys, {}) || ((uintptr_t)out & 7u) ||
        out_token_stride % 4 != 0 || out_head_stride % 4 != 0 || (int64_t)num_units * num_heads > 0x7fffffffLL)
      return LVAMD_ERR_INVALID_ARGUMENT;
    if (num_partial_slots > 0 && (!part_acc || !part_ml)) return LVAMD_ERR_WORKSPACE;
  }
  LatentPrefillArgs a{.by_heads = FastDiv(num_heads)};
  a.q = query;
  a.q_tok_stride = query_token_stride;
  a.q_head_stride = query_head_stride;
  a.qr = query_rope;
  a.qr_tok_stride = rope_token_stride;
  a.qr_head_stride = rope_head_stride;
  a.keys = keys;
  a.values = values;
  a.rope = rope_keys;
  a.num_keys = num_keys;
  a.out = out;
  a.out_tok_stride = out_token_stride;
  a.out_head_stride = out_head_stride;
  a.part_acc = part_acc;
  a.part_ml = part_ml;
  a.heads = num_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int status = prefill_dispatch(dtype, nope_size, rope_size, value_size, [&]<typename T, int N, int P, int V>() -> int {
    if (num_units == 0) return LVAMD_OK;
    hipLaunchKernelGGL((latent_prefill_kernel<T, N, P, V>), dim3((unsigned)(num_units * num_heads)), dim3(256), 0, s, units, a);
    return launch_status();
  });
  if (status != LVAMD_OK || num_units == 0 || num_jobs == 0) return status;
  return launch_merge(part_acc, part_ml, out, out_token_stride, out_head_stride, jobs, num_jobs, num_partial_slots, 0,
                      num_heads, 1, value_size, kUnitColumns / 16, merge_columns, dtype, s, true, NAN);
}
