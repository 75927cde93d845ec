// Prefill and tree-verification attention over the 8-bit cache on gfx950:
// requests of more than one 16-column MFMA tile.
//
// Semantics are the 16-bit prefill kernel's (lvamd_prefill.hip) with K and V
// the cache's values, code * scale; the step's tokens are in the cache already
// (lvamd_kv_append_q8 runs first).  Work units, spans, split keys, partials and
// merge are the same too.
//
// Mapping onto CDNA4:
//   * A unit is up to 128 columns, (query, head-in-group) pairs of one kv head:
//     eight waves of one 16-column tile share every key tile (64 keys, 32 above
//     D = 128).  Four waves of two tiles each read half as much of LDS, but fill
//     the registers: half as many waves per SIMD, none beside it above D = 128.
//     A chunk of 1024 tokens after 4096 (16 heads, 4 kv heads) took 182 us so at
//     D = 160 against 125, 219 against 154 at D = 256; at D = 128 2048 tokens (28
//     heads, 4 kv heads) 73 against 65, and 536 against 555 for 8192.
//   * Units of 256 columns, eight waves of two tiles, for chunks that fill the
//     GPU with them (64 < D <= 128, backend.py's rule): each code is converted
//     for twice the products.  2048 tokens after 14336, 28 heads, 4 kv heads, D
//     = 128: 485 us (930 TFLOP/s) against 545.
//   * Units of 64 columns, four waves, for steps whose requests all have at most
//     64 (tree verification, short chunks): no wave is left without columns, and
//     the registers hold several tiles in flight, as such units are bound by the
//     latency of their few tiles.
//   * A tile's codes go to registers (16 per load and thread) while the last
//     tile computes, become T with their block's scale (exactly, lvamd_q8.h)
//     and are written to the other of two LDS buffers; one barrier per tile.
//     Converting before LDS, each code is converted once per workgroup;
//     direct loads to LDS would leave it to each of the waves.
//   * S^T = K Q^T, O^T = V^T P^T and the softmax sums on MFMA 16x16x32, online
//     softmax in the log2 domain with lazy rescaling, as in the 16-bit kernel.
//   * NaN values of this step's tokens: as in the 8-bit decode kernel, they go
//     to LDS as zero and the columns that see the row get them back.
//
// Bound by the matrix units' schedule in chunks (they are busy 48% of the time;
// LDS reads, the softmax and the conversions share the issue), by the chain of a
// unit's few tiles in tree steps: 32 trees of 9 queries after 500-2560 tokens, 12
// heads over 2, D = 128: 14 us, and 5 for the merge.  A chunk of 1024 tokens after
// 4096 (16 heads over 4) takes 50 us at D = 64, 76 at 128, 124 at 160, 151 at 256.

#include <cmath>

#include "lvamd_q8.h"

namespace lvamd {

namespace {

constexpr float kSlack = 8.0f;  // lazy-rescale threshold, log2 units

struct Q8PrefillArgs {
  const void* q;
  int64_t q_tok_stride, q_head_stride;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* k_scales;
  const float* v_scales;
  void* out;
  int64_t out_tok_stride, out_head_stride;
  const int32_t* __restrict__ tables;
  const uint32_t* __restrict__ vis;
  void* part_acc;
  float* part_ml;
  int32_t group;
  int32_t block_size;
  FastDiv by_block, by_group;
  float scale_log2;
};

// CT: column tiles per wave, 2 or 1; W: waves.
template <int D, int CT, int W>
struct Q8PrefillShape {
  static constexpr int COLUMNS = 16 * W * CT;
  static constexpr int KT = D <= 128 ? 64 : 32;
  static constexpr int KS = KT / 16;
  static constexpr int C8 = D / 16;              // 16-code chunks per row
  static constexpr int CPR = D / 8;              // 16-byte chunks of T per row
  static constexpr int RS = q8_row_stride(CPR);  // LDS row stride in chunks
  static constexpr int THREADS = 64 * W;
  static constexpr int LPT = (KT * C8 + THREADS - 1) / THREADS;  // loads per thread and tensor
  static constexpr int NCH = (D + 31) / 32;
  static constexpr int NT = D / 16;
  static constexpr int PD = CT == 2 || W == 8 ? 1 : D <= 128 ? 4 : 2;  // tiles in flight
};

}  // namespace

// (Waves per SIMD: what the registers and the resident workgroups allow.)
constexpr int prefill_waves_per_eu(int d, int col_tiles, int waves) {
  return waves == 4 ? (d <= 128 ? 2 : 1) : col_tiles == 1 && d <= 128 ? 4 : 2;
}
template <typename T, int D, int CT, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(prefill_waves_per_eu(D, CT, W)))) void q8_prefill_kernel(
    const int32_t* __restrict__ units, const int32_t num_kv_heads, const uint32_t heads_magic, const int32_t heads_shift,
    const Q8PrefillArgs a) {
  using P = Q8PrefillShape<D, CT, W>;
  constexpr int KT = P::KT, KS = P::KS, C8 = P::C8, CPR = P::CPR, RS = P::RS, LPT = P::LPT, NCH = P::NCH, NT = P::NT;
  constexpr int PD = P::PD;
  using V8 = typename std::conditional<std::is_same<T, __bf16>::value, bf16x8, f16x8>::type;
  __shared__ __attribute__((aligned(16))) uint4 klds[2][KT * RS];
  __shared__ __attribute__((aligned(16))) uint4 vlds[2][KT * RS];
  __shared__ int poison[2];  // a buffer's V rows had NaN left out

  const int tid = threadIdx.x & (P::THREADS - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int l16 = lane & 15;
  const int g = lane >> 4;
  const int Hkv = num_kv_heads;
  const int G = a.group;
  const int unit = fast_div((int)blockIdx.x, heads_magic, heads_shift);
  const int kvh = (int)blockIdx.x - unit * Hkv;
  const int32_t* u = units + (int64_t)unit * LVAMD_PREFILL_FIELDS;
  const int col0 = u[1], ncols = u[2], key_begin = u[3], key_end = u[4], slot = u[5];
  const int table_off = u[6], q_start = u[7], computed = u[8], q_len = u[9], vis_off = u[10], vis_words = u[11];
  const int b0 = u[12], b1 = u[13], b2 = u[14], b3 = u[15];  // of the unit's first tile; -1: take them from the table
  if (ncols <= 0) return;  // a padding record (the host's per-XCD unit order)
  const int col_end = col0 + ncols;
  const int kneed = computed + fast_div(col_end - 1, a.by_group) + 1;
  const int kmax = key_end > 0 && key_end < kneed ? key_end : kneed;
  const int tile0 = key_begin / KT;
  const int ntiles = (kmax + KT - 1) / KT - tile0;
  const int bs = a.block_size;
  const int64_t row_bytes = (int64_t)Hkv * D;
  gptr<const uint8_t> const kbase = (gptr<const uint8_t>)(a.k_pool) + (int64_t)kvh * D;
  gptr<const uint8_t> const vbase = (gptr<const uint8_t>)(a.v_pool) + (int64_t)kvh * D;
  gptr<const float> const kscales = (gptr<const float>)(a.k_scales) + kvh;
  gptr<const float> const vscales = (gptr<const float>)(a.v_scales) + kvh;
  const int32_t* table = a.tables + table_off;

  // ---- tile loads: chunk id tid + THREADS j of a tile is chunk id % C8 of row
  // id / C8.  Rows past the piece repeat its last key (masked).
  auto key_pos = [&](int t, int j) -> int {
    const int row = (tid + P::THREADS * j) / C8;
    const int pos = (tile0 + t) * KT + (row < KT ? row : KT - 1);
    return pos < kmax ? pos : kmax - 1;
  };
  auto lookup = [&](int t, int (&block)[LPT]) {
#pragma unroll
    for (int j = 0; j < LPT; ++j) block[j] = table[fast_div(key_pos(t, j), a.by_block)];
  };
  // Tile 0's from the unit's record where it has them: no wait for the table.
  auto lookup_first = [&](int (&block)[LPT]) {
    if (b0 < 0) {
      lookup(0, block);
      return;
    }
#pragma unroll
    for (int j = 0; j < LPT; ++j) {
      const int k = fast_div(key_pos(0, j), a.by_block) - fast_div(key_begin, a.by_block);
      block[j] = k == 0 ? b0 : k == 1 ? b1 : k == 2 ? b2 : b3;
    }
  };
  struct Tile {
    uint4 k[LPT], v[LPT];
    float ks[LPT], vs[LPT];
  };
  auto issue = [&](int t, const int (&block)[LPT], Tile& x) {
#pragma unroll
    for (int j = 0; j < LPT; ++j) {
      const int64_t at = (int64_t)block[j] * Hkv;
      x.ks[j] = kscales[at];
      x.vs[j] = vscales[at];
    }
#pragma unroll
    for (int j = 0; j < LPT; ++j) {
      const int c = (tid + P::THREADS * j) % C8;
      const int pos = key_pos(t, j);
      const int64_t s = (int64_t)block[j] * bs + (pos - fast_div(pos, a.by_block) * bs);
      const int64_t off = s * row_bytes + 16 * c;
      x.k[j] = load16(kbase + off);
      x.v[j] = load16(vbase + off);
    }
  };
  auto stage_rows = [&]<bool NEW>(int first_new, const Tile& x, uint4* kd, uint4* vd, int* flag)
      __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < LPT; ++j) {
      const int id = tid + P::THREADS * j;
      const int row = id / C8, c = id - row * C8;
      uint4 v = x.v[j];
      if constexpr (NEW) {
        if (row >= first_new && q8_has_nan(v)) {
          *flag = 1;
          v = make_uint4(q8_without_nan4(v.x), q8_without_nan4(v.y), q8_without_nan4(v.z), q8_without_nan4(v.w));
        }
      }
      uint4 klo, khi, vlo, vhi;
      q8_values16<T>(x.k[j], x.ks[j], klo, khi);
      q8_values16<T>(v, x.vs[j], vlo, vhi);
      if (P::THREADS * LPT == KT * C8 || row < KT) {
        kd[row * RS + 2 * c] = klo;
        kd[row * RS + 2 * c + 1] = khi;
        vd[row * RS + 2 * c] = vlo;
        vd[row * RS + 2 * c + 1] = vhi;
      }
    }
  };
  auto stage = [&](int t, const Tile& x, uint4* kd, uint4* vd, int* flag) __attribute__((always_inline)) {
    const int first_new = computed - (tile0 + t) * KT;  // rows from it on hold this step's tokens
    if (first_new >= KT) {
      stage_rows.template operator()<false>(first_new, x, kd, vd, flag);
    } else {
      stage_rows.template operator()<true>(first_new, x, kd, vd, flag);
    }
  };

  // ---- this wave's columns: (query qi, head) per column tile, and Q^T chunks
  int qi[CT];
  bool colok[CT];
  uint4 qf[CT][NCH];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = col0 + 16 * (CT * wave + ct) + l16;
    colok[ct] = col < col_end;
    const int colc = colok[ct] ? col : col_end - 1;
    qi[ct] = fast_div(colc, a.by_group);
    const int qhead = kvh * G + (colc - qi[ct] * G);
    const T* qrow = static_cast<const T*>(a.q) + (int64_t)(q_start + qi[ct]) * a.q_tok_stride +
                    (int64_t)qhead * a.q_head_stride;
#pragma unroll
    for (int kk = 0; kk < NCH; ++kk) {
      const int ch = kk * 4 + g;
      qf[ct][kk] = (colok[ct] && ch < CPR) ? load16(qrow + ch * 8) : zero_u4();
    }
  }
  const int wave_col_last = col0 + 16 * CT * (wave + 1) - 1;
  const int wave_kmax = computed + fast_div(wave_col_last < col_end ? wave_col_last : col_end - 1, a.by_group) + 1;
  const bool wave_active = col0 + 16 * CT * wave < col_end;
  const bool tree = vis_off >= 0;
  // Tiles below this bound are visible to every column of the unit.
  const int full_tiles = (tree ? computed : computed + fast_div(col0, a.by_group) + 1) / KT;
  const float c_log2 = a.scale_log2;
  // A tree's ancestor words: the first two of each column's row are loaded here
  // (a load among the tiles' would wait for those before it); longer rows are
  // read where a tile needs them.
  const bool few_words = vis_words <= 2;
  uint32_t row_word0[CT], row_word1[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    row_word0[ct] = tree && few_words ? a.vis[vis_off + qi[ct] * vis_words] : 0u;
    row_word1[ct] = tree && vis_words == 2 ? a.vis[vis_off + qi[ct] * vis_words + 1] : 0u;
  }
  // Whether a column sees the step's token j.
  auto sees = [&](int ct, int j) -> bool {
    if (!tree) return j <= qi[ct];
    return j < q_len && ((a.vis[vis_off + qi[ct] * vis_words + (j >> 5)] >> (j & 31)) & 1u);
  };

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
  auto mm = [&](V8 x, V8 y, f32x4 c) -> f32x4 {
    if constexpr (std::is_same<T, __bf16>::value) {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
    } else {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
    }
  };

  // MASKED: the tile may reach past what every column of the unit sees.  LDS
  // reads run LEAD operands ahead of the matrix instructions, held there by
  // scheduling barriers.
  auto compute = [&]<bool MASKED>(int tr, const uint4* kt, const uint4* vt, const int* flag)
      __attribute__((always_inline)) {
    const int t = tile0 + tr;
    if (!wave_active || (MASKED && t * KT >= wave_kmax)) return;
    f32x4 st[CT][KS];
    __builtin_amdgcn_s_setprio(1);
    {
      constexpr int TOT = KS * NCH, LEAD = TOT < 3 ? TOT : 3;
      auto rd = [&](int i) -> uint4 {
        const int s = i / NCH, ch = (i % NCH) * 4 + g;
        return (CPR % 4 == 0 || ch < CPR) ? kt[(16 * s + l16) * RS + ch] : zero_u4();
      };
      uint4 kf[LEAD];
#pragma unroll
      for (int i = 0; i < LEAD; ++i) kf[i] = rd(i);
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < TOT; ++i) {
        const int s = i / NCH, kk = i % NCH;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) st[ct][s] = Mma<T>::qk(kf[i % LEAD], qf[ct][kk], kk == 0 ? z : st[ct][s]);
        if (i + LEAD < TOT) kf[i % LEAD] = rd(i + LEAD);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if (MASKED && t >= full_tiles) {
      const int j0 = t * KT - computed;  // the tile's first key as a token of the step
      if (!tree) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int last = qi[ct] - j0 - 4 * g;
#pragma unroll
          for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) st[ct][s][r] = 16 * s + r > last ? -INFINITY : st[ct][s][r];
        }
      } else {
        // The row's words that cover the tile's keys, as 16 bits per key group:
        // bits of keys before the step are set, those past it clear.
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          uint32_t low = 0;
#pragma unroll
          for (int i = 0; i <= KT / 32; ++i) {
            const int wi = (j0 >> 5) + i;
            const int left = q_len - 32 * wi;
            const uint32_t valid = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
            const int wc = min(max(wi, 0), vis_words - 1);
            const uint32_t w0 = row_word0[ct], w1 = row_word1[ct];
            uint32_t row = wc == 0 ? w0 + 0u : w1 + 0u;  // (values: a choice of lvalues would put the arrays in memory)
            if (!few_words) row = a.vis[vis_off + qi[ct] * vis_words + wc];
            const uint32_t word = wi < 0 ? ~0u : row & valid;
            if (i > 0) {
              const uint32_t bits = __builtin_amdgcn_alignbit(word, low, j0 & 31) >> (4 * g);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int s = 2 * (i - 1) + (e >> 2);
                st[ct][s][e & 3] = (bits >> (16 * (e >> 2) + (e & 3))) & 1u ? st[ct][s][e & 3] : -INFINITY;
              }
            }
            low = word;
          }
        }
      }
    }
    V8 pb[CT][KS / 2];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float mt = -INFINITY;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) mt = fmaxf(mt, st[ct][s][r]);
      mt = row_max4(mt) * c_log2;
      if (__any(mt > m_run[ct] + kSlack)) {
        const float m_new = fmaxf(m_run[ct], mt);
        const float alpha = (m_new == -INFINITY) ? 1.f : fast_exp2(m_run[ct] - m_new);
        l_run[ct] *= alpha;
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[ct][n] *= alpha;
        m_run[ct] = m_new;
      }
      const float nbase = (m_run[ct] == -INFINITY) ? 0.f : -m_run[ct];
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          // (Rounded to T, as a matrix instruction's operands are of one type; the
          // sum below takes them as rounded.)
          pb[ct][s >> 1][(s & 1) * 4 + r] = from_f32<T>(fast_exp2(__builtin_fmaf(st[ct][s][r], c_log2, nbase)));
    }
    __builtin_amdgcn_s_setprio(1);
    const char* vbytes = reinterpret_cast<const char*>(vt);
    const int q4 = l16 & 3;
    {
      constexpr int TOT = KS / 2 * NT, LEAD = TOT < 2 ? TOT : 2;
      auto rd = [&](int i) -> V8 {
        const int h = i / NT, n = i % NT;
        const int lo = ((32 * h + 4 * g + (l16 >> 2)) * RS + 2 * n + (q4 >> 1)) * 16 + (q4 & 1) * 8;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vbytes + lo));
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vbytes + lo + 16 * RS * 16));
        const s16x4 both[2] = {v0, v1};
        return bitcast<V8>(both);
      };
      V8 vf[LEAD];
#pragma unroll
      for (int i = 0; i < LEAD; ++i) vf[i] = rd(i);
#pragma unroll
      for (int h = 0; h < KS / 2; ++h)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) l_run[ct] = mm(ones, pb[ct][h], l_run[ct]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TOT; ++i) {
        const int h = i / NT, n = i % NT;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) acc[ct][n] = mm(vf[i % LEAD], pb[ct][h], acc[ct][n]);
        if (i + LEAD < TOT) vf[i % LEAD] = rd(i + LEAD);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if (MASKED && *flag) {
      for (int pos = max(t * KT, computed); pos < min((t + 1) * KT, kmax); ++pos) {
        const int lb = fast_div(pos, a.by_block);
        const int64_t s = (int64_t)table[lb] * bs + (pos - lb * bs);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const bool see = sees(ct, pos - computed);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint32_t nan = q8_nan4(*(gptr<const uint32_t>)(vbase + s * row_bytes + 16 * n + 4 * g));
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (see && ((nan >> (8 * r + 7)) & 1u)) acc[ct][n][r] = __uint_as_float(0x7fc00000u);
          }
        }
      }
    }
  };

  // ---- PD tiles' codes are in flight while a tile computes; the table entries
  // of a tile are loaded PD tiles before its codes.  Tile t is staged into buffer
  // t % 2; the barrier after it tells that every wave is done with tile t - 1's
  // predecessor in that buffer.  (A buffer's flag stays set: compute looks at
  // the rows themselves.)  No load is conditional in the steady loop, so that
  // each wait counts only the loads before its own: past the last tile they
  // repeat it.
  const int last_tile = ntiles - 1;
  Tile x[PD];
  int block[PD][LPT];
  if (tid < 2) poison[tid] = 0;
  lookup_first(block[0]);
#pragma unroll
  for (int i = 1; i < PD; ++i) lookup(min(i, last_tile), block[i]);
  int ahead[PD][LPT];
#pragma unroll
  for (int i = 0; i < PD; ++i) lookup(min(PD + i, last_tile), ahead[i]);
#pragma unroll
  for (int i = 0; i < PD; ++i) issue(min(i, last_tile), block[i], x[i]);
  __syncthreads();  // (the flags are clear)
  // PD tiles from t on.  MORE: tiles follow them; MASKED: as compute's.
  auto run = [&]<bool MORE, bool MASKED>(int t0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PD; ++i) {
      const int t = t0 + i;
      if (!MORE && t > last_tile) return;
      const int b = t & 1;
      stage(t, x[i], klds[b], vlds[b], &poison[b]);
      if constexpr (MORE) {
#pragma unroll
        for (int j = 0; j < LPT; ++j) block[i][j] = ahead[i][j];
        lookup(min(t + 2 * PD, last_tile), ahead[i]);
        issue(min(t + PD, last_tile), block[i], x[i]);
      }
      __syncthreads();
      compute.template operator()<MASKED>(t, klds[b], vlds[b], &poison[b]);
    }
  };
  int t = 0;
  if constexpr (PD == 1) {
    // Tiles that every column sees, before the step's own tokens; then the rest.
    const int nfull = min(min(full_tiles, computed / KT) - tile0, last_tile);
    for (; t < nfull; ++t) run.template operator()<true, false>(t);
  }
  for (; t + PD <= last_tile; t += PD) run.template operator()<true, true>(t);
  run.template operator()<false, true>(t);

  // ---- normalised output rows, or this piece's partials
  if (!wave_active) return;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (!colok[ct]) continue;
    const float l_tot = l_run[ct][0];
    const float inv = l_tot > 0.f ? 1.f / l_tot : l_tot == 0.f ? 0.f : l_tot;  // (NaN stays)
    if (slot >= 0) {
      const int64_t cs = ((int64_t)slot * Hkv + kvh) * P::COLUMNS + 16 * (CT * wave + ct) + l16;
      float* row = static_cast<float*>(a.part_acc) + cs * D;
#pragma unroll
      for (int n = 0; n < NT; ++n) store_partial4<true, float>(row + 16 * n + 4 * g, acc[ct][n], inv);
      // (A NaN sum keeps a finite maximum: the merge passes over a partial
      // whose maximum is -inf.)
      const float m = l_tot == l_tot || m_run[ct] != -INFINITY ? m_run[ct] : 0.f;
      if (g == 0) __builtin_nontemporal_store(f32x2{m, l_tot}, reinterpret_cast<f32x2*>(a.part_ml + cs * 2));
      continue;
    }
    const int col = col0 + 16 * (CT * wave + ct) + l16;
    const int qhead = kvh * G + (col - qi[ct] * G);
    T* row = static_cast<T*>(a.out) + (int64_t)(q_start + qi[ct]) * a.out_tok_stride + (int64_t)qhead * a.out_head_stride;
#pragma unroll
    for (int n = 0; n < NT; ++n) store_partial4<false, T>(row + 16 * n + 4 * g, acc[ct][n], inv);
  }
}

namespace {

bool prefill_q8_supported(int dtype, int head_size) {
  return (dtype == LVAMD_BF16 || dtype == LVAMD_F16) && q8_head_size(head_size);
}

// (Units of 256 columns: the head sizes whose two tiles per wave fit the
// registers, and whose products are long enough to gain by them.)
template <typename T, typename F>
int with_wide_head_size(int head_size, F& f) {
  switch (head_size) {
    case 80: return f.template operator()<T, 80, 2, 8>();
    case 96: return f.template operator()<T, 96, 2, 8>();
    case 112: return f.template operator()<T, 112, 2, 8>();
    case 128: return f.template operator()<T, 128, 2, 8>();
    default: return LVAMD_ERR_UNSUPPORTED;
  }
}
bool prefill_q8_columns(int columns) { return columns == 64 || columns == 128 || columns == 256; }
template <typename F>
int dispatch_prefill(int dtype, int head_size, int columns, F f) {
  const bool bf16 = dtype == LVAMD_BF16;
  switch (columns) {
    case 64:
      return q8_dispatch(dtype, head_size, [&]<typename T, int D>() { return f.template operator()<T, D, 1, 4>(); });
    case 128:
      return q8_dispatch(dtype, head_size, [&]<typename T, int D>() { return f.template operator()<T, D, 1, 8>(); });
    default: return bf16 ? with_wide_head_size<__bf16>(head_size, f) : with_wide_head_size<_Float16>(head_size, f);
  }
}

}  // namespace

}  // namespace lvamd

using namespace lvamd;

extern "C" int lvamd_paged_prefill_q8_key_tokens(int32_t dtype, int32_t head_size) {
  if (!prefill_q8_supported(dtype, head_size)) return LVAMD_ERR_UNSUPPORTED;
  return head_size <= 128 ? 64 : 32;
}

extern "C" int lvamd_paged_prefill_q8_resident_units(int32_t dtype, int32_t head_size, int32_t columns) {
  if (!prefill_q8_supported(dtype, head_size) || !prefill_q8_columns(columns)) return LVAMD_ERR_UNSUPPORTED;
  return dispatch_prefill(dtype, head_size, columns, []<typename T, int D, int CT, int W>() -> int {
    int device = 0, cus = 0, per_cu = 0;
    if (hipGetDevice(&device) != hipSuccess) return LVAMD_ERR_LAUNCH;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess)
      return LVAMD_ERR_LAUNCH;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, reinterpret_cast<const void*>(&q8_prefill_kernel<T, D, CT, W>),
                                                     64 * W, 0) != hipSuccess)
      return LVAMD_ERR_LAUNCH;
    return per_cu * cus;
  });
}

extern "C" int lvamd_paged_prefill_q8(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* key_pool,
                                      const float* key_scales, const void* value_pool, const float* value_scales,
                                      void* out, int64_t out_token_stride, int64_t out_head_stride,
                                      const int32_t* tables, const uint32_t* vis, const int32_t* units,
                                      int32_t num_units, void* part_acc, float* part_ml, int64_t num_partial_slots,
                                      int32_t num_kv_heads, int32_t group, int32_t head_size, int32_t columns,
                                      int32_t block_size, float scale, int32_t dtype, lvamd_stream_t stream) {
  if (!prefill_q8_supported(dtype, head_size) || !prefill_q8_columns(columns)) return LVAMD_ERR_UNSUPPORTED;
  if (num_units < 0 || num_kv_heads <= 0 || group <= 0 || block_size <= 0 || num_partial_slots < 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_units == 0) return LVAMD_OK;
  // (The running maximum is taken of the unscaled scores, masked ones -inf.)
  if (!(scale > 0.f)) return LVAMD_ERR_INVALID_ARGUMENT;
  if (!q || !key_pool || !key_scales || !value_pool || !value_scales || !out || !tables || !vis || !units)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_partial_slots > 0 && (!part_acc || !part_ml)) return LVAMD_ERR_WORKSPACE;
  if (((uintptr_t)q & 15u) || ((uintptr_t)key_pool & 15u) || ((uintptr_t)value_pool & 15u) || q_token_stride % 8 != 0 ||
      q_head_stride % 8 != 0 || ((uintptr_t)out & 7u) || out_token_stride % 4 != 0 || out_head_stride % 4 != 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if ((int64_t)num_units * num_kv_heads > 0x7fffffffLL) return LVAMD_ERR_INVALID_ARGUMENT;
  Q8PrefillArgs a{.by_block = FastDiv(block_size), .by_group = FastDiv(group)};
  a.q = q;
  a.q_tok_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.k_pool = static_cast<const uint8_t*>(key_pool);
  a.v_pool = static_cast<const uint8_t*>(value_pool);
  a.k_scales = key_scales;
  a.v_scales = value_scales;
  a.out = out;
  a.out_tok_stride = out_token_stride;
  a.out_head_stride = out_head_stride;
  a.tables = tables;
  a.vis = vis;
  a.part_acc = part_acc;
  a.part_ml = part_ml;
  a.group = group;
  a.block_size = block_size;
  a.scale_log2 = scale * 1.4426950408889634f;
  const FastDiv by_heads(num_kv_heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dispatch_prefill(dtype, head_size, columns, [&]<typename T, int D, int CT, int W>() -> int {
    hipLaunchKernelGGL((q8_prefill_kernel<T, D, CT, W>), dim3((unsigned)(num_units * num_kv_heads)), dim3(64 * W), 0, s,
                       units, num_kv_heads, by_heads.magic, by_heads.shift, a);
    return launch_status();
  });
}
