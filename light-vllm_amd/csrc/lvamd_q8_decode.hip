// Paged decode attention over the 8-bit cache on gfx950: requests whose
// queries x group fit one 16-column MFMA tile (single tokens, short trees).
//
// Semantics are the 16-bit decode kernel's (lvamd_decode.hip) with K and V the
// cache's values, code * scale.  The step's tokens are in the cache already
// (lvamd_kv_append_q8 ran), or the kernel appends them.  The work lists are the
// same too: stream-K pieces over the (request) segments, one wave64 per share,
// split segments merged by lvamd_paged_attention_merge_q8.
//
// Mapping onto CDNA4:
//   * A tile is TT tokens of one kv head, 16 KiB of K and V codes (TT = 64 at
//     D = 128).  Each load instruction reads whole rows, 16 codes per lane,
//     non-temporal; the next tile's loads are in flight while a tile computes.
//   * The codes become T in registers (one conversion instruction per two
//     codes applies the block's scale exactly, lvamd_q8.h) on their way to
//     LDS, so any block size works: each row has its own scale.  Keeping the
//     codes in LDS would halve its traffic, but the V operand holds eight keys
//     per lane, which would have to share one scale.
//   * One LDS tile per wave: a wave writes the next tile after its own reads of
//     the last one, in program order, so no second buffer and no barrier.
//   * Row r of a tile belongs to lane r % 64 for the block table, the slot and
//     the two scales (one load each per tile and wave; the table's a tile ahead
//     of the codes); the lanes that load or convert a row fetch them by shuffles.
//   * S^T = K Q^T and O^T = V^T P^T on MFMA 16x16x32, the online softmax in the
//     log2 domain with lazy rescaling: as in the 16-bit kernel.
//   * Append: with block sizes that divide the tile, each block that the step
//     writes lies in one tile, and a kv head's tile belongs to one wave: that
//     wave quantises the new rows, re-scales the block's others if its scale
//     grows and stores what changed, after it staged the tile (append_rows; one
//     tile per request and kv head).  It saves the append's launch, 3 us of
//     the 12 that a step of short sequences takes per layer, and costs more
//     than that in long ones: an instance of its own (APPEND).
//   * A row that some column does not see may hold NaN (a sibling's draft),
//     which a zero probability would not hide: rows of this step go to LDS
//     with NaN as zero, and the columns that do see such a row get it back
//     (poison, below; code that no ordinary step enters).
//
// HBM-bound in long steps, a chain of dependent round trips in short ones.  28
// heads over 4, D = 128: 64 sequences of 512-4095 tokens (bf16) 34 us for 159 MB,
// 4.7 TB/s; 16 of 32767 (fp16) 86-91 us for 537 MB, 5.9-6.2 TB/s.  4 sequences of
// 37-511 tokens, 14 heads over 2, D = 64: 8 us with the append.

#include <cmath>

#include "lvamd_q8.h"

namespace lvamd {

namespace {

constexpr float kSlack = 8.0f;  // lazy-rescale threshold, log2 units

struct Q8DecodeArgs {
  const void* q;
  int64_t q_tok_stride, q_head_stride;
  const void* k_new;  // this step's K/V [tokens][kv heads][D], or null: nothing to append
  const void* v_new;
  int64_t kn_tok_stride, kn_head_stride, vn_tok_stride, vn_head_stride;
  uint8_t* k_pool;
  uint8_t* v_pool;
  float* k_scales;
  float* v_scales;
  void* out;
  int64_t out_tok_stride, out_head_stride;
  const int32_t* __restrict__ tables;
  const uint32_t* __restrict__ vis;
  void* part_acc;
  float* part_ml;
  int32_t num_kv_heads;
  int32_t group;
  int32_t block_size;
  FastDiv by_block, by_group;
  float scale_log2;
};

template <int D>
struct Q8Tile {
  static constexpr int TT = D <= 64 ? 128 : D <= 128 ? 64 : 32;  // tokens
  static constexpr int SUB = TT / 16;
  static constexpr int C8 = D / 16;                     // 16-code chunks per row
  static constexpr int CPR = D / 8;                     // 16-byte chunks of T per row
  static constexpr int RS = q8_row_stride(CPR);         // LDS row stride in chunks
  static constexpr int LPT = (TT * C8 + 63) / 64;       // loads per lane and tensor
  static constexpr int SPL = (TT + 63) / 64;            // rows whose slot a lane holds
  static constexpr int NCH = (D + 31) / 32;             // MFMA k-steps of QK^T
  static constexpr int NT = D / 16;
};

struct Q8Piece {
  int tok_begin, tok_end, slot, table_off, computed, q_len, q_start, vis_off, vis_words;
};

__device__ __forceinline__ Q8Piece read_q8_piece(const int32_t* __restrict__ pieces, int p) {
  const int32_t* r = pieces + (int64_t)p * LVAMD_PIECE_FIELDS;
  return {r[2], r[3], r[4], r[5], r[6], r[7], r[8], r[9], r[10]};
}

}  // namespace

template <typename T, int D, bool APPEND>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(1, 1))) void q8_decode_kernel(
    const int32_t* __restrict__ wave_first, const int32_t* __restrict__ pieces, const int32_t waves_per_head,
    const uint32_t wg_magic, const int32_t wg_shift, const Q8DecodeArgs a) {
  using S = Q8Tile<D>;
  constexpr int TT = S::TT, SUB = S::SUB, C8 = S::C8, CPR = S::CPR, RS = S::RS, LPT = S::LPT, SPL = S::SPL;
  constexpr int NCH = S::NCH, NT = S::NT;
  using V8 = typename std::conditional<std::is_same<T, __bf16>::value, bf16x8, f16x8>::type;
  __shared__ __attribute__((aligned(16))) uint4 klds[TT * RS];
  __shared__ __attribute__((aligned(16))) uint4 vlds[TT * RS];

  const int lane = threadIdx.x & 63;
  const int l16 = lane & 15;
  const int g = lane >> 4;
  const int Hkv = a.num_kv_heads;
  const int G = a.group;
  const int kvh = fast_div((int)blockIdx.x, wg_magic, wg_shift);
  const int w = (int)blockIdx.x - kvh * waves_per_head;
  int p = wave_first[w];
  const int p_end = wave_first[w + 1];
  if (p >= p_end) return;
  const int64_t row_bytes = (int64_t)Hkv * D;
  gptr<uint8_t> const kbase = (gptr<uint8_t>)(a.k_pool) + (int64_t)kvh * D;
  gptr<uint8_t> const vbase = (gptr<uint8_t>)(a.v_pool) + (int64_t)kvh * D;
  gptr<float> const kscales = (gptr<float>)(a.k_scales) + kvh;
  gptr<float> const vscales = (gptr<float>)(a.v_scales) + kvh;

  // This lane's rows of a tile: their blocks and offsets in them.  (The slot is
  // made of them where the codes are requested: here it would wait for the
  // table's load, and with it for the tile's loads before it.)  Rows past the
  // piece repeat its last one.
  struct Rows {
    int block[SPL], off[SPL];
  };
  auto lookup = [&](int table_off, int t0, int tok_end) -> Rows {
    Rows r;
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      const int pos = min(t0 + 64 * i + lane, tok_end - 1);
      const int lb = fast_div(pos, a.by_block);
      r.block[i] = a.tables[table_off + lb];
      r.off[i] = pos - lb * a.block_size;
    }
    return r;
  };
  auto shuffled = [&](const auto (&v)[SPL], int row) {
    auto x = __shfl(v[0], row & 63);
#pragma unroll
    for (int i = 1; i < SPL; ++i) {
      const auto y = __shfl(v[i], row & 63);
      x = row >= 64 * i ? y : x;
    }
    return x;
  };
  // Chunk id lane + 64 j of a tile: row id / C8, chunk id % C8.
  struct Tile {
    uint4 k[LPT], v[LPT];
    float ks[SPL], vs[SPL];
  };
  auto issue = [&](const Rows& r, Tile& t) {
    // (The scales first: loads return in order, and every row's conversion
    // needs one.)
    int slot[SPL];
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      slot[i] = r.block[i] * a.block_size + r.off[i];
      const int64_t at = (int64_t)r.block[i] * Hkv;
      t.ks[i] = kscales[at];
      t.vs[i] = vscales[at];
    }
#pragma unroll
    for (int j = 0; j < LPT; ++j) {
      const int id = lane + 64 * j;
      const int row = id / C8, c = id - row * C8;
      const int64_t off = (int64_t)shuffled(slot, row & (TT - 1)) * row_bytes + 16 * c;
      t.k[j] = t.v[j] = zero_u4();
      if (64 * LPT == TT * C8 || row < TT) {
        t.k[j] = load16_stream((gptr<const uint8_t>)(kbase + off));
        t.v[j] = load16_stream((gptr<const uint8_t>)(vbase + off));
      }
    }
  };
  // Tile into LDS as T.  NEW: rows from first_new on hold this step's tokens, or
  // are past the end.  Their V rows' NaN values are left out (returns whether
  // there were any); zeros, where this launch has yet to write them.
  auto stage_rows = [&]<bool NEW>(const Tile& t, int first_new) __attribute__((always_inline)) -> bool {
    bool any = false;
#pragma unroll
    for (int j = 0; j < LPT; ++j) {
      const int id = lane + 64 * j;
      const int row = id / C8, c = id - row * C8;
      const float ks = shuffled(t.ks, row & (TT - 1));
      float vs = shuffled(t.vs, row & (TT - 1));
      uint4 v = t.v[j];
      if constexpr (NEW) {
        if (APPEND && row >= first_new) {
          v = zero_u4();
          vs = 0.f;
        }
        const bool nan = row >= first_new && q8_has_nan(v);
        any |= nan;
        if (nan) v = q8_without_nan16(v);
      }
      uint4 klo, khi, vlo, vhi;
      q8_values16<T>(t.k[j], ks, klo, khi);
      q8_values16<T>(v, vs, vlo, vhi);
      if (64 * LPT == TT * C8 || row < TT) {
        klds[row * RS + 2 * c] = klo;
        klds[row * RS + 2 * c + 1] = khi;
        vlds[row * RS + 2 * c] = vlo;
        vlds[row * RS + 2 * c + 1] = vhi;
      }
    }
    return NEW && __any(any);
  };
  // 16 elements of a new token's K and V row.
  struct Raw {
    uint4 k0, k1, v0, v1;
  };
  auto load_new = [&](int tok, int c) -> Raw {
    gptr<const T> const k = (gptr<const T>)(a.k_new) + (int64_t)tok * a.kn_tok_stride + kvh * a.kn_head_stride + 16 * c;
    gptr<const T> const v = (gptr<const T>)(a.v_new) + (int64_t)tok * a.vn_tok_stride + kvh * a.vn_head_stride + 16 * c;
    return {load16(k), load16(k + 8), load16(v), load16(v + 8)};
  };
  // The piece's new rows of the tile at t0 (at most 16: a piece has no more
  // queries), after the tile was staged without them: into the cache, and into
  // LDS as they are stored.  Loops, not unrolled: a launch pays for code that it
  // fetches, and waves that append do it once or twice.
  auto append_rows = [&](const Tile& t, const Rows& rows, const Q8Piece& x, int t0)
      __attribute__((always_inline)) -> bool {
    const int row0 = max(x.computed - t0, 0), end = min(x.tok_end - t0, TT);
    const int n = end - row0;
    const int tok0 = x.q_start + t0 - x.computed;  // row r is token tok0 + r
    const int block0 = fast_div(row0, a.by_block), begin0 = block0 * a.block_size;
    const int blocks = fast_div(end - 1, a.by_block) - block0 + 1;
    const Raw raw = load_new(tok0 + row0 + min(lane, n * C8 - 1) / C8, min(lane, n * C8 - 1) % C8);
    // Lane b < blocks is at block block0 + b.  Only the first may hold earlier rows.
    const bool first = lane == 0 && begin0 < x.computed - t0;
    const int from = min((block0 + lane) * a.block_size, end - 1);
    const int block = shuffled(rows.block, from);
    const int64_t at = (int64_t)block * Hkv;
    const float kheld = shuffled(t.ks, from), vheld = shuffled(t.vs, from);
    const float kold = first ? kheld : 0.f, vold = first ? vheld : 0.f;
    // Each block's largest magnitudes, in the first new rows' place.
    static_assert(D >= 32, "16 words in a row");
    uint32_t* const kmax = reinterpret_cast<uint32_t*>(klds + row0 * RS);
    uint32_t* const vmax = reinterpret_cast<uint32_t*>(vlds + row0 * RS);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < 16) kmax[lane] = vmax[lane] = 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // (All lanes take part in each pass, the last chunk's again past the end: the
    // shuffles read any of them.)
    Raw e = raw;
#pragma unroll 1
    for (int i = 0;;) {
      const int row = row0 + min(i + lane, n * C8 - 1) / C8;
      const int b = fast_div(row, a.by_block) - block0;
      atomicMax(kmax + b, q8_largest16<T>(e.k0, e.k1));
      atomicMax(vmax + b, q8_largest16<T>(e.v0, e.v1));
      if ((i += 64) >= n * C8) break;
      const int id = min(i + lane, n * C8 - 1);
      e = load_new(tok0 + row0 + id / C8, id % C8);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const float kscale = fmaxf(kold, q8_scale(__uint_as_float(kmax[lane & 15])));
    const float vscale = fmaxf(vold, q8_scale(__uint_as_float(vmax[lane & 15])));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < blocks) {
      kscales[at] = kscale;
      vscales[at] = vscale;
    }
    bool nan = false;
    e = raw;
#pragma unroll 1
    for (int i = 0;;) {
      const int id = min(i + lane, n * C8 - 1);
      const int row = row0 + id / C8, c = id % C8;
      const int lb = fast_div(row, a.by_block), b = lb - block0;
      const float ks = __shfl(kscale, b), vs = __shfl(vscale, b);
      const int64_t off = ((int64_t)__shfl(block, b) * a.block_size + (row - lb * a.block_size)) * row_bytes + 16 * c;
      const uint4 kc = q8_codes16<T>(e.k0, e.k1, ks);
      uint4 vc = q8_codes16<T>(e.v0, e.v1, vs);
      store16(kbase + off, kc);
      store16(vbase + off, vc);
      nan |= q8_has_nan(vc);
      vc = q8_without_nan16(vc);
      uint4* const kto = klds + row * RS + 2 * c;
      uint4* const vto = vlds + row * RS + 2 * c;
      q8_values16<T>(kc, ks, kto[0], kto[1]);
      q8_values16<T>(vc, vs, vto[0], vto[1]);
      if ((i += 64) >= n * C8) break;
      const int next = min(i + lane, n * C8 - 1);
      e = load_new(tok0 + row0 + next / C8, next % C8);
    }
    // The first block's other rows, where its scale grew.
    if (__any(first && (kscale > kold || vscale > vold))) {
      const float ks = __shfl(kscale, 0), vs = __shfl(vscale, 0);
      const float kratio = __shfl(kold, 0) * q8_inverse(ks), vratio = __shfl(vold, 0) * q8_inverse(vs);
      const int64_t slot0 = (int64_t)__shfl(block, 0) * a.block_size;
#pragma unroll 1
      for (int id = lane; id < a.block_size * C8; id += 64) {
        const int r = id / C8, c = id % C8;
        const int row = begin0 + r;
        if (row >= row0 && row < end) continue;
        const int64_t off = (slot0 + r) * row_bytes + 16 * c;
        const uint4 kc = q8_rescale16(load16((gptr<const uint8_t>)(kbase + off)), kratio);
        const uint4 vc = q8_rescale16(load16((gptr<const uint8_t>)(vbase + off)), vratio);
        if (kratio < 1.f) store16(kbase + off, kc);
        if (vratio < 1.f) store16(vbase + off, vc);
        if (row >= row0) continue;  // (past the tokens: stale)
        uint4* const kto = klds + row * RS + 2 * c;
        uint4* const vto = vlds + row * RS + 2 * c;
        q8_values16<T>(kc, ks, kto[0], kto[1]);
        q8_values16<T>(vc, vs, vto[0], vto[1]);
      }
    }
    return __any(nan);
  };

  // This lane's column: query qi, head qhead, and which of the step's tokens
  // it sees (bit j; a piece has at most 16 queries).
  struct Column {
    int qi, qhead;
    bool ok;
    uint32_t sees;
  };
  auto column = [&](const Q8Piece& x) -> Column {
    Column c;
    const int ncols = x.q_len * G;
    c.ok = l16 < ncols;
    const int col = c.ok ? l16 : ncols - 1;
    c.qi = fast_div(col, a.by_group);
    c.qhead = kvh * G + (col - c.qi * G);
    c.sees = x.vis_off >= 0 ? a.vis[x.vis_off + c.qi * x.vis_words] : (2u << c.qi) - 1u;
    return c;
  };
  auto load_q = [&](const Q8Piece& x, const Column& c, uint4 (&q)[NCH]) {
    const T* row = static_cast<const T*>(a.q) + (int64_t)(x.q_start + c.qi) * a.q_tok_stride +
                   (int64_t)c.qhead * a.q_head_stride;
#pragma unroll
    for (int kk = 0; kk < NCH; ++kk) {
      const int ch = kk * 4 + g;
      q[kk] = c.ok && ch < CPR ? load16(row + ch * 8) : zero_u4();
    }
  };

  // Tiles in order over the wave's pieces.  The cursor is at the tile whose rows
  // were looked up last: two ahead of the one that computes.
  struct Cursor {
    int p, table_off, t0, tok_end;
  };
  auto advance = [&](Cursor& c) {
    c.t0 += TT;
    if (c.t0 >= c.tok_end && ++c.p < p_end) {
      const int32_t* r = pieces + (int64_t)c.p * LVAMD_PIECE_FIELDS;
      c.t0 = r[2];
      c.tok_end = r[3];
      c.table_off = r[5];
    }
  };

  Q8Piece cur = read_q8_piece(pieces, p);
  Cursor at = {p, cur.table_off, cur.tok_begin, cur.tok_end};
  Rows rows = lookup(at.table_off, at.t0, at.tok_end);
  Tile tile;
  issue(rows, tile);
  Rows staged = rows;
  Column col = column(cur);
  uint4 qf[NCH];
  load_q(cur, col, qf);
  advance(at);
  if (at.p < p_end) rows = lookup(at.table_off, at.t0, at.tok_end);
  int t0 = cur.tok_begin;

  float m_run = -INFINITY, l_run = 0.f;
  f32x4 acc[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};

  Q8Piece nxt = cur;
  Column ncol = col;
  uint4 qn[NCH];
  while (true) {
    bool poisoned = false;
    if (const int first_new = cur.computed - t0; first_new >= TT) {
      stage_rows.template operator()<false>(tile, first_new);
    } else {
      poisoned = stage_rows.template operator()<true>(tile, first_new);
      if constexpr (APPEND) poisoned = append_rows(tile, staged, cur, t0);
    }
    // The next tile's codes, the rows of the one after it and, where the next
    // tile starts a piece, that piece's record and queries.
    const bool has_next = at.p < p_end;
    const bool ends = at.p != p;  // the tile in LDS is its piece's last
    const int nt0 = at.t0;
    if (has_next) {
      issue(rows, tile);
      staged = rows;
      if (ends) {
        p = at.p;
        nxt = read_q8_piece(pieces, p);
        ncol = column(nxt);
        load_q(nxt, ncol, qn);
      }
      advance(at);
      if (at.p < p_end) rows = lookup(at.table_off, at.t0, at.tok_end);
    }

    // ---- scores of the tile in LDS
    f32x4 st[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      st[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < NCH; ++kk) {
        const int ch = kk * 4 + g;
        const uint4 k = (CPR % 4 == 0 || ch < CPR) ? klds[(16 * s + l16) * RS + ch] : zero_u4();
        st[s] = Mma<T>::qk(k, qf[kk], st[s]);
      }
    }
    // Masks, only in tiles that reach the step's tokens or the piece's end.
    const int limit = min(cur.computed, cur.tok_end);
    if (t0 + TT > limit) {
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int pos = t0 + 16 * s + 4 * g + r;
          const int j = pos - cur.computed;
          const bool seen = (int)(j < 0) | (int)((col.sees >> (j & 31)) & 1u);
          const bool vis = (int)seen & (int)(pos < cur.tok_end);
          st[s][r] = vis ? st[s][r] * a.scale_log2 : -INFINITY;
        }
    } else {
#pragma unroll
      for (int s = 0; s < SUB; ++s) st[s] *= a.scale_log2;
    }
    float mt = -INFINITY;
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) mt = fmaxf(mt, st[s][r]);
    mt = row_max4(mt);
    if (__any(mt > m_run + kSlack)) {
      const float m_new = fmaxf(m_run, mt);
      const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n] *= alpha;
      m_run = m_new;
    }
    const float base = m_run == -INFINITY ? 0.f : -m_run;
    V8 pb[SUB / 2];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // The weights are rounded to T for the products with V (a matrix
        // instruction's operands are of one type; bf16 output is off by 1.3 times
        // its own rounding in all, twice the products would spare 0.3); the sum that
        // divides them counts them as rounded, so a weight's rounding moves the
        // result by its share of v - out, not of v.
        const T pr = from_f32<T>(fast_exp2(st[s][r] + base));
        l_run += to_f32(pr);
        pb[s >> 1][(s & 1) * 4 + r] = pr;
      }
    // ---- O^T += V^T P^T, V^T by transpose reads
    const char* vbytes = reinterpret_cast<const char*>(vlds);
    const int q4 = l16 & 3;
#pragma unroll
    for (int hh = 0; hh < SUB / 2; ++hh)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int lo = ((32 * hh + 4 * g + (l16 >> 2)) * RS + 2 * n + (q4 >> 1)) * 16 + (q4 & 1) * 8;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vbytes + lo));
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vbytes + lo + 16 * RS * 16));
        const s16x4 both[2] = {v0, v1};
        if constexpr (std::is_same<T, __bf16>::value) {
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<V8>(both), pb[hh], acc[n], 0, 0, 0);
        } else {
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<V8>(both), pb[hh], acc[n], 0, 0, 0);
        }
      }
    if (poisoned) {
      // NaN values of this step's tokens: every column that sees the row gets
      // NaN in that element, as 0 * NaN would give.
      for (int pos = max(t0, cur.computed); pos < min(t0 + TT, cur.tok_end); ++pos) {
        const int lb = fast_div(pos, a.by_block);
        const int64_t slot = (int64_t)a.tables[cur.table_off + lb] * a.block_size + (pos - lb * a.block_size);
        const bool sees = (col.sees >> ((pos - cur.computed) & 31)) & 1u;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t nan;
          if constexpr (APPEND) {  // (the token's own values: the codes' stores may be on their way)
            const int64_t tok = cur.q_start + pos - cur.computed;
            const T* const v = static_cast<const T*>(a.v_new) + tok * a.vn_tok_stride + kvh * a.vn_head_stride;
            nan = q8_nan4_of<T>(*reinterpret_cast<const uint2*>(v + 16 * n + 4 * g));
          } else {
            nan = q8_nan4(*(gptr<const uint32_t>)(vbase + slot * row_bytes + 16 * n + 4 * g));
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (sees && ((nan >> (8 * r + 7)) & 1u)) acc[n][r] = __uint_as_float(0x7fc00000u);
        }
      }
    }

    // ---- a finished piece: its output rows, or its partials
    if (ends) {
      const float l_tot = row_sum4(l_run);
      const float inv = l_tot > 0.f ? 1.f / l_tot : 0.f;
      if (col.ok) {
        if (cur.slot < 0) {
          T* row = static_cast<T*>(a.out) + (int64_t)(cur.q_start + col.qi) * a.out_tok_stride +
                   (int64_t)col.qhead * a.out_head_stride;
#pragma unroll
          for (int n = 0; n < NT; ++n) store_partial4<false, T>(row + 16 * n + 4 * g, acc[n], l_tot == l_tot ? inv : l_tot);
        } else {
          const int64_t cs = ((int64_t)cur.slot * Hkv + kvh) * 16 + l16;
          float* row = static_cast<float*>(a.part_acc) + cs * D;
#pragma unroll
          for (int n = 0; n < NT; ++n)
            store_partial4<false, float>(row + 16 * n + 4 * g, acc[n], l_tot == l_tot ? inv : l_tot);
          // (A NaN sum keeps a finite maximum: the merge passes over a
          // partial whose maximum is -inf.)
          const float m = l_tot == l_tot || m_run != -INFINITY ? m_run : 0.f;
          if (g == 0) *reinterpret_cast<float2*>(a.part_ml + cs * 2) = make_float2(m, l_tot);
        }
      }
      if (!has_next) break;
      cur = nxt;
      col = ncol;
#pragma unroll
      for (int kk = 0; kk < NCH; ++kk) qf[kk] = qn[kk];
      m_run = -INFINITY;
      l_run = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    t0 = nt0;
  }
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace lvamd

using namespace lvamd;

extern "C" int lvamd_paged_decode_q8(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* new_key,
                                     int64_t new_key_token_stride, int64_t new_key_head_stride, const void* new_value,
                                     int64_t new_value_token_stride, int64_t new_value_head_stride, void* key_pool,
                                     float* key_scales, void* value_pool, float* value_scales, void* out,
                                     int64_t out_token_stride, int64_t out_head_stride, const int32_t* pieces,
                                     const int32_t* wave_first, int32_t waves_per_head, const int32_t* tables,
                                     const uint32_t* vis, void* part_acc, float* part_ml,
                                     int64_t num_partial_slots, int32_t num_kv_heads, int32_t group, int32_t head_size,
                                     int32_t block_size, float scale, int32_t dtype, lvamd_stream_t stream) {
  if ((dtype != LVAMD_BF16 && dtype != LVAMD_F16) || !q8_head_size(head_size)) return LVAMD_ERR_UNSUPPORTED;
  if (waves_per_head < 0 || num_kv_heads <= 0 || group <= 0 || group > 16 || block_size <= 0 || num_partial_slots < 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (waves_per_head == 0) return LVAMD_OK;
  if (!q || !key_pool || !key_scales || !value_pool || !value_scales || !out || !pieces || !wave_first || !tables || !vis)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_partial_slots > 0 && (!part_acc || !part_ml)) return LVAMD_ERR_WORKSPACE;
  if (!aligned16(q) || !aligned16(key_pool) || !aligned16(value_pool) || q_token_stride % 8 != 0 ||
      q_head_stride % 8 != 0 || ((uintptr_t)out & 7u) != 0 || out_token_stride % 4 != 0 || out_head_stride % 4 != 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if ((new_key == nullptr) != (new_value == nullptr)) return LVAMD_ERR_INVALID_ARGUMENT;
  // Appending needs whole blocks per tile.
  if (new_key && (!aligned16(new_key) || !aligned16(new_value) || new_key_token_stride % 8 != 0 ||
                  new_key_head_stride % 8 != 0 || new_value_token_stride % 8 != 0 || new_value_head_stride % 8 != 0 ||
                  lvamd_paged_decode_q8_tile_tokens(dtype, head_size) % block_size != 0))
    return LVAMD_ERR_INVALID_ARGUMENT;
  if ((int64_t)waves_per_head * num_kv_heads > 0x7fffffffLL) return LVAMD_ERR_INVALID_ARGUMENT;
  Q8DecodeArgs a{.by_block = FastDiv(block_size), .by_group = FastDiv(group)};
  a.q = q;
  a.q_tok_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.k_new = new_key;
  a.v_new = new_value;
  a.kn_tok_stride = new_key_token_stride;
  a.kn_head_stride = new_key_head_stride;
  a.vn_tok_stride = new_value_token_stride;
  a.vn_head_stride = new_value_head_stride;
  a.k_pool = static_cast<uint8_t*>(key_pool);
  a.v_pool = static_cast<uint8_t*>(value_pool);
  a.k_scales = key_scales;
  a.v_scales = value_scales;
  a.out = out;
  a.out_tok_stride = out_token_stride;
  a.out_head_stride = out_head_stride;
  a.tables = tables;
  a.vis = vis;
  a.part_acc = part_acc;
  a.part_ml = part_ml;
  a.num_kv_heads = num_kv_heads;
  a.group = group;
  a.block_size = block_size;
  a.scale_log2 = scale * 1.4426950408889634f;
  const dim3 grid((unsigned)(waves_per_head * num_kv_heads));
  const FastDiv by_waves(waves_per_head);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return q8_dispatch(dtype, head_size, [&]<typename T, int D>() -> int {
    hipLaunchKernelGGL((new_key ? q8_decode_kernel<T, D, true> : q8_decode_kernel<T, D, false>), grid, dim3(64), 0, s,
                       wave_first, pieces, waves_per_head, by_waves.magic, by_waves.shift, a);
    return launch_status();
  });
}

extern "C" int lvamd_paged_decode_q8_tile_tokens(int32_t dtype, int32_t head_size) {
  return q8_dispatch(dtype, head_size, []<typename T, int D>() -> int { return Q8Tile<D>::TT; });
}

extern "C" int lvamd_paged_decode_q8_resident_waves(int32_t dtype, int32_t head_size) {
  return q8_dispatch(dtype, head_size, []<typename T, int D>() -> int {
    int device = 0, cus = 0, per_cu = 0;
    if (hipGetDevice(&device) != hipSuccess) return LVAMD_ERR_LAUNCH;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess)
      return LVAMD_ERR_LAUNCH;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(
            &per_cu, reinterpret_cast<const void*>(&q8_decode_kernel<T, D, false>), 64, 0) != hipSuccess)
      return LVAMD_ERR_LAUNCH;
    return per_cu * cus;
  });
}
