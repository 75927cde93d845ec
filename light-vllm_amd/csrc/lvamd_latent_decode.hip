// Attention over a paged cache of latent vectors on gfx950, in latent space
// (the absorbed form): head h's query, multiplied by its key weights already,
// meets the rows themselves,
//   s = scale (q[0..L) . c + q[L..L+P) . r),   out = sum softmax(s) c,
// so all heads share one key of L + P values and one value of L of them.
//
// Query j of a request with c computed tokens sees logical positions [0, c) and
// {c + i : i <= j} (linear) or {c + i : i an ancestor of j, or j} (tree).  The
// step's tokens are in the cache already.
//
// Mapping onto CDNA4:
//   * A column is a (query, head) pair of one request; a workgroup of four waves
//     holds up to 16 NC of them and walks over tiles of 32 rows: stream-K pieces
//     of (request, column group) segments, split segments merged below.
//   * The rows of a tile are loaded once, straight into LDS (global_load_lds, no
//     registers), while the tile before is computed; they serve as keys (rows
//     read as they lie) and as values (transpose reads).
//   * Scores: S^T = K Q^T on MFMA 16x16x32, the 16-row halves of the tile and the
//     column tiles dealt to the waves, queries in registers.  Products: O^T = V^T
//     P^T, a quarter of the latent's dimensions per wave for all columns, so an
//     accumulator takes a quarter of the registers that a whole row would, and
//     each value is read from LDS once.  The probabilities cross over through
//     LDS (the accumulator layout of S^T is the operand layout of P^T).
//   * The waves share each column's running maximum, which moves only when some
//     score passes it by 2^8 (lazy rescaling): a vote per tile in LDS.
//   * A tile has two barriers: its rows are there, its probabilities are there.
//
// LDS tile layout: groups of 64 columns (128 bytes of every row), group-major;
// one load of a wave fills 1 KB = 8 whole 128-byte lines of one group.  Chunk c
// of row r lies in slot c ^ f(r), f = 2 (r2 | (r3 ^ r1) << 1) in the bits of r:
// the key reads (16 rows, 2 chunks) and the transpose reads (8 rows, 32 bytes)
// then cover every bank once.

#include <cmath>

#include "lvamd_latent.h"

namespace lvamd {

namespace {

constexpr float kSlack = 8.0f;  // lazy-rescale threshold, log2 units
constexpr int KT = 32;          // rows per tile
constexpr int kWaves = 4;

typedef const __attribute__((address_space(1))) void* lds_gptr;
typedef __attribute__((address_space(3))) void* lds_lptr;

struct LatentDecodeArgs {
  const void* q;  // [tokens][heads][L], the latent part
  int64_t q_tok_stride, q_head_stride;
  const void* qr;  // [tokens][heads][P], the rotated part
  int64_t qr_tok_stride, qr_head_stride;
  const void* pool;  // [slots][L + P]
  void* out;         // [tokens][heads][L]
  int64_t out_tok_stride, out_head_stride;
  const int32_t* __restrict__ tables;
  const uint32_t* __restrict__ vis;
  float* part_acc;  // [slots][16 NC][L] fp32, rows normalised
  float* part_ml;   // [slots][16 NC][2]: (max, sum)
  int32_t heads, block_size;
  FastDiv by_block, by_heads;
  float scale_log2;
};

struct LatentPiece {
  int group, tok_begin, tok_end, slot, table_off, computed, q_len, q_start, vis_off, vis_words;
};
__device__ __forceinline__ LatentPiece read_latent_piece(const int32_t* __restrict__ pieces, int p) {
  const int32_t* r = pieces + (int64_t)p * LVAMD_PIECE_FIELDS;
  return {r[1], r[2], r[3], r[4], r[5], r[6], r[7], r[8], r[9], r[10]};
}

__device__ __forceinline__ constexpr int swizzle(int row) {
  return (((row >> 2) & 1) << 1) | ((((row >> 3) ^ (row >> 1)) & 1) << 2);
}

// Orders LDS accesses around a workgroup barrier (global loads stay in flight).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int L, int P, int NC>
struct LatentShape {
  static constexpr int ROW = L + P;                   // elements
  static constexpr int CPR = ROW / 8;                 // 16-byte chunks of a row
  static constexpr int GR = (CPR + 7) / 8;            // 128-byte groups
  static constexpr int TILE_BYTES = GR * KT * 128;
  static constexpr int KSTEPS = ROW / 32;             // MFMA steps of a score
  static constexpr int DT = L / 64;                   // 16-dimension tiles per wave
  static constexpr int QKS = NC == 8 ? 2 : 1;         // 16-row halves a wave scores
  static constexpr int QCT = NC >= 4 ? 2 : 1;         // column tiles a wave scores
  static constexpr int REGS = DT * NC * 4 + QCT * KSTEPS * 4;  // accumulators and queries
  static constexpr int WAVES_PER_EU = REGS <= 176 ? 2 : 1;
  static_assert(L % 128 == 0 && P % 32 == 0);
};

template <typename T>
__device__ __forceinline__ bool not_finite(T x) {
  return !(__builtin_fabsf(to_f32(x)) < INFINITY);
}

}  // namespace

template <typename T, int L, int P, int NC>
__global__ __launch_bounds__(64 * kWaves)
__attribute__((amdgpu_waves_per_eu(LatentShape<L, P, NC>::WAVES_PER_EU))) void latent_decode_kernel(
    const int32_t* __restrict__ wave_first, const int32_t* __restrict__ pieces, const LatentDecodeArgs a) {
  using S = LatentShape<L, P, NC>;
  constexpr int GR = S::GR, KSTEPS = S::KSTEPS, DT = S::DT, QKS = S::QKS, QCT = S::QCT;
  constexpr int COLS = 16 * NC;
  using V8 = typename std::conditional<std::is_same<T, __bf16>::value, bf16x8, f16x8>::type;
  // Separate objects: a load into one does not alias a read of another.
  __shared__ __attribute__((aligned(1024))) char tile0[S::TILE_BYTES];
  __shared__ __attribute__((aligned(1024))) char tile1[S::TILE_BYTES];
  __shared__ __attribute__((aligned(16))) uint2 probs[NC * 64 * 2];  // [column tile][lane][half]
  __shared__ float tile_max[2][COLS], col_max[COLS], col_sum[2][COLS];
  __shared__ __attribute__((aligned(16))) uint32_t votes[kWaves];

  const int tid = threadIdx.x & (64 * kWaves - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int l16 = lane & 15;
  const int g = lane >> 4;
  int p = wave_first[blockIdx.x];
  const int p_end = wave_first[blockIdx.x + 1];
  if (p >= p_end) return;

  // ---- this wave's scores: rows [16 ks0, 16 (ks0 + QKS)) of a tile, column
  // tiles ct0 .. ct0 + QCT.
  const bool scores = NC > 1 || wave < 2;
  const int ks0 = NC == 8 ? 0 : wave & 1;
  const int ct0 = NC == 1 ? 0 : NC == 8 ? 2 * wave : QCT * (wave >> 1);

  // ---- tile loads: wave w loads rows 8 w .. 8 w + 7, lane l row 8 w + l / 8
  // into chunk slot l % 8 of every group.
  const int lrow = 8 * wave + (lane >> 3);
  const int lchunk = (lane & 7) ^ swizzle(lrow);
  struct Row {
    int entry, off;
  };
  auto lookup = [&](int table_off, int t0, int tok_end) -> Row {
    const int pos = min(t0 + lrow, tok_end - 1);
    const int lb = fast_div(pos, a.by_block);
    return {a.tables[table_off + lb], pos - lb * a.block_size};
  };
  gptr<const T> const pool = (gptr<const T>)(a.pool);
  auto issue = [&](const Row& r, char* dst) {
    gptr<const T> const row = pool + ((int64_t)r.entry * a.block_size + r.off) * S::ROW;
#pragma unroll
    for (int i = 0; i < GR; ++i) {
      int c = 8 * i + lchunk;
      // (A half-used last group's spare slots take the row's last chunks again.)
      if (8 * GR > S::CPR && i == GR - 1) c = min(c, S::CPR - 1);
      __builtin_amdgcn_global_load_lds((lds_gptr)(row + 8 * c), (lds_lptr)(dst + i * KT * 128 + wave * 1024), 16, 0, 0);
    }
  };

  // ---- columns: queries in registers, what each sees of the step's tokens
  struct Columns {
    int qi[QCT], head[QCT];
    bool ok[QCT];
  };
  auto columns = [&](const LatentPiece& x, int ct, int& qi, int& head) -> bool {
    const int col = x.group * COLS + 16 * ct + l16, ncols = x.q_len * a.heads;
    const bool ok = col < ncols;
    const int c = ok ? col : ncols - 1;
    qi = fast_div(c, a.by_heads);
    head = c - qi * a.heads;
    return ok;
  };
  // Bit k: whether query qi sees the tile's row k (rows of the step only;
  // earlier ones are seen by all, those past the piece by none).
  auto window = [&](const LatentPiece& x, int qi, int t0) -> uint32_t {
    const int j0 = t0 - x.computed;
    uint32_t bits;
    if (x.vis_off < 0) {
      const int n = qi - j0 + 1;
      bits = n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u;
    } else {
      const int w0 = j0 >> 5;
      const uint32_t* row = a.vis + x.vis_off + (int64_t)qi * x.vis_words;
      const uint32_t lo = w0 < 0 ? ~0u : w0 < x.vis_words ? row[w0] : 0u;
      const uint32_t hi = w0 + 1 < 0 ? ~0u : w0 + 1 < x.vis_words ? row[w0 + 1] : 0u;
      bits = __builtin_amdgcn_alignbit(hi, lo, j0 & 31);
    }
    const int left = x.tok_end - t0;
    return left >= 32 ? bits : bits & ((1u << left) - 1u);
  };

  LatentPiece cur = read_latent_piece(pieces, p);
  uint4 qf[QCT][KSTEPS];
  Columns col;
  auto load_queries = [&](const LatentPiece& x) {
#pragma unroll
    for (int c = 0; c < QCT; ++c) {
      col.ok[c] = columns(x, ct0 + c, col.qi[c], col.head[c]);
      const T* q = static_cast<const T*>(a.q) + (int64_t)(x.q_start + col.qi[c]) * a.q_tok_stride +
                   (int64_t)col.head[c] * a.q_head_stride;
      const T* qr = static_cast<const T*>(a.qr) + (int64_t)(x.q_start + col.qi[c]) * a.qr_tok_stride +
                    (int64_t)col.head[c] * a.qr_head_stride;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        const T* from = 32 * k < L ? q + 32 * k + 8 * g : qr + 32 * k - L + 8 * g;
        qf[c][k] = scores && col.ok[c] ? load16(from) : zero_u4();
      }
    }
  };

  // The cursor is at the tile whose rows were looked up last, one ahead of the
  // one in flight.
  struct Cursor {
    int p, table_off, t0, tok_end;
  };
  auto advance = [&](Cursor& c) {
    c.t0 += KT;
    if (c.t0 >= c.tok_end && ++c.p < p_end) {
      const int32_t* r = pieces + (int64_t)c.p * LVAMD_PIECE_FIELDS;
      c.t0 = r[2];
      c.tok_end = r[3];
      c.table_off = r[5];
    }
  };
  Cursor at = {p, cur.table_off, cur.tok_begin, cur.tok_end};
  Row row = lookup(at.table_off, at.t0, at.tok_end);
  issue(row, tile0);
  advance(at);
  if (at.p < p_end) row = lookup(at.table_off, at.t0, at.tok_end);

  float m_run[QCT], l_run[QCT];
  f32x4 acc[NC][DT];
  int t0 = cur.tok_begin;
  bool fresh = true;  // the tile is its piece's first

  // LDS offsets of this lane: key reads (row l16 + 16 ks, chunk 4 k + g) and
  // transpose reads (row 4 g + l16 / 4, +16; 8 bytes of dimensions 16 n + 4 q4).
  const int kbase = l16 * 128;
  const int kslot[2] = {16 * (g ^ swizzle(l16)), 16 * ((4 + g) ^ swizzle(l16))};
  const int vrow = 4 * g + (l16 >> 2);
  const int q4 = l16 & 3;
  auto vaddr = [&](const char* tile, int n) -> const char* {
    const int c = 2 * (wave * DT + n) + (q4 >> 1);
    return tile + (c >> 3) * (KT * 128) + vrow * 128 + 16 * ((c & 7) ^ swizzle(vrow)) + 8 * (q4 & 1);
  };

  // One tile from `here` while the next lands in `there`; false: it was the last.
  auto step = [&](const char* here, char* there) __attribute__((always_inline)) -> bool {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part of the tile
    lds_barrier();                       // everyone's, and the last tile's reads are done
    const bool has_next = at.p < p_end;
    const bool ends = at.p != p;  // the tile is its piece's last
    const int nt0 = at.t0, np = at.p;
    if (has_next) {
      issue(row, there);
      advance(at);
      if (at.p < p_end) row = lookup(at.table_off, at.t0, at.tok_end);
    }
    if (fresh) {
      load_queries(cur);
#pragma unroll
      for (int c = 0; c < QCT; ++c) {
        m_run[c] = -INFINITY;
        l_run[c] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int n = 0; n < DT; ++n) acc[c][n] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (tid < COLS) col_max[tid] = -INFINITY;
      fresh = false;
    }
    const bool masked = t0 + KT > min(cur.computed, cur.tok_end);

    // ---- scores
    f32x4 st[QCT][QKS];
    bool vote = false, odd = false;
    if (scores) {
      // LDS reads run LEAD ahead of the matrix instructions (held there by
      // scheduling barriers: left alone the scheduler hoists them all and the
      // wide instances spill).
      constexpr int TOT = QKS * KSTEPS, LEAD = 4;
      auto rd = [&](int i) -> uint4 {
        const int s = i / KSTEPS, k = i % KSTEPS;
        return *reinterpret_cast<const uint4*>(here + (k >> 1) * (KT * 128) + (ks0 + s) * 16 * 128 + kbase + kslot[k & 1]);
      };
      uint4 key[LEAD];
#pragma unroll
      for (int i = 0; i < LEAD; ++i) key[i] = rd(i);
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < TOT; ++i) {
        const int s = i / KSTEPS, k = i % KSTEPS;
#pragma unroll
        for (int c = 0; c < QCT; ++c) st[c][s] = Mma<T>::qk(key[i % LEAD], qf[c][k], k == 0 ? z : st[c][s]);
        if (i + LEAD < TOT) key[i % LEAD] = rd(i + LEAD);
        if constexpr (QCT == 2) __builtin_amdgcn_sched_barrier(0);
      }
      if (masked) {
        // A row that some column does not see may hold what is not finite (a
        // sibling's draft): zero probabilities do not hide it.  Every score of
        // such a row is not finite either.
#pragma unroll
        for (int c = 0; c < QCT; ++c) {
          const uint32_t bits = window(cur, col.qi[c], t0) >> (16 * ks0 + 4 * g);
#pragma unroll
          for (int s = 0; s < QKS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              odd |= !(__builtin_fabsf(st[c][s][r]) < INFINITY);
              st[c][s][r] = (bits >> (16 * s + r)) & 1u ? st[c][s][r] * a.scale_log2 : -INFINITY;
            }
        }
      } else {
#pragma unroll
        for (int c = 0; c < QCT; ++c)
#pragma unroll
          for (int s = 0; s < QKS; ++s) st[c][s] *= a.scale_log2;
      }
#pragma unroll
      for (int c = 0; c < QCT; ++c) {
        float mt = -INFINITY;
#pragma unroll
        for (int s = 0; s < QKS; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) mt = fmaxf(mt, st[c][s][r]);
        mt = row_max4(mt);
        vote |= mt > m_run[c] + kSlack;
        if (g == 0) tile_max[ks0][16 * (ct0 + c) + l16] = mt;
      }
    }
    auto weigh = [&]() {
#pragma unroll
      for (int c = 0; c < QCT; ++c) {
        const float base = m_run[c] == -INFINITY ? 0.f : -m_run[c];
#pragma unroll
        for (int s = 0; s < QKS; ++s) {
          // The weights are rounded to T for the products (a matrix
          // instruction's operands are of one type); the sum that divides them
          // counts them as rounded.
          T w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            w[r] = from_f32<T>(fast_exp2(st[c][s][r] + base));
            l_run[c] += to_f32(w[r]);
          }
          uint2 both;
          __builtin_memcpy(&both, w, 8);
          probs[((ct0 + c) * 64 + lane) * 2 + ks0 + s] = both;
        }
      }
    };
    const bool any_vote = __any(vote), any_odd = __any(odd);
    if (scores && !any_vote) weigh();
    if (lane == 0) votes[wave] = (any_vote ? 1u : 0u) | (any_odd ? 2u : 0u);
    lds_barrier();
    const uint4 vw = *reinterpret_cast<const uint4*>(votes);
    const uint32_t said = __builtin_amdgcn_readfirstlane(vw.x | vw.y | vw.z | vw.w);
    if (said & 1u) {
      // Some column's maximum moves: all waves move every column to its own.
      auto moved = [&](int c, float& before) -> float {
        const int i = 16 * c + l16;
        before = col_max[i];
        return fmaxf(before, QKS == 2 ? tile_max[0][i] : fmaxf(tile_max[0][i], tile_max[1][i]));
      };
      auto ratio = [](float before, float after) { return after == -INFINITY ? 1.f : fast_exp2(before - after); };
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float before;
        const float after = moved(c, before), alpha = ratio(before, after);
#pragma unroll
        for (int n = 0; n < DT; ++n) acc[c][n] *= alpha;
      }
      if (scores) {
        // (Weights that were formed with the old maximum are taken back.)
        if (!any_vote) {
#pragma unroll
          for (int c = 0; c < QCT; ++c)
#pragma unroll
            for (int s = 0; s < QKS; ++s) {
              const uint2 both = probs[((ct0 + c) * 64 + lane) * 2 + ks0 + s];
              T w[4];
              __builtin_memcpy(w, &both, 8);
#pragma unroll
              for (int r = 0; r < 4; ++r) l_run[c] -= to_f32(w[r]);
            }
        }
#pragma unroll
        for (int c = 0; c < QCT; ++c) {
          float before;
          const float after = moved(ct0 + c, before);
          l_run[c] *= ratio(before, after);
          m_run[c] = after;
        }
        weigh();
      }
      lds_barrier();
      if (scores && g == 0 && ks0 == 0) {
#pragma unroll
        for (int c = 0; c < QCT; ++c) col_max[16 * (ct0 + c) + l16] = m_run[c];
      }
    }
    const bool poisoned = (said & 2u) != 0;
    if (poisoned) {
      // The step's rows without their values that are not finite (and none of
      // the repeated rows past the piece's end).
      const int pos = t0 + lrow;
      if (pos >= cur.computed) {
#pragma unroll 1
        for (int c = 0; c < L / 8; ++c) {
          if ((c & 7) != lchunk) continue;
          T* at8 = reinterpret_cast<T*>(const_cast<char*>(here) + (c >> 3) * (KT * 128) + wave * 1024 + lane * 16);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (not_finite(at8[e])) at8[e] = from_f32<T>(0.f);
        }
      }
      lds_barrier();
    }

    // ---- O^T += V^T P^T
    V8 pb[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) pb[c] = bitcast<V8>(*reinterpret_cast<const uint4*>(probs + (c * 64 + lane) * 2));
#pragma unroll
    for (int n = 0; n < DT; ++n) {
      const char* at8 = vaddr(here, n);
      const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(at8));
      const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(at8 + 16 * 128));
      const s16x4 both[2] = {v0, v1};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if constexpr (std::is_same<T, __bf16>::value) {
          acc[c][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<V8>(both), pb[c], acc[c][n], 0, 0, 0);
        } else {
          acc[c][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<V8>(both), pb[c], acc[c][n], 0, 0, 0);
        }
      }
    }
    if (poisoned) {
      // Every column that sees such a value gets NaN in that dimension, as 0 x
      // NaN, 0 x inf or a weight of a score that is not finite would give: the
      // value times zero is added (zero, for finite ones).
#pragma unroll 1
      for (int pos = max(t0, cur.computed); pos < min(t0 + KT, cur.tok_end); ++pos) {
        const int lb = fast_div(pos, a.by_block);
        gptr<const T> const v =
            pool + ((int64_t)a.tables[cur.table_off + lb] * a.block_size + (pos - lb * a.block_size)) * S::ROW;
        f32x4 zero_or_nan[DT];
#pragma unroll
        for (int n = 0; n < DT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) zero_or_nan[n][r] = to_f32((T)v[16 * (wave * DT + n) + 4 * g + r]) * 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          int qi, head;
          columns(cur, c, qi, head);
          const bool sees = (window(cur, qi, t0) >> (pos - t0)) & 1u;
#pragma unroll
          for (int n = 0; n < DT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[c][n][r] += sees ? zero_or_nan[n][r] : 0.f;
        }
      }
    }

    // ---- a finished piece: its output rows, or its partials
    if (ends) {
      if (scores) {
#pragma unroll
        for (int c = 0; c < QCT; ++c) {
          const float l = row_sum4(l_run[c]);
          if (g == 0) col_sum[ks0][16 * (ct0 + c) + l16] = l;
        }
      }
      lds_barrier();
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int i = 16 * c + l16;
        const float l_tot = QKS == 2 ? col_sum[0][i] : col_sum[0][i] + col_sum[1][i];
        const float inv = l_tot > 0.f ? 1.f / l_tot : l_tot == l_tot ? 0.f : l_tot;
        int qi, head;
        if (!columns(cur, c, qi, head)) continue;
        if (cur.slot < 0) {
          T* to = static_cast<T*>(a.out) + (int64_t)(cur.q_start + qi) * a.out_tok_stride + (int64_t)head * a.out_head_stride;
#pragma unroll
          for (int n = 0; n < DT; ++n) store_partial4<false, T>(to + 16 * (wave * DT + n) + 4 * g, acc[c][n], inv);
        } else {
          const int64_t cs = (int64_t)cur.slot * COLS + i;
          float* to = a.part_acc + cs * L;
#pragma unroll
          for (int n = 0; n < DT; ++n) store_partial4<false, float>(to + 16 * (wave * DT + n) + 4 * g, acc[c][n], inv);
          // (A NaN sum keeps a finite maximum: the merge passes over a partial
          // whose maximum is -inf.)
          const float m = col_max[i];
          if (wave == 0 && g == 0)
            *reinterpret_cast<float2*>(a.part_ml + cs * 2) = make_float2(l_tot == l_tot || m != -INFINITY ? m : 0.f, l_tot);
        }
      }
      if (!has_next) return false;
      p = np;
      cur = read_latent_piece(pieces, p);
      fresh = true;
    }
    t0 = nt0;
    return true;
  };
  while (step(tile0, tile1) && step(tile1, tile0)) {
  }
}

// ---------------------------------------------------------------------------
// Merge: a workgroup per (job, column), a thread per four dimensions.  With
// partial i's maximum m_i (log2) and sum l_i, out = sum 2^(m_i - M) l_i o_i /
// sum 2^(m_i - M) l_i.
// ---------------------------------------------------------------------------
template <typename T, int L>
__global__ __launch_bounds__(L / 4) void latent_merge_kernel(const int32_t* __restrict__ jobs, const int32_t cols,
                                                             const LatentDecodeArgs a) {
  const int32_t* jb = jobs + (int64_t)blockIdx.x * LVAMD_MERGE_FIELDS;
  const int group = jb[1], slot0 = jb[2], np = jb[3], q_start = jb[4], q_len = jb[5];
  const int i = blockIdx.y;
  const int col = group * cols + i;
  if (col >= q_len * a.heads) return;
  const float* ml = a.part_ml + ((int64_t)slot0 * cols + i) * 2;
  const int64_t ml_step = 2 * cols;
  float m = -INFINITY;
  for (int k = 0; k < np; ++k) m = fmaxf(m, ml[k * ml_step]);
  const float* from = a.part_acc + ((int64_t)slot0 * cols + i) * L + 4 * threadIdx.x;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  float total = 0.f;
#pragma unroll 4
  for (int k = 0; k < np; ++k) {
    const f32x4 o = *reinterpret_cast<const f32x4*>(from + (int64_t)k * cols * L);
    const float mk = ml[k * ml_step];
    const float w = mk == -INFINITY ? 0.f : fast_exp2(mk - m) * ml[k * ml_step + 1];
    total += w;
    sum += o * w;
  }
  const int qi = fast_div(col, a.by_heads), head = col - qi * a.heads;
  T* to = static_cast<T*>(a.out) + (int64_t)(q_start + qi) * a.out_tok_stride + (int64_t)head * a.out_head_stride;
  const float inv = total > 0.f ? 1.f / total : total == total ? 0.f : total;
  store_partial4<false, T>(to + 4 * threadIdx.x, sum, inv);
}

template <typename T, int L, int P>
static const void* latent_decode_fn(int col_tiles) {
  switch (col_tiles) {
    case 1: return (const void*)&latent_decode_kernel<T, L, P, 1>;
    case 2: return (const void*)&latent_decode_kernel<T, L, P, 2>;
    case 4: return (const void*)&latent_decode_kernel<T, L, P, 4>;
    default: return nullptr;
  }
}

}  // namespace lvamd

using namespace lvamd;

extern "C" int lvamd_latent_decode_tile_tokens(void) { return KT; }

extern "C" int lvamd_latent_decode_resident_groups(int32_t dtype, int32_t latent_size, int32_t rope_size, int32_t col_tiles) {
  return latent_dispatch(dtype, latent_size, rope_size, [&]<typename T, int L, int P>() -> int {
    const void* fn = latent_decode_fn<T, L, P>(col_tiles);
    int device = 0, cus = 0, per_cu = 0;
    if (!fn) return LVAMD_ERR_UNSUPPORTED;
    if (hipGetDevice(&device) != hipSuccess) return LVAMD_ERR_LAUNCH;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess) return LVAMD_ERR_LAUNCH;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, fn, 64 * kWaves, 0) != hipSuccess) return LVAMD_ERR_LAUNCH;
    return per_cu * cus;
  });
}

extern "C" int lvamd_latent_decode(const void* query, int64_t query_token_stride, int64_t query_head_stride,
                                   const void* query_rope, int64_t rope_token_stride, int64_t rope_head_stride,
                                   const void* pool, void* out, int64_t out_token_stride, int64_t out_head_stride,
                                   const int32_t* pieces, const int32_t* group_first, int32_t num_groups,
                                   const int32_t* jobs, int32_t num_jobs, int32_t merge_columns, const int32_t* tables,
                                   const uint32_t* vis, float* part_acc, float* part_ml, int64_t num_partial_slots,
                                   int32_t num_heads, int32_t latent_size, int32_t rope_size, int32_t col_tiles,
                                   int32_t block_size, float scale, int32_t dtype, lvamd_stream_t stream) {
  if (!latent_sizes(latent_size, rope_size) || !latent_dtype(dtype)) return LVAMD_ERR_UNSUPPORTED;
  if (num_groups < 0 || num_jobs < 0 || num_heads <= 0 || block_size <= 0 || num_partial_slots < 0 || merge_columns < 0 ||
      merge_columns > 65535)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_groups == 0) return LVAMD_OK;
  if (!query || !query_rope || !pool || !out || !pieces || !group_first || !tables || !vis || (num_jobs > 0 && !jobs))
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_partial_slots > 0 && (!part_acc || !part_ml)) return LVAMD_ERR_WORKSPACE;
  if (!rows16(query, {query_token_stride, query_head_stride}) || !rows16(query_rope, {rope_token_stride, rope_head_stride}) ||
      !rows16(pool, {}) || ((uintptr_t)out & 7u) || out_token_stride % 4 != 0 || out_head_stride % 4 != 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  LatentDecodeArgs a{.by_block = FastDiv(block_size), .by_heads = FastDiv(num_heads)};
  a.q = query;
  a.q_tok_stride = query_token_stride;
  a.q_head_stride = query_head_stride;
  a.qr = query_rope;
  a.qr_tok_stride = rope_token_stride;
  a.qr_head_stride = rope_head_stride;
  a.pool = pool;
  a.out = out;
  a.out_tok_stride = out_token_stride;
  a.out_head_stride = out_head_stride;
  a.tables = tables;
  a.vis = vis;
  a.part_acc = part_acc;
  a.part_ml = part_ml;
  a.heads = num_heads;
  a.block_size = block_size;
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return latent_dispatch(dtype, latent_size, rope_size, [&]<typename T, int L, int P>() -> int {
    const dim3 grid((unsigned)num_groups), block(64 * kWaves);
    switch (col_tiles) {
      case 1: hipLaunchKernelGGL((latent_decode_kernel<T, L, P, 1>), grid, block, 0, s, group_first, pieces, a); break;
      case 2: hipLaunchKernelGGL((latent_decode_kernel<T, L, P, 2>), grid, block, 0, s, group_first, pieces, a); break;
      case 4: hipLaunchKernelGGL((latent_decode_kernel<T, L, P, 4>), grid, block, 0, s, group_first, pieces, a); break;
      default: return LVAMD_ERR_UNSUPPORTED;
    }
    if (const int status = launch_status(); status != LVAMD_OK) return status;
    if (num_jobs == 0) return LVAMD_OK;
    hipLaunchKernelGGL((latent_merge_kernel<T, L>), dim3((unsigned)num_jobs, (unsigned)merge_columns), dim3(L / 4), 0, s,
                       jobs, 16 * col_tiles, a);
    return launch_status();
  });
}
