// Attention over a paged cache of latent vectors on gfx950, in latent space
// (the absorbed form): head h's query, multiplied by its key weights already,
// meets the rows themselves,
//   s = scale (q[0..L) . c + q[L..L+P) . r),   out = sum softmax(s) c,
// so all heads share one key of L + P values and one value of L of them.
//
// Query j of a request with c computed tokens sees logical positions [0, c) and
// {c + i : i <= j} (linear) or {c + i : i an ancestor of j, or j} (tree).  The
// step's tokens are in the cache already, or the launch appends them.
//
// Mapping onto CDNA4:
//   * A column is a (query, head) pair of one request; a workgroup (four waves, or
//     eight of 64 columns and more) holds up to 16 NC of them and walks over tiles
//     of 32 rows (64 with 64 columns): stream-K pieces of (request, column group)
//     segments, split segments merged below.
//   * The rows of a tile are loaded once, straight into LDS (global_load_lds, no
//     registers), while the tile before is computed; they serve as keys (rows
//     read as they lie) and as values (transpose reads).
//   * Scores: S^T = K Q^T on MFMA 16x16x32, the 16-row parts of the tile and the
//     column tiles dealt to the waves, queries in registers.  Products: O^T = V^T
//     P^T, a share of the latent's dimensions per wave for all columns, so an
//     accumulator takes a share of the registers that a whole row would, and
//     each value is read from LDS once.  The probabilities cross over through
//     LDS (the accumulator layout of S^T is the operand layout of P^T).
//   * The waves share each column's running maximum, which moves only when some
//     score passes it by 2^8 (lazy rescaling): a vote per tile in LDS.
//   * A row that some column does not see may hold anything: its scores, which are not
//     finite then, raise a flag beside the vote.  Scores and weights stay; the tile's
//     values that are not finite become zeros in LDS, and each column that sees such a
//     row adds the row's values times zero.
//   * Append: a tile's rows of this step are loaded from the step's tensors, and
//     one column group writes them to the pool; keys and queries are turned on the
//     way.  On the GPU it costs what the append's launch takes (48 requests: 30.4
//     against 26.1 + 3.4 us), on the host it saves that launch (one request: 23
//     against 30 us a call).
//   * A tile has two barriers: its rows are there, its probabilities are there.
//     The values of up to 64 columns are read before the softmax (43 against 45 us
//     for 64 requests of 32 columns, 232 against 258 for 8 x 32767 x 128 columns).
//
// What bounds it.  Up to 32 columns two workgroups of a CU keep a tile of 37 KB
// each in flight: 64 requests of 512 to 4,095 tokens (16 heads, 512 + 64, bf16, 182
// MB) 41 to 43 us, 4.4 TB/s, of which 6 pass before the first tile and 31 at the full
// rate; 16 x 32767 tokens (32 heads, fp16, 605 MB) 109 us, 5.5 TB/s.  From 64 columns on
// the tile's own work: about 2.8 us for 64 rows and 64 columns, of which the matrix units
// are busy 0.9 and LDS 1.1; the rest is vector instructions (two waves a SIMD, one
// workgroup a CU) and the round trips between the phases.  32 requests of 128 heads (97
// MB, 21 GFLOP) 54 us: 7 to the first tile, 9 to 10 tiles, 3 for the partials; over the
// launch the matrix units are busy 16 %, LDS 14 %, waves wait 43 %.  The groups of one
// request over the same tokens run on one XCD, whose L2 serves a part of the second's (159
// of 209 MB come from memory): 63 to 51 us for 32 x 2300 tokens.  Eight waves rather than four from 64 columns on: 140 against
// 145 us for 8 x 32767 x 128 heads.  Up to 32 columns tile loads are non-temporal: 50
// against 55 us for the 64 requests.  Dealing the loads between the score products
// measured slower (258 against 232 us).
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
// Rows per tile.  64 columns leave registers and LDS for 64 rows, which halves a
// row's share of the barriers and round trips (128 against 147 us for 8 x 32767 tokens
// of 128 heads, 95 against 104 for 64 x 2300); 128 columns do not, and two workgroups
// of a CU do not fit with fewer.
constexpr int tile_rows(int col_tiles) { return col_tiles == 4 ? 64 : 32; }

typedef const __attribute__((address_space(1))) void* lds_gptr;
typedef __attribute__((address_space(3))) void* lds_lptr;

struct LatentDecodeArgs {
  const void* q;  // [rows][heads][L], the latent part; a piece names its request's first row
  int64_t q_tok_stride, q_head_stride;
  const void* qr;  // [tokens][heads][P], the rotated part
  int64_t qr_tok_stride, qr_head_stride;
  void* pool;  // [slots][L + P]
  // The step's rows, where this launch appends them, or null: the pool has them.
  const void* latent_new;
  const void* rope_new;
  int64_t latent_stride, rope_stride;
  const float* cosines;  // [tokens][P / 2], or null: queries and keys are turned already
  const float* sines;
  int64_t angle_stride;
  void* out;  // [rows][heads][L]
  int64_t out_tok_stride, out_head_stride;
  const int32_t* __restrict__ tables;
  const uint32_t* __restrict__ vis;
  float* part_acc;  // [slots][16 NC][L] fp32, rows normalised
  float* part_ml;   // [slots][16 NC][2]: (max, sum)
  int32_t heads, block_size, interleaved;
  FastDiv by_block, by_heads;
  float scale_log2;
};

// A piece's record: pieces[blockIdx.x] is a workgroup's first, next its next (-1:
// none); blocks are the first four of its table entries (-1: look them up).
struct LatentPiece {
  int row, group, tok_begin, tok_end, slot, table_off, computed, q_len, q_start, vis_off, vis_words, next;
};
__device__ __forceinline__ LatentPiece read_latent_piece(const int32_t* __restrict__ pieces, int p) {
  const int32_t* r = pieces + (int64_t)p * LVAMD_PIECE_FIELDS;
  return {r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7], r[8], r[9], r[10], r[11]};
}

__device__ __forceinline__ constexpr int swizzle(int row) {
  return (((row >> 2) & 1) << 1) | ((((row >> 3) ^ (row >> 1)) & 1) << 2);
}

// Orders LDS accesses around a workgroup barrier.  (A release fence would also
// wait for the tile loads in flight, which write LDS too.)
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

constexpr int wait_vm(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); }  // s_waitcnt vmcnt(n)

template <int L, int P, int NC>
struct LatentShape {
  static constexpr int ROW = L + P;                   // elements
  static constexpr int CPR = ROW / 8;                 // 16-byte chunks of a row
  static constexpr int GR = (CPR + 7) / 8;            // 128-byte groups
  static constexpr int KT = tile_rows(NC);
  static constexpr int TILE_BYTES = GR * KT * 128;
  static constexpr int KSTEPS = ROW / 32;             // MFMA steps of a score
  static constexpr int W = NC >= 4 ? 8 : 4;           // waves
  static constexpr int DT = L / (16 * W);             // 16-dimension tiles per wave
  static constexpr int QKS = NC >= 4 ? 2 : 1;         // 16-row parts a wave scores
  static constexpr int NB = 2;                        // tiles in LDS
  static constexpr int WAVES_PER_EU = 2;
  static constexpr bool APPEND = NC < 8;              // (128 columns: no registers left for it)
  static_assert(L % 128 == 0 && P % 32 == 0);
};

template <typename T>
__device__ __forceinline__ bool not_finite(T x) {
  return !(__builtin_fabsf(to_f32(x)) < INFINITY);
}

}  // namespace

template <typename T, int L, int P, int NC>
__global__ __launch_bounds__(NC >= 4 ? 512 : 256)
__attribute__((amdgpu_waves_per_eu(LatentShape<L, P, NC>::WAVES_PER_EU))) void latent_decode_kernel(
    const int32_t* __restrict__ pieces, const LatentDecodeArgs a) {
  using S = LatentShape<L, P, NC>;
  constexpr int KT = S::KT, GR = S::GR, KSTEPS = S::KSTEPS, DT = S::DT, QKS = S::QKS, W = S::W;
  constexpr int COLS = 16 * NC;
  constexpr bool APPEND = S::APPEND;
  using V8 = typename std::conditional<std::is_same<T, __bf16>::value, bf16x8, f16x8>::type;
  // Separate objects: a load into one does not alias a read of another.
  __shared__ __attribute__((aligned(1024))) char tile0[S::TILE_BYTES];
  __shared__ __attribute__((aligned(1024))) char tile1[S::TILE_BYTES];
  __shared__ __attribute__((aligned(16))) uint2 probs[KT / 32 * NC * 64 * 2];  // [32 rows][column tile][lane][half]
  __shared__ float tile_max[2][COLS], col_max[COLS], col_sum[2][COLS];
  __shared__ __attribute__((aligned(16))) uint32_t votes[W];

  const int tid = threadIdx.x & (64 * W - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;

  // ---- this wave's scores: rows [16 ks0, 16 (ks0 + QKS)) of a tile, column tile ct0.
  const bool scores = NC > 1 || wave < 2;
  constexpr int HALVES = KT / (16 * QKS);  // waves that share a column tile
  const int half = HALVES == 1 ? 0 : wave & 1, ks0 = QKS * half;
  const int ct0 = NC == 1 ? 0 : HALVES == 1 ? wave : wave >> 1;

  // ---- tile loads: wave w loads rows 8 (w % RB) .. + 7 of the groups w / RB, + W / RB,
  // ..; lane l row l / 8 of them into chunk slot l % 8 of a group.
  constexpr int RB = KT / 8, GSTEP = W / RB;
  const int rb = wave % RB;
  // The load cursor: the tile whose rows are looked up next.  first_new: the
  // position from which rows are the step's own, read from its tensors.
  struct Cursor {
    int table_off, t0, tok_end, next;  // tok_end 0: no more tiles
    int first_new, q_start;
  };
  struct Row {
    int entry, off, tok;  // tok: of the step, or -1
  };
  auto first_new = [&](int computed) { return APPEND && a.latent_new ? computed : 0x7fffffff; };
  auto lookup = [&](int ln, const Cursor& c) -> Row {
    const int pos = min(c.t0 + 8 * rb + (ln >> 3), c.tok_end - 1);
    const int lb = fast_div(pos, a.by_block);
    return {a.tables[c.table_off + lb], pos - lb * a.block_size, pos >= c.first_new ? c.q_start + pos - c.first_new : -1};
  };
  gptr<T> const pool = (gptr<T>)(a.pool);
  auto issue = [&](int ln, const Row& r, char* dst) {
    const int lchunk = (ln & 7) ^ swizzle(8 * rb + (ln >> 3));
    gptr<const T> row = pool + ((int64_t)r.entry * a.block_size + r.off) * S::ROW, key = row;
    if (APPEND && __any(r.tok >= 0)) {
      row = r.tok >= 0 ? (gptr<const T>)(a.latent_new) + r.tok * a.latent_stride : row;
      key = r.tok >= 0 ? (gptr<const T>)(a.rope_new) + r.tok * a.rope_stride - L : key;
    }
#pragma unroll
    for (int i = 0; i < (GR + GSTEP - 1) / GSTEP; ++i) {
      const int gr = wave / RB + i * GSTEP;
      if (GR % GSTEP != 0 && gr >= GR) break;
      int c = 8 * gr + lchunk;
      // (A half-used last group's spare slots take the row's last chunk again.)
      if (8 * GR > S::CPR && gr == GR - 1) c = min(c, S::CPR - 1);
      // Non-temporal where a row is read once (16 and 32 columns are a whole request);
      // 64 columns are often one of several groups, which share an L2 (51 against 56 us
      // for 32 x 2300 tokens of 128 heads).  128 measured alike either way.
      __builtin_amdgcn_global_load_lds((lds_gptr)((gr < L / 64 ? row : key) + 8 * c),
                                       (lds_lptr)(dst + (gr * KT * 128 + rb * 1024)), 16, 0, NC == 4 ? 0 : 2);
    }
  };

  // Keys of the step's rows that are still to be turned: a lane's chunk of the key
  // and its angles (with the half layout also the chunk that holds the pairs' other
  // values), loaded beside the tile.
  struct Key {
    uint4 lo, hi;
    f32x4 c[2], s[2];
  };
  constexpr int HALF = P / 16;  // chunks of half a key
  constexpr int KEY_GROUP = L / 64;
  auto key_chunk = [&](int ln) -> int {  // -1: not this lane's
    const int c = (ln & 7) ^ swizzle(8 * rb + (ln >> 3));
    return (GSTEP == 1 || wave / RB == KEY_GROUP % GSTEP) && c < 2 * HALF ? c : -1;
  };
  auto key_place = [&](int ln, char* tile) -> uint4* {
    return reinterpret_cast<uint4*>(tile + (KEY_GROUP * (KT * 128) + rb * 1024 + ln * 16));
  };
  auto load_key = [&](int ln, const Row& r, Key& k) {
    const int c = key_chunk(ln);
    if (r.tok < 0 || c < 0) return;
    gptr<const T> const from = (gptr<const T>)(a.rope_new) + (int64_t)r.tok * a.rope_stride;
    const float* cs = a.cosines + (int64_t)r.tok * a.angle_stride;
    const float* sn = a.sines + (int64_t)r.tok * a.angle_stride;
    // (The same loads for both layouts: interleaved pairs need the first of each two.)
    const int low = c & (HALF - 1), at = a.interleaved ? 4 * c : 8 * low, more = a.interleaved ? 0 : 4;
    k.c[0] = *reinterpret_cast<const f32x4*>(cs + at);
    k.s[0] = *reinterpret_cast<const f32x4*>(sn + at);
    k.c[1] = *reinterpret_cast<const f32x4*>(cs + at + more);
    k.s[1] = *reinterpret_cast<const f32x4*>(sn + at + more);
    k.lo = load16(from + 8 * (a.interleaved ? c : low));
    k.hi = load16(from + 8 * (a.interleaved ? c : low + HALF));
  };
  auto turned = [&](int ln, const Key& k) -> uint4 {
    if (a.interleaved) return turn_chunk<T>(k.lo, k.c[0], k.s[0]);
    uint4 lo = k.lo, hi = k.hi;
    turn_chunks<T>(lo, hi, k.c, k.s);
    const bool low = key_chunk(ln) < HALF;
    return make_uint4(low ? lo.x : hi.x, low ? lo.y : hi.y, low ? lo.z : hi.z, low ? lo.w : hi.w);
  };

  // ---- columns: queries in registers, what each sees of the step's tokens
  auto columns = [&](int ln, const LatentPiece& x, int ct, int& qi, int& head) -> bool {
    const int col = x.group * COLS + 16 * ct + (ln & 15), ncols = x.q_len * a.heads;
    const bool ok = col < ncols;
    const int c = ok ? col : ncols - 1;
    qi = fast_div(c, a.by_heads);
    head = c - qi * a.heads;
    return ok;
  };
  // Bit k: whether query qi sees row t0 + k, 32 rows (rows of the step only;
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
    return left >= 32 ? bits : left <= 0 ? 0u : bits & ((1u << left) - 1u);
  };

  LatentPiece cur = read_latent_piece(pieces, blockIdx.x);
  uint4 qf[KSTEPS];
  int qi0 = 0;
  auto load_queries = [&](int ln, const LatentPiece& x) {
    const int g = ln >> 4;
    int head;
    const bool ok = columns(ln, x, ct0, qi0, head);
    const T* q = static_cast<const T*>(a.q) + (int64_t)(x.row + qi0) * a.q_tok_stride + (int64_t)head * a.q_head_stride + 8 * g;
    const T* qr = static_cast<const T*>(a.qr) + (int64_t)(x.q_start + qi0) * a.qr_tok_stride +
                  (int64_t)head * a.qr_head_stride + 8 * g;
    const bool mine = scores && ok;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) qf[k] = mine ? load16(32 * k < L ? q + 32 * k : qr + 32 * k - L) : zero_u4();
    if (APPEND && a.cosines) {
      // Turned here: chunk (32 k - L) / 8 + g of the rotated part.
      const float* cs = a.cosines + (int64_t)(x.q_start + qi0) * a.angle_stride;
      const float* sn = a.sines + (int64_t)(x.q_start + qi0) * a.angle_stride;
#pragma unroll
      for (int k = L / 32; k < KSTEPS; ++k) {
        const int c = (32 * k - L) / 8 + g;
        if (mine && a.interleaved) qf[k] = turn_chunk<T>(qf[k], cs + 4 * c, sn + 4 * c);
        if (mine && !a.interleaved) {
          const int at = 8 * (c & (HALF - 1));
          uint4 lo = load16(qr - 8 * g + 8 * (c & (HALF - 1))), hi = load16(qr - 8 * g + 8 * (c | HALF));
          turn_chunks<T>(lo, hi, cs + at, sn + at);
          const bool low = c < HALF;
          qf[k] = make_uint4(low ? lo.x : hi.x, low ? lo.y : hi.y, low ? lo.z : hi.z, low ? lo.w : hi.w);
        }
      }
    }
  };

  auto advance = [&](Cursor& c) {
    c.t0 += KT;
    if (c.t0 >= c.tok_end) {
      if (c.next < 0) {
        c.tok_end = 0;
        return;
      }
      const int32_t* r = pieces + (int64_t)c.next * LVAMD_PIECE_FIELDS;
      c.t0 = r[2];
      c.tok_end = r[3];
      c.table_off = r[5];
      c.first_new = first_new(r[6]);
      c.q_start = r[8];
      c.next = r[11];
    }
  };
  Cursor at = {cur.table_off, cur.tok_begin, cur.tok_end, cur.next, first_new(cur.computed), cur.q_start};
  Row row;
  {
    // The first tile's rows lie in the record's blocks.
    const int32_t* r = pieces + (int64_t)blockIdx.x * LVAMD_PIECE_FIELDS;
    const int b0 = r[12], b1 = r[13], b2 = r[14], b3 = r[15];
    if (b0 >= 0) {
      const int pos = min(at.t0 + 8 * rb + (lane >> 3), at.tok_end - 1);
      const int lb = fast_div(pos, a.by_block), k = lb - fast_div(at.t0, a.by_block);
      row = {k == 0 ? b0 : k == 1 ? b1 : k == 2 ? b2 : b3, pos - lb * a.block_size,
             pos >= at.first_new ? at.q_start + pos - at.first_new : -1};
    } else {
      row = lookup(lane, at);
    }
  }
  Row held = row;  // of the tile that is computed next, while it holds rows of the step
  Key held_key;
  issue(lane, row, tile0);
  if (APPEND && a.cosines) load_key(lane, row, held_key);
  load_queries(lane, cur);
  advance(at);
  if (at.tok_end > 0) row = lookup(lane, at);

  float m_run, l_run;
  f32x4 acc[NC][DT];
  int t0 = cur.tok_begin;
  bool fresh = true;  // the tile is its piece's first

  auto key_base = [&](int ln) -> int {
    return (16 * ks0 + (ln & 15)) * 128 + 16 * ((ln >> 4) ^ swizzle(ln & 15));  // (^ 64: chunk 4 + g)
  };
  auto value_address = [&](int ln, int n) -> int {
    const int vrow = 4 * (ln >> 4) + ((ln & 15) >> 2), q4 = ln & 3, c = 2 * (wave * DT + n) + (q4 >> 1);
    return (c >> 3) * (KT * 128) + vrow * 128 + 16 * ((c & 7) ^ swizzle(vrow)) + 8 * (q4 & 1);
  };
  constexpr bool EARLY_V = NC < 8;
  const int kept_kbase = key_base(lane);
  int kept_vaddr[DT];
#pragma unroll
  for (int n = 0; n < DT; ++n) kept_vaddr[n] = value_address(lane, n);

  // One tile from `here` while the next lands in `there`; false: it was the last.
  auto step = [&](const char* here, char* there) __attribute__((always_inline)) -> bool {
    // (Everything that depends on the lane is formed anew in each step, a few
    // instructions: kept from step to step it would not fit the registers of the
    // wide instances.)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int l16 = ln & 15, g = ln >> 4;
    // LDS offsets: key reads (row l16 + 16 ks, chunk 4 k + g) and transpose reads (row
    // 4 g + l16 / 4, +16; 8 bytes of dimensions 16 n + 4 q4).  (Each read is one
    // offset from its tile: the compiler tells a read of one tile from a load into
    // the other only where few steps of arithmetic lie between the array and the
    // access; otherwise it waits for the load before every read.)
    const int kbase = EARLY_V ? kept_kbase : key_base(ln);
    auto vaddr = [&](int n) -> int { return EARLY_V ? kept_vaddr[n] : value_address(ln, n); };
    __builtin_amdgcn_s_waitcnt(wait_vm(0));  // this wave's part of the tile
    lds_barrier();                           // everyone's, and the last tile's reads are done
    const bool masked = t0 + KT > min(cur.computed, cur.tok_end);
    // The step's own rows among the tile's: the turned keys go to LDS, and the group
    // with a token's first column writes its row to the pool (below, behind the
    // tile's matrix work).
    const bool has_new = APPEND && masked && a.latent_new;
    int slot = -1;
    if (has_new) {
      if (a.cosines && held.tok >= 0 && key_chunk(ln) >= 0) *key_place(ln, const_cast<char*>(here)) = turned(ln, held_key);
      const int pos = t0 + 8 * rb + (ln >> 3);
      const int col = (pos - cur.computed) * a.heads - cur.group * COLS;
      if (pos >= cur.computed && pos < cur.tok_end && col >= 0 && col < COLS) slot = held.entry * a.block_size + held.off;
    }
    if (at.tok_end > 0) {
      issue(ln, row, there);
      if (APPEND) held = row;
      if (APPEND && a.cosines) load_key(ln, row, held_key);
      advance(at);
      if (at.tok_end > 0) row = lookup(ln, at);
    }
    if (has_new && a.cosines) lds_barrier();
    if (fresh) {
      m_run = -INFINITY;
      l_run = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int n = 0; n < DT; ++n) acc[c][n] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (tid < COLS) col_max[tid] = -INFINITY;
      fresh = false;
    }
    // ---- scores
    auto rdv = [&](int n, int step = 0) -> V8 {
      const int at8 = vaddr(n) + step * 32 * 128;
      const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(here + at8));
      const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(here + (at8 + 16 * 128)));
      const s16x4 both[2] = {v0, v1};
      return bitcast<V8>(both);
    };
    constexpr int STEPS = KT / 32;
    V8 vals[EARLY_V ? DT : 1];
    f32x4 st[QKS];
    bool vote = false, odd = false;
    if (scores) {
      // LDS reads run LEAD ahead of the matrix instructions; two sums per score, so
      // that an instruction does not wait for the one before it.
      constexpr int TOT = QKS * KSTEPS, LEAD = NC == 8 ? 3 : 6, CH = QKS == 1 ? 2 : 1;
      auto rd = [&](int i) -> uint4 {
        const int group = (i / QKS) >> 1, odd_chunks = (i / QKS) & 1;
        return *reinterpret_cast<const uint4*>(here + (group * (KT * 128) + (i % QKS) * 16 * 128 + (kbase ^ (odd_chunks ? 64 : 0))));
      };
      uint4 key[LEAD];
#pragma unroll
      for (int i = 0; i < LEAD; ++i) key[i] = rd(i);
      f32x4 sum[2];
#pragma unroll
      for (int i = 0; i < TOT; ++i) {
        const int k = i / QKS, to = QKS == 2 ? i % 2 : k % 2;
        sum[to] = Mma<T>::qk(key[i % LEAD], qf[k], i < 2 ? f32x4{0.f, 0.f, 0.f, 0.f} : sum[to]);
        if (i + LEAD < TOT) key[i % LEAD] = rd(i + LEAD);
        if constexpr (NC == 8) __builtin_amdgcn_sched_barrier(0);  // (hoisted reads would spill)
      }
      if constexpr (EARLY_V) {
#pragma unroll
        for (int n = 0; n < DT; ++n) vals[n] = rdv(n);
      }
      if constexpr (CH == 2) {
        st[0] = sum[0] + sum[1];
      } else {
        st[0] = sum[0];
        st[QKS - 1] = sum[1];
      }
      if (masked) {
        // A row that some column does not see may hold what is not finite (a
        // sibling's draft): zero weights do not hide it.  Every score of such a row is not
        // finite either (the row is the key too).
        const uint32_t bits = window(cur, qi0, t0 + 16 * (ks0 & ~1)) >> (16 * (ks0 & 1) + 4 * g);
#pragma unroll
        for (int s = 0; s < QKS; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            odd |= !(__builtin_fabsf(st[s][r]) < INFINITY);
            st[s][r] = (bits >> (16 * s + r)) & 1u ? st[s][r] * a.scale_log2 : -INFINITY;
          }
        // (Loads of rare branches are waited for in them: where the compiler has to
        // assume them pending, it would wait for the tile in flight.)
        __builtin_amdgcn_s_waitcnt(wait_vm(0));
      } else {
#pragma unroll
        for (int s = 0; s < QKS; ++s) st[s] *= a.scale_log2;
      }
      float mt = -INFINITY;
#pragma unroll
      for (int s = 0; s < QKS; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) mt = fmaxf(mt, st[s][r]);
      mt = row_max4(mt);
      vote = mt > m_run + kSlack;
      if (g == 0) tile_max[half][16 * ct0 + l16] = mt;
    }
    if (EARLY_V && !scores) {
#pragma unroll
      for (int n = 0; n < DT; ++n) vals[EARLY_V ? n : 0] = rdv(n);
    }
    // The weights are rounded to T for the products (a matrix instruction's
    // operands are of one type); the sum that divides them counts them as rounded.
    auto weigh = [&]() {
      const float base = m_run == -INFINITY ? 0.f : kWeightLift<T> - m_run;
#pragma unroll
      for (int s = 0; s < QKS; ++s) {
        T w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          w[r] = from_f32<T>(fast_exp2(st[s][r] + base));
          l_run += to_f32(w[r]);
        }
        uint2 both;
        __builtin_memcpy(&both, w, 8);
        probs[(((ks0 + s) / 2 * NC + ct0) * 64 + ln) * 2 + (ks0 + s) % 2] = both;
      }
    };
    const bool any_vote = __any(vote), any_odd = __any(odd);
    const float l_before = l_run;
    if (scores && !any_vote) weigh();
    if (ln == 0) votes[wave] = (any_vote ? 1u : 0u) | (any_odd ? 2u : 0u);
    lds_barrier();
    uint32_t said = 0;
#pragma unroll
    for (int w = 0; w < W; w += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(votes + w);
      said |= v.x | v.y | v.z | v.w;
    }
    said = __builtin_amdgcn_readfirstlane(said);
    if (said & 1u) {
      // Some column's maximum moves: all waves move every column to its own.
      auto moved = [&](int c, float& before) -> float {
        const int i = 16 * c + l16;
        before = col_max[i];
        return fmaxf(before, HALVES == 1 ? tile_max[0][i] : fmaxf(tile_max[0][i], tile_max[1][i]));
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
        // (Weights that were formed with the old maximum count anew.)
        float before;
        const float after = moved(ct0, before);
        l_run = l_before * ratio(before, after);
        m_run = after;
        weigh();
      }
      lds_barrier();
      if (scores && g == 0 && half == 0) col_max[16 * ct0 + l16] = m_run;
    }
    if (APPEND && masked && __any(slot >= 0)) {
      if (slot >= 0) {
        const int lchunk = (ln & 7) ^ swizzle(8 * rb + (ln >> 3));
        gptr<T> const to = pool + (int64_t)slot * S::ROW;
#pragma unroll
        for (int i = 0; i < (GR + GSTEP - 1) / GSTEP; ++i) {
          const int gr = wave / RB + i * GSTEP, c = 8 * gr + lchunk;
          if (c < S::CPR)
            store16(to + 8 * c, *reinterpret_cast<const uint4*>(here + (gr * (KT * 128) + rb * 1024 + ln * 16)));
        }
      }
    }
    const bool poisoned = (said & 2u) != 0;
    if (poisoned) {
      lds_barrier();  // (the rows on their way to the pool have been read)
      // The step's rows without their values that are not finite (and none of
      // the repeated rows past the piece's end).
      const int lrow = 8 * rb + (ln >> 3);
      if (t0 + lrow >= cur.computed && wave < RB) {
#pragma unroll 1
        for (int c = 0; c < L / 8; ++c) {
          if ((c & 7) != ((ln & 7) ^ swizzle(lrow))) continue;
          uint4* const at8 = reinterpret_cast<uint4*>(const_cast<char*>(here) + ((c >> 3) * (KT * 128) + rb * 1024 + ln * 16));
          T v[8];
          const uint4 had = *at8;
          __builtin_memcpy(v, &had, 16);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (not_finite(v[e])) v[e] = from_f32<T>(0.f);
          uint4 has;
          __builtin_memcpy(&has, v, 16);
          *at8 = has;
        }
      }
      lds_barrier();
      if constexpr (EARLY_V) {
#pragma unroll
        for (int n = 0; n < DT; ++n) vals[n] = rdv(n);
      }
    }

    // ---- O^T += V^T P^T.  The fewer of the two operands' registers are held (all
    // of a wave's values, or all columns' weights), the other is read LEAD ahead.
    {
      auto rdp = [&](int c) -> V8 { return bitcast<V8>(*reinterpret_cast<const uint4*>(probs + (c * 64 + ln) * 2)); };
      auto mm = [&](V8 v, V8 w, f32x4 x) -> f32x4 {
        if constexpr (std::is_same<T, __bf16>::value) {
          return __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, w, x, 0, 0, 0);
        } else {
          return __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w, x, 0, 0, 0);
        }
      };
      if constexpr (EARLY_V) {
#pragma unroll
        for (int step = 0; step < STEPS; ++step) {
          V8 w[NC], more[DT];
#pragma unroll
          for (int c = 0; c < NC; ++c) w[c] = rdp(step * NC + c);
          if (step + 1 < STEPS) {
#pragma unroll
            for (int n = 0; n < DT; ++n) more[n] = rdv(n, step + 1);
          }
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int n = 0; n < DT; ++n) acc[c][n] = mm(vals[n], w[c], acc[c][n]);
          if (step + 1 < STEPS) {
#pragma unroll
            for (int n = 0; n < DT; ++n) vals[n] = more[n];
          }
        }
      } else {
        constexpr bool HOLD_V = NC > DT;
        constexpr int HELD = HOLD_V ? DT : NC, TOT = HOLD_V ? NC : DT, LEAD = TOT < 2 ? TOT : 2;
        V8 held[HELD], ahead[LEAD];
#pragma unroll
        for (int i = 0; i < HELD; ++i) held[i] = HOLD_V ? rdv(i) : rdp(i);
#pragma unroll
        for (int i = 0; i < LEAD; ++i) ahead[i] = HOLD_V ? rdp(i) : rdv(i);
        if constexpr (NC == 8) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TOT; ++i) {
          const V8 x = ahead[i % LEAD];
          if (i + LEAD < TOT) ahead[i % LEAD] = HOLD_V ? rdp(i + LEAD) : rdv(i + LEAD);
#pragma unroll
          for (int k = 0; k < HELD; ++k) {
            f32x4& to = acc[HOLD_V ? i : k][HOLD_V ? k : i];
            to = HOLD_V ? mm(held[k], x, to) : mm(x, held[k], to);
          }
          if constexpr (NC == 8) __builtin_amdgcn_sched_barrier(0);
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
            APPEND && a.latent_new ? (gptr<const T>)(a.latent_new) + (int64_t)(cur.q_start + pos - cur.computed) * a.latent_stride
                         : pool + ((int64_t)a.tables[cur.table_off + lb] * a.block_size + (pos - lb * a.block_size)) * S::ROW;
        uint32_t sees = 0;  // bit c: this lane's column of tile c
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          int qi, head;
          columns(ln, cur, c, qi, head);
          sees |= ((window(cur, qi, t0 + ((pos - t0) & ~31)) >> ((pos - t0) & 31)) & 1u) << c;
        }
#pragma unroll
        for (int n = 0; n < DT; ++n) {
          f32x4 zero_or_nan;
#pragma unroll
          for (int r = 0; r < 4; ++r) zero_or_nan[r] = to_f32((T)v[16 * (wave * DT + n) + 4 * g + r]) * 0.f;
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[c][n][r] += (sees >> c) & 1u ? zero_or_nan[r] : 0.f;
        }
      }
      __builtin_amdgcn_s_waitcnt(wait_vm(0));
    }

    t0 += KT;
    if (t0 < cur.tok_end) return true;
    // ---- a finished piece: its output rows, or its partials
    if (scores) {
      const float l = row_sum4(l_run);
      if (g == 0) col_sum[half][16 * ct0 + l16] = l;
    }
    lds_barrier();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = 16 * c + l16;
      const float l_tot = HALVES == 1 ? col_sum[0][i] : col_sum[0][i] + col_sum[1][i];
      // (A piece may hold no row that a column sees, and weighs nothing then; a whole
      // request's softmax without a finite score is NaN.)
      const float inv = l_tot > 0.f ? 1.f / l_tot : cur.slot < 0 ? NAN : l_tot == l_tot ? 0.f : l_tot;
      int qi, head;
      if (!columns(ln, cur, c, qi, head)) continue;
      if (cur.slot < 0) {
        T* to = static_cast<T*>(a.out) + (int64_t)(cur.row + qi) * a.out_tok_stride + (int64_t)head * a.out_head_stride;
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
    if (cur.next < 0) return false;
    // (The next piece's queries arrive with its first tile: the wait at the top
    // of a step is for both.)
    cur = read_latent_piece(pieces, cur.next);
    load_queries(ln, cur);
    t0 = cur.tok_begin;
    fresh = true;
    return true;
  };
  while (step(tile0, tile1) && step(tile1, tile0)) {
  }
}

// ---------------------------------------------------------------------------
// Merge: a workgroup per (job, column), a thread per four dimensions and other
// piece; the two shares of the pieces join in LDS, in order.  (64 requests of 16
// heads 5.1 us, 6.8 with one share in two passes; 32 of 144 columns 13.1, 16.8 with
// four shares; bound by the partials, 2 KB a column and piece.)  With partial i's
// maximum m_i (log2) and sum l_i, out = sum 2^(m_i - M) l_i o_i / sum 2^(m_i - M) l_i,
// taken in one pass: a share's sums are scaled when its maximum moves.
// ---------------------------------------------------------------------------
constexpr int MERGE_SHARES = 2;
template <typename T, int L>
__global__ __launch_bounds__(L / 4 * MERGE_SHARES) void latent_merge_kernel(const int32_t* __restrict__ jobs, const int32_t cols,
                                                                            const LatentDecodeArgs a) {
  constexpr int LANES = L / 4, S = MERGE_SHARES, AT_ONCE = 4;
  __shared__ f32x4 sums[S - 1][LANES];
  __shared__ float maxima[S], totals[S];
  const int32_t* jb = jobs + (int64_t)blockIdx.x * LVAMD_MERGE_FIELDS;
  const int row = jb[0], group = jb[1], slot0 = jb[2], np = jb[3], q_len = jb[5];
  const int i = blockIdx.y;
  const int col = group * cols + i;
  if (col >= q_len * a.heads) return;
  const int at = threadIdx.x % LANES, share = threadIdx.x / LANES;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (int64_t)slot0 * cols + i;
  const float* from = a.part_acc + ((int64_t)slot0 * cols + i) * L + 4 * at;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, total = 0.f;
  for (int k0 = share; k0 < np; k0 += S * AT_ONCE) {
    f32x4 o[AT_ONCE];
    float2 of[AT_ONCE];
    float top = m;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int k = min(k0 + S * j, np - 1);
      of[j] = ml[(int64_t)k * cols];
      o[j] = *reinterpret_cast<const f32x4*>(from + (int64_t)k * cols * L);
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (k0 + S * j < np) top = fmaxf(top, of[j].x);
    const float had = m == -INFINITY ? 0.f : fast_exp2(m - top);
    sum *= had;
    total *= had;
    m = top;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      if (k0 + S * j >= np) break;
      const float w = of[j].x == -INFINITY ? 0.f : fast_exp2(of[j].x - m) * of[j].y;
      total += w;
      sum += o[j] * w;
    }
  }
  if (share) sums[share - 1][at] = sum;
  if (at == 0) {
    maxima[share] = m;
    totals[share] = total;
  }
  __syncthreads();
  if (share) return;
  float top = m;
#pragma unroll
  for (int s = 1; s < S; ++s) top = fmaxf(top, maxima[s]);
  const float had = m == -INFINITY ? 0.f : fast_exp2(m - top);
  sum *= had;
  total *= had;
#pragma unroll
  for (int s = 1; s < S; ++s) {
    const float w = maxima[s] == -INFINITY ? 0.f : fast_exp2(maxima[s] - top);
    total += totals[s] * w;
    sum += sums[s - 1][at] * w;
  }
  const int qi = fast_div(col, a.by_heads), head = col - qi * a.heads;
  T* to = static_cast<T*>(a.out) + (int64_t)(row + qi) * a.out_tok_stride + (int64_t)head * a.out_head_stride;
  const float inv = total > 0.f ? 1.f / total : NAN;  // (no finite score in any piece)
  store_partial4<false, T>(to + 4 * at, sum, inv);
}

template <typename T, int L, int P>
static const void* latent_decode_fn(int col_tiles) {
  switch (col_tiles) {
    case 1: return (const void*)&latent_decode_kernel<T, L, P, 1>;
    case 2: return (const void*)&latent_decode_kernel<T, L, P, 2>;
    case 4: return (const void*)&latent_decode_kernel<T, L, P, 4>;
    case 8: return (const void*)&latent_decode_kernel<T, L, P, 8>;
    default: return nullptr;
  }
}

}  // namespace lvamd

using namespace lvamd;

extern "C" int lvamd_latent_decode_tile_tokens(int32_t col_tiles) { return tile_rows(col_tiles); }

extern "C" int lvamd_latent_decode_resident_groups(int32_t dtype, int32_t latent_size, int32_t rope_size, int32_t col_tiles) {
  return latent_dispatch(dtype, latent_size, rope_size, [&]<typename T, int L, int P>() -> int {
    const void* fn = latent_decode_fn<T, L, P>(col_tiles);
    int device = 0, cus = 0, per_cu = 0;
    if (!fn) return LVAMD_ERR_UNSUPPORTED;
    if (hipGetDevice(&device) != hipSuccess) return LVAMD_ERR_LAUNCH;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess) return LVAMD_ERR_LAUNCH;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, fn, col_tiles >= 4 ? 512 : 256, 0) != hipSuccess) return LVAMD_ERR_LAUNCH;
    return per_cu * cus;
  });
}

extern "C" int lvamd_latent_decode(const void* query, int64_t query_token_stride, int64_t query_head_stride,
                                   const void* query_rope, int64_t rope_token_stride, int64_t rope_head_stride,
                                   const void* latent, int64_t latent_token_stride, const void* rope_key,
                                   int64_t rope_key_token_stride, const float* cosines, const float* sines,
                                   int64_t angle_token_stride, int32_t interleaved, void* pool, void* out,
                                   int64_t out_token_stride, int64_t out_head_stride,
                                   const int32_t* pieces, int32_t num_groups,
                                   const int32_t* jobs, int32_t num_jobs, int32_t merge_columns, const int32_t* tables,
                                   const uint32_t* vis, float* part_acc, float* part_ml, int64_t num_partial_slots,
                                   int32_t num_heads, int32_t latent_size, int32_t rope_size, int32_t col_tiles,
                                   int32_t block_size, float scale, int32_t dtype, lvamd_stream_t stream) {
  if (!latent_sizes(latent_size, rope_size) || !latent_dtype(dtype)) return LVAMD_ERR_UNSUPPORTED;
  if (num_groups < 0 || num_jobs < 0 || num_heads <= 0 || block_size <= 0 || num_partial_slots < 0 || merge_columns < 0 ||
      merge_columns > 65535)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_groups == 0) return LVAMD_OK;
  if (!query || !query_rope || !pool || !out || !pieces || !tables || !vis || (num_jobs > 0 && !jobs))
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_partial_slots > 0 && (!part_acc || !part_ml)) return LVAMD_ERR_WORKSPACE;
  if (!rows16(query, {query_token_stride, query_head_stride}) || !rows16(query_rope, {rope_token_stride, rope_head_stride}) ||
      !rows16(pool, {}) || ((uintptr_t)out & 7u) || out_token_stride % 4 != 0 || out_head_stride % 4 != 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (col_tiles > 4 && (latent || cosines)) return LVAMD_ERR_UNSUPPORTED;
  if ((latent == nullptr) != (rope_key == nullptr) || (cosines == nullptr) != (sines == nullptr) ||
      (latent && (!rows16(latent, {latent_token_stride}) || !rows16(rope_key, {rope_key_token_stride}))) ||
      (cosines && (((uintptr_t)cosines & 15u) || ((uintptr_t)sines & 15u) || angle_token_stride % 4 != 0)))
    return LVAMD_ERR_INVALID_ARGUMENT;
  LatentDecodeArgs a{.by_block = FastDiv(block_size), .by_heads = FastDiv(num_heads)};
  a.latent_new = latent;
  a.rope_new = rope_key;
  a.latent_stride = latent_token_stride;
  a.rope_stride = rope_key_token_stride;
  a.cosines = cosines;
  a.sines = sines;
  a.angle_stride = angle_token_stride;
  a.interleaved = interleaved;
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
    auto launch = [&]<int NC>() {
      hipLaunchKernelGGL((latent_decode_kernel<T, L, P, NC>), dim3((unsigned)num_groups), dim3(64 * LatentShape<L, P, NC>::W),
                         0, s, pieces, a);
    };
    switch (col_tiles) {
      case 1: launch.template operator()<1>(); break;
      case 2: launch.template operator()<2>(); break;
      case 4: launch.template operator()<4>(); break;
      case 8: launch.template operator()<8>(); break;
      default: return LVAMD_ERR_UNSUPPORTED;
    }
    if (const int status = launch_status(); status != LVAMD_OK) return status;
    if (num_jobs == 0) return LVAMD_OK;
    hipLaunchKernelGGL((latent_merge_kernel<T, L>), dim3((unsigned)num_jobs, (unsigned)merge_columns), dim3(L / 4 * MERGE_SHARES), 0, s,
                       jobs, 16 * col_tiles, a);
    return launch_status();
  });
}
