// Verification of drafted tokens against the target model's probabilities, from
// given uniform numbers.
//
// A request has a tree of drafts (a chain is one) and one row of target
// probabilities p per node: the root (before any draft) and every draft.
// With one uniform u per node, a node's children c1..ck are tried in order:
//   * drafts without probabilities (looked up, not drawn): child j is accepted
//     when p(c1) + .. + p(cj-1) <= u < p(c1) + .. + p(cj).  No child: the node's
//     token is drawn from p without the children's tokens.
//   * chains drawn from draft probabilities q: the child is accepted when
//     u * q(c) < p(c), else the token is drawn from max(p - q, 0).
// Either way the accepted tokens and the last one follow the target's
// distribution.  The walk ends at a node that accepts no child (or has none);
// its residual r is drawn from by inverse distribution: the first x with
// r(0) + .. + r(x) > u' * sum(r), u' one uniform per request.  A residual of
// zeros (p <= q everywhere by rounding) falls back to p.  Entries that are not
// finite and positive count as zero; with nothing to draw from the token is -1.
//
// All sums are in fp64: how they are split can change the drawn index only where
// the number lies within their rounding error (1e-13 of the sum) of a border.
//
// HBM-bound in large batches: one row of p per request (and one of q), 16-byte
// loads, several per lane in flight; a chain of round trips in small ones, over
// two dependent launches.  The accept tests need only p and q at the drafts
// themselves, so every workgroup of the first launch finds its request's last
// node itself (a gather of n values and a walk in LDS, in place of a launch
// before it); then its waves sum chunks of the residual, 4 KiB of a row each.
// The second launch is one wave per request, without a barrier: it scans the
// chunks' sums, then the one chunk that holds the draw.
//
// One request of 4 drafts, 151,936 tokens, fp32 with q: 4.9 + 4.0 us.  128 trees
// over 100,003 tokens, bf16: 12.9 + 4.8 us for 26 MB, of which the walk's two
// rounds of loads take about 4.  One launch of a workgroup per request won 1-2 us
// below 1000 tokens and lost up to four times at 151,936 (one CU then converts
// and adds every element).

#include <algorithm>
#include <cmath>

#include "lvamd_common.h"

namespace lvamd {

namespace {

constexpr int kMaxDrafts = LVAMD_VERIFY_MAX_DRAFTS;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kLoads = 4;  // 16-byte loads per lane and chunk

// What the first launch leaves the second: the last node (0: the root), its
// children, and the draft whose q is subtracted there (-1: none).
struct Stop {
  int32_t node, num_children, draft, unused;
};

struct VerifyArgs {
  const void* target;
  int64_t target_stride;
  const void* draft_probs;  // null: drafts without probabilities
  int64_t draft_stride;
  const int32_t* starts;    // [requests + 1]: first draft
  const int64_t* tokens;    // [drafts]
  const int32_t* parents;   // [drafts]: index within the request, -1 the root
  const int32_t* siblings;  // [drafts]: the sibling before it, or -1
  const void* node_uniforms;
  const void* sample_uniforms;
  double2* sums;            // [requests][chunks]: the residual's sum, p's sum
  Stop* stops;              // [requests]
  int32_t* children;        // [drafts]: the last node's children's tokens, from the request's first draft on
  int32_t* counts;
  int32_t* paths;
  int64_t* out_tokens;
  int32_t vocab, chunks, path_width;
  int32_t uniforms_f64;
};

// (Finite and positive: else zero.  Class bits: positive subnormal or normal.)
__device__ __forceinline__ float mass(float p) { return __builtin_amdgcn_classf(p, 0x180) ? p : 0.f; }

__device__ __forceinline__ double uniform_at(const void* u, int64_t i, int f64) {
  return f64 ? static_cast<const double*>(u)[i] : (double)static_cast<const float*>(u)[i];
}

template <typename T>
struct Wide {
  static constexpr int N = 16 / (int)sizeof(T);   // elements per load
  static constexpr int CHUNK = 64 * kLoads * N;   // elements per chunk
};

// 16 bytes of a row (its alignment is that of its elements: rows of odd length
// start anywhere): elements [at, at + N), at = i but for the row's end, where
// the load begins earlier and its elements before i do not count.
template <typename T>
struct Pack {
  typedef T Vec __attribute__((ext_vector_type(Wide<T>::N)));
  Vec e;
};
template <typename T>
__device__ __forceinline__ int pack_at(int i, int end) {
  return min(i, max(end - Wide<T>::N, 0));
}
template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const T* row, int i, int end) {
  constexpr int N = Wide<T>::N;
  Pack<T> v;
  if (end >= N) {
    typedef T Loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    v.e = *reinterpret_cast<const Loose*>(row + pack_at<T>(i, end));
  } else {  // a row shorter than the load
#pragma unroll
    for (int k = 0; k < N; ++k) v.e[k] = row[min(k, end - 1)];
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void masses(const Pack<T>& v, int i, int end, float (&x)[Wide<T>::N]) {
  const int at = pack_at<T>(i, end);
#pragma unroll
  for (int k = 0; k < Wide<T>::N; ++k)
    x[k] = at + k >= i && at + k < end ? mass(to_f32((T)v.e[k])) : 0.f;
}

// A lane's packs of a chunk, pack j from element first + j * step on.
template <typename T>
struct Packs {
  Pack<T> v[kLoads];
  int first, step;
  __device__ __forceinline__ int from(int j) const { return first + j * step; }
};
template <typename T>
__device__ __forceinline__ void load_packs(Packs<T>& x, const T* row, int first, int step, int end) {
  x.first = first;
  x.step = step;
#pragma unroll
  for (int j = 0; j < kLoads; ++j) x.v[j] = load_pack<T>(row, x.from(j), end);
}
// The children's tokens that lie in the chunk from `begin` on taken out; whether
// there are any.
template <typename T>
__device__ __forceinline__ bool take_out(Packs<T>& x, const int32_t* kids, int nkids, int begin, int end) {
  bool any = false;
  for (int c = 0; c < nkids; ++c) {
    const int kid = kids[c];
    if (kid < begin || kid >= begin + Wide<T>::CHUNK) continue;  // (uniform)
    any = true;
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
#pragma unroll
      for (int k = 0; k < Wide<T>::N; ++k)
        if (pack_at<T>(x.from(j), end) + k == kid) x.v[j].e[k] = (T)0.f;
  }
  return any;
}
// Residual of pack j's elements: p, or p - q (exact in fp64: two 24-bit values)
// where that is positive.
template <typename T, bool DRAWN>
__device__ __forceinline__ void residual(const Packs<T>& p, const Packs<T>& q, int j, int end, double (&r)[Wide<T>::N]) {
  constexpr int N = Wide<T>::N;
  float x[N];
  masses<T>(p.v[j], p.from(j), end, x);
  if constexpr (DRAWN) {
    float y[N];
    masses<T>(q.v[j], q.from(j), end, y);
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = x[k] > y[k] ? (double)x[k] - (double)y[k] : 0.0;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = (double)x[k];
  }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// Sum over the wave's lanes up to each.
__device__ __forceinline__ double wave_scan(double v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

template <bool DRAWN>
struct WalkShared {
  float p[kMaxDrafts], q[DRAWN ? kMaxDrafts : 1];  // the drafts' own probabilities
  int16_t next[kMaxDrafts + 1];                       // per node, the draft accepted there (plus one), or -1
  int16_t after[DRAWN ? 1 : kMaxDrafts];              // per draft, the next sibling, or -1
  int32_t kids[kMaxDrafts];
  int node, num_kids, kid_draft;
};

// The request's last node, its children's tokens (s.kids) and its one draft
// (chains drawn from q), found by a workgroup: two rounds of loads and a walk in
// LDS.  `leader` writes the accepted path.
template <typename T, bool DRAWN, int THREADS>
__device__ __forceinline__ Stop walk(const VerifyArgs& a, int req, bool leader, WalkShared<DRAWN>& s) {
  constexpr int PER = kMaxDrafts / THREADS;
  const int first = a.starts[req];
  const int n = min(a.starts[req + 1] - first, kMaxDrafts);
  const int64_t row0 = (int64_t)first + req;  // the root's row
  const T* target = static_cast<const T*>(a.target);
  const T* drafts = static_cast<const T*>(a.draft_probs);
  if (threadIdx.x == 0) {
    s.node = s.num_kids = 0;
    s.kid_draft = -1;
  }
  int parent[PER], token[PER], sibling[PER];
  double u[PER];
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = threadIdx.x + THREADS * i;
      if (c >= n) break;
      const int64_t tok = a.tokens[first + c];
      token[i] = tok >= 0 && tok < a.vocab ? (int)tok : -1;
      parent[i] = a.parents[first + c] + 1;
      sibling[i] = a.siblings[first + c];
      s.next[c] = -1;
      if constexpr (!DRAWN) s.after[c] = -1;
    }
    if (threadIdx.x == 0) s.next[n] = -1;
    if constexpr (!DRAWN) __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = threadIdx.x + THREADS * i;
      if (c >= n) break;
      if constexpr (!DRAWN)
        if (sibling[i] >= 0 && sibling[i] < c) s.after[sibling[i]] = (int16_t)c;
      const int64_t tok = max(token[i], 0);
      const float p = to_f32(target[(row0 + parent[i]) * a.target_stride + tok]);
      u[i] = uniform_at(a.node_uniforms, row0 + parent[i], a.uniforms_f64);
      if constexpr (DRAWN) {
        const float q = to_f32(drafts[(int64_t)(first + c) * a.draft_stride + tok]);
        s.q[c] = token[i] >= 0 ? mass(q) : 0.f;
      }
      s.p[c] = token[i] >= 0 ? mass(p) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = threadIdx.x + THREADS * i;
      if (c >= n) break;
      if constexpr (DRAWN) {
        if (u[i] * (double)s.q[c] < (double)s.p[c]) s.next[parent[i]] = (int16_t)(c + 1);
      } else if (sibling[i] < 0 && u[i] >= 0.0) {
        // A node's first child takes them all in order, so an interval's upper
        // border is the next one's lower border bit for bit.
        double upto = 0.0;
        for (int k = c; k >= 0; k = s.after[k]) {
          upto += (double)s.p[k];
          if (u[i] < upto) {
            s.next[parent[i]] = (int16_t)(k + 1);
            break;
          }
        }
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    int node = 0, count = 0;
    if (n > 0)
      for (int to = s.next[0]; to >= 0 && count < n; to = s.next[to]) {
        node = to;
        if (leader && count < a.path_width) a.paths[(int64_t)req * a.path_width + count] = node - 1;
        ++count;
      }
    s.node = node;
    if (leader) {
      a.counts[req] = count;
      for (int i = count; i < a.path_width; ++i) a.paths[(int64_t)req * a.path_width + i] = -1;
    }
  }
  __syncthreads();
  const int node = s.node;
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = threadIdx.x + THREADS * i;
      if (c >= n) break;
      if (parent[i] == node) {
        s.kids[atomicAdd(&s.num_kids, 1)] = token[i];
        s.kid_draft = first + c;  // (a chain has one)
      }
    }
    __syncthreads();
  }
  return {node, s.num_kids, DRAWN ? s.kid_draft : -1, 0};
}

// The rows at the request's last node: p, and what is subtracted from it (null:
// nothing).
template <typename T>
struct Rows {
  const T *p, *q;
};
template <typename T, bool DRAWN>
__device__ __forceinline__ Rows<T> rows_at(const VerifyArgs& a, int req, const Stop& stop) {
  const int64_t row = (int64_t)a.starts[req] + req + stop.node;
  return {static_cast<const T*>(a.target) + row * a.target_stride,
          DRAWN && stop.draft >= 0 ? static_cast<const T*>(a.draft_probs) + (int64_t)stop.draft * a.draft_stride : nullptr};
}

// A lane's part of a chunk's sums: the residual's, and p's.
template <typename T, bool DRAWN>
struct Chunk {
  static constexpr int N = Wide<T>::N;
  Packs<T> p, q = {};
  __device__ __forceinline__ void load(const Rows<T>& rows, int chunk, int lane, int vocab) {
    load_packs<T>(p, rows.p, chunk * Wide<T>::CHUNK + lane * N, 64 * N, vocab);
    if constexpr (DRAWN) {
      if (rows.q) load_packs<T>(q, rows.q, chunk * Wide<T>::CHUNK + lane * N, 64 * N, vocab);  // (else zeros)
    }
  }
  template <bool LESS>
  __device__ __forceinline__ double sum(int vocab) const {
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      double r[N];
      residual<T, LESS>(p, q, j, vocab, r);
#pragma unroll
      for (int k = 0; k < N; ++k) s += r[k];
    }
    return s;
  }
  __device__ __forceinline__ double2 sums(const Rows<T>& rows, const int32_t* kids, int nkids, int chunk, int vocab) {
    const double full = sum<false>(vocab);
    double rest = full;
    if constexpr (DRAWN) {
      if (rows.q) rest = sum<true>(vocab);
    } else {
      if (take_out<T>(p, kids, nkids, chunk * Wide<T>::CHUNK, vocab)) rest = sum<false>(vocab);
    }
    return make_double2(wave_sum(rest), wave_sum(full));
  }
};

// The draw, by one wave: the chunk that holds it from the chunks' sums, then the
// element.
template <typename T, bool DRAWN>
__device__ __forceinline__ void draw(const VerifyArgs& a, int req, int lane, const double2* sums, const Rows<T>& rows,
                                     const int32_t* kids, int nkids) {
  constexpr int N = Wide<T>::N;
  constexpr int kHeld = 4;  // rounds of 64 chunks whose sums stay in registers
  const double u = uniform_at(a.sample_uniforms, req, a.uniforms_f64);
  double2 held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = 64 * i + lane < a.chunks ? sums[64 * i + lane] : make_double2(0.0, 0.0);
  double rest = 0.0, full = 0.0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    rest += held[i].x;
    full += held[i].y;
  }
  for (int c = 64 * kHeld + lane; c < a.chunks; c += 64) {
    rest += sums[c].x;
    full += sums[c].y;
  }
  rest = wave_sum(rest);
  full = wave_sum(full);
  const bool residual_left = rest > 0.0;
  const double goal = u * (residual_left ? rest : full);
  // The first chunk whose sums pass the goal; the last that holds anything
  // where none does (u >= 1, or by rounding).
  int at = -1, tail = -1;
  double done = 0.0, base = 0.0, tail_base = 0.0;
  auto round = [&](int r, double2 s) {
    const double mine = residual_left ? s.x : s.y;
    const double upto = done + wave_scan(mine, lane);
    const uint64_t pass = __ballot(upto > goal), some = __ballot(mine > 0.0);
    if (pass && at < 0) {
      const int l = __builtin_ctzll(pass);
      at = 64 * r + l;
      base = __shfl(upto - mine, l);
    }
    if (some) {
      const int l = 63 - __builtin_clzll(some);
      tail = 64 * r + l;
      tail_base = __shfl(upto - mine, l);
    }
    done = __shfl(upto, 63);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (at < 0 && 64 * i < a.chunks) round(i, held[i]);
  for (int i = kHeld; at < 0 && 64 * i < a.chunks; ++i)
    round(i, 64 * i + lane < a.chunks ? sums[64 * i + lane] : make_double2(0.0, 0.0));
  if (at < 0) {
    at = tail;
    base = tail_base;
  }
  if (at < 0) {
    if (lane == 0) a.out_tokens[req] = -1;
    return;
  }
  // The chunk, kLoads * N elements in a row per lane.
  const T* qrow = residual_left ? rows.q : nullptr;
  const int begin = at * Wide<T>::CHUNK + lane * kLoads * N;
  Packs<T> p, q = {};
  load_packs<T>(p, rows.p, begin, N, a.vocab);
  if constexpr (DRAWN) {
    if (qrow) load_packs<T>(q, qrow, begin, N, a.vocab);
  } else {
    if (residual_left) take_out<T>(p, kids, nkids, at * Wide<T>::CHUNK, a.vocab);
  }
  double r[kLoads][N], s = 0.0;
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    residual<T, DRAWN>(p, q, j, a.vocab, r[j]);
#pragma unroll
    for (int k = 0; k < N; ++k) s += r[j][k];
  }
  double c = base + (wave_scan(s, lane) - s);
  int hit = -1, last = -1;
#pragma unroll
  for (int j = 0; j < kLoads; ++j)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      c += r[j][k];
      if (r[j][k] > 0.0) {
        last = pack_at<T>(begin + j * N, a.vocab) + k;
        if (c > goal && hit < 0) hit = last;
      }
    }
  const uint64_t hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
  const int token = hits ? __shfl(hit, __builtin_ctzll(hits)) : lasts ? __shfl(last, 63 - __builtin_clzll(lasts)) : -1;
  if (lane == 0) a.out_tokens[req] = token;
}

}  // namespace

// Grid of the first launch: (workgroups per request, requests); every
// workgroup walks, then a request's waves take its chunks in turn.
template <typename T, bool DRAWN>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4))) void verify_sums_kernel(
    const VerifyArgs a) {
  __shared__ WalkShared<DRAWN> s;
  const int req = blockIdx.y;
  const bool leader = blockIdx.x == 0;  // writes what is found
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const Stop stop = walk<T, DRAWN, kThreads>(a, req, leader, s);
  if (leader) {
    if (threadIdx.x == 0) a.stops[req] = stop;
    for (int c = threadIdx.x; c < stop.num_children; c += kThreads) a.children[a.starts[req] + c] = s.kids[c];
  }
  const Rows<T> rows = rows_at<T, DRAWN>(a, req, stop);
  for (int chunk = blockIdx.x * kWaves + wave; chunk < a.chunks; chunk += gridDim.x * kWaves) {
    Chunk<T, DRAWN> x;
    x.load(rows, chunk, lane, a.vocab);
    const double2 sum = x.sums(rows, s.kids, stop.num_children, chunk, a.vocab);
    if (lane == 0) a.sums[(int64_t)req * a.chunks + chunk] = sum;
  }
}

// Grid of the second: requests, one wave each.
template <typename T, bool DRAWN>
__global__ __launch_bounds__(64) void verify_draw_kernel(const VerifyArgs a) {
  const int req = blockIdx.x;
  const Stop stop = a.stops[req];
  draw<T, DRAWN>(a, req, threadIdx.x & 63, a.sums + (int64_t)req * a.chunks, rows_at<T, DRAWN>(a, req, stop),
                 a.children + a.starts[req], stop.num_children);
}

}  // namespace lvamd

using namespace lvamd;

static int verify_chunks(int32_t vocab, int32_t dtype) {
  const int chunk = 64 * kLoads * (dtype == LVAMD_F32 ? 4 : 8);
  return (vocab + chunk - 1) / chunk;
}

extern "C" int64_t lvamd_verify_drafts_workspace_size(int64_t num_requests, int64_t num_drafts, int32_t vocab,
                                                      int32_t dtype) {
  if (num_requests <= 0 || num_drafts < 0 || vocab <= 0) return 0;
  return num_requests * ((int64_t)verify_chunks(vocab, dtype) * (int64_t)sizeof(double2) + (int64_t)sizeof(Stop)) +
         num_drafts * 4;
}

extern "C" int lvamd_verify_drafts(const void* target, int64_t target_row_stride, const void* draft_probs,
                                   int64_t draft_row_stride, int32_t vocab, int32_t dtype, const int32_t* draft_starts,
                                   const int64_t* draft_tokens, const int32_t* parents, const int32_t* siblings,
                                   int64_t num_requests, int64_t num_drafts, const void* node_uniforms,
                                   const void* sample_uniforms, int32_t uniforms_f64, int32_t* counts, int32_t* paths, int32_t path_width,
                                   int64_t* out_tokens, void* workspace, int64_t workspace_bytes,
                                   lvamd_stream_t stream) {
  if (dtype_size(dtype) == 0) return LVAMD_ERR_UNSUPPORTED;
  if (num_requests < 0 || num_requests > 65535 || num_drafts < 0 || vocab <= 0 || vocab > (1 << 30) || path_width < 1 ||
      target_row_stride < 0 || draft_row_stride < 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_requests == 0) return LVAMD_OK;
  if (!target || !draft_starts || !draft_tokens || !parents || !siblings || !node_uniforms || !sample_uniforms ||
      !counts || !paths || !out_tokens)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (!workspace || ((uintptr_t)workspace & 15u) != 0 ||
      workspace_bytes < lvamd_verify_drafts_workspace_size(num_requests, num_drafts, vocab, dtype))
    return LVAMD_ERR_WORKSPACE;
  VerifyArgs a{};
  a.target = target;
  a.target_stride = target_row_stride;
  a.draft_probs = draft_probs;
  a.draft_stride = draft_row_stride;
  a.starts = draft_starts;
  a.tokens = draft_tokens;
  a.parents = parents;
  a.siblings = siblings;
  a.node_uniforms = node_uniforms;
  a.sample_uniforms = sample_uniforms;
  a.chunks = verify_chunks(vocab, dtype);
  a.sums = static_cast<double2*>(workspace);
  a.stops = reinterpret_cast<Stop*>(a.sums + num_requests * a.chunks);
  a.children = reinterpret_cast<int32_t*>(a.stops + num_requests);
  a.counts = counts;
  a.paths = paths;
  a.path_width = path_width;
  a.out_tokens = out_tokens;
  a.vocab = vocab;
  a.uniforms_f64 = uniforms_f64 != 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  // A chunk per wave while kWorkgroups (six per CU, all resident) suffice; several
  // in larger batches, which spreads the walk over more of the row.  (512 requests
  // of 151,936 fp32 tokens: 1024 91 us, 1536 78, 2048 93, 4096 83; 128 of 100,003:
  // 20.9, 19.2, 22.4, 21.8; up to 8 requests no difference.)
  constexpr int64_t kWorkgroups = 1536;
  const int64_t most = (a.chunks + kWaves - 1) / kWaves;
  const int64_t share = std::max<int64_t>(1, std::min<int64_t>(most, kWorkgroups / num_requests));
  const dim3 grid((unsigned)share, (unsigned)num_requests), draw((unsigned)num_requests), threads(kThreads);
  auto launch = [&]<typename T, bool DRAWN>() -> int {
    hipLaunchKernelGGL((verify_sums_kernel<T, DRAWN>), grid, threads, 0, s, a);
    const int status = launch_status();
    if (status != LVAMD_OK) return status;
    hipLaunchKernelGGL((verify_draw_kernel<T, DRAWN>), draw, dim3(64), 0, s, a);
    return launch_status();
  };
  auto launch_t = [&]<typename T>() -> int {
    return draft_probs ? launch.template operator()<T, true>() : launch.template operator()<T, false>();
  };
  switch (dtype) {
    case LVAMD_BF16: return launch_t.template operator()<__bf16>();
    case LVAMD_F16: return launch_t.template operator()<_Float16>();
    default: return launch_t.template operator()<float>();
  }
}
