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
// All sums are in fp64, so the drawn index does not depend on how they are
// split (a sum's error, 1e-13, against the 1e-6 of a 150,000-token border).
//
// HBM-bound in large batches: one row of p per request (and one of q), 16-byte
// loads; two dependent launches otherwise.  The accept tests need only p and q
// at the drafts themselves, so every workgroup of the first launch finds its
// request's last node itself (a gather of n values and a walk in LDS, in place
// of a launch before it), then sums its chunk of the residual; the second
// finds the chunk that holds the draw and scans it.

#include <cmath>

#include "lvamd_common.h"

namespace lvamd {

namespace {

constexpr int kMaxDrafts = LVAMD_VERIFY_MAX_DRAFTS;
constexpr int kThreads = 256;
constexpr int kMaxChunks = kThreads;  // one partial sum per thread of the second launch

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
  double* sums;             // [requests][chunks][2]: the residual's sum, p's sum
  int32_t* stops;           // [requests]: the last node, 0 the root
  int32_t* counts;
  int32_t* paths;
  int64_t* out_tokens;
  int32_t vocab, chunks, chunk, path_width;
  int32_t uniforms_f64;
};

// (Finite and positive: else zero.)
__device__ __forceinline__ float mass(float p) { return p > 0.f && p < INFINITY ? p : 0.f; }

__device__ __forceinline__ double uniform_at(const void* u, int64_t i, int f64) {
  return f64 ? static_cast<const double*>(u)[i] : (double)static_cast<const float*>(u)[i];
}

template <typename T>
struct Wide {
  static constexpr int N = 16 / (int)sizeof(T);
};

// N = 16 bytes of a row from element i on (the row's alignment is that of its
// elements: rows of odd length start anywhere); elements from `end` on are 0.
template <typename T>
__device__ __forceinline__ void load_wide(const T* row, int i, int end, float (&x)[Wide<T>::N]) {
  constexpr int N = Wide<T>::N;
  if (i + N <= end) {
    struct __attribute__((packed, aligned(sizeof(T)))) V {
      T e[N];
    };
    const V v = *reinterpret_cast<const V*>(row + i);
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = mass(to_f32(v.e[k]));
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = i + k < end ? mass(to_f32(row[i + k])) : 0.f;
  }
}

// The node's children: their tokens (any order), and the draft whose q is
// subtracted (the first found; a chain has one).
struct Children {
  int count, draft;
};
__device__ __forceinline__ void list_children(const VerifyArgs& a, int first, int n, int node, int64_t* tokens,
                                              Children* found) {
  if (threadIdx.x == 0) *found = {0, -1};
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += kThreads)
    if (a.parents[first + c] + 1 == node) {
      tokens[atomicAdd(&found->count, 1)] = a.tokens[first + c];
      found->draft = first + c;
    }
  __syncthreads();
}

// Residual and p of N elements from i on.  p is exact, and so is p - q in
// fp64 (the residual of two 24-bit values).
template <typename T>
__device__ __forceinline__ void residual(const T* prow, const T* qrow, const int64_t* kids, int nkids, int i, int end,
                                         float (&p)[Wide<T>::N], double (&r)[Wide<T>::N]) {
  constexpr int N = Wide<T>::N;
  load_wide<T>(prow, i, end, p);
  if (qrow != nullptr) {
    float q[N];
    load_wide<T>(qrow, i, end, q);
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = p[k] > q[k] ? (double)p[k] - (double)q[k] : 0.0;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = (double)p[k];
    for (int c = 0; c < nkids; ++c) {
      const int64_t at = kids[c] - i;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (at == k) r[k] = 0.0;
    }
  }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

}  // namespace

// Grid: (chunks, requests).
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(const VerifyArgs a) {
  __shared__ float mp[kMaxDrafts], mq[kMaxDrafts];
  __shared__ int next[kMaxDrafts + 1];
  __shared__ int64_t kids[kMaxDrafts];
  __shared__ Children found;
  __shared__ int stop;
  __shared__ double part[kThreads / 64][2];
  const int req = blockIdx.y;
  const int first = a.starts[req];
  const int n = min(a.starts[req + 1] - first, kMaxDrafts);
  const int64_t row0 = (int64_t)first + req;  // the root's row
  const T* target = static_cast<const T*>(a.target);
  const T* drafts = static_cast<const T*>(a.draft_probs);
  for (int c = threadIdx.x; c < n; c += kThreads) {
    const int64_t tok = a.tokens[first + c];
    const bool in = tok >= 0 && tok < a.vocab;
    mp[c] = in ? mass(to_f32(target[(row0 + a.parents[first + c] + 1) * a.target_stride + tok])) : 0.f;
    mq[c] = in && drafts ? mass(to_f32(drafts[(int64_t)(first + c) * a.draft_stride + tok])) : 0.f;
  }
  for (int c = threadIdx.x; c <= n; c += kThreads) next[c] = -1;
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += kThreads) {
    const int parent = a.parents[first + c] + 1;
    const double u = uniform_at(a.node_uniforms, row0 + parent, a.uniforms_f64);
    bool taken;
    if (drafts) {
      taken = u * (double)mq[c] < (double)mp[c];
    } else {
      double before = 0.0;
      for (int s = a.siblings[first + c]; s >= 0; s = a.siblings[first + s]) before += (double)mp[s];
      taken = u >= before && u < before + (double)mp[c];
    }
    if (taken) next[parent] = c + 1;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool write = blockIdx.x == 0;
    int node = 0, count = 0;
    for (int to = next[0]; to >= 0 && count < n; to = next[to]) {
      node = to;
      if (write && count < a.path_width) a.paths[(int64_t)req * a.path_width + count] = node - 1;
      ++count;
    }
    stop = node;
    if (write) {
      a.counts[req] = count;
      a.stops[req] = node;
      for (int i = count; i < a.path_width; ++i) a.paths[(int64_t)req * a.path_width + i] = -1;
    }
  }
  __syncthreads();
  const int node = stop;
  list_children(a, first, n, node, kids, &found);
  const T* prow = target + (row0 + node) * a.target_stride;
  const T* qrow = drafts && found.draft >= 0 ? drafts + (int64_t)found.draft * a.draft_stride : nullptr;
  const int nkids = drafts ? 0 : found.count;
  const int begin = blockIdx.x * a.chunk;
  const int end = min(begin + a.chunk, a.vocab);
  constexpr int N = Wide<T>::N;
  double rest = 0.0, full = 0.0;
  for (int i = begin + threadIdx.x * N; i < end; i += kThreads * N) {
    float p[N];
    double r[N];
    residual<T>(prow, qrow, kids, nkids, i, end, p, r);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      rest += r[k];
      full += (double)p[k];
    }
  }
  rest = wave_sum(rest);
  full = wave_sum(full);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    part[wave][0] = rest;
    part[wave][1] = full;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) s += part[i][threadIdx.x];
    a.sums[((int64_t)req * a.chunks + blockIdx.x) * 2 + threadIdx.x] = s;
  }
}

namespace {

// Inclusive sum over the workgroup's threads, in thread order.
__device__ __forceinline__ double scan(double v, double* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  double before = 0.0;
  for (int i = 0; i < wave; ++i) before += waves[i];
  return before + v;
}

}  // namespace

// Grid: requests.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(const VerifyArgs a) {
  __shared__ int64_t kids[kMaxDrafts];
  __shared__ Children found;
  __shared__ double waves[kThreads / 64];
  __shared__ double ends[kThreads];  // inclusive sums per chunk
  __shared__ int hit, tail;
  const int req = blockIdx.x;
  const int tid = threadIdx.x;
  const int first = a.starts[req];
  const int n = min(a.starts[req + 1] - first, kMaxDrafts);
  const int node = a.stops[req];
  const double u = uniform_at(a.sample_uniforms, req, a.uniforms_f64);
  const double* sums = a.sums + (int64_t)req * a.chunks * 2;
  const double rest = tid < a.chunks ? sums[2 * tid] : 0.0;
  const double full = tid < a.chunks ? sums[2 * tid + 1] : 0.0;
  if (tid == 0) {
    hit = kThreads;
    tail = -1;
  }
  list_children(a, first, n, node, kids, &found);
  const bool residual_left = __syncthreads_or(rest > 0.0);
  const double mine = residual_left ? rest : full;
  const double upto = scan(mine, waves);
  ends[tid] = upto;
  __syncthreads();
  const double goal = u * ends[kThreads - 1];
  if (upto > goal) atomicMin(&hit, tid);
  if (mine > 0.0) atomicMax(&tail, tid);
  __syncthreads();
  const int at = hit < kThreads ? hit : tail;  // (u >= 1: the last chunk that holds anything)
  if (at < 0) {
    if (tid == 0) a.out_tokens[req] = -1;
    return;
  }
  const double base = at > 0 ? ends[at - 1] : 0.0;
  __syncthreads();
  if (tid == 0) {
    hit = 0x7fffffff;
    tail = -1;
  }
  __syncthreads();
  // The chunk, N elements per thread and round, until the draw is reached.
  const T* drafts = static_cast<const T*>(a.draft_probs);
  const T* prow = static_cast<const T*>(a.target) + ((int64_t)first + req + node) * a.target_stride;
  const T* qrow =
      residual_left && drafts && found.draft >= 0 ? drafts + (int64_t)found.draft * a.draft_stride : nullptr;
  const int nkids = residual_left && !drafts ? found.count : 0;
  constexpr int N = Wide<T>::N;
  const int begin = at * a.chunk;
  const int end = min(begin + a.chunk, a.vocab);
  double done = base;
  for (int i0 = begin; i0 < end; i0 += kThreads * N) {
    const int i = i0 + tid * N;
    float p[N];
    double r[N];
    residual<T>(prow, qrow, kids, nkids, min(i, end), end, p, r);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < N; ++k) s += r[k];
    const double last = done + scan(s, waves);
    double c = last - s;
    // Sums over the elements again, from the thread's own start: the first
    // that passes the goal (the thread's end passes it too, to rounding).
    int mine_hit = 0x7fffffff, mine_tail = -1;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      c += r[k];
      if (r[k] > 0.0) {
        if (c > goal && mine_hit == 0x7fffffff) mine_hit = i + k;
        mine_tail = i + k;
      }
    }
    if (mine_hit != 0x7fffffff) atomicMin(&hit, mine_hit);
    if (mine_tail >= 0) atomicMax(&tail, mine_tail);
    __syncthreads();
    if (hit != 0x7fffffff) break;
    if (tid == kThreads - 1) ends[0] = last;
    __syncthreads();
    done = ends[0];
  }
  if (tid == 0) a.out_tokens[req] = hit != 0x7fffffff ? hit : tail;
}

}  // namespace lvamd

using namespace lvamd;

// Chunks of a row: about 2,048 workgroups over the batch, each with at least
// one 16-byte load per thread, at most kMaxChunks.
static int verify_chunks(int64_t requests, int32_t vocab, int32_t dtype) {
  const int64_t least = kThreads * (dtype == LVAMD_F32 ? 4 : 8);
  const int64_t most = (vocab + least - 1) / least;
  const int64_t want = requests > 0 ? (2048 + requests - 1) / requests : 1;
  const int64_t n = most < want ? most : want;
  return (int)(n < 1 ? 1 : n > kMaxChunks ? kMaxChunks : n);
}

extern "C" int64_t lvamd_verify_drafts_workspace_size(int64_t num_requests, int32_t vocab, int32_t dtype) {
  if (num_requests <= 0 || vocab <= 0) return 0;
  return num_requests * ((int64_t)verify_chunks(num_requests, vocab, dtype) * 16 + 4);
}

extern "C" int lvamd_verify_drafts(const void* target, int64_t target_row_stride, const void* draft_probs,
                                   int64_t draft_row_stride, int32_t vocab, int32_t dtype, const int32_t* draft_starts,
                                   const int64_t* draft_tokens, const int32_t* parents, const int32_t* siblings,
                                   int64_t num_requests, const void* node_uniforms, const void* sample_uniforms,
                                   int32_t uniforms_f64, int32_t* counts, int32_t* paths, int32_t path_width,
                                   int64_t* out_tokens, void* workspace, int64_t workspace_bytes,
                                   lvamd_stream_t stream) {
  if (dtype_size(dtype) == 0) return LVAMD_ERR_UNSUPPORTED;
  if (num_requests < 0 || num_requests > 65535 || vocab <= 0 || vocab > (1 << 30) || path_width < 1 ||
      target_row_stride < 0 || draft_row_stride < 0)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (num_requests == 0) return LVAMD_OK;
  if (!target || !draft_starts || !draft_tokens || !parents || !siblings || !node_uniforms || !sample_uniforms ||
      !counts || !paths || !out_tokens)
    return LVAMD_ERR_INVALID_ARGUMENT;
  if (!workspace || ((uintptr_t)workspace & 7u) != 0 ||
      workspace_bytes < lvamd_verify_drafts_workspace_size(num_requests, vocab, dtype))
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
  a.chunks = verify_chunks(num_requests, vocab, dtype);
  // (Whole 16-byte groups.)
  a.chunk = (((vocab + a.chunks - 1) / a.chunks) + 7) / 8 * 8;
  a.sums = static_cast<double*>(workspace);
  a.stops = reinterpret_cast<int32_t*>(a.sums + num_requests * a.chunks * 2);
  a.counts = counts;
  a.paths = paths;
  a.path_width = path_width;
  a.out_tokens = out_tokens;
  a.vocab = vocab;
  a.uniforms_f64 = uniforms_f64 != 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)a.chunks, (unsigned)num_requests), draw((unsigned)num_requests), threads(kThreads);
  switch (dtype) {
    case LVAMD_BF16: hipLaunchKernelGGL((verify_sums_kernel<__bf16>), grid, threads, 0, s, a); break;
    case LVAMD_F16: hipLaunchKernelGGL((verify_sums_kernel<_Float16>), grid, threads, 0, s, a); break;
    default: hipLaunchKernelGGL((verify_sums_kernel<float>), grid, threads, 0, s, a); break;
  }
  const int status = launch_status();
  if (status != LVAMD_OK) return status;
  switch (dtype) {
    case LVAMD_BF16: hipLaunchKernelGGL((verify_draw_kernel<__bf16>), draw, threads, 0, s, a); break;
    case LVAMD_F16: hipLaunchKernelGGL((verify_draw_kernel<_Float16>), draw, threads, 0, s, a); break;
    default: hipLaunchKernelGGL((verify_draw_kernel<float>), draw, threads, 0, s, a); break;
  }
  return launch_status();
}
