// Moves of cached states in place: the reorder of beams (tabby_states_reorder_async) and the
// acceptance of a drafted tree with its closing of the cache's gaps (tabby_tree_accept_async).
//
// A thread owns a column: the same W bytes of every row (or cache entry) that takes part, so
// what it overwrites is read by nobody else and no second buffer is needed. It first loads all
// rows that move, then stores them. W is the widest power of two that divides the layout (and,
// for many beams, keeps one value a beam in registers).
#include <math.h>

#include <algorithm>
#include <cmath>

#include "decode_internal.h"

namespace tabby {
namespace {

constexpr int kMaxStates = 256;  // pointers a launch carries as parameters
constexpr int kMoveThreads = 128;

struct StatePtrs {
  unsigned char *p[kMaxStates];
};

struct ReorderArgs {
  tabby_state_layout l;
  int32_t beams;
  const int32_t *parents, *lengths;
  int32_t vpe;     // columns an entry
  int32_t packed;  // a segment's entries lie end to end
  int64_t chunks;  // blocks a segment
};

template <int W> struct Vec;
template <> struct Vec<16> { typedef uint4 T; };
template <> struct Vec<8> { typedef uint2 T; };
template <> struct Vec<4> { typedef uint32_t T; };
template <> struct Vec<2> { typedef uint16_t T; };
template <> struct Vec<1> { typedef uint8_t T; };

// blockIdx.x = ((state * batch + b) * segments + g) * chunks + chunk. A thread takes U columns of
// a chunk, so that a row's part of it is U * 128 * W contiguous bytes and enough loads are on
// their way before the first store.
template <int W, int K, int U>
__global__ void __launch_bounds__(kMoveThreads) reorder_kernel(const __grid_constant__ ReorderArgs a,
                                                               const __grid_constant__ StatePtrs s,
                                                               int32_t batch) {
  typedef typename Vec<W>::T V;
  __shared__ int32_t from[K];
  int64_t u = blockIdx.x;
  const int64_t chunk = u % a.chunks;
  u /= a.chunks;
  const int g = (int)(u % a.l.segments);
  u /= a.l.segments;
  const int b = (int)(u % batch);
  const int state = (int)(u / batch);
  if (threadIdx.x < K) {
    int f = -1;
    if ((int)threadIdx.x < a.beams) {
      f = a.parents[(int64_t)b * a.beams + threadIdx.x];
      if (f < 0 || f >= a.beams || f == (int)threadIdx.x) f = -1;
    }
    from[threadIdx.x] = f;
  }
  const int64_t len =
      a.lengths ? min(max(a.lengths[b], 0), a.l.entries) : a.l.entries;
  __syncthreads();
  const int64_t base = chunk * (U * kMoveThreads);  // the block's first column of the segment
  const int64_t cols = len * a.vpe;
  if (base >= cols) return;
  unsigned char *p0 = s.p[state] + (int64_t)b * a.beams * a.l.row_stride + g * a.l.segment_stride;
  V v[U][K];
  unsigned char *p[U];
#pragma unroll
  for (int j = 0; j < U; j++) {
    const uint32_t i = j * kMoveThreads + threadIdx.x;
    p[j] = nullptr;
    if (base + i < cols) {
      if (a.packed) {
        p[j] = p0 + (base + i) * W;
      } else {
        const uint32_t local = (uint32_t)(base % a.vpe) + i;
        p[j] = p0 + (base / a.vpe + local / (uint32_t)a.vpe) * a.l.entry_stride +
               (int64_t)(local % (uint32_t)a.vpe) * W;
      }
    }
#pragma unroll
    for (int k = 0; k < K; k++)
      if (p[j] && from[k] >= 0) v[j][k] = *reinterpret_cast<const V *>(p[j] + from[k] * a.l.row_stride);
  }
#pragma unroll
  for (int j = 0; j < U; j++)
#pragma unroll
    for (int k = 0; k < K; k++)
      if (p[j] && from[k] >= 0) *reinterpret_cast<V *>(p[j] + k * a.l.row_stride) = v[j][k];
}

struct AcceptArgs {
  const int32_t *sampled;
  int64_t sampled_batch_stride, sampled_stride;
  const int32_t *tokens, *parents;
  int64_t parents_stride;
  int32_t batch, nodes;
  const int32_t *lengths;
  int32_t *path, *counts, *next_tokens, *next_lengths;
  tabby_state_layout l;
  int64_t entries;  // slots at or past this entry are unused
  int32_t n_caches;
  int32_t vpe;      // columns an entry; 0 without caches
  int64_t chunks;   // blocks a (cache, sequence)
  bool report;      // writes path, counts, next_tokens, next_lengths
};

// blockIdx.x = (cache * batch + b) * chunks + chunk. Every block walks its sequence's tree
// (a warp finds each step's slot by a ballot); the first block of a sequence writes the outcome.
template <int W>
__global__ void __launch_bounds__(kMoveThreads) accept_kernel(const __grid_constant__ AcceptArgs a,
                                                              const __grid_constant__ StatePtrs s) {
  typedef typename Vec<W>::T V;
  __shared__ int32_t parents[TABBY_TREE_MAX_NODES], tokens[TABBY_TREE_MAX_NODES];
  __shared__ int32_t sampled[TABBY_TREE_MAX_NODES], path[TABBY_TREE_MAX_NODES];
  __shared__ int32_t n_path;
  int64_t u = blockIdx.x;
  const int64_t chunk = u % a.chunks;
  u /= a.chunks;
  const int64_t b = u % a.batch;
  const int cache = (int)(u / a.batch);
  const int t = threadIdx.x;
  const int64_t start = a.lengths[b];
  if (t < a.nodes) {
    parents[t] = a.parents[b * a.parents_stride + t];
    tokens[t] = a.tokens[b * a.nodes + t];
    sampled[t] = a.sampled[b * a.sampled_batch_stride + t * a.sampled_stride];
  }
  __syncthreads();
  if (t < 32) {  // a warp, two slots a lane
    bool used[2];
    for (int h = 0; h < 2; h++) {
      const int j = t + 32 * h;
      used[h] = j < a.nodes && start >= 0 && start + j < a.entries && tree_sees(parents, j) != 0;
    }
    int n = 0, cur = 0;
    if (__shfl_sync(0xffffffffu, used[0], 0) && parents[0] == -1) {
      while (true) {
        if (t == 0) path[n] = cur;
        n++;
        const int want = sampled[cur];
        const unsigned lo =
            __ballot_sync(0xffffffffu, used[0] && parents[t] == cur && tokens[t] == want);
        const unsigned hi = __ballot_sync(
            0xffffffffu, used[1] && parents[t + 32] == cur && tokens[t + 32] == want);
        if (lo) cur = __ffs(lo) - 1;
        else if (hi) cur = 31 + __ffs(hi);
        else break;
      }
    }
    if (t == 0) n_path = n;
  }
  __syncthreads();
  const int n = n_path;
  if (a.report && cache == 0 && chunk == 0) {
    if (t < a.nodes) a.path[b * a.nodes + t] = t < n ? path[t] : -1;
    if (t == 0) {
      a.counts[b] = n;
      a.next_tokens[b] = n > 0 ? sampled[path[n - 1]] : -1;
      a.next_lengths[b] = (int32_t)(start + n);
    }
  }
  if (a.vpe == 0) return;
  const int64_t col = chunk * kMoveThreads + t;
  if (col >= (int64_t)a.l.segments * a.vpe) return;
  unsigned char *p = s.p[cache] + b * a.l.row_stride + (col / a.vpe) * a.l.segment_stride +
                     start * a.l.entry_stride + (col % a.vpe) * W;
  // path[r] >= r and the path rises, so no entry is overwritten before it is read; eight loads
  // are on their way at a time.
  for (int r0 = 1; r0 < n; r0 += 8) {
    V v[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (r0 + i < n && path[r0 + i] != r0 + i)
        v[i] = *reinterpret_cast<const V *>(p + path[r0 + i] * a.l.entry_stride);
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (r0 + i < n && path[r0 + i] != r0 + i)
        *reinterpret_cast<V *>(p + (r0 + i) * a.l.entry_stride) = v[i];
  }
}

// The widest power of two up to `most` that divides every address of the states.
int vector_bytes(const tabby_state_layout &l, void *const *states, int32_t n, int most) {
  uint64_t bits = (uint64_t)l.entry_bytes | (uint64_t)l.row_stride;
  if (l.segments > 1) bits |= (uint64_t)l.segment_stride;
  if (l.entries > 1) bits |= (uint64_t)l.entry_stride;
  for (int32_t i = 0; i < n; i++) bits |= reinterpret_cast<uintptr_t>(states[i]);
  int w = most;
  while (w > 1 && (bits & (uint64_t)(w - 1))) w >>= 1;
  return w;
}

// The same places as a layout with as few segments and as long entries as it allows.
tabby_state_layout merged(tabby_state_layout l) {
  if (l.segments > 1 && l.segment_stride == l.entry_bytes &&
      l.entry_bytes * l.segments < (int64_t)1 << 31 &&
      (l.entries == 1 || l.entry_stride >= l.entry_bytes * l.segments)) {  // [tokens][heads][dim]
    l.entry_bytes *= l.segments;
    l.segments = 1;
  }
  return l;
}

// Columns a thread, by the bytes of registers that it holds for each (4 at least a value).
constexpr int columns_of(int w, int k) {
  const int bytes = std::max(w, 4) * k;
  return bytes <= 64 ? 4 : bytes <= 128 ? 2 : 1;
}

template <int W, int K>
void reorder_launch(ReorderArgs a, const StatePtrs &s, int32_t n, int32_t batch, cudaStream_t q) {
  constexpr int kColumns = columns_of(W, K) * kMoveThreads;
  a.chunks = ((int64_t)a.l.entries * a.vpe + kColumns - 1) / kColumns;
  const unsigned grid = (unsigned)((int64_t)n * batch * a.l.segments * a.chunks);
  reorder_kernel<W, K, columns_of(W, K)><<<grid, kMoveThreads, 0, q>>>(a, s, batch);
}

template <int W>
void reorder_launch_beams(const ReorderArgs &a, const StatePtrs &s, int32_t n, int32_t batch,
                          cudaStream_t q) {
  if (a.beams <= 4) return reorder_launch<W, 4>(a, s, n, batch, q);
  if (a.beams <= 8) return reorder_launch<W, 8>(a, s, n, batch, q);
  if (a.beams <= 16) return reorder_launch<W, 16>(a, s, n, batch, q);
  if constexpr (W <= 8) {
    if (a.beams <= 32) return reorder_launch<W, 32>(a, s, n, batch, q);
  }
  if constexpr (W <= 4) reorder_launch<W, 64>(a, s, n, batch, q);
}

}  // namespace
}  // namespace tabby

extern "C" {

int tabby_states_reorder_async(int32_t device, void *const *h_states, int32_t n_states,
                               const tabby_state_layout *layout, int32_t batch, int32_t beams,
                               const int32_t *d_parents, const int32_t *d_lengths,
                               void *stream) {
  using namespace tabby;
  if (n_states < 0 || batch < 0)
    return decode_fail(TABBY_EINVAL, "states_reorder: n_states and batch must be >= 0");
  if (beams < 1 || beams > TABBY_BEAM_MAX)
    return decode_fail(TABBY_EINVAL, "states_reorder: beams must be in [1, %d], got %d",
                       TABBY_BEAM_MAX, beams);
  const int st = check_layout("states_reorder", layout, (int64_t)batch * beams);
  if (st) return st;
  ReorderArgs a;
  a.l = merged(*layout);
  // By the layout alone, whatever the pointers allow: a call without states tells whether one with
  // states of this layout is refused. (Columns of a byte; wider ones are fewer.)
  const double blocks = (double)batch * a.l.segments *
                        std::ceil((double)a.l.entries * a.l.entry_bytes / kMoveThreads);
  if (blocks > 2147483647.0)
    return decode_fail(TABBY_EINVAL, "states_reorder: a state is too large for one launch");
  if (n_states == 0 || batch == 0) return TABBY_OK;
  if (!h_states || !d_parents)
    return decode_fail(TABBY_EINVAL, "states_reorder: states and parents must not be NULL");
  for (int32_t i = 0; i < n_states; i++)
    if (!h_states[i]) return decode_fail(TABBY_EINVAL, "states_reorder: state %d is NULL", i);
  const int w = vector_bytes(a.l, h_states, n_states, beams <= 16 ? 16 : beams <= 32 ? 8 : 4);
  a.beams = beams;
  a.parents = d_parents;
  a.lengths = d_lengths;
  a.vpe = (int32_t)(a.l.entry_bytes / w);
  a.packed = a.l.entries == 1 || a.l.entry_stride == a.l.entry_bytes;
  const int32_t most =
      (int32_t)std::min<double>(kMaxStates, std::max(1.0, 2147483647.0 / blocks));
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return decode_cuda_fail(scope.err, "cudaSetDevice");
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  for (int32_t s0 = 0; s0 < n_states; s0 += most) {
    const int32_t n = std::min(n_states - s0, most);
    StatePtrs s;
    for (int32_t i = 0; i < n; i++) s.p[i] = static_cast<unsigned char *>(h_states[s0 + i]);
    switch (w) {
      case 16: reorder_launch_beams<16>(a, s, n, batch, q); break;
      case 8: reorder_launch_beams<8>(a, s, n, batch, q); break;
      case 4: reorder_launch_beams<4>(a, s, n, batch, q); break;
      case 2: reorder_launch_beams<2>(a, s, n, batch, q); break;
      default: reorder_launch_beams<1>(a, s, n, batch, q); break;
    }
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return decode_cuda_fail(err, "reorder_kernel launch");
  }
  return TABBY_OK;
}

int tabby_tree_accept_async(int32_t device, const int32_t *d_sampled,
                            int64_t sampled_batch_stride, int64_t sampled_stride,
                            const int32_t *d_tokens, const int32_t *d_parents,
                            int64_t parents_stride, int32_t batch, int32_t nodes,
                            const int32_t *d_lengths, int32_t *d_path, int32_t *d_counts,
                            int32_t *d_next_tokens, int32_t *d_next_lengths,
                            void *const *h_caches, int32_t n_caches,
                            const tabby_state_layout *layout, void *stream) {
  using namespace tabby;
  if (batch < 0 || n_caches < 0)
    return decode_fail(TABBY_EINVAL, "tree_accept: batch and n_caches must be >= 0");
  if (nodes < 1 || nodes > TABBY_TREE_MAX_NODES)
    return decode_fail(TABBY_EINVAL, "tree_accept: nodes must be in [1, %d], got %d",
                       TABBY_TREE_MAX_NODES, nodes);
  if (sampled_batch_stride < 0 || sampled_stride < 0 || parents_stride < 0)
    return decode_fail(TABBY_EINVAL, "tree_accept: strides must be >= 0");
  if (n_caches > 0) {
    const int st = check_layout("tree_accept", layout, batch);
    if (st) return st;
  }
  if (batch == 0) return TABBY_OK;
  if (!d_sampled || !d_tokens || !d_parents || !d_lengths || !d_path || !d_counts ||
      !d_next_tokens || !d_next_lengths || (n_caches > 0 && !h_caches))
    return decode_fail(TABBY_EINVAL, "tree_accept: a required pointer is NULL");
  for (int32_t i = 0; i < n_caches; i++)
    if (!h_caches[i]) return decode_fail(TABBY_EINVAL, "tree_accept: cache %d is NULL", i);
  AcceptArgs a = {};
  a.sampled = d_sampled;
  a.sampled_batch_stride = sampled_batch_stride;
  a.sampled_stride = sampled_stride;
  a.tokens = d_tokens;
  a.parents = d_parents;
  a.parents_stride = parents_stride;
  a.batch = batch;
  a.nodes = nodes;
  a.lengths = d_lengths;
  a.path = d_path;
  a.counts = d_counts;
  a.next_tokens = d_next_tokens;
  a.next_lengths = d_next_lengths;
  a.entries = INT64_MAX;
  a.chunks = 1;
  int w = 1;
  if (n_caches > 0) {
    a.l = merged(*layout);
    w = vector_bytes(a.l, h_caches, n_caches, 16);
    a.entries = a.l.entries;
    a.vpe = (int32_t)(a.l.entry_bytes / w);
    a.chunks = ((int64_t)a.l.segments * a.vpe + kMoveThreads - 1) / kMoveThreads;
  }
  const double blocks = (double)batch * (double)a.chunks;
  if (blocks > 2147483647.0)
    return decode_fail(TABBY_EINVAL, "tree_accept: a cache is too large for one launch");
  const int32_t most =
      (int32_t)std::min<double>(kMaxStates, std::max(1.0, 2147483647.0 / blocks));
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return decode_cuda_fail(scope.err, "cudaSetDevice");
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  for (int32_t c0 = 0; c0 < std::max(n_caches, 1); c0 += most) {
    a.n_caches = std::min(n_caches - c0, most);
    a.report = c0 == 0;
    StatePtrs s;
    for (int32_t i = 0; i < a.n_caches; i++)
      s.p[i] = static_cast<unsigned char *>(h_caches[c0 + i]);
    const unsigned grid = (unsigned)((int64_t)std::max(a.n_caches, 1) * batch * a.chunks);
    switch (w) {
      case 16: accept_kernel<16><<<grid, kMoveThreads, 0, q>>>(a, s); break;
      case 8: accept_kernel<8><<<grid, kMoveThreads, 0, q>>>(a, s); break;
      case 4: accept_kernel<4><<<grid, kMoveThreads, 0, q>>>(a, s); break;
      case 2: accept_kernel<2><<<grid, kMoveThreads, 0, q>>>(a, s); break;
      default: accept_kernel<1><<<grid, kMoveThreads, 0, q>>>(a, s); break;
    }
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return decode_cuda_fail(err, "accept_kernel launch");
  }
  return TABBY_OK;
}

}  // extern "C"
