// Beam search's selection (tabby_beam_step_async): log-softmax of every live beam's logits,
// the n_out best continuations of a prompt over beams and vocabulary.
//
//   lse(i) = max + log(sum exp(x - max)),  key(i, v) = score(i) + (x - lse(i)) in 64 bits
//
// beam_row_kernel: one CTA a row; maximum, sum, then the row's n best logits one after the
// other, each a pass over the row (the best one behind the last in the order value falling,
// index rising). beam_pick_kernel: one CTA a prompt merges its rows' lists the same way.
#include <math.h>

#include "decode_internal.h"

namespace tabby {
namespace {

constexpr int kThreads = 256;

struct BeamArgs {
  const void *logits;
  int64_t batch_stride, beam_stride;
  int32_t batch, beams, vocab;
  const float *scores;
  const uint8_t *finished;
  int32_t eos, n_out;
  float *next_scores;
  int32_t *parents, *tokens;
  uint8_t *next_finished;
  int32_t *status;
  double *lse;     // [rows]; NaN: bad input
  float *values;   // [rows][n_out] best logits, falling
  int32_t *ids;    // [rows][n_out]; -1 behind the last
};

// (a, i) stands before (b, j): the larger value, then the lower index.
template <typename T>
__device__ __forceinline__ bool before(T a, int64_t i, T b, int64_t j) {
  return a > b || (a == b && i < j);
}

// The first of all threads' (v, id); id < 0 stands behind every other.
template <typename T>
__device__ void block_first(T &v, int64_t &id, T *sv, int64_t *si) {
  const int t = threadIdx.x;
  __syncthreads();
  sv[t] = v;
  si[t] = id;
  __syncthreads();
  for (int o = kThreads / 2; o > 0; o >>= 1) {
    if (t < o && si[t + o] >= 0 && (si[t] < 0 || before(sv[t + o], si[t + o], sv[t], si[t]))) {
      sv[t] = sv[t + o];
      si[t] = si[t + o];
    }
    __syncthreads();
  }
  v = sv[0];
  id = si[0];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) beam_row_kernel(BeamArgs a) {
  __shared__ double sd[kThreads];
  __shared__ float sv[kThreads];
  __shared__ int64_t si[kThreads];
  const int row = blockIdx.x, t = threadIdx.x;
  const int b = row / a.beams, i = row % a.beams;
  const float score = a.scores[row];
  const bool skip = score == -INFINITY || (a.finished && a.finished[row]);
  const T *x = static_cast<const T *>(a.logits) + b * a.batch_stride + i * a.beam_stride;
  float *values = a.values + (int64_t)row * a.n_out;
  int32_t *ids = a.ids + (int64_t)row * a.n_out;
  if (skip) {
    for (int j = t; j < a.n_out; j += kThreads) ids[j] = -1;
    if (t == 0) a.lse[row] = 0;
    return;
  }
  float m = -INFINITY;
  bool bad = false;
  for (int v = t; v < a.vocab; v += kThreads) {
    const float f = to_f32(x[v]);
    bad |= !(f < INFINITY);
    m = fmaxf(m, f);
  }
  bad = __syncthreads_or(bad);
  int64_t id = t;
  block_first(m, id, sv, si);
  double s = 0;
  if (m > -INFINITY)
    for (int v = t; v < a.vocab; v += kThreads) s += exp((double)to_f32(x[v]) - (double)m);
  sd[t] = s;
  __syncthreads();
  for (int o = kThreads / 2; o > 0; o >>= 1) {
    if (t < o) sd[t] += sd[t + o];
    __syncthreads();
  }
  if (t == 0) a.lse[row] = bad ? (double)NAN : (double)m + log(sd[0]);
  float pv = INFINITY;
  int64_t pi = -1;
  for (int j = 0; j < a.n_out; j++) {
    float best = -INFINITY;
    int64_t at = -1;
    if (!bad && pi < INT32_MAX) {
      for (int v = t; v < a.vocab; v += kThreads) {
        const float f = to_f32(x[v]);
        if (f > -INFINITY && before(pv, pi, f, (int64_t)v) &&
            (at < 0 || before(f, (int64_t)v, best, at))) {
          best = f;
          at = v;
        }
      }
    }
    block_first(best, at, sv, si);
    if (t == 0) {
      values[j] = best;
      ids[j] = (int32_t)at;
    }
    pv = best;
    pi = at < 0 ? INT32_MAX : at;
  }
}

__global__ void __launch_bounds__(kThreads) beam_pick_kernel(BeamArgs a) {
  __shared__ double sv[kThreads];
  __shared__ int64_t si[kThreads];
  const int b = blockIdx.x, t = threadIdx.x;
  const int64_t row0 = (int64_t)b * a.beams;
  bool bad = false;
  for (int i = t; i < a.beams; i += kThreads) {
    const float s = a.scores[row0 + i];
    bad |= !(s < INFINITY) || isnan(a.lse[row0 + i]);
  }
  bad = __syncthreads_or(bad);
  double pv = INFINITY;
  int64_t pi = -1;
  bool none = bad;
  for (int j = 0; j < a.n_out; j++) {
    double best = -INFINITY;
    int64_t at = -1;
    if (!none) {
      for (int c = t; c < a.beams * a.n_out; c += kThreads) {
        const int i = c / a.n_out, e = c % a.n_out;
        const int64_t row = row0 + i;
        const float score = a.scores[row];
        if (score == -INFINITY) continue;
        double key;
        int64_t id;
        if (a.finished && a.finished[row]) {
          if (e != 0) continue;
          key = score;
          id = (int64_t)i * a.vocab + a.eos;
        } else {
          const int32_t v = a.ids[row * a.n_out + e];
          if (v < 0) continue;
          key = (double)score + ((double)a.values[row * a.n_out + e] - a.lse[row]);
          id = (int64_t)i * a.vocab + v;
        }
        if (before(pv, pi, key, id) && (at < 0 || before(key, id, best, at))) {
          best = key;
          at = id;
        }
      }
    }
    block_first(best, at, sv, si);
    none |= at < 0;
    if (t == 0) {
      const int64_t o = (int64_t)b * a.n_out + j;
      const int32_t parent = none ? -1 : (int32_t)(at / a.vocab);
      const int32_t token = none ? -1 : (int32_t)(at % a.vocab);
      a.next_scores[o] = none ? -INFINITY : (float)best;
      a.parents[o] = parent;
      a.tokens[o] = token;
      if (a.next_finished)
        a.next_finished[o] =
            none || token == a.eos || (a.finished && a.finished[row0 + parent]) ? 1 : 0;
    }
    pv = best;
    pi = at;
  }
  if (t == 0) a.status[b] = bad ? TABBY_EINPUT : TABBY_OK;
}

int check_sizes(int32_t batch, int32_t beams, int32_t vocab, int32_t n_out) {
  if (batch < 0) return decode_fail(TABBY_EINVAL, "beam_step: batch must be >= 0");
  if (beams < 1 || beams > TABBY_BEAM_MAX)
    return decode_fail(TABBY_EINVAL, "beam_step: beams must be in [1, %d], got %d",
                       TABBY_BEAM_MAX, beams);
  if (vocab < 1 || vocab > (1 << 30))
    return decode_fail(TABBY_EINVAL, "beam_step: vocab must be in [1, 2^30], got %d", vocab);
  if (n_out < 1 || n_out > TABBY_BEAM_MAX_OUT)
    return decode_fail(TABBY_EINVAL, "beam_step: n_out must be in [1, %d], got %d",
                       TABBY_BEAM_MAX_OUT, n_out);
  if ((int64_t)batch * beams > (1 << 22))
    return decode_fail(TABBY_EINVAL, "beam_step: batch * beams must be at most 2^22");
  return TABBY_OK;
}

}  // namespace
}  // namespace tabby

extern "C" {

int tabby_beam_workspace_bytes(int32_t batch, int32_t beams, int32_t vocab, int32_t n_out,
                               size_t *bytes) {
  using namespace tabby;
  const int st = check_sizes(batch, beams, vocab, n_out);
  if (st) return st;
  if (!bytes) return decode_fail(TABBY_EINVAL, "beam_step: bytes is NULL");
  const size_t rows = (size_t)batch * beams;
  *bytes = rows * 8 + rows * n_out * 8;
  return TABBY_OK;
}

int tabby_beam_step_async(int32_t device, const void *d_logits, int32_t dtype,
                          int64_t batch_stride, int64_t beam_stride, int32_t batch,
                          int32_t beams, int32_t vocab, const float *d_scores,
                          const uint8_t *d_finished, int32_t eos_id, int32_t n_out,
                          float *d_next_scores, int32_t *d_parents, int32_t *d_tokens,
                          uint8_t *d_next_finished, int32_t *d_status, void *d_workspace,
                          size_t workspace_bytes, void *stream) {
  using namespace tabby;
  size_t need = 0;
  const int st = tabby_beam_workspace_bytes(batch, beams, vocab, n_out, &need);
  if (st) return st;
  if (dtype != TABBY_F32 && dtype != TABBY_BF16 && dtype != TABBY_F16)
    return decode_fail(TABBY_EINVAL, "beam_step: unknown dtype %d", dtype);
  if (eos_id < -1 || eos_id >= vocab)
    return decode_fail(TABBY_EINVAL, "beam_step: eos_id must be in [-1, vocab), got %d", eos_id);
  if (d_finished && eos_id < 0)
    return decode_fail(TABBY_EINVAL, "beam_step: finished beams need an eos_id");
  if (batch_stride < 0 || beam_stride < 0)
    return decode_fail(TABBY_EINVAL, "beam_step: strides must be >= 0");
  if (batch == 0) return TABBY_OK;
  if (!d_logits || !d_scores || !d_next_scores || !d_parents || !d_tokens || !d_status)
    return decode_fail(TABBY_EINVAL, "beam_step: a required pointer is NULL");
  if (!aligned_to(d_logits, dtype == TABBY_F32 ? 4 : 2))
    return decode_fail(TABBY_EINVAL, "beam_step: logits must be aligned to their type");
  if (!d_workspace || workspace_bytes < need || !aligned_to(d_workspace, 16))
    return decode_fail(TABBY_EINVAL,
                       "beam_step: needs a 16-byte aligned workspace of %zu bytes, got %zu", need,
                       d_workspace ? workspace_bytes : (size_t)0);
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return decode_cuda_fail(scope.err, "cudaSetDevice");
  BeamArgs a;
  a.logits = d_logits;
  a.batch_stride = batch_stride;
  a.beam_stride = beam_stride;
  a.batch = batch;
  a.beams = beams;
  a.vocab = vocab;
  a.scores = d_scores;
  a.finished = d_finished;
  a.eos = eos_id;
  a.n_out = n_out;
  a.next_scores = d_next_scores;
  a.parents = d_parents;
  a.tokens = d_tokens;
  a.next_finished = d_next_finished;
  a.status = d_status;
  const size_t rows = (size_t)batch * beams;
  a.lse = static_cast<double *>(d_workspace);
  a.values = reinterpret_cast<float *>(a.lse + rows);
  a.ids = reinterpret_cast<int32_t *>(a.values + rows * n_out);
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  if (dtype == TABBY_F32)
    beam_row_kernel<float><<<(unsigned)rows, kThreads, 0, q>>>(a);
  else if (dtype == TABBY_BF16)
    beam_row_kernel<__nv_bfloat16><<<(unsigned)rows, kThreads, 0, q>>>(a);
  else
    beam_row_kernel<__half><<<(unsigned)rows, kThreads, 0, q>>>(a);
  beam_pick_kernel<<<(unsigned)batch, kThreads, 0, q>>>(a);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return decode_cuda_fail(err, "beam_step launch");
  return TABBY_OK;
}

}  // extern "C"
