// Beam search's selection (tabby_beam_step_async): log-softmax of every live beam's logits,
// the n_out best continuations of a prompt over beams and vocabulary.
//
//   lse(i) = max + log(sum exp(x - max)),  key(i, v) = score(i) + (x - lse(i)) in 64 bits
//
//   beam_scan_kernel  reads every logit once. A CTA of 128 threads takes a chunk of a row (6144
//                     logits, or 2048 where there are few rows) into registers, all loads at
//                     once; the chunk's maximum, its sum of exponentials and the logits that
//                     can be among its n_out best are found from there. A bound on the n_out-th
//                     best: of the 4 warps' thread maxima the ceil(n_out / 4) best each are at
//                     least n_out logits, so all that matters is no smaller than the least of
//                     them. Where more logits than a list holds pass it (ties, or warps without
//                     logits) the exact n_out-th best is found by bisection over the values.
//   beam_pick_kernel  a CTA a prompt: the beams' log-sum-exps from the chunks' statistics, the
//                     keys of the listed logits, the n_out best of them.
//
// The sums of a chunk are in fp32, so a lse is off by up to gap / 2 (gap_of below), and keys of
// different beams that are closer than the gap might be out of order. Such pairs are rare; where
// the sorted result has one, the lse of the beams in it is computed again in 64 bits from all
// their logits (the rows are read once more, by a cluster of CTAs) and the listed keys are sorted
// again.
#include <math.h>

#include <algorithm>

#include "decode_internal.h"
#include "sm100.cuh"

namespace tabby {
namespace {

constexpr int kScanThreads = 128;
constexpr int kScanWarps = kScanThreads / 32;
constexpr int kMaxHelpers = 8;
constexpr int kPickCap = 1024;  // keys a prompt's selection may keep

struct ChunkStats {
  double sum;  // of exp(x - max)
  float max;   // -inf: no logit; NaN: bad input
  float floor; // n_out logits of the chunk are no smaller (-inf: there may be fewer)
  int32_t count;
};
// More keys than this are worth a tighter bound (12 x 5 beams, first steps among them: 15.5 us a
// step with 256, 15.4 with 128, 16.5 with 64; 4 x 32 beams: 23.9, 23.7 and 31.9; over 16 inputs).
constexpr int kPickTight = 128;

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
  int32_t helpers;    // CTAs a prompt of the pick: a cluster
  int32_t chunks;     // a row
  int32_t cap;        // entries of a chunk's list
  double gap;
  ChunkStats *stats;  // [rows][chunks]
  float2 *lists;      // [rows][chunks][cap]: logit, token (bits)
};

// A row's terms exp(x - max) are each off by at most (2.25 |x - max| + 4) u relative (u = 2^-24:
// the difference, its product with log2(e), the constant; ex2's 4 u); weighted by the
// probabilities |x - max| averages to at most ln(vocab). Their fp32 sums add 13 u (runs of 6, 3
// sums of those, 5 steps of a warp's tree). Two lse's differ by twice that.
double gap_of(int32_t vocab) {
  return 2.0 * (2.25 * log((double)std::max(vocab, 2)) + 17.0) * 5.9604644775390625e-8;
}

template <typename T> struct Vec16;  // the values of 16 bytes
template <> struct Vec16<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void get(uint4 v, float *x) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
};
template <> struct Vec16<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void get(uint4 v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Vec16<__half> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void get(uint4 v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};

// Logits are read once: past L1.
__device__ __forceinline__ uint4 load_once(const void *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
// Order-preserving key with -0 folded onto +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = x == 0.f ? 0u : __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ const T *row_of(const BeamArgs &a, int row) {
  return static_cast<const T *>(a.logits) + (row / a.beams) * a.batch_stride +
         (row % a.beams) * a.beam_stride;
}
// 16-byte pieces of a row: piece v holds the elements v * kN - lead + 0 .. kN - 1 of it.
template <typename T>
__device__ __forceinline__ int lead_of(const T *x) {
  return (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
}

// The k best of the n logits in `x` (shared memory, in the order of their indexes, the first of
// which is e0; at least k above -inf), ties to the lower index, in any order into `list`. The k-th
// best value is found by bisection over the keys, bit by bit; then all above it are taken and, of
// those equal to it, the first ones. All threads of the block call; returns k.
__device__ __noinline__ int exact_list(const float *x, int n, int e0, int k, float2 *list) {
  __shared__ int s_warp[kScanWarps], s_taken;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t kstar = 0;
  for (int bit = 31; bit >= 0; bit--) {
    const uint32_t probe = kstar | 1u << bit;
    __syncthreads();
    int c = 0;
    for (int i = tid; i < n; i += kScanThreads) c += order_key(x[i]) >= probe ? 1 : 0;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) s_warp[warp] = c;
    __syncthreads();
    c = 0;
    for (int w = 0; w < kScanWarps; w++) c += s_warp[w];
    if (c >= k) kstar = probe;
  }
  if (tid == 0) s_taken = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kScanThreads)
    if (order_key(x[i]) > kstar) list[atomicAdd(&s_taken, 1)] = make_float2(x[i], __int_as_float(e0 + i));
  __syncthreads();
  int taken = s_taken;  // below k
  for (int i0 = 0; i0 < n && taken < k; i0 += kScanThreads) {
    const bool eq = i0 + tid < n && order_key(x[i0 + tid]) == kstar;
    const unsigned m = __ballot_sync(0xffffffffu, eq);
    __syncthreads();
    if (lane == 0) s_warp[warp] = __popc(m);
    __syncthreads();
    int at = taken + __popc(m & ((1u << lane) - 1u)), all = 0;
    for (int w = 0; w < kScanWarps; w++) {
      if (w < warp) at += s_warp[w];
      all += s_warp[w];
    }
    if (eq && at < k) list[at] = make_float2(x[i0 + tid], __int_as_float(e0 + i0 + tid));
    taken = min(k, taken + all);
  }
  return k;
}

// NV pieces a thread: NV * kN logits in registers.
template <typename T, int NV>
__global__ void __launch_bounds__(kScanThreads, 7) beam_scan_kernel(const __grid_constant__ BeamArgs a) {
  constexpr int kN = Vec16<T>::kN, kE = NV * kN;
  __shared__ float s_max[kScanWarps], s_sum[kScanWarps];
  __shared__ uint32_t s_bound[kScanWarps];
  __shared__ int s_count;
  __shared__ float s_x[kE * kScanThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  ChunkStats *stats = a.stats + blockIdx.x;
  float2 *list = a.lists + (int64_t)blockIdx.x * a.cap;
  const float score = a.scores[row];
  if (score == -INFINITY || (a.finished && a.finished[row])) {
    if (tid == 0) *stats = {0.0, -INFINITY, -INFINITY, 0};
    return;
  }
  const T *x0 = row_of<T>(a, row);
  const int lead = lead_of(x0);
  const T *base = x0 - lead;
  const int pieces = (lead + a.vocab + kN - 1) / kN;
  const int even = pieces / a.chunks, more = pieces - even * a.chunks;
  const int v0 = chunk * even + min(chunk, more), v1 = v0 + even + (chunk < more ? 1 : 0);
  float x[kE];
  if ((int64_t)v0 * kN >= lead && (int64_t)v1 * kN - lead <= a.vocab) {  // whole pieces only
    const T *p = base + (int64_t)(v0 + tid) * kN;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      if (j * kScanThreads + tid < v1 - v0) {
        Vec16<T>::get(load_once(p + j * kScanThreads * kN), x + j * kN);
      } else {
#pragma unroll
        for (int i = 0; i < kN; i++) x[j * kN + i] = -INFINITY;
      }
    }
  } else {  // a row's ragged ends
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int v = v0 + j * kScanThreads + tid;
      const int64_t e = (int64_t)v * kN - lead;  // the piece's first element
#pragma unroll
      for (int i = 0; i < kN; i++)
        x[j * kN + i] =
            v < v1 && e + i >= 0 && e + i < a.vocab ? to_f32(x0[e + i]) : -INFINITY;
    }
  }
  float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int i = 4; i < kE - 4; i += 8)
#pragma unroll
    for (int k = 0; k < 4; k++) mx[k] = max3_nan(mx[k], x[i + 2 * k], x[i + 2 * k + 1]);
  const float top =
      max3_nan(max3_nan(mx[0], mx[1], x[kE - 4]), max3_nan(mx[2], mx[3], x[kE - 3]),
               max3_nan(x[kE - 2], x[kE - 1], x[0]));
  const bool bad = !(top < INFINITY);
  // The warp's maximum and its ceil(n_out / 4)-th best thread maximum.
  const uint32_t key = bad ? 0u : order_key(top);
  uint32_t rest = key, kth = 0;
  const uint32_t best = __reduce_max_sync(0xffffffffu, key);
  for (int left = (a.n_out + kScanWarps - 1) / kScanWarps; left > 0;) {
    kth = __reduce_max_sync(0xffffffffu, rest);
    const unsigned eq = __ballot_sync(0xffffffffu, rest == kth);
    left -= __popc(eq);
    if (rest == kth) rest = 0;
    if (kth == 0) break;
  }
  const float wmax = best ? key_value(best) : -INFINITY;
  // The sum relative to the warp's maximum.
  float2 sum[4] = {};
  if (wmax > -INFINITY) {
    constexpr float kLog2e = 1.4426950408889634f;
    const float2 m2 = make_float2(-wmax, -wmax), l2 = make_float2(kLog2e, kLog2e);
#pragma unroll
    for (int i = 0; i < kE; i += 2) {
      const float2 t = mul2(add2(make_float2(x[i], x[i + 1]), m2), l2);
      sum[(i >> 1) & 3] = add2(sum[(i >> 1) & 3], make_float2(ex2_fast(t.x), ex2_fast(t.y)));
    }
  }
  const float2 sums = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
  float total = sums.x + sums.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) {
    s_max[warp] = wmax;
    s_sum[warp] = total;
    s_bound[warp] = kth;
  }
  if (tid == 0) s_count = 0;
  const bool any_bad = __syncthreads_or(bad);
  if (any_bad) {
    if (tid == 0) *stats = {0.0, NAN, -INFINITY, 0};
    return;
  }
  uint32_t bound = s_bound[0];
  float cmax = s_max[0];
#pragma unroll
  for (int w = 1; w < kScanWarps; w++) {
    bound = min(bound, s_bound[w]);
    cmax = fmaxf(cmax, s_max[w]);
  }
  if (cmax == -INFINITY) {
    if (tid == 0) *stats = {0.0, -INFINITY, -INFINITY, 0};
    return;
  }
  // Candidates: no smaller than the bound, above -inf.
  const float least = bound <= order_key(-INFINITY) ? -3.402823466e38f : key_value(bound);
  if (top >= least) {
    unsigned long long pass = 0;
#pragma unroll
    for (int i = 0; i < kE; i++) pass |= x[i] >= least ? 1ull << i : 0ull;
    int at = atomicAdd(&s_count, __popcll(pass));
    for (; pass; pass &= pass - 1, at++) {
      const int i = __ffsll(pass) - 1;
      const int e = (v0 + i / kN * kScanThreads + tid) * kN - lead + i % kN;
      if (at < a.cap) list[at] = make_float2(to_f32(x0[e]), __int_as_float(e));
    }
  }
  __syncthreads();
  int count = s_count;
  if (count > a.cap) {  // block-uniform
#pragma unroll
    for (int i = 0; i < kE; i++)
      s_x[((i / kN) * kScanThreads + tid) * kN + i % kN] = x[i];
    count = exact_list(s_x, kE * kScanThreads, v0 * kN - lead, a.n_out, list);
  }
  if (warp == 0) {
    double t = 0;
    if (lane < kScanWarps && s_max[lane] > -INFINITY)
      t = (double)s_sum[lane] * exp((double)s_max[lane] - (double)cmax);
    t = warp_sum(t);
    if (lane == 0)
      *stats = {t, cmax, bound > order_key(-INFINITY) ? key_value(bound) : -INFINITY, count};
  }
}

// A candidate: its key, its place (beam, then token), its logit.
struct Cand {
  double key;
  float x;
  int32_t beam, token;
};
// The larger key, then the lower beam; within a beam the larger logit (different ones can round
// to the same key), then the lower token. (Within a beam keys rise with the logits.)
__device__ __forceinline__ bool stands_before(const Cand &p, const Cand &q) {
  if (p.key != q.key) return p.key > q.key;
  if (p.beam != q.beam) return p.beam < q.beam;
  return p.x > q.x || (p.x == q.x && p.token < q.token);
}
// Order-preserving integer of a key (-0 folded onto +0), and back.
__device__ __forceinline__ int64_t key_bits(double k) {
  const int64_t b = __double_as_longlong(k + 0.0);
  return b ^ (int64_t)((uint64_t)(b >> 63) >> 1);
}
__device__ __forceinline__ double bits_key(int64_t b) {
  return __longlong_as_double(b ^ (int64_t)((uint64_t)(b >> 63) >> 1));
}
// A prompt's candidates in shared memory, as integers that order them: the larger key, then the
// smaller tie (beam, then falling logit), then the lower token.
struct CandTable {
  int64_t key[kPickCap];
  uint64_t tie[kPickCap];
  int32_t token[kPickCap];
  __device__ __forceinline__ void put(int i, const Cand &c) {
    key[i] = key_bits(c.key);
    tie[i] = (uint64_t)c.beam << 32 | (uint32_t)~order_key(c.x);
    token[i] = c.token;
  }
  __device__ __forceinline__ Cand get(int i) const {
    Cand c;
    c.key = bits_key(key[i]);
    c.x = key_value(~(uint32_t)tie[i]);
    c.beam = (int32_t)(tie[i] >> 32);
    c.token = token[i];
    return c;
  }
};

// (Aligned, like the wait: the warp has to be converged, whatever branch stood before.)
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of a shared variable's copy in a CTA of the cluster.
__device__ __forceinline__ uint32_t in_cta(const void *p, int cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
  return r;
}
__device__ __forceinline__ uint32_t in_first_cta(const void *p) { return in_cta(p, 0); }
__device__ __forceinline__ uint32_t load_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

// exp(d) for d <= 0 in 64 bits: 2^n 2^f with n the nearest integer to d log2(e) and 2^f by its
// Taylor polynomial of degree 10 on [-1/2, 1/2] (off by less than 3e-13); 0 below 2^-1000.
__device__ __forceinline__ double exp_below(double d) {
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const double t = d * 1.4426950408889634;
  if (!(t > -1000.0)) return 0.0;
  const double r = t + kRound, f = t - (r - kRound);
  double p = 7.0549116208011209e-09;
  p = fma(p, f, 1.0178086009239696e-07);
  p = fma(p, f, 1.3215486790144305e-06);
  p = fma(p, f, 1.5252733804059838e-05);
  p = fma(p, f, 0.00015403530393381606);
  p = fma(p, f, 0.0013333558146428441);
  p = fma(p, f, 0.0096181291076284769);
  p = fma(p, f, 0.055504108664821576);
  p = fma(p, f, 0.24022650695910069);
  p = fma(p, f, 0.69314718055994529);
  p = fma(p, f, 1);
  return __longlong_as_double(__double_as_longlong(p) + (__double_as_longlong(r) << 52));
}
// A CTA's share of sum exp(x - m) over the logits of row `row`, in 64 bits, to `to` (in the
// cluster's first CTA).
template <typename T, int kThreads>
__device__ __noinline__ void share_sum(const BeamArgs &a, int row, float m, int helper,
                                       double *s_warp, uint32_t to) {
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T *x = row_of<T>(a, row);
  const int n = (a.vocab + a.helpers - 1) / a.helpers, end = min(a.vocab, (helper + 1) * n);
  double sum = 0;
  for (int v = helper * n + tid; v < end; v += 16 * kThreads) {
    float y[16];  // all on their way before the first is used
#pragma unroll
    for (int i = 0; i < 16; i++)
      y[i] = v + i * kThreads < end ? to_f32(x[v + i * kThreads]) : -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; i++) sum += exp_below((double)y[i] - (double)m);
  }
  sum = warp_sum(sum);
  __syncthreads();
  if (lane == 0) s_warp[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    sum = warp_sum(lane < kWarps ? s_warp[lane] : 0.0);
    if (lane == 0) store_cluster(to, sum);
  }
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) beam_pick_kernel(const __grid_constant__ BeamArgs a) {
  constexpr int kWarps = kThreads / 32;
  __shared__ double s_lse[TABBY_BEAM_MAX], s_score[TABBY_BEAM_MAX];
  __shared__ double s_bound[kWarps];
  __shared__ CandTable s_cand;
  __shared__ int16_t s_order[kPickCap];
  __shared__ int s_rank[kPickCap];
  __shared__ float s_rowmax[TABBY_BEAM_MAX];
  __shared__ uint8_t s_done[TABBY_BEAM_MAX];
  __shared__ uint32_t s_again[TABBY_BEAM_MAX], s_need;
  __shared__ double s_part[kMaxHelpers][TABBY_BEAM_MAX];
  __shared__ int s_count;
  __shared__ uint32_t s_floor, s_top;
  const int b = blockIdx.x / a.helpers, helper = blockIdx.x - b * a.helpers;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = b * a.beams, lists = a.beams * a.chunks;
  cluster_arrive();  // all of the cluster run once this is complete
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const ChunkStats *stats = a.stats + (int64_t)row0 * a.chunks;
  if (helper > 0) {  // waits for the first CTA's word
    cluster_wait();
    cluster_arrive();
    cluster_wait();
    if (!s_need) return;
    for (int i = 0; i < a.beams; i++)
      if (load_cluster(in_first_cta(&s_again[i])))
        share_sum<T, kThreads>(a, row0 + i,
                               __uint_as_float(load_cluster(in_first_cta(&s_rowmax[i]))), helper,
                               s_bound, in_first_cta(&s_part[helper][i]));
    cluster_arrive();
    cluster_wait();
    return;
  }
  // The word to the others, whether they are needed; a cluster_wait() stands behind it.
  auto tell = [&](uint32_t need) {
    cluster_wait();
    if (tid > 0 && tid < a.helpers) store_cluster(in_cta(&s_need, tid), need);
    cluster_arrive();
  };
  if (tid == 0) s_floor = s_top = 0;
  // Log-sum-exps, a warp a beam.
  bool bad = false;
  for (int i = warp; i < a.beams; i += kWarps) {
    const float score = a.scores[row0 + i];
    const bool done = a.finished && a.finished[row0 + i] && score != -INFINITY;
    float m = -INFINITY;
    for (int c = lane; c < a.chunks; c += 32) {
      const float y = stats[i * a.chunks + c].max;
      bad |= isnan(y);
      m = fmaxf(m, y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    double sum = 0;
    for (int c = lane; c < a.chunks; c += 32) {
      const ChunkStats s = stats[i * a.chunks + c];
      if (s.max > -INFINITY) sum += s.sum * exp((double)s.max - (double)m);
    }
    sum = warp_sum(sum);
    bad |= !(score < INFINITY);
    if (lane == 0) {
      s_rowmax[i] = m;
      s_lse[i] = m > -INFINITY ? (double)m + log(sum) : 0.0;
      s_score[i] = score;
      s_done[i] = done;
      s_again[i] = 0;
    }
  }
  bad = __syncthreads_or(bad);
  auto write = [&](int j, bool none, const Cand &c) {
    const int64_t o = (int64_t)b * a.n_out + j;
    a.next_scores[o] = none ? -INFINITY : (float)c.key;
    a.parents[o] = none ? -1 : c.beam;
    a.tokens[o] = none ? -1 : c.token;
    if (a.next_finished) a.next_finished[o] = none || c.token == a.eos || s_done[c.beam] ? 1 : 0;
  };
  if (tid == 0) a.status[b] = bad ? TABBY_EINPUT : TABBY_OK;
  if (bad) {
    tell(0);
    for (int j = tid; j < a.n_out; j += kThreads) write(j, true, Cand());
    cluster_wait();
    return;
  }
  // A beam's entry of a list, a list's best key.
  auto entry = [&](int beam, float2 y) {
    Cand c;
    c.beam = beam;
    c.token = __float_as_int(y.y);
    c.x = y.x;
    c.key = s_score[c.beam] + ((double)y.x - s_lse[c.beam]);
    return c;
  };
  auto key_of = [&](int l, float x) {  // a logit's of list l
    const int i = l / a.chunks;
    return x > -INFINITY ? s_score[i] + ((double)x - s_lse[i]) : -INFINITY;
  };
  auto list_top = [&](int l) { return key_of(l, stats[l].max); };
  auto finished = [&](int i) {
    Cand c;
    c.beam = i;
    c.token = a.eos;
    c.x = 0.f;
    c.key = s_score[i];
    return c;
  };
  // A bound that at least n_out keys reach: the n_out-th largest of the threads' values (-inf
  // where there are fewer), rounded down, by bisection over the exponent and 8 more bits, as fp32,
  // of how far they lie below the prompt's best. (Of the keys themselves as many bits are steps
  // of 8 to 32 where the running scores of long sequences lie, at minus some thousands: at scores
  // near -5000 32 x 8 beams of 151936 take 42.6 us a step like this and took 382 by the keys, one
  // bit more of them even; 4 x 32 of 49152, 64 out, 25.1 and 1113.)
  auto bound_of = [&](double top) {
    const double best = s_top > order_key(-INFINITY) ? (double)key_value(s_top) : 0.0;
    const uint32_t key = order_key(__double2float_rd(__dsub_rd(top, best)));
    uint32_t kth = 0;
    for (int bit = 30; bit >= 15; bit--) {  // the sign is known
      const uint32_t probe = kth | 1u << bit;
      if (__syncthreads_count(key >= probe) >= a.n_out) kth = probe;
    }
    return kth > order_key(-INFINITY) ? __dadd_rd(best, (double)key_value(kth)) : -INFINITY;
  };
  auto keep = [&](const Cand &c, double least) {
    if (c.key < least) return;
    const int at = atomicAdd(&s_count, 1);
    if (at < kPickCap) s_cand.put(at, c);
  };
  // Goes over the entries of the lists whose best reaches `least`, four entries a lane on their way
  // at a time. A warp looks at 32 lists. Where lists are long (the CTAs of 1024 threads) its lanes
  // then go through one after the other; where they are short they are laid end to end. (4 x 32
  // beams, 64 out: 22.0 us a step one after the other, 24.7 end to end; 2 x 4 beams, 8 out: 11.7
  // and 10.3.)
  auto each_entry = [&](double least, auto use) {
    for (int l0 = warp; l0 < lists; l0 += 32 * kWarps) {
      const int mine = l0 + lane * kWarps;
      int count = mine < lists ? stats[mine].count : 0;
      if (count > 0 && !(list_top(mine) >= least)) count = 0;
      if constexpr (kThreads > 256) {
        for (unsigned in = __ballot_sync(0xffffffffu, count > 0); in; in &= in - 1) {
          const int f = __ffs(in) - 1, n = __shfl_sync(0xffffffffu, count, f);
          const int l = l0 + f * kWarps, beam = l / a.chunks;
          const float2 *list = a.lists + ((int64_t)row0 * a.chunks + l) * a.cap;
          for (int e = lane; e < n; e += 128) {
            float2 y[4];
#pragma unroll
            for (int k = 0; k < 4; k++) y[k] = list[min(e + 32 * k, n - 1)];
#pragma unroll
            for (int k = 0; k < 4; k++)
              if (e + 32 * k < n) use(entry(beam, y[k]));
          }
          __syncwarp();
        }
      } else {
        const int beam = mine / a.chunks;
        int end = count;  // inclusive over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, end, o);
          if (lane >= o) end += y;
        }
        const int all = __shfl_sync(0xffffffffu, end, 31);
        for (int f0 = 0; f0 < all; f0 += 128) {
          float2 y[4];
          int of[4];
#pragma unroll
          for (int k = 0; k < 4; k++) {
            if (f0 + 32 * k >= all) break;  // the whole warp
            const int f = min(f0 + 32 * k + lane, all - 1);
            int lo = 0;  // the first list that ends behind f
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
              if (__shfl_sync(0xffffffffu, end, lo + o - 1) <= f) lo += o;
            const int e = f - __shfl_sync(0xffffffffu, end - count, lo);
            y[k] = a.lists[((int64_t)row0 * a.chunks + l0 + lo * kWarps) * a.cap + e];
            of[k] = __shfl_sync(0xffffffffu, beam, lo);
          }
#pragma unroll
          for (int k = 0; k < 4; k++)
            if (f0 + 32 * k + lane < all) use(entry(of[k], y[k]));
          __syncwarp();
        }
      }
    }
  };
  // What is no smaller than a bound, less what more exact keys might bring up.
  auto collect = [&](double bound) {
    const double least = bound - 2 * a.gap;
    if (tid == 0) s_count = 0;
    __syncthreads();
    each_entry(least, [&](const Cand &c) { keep(c, least); });
    for (int i = tid; i < a.beams; i += kThreads)
      if (s_done[i]) keep(finished(i), least);
    __syncthreads();
  };
  // A bound from the lists' bests, or the best of the lists' own floors; where too much passes it,
  // one from the entries.
  double top = -INFINITY, floor = -INFINITY;
  for (int l = lane * kWarps + warp; l < lists; l += kThreads) {
    top = fmax(top, list_top(l));
    floor = fmax(floor, key_of(l, stats[l].floor));
  }
  const uint32_t floors = __reduce_max_sync(0xffffffffu, order_key(__double2float_rd(floor)));
  const uint32_t tops = __reduce_max_sync(0xffffffffu, order_key(__double2float_ru(top)));
  if (lane == 0) {
    atomicMax(&s_floor, floors);
    atomicMax(&s_top, tops);
  }
  __syncthreads();
  double bound = bound_of(top);
  bound = fmax(bound, s_floor > order_key(-INFINITY) ? (double)key_value(s_floor) : -INFINITY);
  collect(bound);
  if (s_count > kPickTight) {
    top = -INFINITY;
    each_entry(bound, [&](const Cand &c) { top = fmax(top, c.key); });
    __syncthreads();
    bound = fmax(bound, bound_of(top));
    collect(bound);
  }
  // The lse of the marked beams in 64 bits, from all their logits, with the cluster's help.
  auto refine = [&]() {
    tell(1);
    cluster_wait();
    for (int i = 0; i < a.beams; i++)
      if (s_again[i])
        share_sum<T, kThreads>(a, row0 + i, s_rowmax[i], 0, s_bound, in_first_cta(&s_part[0][i]));
    cluster_arrive();
    cluster_wait();
    for (int i = tid; i < a.beams; i += kThreads) {
      if (!s_again[i]) continue;
      double sum = 0;
      for (int k = 0; k < a.helpers; k++) sum += s_part[k][i];
      s_lse[i] = (double)s_rowmax[i] + log(sum);
    }
    __syncthreads();
  };
  const bool many = s_count > kPickCap;
  if (many) {
    // Too many for the table, by ties or near ties: with all keys exact, the best one after the
    // other.
    __syncthreads();
    if (tid == 0) s_count = 0;
    for (int i = tid; i < a.beams; i += kThreads)
      s_again[i] = !s_done[i] && s_rowmax[i] > -INFINITY;
    __syncthreads();
    refine();
    __shared__ Cand s_best[kWarps], s_last;
    Cand last;
    last.key = INFINITY;
    last.x = INFINITY;
    last.beam = -1;
    last.token = -1;
    for (int j = 0; j < a.n_out; j++) {
      Cand best;
      best.beam = -1;
      auto consider = [&](const Cand &c) {
        if ((last.beam < 0 || stands_before(last, c)) &&
            (best.beam < 0 || stands_before(c, best)))
          best = c;
      };
      each_entry(-INFINITY, consider);
      for (int i = tid; i < a.beams; i += kThreads)
        if (s_done[i]) consider(finished(i));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        Cand c;
        c.key = __shfl_xor_sync(0xffffffffu, best.key, o);
        c.x = __shfl_xor_sync(0xffffffffu, best.x, o);
        c.beam = __shfl_xor_sync(0xffffffffu, best.beam, o);
        c.token = __shfl_xor_sync(0xffffffffu, best.token, o);
        if (c.beam >= 0 && (best.beam < 0 || stands_before(c, best))) best = c;
      }
      if (lane == 0) s_best[warp] = best;
      __syncthreads();
      if (tid == 0) {
        best = s_best[0];
        for (int w = 1; w < kWarps; w++)
          if (s_best[w].beam >= 0 && (best.beam < 0 || stands_before(s_best[w], best)))
            best = s_best[w];
        s_last = best;
        if (best.beam >= 0) s_cand.put(s_count++, best);
      }
      __syncthreads();
      last = s_last;
      if (last.beam < 0) break;
    }
    __syncthreads();
  }
  const int n = s_count;
  // 1 where candidate 2 stands before; without branches, of which each costs tens of cycles.
  auto before = [](int64_t key2, uint64_t tie2, int32_t token2, int64_t key, uint64_t tie,
                   int32_t token) {
    const unsigned less = (unsigned)(tie2 < tie) |
                          ((unsigned)(tie2 == tie) & (unsigned)(token2 < token));
    return (int)((unsigned)(key2 > key) | ((unsigned)(key2 == key) & less));
  };
  auto rank = [&]() {  // s_order[j]: the candidate of rank j
    if (n <= 32) {  // a warp, a candidate a lane
      if (warp == 0) {
        const int me = min(lane, max(n, 1) - 1);
        const int64_t key = s_cand.key[me];
        const uint64_t tie = s_cand.tie[me];
        const int32_t token = s_cand.token[me];
        int r = 0;
        for (int k = 0; k < n; k++)
          r += before(__shfl_sync(0xffffffffu, key, k), __shfl_sync(0xffffffffu, tie, k),
                      __shfl_sync(0xffffffffu, token, k), key, tie, token);
        if (lane < n) s_order[r] = (int16_t)lane;
      }
      __syncthreads();
      return;
    }
    const int parts = max(1, kThreads / n);  // a few threads a candidate
    for (int i = tid; i < n; i += kThreads) s_rank[i] = 0;
    __syncthreads();
    for (int i = tid; i < n * parts; i += kThreads) {
      const int p = i / n, me = i - p * n;
      const int64_t key = s_cand.key[me];
      const uint64_t tie = s_cand.tie[me];
      const int32_t token = s_cand.token[me];
      int r = 0;
#pragma unroll 4
      for (int k = p; k < n; k += parts)
        r += before(s_cand.key[k], s_cand.tie[k], s_cand.token[k], key, tie, token);
      if (r) atomicAdd(&s_rank[me], r);
    }
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) s_order[s_rank[i]] = (int16_t)i;
    __syncthreads();
  };
  rank();
  // Neighbours of different beams that are too close to be told apart by fp32 sums, down to
  // those that are as close to the last one chosen.
  bool close = false;
  const double lowest = n > 0 ? s_cand.get(s_order[min(n, a.n_out) - 1]).key - a.gap : 0.0;
  for (int j = tid; !many && j < n - 1; j += kThreads) {
    const Cand p = s_cand.get(s_order[j]), q = s_cand.get(s_order[j + 1]);
    if (q.key >= lowest && p.beam != q.beam && p.key - q.key < a.gap) {
      if (!s_done[p.beam]) s_again[p.beam] = 1, close = true;
      if (!s_done[q.beam]) s_again[q.beam] = 1, close = true;
    }
  }
  const bool again = __syncthreads_or(close);
  if (again) {
    refine();
    for (int i = tid; i < n; i += kThreads)
      if (const Cand c = s_cand.get(i); s_again[c.beam])
        s_cand.key[i] = key_bits(s_score[c.beam] + ((double)c.x - s_lse[c.beam]));
    __syncthreads();
    rank();
  }
  if (!again && !many) tell(0);
  for (int j = tid; j < a.n_out; j += kThreads)
    write(j, j >= n, j < n ? s_cand.get(s_order[j]) : Cand());
  if (!again && !many) cluster_wait();
}

// Chunks of a row: at most 128 threads' worth of pieces each.
struct ScanPlan {
  int nv;      // pieces a thread
  int chunks;  // a row
  int cap;     // entries of a list
};
ScanPlan scan_plan(int64_t rows, int32_t vocab, int32_t dtype, int32_t n_out) {
  const int n = dtype == TABBY_F32 ? 4 : 8;
  const int64_t pieces = ((int64_t)vocab + 2 * n - 2) / n;  // at most, however a row is aligned
  auto chunks = [&](int nv) {
    return (int)((pieces + (int64_t)nv * kScanThreads - 1) / ((int64_t)nv * kScanThreads));
  };
  ScanPlan p;
  p.nv = 48 / n;
  // Few rows: smaller chunks, so that more SMs have one (8 rows of 50257 bf16: 10.5 us as 200
  // chunks of 2048, 11.7 as 72 of 6144; but 4 rows of 151936: 11.7 as 300, 11.0 as 100).
  if (rows * chunks(p.nv) < 74) p.nv = 16 / n;
  p.chunks = chunks(p.nv);
  p.cap = std::max(128, 4 * n_out);
  return p;
}

// Threads of a pick CTA. Many lists with many entries: more of them (rows of 50257 bf16, us a step
// with 256 and with 1024 threads: 4 x 32 beams, 64 out 37.5 and 25.6; 32 x 8, 32 out 27.6 and 26.4;
// 4 x 8, 16 out 13.1 and 14.6; 32 x 8, 16 out 23.2 and 24.0).
int pick_threads(int32_t beams, int32_t n_out) { return beams * n_out >= 256 ? 1024 : 256; }
// CTAs a prompt of the pick: where SMs are left over they help with the rare sums in 64 bits, as
// many as find a place at once. A CTA of 1024 threads takes an SM, and a cluster of them has to lie
// in one group of SMs: 15 clusters of 8 fit, 33 of 4. (4 beams, 64 out: 16 prompts with 8 CTAs each
// 38.8 us a step, with 4 24.4; 64 prompts with 8, 4, 2 and 1 each 100, 53.1, 36.3 and 36.3; of a
// step that needs the sums 145, 78.3, 56.2 and 69.3. CTAs of 256 threads, 64 x 4 beams, 8 out: 27.4
// with 8 each, 21.4 with 4, 21.1 with 1, and 53.0, 48.4 and 84.6 with the sums.)
int pick_helpers(int32_t batch, int threads) {
  int n = kMaxHelpers;
  // (The larger a cluster, the more SMs of the groups it leaves over.)
  while (n > 1 && (int64_t)batch * n > (threads == 1024 ? 148 - 5 * n : 296)) n /= 2;
  return n;
}

template <typename T>
cudaError_t launch_beam(const BeamArgs &a, int nv, cudaStream_t q) {
  constexpr int kN = Vec16<T>::kN;
  const dim3 grid((unsigned)a.batch * (unsigned)a.beams * (unsigned)a.chunks);
  cudaError_t err =
      nv == 48 / kN ? launch_pdl(beam_scan_kernel<T, 48 / kN>, grid, kScanThreads, 0, q, a)
                    : launch_pdl(beam_scan_kernel<T, 16 / kN>, grid, kScanThreads, 0, q, a);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.batch * a.helpers));
  const int threads = pick_threads(a.beams, a.n_out);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = q;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)a.helpers, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return threads == 256 ? cudaLaunchKernelEx(&cfg, beam_pick_kernel<T, 256>, a)
                        : cudaLaunchKernelEx(&cfg, beam_pick_kernel<T, 1024>, a);
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
  if ((int64_t)beams * vocab > INT32_MAX)
    return decode_fail(TABBY_EINVAL, "beam_step: beams * vocab must be below 2^31");
  for (int32_t dtype : {TABBY_F32, TABBY_BF16, TABBY_F16})
    if ((int64_t)batch * beams >
        INT32_MAX / scan_plan((int64_t)batch * beams, vocab, dtype, n_out).chunks)
      return decode_fail(TABBY_EINVAL, "beam_step: batch * beams * vocab is too large");
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
  // The most that any type's plan takes.
  *bytes = 0;
  for (int32_t dtype : {TABBY_F32, TABBY_BF16, TABBY_F16}) {
    const ScanPlan p = scan_plan((int64_t)batch * beams, vocab, dtype, n_out);
    *bytes = std::max(*bytes, (size_t)batch * beams * p.chunks *
                                  (sizeof(ChunkStats) + p.cap * sizeof(float2)));
  }
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
  const ScanPlan plan = scan_plan((int64_t)rows, vocab, dtype, n_out);
  a.chunks = plan.chunks;
  a.cap = plan.cap;
  a.helpers = pick_helpers(batch, pick_threads(beams, n_out));
  a.gap = gap_of(vocab);
  a.stats = static_cast<ChunkStats *>(d_workspace);
  a.lists = reinterpret_cast<float2 *>(a.stats + rows * plan.chunks);
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == TABBY_F32    ? launch_beam<float>(a, plan.nv, q)
                          : dtype == TABBY_BF16 ? launch_beam<__nv_bfloat16>(a, plan.nv, q)
                                                : launch_beam<__half>(a, plan.nv, q);
  if (err != cudaSuccess) return decode_cuda_fail(err, "beam_step launch");
  return TABBY_OK;
}

}  // extern "C"
