// Attention of a drafted tree over a key/value cache (tabby_tree_attention_async).
//
//   out[b][j][h] = sum_t softmax_t(scale q.k[t]) v[t],  t < L or t = L + (j or an ancestor)
//
// One CTA a (sequence, slot, head): each warp takes every fourth key, its lanes four of the
// dim values each, with a running maximum and sum; the warps' partial results are joined
// through shared memory.
#include <math.h>

#include "decode_internal.h"

namespace tabby {
namespace {

constexpr int kWarps = 4;

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) tree_kernel(tabby_tree_attention_args a) {
  __shared__ int32_t parents[TABBY_TREE_MAX_NODES];
  __shared__ float so[kWarps][TABBY_TREE_MAX_DIM], sm[kWarps], sl[kWarps];
  const int j = blockIdx.x % a.nodes, h = (blockIdx.x / a.nodes) % a.heads;
  const int64_t b = blockIdx.x / a.nodes / a.heads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if ((int)threadIdx.x < a.nodes)
    parents[threadIdx.x] = a.parents[b * a.parents_stride + threadIdx.x];
  __syncthreads();
  const int64_t start = a.lengths[b];
  const unsigned long long sees =
      start >= 0 && start + j < a.entries ? tree_sees(parents, j) : 0;
  T *out = static_cast<T *>(a.out) + b * a.out_batch_stride + j * a.out_node_stride +
           h * a.out_head_stride;
  const int d0 = 4 * lane;
  if (sees == 0) {
    if (warp == 0 && d0 < a.dim)
      for (int c = 0; c < 4; c++) out[d0 + c] = T(0.f);
    return;
  }
  const int hk = h / (a.heads / a.kv_heads);
  const T *q = static_cast<const T *>(a.q) + b * a.q_batch_stride + j * a.q_node_stride +
               h * a.q_head_stride;
  const T *k = static_cast<const T *>(a.k) + b * a.k_batch_stride + hk * a.k_head_stride;
  const T *v = static_cast<const T *>(a.v) + b * a.v_batch_stride + hk * a.v_head_stride;
  float qf[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
  for (int c = 0; c < 4; c++) qf[c] = d0 < a.dim ? to_f32(q[d0 + c]) * a.scale : 0;
  const int64_t end = min(start + a.nodes, (int64_t)a.entries);
  for (int64_t t = warp; t < end; t += kWarps) {
    if (t >= start && !(sees >> (t - start) & 1)) continue;
    float x = 0;
    if (d0 < a.dim)
      for (int c = 0; c < 4; c++) x += qf[c] * to_f32(k[t * a.k_entry_stride + d0 + c]);
    for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
    const float m2 = fmaxf(m, x), f = expf(m - m2), p = expf(x - m2);
    l = l * f + p;
    m = m2;
    if (d0 < a.dim)
      for (int c = 0; c < 4; c++)
        o[c] = o[c] * f + p * to_f32(v[t * a.v_entry_stride + d0 + c]);
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  for (int c = 0; c < 4; c++) so[warp][d0 + c] = o[c];
  __syncthreads();
  if (warp == 0 && d0 < a.dim) {
    float mm = -INFINITY, ll = 0, oo[4] = {0, 0, 0, 0};
    for (int w = 0; w < kWarps; w++) mm = fmaxf(mm, sm[w]);
    for (int w = 0; w < kWarps; w++) {
      const float f = expf(sm[w] - mm);
      ll += sl[w] * f;
      for (int c = 0; c < 4; c++) oo[c] += so[w][d0 + c] * f;
    }
    for (int c = 0; c < 4; c++) out[d0 + c] = T(oo[c] / ll);
  }
}

int check_tree(int32_t batch, int32_t nodes, int32_t heads, int32_t kv_heads, int32_t dim) {
  if (batch < 0) return decode_fail(TABBY_EINVAL, "tree_attention: batch must be >= 0");
  if (nodes < 1 || nodes > TABBY_TREE_MAX_NODES)
    return decode_fail(TABBY_EINVAL, "tree_attention: nodes must be in [1, %d], got %d",
                       TABBY_TREE_MAX_NODES, nodes);
  if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads > 65536)
    return decode_fail(TABBY_EINVAL,
                       "tree_attention: heads (%d) must be a multiple of kv_heads (%d), at most "
                       "65536",
                       heads, kv_heads);
  if (dim < 8 || dim > TABBY_TREE_MAX_DIM || dim % 8 != 0)
    return decode_fail(TABBY_EINVAL,
                       "tree_attention: dim must be a multiple of 8 in [8, %d], got %d",
                       TABBY_TREE_MAX_DIM, dim);
  if ((int64_t)batch * heads * nodes > INT32_MAX)
    return decode_fail(TABBY_EINVAL, "tree_attention: batch * heads * nodes exceeds 2^31 - 1");
  return TABBY_OK;
}

}  // namespace
}  // namespace tabby

extern "C" {

int tabby_tree_workspace_bytes(int32_t batch, int32_t nodes, int32_t heads, int32_t kv_heads,
                               int32_t dim, size_t *bytes) {
  using namespace tabby;
  const int st = check_tree(batch, nodes, heads, kv_heads, dim);
  if (st) return st;
  if (!bytes) return decode_fail(TABBY_EINVAL, "tree_attention: bytes is NULL");
  *bytes = 16;
  return TABBY_OK;
}

int tabby_tree_attention_async(int32_t device, const tabby_tree_attention_args *h_args,
                               void *stream) {
  using namespace tabby;
  if (!h_args) return decode_fail(TABBY_EINVAL, "tree_attention: args is NULL");
  const tabby_tree_attention_args a = *h_args;
  size_t need = 0;
  const int st =
      tabby_tree_workspace_bytes(a.batch, a.nodes, a.heads, a.kv_heads, a.dim, &need);
  if (st) return st;
  if (a.dtype != TABBY_BF16 && a.dtype != TABBY_F16)
    return decode_fail(TABBY_EINVAL, "tree_attention: dtype must be TABBY_BF16 or TABBY_F16");
  if (a.entries < 1) return decode_fail(TABBY_EINVAL, "tree_attention: entries must be >= 1");
  if (!(a.scale > -INFINITY && a.scale < INFINITY))
    return decode_fail(TABBY_EINVAL, "tree_attention: scale must be finite");
  if (a.batch == 0) return TABBY_OK;
  if (!a.q || !a.k || !a.v || !a.out || !a.lengths || !a.parents)
    return decode_fail(TABBY_EINVAL, "tree_attention: a required pointer is NULL");
  if (!aligned_to(a.q, 16) || !aligned_to(a.k, 16) || !aligned_to(a.v, 16) ||
      !aligned_to(a.out, 16))
    return decode_fail(TABBY_EINVAL, "tree_attention: q, k, v and out must be 16-byte aligned");
  const int64_t strides[12] = {a.q_batch_stride,   a.q_node_stride,    a.q_head_stride,
                               a.k_batch_stride,   a.k_head_stride,    a.k_entry_stride,
                               a.v_batch_stride,   a.v_head_stride,    a.v_entry_stride,
                               a.out_batch_stride, a.out_node_stride,  a.out_head_stride};
  for (int64_t s : strides)
    if (s < 0 || s % 8 != 0)
      return decode_fail(TABBY_EINVAL,
                         "tree_attention: strides must be multiples of 8 elements, >= 0");
  if (a.parents_stride < 0)
    return decode_fail(TABBY_EINVAL, "tree_attention: parents_stride must be >= 0");
  if (!a.workspace || a.workspace_bytes < need || !aligned_to(a.workspace, 16))
    return decode_fail(TABBY_EINVAL,
                       "tree_attention: needs a 16-byte aligned workspace of %zu bytes", need);
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return decode_cuda_fail(scope.err, "cudaSetDevice");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)((int64_t)a.batch * a.heads * a.nodes);
  if (a.dtype == TABBY_BF16)
    tree_kernel<__nv_bfloat16><<<grid, 32 * kWarps, 0, s>>>(a);
  else
    tree_kernel<__half><<<grid, 32 * kWarps, 0, s>>>(a);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return decode_cuda_fail(err, "tree_attention launch");
  return TABBY_OK;
}

}  // extern "C"
