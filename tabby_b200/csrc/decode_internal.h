// What the files of libtabbydecode.so share (include/tabby_decode.h is the public surface).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "sampler_internal.h"  // DeviceScope
#include "tabby_decode.h"

namespace tabby {

// Records a message for tabby_decode_last_error() and returns `status`.
int decode_fail(int status, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int decode_cuda_fail(cudaError_t err, const char *what);

inline bool aligned_to(const void *p, uintptr_t n) {
  return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

// Checks a state layout of `rows` rows (tabby_decode.h); `what` names the call in the message.
int check_layout(const char *what, const tabby_state_layout *l, int64_t rows);

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

// A slot of a drafted tree is in use when its way up over ever lower slots ends in a root;
// returns the slots it sees (itself and its ancestors) as a bit mask, 0 when it is unused.
// `parents` may lie in shared memory; the way has at most 64 steps.
__device__ __forceinline__ unsigned long long tree_sees(const int32_t *parents, int j) {
  unsigned long long m = 0;
  while (true) {
    m |= 1ull << j;
    const int p = parents[j];
    if (p == -1) return m;
    if (p < 0 || p >= j) return 0;
    j = p;
  }
}

}  // namespace tabby
