// Errors, version and shared argument checks of libtabbydecode.so (include/tabby_decode.h).
#include <stdarg.h>
#include <stdio.h>

#include <utility>

#include "decode_internal.h"

namespace {
thread_local char g_error[512] = "";
}

int tabby::decode_fail(int status, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return status;
}

int tabby::decode_cuda_fail(cudaError_t err, const char *what) {
  return decode_fail(TABBY_ECUDA, "%s: %s (%s)", what, cudaGetErrorName(err),
                     cudaGetErrorString(err));
}

int tabby::check_layout(const char *what, const tabby_state_layout *l, int64_t rows) {
  if (!l) return decode_fail(TABBY_EINVAL, "%s: layout is NULL", what);
  if (l->segments < 1 || l->entries < 1 || l->entry_bytes < 1)
    return decode_fail(TABBY_EINVAL, "%s: segments, entries and entry_bytes must be >= 1", what);
  if (l->entry_bytes >= (int64_t)1 << 31)
    return decode_fail(TABBY_EINVAL, "%s: entry_bytes must be below 2^31", what);
  if (l->row_stride < 0 || l->segment_stride < 0 || l->entry_stride < 0)
    return decode_fail(TABBY_EINVAL, "%s: strides must be >= 0", what);
  // Taken from the smallest stride up, each must pass everything the ones below it span.
  struct {
    int64_t n, stride;
  } d[3] = {{rows, l->row_stride}, {l->segments, l->segment_stride}, {l->entries, l->entry_stride}};
  if (d[0].stride > d[1].stride) std::swap(d[0], d[1]);
  if (d[1].stride > d[2].stride) std::swap(d[1], d[2]);
  if (d[0].stride > d[1].stride) std::swap(d[0], d[1]);
  __int128 span = l->entry_bytes;
  for (const auto &x : d) {
    if (x.n <= 1) continue;
    if (x.stride < span) return decode_fail(TABBY_EINVAL, "%s: the states' parts overlap", what);
    span += (__int128)x.stride * (x.n - 1);
  }
  return TABBY_OK;
}

extern "C" {

int32_t tabby_decode_abi_version(void) { return TABBY_DECODE_ABI_VERSION; }

const char *tabby_decode_last_error(void) { return g_error; }

}  // extern "C"
