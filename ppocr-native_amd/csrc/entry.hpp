// What the C entries of the decoder layers share (decoder.cpp, writer.cpp):
// refusals, the stream's device, checks of pointers, strides and caches.
// Nothing here allocates, waits or throws.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "decoder.hpp"
#include "ppocr_hip.h"

namespace {

using namespace ppocr;

struct Fail {
  char *err;
  size_t len;
  __attribute__((format(printf, 2, 3))) int operator()(const char *fmt, ...) const {
    if (err && len) {
      va_list ap;
      va_start(ap, fmt);
      vsnprintf(err, len, fmt, ap);
      va_end(ap);
    }
    return int(hipErrorInvalidValue);
  }
  int hip(const char *what, hipError_t e) const {
    if (e == hipSuccess) return 0;
    (*this)("%s: %s", what, hipGetErrorString(e));
    return int(e);
  }
};

// Makes the stream's device current for the launch, if it is another. Two
// handles are numbers and no streams: that of the thread's own stream, which is
// the current device's, and that of the legacy default stream, which ended the
// process in the runtime and is refused (NULL is that stream).
struct OnDevice {
  int before = -1;
  hipError_t e = hipSuccess;
  explicit OnDevice(hipStream_t s) {
    if (s == hipStreamLegacy) {
      e = hipErrorInvalidHandle;
      return;
    }
    if (!s || s == hipStreamPerThread) return;
    hipDevice_t of = 0;
    int now = 0;
    if ((e = hipGetDevice(&now)) != hipSuccess || (e = hipStreamGetDevice(s, &of)) != hipSuccess) return;
    if (of == now) return;
    if ((e = hipSetDevice(of)) == hipSuccess) before = now;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

constexpr size_t kMost = size_t(1) << 30;  // most rows, values a row and the like
constexpr size_t kMostStride = size_t(1) << 40;

inline bool is_real(int t) { return t == PPOCR_F32 || t == PPOCR_BF16 || t == PPOCR_F16; }
inline size_t size_of(int t) { return t == PPOCR_F32 ? 4 : t == PPOCR_BF16 || t == PPOCR_F16 ? 2 : 1; }
inline bool aligned(const void *p, size_t n) { return uintptr_t(p) % n == 0; }

// A softmax's scale for 2-logarithms: positive (a hidden product, -inf, times
// 0 would be NaN; 1e-30 makes the weights equal just as well).
inline float scale_of(float scale) { return std::fmax(std::fabs(scale) * 1.44269504088896340736f, 1e-30f); }

// A stride's value: rows without a gap where it is 0.
inline bool stride_of(size_t given, size_t width, long *out) {
  *out = long(given ? given : width);
  return (!given || given >= width) && given <= kMostStride;
}

// The cache's own checks; fills `c`.
inline int cache_of(const Fail &fail, const char *what, const ppocr_kv_cache *k, const int32_t *table, size_t table_width,
             const int32_t *lengths, CacheArgs &c) {
  if (!k || !k->k || !k->v || !table || !lengths) return fail("%s: no cache, page table or lengths", what);
  if (!is_real(k->type)) return fail("%s: a cache of type %d", what, k->type);
  if (!aligned(k->k, size_of(k->type)) || !aligned(k->v, size_of(k->type)) || !aligned(table, 4) ||
      !aligned(lengths, 4))
    return fail("%s: a pointer is not aligned to its type", what);
  if (!k->pages || !k->page_size || !k->heads || !k->dim || k->pages > kMost || k->page_size > kMost ||
      k->heads > 65535)
    return fail("%s: a cache of %zu pages of %zu tokens of %zu heads", what, k->pages, k->page_size, k->heads);
  if (k->dim > 256) return fail("%s: heads of %zu values: 1 to 256 are taken", what, k->dim);
  if (!table_width || table_width > kMost || table_width * k->page_size > (size_t(1) << 31) - 4096)
    return fail("%s: a page table of %zu pages of %zu tokens a text", what, table_width, k->page_size);
  const size_t row = k->heads * k->dim;
  if (!k->page_stride && !k->token_stride && !k->head_stride) {
    c.head_stride = long(k->dim), c.token_stride = long(row), c.page_stride = long(row * k->page_size);
  } else {
    if (k->head_stride < k->dim || k->token_stride < k->dim || k->page_stride < k->dim ||
        k->head_stride > kMostStride || k->token_stride > kMostStride || k->page_stride > kMostStride)
      return fail("%s: cache strides %zu, %zu, %zu for heads of %zu values", what, k->page_stride, k->token_stride,
                  k->head_stride, k->dim);
    c.head_stride = long(k->head_stride), c.token_stride = long(k->token_stride), c.page_stride = long(k->page_stride);
  }
  c.k = k->k, c.v = k->v;
  c.pages = int(k->pages), c.page_size = int(k->page_size), c.heads = int(k->heads), c.dim = int(k->dim);
  c.by_page = Divide(c.page_size);
  c.table = table, c.table_width = long(table_width), c.lengths = lengths;
  return 0;
}

}  // namespace
