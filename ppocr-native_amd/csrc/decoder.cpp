// The C entries of the decoder layers (include/ppocr_hip.h): checks of the
// arguments, the stream's device, and the launch. Nothing here allocates,
// waits or throws.
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

bool is_real(int t) { return t == PPOCR_F32 || t == PPOCR_BF16 || t == PPOCR_F16; }
size_t size_of(int t) { return t == PPOCR_F32 ? 4 : t == PPOCR_BF16 || t == PPOCR_F16 ? 2 : 1; }
bool aligned(const void *p, size_t n) { return uintptr_t(p) % n == 0; }

// A softmax's scale for 2-logarithms: positive (a hidden product, -inf, times
// 0 would be NaN; 1e-30 makes the weights equal just as well).
float scale_of(float scale) { return std::fmax(std::fabs(scale) * 1.44269504088896340736f, 1e-30f); }

// A stride's value: rows without a gap where it is 0.
bool stride_of(size_t given, size_t width, long *out) {
  *out = long(given ? given : width);
  return (!given || given >= width) && given <= kMostStride;
}

// Whether the 4-bit product takes these sizes.
bool q4_sizes(size_t m, size_t n, size_t k) {
  return k && k <= size_t(1) << 24 && n <= kMost && m <= size_t(1) << 20 &&
         (n + 15) / 16 * ((m + 15) / 16) <= size_t(1) << 24;
}

// The cache's own checks; fills `c`.
int cache_of(const Fail &fail, const char *what, const ppocr_kv_cache *k, const int32_t *table, size_t table_width,
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

extern "C" {

int ppocr_hip_rms_norm(const void *x, size_t x_stride, const void *residual, size_t residual_stride,
                       const void *weight, void *sum, size_t sum_stride, void *y, size_t y_stride, float *scales,
                       size_t rows, size_t c, int type, int y_type, size_t group, float eps, void *stream, char *err,
                       size_t err_len) {
  const Fail fail{err, err_len};
  if (!is_real(type)) return fail("rms norm: type %d", type);
  const bool y8 = y_type == PPOCR_E4M3 || y_type == PPOCR_I8;
  if (!y8 && y_type != type) return fail("rms norm: type %d gives type %d, e4m3 or 8-bit integers, not %d", type, type, y_type);
  if (rows == 0) return 0;
  if (!c || c > kMost || rows > kMost) return fail("rms norm: %zu rows of %zu values", rows, c);
  if (!x || !weight || !y || (y8 && !scales)) return fail("rms norm: x, weight, y and (for 8 bits) scales are needed");
  const size_t s = size_of(type);
  if (!aligned(x, s) || !aligned(residual, s) || !aligned(weight, s) || !aligned(sum, s) || !aligned(y, size_of(y_type)) ||
      !aligned(scales, 4))
    return fail("rms norm: a pointer is not aligned to its type");
  if (y8 && group != 0 && group != 32 && group != 64 && group != 128)
    return fail("rms norm: groups of %zu values: 0 (a row), 32, 64 or 128 are taken", group);
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail("rms norm: eps %g", double(eps));
  NormArgs a{};
  if (!stride_of(x_stride, c, &a.x_stride) || !stride_of(residual_stride, c, &a.residual_stride) ||
      !stride_of(sum_stride, c, &a.sum_stride) || !stride_of(y_stride, c, &a.y_stride))
    return fail("rms norm: rows of %zu values with strides %zu, %zu, %zu, %zu", c, x_stride, residual_stride,
                sum_stride, y_stride);
  a.x = x, a.residual = residual, a.weight = weight, a.sum = sum, a.y = y, a.scales = scales;
  a.rows = long(rows), a.c = int(c), a.eps = eps, a.inverse_c = float(1.0 / double(c));
  a.group = group && y8 ? int(group) : int(c);
  a.groups = int((c + a.group - 1) / a.group);
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip("rms norm", on.e);
  return fail.hip("rms norm", launch_rms_norm(a, type, y_type, hipStream_t(stream)));
}

int ppocr_hip_q4_product(const void *x, size_t x_stride, const float *x_scales, size_t x_group, const uint8_t *q,
                         const void *scales, const uint8_t *zeros, const void *bias, void *y, size_t y_stride,
                         size_t m, size_t n, size_t k, size_t group, int x_type, int scale_type, int y_type,
                         void *stream, char *err, size_t err_len) {
  const Fail fail{err, err_len};
  const bool x8 = x_type == PPOCR_E4M3 || x_type == PPOCR_I8;
  if (!is_real(x_type) && !x8) return fail("4-bit product: x of type %d", x_type);
  if (!is_real(scale_type)) return fail("4-bit product: scales of type %d", scale_type);
  if (!is_real(y_type)) return fail("4-bit product: y of type %d", y_type);
  if (group != 32 && group != 64 && group != 128)
    return fail("4-bit product: groups of %zu inputs: 32, 64 or 128 are taken", group);
  if (m == 0 || n == 0) return 0;
  if (!q4_sizes(m, n, k))
    return fail("4-bit product: %zu rows of %zu inputs to %zu outputs", m, k, n);
  if (!x || !q || !scales || !y || (x8 && !x_scales))
    return fail("4-bit product: x, q, scales, y and (for 8-bit x) x_scales are needed");
  if (x8 && x_group != 0 && x_group != group)
    return fail("4-bit product: x with a scale each %zu inputs, the weights each %zu", x_group, group);
  if (!aligned(x, size_of(x_type)) || !aligned(x_scales, 4) || !aligned(scales, size_of(scale_type)) ||
      !aligned(bias, size_of(y_type)) || !aligned(y, size_of(y_type)))
    return fail("4-bit product: a pointer is not aligned to its type");
  Q4Args a{};
  if (!stride_of(x_stride, k, &a.x_stride) || a.x_stride > 1 << 24 || !stride_of(y_stride, n, &a.y_stride))
    return fail("4-bit product: strides %zu for %zu inputs, %zu for %zu outputs", x_stride, k, y_stride, n);
  a.x = x, a.x_scales = x_scales, a.q = q, a.scales = scales, a.zeros = zeros, a.bias = bias, a.y = y;
  a.m = int(m), a.n = int(n), a.k = int(k), a.group = int(group), a.groups = int((k + group - 1) / group);
  a.x_group = int(x_group);
  a.scale_type = scale_type, a.y_type = y_type;
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip("4-bit product", on.e);
  const hipStream_t st = hipStream_t(stream);
  return fail.hip("4-bit product", x_type == PPOCR_F32    ? launch_q4_f32(a, 0, st)
                                   : x_type == PPOCR_BF16 ? launch_q4_bf16(a, 0, st)
                                   : x_type == PPOCR_F16  ? launch_q4_f16(a, 0, st)
                                                          : launch_q4_i8(a, x_type == PPOCR_E4M3, st));
}

size_t ppocr_hip_q4_product_tiles(size_t m, size_t n, size_t k, int x_type) {
  if (x_type < PPOCR_F32 || x_type > PPOCR_I8 || !m || !n || !q4_sizes(m, n, k)) return 0;
  return size_t(q4_tiles(x_type, int(m), int(n), int(k)));
}

int ppocr_hip_kv_append(const void *k, size_t k_stride, const void *v, size_t v_stride, const ppocr_kv_cache *cache,
                        const int32_t *table, size_t table_width, const int32_t *lengths, const int32_t *starts,
                        size_t batch, size_t rows, void *stream, char *err, size_t err_len) {
  const Fail fail{err, err_len};
  AppendArgs a{};
  if (const int rc = cache_of(fail, "cache append", cache, table, table_width, lengths, a.c)) return rc;
  if (batch == 0 || rows == 0) return 0;
  if (batch > 65535 || rows > kMost) return fail("cache append: %zu rows of %zu texts", rows, batch);
  if (!starts && rows != batch) return fail("cache append: %zu rows for %zu texts need starts", rows, batch);
  if (!k || !v) return fail("cache append: k and v are needed");
  const size_t s = size_of(cache->type), width = cache->heads * cache->dim;
  if (!aligned(k, s) || !aligned(v, s) || !aligned(starts, 4))
    return fail("cache append: a pointer is not aligned to its type");
  if (!stride_of(k_stride, width, &a.k_stride) || !stride_of(v_stride, width, &a.v_stride))
    return fail("cache append: strides %zu, %zu for rows of %zu values", k_stride, v_stride, width);
  a.k = k, a.v = v, a.starts = starts, a.rows = long(rows), a.batch = int(batch);
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip("cache append", on.e);
  return fail.hip("cache append", launch_kv_append(a, cache->type, hipStream_t(stream)));
}

size_t ppocr_hip_paged_attention_workspace(const ppocr_kv_cache *cache, size_t batch, size_t heads, size_t longest) {
  if (!cache || !is_real(cache->type) || !cache->heads || !cache->dim || cache->dim > 256 || !batch ||
      batch > 65535 || !heads || heads > 65535 || heads % cache->heads)
    return 0;
  if (!longest || longest > (size_t(1) << 31)) longest = size_t(1) << 31;
  const int n = paged_parts(int(batch), int(heads), int(cache->heads), cache->type, long(longest)).splits;
  return n > 1 ? batch * heads * size_t(n) * (cache->dim + 2) * sizeof(float) : 0;
}

int ppocr_hip_paged_attention(const void *q, size_t q_stride, const ppocr_kv_cache *cache, const int32_t *table,
                              size_t table_width, const int32_t *lengths, void *y, size_t y_stride, size_t batch,
                              size_t heads, float scale, size_t window, size_t sinks, size_t longest,
                              void *workspace, size_t workspace_bytes, void *stream, char *err, size_t err_len) {
  const Fail fail{err, err_len};
  PagedArgs a{};
  if (const int rc = cache_of(fail, "paged attention", cache, table, table_width, lengths, a.c)) return rc;
  if (batch == 0) return 0;
  if (batch > 65535 || !heads || heads > 65535 || heads % cache->heads)
    return fail("paged attention: %zu texts, %zu query heads over %zu", batch, heads, cache->heads);
  if (!q || !y) return fail("paged attention: q and y are needed");
  const size_t s = size_of(cache->type), width = heads * cache->dim;
  if (!aligned(q, s) || !aligned(y, s) || (workspace && !aligned(workspace, 16)))
    return fail("paged attention: a pointer is not aligned");
  if (!stride_of(q_stride, width, &a.q_stride) || !stride_of(y_stride, width, &a.y_stride))
    return fail("paged attention: strides %zu, %zu for rows of %zu values", q_stride, y_stride, width);
  if (!std::isfinite(scale)) return fail("paged attention: scale %g", double(scale));
  const size_t capacity = table_width * cache->page_size;
  if (!longest || longest > capacity) longest = capacity;
  const size_t seen = window && window < longest && sinks < longest ? window + sinks + 64 : longest;
  const PagedParts parts =
      paged_parts(int(batch), int(heads), int(cache->heads), cache->type, long(seen < longest ? seen : longest));
  int n = parts.splits;
  const size_t a_part = batch * heads * (cache->dim + 2) * sizeof(float);
  const size_t most = workspace ? workspace_bytes / a_part : 0;
  if (size_t(n) > most) n = most > 1 ? int(most) : 1;
  a.q = q, a.y = y, a.batch = int(batch), a.heads = int(heads), a.splits = n, a.each = parts.each;
  a.window = int(window < (size_t(1) << 31) - 1 ? window : 0);
  a.sinks = int(sinks < (size_t(1) << 30) ? sinks : size_t(1) << 30);
  a.scale = scale_of(scale), a.turn = scale < 0.0f;
  a.part = static_cast<float *>(workspace);
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip("paged attention", on.e);
  return fail.hip("paged attention", launch_paged_attention(a, cache->type, hipStream_t(stream)));
}

int ppocr_hip_window_attention(const void *q, size_t q_stride, const void *k, size_t k_stride, const void *v,
                               size_t v_stride, void *y, size_t y_stride, const int32_t *starts_q,
                               const int32_t *starts_k, size_t batch, size_t rows_q, size_t rows_k, size_t heads,
                               size_t kv_heads, size_t dim, int type, float scale, size_t window, size_t sinks,
                               void *stream, char *err, size_t err_len) {
  const Fail fail{err, err_len};
  if (!is_real(type)) return fail("window attention: type %d", type);
  if (!kv_heads || !heads || heads > 65535 || heads % kv_heads)
    return fail("window attention: %zu query heads over %zu", heads, kv_heads);
  if (!dim || dim > 256) return fail("window attention: heads of %zu values: 1 to 256 are taken", dim);
  if (batch == 0 || rows_q == 0) return 0;
  // (A launch has fewer than 2^24 workgroups of 32 or more queries of a head.)
  if (batch > 32768 || rows_q > size_t(1) << 24 || rows_k > kMost || heads * (rows_q / 32 + batch) >= size_t(1) << 24)
    return fail("window attention: %zu queries and %zu keys of %zu texts", rows_q, rows_k, batch);
  if (!q || !y || !starts_q || !starts_k || (rows_k && (!k || !v)))
    return fail("window attention: q, k, v, y and starts are needed");
  const size_t s = size_of(type);
  if (!aligned(q, s) || !aligned(k, s) || !aligned(v, s) || !aligned(y, s) || !aligned(starts_q, 4) ||
      !aligned(starts_k, 4))
    return fail("window attention: a pointer is not aligned to its type");
  PromptArgs a{};
  if (!stride_of(q_stride, heads * dim, &a.q_stride) || !stride_of(y_stride, heads * dim, &a.y_stride) ||
      !stride_of(k_stride, kv_heads * dim, &a.k_stride) || !stride_of(v_stride, kv_heads * dim, &a.v_stride))
    return fail("window attention: strides %zu, %zu, %zu, %zu for %zu and %zu heads of %zu", q_stride, k_stride,
                v_stride, y_stride, heads, kv_heads, dim);
  if (!std::isfinite(scale)) return fail("window attention: scale %g", double(scale));
  a.q = q, a.k = k, a.v = v, a.y = y, a.starts_q = starts_q, a.starts_k = starts_k;
  a.batch = int(batch), a.rows_q = int(rows_q), a.rows_k = int(rows_k);
  a.heads = int(heads), a.kv_heads = int(kv_heads), a.dim = int(dim);
  a.window = int(window < rows_k ? window : 0);  // (no text has more keys)
  a.sinks = int(sinks < (size_t(1) << 30) ? sinks : size_t(1) << 30);
  a.scale = scale_of(scale), a.turn = scale < 0.0f;
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip("window attention", on.e);
  return fail.hip("window attention", launch_window_attention(a, type, hipStream_t(stream)));
}

}  // extern "C"
