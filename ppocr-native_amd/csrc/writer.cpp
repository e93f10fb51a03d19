// The C entries of what a text decoder writes with (include/ppocr_hip.h): the
// append with the rotation of positions, the cache in 4 bits, beam search.
// Checks of the arguments, the stream's device, and the launch. Nothing here
// allocates, waits or throws.
#include "writer.hpp"

#include "entry.hpp"

namespace {

// A 4-bit cache's geometry: 32s of a padded head, values a group (256: a whole
// head) and groups. False where it is refused.
bool kv4_sizes(size_t page_size, size_t heads, size_t dim, size_t group, Kv4Args &c) {
  if (!page_size || page_size % 16 || page_size > size_t(1) << 20 || !heads || heads > 65535 || !dim || dim > 256 ||
      (group != 0 && group != 32 && group != 64))
    return false;
  const int nc = int((dim + 31) / 32);
  c.nc = nc == 5 ? 6 : nc == 7 ? 8 : nc;
  c.group = group == 0 || int(group) >= 32 * c.nc ? 256 : int(group);
  c.groups = (32 * c.nc + c.group - 1) / c.group;
  c.page_size = int(page_size), c.heads = int(heads), c.dim = int(dim);
  const int codes = c.page_size * 16 * c.nc, few = c.page_size * 2 * c.groups;
  c.at_ks = codes, c.at_km = codes + few, c.at_v = codes + 2 * few;
  c.at_vs = c.at_v + codes, c.at_vm = c.at_vs + few, c.chunk = c.at_vm + few;
  return true;
}

int kv4_of(const Fail &fail, const char *what, const ppocr_kv4_cache *k, const int32_t *table, size_t table_width,
           const int32_t *lengths, Kv4Args &c) {
  if (!k || !k->data || !table || !lengths) return fail("%s: no cache, page table or lengths", what);
  if (!kv4_sizes(k->page_size, k->heads, k->dim, k->group, c))
    return fail("%s: pages of %zu tokens (a multiple of 16 up to 2^20 is taken), %zu heads of %zu values (1 to 256) in "
                "groups of %zu (0, a whole head, 32 or 64)", what, k->page_size, k->heads, k->dim, k->group);
  if (!k->pages || k->pages > kMost) return fail("%s: a cache of %zu pages", what, k->pages);
  if (!aligned(k->data, 16) || !aligned(table, 4) || !aligned(lengths, 4))
    return fail("%s: a pointer is not aligned (a 4-bit cache to 16 bytes)", what);
  const size_t page = size_t(c.chunk) * k->heads;
  c.page_stride = long(k->page_stride ? k->page_stride : page);
  if (size_t(c.page_stride) < page || c.page_stride % 16 || size_t(c.page_stride) > kMostStride)
    return fail("%s: pages of %zu bytes, %zu apart (a multiple of 16 is taken)", what, page, k->page_stride);
  if (!table_width || table_width > kMost || table_width * k->page_size > (size_t(1) << 31) - 4096)
    return fail("%s: a page table of %zu pages of %zu tokens a text", what, table_width, k->page_size);
  c.data = static_cast<char *>(k->data), c.pages = int(k->pages);
  c.by_page = Divide(c.page_size);
  c.table = table, c.table_width = long(table_width), c.lengths = lengths;
  return 0;
}

// The rows of keys and values of a call, and the queries and rotation with them.
int rows_of(const Fail &fail, const char *what, const void *k, const void *v, size_t *k_stride, size_t *v_stride,
            size_t width, int type, const int32_t *starts, size_t batch, size_t rows) {
  if (!is_real(type)) return fail("%s: type %d", what, type);
  if (batch > 65535 || rows > kMost) return fail("%s: %zu rows of %zu texts", what, rows, batch);
  if (!starts && rows != batch) return fail("%s: %zu rows for %zu texts need starts", what, rows, batch);
  if (!k || !v) return fail("%s: k and v are needed", what);
  if (!aligned(k, size_of(type)) || !aligned(v, size_of(type)) || !aligned(starts, 4))
    return fail("%s: a pointer is not aligned to its type", what);
  long a, b;
  if (!stride_of(*k_stride, width, &a) || !stride_of(*v_stride, width, &b))
    return fail("%s: strides %zu, %zu for rows of %zu values", what, *k_stride, *v_stride, width);
  *k_stride = size_t(a), *v_stride = size_t(b);
  return 0;
}

int turn_of(const Fail &fail, const char *what, const void *q, size_t q_stride, void *q_out, size_t q_out_stride,
            size_t heads, const float *freqs, const int32_t *positions, size_t rotary, int pairs, size_t dim,
            size_t kv_heads, int type, TurnArgs &t) {
  if (rotary % 2 || rotary > dim) return fail("%s: %zu dims of heads of %zu turned", what, rotary, dim);
  if (rotary && !freqs) return fail("%s: %zu dims turned without frequencies", what, rotary);
  if ((q && (!heads || heads > 65535)) || (!q && heads) || !q != !q_out)
    return fail("%s: %zu query heads, and q and q_out are given together or not at all", what, heads);
  if (q && heads % kv_heads) return fail("%s: %zu query heads over %zu", what, heads, kv_heads);
  if (!aligned(q, size_of(type)) || !aligned(q_out, size_of(type)) || !aligned(freqs, 4) || !aligned(positions, 4))
    return fail("%s: a pointer is not aligned to its type", what);
  if (!stride_of(q_stride, heads * dim, &t.q_stride) || !stride_of(q_out_stride, heads * dim, &t.q_out_stride))
    return fail("%s: strides %zu, %zu for rows of %zu query values", what, q_stride, q_out_stride, heads * dim);
  t.q = q, t.q_out = q_out, t.heads = int(heads), t.freqs = freqs, t.positions = positions;
  t.rotary = int(rotary), t.pairs = pairs != 0;
  return 0;
}

}  // namespace

extern "C" {

int ppocr_hip_kv_append_rotated(const void *q, size_t q_stride, void *q_out, size_t q_out_stride, size_t heads,
                                const void *k, size_t k_stride, const void *v, size_t v_stride,
                                const ppocr_kv_cache *cache, const int32_t *table, size_t table_width,
                                const int32_t *lengths, const int32_t *starts, const int32_t *positions,
                                const float *freqs, size_t rotary, int pairs, size_t batch, size_t rows, void *stream,
                                char *err, size_t err_len) {
  const Fail fail{err, err_len};
  const char *what = "rotated append";
  TurnedAppendArgs a{};
  if (const int rc = cache_of(fail, what, cache, table, table_width, lengths, a.a.c)) return rc;
  if (const int rc = turn_of(fail, what, q, q_stride, q_out, q_out_stride, heads, freqs, positions, rotary, pairs,
                             cache->dim, cache->heads, cache->type, a.t))
    return rc;
  if (batch == 0 || rows == 0) return 0;
  if (const int rc = rows_of(fail, what, k, v, &k_stride, &v_stride, cache->heads * cache->dim, cache->type, starts,
                             batch, rows))
    return rc;
  a.a.k = k, a.a.v = v, a.a.k_stride = long(k_stride), a.a.v_stride = long(v_stride);
  a.a.starts = starts, a.a.rows = long(rows), a.a.batch = int(batch);
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip(what, on.e);
  return fail.hip(what, launch_kv_append_turned(a, cache->type, hipStream_t(stream)));
}

size_t ppocr_hip_kv4_page_bytes(size_t page_size, size_t heads, size_t dim, size_t group) {
  Kv4Args c{};
  return kv4_sizes(page_size, heads, dim, group, c) ? heads * size_t(c.chunk) : 0;
}

int ppocr_hip_kv4_append(const void *q, size_t q_stride, void *q_out, size_t q_out_stride, size_t heads, const void *k,
                         size_t k_stride, const void *v, size_t v_stride, const ppocr_kv4_cache *cache,
                         const int32_t *table, size_t table_width, const int32_t *lengths, const int32_t *starts,
                         const int32_t *positions, const float *freqs, size_t rotary, int pairs, size_t batch,
                         size_t rows, int type, void *stream, char *err, size_t err_len) {
  const Fail fail{err, err_len};
  const char *what = "4-bit append";
  Append4Args a{};
  if (const int rc = kv4_of(fail, what, cache, table, table_width, lengths, a.c)) return rc;
  if (!is_real(type)) return fail("%s: type %d", what, type);
  if (const int rc = turn_of(fail, what, q, q_stride, q_out, q_out_stride, heads, freqs, positions, rotary, pairs,
                             cache->dim, cache->heads, type, a.t))
    return rc;
  if (batch == 0 || rows == 0) return 0;
  if (const int rc = rows_of(fail, what, k, v, &k_stride, &v_stride, cache->heads * cache->dim, type, starts, batch,
                             rows))
    return rc;
  a.k = k, a.v = v, a.k_stride = long(k_stride), a.v_stride = long(v_stride);
  a.starts = starts, a.rows = long(rows), a.batch = int(batch);
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip(what, on.e);
  return fail.hip(what, launch_kv4_append(a, type, hipStream_t(stream)));
}

int ppocr_hip_kv4_read(void *k, size_t k_stride, void *v, size_t v_stride, const ppocr_kv4_cache *cache,
                       const int32_t *table, size_t table_width, const int32_t *lengths, const int32_t *starts,
                       size_t batch, size_t rows, int type, void *stream, char *err, size_t err_len) {
  const Fail fail{err, err_len};
  const char *what = "4-bit read";
  Read4Args a{};
  if (const int rc = kv4_of(fail, what, cache, table, table_width, lengths, a.c)) return rc;
  if (!is_real(type)) return fail("%s: type %d", what, type);
  if (batch == 0 || rows == 0) return 0;
  if (const int rc = rows_of(fail, what, k, v, &k_stride, &v_stride, cache->heads * cache->dim, type, starts, batch,
                             rows))
    return rc;
  a.k = k, a.v = v, a.k_stride = long(k_stride), a.v_stride = long(v_stride);
  a.starts = starts, a.rows = long(rows), a.batch = int(batch);
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip(what, on.e);
  return fail.hip(what, launch_kv4_read(a, type, hipStream_t(stream)));
}

size_t ppocr_hip_kv4_attention_workspace(const ppocr_kv4_cache *cache, size_t batch, size_t heads, size_t longest) {
  if (!cache || !cache->heads || cache->heads > 65535 || !cache->dim || cache->dim > 256 || !batch || batch > 65535 ||
      !heads || heads > 65535 || heads % cache->heads)
    return 0;
  if (!longest || longest > (size_t(1) << 31)) longest = size_t(1) << 31;
  const int n = kv4_parts(int(batch), int(heads), int(cache->heads), long(longest)).splits;
  return n > 1 ? batch * heads * size_t(n) * (cache->dim + 2) * sizeof(float) : 0;
}

int ppocr_hip_kv4_attention(const void *q, size_t q_stride, const ppocr_kv4_cache *cache, const int32_t *table,
                            size_t table_width, const int32_t *lengths, void *y, size_t y_stride, size_t batch,
                            size_t heads, int type, float scale, size_t window, size_t sinks, size_t longest,
                            void *workspace, size_t workspace_bytes, void *stream, char *err, size_t err_len) {
  const Fail fail{err, err_len};
  const char *what = "4-bit attention";
  Attend4Args a{};
  if (const int rc = kv4_of(fail, what, cache, table, table_width, lengths, a.c)) return rc;
  if (!is_real(type)) return fail("%s: type %d", what, type);
  if (batch == 0) return 0;
  if (batch > 65535 || !heads || heads > 65535 || heads % cache->heads)
    return fail("%s: %zu texts, %zu query heads over %zu", what, batch, heads, cache->heads);
  if (!q || !y) return fail("%s: q and y are needed", what);
  const size_t s = size_of(type), width = heads * cache->dim;
  if (!aligned(q, s) || !aligned(y, s) || !aligned(workspace, 16)) return fail("%s: a pointer is not aligned", what);
  if (!stride_of(q_stride, width, &a.q_stride) || !stride_of(y_stride, width, &a.y_stride))
    return fail("%s: strides %zu, %zu for rows of %zu values", what, q_stride, y_stride, width);
  if (!std::isfinite(scale)) return fail("%s: scale %g", what, double(scale));
  const size_t capacity = table_width * cache->page_size;
  if (!longest || longest > capacity) longest = capacity;
  const size_t seen = window && window < longest && sinks < longest ? window + sinks + 64 : longest;
  const PagedParts parts =
      kv4_parts(int(batch), int(heads), int(cache->heads), long(seen < longest ? seen : longest));
  int n = parts.splits;
  const size_t a_part = batch * heads * (cache->dim + 2) * sizeof(float);
  const size_t most = workspace ? workspace_bytes / a_part : 0;
  if (size_t(n) > most) n = most > 1 ? int(most) : 1;
  a.q = q, a.y = y, a.type = type, a.batch = int(batch), a.heads = int(heads), a.splits = n, a.each = parts.each;
  a.window = int(window < (size_t(1) << 31) - 1 ? window : 0);
  a.sinks = int(sinks < (size_t(1) << 30) ? sinks : size_t(1) << 30);
  a.scale = std::fabs(scale), a.turn = scale < 0.0f;
  a.part = static_cast<float *>(workspace);
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip(what, on.e);
  return fail.hip(what, type == PPOCR_F32 ? launch_kv4_attention_32(a, hipStream_t(stream))
                                          : launch_kv4_attention_16(a, hipStream_t(stream)));
}

}  // extern "C"
