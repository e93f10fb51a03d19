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

bool select_sizes(size_t batch, size_t beams, size_t vocab, size_t keep) {
  if (!batch || batch > 65535 || !beams || beams > kMostBeams || !vocab || vocab > size_t(1) << 24 || !keep ||
      keep > kMostKeep)
    return false;
  const long rows = long(batch * beams);
  return rows * select_parts(rows, int(vocab)).parts < 1 << 24;
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
  return fail.hip(what, launch_kv4_attention(a, hipStream_t(stream)));
}

size_t ppocr_hip_beam_select_workspace(size_t batch, size_t beams, size_t vocab, size_t keep) {
  if (!select_sizes(batch, beams, vocab, keep)) return 0;
  const long rows = long(batch * beams);
  return size_t(rows) * select_parts(rows, int(vocab)).parts * (keep + 1) * 8;
}

int ppocr_hip_beam_select(const void *logits, size_t stride, const float *scores, const uint8_t *ended,
                          float *out_scores, int32_t *parents, int32_t *tokens, uint8_t *out_ended, int32_t end,
                          size_t batch, size_t beams, size_t vocab, size_t keep, int type, void *workspace,
                          size_t workspace_bytes, void *stream, char *err, size_t err_len) {
  const Fail fail{err, err_len};
  const char *what = "beam selection";
  if (!is_real(type)) return fail("%s: type %d", what, type);
  if (batch == 0) return 0;
  if (!select_sizes(batch, beams, vocab, keep))
    return fail("%s: %zu of %zu beams of %zu texts and %zu tokens (up to %d beams, %d kept, 2^24 tokens and 2^24 parts "
                "of rows are taken)", what, keep, beams, batch, vocab, kMostBeams, kMostKeep);
  if (!logits || !scores || !out_scores || !parents || !tokens)
    return fail("%s: logits, scores, out_scores, parents and tokens are needed", what);
  if (!aligned(logits, size_of(type)) || !aligned(scores, 4) || !aligned(out_scores, 4) || !aligned(parents, 4) ||
      !aligned(tokens, 4) || !aligned(workspace, 16))
    return fail("%s: a pointer is not aligned", what);
  if (end < -1 || (end >= 0 && size_t(end) >= vocab) || (ended && end < 0))
    return fail("%s: end token %d of %zu%s", what, int(end), vocab, ended ? ", and beams that have ended need one" : "");
  SelectArgs a{};
  if (!stride_of(stride, vocab, &a.stride)) return fail("%s: stride %zu for %zu tokens", what, stride, vocab);
  const size_t need = ppocr_hip_beam_select_workspace(batch, beams, vocab, keep);
  if (!workspace || workspace_bytes < need)
    return fail("%s: a workspace of %zu bytes is needed, not %zu", what, need, workspace ? workspace_bytes : 0);
  a.logits = logits, a.scores = scores, a.ended = ended, a.out_scores = out_scores;
  a.parents = parents, a.tokens = tokens, a.out_ended = out_ended, a.end = int(end);
  a.batch = int(batch), a.beams = int(beams), a.vocab = int(vocab), a.keep = int(keep);
  const SelectParts parts = select_parts(long(batch * beams), a.vocab);
  a.parts = parts.parts, a.chunk = parts.chunk;
  a.keys = static_cast<uint64_t *>(workspace);
  a.stats = reinterpret_cast<float *>(a.keys + batch * beams * size_t(a.parts) * keep);
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip(what, on.e);
  return fail.hip(what, launch_beam_select(a, type, hipStream_t(stream)));
}

int ppocr_hip_beam_reorder(const ppocr_kv_cache *caches, size_t n_caches, const ppocr_kv4_cache *caches4,
                           size_t n_caches4, const ppocr_beam_state *states, size_t n_states, const int32_t *parents,
                           const int32_t *table, int32_t *table_out, size_t table_width, const int32_t *lengths,
                           const int32_t *spare, int32_t *spare_out, size_t batch, size_t beams, void *stream,
                           char *err, size_t err_len) {
  const Fail fail{err, err_len};
  const char *what = "beam reordering";
  if ((n_caches && !caches) || (n_caches4 && !caches4) || (n_states && !states))
    return fail("%s: a list is missing", what);
  if (n_caches && n_caches4) return fail("%s: caches of one kind are taken, not %zu and %zu", what, n_caches, n_caches4);
  if (n_states > kMostStates || n_caches > 4096 || n_caches4 > 4096)
    return fail("%s: %zu states, %zu caches: %d and 4096 are taken", what, n_states, n_caches + n_caches4, kMostStates);
  if (batch == 0) return 0;
  if (!beams || beams > kMost || batch > 65535 || batch * beams > 65535)
    return fail("%s: %zu texts of %zu beams: up to 65535 beams in all are taken", what, batch, beams);
  if (!parents || !aligned(parents, 4)) return fail("%s: parents are needed, aligned to their type", what);
  ReorderArgs a{};
  a.rows = int(batch * beams), a.beams = int(beams), a.by_beams = Divide(a.beams), a.parents = parents;
  const bool paged = n_caches || n_caches4;
  // Each cache's planes, its pages and a page's tokens, twice: counted and checked, then launched.
  Plane planes[6];
  int pages = 0, tokens = 0, page_size = 0;
  auto planes_of = [&](size_t i, int &n) -> int {
    n = 0;
    if (n_caches4) {
      Kv4Args c{};
      if (const int rc = kv4_of(fail, what, caches4 + i, table, table_width, lengths, c)) return rc;
      const int at[6] = {0, c.at_ks, c.at_km, c.at_v, c.at_vs, c.at_vm};
      for (int k = 0; k < 6; k++) {
        const int bytes = k % 3 ? 2 * c.groups : 16 * c.nc;
        planes[n++] = Plane{c.data + at[k], c.page_stride, bytes, c.chunk, c.heads, bytes};
      }
      pages = c.pages, tokens = c.page_size;
    } else {
      CacheArgs c{};
      if (const int rc = cache_of(fail, what, caches + i, table, table_width, lengths, c)) return rc;
      const long size = long(size_of(caches[i].type));
      const bool rows = c.head_stride == c.dim && c.token_stride == long(c.heads) * c.dim;
      // (Where a head's tokens do not lie together, its rows are counted in 32 bits.)
      if (!rows && c.token_stride != c.dim && caches[i].page_size * caches[i].heads > (size_t(1) << 31) - 4096)
        return fail("%s: pages of %zu tokens of %zu heads, which do not lie together", what, caches[i].page_size, caches[i].heads);
      for (void *p : {c.k, c.v})
        planes[n++] = rows ? Plane{static_cast<char *>(p), c.page_stride * size, c.token_stride * size, 0, 1,
                                   int(c.token_stride * size)}
                           : Plane{static_cast<char *>(p), c.page_stride * size, c.token_stride * size,
                                   c.head_stride * size, c.heads, int(c.dim * size)};
      pages = c.pages, tokens = c.page_size;
    }
    return 0;
  };
  const size_t count = n_caches + n_caches4;
  for (size_t i = 0; i < count; i++) {
    int n;
    if (const int rc = planes_of(i, n)) return rc;
    if (i && tokens != page_size) return fail("%s: caches of pages of %d and %d tokens", what, page_size, tokens);
    // Pages that all caches have: a page's copy and its place in the tables go by the same in every launch.
    a.pages = i && a.pages < pages ? a.pages : pages, page_size = tokens;
  }
  if (paged) {
    if (!table_out || !spare || !spare_out || table_out == table || spare_out == spare)
      return fail("%s: table_out, spare and spare_out are needed, apart from table and spare", what);
    if (!aligned(table_out, 4) || !aligned(spare, 4) || !aligned(spare_out, 4))
      return fail("%s: a pointer is not aligned to its type", what);
    a.table = table, a.table_out = table_out, a.table_width = long(table_width);
    a.lengths = lengths, a.spare = spare, a.spare_out = spare_out;
    a.by_page = Divide(page_size), a.whole4 = n_caches4 != 0;
  }
  for (size_t i = 0; i < n_states; i++) {
    const ppocr_beam_state &s = states[i];
    if (!s.from || !s.to || s.from == s.to) return fail("%s: state %zu needs from and to, apart", what, i);
    const size_t from_stride = s.from_stride ? s.from_stride : s.bytes, to_stride = s.to_stride ? s.to_stride : s.bytes;
    if (s.bytes > kMostStride || from_stride < s.bytes || to_stride < s.bytes || from_stride > kMostStride ||
        to_stride > kMostStride)
      return fail("%s: state %zu of %zu bytes with strides %zu, %zu", what, i, s.bytes, s.from_stride, s.to_stride);
    a.states[i] = BeamState{static_cast<const char *>(s.from), static_cast<char *>(s.to), long(s.bytes),
                            long(from_stride), long(to_stride)};
  }
  a.n_states = int(n_states);
  size_t most = 0;
  for (size_t i = 0; i < n_states; i++) most = states[i].bytes > most ? states[i].bytes : most;
  a.state_splits = most < 65536 ? 1 : most < 1 << 20 ? int(most >> 15) : 32;
  if (!paged && !n_states) return 0;
  const OnDevice on{hipStream_t(stream)};
  if (on.e != hipSuccess) return fail.hip(what, on.e);
  // As many planes a launch as its arguments hold; the tables and states in the first.
  const int a_cache = n_caches4 ? 6 : 2;
  size_t i = 0;
  do {
    a.tables = i == 0, a.n_planes = 0;
    for (; i < count && a.n_planes + a_cache <= kMostPlanes; i++) {
      int n;
      if (const int rc = planes_of(i, n)) return rc;
      for (int k = 0; k < n; k++) a.planes[a.n_planes++] = planes[k];
    }
    // A plane's tokens in parts while there are few rows and planes.
    const long work = long(a.n_planes) * a.rows;
    a.splits = work >= 1024 || !work ? 1 : work >= 512 ? 2 : work >= 256 ? 4 : 8;
    if (const int rc = fail.hip(what, launch_beam_reorder(a, hipStream_t(stream)))) return rc;
  } while (i < count);
  return 0;
}

}  // extern "C"
