// The paged cache of keys and values: appending to it (ppocr_hip_kv_append)
// and attention of one new token a text over it (ppocr_hip_paged_attention).
#include <algorithm>

#include "attend.hpp"

namespace ppocr {
namespace {

// ------------------------------------------------------------------- append

// Text blockIdx.y; its new tokens are shared by the waves of gridDim.x
// workgroups, a token a wave at a time: its place is the same in all lanes,
// its rows of k and v are copied in 16-byte pieces of a head, two of each on
// their way. Memory bound: 5400 tokens of 8 heads of 128 in 16 bits (44 MB) in
// 9.2 us, 4.8 TB/s; at a token a text bound by the launch.
// WHOLE: heads are whole pieces.
template <typename V>
__device__ __forceinline__ v4u load16(const V *p) {
  v4u v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
template <typename V>
__device__ __forceinline__ void store16(V *p, v4u v) {
  __builtin_memcpy(p, &v, 16);
}

template <typename V, bool WHOLE>
__global__ __launch_bounds__(256) void kv_append_rows(AppendArgs a) {
  constexpr int N = 16 / sizeof(V);
  const int b = blockIdx.y, lane = threadIdx.x % 64;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / 64), waves = gridDim.x * 4;
  long first = b, last = b + 1L;
  if (a.starts) first = a.starts[b], last = a.starts[b + 1];
  const long count = last - first;
  const int end = a.c.lengths[b];
  const int pieces = (a.c.dim + N - 1) / N, all = a.c.heads * pieces;
  // Those that have a row and a place: starts and lengths may say anything.
  const long begin = max(max(0L, -first), count - end), stop = min(count, a.rows - first);
  for (long i = begin + wave; i < stop; i += waves) {
    const long row = first + i, at = end - count + i;
    const int slot = a.c.by_page((int)at);  // (at < end, an int)
    if (slot >= a.c.table_width) continue;
    const int page = a.c.table[b * a.c.table_width + slot];
    if (page < 0 || page >= a.c.pages) continue;
    const long to = page * a.c.page_stride + (at - (long)slot * a.c.page_size) * a.c.token_stride;
    const V *kr = (const V *)a.k + row * a.k_stride, *vr = (const V *)a.v + row * a.v_stride;
    if constexpr (WHOLE) {
      for (int p = lane; p < all; p += 128) {
        const int p2 = min(p + 64, all - 1);  // (past the last: the last again)
        const int h1 = p / pieces, d1 = (p - h1 * pieces) * N, h2 = p2 / pieces, d2 = (p2 - h2 * pieces) * N;
        const long f1 = (long)h1 * a.c.dim + d1, f2 = (long)h2 * a.c.dim + d2;
        const v4u k1 = load16(kr + f1), v1 = load16(vr + f1), k2 = load16(kr + f2), v2 = load16(vr + f2);
        const long t1 = to + h1 * a.c.head_stride + d1, t2 = to + h2 * a.c.head_stride + d2;
        store16((V *)a.c.k + t1, k1);
        store16((V *)a.c.v + t1, v1);
        if (p + 64 < all) {
          store16((V *)a.c.k + t2, k2);
          store16((V *)a.c.v + t2, v2);
        }
      }
    } else {
      for (int p = lane; p < all; p += 64) {
        const int head = p / pieces, d = (p - head * pieces) * N, left = a.c.dim - d;
        const long from = (long)head * a.c.dim + d, into = to + head * a.c.head_stride + d;
        V k[N], v[N];
        load_n(kr + from, left, k);
        load_n(vr + from, left, v);
        store_n((V *)a.c.k + into, left, k);
        store_n((V *)a.c.v + into, left, v);
      }
    }
  }
}

// ---------------------------------------------------------- decode attention

constexpr int kWaves = 4;  // waves of a workgroup, each its own tiles

// What of a text is seen, in tiles of KEYS tokens: those with sinks first,
// then those of the window, whose first starts at a multiple of KEYS (and of
// 16, so that a tile's halves lie in one page where pages are multiples of 16).
struct Seen {
  int length, low;     // tokens low .. length - 1 are in the window
  int sinks, first;    // tokens 0 .. sinks - 1 too; the window's first tile's start
  int sink_tiles, tiles;
};

__device__ __forceinline__ Seen seen_of(int length, int window, int sinks, int keys) {
  Seen s;
  s.length = max(length, 0);
  s.low = window > 0 && window < s.length ? s.length - window : 0;
  s.first = s.low / keys * keys;
  s.sinks = min(sinks, s.low);
  // A tile that holds sinks and the window's start is the window's.
  s.sink_tiles = min((s.sinks + keys - 1) / keys, s.first / keys);
  s.tiles = s.sink_tiles + (s.length - s.first + keys - 1) / keys;
  return s;
}

// Tiles of a part: as many in every text, so that workgroups have equal work
// where texts do not, unless a text is longer than was said.
__device__ __forceinline__ int tiles_a_part(int tiles, int each, int splits) {
  return max((tiles + splits - 1) / splits, each);
}

// Reading the seen keys and values bounds it: 32 texts of up to 16384 tokens, 8
// key heads of 128 in bf16 (1.08 GB), 217 us and 6 for the join, 5.0 TB/s, where
// a kernel that only reads has 6.7; the address unit is 76 % busy, as a wave's
// load of K takes 16 bytes of each of 16 rows. Each wave keeps one tile's loads
// on their way while it takes in the one before (367 us when it asked for a tile
// as it came to it), and the key heads of one part of a text run side by side, so
// that they read whole rows of a page together (264 us with the parts of one head
// side by side).
//
// Text blockIdx.z, a key head's 16 (or fewer) query heads blockIdx.x, part
// blockIdx.y of its tiles. PAGED16: pages are multiples of 16 tokens.
template <int T, int DP, int DIMS, bool PAGED16>
__global__ __launch_bounds__(64 * kWaves, (DP <= 128 ? 2 : 1)) void paged_attention_parts(PagedArgs a) {
  typedef Attend<T, DP, DIMS> A;
  typedef typename A::V V;
  constexpr int K = A::KEYS;
  __shared__ float lds_o[kWaves][16][DP + 4];
  __shared__ float lds_m[kWaves][16], lds_l[kWaves][16];
  __shared__ int lds_bad;
  const int lane = threadIdx.x % 64, col = lane % 16, quarter = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int b = blockIdx.z, per = a.heads / a.c.heads, blocks = (per + 15) / 16;
  const int kv = blockIdx.x / blocks, h0 = kv * per + blockIdx.x % blocks * 16;
  const int rows = min(16, kv * per + per - h0);
  const long capacity = a.c.table_width * a.c.page_size;
  const int length = a.c.lengths[b];
  const bool too_long = length > capacity;
  const Seen s = seen_of(too_long ? 0 : length, a.window, a.sinks, K);
  const int each = tiles_a_part(s.tiles, a.each, a.splits);
  const int begin = blockIdx.y * each, end = min(begin + each, s.tiles);
  if (begin >= end && blockIdx.y) return;  // part 0 of an empty text writes its zeros
  if (threadIdx.x == 0) lds_bad = too_long;
  __syncthreads();

  A at;
  at.start((const V *)a.q + b * a.q_stride + (long)(h0 + min(col, rows - 1)) * a.c.dim, a.c.dim, quarter,
           a.turn);
  const int *table = a.c.table + b * a.c.table_width;
  const V *ck = (const V *)a.c.k + kv * a.c.head_stride, *cv = (const V *)a.c.v + kv * a.c.head_stride;
  bool bad = false;
  auto tile_key = [&](int t) { return t < s.sink_tiles ? t * K : s.first + (t - s.sink_tiles) * K; };
  // Token k's row in its page, or -1 where that does not exist.
  auto row_of = [&](int k) -> long {
    const int slot = a.c.by_page(k), page = table[slot];
    return page < 0 || page >= a.c.pages
               ? -1
               : page * a.c.page_stride + (long)(k - slot * a.c.page_size) * a.c.token_stride;
  };

  // Tiles that are seen whole: their loads run one tile ahead.
  const int whole0 = max(begin, s.sink_tiles + (s.first < s.low ? 1 : 0));
  const int whole1 = min(end, s.sink_tiles + (s.length - s.first) / K);
  typename A::Tile ta, tb;
  // The rows of tile t: with pages of multiples of 16 tokens where its halves
  // start, the same in all lanes; else lane i's is token i's. (A page that
  // does not exist is read as page 0, and the text's result is NaN.)
  struct Rows {
    long at[PAGED16 ? A::H : 1];
  };
  auto find = [&](int t) {
    Rows r;
    const int k0 = tile_key(min(t, whole1 - 1));
    if constexpr (PAGED16) {
#pragma unroll
      for (int h = 0; h < A::H; h++) r.at[h] = row_of(k0 + 16 * h);
    } else {
      r.at[0] = row_of(k0 + lane % K);
    }
    return r;
  };
  auto load = [&](typename A::Tile &tile, Rows &r) {
#pragma unroll
    for (int h = 0; h < (PAGED16 ? A::H : 1); h++) {
      bad |= r.at[h] < 0;
      r.at[h] = max(r.at[h], 0L);
    }
    auto row = [&](const V *c, int i) -> const V * {
      if constexpr (PAGED16) return c + r.at[i / 16] + (i % 16) * a.c.token_stride;
      return c + (long)(((uint64_t)(uint32_t)__shfl((int)(r.at[0] >> 32), i) << 32) | (uint32_t)__shfl((int)r.at[0], i));
    };
    A::load(tile, [&](int i) { return row(ck, i); }, [&](int i) { return row(cv, i); }, a.c.dim, lane);
  };
  auto all = [](int) { return true; };
  int t = whole0 + wave;
  if (t < whole1) {
    Rows r = find(t);
    load(ta, r);
    r = find(t + kWaves);
    while (true) {
      if (t + kWaves < whole1) load(tb, r);
      r = find(t + 2 * kWaves);
      at.template use<false>(ta, all, all, false, a.c.dim, a.scale, lane);
      t += kWaves;
      if (t >= whole1) break;
      if (t + kWaves < whole1) load(ta, r);
      r = find(t + 2 * kWaves);
      at.template use<false>(tb, all, all, false, a.c.dim, a.scale, lane);
      t += kWaves;
      if (t >= whole1) break;
    }
  }
  // The others: sinks, and the two ends of the window.
  for (int u = begin + wave; u < end; u += kWaves) {
    if (u >= whole0 && u < whole1) continue;
    const int k0 = tile_key(u);
    auto seen = [&](int i) { return k0 + i < s.length && (k0 + i >= s.low || k0 + i < s.sinks); };
    long mine = 0;  // token lane % K's row; the cache's first where it is not seen
    if (seen(lane % K)) {
      mine = row_of(k0 + lane % K);
      bad |= mine < 0;
      mine = max(mine, 0L);
    }
    auto row = [&](const V *c, int i) -> const V * {
      const long o = (long)(((uint64_t)(uint32_t)__shfl((int)(mine >> 32), i) << 32) | (uint32_t)__shfl((int)mine, i));
      return c + o;
    };
    A::load(ta, [&](int i) { return row(ck, i); }, [&](int i) { return row(cv, i); }, a.c.dim, lane);
    at.template use<false>(ta, seen, seen, true, a.c.dim, a.scale, lane);
  }
  // The waves' parts, joined.
  if (bad) lds_bad = 1;
  const float l = at.total();
  if (quarter == 0) lds_m[wave][col] = at.m, lds_l[wave][col] = l;
#pragma unroll
  for (int e = 0; e < A::E; e++)
#pragma unroll
    for (int r = 0; r < 4; r++) lds_o[wave][col][A::E * (4 * quarter + r) + e] = at.o[e][r];
  __syncthreads();
  const bool split = a.splits > 1;
  for (int i = threadIdx.x; i < rows * DP; i += 64 * kWaves) {
    const int row = i / DP, d = i % DP;
    if (d >= a.c.dim) continue;
    float m = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) m = fmaxf(m, lds_m[w][row]);
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float f = lds_m[w][row] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((lds_m[w][row] - m) * a.scale);
      sum += f * lds_l[w][row];
      o += f * lds_o[w][row][d];
    }
    if (lds_bad) sum = o = __uint_as_float(0x7fc00000u);
    if (split) {
      float *p = a.part + (((long)b * a.heads + h0 + row) * a.splits + blockIdx.y) * (a.c.dim + 2);
      p[d + 2] = o;
      if (d == 0) p[0] = m, p[1] = sum;
    } else {
      ((V *)a.y)[b * a.y_stride + (long)(h0 + row) * a.c.dim + d] = Num<T>::put(sum == 0.0f ? 0.0f : o / sum);
    }
  }
}

// Joins a row's parts, a workgroup a head of a text: lane i of each wave has
// parts i and i + 64's factors, wave w adds parts w, w + 4, ... of them.
constexpr int kMostParts = 128;

// J: 64s of dim, rounded up to a power of two.
template <int T, int J>
__global__ __launch_bounds__(256) void paged_attention_join(PagedArgs a) {
  typedef num_t<T> V;
  __shared__ float lds_o[4][256], lds_f[kMostParts];
  const int head = blockIdx.x, b = blockIdx.y, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int length = a.c.lengths[b];
  const Seen s = seen_of(length > a.c.table_width * a.c.page_size ? 0 : length, a.window, a.sinks,
                         T == PPOCR_F32 ? 16 : 32);
  const int each = tiles_a_part(s.tiles, a.each, a.splits);
  const int parts = max(1, (s.tiles + each - 1) / each), dim = a.c.dim, row = dim + 2;
  const float *p = a.part + ((long)b * a.heads + head) * a.splits * row;
  const float m0 = lane < parts ? p[(long)lane * row] : -INFINITY, l0 = lane < parts ? p[(long)lane * row + 1] : 0.0f;
  const int far = lane + 64;
  const float m1 = far < parts ? p[(long)far * row] : -INFINITY, l1 = far < parts ? p[(long)far * row + 1] : 0.0f;
  float m = fmaxf(m0, m1);
#pragma unroll
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  // A part's maximum is -inf only where nothing of it is seen (or a seen page
  // does not exist: then its sum is NaN, and so is the whole).
  auto factor = [&](float mi, float li) {
    return mi == -INFINITY ? (li == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f((mi - m) * a.scale);
  };
  const float f0 = factor(m0, l0), f1 = factor(m1, l1);
  float sum = f0 * l0 + f1 * l1;
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  if (wave == 0) lds_f[lane] = f0, lds_f[far] = f1;
  __syncthreads();
  float o[J] = {};
#pragma unroll 8
  for (int i = wave; i < parts; i += 4) {
    const float f = lds_f[i];
#pragma unroll
    for (int j = 0; j < J; j++)  // (past dim: its last value, not kept)
      o[j] = fmaf(f, p[i * row + 2 + min(lane + 64 * j, dim - 1)], o[j]);
  }
#pragma unroll
  for (int j = 0; j < J; j++) lds_o[wave][lane + 64 * j] = o[j];
  __syncthreads();
  const int d = threadIdx.x;
  if (d < dim) {
    const float v = (lds_o[0][d] + lds_o[1][d]) + (lds_o[2][d] + lds_o[3][d]);
    ((V *)a.y)[b * a.y_stride + (long)head * dim + d] = Num<T>::put(sum == 0.0f ? 0.0f : v / sum);
  }
}

template <int T, int DP, int DIMS, bool PAGED16>
hipError_t launch_parts_of(const PagedArgs &a, hipStream_t s) {
  const int per = a.heads / a.c.heads;
  const dim3 grid(a.c.heads * ((per + 15) / 16), a.splits, a.batch), block(64 * kWaves);
  return launch_kernel(paged_attention_parts<T, DP, DIMS, PAGED16>, grid, block, 0, s, a);
}

template <int T, int DP>
hipError_t launch_whole(const PagedArgs &a, hipStream_t s) {
  if (a.c.page_size % 16 == 0) return launch_parts_of<T, DP, DIMS_WHOLE, true>(a, s);
  return launch_parts_of<T, DP, DIMS_WHOLE, false>(a, s);
}

template <int T, int DP>
hipError_t launch_parts(const PagedArgs &a, hipStream_t s) {
  if (a.c.dim == DP) return launch_whole<T, DP>(a, s);
  if (a.c.dim % 8) return launch_parts_of<T, DP, DIMS_ANY, false>(a, s);
  if (a.c.page_size % 16 == 0) return launch_parts_of<T, DP, DIMS_EVEN, true>(a, s);
  return launch_parts_of<T, DP, DIMS_EVEN, false>(a, s);
}

template <int T>
hipError_t launch_paged(const PagedArgs &a, hipStream_t s) {
  // Heads of 96 and 192 in a kernel of their own size: 32 texts of up to 8000
  // tokens, 8 key heads in bf16, 126 to 109 and 476 to 238 us against those of
  // 128 and 256, whose loads past dim are requests all the same. Other heads
  // run in the next power of two (80: 120 us, 136: 467, 200: 495 to 501), which
  // spills at 256, and those that are no multiple of 8 value by value, with two
  // tiles in registers and up to 600 of them spilled (100: 866 us, 129: 2418).
  const hipError_t e = a.c.dim <= 32    ? launch_parts<T, 32>(a, s)
                       : a.c.dim <= 64  ? launch_parts<T, 64>(a, s)
                       : a.c.dim == 96  ? launch_whole<T, 96>(a, s)
                       : a.c.dim <= 128 ? launch_parts<T, 128>(a, s)
                       : a.c.dim == 192 ? launch_whole<T, 192>(a, s)
                                        : launch_parts<T, 256>(a, s);
  if (e != hipSuccess || a.splits == 1) return e;
  const dim3 grid(a.heads, a.batch), block(256);
  if (a.c.dim <= 64) return launch_kernel(paged_attention_join<T, 1>, grid, block, 0, s, a);
  if (a.c.dim <= 128) return launch_kernel(paged_attention_join<T, 2>, grid, block, 0, s, a);
  return launch_kernel(paged_attention_join<T, 4>, grid, block, 0, s, a);
}

}  // namespace

PagedParts paged_parts(int batch, int heads, int kv_heads, int type, long longest) {
  // Parts so long that, were all texts the longest, 4096 workgroups would come
  // of it: eight times what the card holds at once, so that the last of them
  // end together; but of 16 tiles (four a wave) at least, or of four where
  // that leaves too few for the card. A text of 16 tiles is done without a
  // join.
  const int keys = type == PPOCR_F32 ? 16 : 32, per = heads / kv_heads;
  const long groups = (long)batch * kv_heads * ((per + 15) / 16), tiles = (longest + keys - 1) / keys + 2;
  long each = (tiles * groups + 4095) / 4096;
  if (each < 16) {
    const long few = (tiles * groups + 511) / 512;
    each = tiles <= 16 ? 16 : few < 4 ? 4 : few < 16 ? few : 16;
  }
  if (each < (tiles + kMostParts - 1) / kMostParts) each = (tiles + kMostParts - 1) / kMostParts;
  const long splits = (tiles + each - 1) / each;
  return {int(splits < 1 ? 1 : splits), int(each)};
}

hipError_t launch_kv_append(const AppendArgs &a, int type, hipStream_t s) {
  // A token a wave where the texts' shares are even, up to 8192 waves. (Where they
  // are not, one text's waves take many in turn: 8192 tokens of one text and one
  // each of 63 others take 54.6 us, 129 each of 64 take 12.0.)
  const long share = (a.rows + a.batch - 1) / a.batch, most = 2048 / a.batch + 1;
  const long x = std::min((share + 3) / 4, most);
  const dim3 grid(unsigned(std::max(x, 1L)), a.batch);
  const dim3 block(256);
  if (type == PPOCR_F32 && a.c.dim % 4 == 0)
    return launch_kernel(kv_append_rows<uint32_t, true>, grid, block, 0, s, a);
  if (type == PPOCR_F32) return launch_kernel(kv_append_rows<uint32_t, false>, grid, block, 0, s, a);
  if (a.c.dim % 8 == 0) return launch_kernel(kv_append_rows<uint16_t, true>, grid, block, 0, s, a);
  return launch_kernel(kv_append_rows<uint16_t, false>, grid, block, 0, s, a);
}

hipError_t launch_paged_attention(const PagedArgs &a, int type, hipStream_t s) {
  switch (type) {
    case PPOCR_F32: return launch_paged<PPOCR_F32>(a, s);
    case PPOCR_BF16: return launch_paged<PPOCR_BF16>(a, s);
    case PPOCR_F16: return launch_paged<PPOCR_F16>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ppocr
