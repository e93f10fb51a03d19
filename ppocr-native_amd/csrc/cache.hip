// The paged cache of keys and values: appending to it (ppocr_hip_kv_append)
// and attention of one new token a text over it (ppocr_hip_paged_attention).
#include "attend.hpp"

namespace ppocr {
namespace {

// ------------------------------------------------------------------- append

// Text blockIdx.y; its new tokens are shared by the waves of gridDim.x
// workgroups, a token a wave at a time. A token's rows of k and v are read
// and written in 16-byte pieces of a head: memory bound, and at a token a
// text bound by the launch.
template <typename V>
__global__ __launch_bounds__(256) void kv_append_rows(AppendArgs a) {
  constexpr int N = 16 / sizeof(V);
  const int b = blockIdx.y, lane = threadIdx.x % 64;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / 64), waves = gridDim.x * 4;
  long first = b, last = b + 1L;
  if (a.starts) first = a.starts[b], last = a.starts[b + 1];
  const long count = last - first;
  const long end = a.c.lengths[b];
  const int pieces = (a.c.dim + N - 1) / N, all = a.c.heads * pieces;
  for (long i = wave; i < count; i += waves) {
    const long row = first + i, at = end - count + i;
    if (row < 0 || row >= a.rows || at < 0) continue;
    const long slot = at / a.c.page_size;
    if (slot >= a.c.table_width) continue;
    const int page = a.c.table[b * a.c.table_width + slot];
    if (page < 0 || page >= a.c.pages) continue;
    const long to = page * a.c.page_stride + (at - slot * a.c.page_size) * a.c.token_stride;
    const V *k = (const V *)a.k + row * a.k_stride, *v = (const V *)a.v + row * a.v_stride;
    for (int p = lane; p < all; p += 64) {
      const int head = p / pieces, d = (p - head * pieces) * N;
      const long from = (long)head * a.c.dim + d, into = to + head * a.c.head_stride + d;
      V kv[N], vv[N];
      load_n(k + from, a.c.dim - d, kv);
      load_n(v + from, a.c.dim - d, vv);
      store_n((V *)a.c.k + into, a.c.dim - d, kv);
      store_n((V *)a.c.v + into, a.c.dim - d, vv);
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

// Tiles of a part: all parts but the last that is not empty have as many.
constexpr int kLeastTiles = 4;
__device__ __forceinline__ int tiles_a_part(int tiles, int splits) {
  return max((tiles + splits - 1) / splits, kLeastTiles);
}

// Text blockIdx.z, a key head's 16 (or fewer) query heads blockIdx.y, part
// blockIdx.x of its tiles. PAGED16: pages are multiples of 16 tokens.
template <int T, int DP, bool EVEN, bool PAGED16>
__global__ __launch_bounds__(64 * kWaves) void paged_attention_parts(PagedArgs a) {
  typedef Attend<T, DP, EVEN> A;
  typedef typename A::V V;
  constexpr int K = A::KEYS;
  __shared__ float lds_o[kWaves][16][DP + 4];
  __shared__ float lds_m[kWaves][16], lds_l[kWaves][16];
  __shared__ int lds_bad;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, col = lane % 16, quarter = lane / 16;
  const int b = blockIdx.z, per = a.heads / a.c.heads, blocks = (per + 15) / 16;
  const int kv = blockIdx.y / blocks, h0 = kv * per + blockIdx.y % blocks * 16;
  const int rows = min(16, kv * per + per - h0);
  const long capacity = a.c.table_width * a.c.page_size;
  const int length = a.c.lengths[b];
  const bool too_long = length > capacity;
  const Seen s = seen_of(too_long ? 0 : length, a.window, a.sinks, K);
  const int each = tiles_a_part(s.tiles, a.splits);
  const int begin = blockIdx.x * each, end = min(begin + each, s.tiles);
  if (begin >= end && blockIdx.x) return;  // part 0 of an empty text writes its zeros
  if (threadIdx.x == 0) lds_bad = too_long;
  __syncthreads();

  A at;
  at.start((const V *)a.q + b * a.q_stride + (long)(h0 + min(col, rows - 1)) * a.c.dim, a.c.dim, quarter,
           a.turn);
  const int *table = a.c.table + b * a.c.table_width;
  const V *ck = (const V *)a.c.k + kv * a.c.head_stride, *cv = (const V *)a.c.v + kv * a.c.head_stride;
  bool bad = false;
  for (int t = begin + wave; t < end; t += kWaves) {
    const int k0 = t < s.sink_tiles ? t * K : s.first + (t - s.sink_tiles) * K;
    const bool masked = k0 + K > s.length || k0 < s.low;
    auto seen = [&](int i) { return k0 + i < s.length && (k0 + i >= s.low || k0 + i < s.sinks); };
    if constexpr (PAGED16) {
      long base[A::H];
#pragma unroll
      for (int h = 0; h < A::H; h++) {
        const int k = k0 + 16 * h;  // the half's first token; a half past the text is not looked up
        const int slot = k / a.c.page_size;
        const int page = k < s.length ? table[slot] : 0;
        base[h] = page * a.c.page_stride + (long)(k - slot * a.c.page_size) * a.c.token_stride;
        if (page < 0 || page >= a.c.pages) base[h] = -1;
        // (A half of which only unseen tokens lie in the text is not read.)
        bool any = false;
        if (base[h] < 0) {
          for (int i = 0; i < 16; i++) any = any || seen(16 * h + i);
          bad = bad || any;
        }
      }
      auto row = [&](const V *c, int i) -> const V * {
        const long o = base[i / 16];
        return o < 0 || (masked && !seen(i)) ? nullptr : c + o + (i % 16) * a.c.token_stride;
      };
      at.template tile<false>([&](int i) { return row(ck, i); }, [&](int i) { return row(cv, i); }, seen, masked, a.c.dim, a.scale,
              lane);
    } else {
      auto row = [&](const V *c, int i) -> const V * {
        if (masked && !seen(i)) return nullptr;
        const int k = k0 + i, slot = k / a.c.page_size, page = table[slot];
        if (page < 0 || page >= a.c.pages) {
          bad = true;
          return nullptr;
        }
        return c + page * a.c.page_stride + (long)(k - slot * a.c.page_size) * a.c.token_stride;
      };
      at.template tile<false>([&](int i) { return row(ck, i); }, [&](int i) { return row(cv, i); }, seen, masked, a.c.dim, a.scale,
              lane);
    }
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
      float *p = a.part + ((long)(b * a.heads + h0 + row) * a.splits + blockIdx.x) * (a.c.dim + 2);
      p[d + 2] = o;
      if (d == 0) p[0] = m, p[1] = sum;
    } else {
      ((V *)a.y)[b * a.y_stride + (long)(h0 + row) * a.c.dim + d] = Num<T>::put(sum == 0.0f ? 0.0f : o / sum);
    }
  }
}

// Joins a row's parts: a wave a head of a text.
template <int T>
__global__ __launch_bounds__(64) void paged_attention_join(PagedArgs a) {
  typedef num_t<T> V;
  const int head = blockIdx.x, b = blockIdx.y, lane = threadIdx.x;
  const int length = a.c.lengths[b];
  const Seen s = seen_of(length > a.c.table_width * a.c.page_size ? 0 : length, a.window, a.sinks,
                         T == PPOCR_F32 ? 16 : 32);
  const int each = tiles_a_part(s.tiles, a.splits);
  const int parts = max(1, (s.tiles + each - 1) / each), dim = a.c.dim;
  const float *p = a.part + (long)(b * a.heads + head) * a.splits * (dim + 2);
  float m = -INFINITY;
  for (int i = 0; i < parts; i++) m = fmaxf(m, p[(long)i * (dim + 2)]);
  float sum = 0.0f, o[4] = {0, 0, 0, 0};
  for (int i = 0; i < parts; i++) {
    const float *part = p + (long)i * (dim + 2);
    // A part's maximum is -inf only where nothing of it is seen (or a seen
    // page does not exist: then its sum is NaN, and so is the whole).
    const float f = part[0] == -INFINITY ? (part[1] == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f((part[0] - m) * a.scale);
    sum += f * part[1];
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (lane + 64 * j < dim) o[j] += f * part[2 + lane + 64 * j];
  }
  V *y = (V *)a.y + b * a.y_stride + (long)head * dim;
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (lane + 64 * j < dim) y[lane + 64 * j] = Num<T>::put(sum == 0.0f ? 0.0f : o[j] / sum);
}

template <int T, int DP>
void launch_parts(const PagedArgs &a, hipStream_t s) {
  const int per = a.heads / a.c.heads;
  const dim3 grid(a.splits, a.c.heads * ((per + 15) / 16), a.batch), block(64 * kWaves);
  const bool even = a.c.dim % 8 == 0, paged16 = a.c.page_size % 16 == 0;
  if (even && paged16)
    hipLaunchKernelGGL((paged_attention_parts<T, DP, true, true>), grid, block, 0, s, a);
  else if (even)
    hipLaunchKernelGGL((paged_attention_parts<T, DP, true, false>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((paged_attention_parts<T, DP, false, false>), grid, block, 0, s, a);
}

template <int T>
hipError_t launch_paged(const PagedArgs &a, hipStream_t s) {
  if (a.c.dim <= 64)
    launch_parts<T, 64>(a, s);
  else if (a.c.dim <= 128)
    launch_parts<T, 128>(a, s);
  else
    launch_parts<T, 256>(a, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL((paged_attention_join<T>), dim3(a.heads, a.batch), dim3(64), 0, s, a);
  return hipGetLastError();
}

}  // namespace

int paged_splits(int batch, int heads, int kv_heads, int type, long longest) {
  // Enough workgroups to fill 256 CUs four times; a part has kLeastTiles
  // tiles at least.
  const int keys = type == PPOCR_F32 ? 16 : 32, per = heads / kv_heads;
  const long groups = (long)batch * kv_heads * ((per + 15) / 16);
  const long most = (longest + (long)keys * kLeastTiles - 1) / ((long)keys * kLeastTiles);
  const long want = (1024 + groups - 1) / groups;
  const long n = want < most ? want : most;
  return n < 1 ? 1 : n > 128 ? 128 : (int)n;
}

hipError_t launch_kv_append(const AppendArgs &a, int type, hipStream_t s) {
  // Waves: one a token where the texts' shares are even, up to 4096.
  const long share = (a.rows + a.batch - 1) / a.batch;
  long x = (share + 3) / 4;
  const long most = 1024 / a.batch + 1;
  if (x > most) x = most;
  const dim3 grid(unsigned(x < 1 ? 1 : x), a.batch);
  if (type == PPOCR_F32)
    hipLaunchKernelGGL((kv_append_rows<uint32_t>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((kv_append_rows<uint16_t>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
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
