// Appending keys and values to a paged cache with the rotation of keys and
// queries by their positions on the way (ppocr_hip_kv_append_rotated).
#include <algorithm>

#include "turn.hpp"

namespace ppocr {
namespace {

constexpr long kNoText = -(1L << 40);  // below every token's number

// TOKENS rows a workgroup: their loads need no more than the rows' numbers, so
// they are on their way while waves find the texts, places and angles; a thread
// has the same unit of each row. Memory bound: six prompts, 5400 rows of 32 heads
// of 128 and 8 key heads in f16, 133 MB, take 25 us, 5.3 TB/s (a copy of as much
// has 5.2; 28 us without the stores as a stream). At a token a text the chain of
// waits is the whole: 64 take 4.7 us. Where a turned half is no multiple of 16
// bytes a piece is one value and a workgroup has one row: heads of 96 with 24
// turned, the same prompts, take 43 us (100 MB, 2.3 TB/s), with 96 turned 22.
template <int T, int N, int TOKENS>
__global__ __launch_bounds__(512) void kv_append_turned(TurnedAppendArgs g) {
  typedef num_t<T> V;
  __shared__ v2f cs[TOKENS][128];
  __shared__ long place[TOKENS][2];  // of a row: the token's number in its text, or -1; where it goes, or -1
  const AppendArgs &a = g.a;
  const TurnArgs &t = g.t;
  const int heads = t.heads, kv = a.c.heads, items = (heads + 2 * kv) * g.units, half = t.rotary / 2;
  const long row0 = ((long)blockIdx.y * gridDim.x + blockIdx.x) * TOKENS;

  // Item i: a unit of q's heads, then of k's, then of v's.
  V p[TOKENS][N], r[TOKENS][N];
  Unit o;
  int h;
  auto load = [&](int i) {
    h = g.by_unit(i);
    o = unit_of<N>(i - h * g.units, a.c.dim, t.rotary, t.pairs);
    const int in = h < heads ? h : h < heads + kv ? h - heads : h - heads - kv;
    const V *from = h < heads ? (const V *)t.q : h < heads + kv ? (const V *)a.k : (const V *)a.v;
    const long stride = h < heads ? t.q_stride : h < heads + kv ? a.k_stride : a.v_stride;
    const int d2 = o.d2 < a.c.dim ? o.d2 : o.d1;
#pragma unroll
    for (int j = 0; j < TOKENS; j++) {
      const V *at = from + min(row0 + j, a.rows - 1) * stride + (long)in * a.c.dim;
      __builtin_memcpy(p[j], at + o.d1, sizeof p[j]);
      __builtin_memcpy(r[j], at + d2, sizeof r[j]);
    }
  };
  load(min((int)threadIdx.x, items - 1));

  // A wave's rows: where they go.
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64;
  for (int j = wave; j < TOKENS; j += waves) {
    const long row = row0 + j;
    long at = -1, to = -1;
    int b = row < a.rows ? (int)row : -1;
    if (a.starts && b >= 0) b = last_not_past(a.batch + 1, row, [&](int i) { return (long)a.starts[i]; });
    b = __builtin_amdgcn_readfirstlane(b);
    if (b >= 0 && b < a.batch) {
      long first = b, last = b + 1L;
      if (a.starts) first = a.starts[b], last = a.starts[b + 1];
      const int end = a.c.lengths[b];
      if (row >= first && row < last) {
        at = end - (last - row);  // (below end, an int)
        const int slot = at >= 0 ? a.c.by_page((int)at) : a.c.table_width;
        if (slot < a.c.table_width) {
          const int page = a.c.table[b * a.c.table_width + slot];
          if (page >= 0 && page < a.c.pages)
            to = page * a.c.page_stride + (at - (long)slot * a.c.page_size) * a.c.token_stride;
        }
      } else {
        b = -1;
      }
    }
    if (b < 0 || b >= a.batch) at = kNoText;
    if (threadIdx.x % 64 == 0) place[j][0] = at, place[j][1] = to;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < TOKENS * half; i += blockDim.x) {
    const int j = TOKENS == 1 ? 0 : g.by_half(i), n = i - j * half;
    const double at = t.positions ? (double)t.positions[min(row0 + j, a.rows - 1)] : (double)place[j][0];
    cs[j][n] = cosine_sine(at * (double)t.freqs[n]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += blockDim.x) {
    if (i != threadIdx.x) load(i);
    const bool query = h < heads, turned = h < heads + kv && o.turned;
    V *into = query ? (V *)t.q_out + row0 * t.q_out_stride + (long)h * a.c.dim
              : h < heads + kv ? (V *)a.c.k + (h - heads) * a.c.head_stride
                               : (V *)a.c.v + (h - heads - kv) * a.c.head_stride;
#pragma unroll
    for (int j = 0; j < TOKENS; j++) {
      if (turned) turn_unit<T, N>(p[j], r[j], cs[j], o, t.rotary, t.pairs);
      const long to = query ? (place[j][0] == kNoText ? -1 : j * t.q_out_stride) : place[j][1];
      if (to >= 0) {
        stream_out(into + to + o.d1, p[j]);
        if (o.d2 < a.c.dim) stream_out(into + to + o.d2, r[j]);
      }
    }
  }
}

template <int T, int N>
hipError_t launch_turned(TurnedAppendArgs a, hipStream_t s) {
  a.units = units_of(N, a.a.c.dim, a.t.rotary, a.t.pairs);
  a.by_unit = Divide(a.units);
  // As many threads as units, or as few as share them evenly; at least one an angle.
  const long items = (a.t.heads + 2L * a.a.c.heads) * a.units, rounds = (items + 511) / 512;
  const int threads = std::max(int(((items + rounds - 1) / rounds + 63) / 64 * 64), 128);
  const dim3 block(threads);
  a.by_half = Divide(std::max(a.t.rotary / 2, 1));
  // Two rows a workgroup where that leaves every compute unit two (the six
  // prompts above: 38 us with one row, 28 with two, 30 with four, all without streams).
  const bool two = N > 1 && a.a.rows >= 4 * 256;
  const long groups = two ? (a.a.rows + 1) / 2 : a.a.rows, wide = std::min(groups, 1L << 20);
  const dim3 grid(unsigned(wide), unsigned((groups + wide - 1) / wide));
  return two ? launch_kernel(kv_append_turned<T, N, N == 1 ? 1 : 2>, grid, block, 0, s, a)
              : launch_kernel(kv_append_turned<T, N, 1>, grid, block, 0, s, a);
}

}  // namespace

hipError_t launch_kv_append_turned(const TurnedAppendArgs &a, int type, hipStream_t s) {
  const int n = type == PPOCR_F32 ? 4 : 8;
  const bool whole = whole_pieces(n, a.a.c.dim, a.t.rotary, a.t.pairs);
  switch (type) {
    case PPOCR_F32: return whole ? launch_turned<PPOCR_F32, 4>(a, s) : launch_turned<PPOCR_F32, 1>(a, s);
    case PPOCR_BF16: return whole ? launch_turned<PPOCR_BF16, 8>(a, s) : launch_turned<PPOCR_BF16, 1>(a, s);
    case PPOCR_F16: return whole ? launch_turned<PPOCR_F16, 8>(a, s) : launch_turned<PPOCR_F16, 1>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ppocr
