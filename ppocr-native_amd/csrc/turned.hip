// Appending keys and values to a paged cache with the rotation of keys and
// queries by their positions on the way (ppocr_hip_kv_append_rotated).
#include <algorithm>

#include "turn.hpp"

namespace ppocr {
namespace {

// A new token a workgroup: its row's loads need no more than its number, so
// they are on their way while the waves find its text, place and angles.
// Memory bound; at a token a text bound by that chain of waits.
template <int T, int N>
__global__ __launch_bounds__(512) void kv_append_turned(TurnedAppendArgs g) {
  typedef num_t<T> V;
  __shared__ v2f cs[128];
  const AppendArgs &a = g.a;
  const TurnArgs &t = g.t;
  const int heads = t.heads, kv = a.c.heads, items = (heads + 2 * kv) * g.units, half = t.rotary / 2;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    int b = (int)row;
    if (a.starts) b = last_not_past(a.batch + 1, row, [&](int i) { return (long)a.starts[i]; });
    b = __builtin_amdgcn_readfirstlane(b);

    // Item i: a unit of q's heads, then of k's, then of v's.
    V p[N], r[N];
    Unit o;
    int h;
    auto load = [&](int i) {
      h = g.by_unit(i);
      o = unit_of<N>(i - h * g.units, a.c.dim, t.rotary, t.pairs);
      const V *from = h < heads        ? (const V *)t.q + row * t.q_stride + (long)h * a.c.dim
                      : h < heads + kv ? (const V *)a.k + row * a.k_stride + (long)(h - heads) * a.c.dim
                                       : (const V *)a.v + row * a.v_stride + (long)(h - heads - kv) * a.c.dim;
      __builtin_memcpy(p, from + o.d1, sizeof p);
      __builtin_memcpy(r, from + (o.d2 < a.c.dim ? o.d2 : o.d1), sizeof r);
    };
    int i = threadIdx.x;
    if (i < items) load(i);

    if (b < 0 || b >= a.batch) continue;
    long first = b, last = b + 1L;
    if (a.starts) first = a.starts[b], last = a.starts[b + 1];
    if (row < first || row >= last) continue;
    const int end = a.c.lengths[b];
    const long at = end - (last - row);  // (below end, an int)
    long to = -1;
    if (at >= 0) {
      const int slot = a.c.by_page((int)at);
      if (slot < a.c.table_width) {
        const int page = a.c.table[b * a.c.table_width + slot];
        if (page >= 0 && page < a.c.pages)
          to = page * a.c.page_stride + (at - (long)slot * a.c.page_size) * a.c.token_stride;
      }
    }
    const double position = t.positions ? (double)t.positions[row] : (double)at;
    if (threadIdx.x < half) cs[threadIdx.x] = cosine_sine(position * (double)t.freqs[threadIdx.x]);
    __syncthreads();
    for (; i < items; i += blockDim.x) {
      if (i != threadIdx.x) load(i);
      if (h < heads + kv && o.turned) turn_unit<T, N>(p, r, cs, o, t.rotary, t.pairs);
      V *into = h < heads        ? (V *)t.q_out + row * t.q_out_stride + (long)h * a.c.dim
                : h < heads + kv ? (V *)a.c.k + to + (h - heads) * a.c.head_stride
                                 : (V *)a.c.v + to + (h - heads - kv) * a.c.head_stride;
      if (h < heads || to >= 0) {
        __builtin_memcpy(into + o.d1, p, sizeof p);
        if (o.d2 < a.c.dim) __builtin_memcpy(into + o.d2, r, sizeof r);
      }
    }
    if (gridDim.x < a.rows) __syncthreads();  // before the next token's angles
  }
}

template <int T, int N>
hipError_t launch_turned(TurnedAppendArgs a, hipStream_t s) {
  a.units = units_of(N, a.a.c.dim, a.t.rotary, a.t.pairs);
  a.by_unit = Divide(a.units);
  // As many threads as units, or as few as share them evenly; at least one an angle.
  const long items = (a.t.heads + 2L * a.a.c.heads) * a.units, rounds = (items + 511) / 512;
  const int threads = std::max(int(((items + rounds - 1) / rounds + 63) / 64 * 64), 128);
  const dim3 grid(unsigned(std::min(a.a.rows, 1L << 20))), block(threads);
  return launch_kernel(kv_append_turned<T, N>, grid, block, 0, s, a);
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
