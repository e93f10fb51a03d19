// The rotation of queries and keys by their positions, and the finding of a
// row's text, shared by the appends to the plain cache and to the one in 4 bits.
//
//   a = position freq_j,  x1' = x1 cos a - x2 sin a,  x2' = x2 cos a + x1 sin a
//
// for the dims x1 and x2 of pair j. Cosine and sine are computed in f64 and
// rounded to f32 once: an f32 angle of position 10^6 is off by 0.03, and
// results do not depend on how a library rounds its f32 functions. A token's
// angles are computed once, into LDS, for all of its heads.
#pragma once
#include <type_traits>

#include "writer.hpp"

namespace ppocr {

// Cosine and sine of a, as f32. a less the nearest multiple of pi / 2 (in two
// parts, 106 bits) is at most pi / 4, where Taylor's series to the 17th power
// are exact to 2^-55.
__device__ __forceinline__ v2f cosine_sine(double a) {
  const double n = __builtin_rint(a * 0.63661977236758134308);
  double r = fma(-n, 1.57079632679489661923, a);
  r = fma(-n, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double s = 1.0 / 355687428096000.0;
  s = fma(-s, z, 1.0 / 1307674368000.0);
  s = fma(-s, z, 1.0 / 6227020800.0);
  s = fma(-s, z, 1.0 / 39916800.0);
  s = fma(-s, z, 1.0 / 362880.0);
  s = fma(-s, z, 1.0 / 5040.0);
  s = fma(-s, z, 1.0 / 120.0);
  s = fma(-s, z, 1.0 / 6.0);
  s = fma(-s * z, r, r);
  double c = 1.0 / 20922789888000.0;
  c = fma(-c, z, 1.0 / 87178291200.0);
  c = fma(-c, z, 1.0 / 479001600.0);
  c = fma(-c, z, 1.0 / 3628800.0);
  c = fma(-c, z, 1.0 / 40320.0);
  c = fma(-c, z, 1.0 / 720.0);
  c = fma(-c, z, 1.0 / 24.0);
  c = fma(-c, z, 0.5);
  c = fma(-c, z, 1.0);
  const int turn = (int)(long)n & 3;  // quarter turns
  const float fc = (float)(turn & 1 ? s : c), fs = (float)(turn & 1 ? c : s);
  return v2f{turn == 1 || turn == 2 ? -fc : fc, turn >= 2 ? -fs : fs};
}

// Stores of values that are not looked at again soon, as a stream.
template <class V, int N>
__device__ __forceinline__ void stream_out(V *p, const V (&v)[N]) {
  constexpr int kBytes = N * sizeof(V), kWord = kBytes < 16 ? kBytes : 16;
  typedef std::conditional_t<kWord == 16, v4u, std::conditional_t<kWord == 8, v2u, std::conditional_t<kWord == 4, uint32_t, uint16_t>>> Word;
  typedef Word __attribute__((aligned(sizeof(V)))) Loose;  // (a caller's rows are aligned to their values only)
  Word w[kBytes / kWord];
  __builtin_memcpy(w, v, kBytes);
#pragma unroll
  for (int i = 0; i < kBytes / kWord; i++) __builtin_nontemporal_store(w[i], (Loose *)p + i);
}

// The last of `n` not decreasing numbers at(0), at(1), ... that is not past
// `row`, or -1: 64 of them a step, by all lanes of a wave.
template <class At>
__device__ __forceinline__ int last_not_past(int n, long row, At at) {
  const int lane = threadIdx.x % 64;
  int low = 0;
  while (true) {
    const int step = (n + 63) / 64, i = lane * step;
    const int found = __popcll(__ballot(i < n && at(low + min(i, n - 1)) <= row));
    if (found == 0) return -1;
    low += (found - 1) * step;
    if (step == 1) return low;
    n = min(step, n - (found - 1) * step);
  }
}

// Where a head's unit of two pieces lies. A unit is turned (its pieces are the
// two halves' N values each, or hold whole pairs) or copied.
struct Unit {
  int d1, d2;  // the second is not there where d2 >= dim
  int pair;    // the first pair's number
  bool turned;
};
template <int N>
__device__ __forceinline__ Unit unit_of(int u, int dim, int rotary, int pairs) {
  Unit o;
  const int half = rotary / 2;
  if (pairs && N > 1) {
    o.d1 = 2 * u * N, o.d2 = o.d1 + N, o.pair = u * N, o.turned = o.d1 < rotary;
  } else if (pairs) {
    o.d1 = 2 * u, o.d2 = o.d1 + 1, o.pair = u, o.turned = u < half;
  } else {
    o.turned = u * N < half;
    const int rest = u * N - half;
    o.d1 = o.turned ? u * N : rotary + 2 * rest;
    o.d2 = o.turned ? half + u * N : o.d1 + N;
    o.pair = u * N;
  }
  return o;
}

// Turns a unit's pieces; `cs`: the token's cosines and sines.
template <int T, int N>
__device__ __forceinline__ void turn_unit(num_t<T> (&p)[N], num_t<T> (&r)[N], const v2f *cs, const Unit &o, int rotary,
                                          int pairs) {
  typedef Num<T> F;
  if (N > 1 && pairs) {
#pragma unroll
    for (int j = 0; j + 1 < N; j += 2) {
      const v2f t = cs[o.pair + j / 2];
      const float a = F::get(p[j]), b = F::get(p[j + 1]);
      p[j] = F::put(a * t[0] - b * t[1]), p[j + 1] = F::put(b * t[0] + a * t[1]);
    }
    if (o.d2 < rotary) {
#pragma unroll
      for (int j = 0; j + 1 < N; j += 2) {
        const v2f t = cs[o.pair + N / 2 + j / 2];
        const float a = F::get(r[j]), b = F::get(r[j + 1]);
        r[j] = F::put(a * t[0] - b * t[1]), r[j + 1] = F::put(b * t[0] + a * t[1]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j++) {
      const v2f t = cs[o.pair + j];
      const float a = F::get(p[j]), b = F::get(r[j]);
      p[j] = F::put(a * t[0] - b * t[1]), r[j] = F::put(b * t[0] + a * t[1]);
    }
  }
}

// The units of a head: every value is in one. N: values a piece.
inline int units_of(int n, int dim, int rotary, int pairs) {
  if (pairs) return (dim + 2 * n - 1) / (2 * n);
  return rotary / 2 / n + (dim - rotary + 2 * n - 1) / (2 * n);
}
// Whether pieces of n values hold no part of what is turned apart.
inline bool whole_pieces(int n, int dim, int rotary, int pairs) {
  return dim % n == 0 && (pairs ? rotary % n == 0 : rotary / 2 % n == 0);
}

}  // namespace ppocr
