// Attention of one new token a text over a cache in 4 bits
// (ppocr_hip_kv4_attention): the kernel, compiled for 16-bit and for 32-bit
// queries (attend4_16_*.hip, attend4_32_*.hip).
//
// A key is n s + m with codes n of 0 .. 15 and a scale and a minimum a group:
//   S[key][row] = sum over groups g of  s_g (sum of n q over g) + m_g (sum of q over g)
//   O[row][d]   = sum over keys of  (P s_g) n + P m_g
// so that the products are of codes, which f16 holds exactly, and scales and
// minima meet sums of 32 bits: nothing of the cache is rounded.
//
// Four bits are an f16 as they are: shifted to bits 6 .. 9 of a 16-bit half they
// are n 2^-18, below the smallest normal number. So eight codes of a word cost four
// masks and four shifts. The matrix cores take such numbers, but line a product's
// terms up by exponents that leave out the zeros in front, and cut them 2^-24 below
// the largest of those: n q is off by 2^-20 of the largest q, a sum of weights times
// codes by 2^-20 of the largest weight a tile, where 16-bit results keep 2^-9 or
// 2^-12 of theirs. (Without the shifts, n 2^-24, it would be 2^-14.) For f32 queries
// masks of bits 0 .. 3 and 4 .. 7, one shift and four packed products with 2^15 make
// them normal numbers, n 2^-9 and n 2^-5; the 2^4 between the two goes into q (K) or
// into the result (V). K's words have eight dims of a token; V's have two dims of four
// tokens, so that codes of a word side by side are pairs of keys, which is what the
// product over keys wants.
//
// The sixteen columns of a product are a key head's query heads, or where those
// are eight or four at most, two or four of each: then a column has every second
// or fourth 16 keys, and its own largest and sum, and a lane half or a quarter of
// the softmax's work (32 texts to 16384 tokens, four query heads a key head, 8 key
// heads of 128 in bf16 and groups of 64, 305 MB: 97 us with one column a row, 73 with
// four). What else counted there: codes read as a stream (69), parts by the lengths
// that there are, so that no workgroup is left over for a last, short round (63; 65 with
// a power of two a group, 4.7 TB/s). Of the 73 the loads alone took 66, the arithmetic
// alone 51. Now the vector units have work for 78 % of the time: 530 instructions a tile
// of 64 keys, of which 267 are masks and shifts of codes and 76 selects for the columns.
#pragma once
#include <algorithm>
#include <type_traits>

#include "parts4.hpp"

namespace ppocr {

constexpr int kWaves4 = 4;

__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
// Codes I of a word's halves (of four): n 2^-18, or as normal numbers n 2^-9, and
// n 2^-5 where I is odd.
template <bool NORMAL, int I>
__device__ __forceinline__ uint32_t codes16(uint32_t w) {
  if constexpr (NORMAL) {
    const uint32_t n = (I < 2 ? w : w >> 8) & (I % 2 ? 0x00f000f0u : 0x000f000fu);
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, n) * v2h{(_Float16)0x1p15f, (_Float16)0x1p15f});
  } else {
    return (I == 0 ? w << 6 : I == 1 ? w << 2 : I == 2 ? w >> 2 : w >> 6) & 0x03c003c0u;
  }
}
__device__ __forceinline__ uint32_t pair16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// N dwords, in the widest pieces there are.
template <int N>
struct Words {
  typedef std::conditional_t<N % 4 == 0, v4u, std::conditional_t<N % 2 == 0, v2u, uint32_t>> Piece;
  Piece w[4 * N / sizeof(Piece)];
};
template <int N>
__device__ __forceinline__ Words<N> words_at(const char *p) {
  Words<N> w;
  __builtin_memcpy(&w, p, sizeof w);
  return w;
}
// The same as a stream: codes are read once.
template <int N>
__device__ __forceinline__ void stream_in(uint32_t (&n)[N], const char *p) {
  typedef typename Words<N>::Piece Piece;
  Words<N> w;
#pragma unroll
  for (int j = 0; j < int(sizeof w / sizeof(Piece)); j++) w.w[j] = __builtin_nontemporal_load((const Piece *)p + j);
  __builtin_memcpy(n, &w, sizeof w);
}

// The state of 16 columns, a wave's worth: a lane has column lane % 16, row lane %
// (16 / CP) of the query heads, and of each 16 keys the four of quarter lane / 16.
// NC: 32s of a padded head; GC: those of a group; TWO: q in two f16 parts (23
// bits) instead of one (11 bits, all that 16-bit queries have); CP: columns a row.
template <int NC, int GC, bool TWO, int CP>
struct Rows4 {
  static constexpr int G = (NC + GC - 1) / GC, DP = 32 * NC, E = 2 * NC;
  static constexpr int H = halves4(CP), L = H / CP;  // 16s of keys a tile, and a lane
  static constexpr int UNIT = TWO ? 9 : 18;  // codes are multiplied as n 2^-UNIT
  static constexpr int FEW = H * G / 2;      // dwords of a tile's scales and minima a lane brings
  v4u q[TWO ? 2 : 1][NC];  // times 2^e of the row; TWO: odd dims 2^-4 of that
  float qs[G];             // sums of q over a group, times 2^(e - UNIT)
  v4f o[E];                // lane's column, dim 32 c + 2 (4 quarter + r) + b in o[2 c + b][r]
  float om[G];             // this lane's share of sum P m
  // Weights are 2^(S scale - base), base the largest S scale when it was set (before
  // that -2^126, below all that are finite). Their products with a group's scales of V
  // are taken times f, a power of two that brought the largest product, of all that a
  // column has seen of the group, to 2^11 or more and below 2^12: so f16's range is a
  // group's own, and neither another group's scale nor that of a token without weight
  // takes bits from it. Products of 2^-13 of the largest or more keep 23 bits, smaller
  // ones are off by 2^-36 of it. Results are scaled anew only where a weight passes
  // 2^kSlack or a product 2^15: with each new largest it would be in most tiles.
  static constexpr float kSlack = 3.0f, kMostF = 0x1p100f;
  // The base is near + far, one of which is 0. Below 2^24 S scale - near is rounded
  // once; beyond, half a step of the base can be any power of two, and S scale is
  // rounded as the base was, so that the largest has 0 and equal ones are equal.
  float l, near, far, scale, f[G];

  // Eight neighbouring dims of a row from d, as they are stored; past dim some
  // others of the row. EIGHTS: heads are of a multiple of 8 dims.
  template <bool EIGHTS, class V>
  static __device__ __forceinline__ void load8(const V *p, int d, int dim, V (&v)[8]) {
    if constexpr (EIGHTS) {
      __builtin_memcpy(v, p + min(d, dim - 8), sizeof v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = p[min(d + j, dim - 1)];
    }
  }

  template <bool EIGHTS>
  __device__ __forceinline__ void start(const void *q_, long at, int type, int dim, int quarter, float by, bool turn) {
    typedef std::conditional_t<TWO, uint32_t, uint16_t> Raw;
    constexpr Raw kSign = TWO ? 0x80000000u : 0x8000u;
    Raw raw[NC][8];
#pragma unroll
    for (int c = 0; c < NC; c++) load8<EIGHTS>((const Raw *)q_ + at, 32 * c + 8 * quarter, dim, raw[c]);
    if (dim != DP) {
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (32 * c + 8 * quarter + j >= dim) raw[c][j] = 0;
    }
    // The largest, as bits without the sign.
    uint32_t top = 0;
    if constexpr (TWO) {
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, raw[c][j] & 0x7fffffffu);
    } else {
      typedef uint16_t v2s __attribute__((ext_vector_type(2)));
      v2s two{0, 0};
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          two = __builtin_elementwise_max(two, v2s{raw[c][j], raw[c][j + 1]} & (v2s)(0x7fff));
      top = max((uint32_t)two[0], (uint32_t)two[1]);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    if constexpr (!TWO)
      top = type == PPOCR_BF16 ? top << 16 : __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)top));
    // q's largest is 2^13 or more, below 2^14 (less only where all are below f32's normal numbers).
    const int e = 13 - ((int)(top >> 23) - 127);
    // 2^100 keeps sums times it finite: at such a scale one key has all the weight. 2^-126 stands for 0, which a
    // hidden key's -infinity could not be multiplied with.
    scale = fmaxf(fminf(__builtin_ldexpf(by, UNIT - e) * 1.44269504088896340736f, 0x1p100f), 0x1p-126f);
    if (top >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u);  // an infinity or NaN in q: NaN
    if (turn) {
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) raw[c][j] ^= kSign;
    }
    // (16-bit numbers fit f16's 11 bits: rounding to 0 changes none that is not below its steps.)
    auto fill = [&](auto value) {
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float x = __builtin_ldexpf(value(raw[c][i]), TWO && i & 1 ? e - 4 : e), y = __builtin_ldexpf(value(raw[c][i + 4]), TWO && i & 1 ? e - 4 : e);
          if constexpr (TWO) {
            const v2h high = __builtin_convertvector(v2f{x, y}, v2h);
            q[0][c][i] = __builtin_bit_cast(uint32_t, high);
            q[TWO][c][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{x - (float)high[0], y - (float)high[1]}, v2h));
          } else {
            q[0][c][i] = pair16(x, y);
          }
        }
    };
    if constexpr (TWO)
      fill([](uint32_t u) { return __uint_as_float(u); });
    else if (type == PPOCR_BF16)
      fill([](uint16_t u) { return __uint_as_float((uint32_t)u << 16); });
    else
      fill([](uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); });
    const v2h one{(_Float16)0x1p-9f, (_Float16)0x1p-9f}, few_{(_Float16)0x1p-5f, (_Float16)0x1p-5f};
#pragma unroll
    for (int g = 0; g < G; g++) {
      float sum = 0.0f;
#pragma unroll
      for (int c = g * GC; c < NC && c < (g + 1) * GC; c++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int part = 0; part <= TWO; part++) {
            const uint32_t two = q[part][c][i];
            sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, two), TWO && i & 1 ? few_ : one, sum, false);
          }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      qs[g] = TWO ? sum : sum * 0x1p-9f;
      om[g] = 0.0f;
      f[g] = kMostF;
    }
#pragma unroll
    for (int i = 0; i < E; i++) o[i] = v4f{0, 0, 0, 0};
    near = l = 0.0f;
    far = -0x1p126f;
  }

  // A tile's codes: 16s of keys, of which this lane has row lane % 16 of K and the
  // four keys 4 quarter .. 4 quarter + 3 of V. (Its scales and minima, 128 H G
  // bytes, go through LDS: as loads of a lane's own they would be 4 H times as many.)
  uint32_t k[H][NC], v[H][NC];

  // Of 16 keys' 4 quarter .. + 3, for each group: plane 0 K's scales, 1 its minima, 2 and 3 V's.
  struct Few {
    _Float16 of[4 * G];
  };
  static __device__ __forceinline__ Few few_of(const char *lds, int half, int plane, int quarter) {
    Few f;
    __builtin_memcpy(f.of, __builtin_assume_aligned(lds + ((half * 4 + plane) * 4 + quarter) * 8 * G, G % 2 ? 8 : 16), 8 * G);
    return f;
  }

  // Of a column's four lanes. (Rows of 16 lanes change places between two registers:
  // a chain of waits on LDS less than shuffles, where a tile needs three of these.)
  static __device__ __forceinline__ float largest(float v) {
    auto two = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(two[0]), __uint_as_float(two[1]));
    two = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(two[0]), __uint_as_float(two[1]));
  }
  __device__ __forceinline__ float above_base(float z) const { return fmaf(z, scale, -near) - far; }
  // Raises the base to a tile's largest S; by how much, as a 2-logarithm.
  __device__ __forceinline__ float raise(float top) {
    const float base = near + far, next = fmaxf(base, largest(top) * scale), rise = next - base;
    const float shrink = __builtin_amdgcn_exp2f(-rise);
    l *= shrink;
#pragma unroll
    for (int g = 0; g < G; g++) om[g] *= shrink;
    near = fabsf(next) < 0x1p24f ? next : 0.0f;
    far = next - near;
    return rise;
  }
  // After that, or where a product passes 2^15: a group's results, and its f, which
  // goes up as they went down, but no further than the tile's products allow.
  __device__ __forceinline__ void fit(int g, float product, float rise) {
    const int up = min((int)fminf(rise, 256.0f), 100 + 127 - (int)(__float_as_uint(f[g]) >> 23));
    const float now = __builtin_ldexpf(f[g], up), most = largest(product) * now;
    const int down = most > 0x1p15f ? (int)(__float_as_uint(most) >> 23) - 126 - 12 : 0;  // most < 2^(12 + down)
    f[g] = __builtin_ldexpf(now, -down);
    const float by = __builtin_ldexpf(__builtin_amdgcn_exp2f((float)up - rise), -down);
#pragma unroll
    for (int c = g * GC; c < NC && c < (g + 1) * GC; c++) o[2 * c] *= by, o[2 * c + 1] *= by;
  }

  // Takes in the tile in k and v, its scales and minima at `lds`. seen(key of the
  // tile): whether the rows see it (asked where `masked`); next_k() and next_v()
  // ask for the next tile's as soon as this one's are used.
  template <class Seen, class NextK, class NextV>
  __device__ __forceinline__ void use(const char *lds, Seen seen, bool masked, int lane, NextK next_k, NextV next_v) {
    const int quarter = lane / 16, copy = lane % 16 / (16 / CP);
    // The products of K with q: of a lane's own 16s of keys.
    v4f s[L][G];
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
      for (int g = 0; g < G; g++) {
        v4f sum{0, 0, 0, 0};
#pragma unroll
        for (int c = g * GC; c < NC && c < (g + 1) * GC; c++) {
          const uint32_t w = k[h][c];
          const v4u a{codes16<TWO, 0>(w), codes16<TWO, 1>(w), codes16<TWO, 2>(w), codes16<TWO, 3>(w)};
          sum = mfma16(a, q[0][c], sum);
          if constexpr (TWO) sum = mfma16(a, q[1][c], sum);
        }
        if (h / L == 0) {
          s[h % L][g] = sum;
        } else {
#pragma unroll
          for (int r = 0; r < 4; r++) s[h % L][g][r] = copy == h / L ? sum[r] : s[h % L][g][r];
        }
      }
    next_k();
    Few vs[L], vm[L];
    float z[L][4];
#pragma unroll
    for (int j = 0; j < L; j++) {
      const int half = copy * L + j;
      const Few ks = few_of(lds, half, 0, quarter), km = few_of(lds, half, 1, quarter);
      vs[j] = few_of(lds, half, 2, quarter), vm[j] = few_of(lds, half, 3, quarter);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        z[j][r] = 0.0f;
#pragma unroll
        for (int g = 0; g < G; g++) {
          z[j][r] = fmaf((float)km.of[r * G + g], qs[g], z[j][r]);
          z[j][r] = fmaf((float)ks.of[r * G + g], s[j][g][r], z[j][r]);
        }
      }
      if (masked) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const bool on = seen(16 * half + 4 * quarter + r);
          z[j][r] = on ? z[j][r] : -INFINITY;
#pragma unroll
          for (int g = 0; g < G; g++) {
            vs[j].of[r * G + g] = on ? vs[j].of[r * G + g] : (_Float16)0.0f;
            vm[j].of[r * G + g] = on ? vm[j].of[r * G + g] : (_Float16)0.0f;
          }
        }
      }
    }
    float top = -INFINITY, rise = 0.0f;
#pragma unroll
    for (int j = 0; j < L; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) top = fmaxf(top, z[j][r]);
    const bool higher = __any(above_base(top) > kSlack);
    if (higher) rise = raise(top);
    float p[L][4];
#pragma unroll
    for (int j = 0; j < L; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[j][r] = __builtin_amdgcn_exp2f(above_base(z[j][r]));
        l += p[j][r];
#pragma unroll
        for (int g = 0; g < G; g++) om[g] = fmaf(p[j][r], (float)vm[j].of[r * G + g], om[g]);
      }
    // Weights times scales, 16 or 24 at a time.
    constexpr int SOME = G % 4 == 0 && L == 1 ? 4 : G % 3 == 0 ? 3 : G % 2 == 0 ? 2 : 1;
    float w[SOME][L][4];
#pragma unroll
    for (int g = 0; g < G; g++) {
      if (g % SOME == 0) {
        float product[SOME] = {};
        bool past = false;
#pragma unroll
        for (int i = 0; i < SOME; i++) {
#pragma unroll
          for (int j = 0; j < L; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              w[i][j][r] = fmaf(p[j][r], (float)vs[j].of[r * G + g + i], 0.0f);
              product[i] = fmaxf(product[i], w[i][j][r]);
            }
          past = past || product[i] * f[g + i] > 0x1p15f;
        }
        if (higher || __any(past)) {
#pragma unroll
          for (int i = 0; i < SOME; i++) fit(g + i, product[i], rise);
        }
      }
      // In two f16 parts, each rounded to the nearest: 23 bits, and off to neither side. Keys r and r + 2 of a quarter
      // side by side, as the masks leave V's; a column has its own 16s of keys and zeros for the others.
      uint32_t high[L][2], low[L][2];
#pragma unroll
      for (int j = 0; j < L; j++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const float x = w[g % SOME][j][r] * f[g], y = w[g % SOME][j][r + 2] * f[g];
          const v2h first = __builtin_convertvector(v2f{x, y}, v2h);
          const v2f rest{fmaf((float)first[0], -1.0f, x), fmaf((float)first[1], -1.0f, y)};
          high[j][r] = __builtin_bit_cast(uint32_t, first);
          low[j][r] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, v2h));
        }
#pragma unroll
      for (int h = 0; h < H; h += 2) {
        v4u a, b;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int of = (h + i / 2) / L, j = (h + i / 2) % L;
          a[i] = CP == 1 || copy == of ? high[j][i % 2] : 0u;
          b[i] = CP == 1 || copy == of ? low[j][i % 2] : 0u;
        }
#pragma unroll
        for (int c = g * GC; c < NC && c < (g + 1) * GC; c++) {
          const uint32_t w0 = v[h][c], w1 = v[h + 1][c];
          const v4u even{codes16<TWO, 0>(w0), codes16<TWO, 2>(w0), codes16<TWO, 0>(w1), codes16<TWO, 2>(w1)};
          const v4u odd{codes16<TWO, 1>(w0), codes16<TWO, 3>(w0), codes16<TWO, 1>(w1), codes16<TWO, 3>(w1)};
          o[2 * c] = mfma16(even, b, o[2 * c]);
          o[2 * c + 1] = mfma16(odd, b, o[2 * c + 1]);
          o[2 * c] = mfma16(even, a, o[2 * c]);
          o[2 * c + 1] = mfma16(odd, a, o[2 * c + 1]);
        }
      }
    }
    next_v();
  }

  // The column's whole sum, and its sums of P m, in all four quarters.
  __device__ __forceinline__ float total() {
#pragma unroll
    for (int g = 0; g < G; g++) {
      om[g] += __shfl_xor(om[g], 16);
      om[g] += __shfl_xor(om[g], 32);
    }
    const float t = l + __shfl_xor(l, 16);
    return t + __shfl_xor(t, 32);
  }
};

// Waves that a SIMD's 512 registers a lane hold without spilling: results, q,
// codes, the tile's products, scales and minima, and some 55 others. (Four columns
// of 16-bit queries over one group spill with four waves: the texts above, with heads
// of 64 and of 96, take 47 and 57 us so, and 45 and 53 with three. With more groups,
// f32 queries or fewer columns four waves are the faster by 1 to 5 %.)
template <int NC, int GC, bool TWO, int CP>
constexpr int waves_a_simd4() {
  typedef Rows4<NC, GC, TWO, CP> A;
  constexpr int n = NC * (8 + (TWO ? 8 : 4) + 2 * A::H) + A::FEW + A::G * (4 * A::L + 8 * A::L) + 55;
  return n <= (A::G == 1 && CP == 4 && !TWO ? 105 : 130) ? 4 : n <= 170 ? 3 : n <= 250 ? 2 : 1;
}

// A key head's 16 (or fewer) query heads blockIdx.x, text blockIdx.z and part
// blockIdx.y of its tiles, or the parts' number blockIdx.y where there are
// `pieces`; a tile a wave at a time. EIGHTS: heads are of a multiple of 8 dims.
template <int NC, int GC, bool TWO, int CP, bool EIGHTS>
__global__ __launch_bounds__(64 * kWaves4, (waves_a_simd4<NC, GC, TWO, CP>())) void kv4_attention_parts(Attend4Args a) {
  typedef Rows4<NC, GC, TWO, CP> A;
  constexpr int DP = A::DP, H = A::H, KEYS = 16 * H, R = 16 / CP, kTable = 64 / H;
  __shared__ float lds_o[kWaves4][16][DP + 4];
  __shared__ float lds_b[kWaves4][16], lds_l[kWaves4][16];
  __shared__ __attribute__((aligned(16))) char lds_few[kWaves4][256 * A::FEW];
  __shared__ int lds_bad;
  const int lane = threadIdx.x % 64, col = lane % 16, quarter = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int wanted = each4(a, KEYS);
  int b = blockIdx.z, part = blockIdx.y;
  if (a.pieces) {
    const Piece4 piece = piece4(a, KEYS, wanted, part);
    if (piece.b < 0) return;
    b = piece.b, part = piece.part;
  }
  const int per = a.heads / a.c.heads, blocks = (per + 15) / 16;
  const int kv = blockIdx.x / blocks, h0 = kv * per + blockIdx.x % blocks * 16;
  const int rows = min(16, kv * per + per - h0);
  const int length = a.c.lengths[b];
  const bool too_long = length > a.c.table_width * a.c.page_size;
  const Seen s = seen_of(too_long ? 0 : length, a.window, a.sinks, KEYS);
  const int each = tiles_a_part(s.tiles, wanted, a.splits);
  const int begin = part * each, end = min(begin + each, s.tiles);
  if (begin >= end && part) return;  // part 0 of an empty text writes its zeros
  if (threadIdx.x == 0) lds_bad = too_long;
  __syncthreads();

  A at;
  at.template start<EIGHTS>(a.q, b * a.q_stride + (long)(h0 + min(col % R, rows - 1)) * a.c.dim, a.type, a.c.dim, quarter,
                            a.scale, a.turn);
  const int *table = a.c.table + b * a.c.table_width;
  const char *data = a.c.data + (long)kv * a.c.chunk;
  bool bad = false;
  auto tile_key = [&](int t) { return t < s.sink_tiles ? t * KEYS : s.first + (t - s.sink_tiles) * KEYS; };
  const int whole0 = s.sink_tiles + (s.first < s.low ? 1 : 0), whole1 = s.sink_tiles + (s.length - s.first) / KEYS;
  const uint32_t k_at = (col * 4 + quarter) * 4 * NC, v_at = a.c.at_v + lane * 4 * NC;
  // This lane's share of a tile's scales and minima: of 16 keys, a plane, a piece.
  const int half = lane / kTable, plane = lane / (16 / H) % 4;
  const uint32_t few_at = (plane == 0 ? a.c.at_ks : plane == 1 ? a.c.at_km : plane == 2 ? a.c.at_vs : a.c.at_vm) +
                          lane % (16 / H) * 4 * A::FEW;
  char *few = lds_few[wave];
  // A wave takes each fourth tile. Of its next ones, each lane finds where 16
  // keys lie: the page's offset and the first token's slot in it. (A page that
  // does not exist is read as page 0, and the text's result is NaN.)
  for (int t0 = begin + wave; t0 < end; t0 += kTable * kWaves4) {
    long my_page = 0;
    int my_slot = 0;
    {
      const int t = t0 + lane / H * kWaves4, k = tile_key(min(t, end - 1)) + lane % H * 16;
      // Of 16 neighbours some is seen if one is below the length and above the window's start, or below the sinks' end.
      if (t < end && k < s.length && (k + 15 >= s.low || k < s.sinks)) {
        const int n = a.c.by_page(k), page = table[n];
        if (page >= 0 && page < a.c.pages)
          my_page = page * a.c.page_stride, my_slot = k - n * a.c.page_size;
        else
          bad = true;
      }
    }
    auto page_of = [&](int i) {
      return data + (long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(my_page >> 32), i) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)my_page, i));
    };
    auto slot_of = [&](int i) { return __builtin_amdgcn_readlane(my_slot, i); };
    auto load_codes = [&](uint32_t (&n)[H][NC], int i, uint32_t at_) {
#pragma unroll
      for (int h = 0; h < H; h++)
        stream_in(n[h], page_of(H * i + h) + slot_of(H * i + h) * 16 * NC + at_);
    };
    // A lane's share of a tile's scales and minima.
    auto load_few = [&](int i) {
      const int from = H * i + half;
      const long o = (long)((uint64_t)(uint32_t)__shfl((int)(my_page >> 32), from) << 32 | (uint32_t)__shfl((int)my_page, from));
      return words_at<A::FEW>(data + o + (uint32_t)(__shfl(my_slot, from) * 2 * A::G) + few_at);
    };
    auto put_few = [&](const Words<A::FEW> &w) {
      __builtin_amdgcn_wave_barrier();  // (a wave's LDS operations are done in order)
      *(Words<A::FEW> *)(few + lane * 4 * A::FEW) = w;
      __builtin_amdgcn_wave_barrier();
    };
    const int n = min((end - t0 + kWaves4 - 1) / kWaves4, kTable);
    Words<A::FEW> share = load_few(0);
    load_codes(at.k, 0, k_at);
    load_codes(at.v, 0, v_at);
    put_few(share);
    for (int i = 0; i < n; i++) {
      const int next = min(i + 1, n - 1);  // (the last one again, rather than loads behind a branch, which would be waited for)
      share = load_few(next);
      const int t = t0 + i * kWaves4, k = tile_key(t);
      at.use(few, [&](int j) { return k + j < s.length && (k + j >= s.low || k + j < s.sinks); }, t < whole0 || t >= whole1,
             lane, [&] { load_codes(at.k, next, k_at); },
             [&] {
               put_few(share);
               load_codes(at.v, next, v_at);
             });
    }
  }
  // The waves' columns, joined.
  if (bad) lds_bad = 1;
  const float l = at.total();
  if (quarter == 0) lds_b[wave][col] = at.near + at.far, lds_l[wave][col] = l;
#pragma unroll
  for (int c = 0; c < NC; c++)
#pragma unroll
    for (int odd = 0; odd < 2; odd++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        lds_o[wave][col][32 * c + 2 * (4 * quarter + r) + odd] =
            fmaf(at.o[2 * c + odd][r], (TWO ? (odd ? 0x1p5f : 0x1p9f) : 0x1p18f) / at.f[c / GC], at.om[c / GC]);
  __syncthreads();
  // A column's factor, and a row's sum: a wave's columns in 16 neighbouring lanes.
  {
    const int row = col % R;
    float bw = lane < 16 * kWaves4 ? lds_b[lane / 16][col] : -INFINITY, base_ = bw;
    auto all = [&](float v, auto join) {
#pragma unroll
      for (int o = R; o < 64; o *= 2) v = join(v, __shfl_xor(v, o));
      return v;
    };
    base_ = all(base_, [](float x, float y) { return fmaxf(x, y); });
    const float f = __builtin_amdgcn_exp2f(bw - base_);
    const float sum = all(f * lds_l[lane / 16][col], [](float x, float y) { return x + y; });
    __syncthreads();
    if (wave == 0) {
      lds_b[lane / 16][col] = f;
      if (lane < R) lds_l[0][row] = lds_bad ? __uint_as_float(0x7fc00000u) : sum, lds_l[1][row] = base_;
    }
    __syncthreads();
  }
  const bool split = a.splits > 1;
  for (int i = threadIdx.x; i < rows * DP; i += 64 * kWaves4) {
    const int row = i / DP, d = i % DP;
    if (d >= a.c.dim) continue;
    const float sum = lds_l[0][row];
    float o = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves4 * CP; w++)
      o = fmaf(lds_b[w / CP][w % CP * R + row], lds_o[w / CP][w % CP * R + row][d], o);
    if (split) {
      float *p = a.part + (((long)b * a.heads + h0 + row) * a.splits + part) * (a.c.dim + 2);
      p[d + 2] = o;
      if (d == 0) p[0] = lds_l[1][row], p[1] = sum;
    } else {
      put_at(a.y, b * a.y_stride + (long)(h0 + row) * a.c.dim + d, a.type, sum == 0.0f ? 0.0f : o / sum);
    }
  }
}

// As many parts as the card holds workgroups at once, or a multiple of it of two
// and a half parts a text, less the half part a text that their lengths leave; with
// many texts and heads, or few workgroups in all, as the host chose.
template <int NC, int GC, bool TWO, int CP>
hipError_t launch_parts4(Attend4Args &a, hipStream_t s) {
  typedef Rows4<NC, GC, TWO, CP> A;
  constexpr int kLds = kWaves4 * (16 * (A::DP + 4) * 4 + 256 * A::FEW + 128) + 64;
  constexpr int kHeld = 256 * std::min(waves_a_simd4<NC, GC, TWO, CP>(), (160 << 10) / kLds);
  const int per = a.heads / a.c.heads, groups = a.c.heads * ((per + 15) / 16);
  if (a.splits > 1 && long(a.batch) * groups <= kShared4 && long(a.splits) * a.batch * groups > kHeld) {
    const long wanted = (5L * a.batch * groups + 1) / 2, times = std::max((wanted + kHeld - 1) / kHeld, 1L);
    a.pieces = int(std::max(times * kHeld / groups - a.batch / 2, 1L));
  }
  const dim3 grid = a.pieces ? dim3(groups, a.pieces + a.batch + 1) : dim3(groups, a.splits, a.batch), block(64 * kWaves4);
  if (a.c.dim % 8 == 0) return launch_kernel(kv4_attention_parts<NC, GC, TWO, CP, true>, grid, block, 0, s, a);
  return launch_kernel(kv4_attention_parts<NC, GC, TWO, CP, false>, grid, block, 0, s, a);
}

// Groups of a whole head, of 32 and of 64 (where a head has more than one).
template <int NC, bool TWO, int CP>
hipError_t launch_groups4(Attend4Args &a, hipStream_t s) {
  if constexpr (NC > 1) {
    if (a.c.group == 32) return launch_parts4<NC, 1, TWO, CP>(a, s);
  }
  if constexpr (NC > 2) {
    if (a.c.group == 64) return launch_parts4<NC, 2, TWO, CP>(a, s);
  }
  return launch_parts4<NC, NC, TWO, CP>(a, s);
}

template <bool TWO, int CP>
hipError_t launch_attention4(Attend4Args &a, hipStream_t s) {
  switch (a.c.nc) {
    case 1: return launch_groups4<1, TWO, CP>(a, s);
    case 2: return launch_groups4<2, TWO, CP>(a, s);
    case 3: return launch_groups4<3, TWO, CP>(a, s);
    case 4: return launch_groups4<4, TWO, CP>(a, s);
    case 6: return launch_groups4<6, TWO, CP>(a, s);
    case 8: return launch_groups4<8, TWO, CP>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ppocr
