// Attention of one new token a text over a cache in 4 bits
// (ppocr_hip_kv4_attention): the kernel, compiled for 16-bit and for 32-bit
// queries (attend4_16.hip, attend4_32.hip).
//
// A key is n s + m with codes n of 0 .. 15 and a scale and a minimum a group:
//   S[key][row] = sum over groups g of  s_g (sum of n q over g) + m_g (sum of q over g)
//   O[row][d]   = sum over keys of  (P s_g) n + P m_g
// so that the products are of codes, which f16 holds exactly, and scales and
// minima meet sums of 32 bits: nothing of the cache is rounded.
//
// Four bits are an f16 as they are: bits 0 .. 3 of a 16-bit half are n 2^-24,
// bits 4 .. 7 are n 2^-20, both below the smallest normal number. So eight codes
// of a word cost four masks and one shift, and four packed products with 2^15
// to make them normal numbers, n 2^-9 and n 2^-5: the matrix cores take the
// others too, but line products up by exponents that leave out the zeros in
// front, and cut them 2^-20 of the largest from the top (4 % faster, and 16-bit
// results hardly show it; f32 ones were off by 2^-13). The 2^4 between the two
// goes into q (K) or into the result (V). K's words have eight dims of a token;
// V's have two dims of four tokens, so that the same masks give pairs of keys,
// which is what the product over keys wants.
#pragma once
#include "seen.hpp"
#include "writer.hpp"

namespace ppocr {

constexpr int kWaves4 = 4, kKeys4 = 32;

__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
// The codes that a mask leaves, as normal numbers.
__device__ __forceinline__ uint32_t codes16(uint32_t w, uint32_t mask) {
  const uint32_t n = w & mask;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, n) * v2h{(_Float16)0x1p15f, (_Float16)0x1p15f});
}
__device__ __forceinline__ uint32_t pair16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
__device__ __forceinline__ void put_at(void *p, long i, int type, float v) {
  if (type == PPOCR_F32)
    ((float *)p)[i] = v;
  else if (type == PPOCR_BF16)
    ((__bf16 *)p)[i] = (__bf16)v;
  else
    ((_Float16 *)p)[i] = (_Float16)v;
}

// The state of 16 rows (query heads of a key head), a wave's worth: a lane has
// row lane % 16, quarter lane / 16 of the keys. NC: 32s of a padded head; GC:
// those of a group; TWO: q in two f16 parts (22 bits) instead of one (11 bits,
// all that 16-bit queries have).
template <int NC, int GC, bool TWO>
struct Rows4 {
  static constexpr int G = (NC + GC - 1) / GC, DP = 32 * NC, E = 2 * NC;
  v4u q[TWO ? 2 : 1][NC];  // times 2^e of the row, odd dims 2^-4 of that
  float qs[G];             // sums of q over a group, times 2^(e - 9)
  v4f o[E];                // lane's row, dim 32 c + 2 (4 quarter + r) + b in o[2 c + b][r]
  float om[G];             // this lane's share of sum P m
  // Weights are 2^(S scale - base); base is the largest S scale less `up`, and
  // 2^up times any scale of V is at most 2^15, so that products of the two
  // fill f16's range. `most`: the largest scale of V so far, as a power of two
  // above it.
  float m, l, base, scale, most, up;

  // Eight neighbouring dims of a row from d, as they are stored; past dim the
  // last one (all loads are on their way before the first is used).
  template <class V>
  static __device__ __forceinline__ void load8(const V *p, int d, int dim, V (&v)[8]) {
    if (dim % 8 == 0) {
      __builtin_memcpy(v, p + min(d, dim - 8), sizeof v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = p[min(d + j, dim - 1)];
    }
  }

  __device__ __forceinline__ void start(const void *q_, long at, int type, int dim, int quarter, float by, bool turn) {
    float x[NC][8];
    uint32_t top = 0;
    if constexpr (TWO) {
#pragma unroll
      for (int c = 0; c < NC; c++) load8((const float *)q_ + at, 32 * c + 8 * quarter, dim, x[c]);
    } else {
      uint16_t raw[NC][8];
#pragma unroll
      for (int c = 0; c < NC; c++) load8((const uint16_t *)q_ + at, 32 * c + 8 * quarter, dim, raw[c]);
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          x[c][j] = type == PPOCR_BF16 ? __uint_as_float((uint32_t)raw[c][j] << 16)
                                       : (float)__builtin_bit_cast(_Float16, raw[c][j]);
    }
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (32 * c + 8 * quarter + j >= dim) x[c][j] = 0.0f;
        top = max(top, __float_as_uint(x[c][j]) & 0x7fffffffu);
      }
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    // q's largest is 2^13 or more, below 2^14 (less only where all are below f32's normal numbers).
    const int e = 13 - ((int)(top >> 23) - 127);
    // 2^100 keeps sums times it finite: at such a scale one key has all the weight. 2^-126 stands for 0, which a
    // hidden key's -infinity could not be multiplied with.
    scale = fmaxf(fminf(__builtin_ldexpf(by, 9 - e) * 1.44269504088896340736f, 0x1p100f), 0x1p-126f);
    if (top >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u);  // an infinity or NaN in q: NaN
#pragma unroll
    for (int g = 0; g < G; g++) qs[g] = 0.0f, om[g] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; c++) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        x[c][j] = __builtin_ldexpf(turn ? -x[c][j] : x[c][j], e);
        sum += x[c][j];
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      qs[c / GC] += sum * 0x1p-9f;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float odd = i & 1 ? 0x1p-4f : 1.0f, a = x[c][i] * odd, b = x[c][i + 4] * odd;
        const v2h high = __builtin_convertvector(v2f{a, b}, v2h);
        q[0][c][i] = __builtin_bit_cast(uint32_t, high);
        if constexpr (TWO)
          q[1][c][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a - (float)high[0], b - (float)high[1]}, v2h));
      }
    }
#pragma unroll
    for (int i = 0; i < E; i++) o[i] = v4f{0, 0, 0, 0};
    m = base = -INFINITY;
    l = most = 0.0f;
    up = 15.0f;
  }

  // Half a tile's codes of 16 keys, of which this lane has row lane % 16 of K and
  // the four keys 4 quarter .. 4 quarter + 3 of V and of all scales and minima.
  struct Half {
    uint32_t n[NC];
    _Float16 s[4 * G], m[4 * G];
  };
  Half k[2], v[2];

  // `p`: the page's chunk, `slot`: the half's first token in the page.
  static __device__ __forceinline__ void load(Half &t, const char *p, int codes, int scales, int minima, int slot,
                                              int at, int quarter) {
    const int few = 2 * G * (slot + 4 * quarter);
    __builtin_memcpy(t.n, p + codes + slot * 16 * NC + at * 4 * NC, 4 * NC);
    __builtin_memcpy(t.s, p + scales + few, 8 * G);
    __builtin_memcpy(t.m, p + minima + few, 8 * G);
  }
  __device__ __forceinline__ void load_k(int half, const char *p, int slot, const Kv4Args &c, int lane) {
    load(k[half], p, 0, c.at_ks, c.at_km, slot, lane % 16 * 4 + lane / 16, lane / 16);
  }
  __device__ __forceinline__ void load_v(int half, const char *p, int slot, const Kv4Args &c, int lane) {
    load(v[half], p, c.at_v, c.at_vs, c.at_vm, slot, lane, lane / 16);
  }

  // The products of K's half with q.
  __device__ __forceinline__ v4f products(const Half &t) const {
    constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;
    v4f sum[G], s{0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < G; g++) {
      sum[g] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int c = g * GC; c < NC && c < (g + 1) * GC; c++) {
        const uint32_t w = t.n[c], u = w >> 8;
        const v4u a{codes16(w, kLow), codes16(w, kHigh), codes16(u, kLow), codes16(u, kHigh)};
        sum[g] = mfma16(a, q[0][c], sum[g]);
        if constexpr (TWO) sum[g] = mfma16(a, q[1][c], sum[g]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int g = 0; g < G; g++) {
        s[r] = fmaf((float)t.m[r * G + g], qs[g], s[r]);
        s[r] = fmaf((float)t.s[r * G + g], sum[g][r], s[r]);
      }
    return s;
  }

  // Raises the largest product and V's largest scale to a tile's.
  __device__ __forceinline__ void raise(float now, float large) {
    large = fmaxf(large, __shfl_xor(large, 16));
    large = fmaxf(large, __shfl_xor(large, 32));
    if (large > most) {
      const int e = min((int)(__float_as_uint(large) >> 23) - 126, 17);  // large <= 2^e
      most = __builtin_ldexpf(1.0f, e);
      up = (float)(15 - e);
    }
    const float next = now == -INFINITY ? -INFINITY : fmaf(now, scale, -up);
    const float shrink = base == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(base - next);
    l *= shrink;
#pragma unroll
    for (int i = 0; i < E; i++) o[i] *= shrink;
#pragma unroll
    for (int g = 0; g < G; g++) om[g] *= shrink;
    m = now;
    base = next;
  }

  // Takes in the tile in k and v. seen(key of the tile): whether the rows see it
  // (asked where `masked`); next_k() and next_v() ask for the next tile's as soon
  // as this one's are used.
  template <class Seen, class NextK, class NextV>
  __device__ __forceinline__ void use(Seen seen, bool masked, int quarter, NextK next_k, NextV next_v) {
    constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;
    v4f s[2] = {products(k[0]), products(k[1])};
    next_k();
    if (masked) {
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const bool on = seen(16 * h + 4 * quarter + r);
          s[h][r] = on ? s[h][r] : -INFINITY;
#pragma unroll
          for (int g = 0; g < G; g++) {
            v[h].s[r * G + g] = on ? v[h].s[r * G + g] : (_Float16)0.0f;
            v[h].m[r * G + g] = on ? v[h].m[r * G + g] : (_Float16)0.0f;
          }
        }
    }
    float top = -INFINITY;
    v2h wide{0, 0};
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int r = 0; r < 4; r++) top = fmaxf(top, s[h][r]);
#pragma unroll
      for (int i = 0; i < 4 * G; i += 2) wide = __builtin_elementwise_max(wide, v2h{v[h].s[i], v[h].s[i + 1]});
    }
    const float large = (float)__builtin_elementwise_max(wide[0], wide[1]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float now = fmaxf(m, top);
    if (__any(now != m || large > most)) raise(now, large);
    const float from = base == -INFINITY ? 0.0f : base;
    float p[2][4];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[h][r] = __builtin_amdgcn_exp2f(fmaf(s[h][r], scale, -from));
        l += p[h][r];
#pragma unroll
        for (int g = 0; g < G; g++) om[g] = fmaf(p[h][r], (float)v[h].m[r * G + g], om[g]);
      }
#pragma unroll
    for (int g = 0; g < G; g++) {
      // Weights times scales in two f16 parts: 22 bits.
      v4u high, low;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int h = i / 2, r = i % 2;  // keys r and r + 2 of the quarter, as the masks leave V's
        const float x = fmaf(p[h][r], (float)v[h].s[r * G + g], 0.0f);
        const float y = fmaf(p[h][r + 2], (float)v[h].s[(r + 2) * G + g], 0.0f);
        const uint32_t both = pair16(x, y);
        const v2h back = __builtin_bit_cast(v2h, both);
        high[i] = both;
        low[i] = pair16(fmaf((float)back[0], -1.0f, x), fmaf((float)back[1], -1.0f, y));
      }
#pragma unroll
      for (int c = g * GC; c < NC && c < (g + 1) * GC; c++) {
        const uint32_t w0 = v[0].n[c], w1 = v[1].n[c], u0 = w0 >> 8, u1 = w1 >> 8;
        const v4u even{codes16(w0, kLow), codes16(u0, kLow), codes16(w1, kLow), codes16(u1, kLow)};
        const v4u odd{codes16(w0, kHigh), codes16(u0, kHigh), codes16(w1, kHigh), codes16(u1, kHigh)};
        o[2 * c] = mfma16(even, low, o[2 * c]);
        o[2 * c + 1] = mfma16(odd, low, o[2 * c + 1]);
        o[2 * c] = mfma16(even, high, o[2 * c]);
        o[2 * c + 1] = mfma16(odd, high, o[2 * c + 1]);
      }
    }
    next_v();
  }

  // The row's whole sum, and its sums of P m, in all four quarters.
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

// Waves that a SIMD's 512 registers a lane hold without spilling: results, q and
// codes, scales and minima, and about 45 others.
template <int NC, int GC, bool TWO>
constexpr int waves_a_simd4() {
  constexpr int n = NC * (8 + (TWO ? 8 : 4) + 4) + 16 * ((NC + GC - 1) / GC) + 45;
  return n <= 128 ? 4 : n <= 168 ? 3 : n <= 250 ? 2 : 1;
}

// Text blockIdx.z, a key head's 16 (or fewer) query heads blockIdx.x, part
// blockIdx.y of its tiles of 32 tokens, a tile a wave at a time: a tile's halves
// lie in one page each, whose number all lanes look up alike.
template <int NC, int GC, bool TWO>
__global__ __launch_bounds__(64 * kWaves4, (waves_a_simd4<NC, GC, TWO>())) void kv4_attention_parts(Attend4Args a) {
  typedef Rows4<NC, GC, TWO> A;
  constexpr int DP = A::DP;
  __shared__ float lds_o[kWaves4][16][DP + 4];
  __shared__ float lds_b[kWaves4][16], lds_l[kWaves4][16];
  __shared__ int lds_bad;
  const int lane = threadIdx.x % 64, col = lane % 16, quarter = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int b = blockIdx.z, per = a.heads / a.c.heads, blocks = (per + 15) / 16;
  const int kv = blockIdx.x / blocks, h0 = kv * per + blockIdx.x % blocks * 16;
  const int rows = min(16, kv * per + per - h0);
  const int length = a.c.lengths[b];
  const bool too_long = length > a.c.table_width * a.c.page_size;
  const Seen s = seen_of(too_long ? 0 : length, a.window, a.sinks, kKeys4);
  const int each = tiles_a_part(s.tiles, a.each, a.splits);
  const int begin = blockIdx.y * each, end = min(begin + each, s.tiles);
  if (begin >= end && blockIdx.y) return;  // part 0 of an empty text writes its zeros
  if (threadIdx.x == 0) lds_bad = too_long;
  __syncthreads();

  A at;
  at.start(a.q, b * a.q_stride + (long)(h0 + min(col, rows - 1)) * a.c.dim, a.type, a.c.dim, quarter, a.scale, a.turn);
  const int *table = a.c.table + b * a.c.table_width;
  const char *data = a.c.data + (long)kv * a.c.chunk;
  bool bad = false;
  auto tile_key = [&](int t) { return t < s.sink_tiles ? t * kKeys4 : s.first + (t - s.sink_tiles) * kKeys4; };
  // Where the 16 tokens from k lie, some of which are seen if `wanted`. (A page
  // that does not exist is read as page 0, and the text's result is NaN.)
  struct Place {
    const char *page;
    int slot;
  };
  auto find = [&](int k, bool wanted) -> Place {
    int page = -1, slot = 0;
    if (wanted) {
      const int n = a.c.by_page(k);
      page = table[n];
      slot = k - n * a.c.page_size;
      bad |= page < 0 || page >= a.c.pages;
    }
    const bool there = page >= 0 && page < a.c.pages;
    return {data + (there ? page * a.c.page_stride : 0), there ? slot : 0};
  };
  struct Places {
    Place half[2];
  };
  // Of 16 neighbours some is seen if one is below the length and above the window's start, or below the sinks' end.
  auto find_tile = [&](int t) -> Places {
    const int k = tile_key(min(t, end - 1));
    return {find(k, k < s.length && (k + 15 >= s.low || k < s.sinks)),
            find(k + 16, k + 16 < s.length && (k + 31 >= s.low || k + 16 < s.sinks))};
  };
  const int whole0 = s.sink_tiles + (s.first < s.low ? 1 : 0), whole1 = s.sink_tiles + (s.length - s.first) / kKeys4;
  int t = begin + wave;
  if (t < end) {
    Places at_now = find_tile(t);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      at.load_k(h, at_now.half[h].page, at_now.half[h].slot, a.c, lane);
      at.load_v(h, at_now.half[h].page, at_now.half[h].slot, a.c, lane);
    }
    for (; t < end; t += kWaves4) {
      // (Past the last tile the last one again.)
      const Places next = find_tile(t + kWaves4);
      const int k = tile_key(t);
      at.use([&](int i) { return k + i < s.length && (k + i >= s.low || k + i < s.sinks); }, t < whole0 || t >= whole1,
             quarter,
             [&] {
#pragma unroll
               for (int h = 0; h < 2; h++) at.load_k(h, next.half[h].page, next.half[h].slot, a.c, lane);
             },
             [&] {
#pragma unroll
               for (int h = 0; h < 2; h++) at.load_v(h, next.half[h].page, next.half[h].slot, a.c, lane);
             });
    }
  }
  // The waves' parts, joined.
  if (bad) lds_bad = 1;
  const float l = at.total();
  if (quarter == 0) lds_b[wave][col] = at.base, lds_l[wave][col] = l;
#pragma unroll
  for (int c = 0; c < NC; c++)
#pragma unroll
    for (int odd = 0; odd < 2; odd++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        lds_o[wave][col][32 * c + 2 * (4 * quarter + r) + odd] =
            fmaf(at.o[2 * c + odd][r], odd ? 0x1p5f : 0x1p9f, at.om[c / GC]);
  __syncthreads();
  const bool split = a.splits > 1;
  for (int i = threadIdx.x; i < rows * DP; i += 64 * kWaves4) {
    const int row = i / DP, d = i % DP;
    if (d >= a.c.dim) continue;
    float base = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves4; w++) base = fmaxf(base, lds_b[w][row]);
#pragma unroll
    for (int w = 0; w < kWaves4; w++) {
      // (A base is -infinity where the wave had no key; NaN where q is not finite.)
      const float f = lds_b[w][row] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lds_b[w][row] - base);
      sum += f * lds_l[w][row];
      o += f * lds_o[w][row][d];
    }
    if (lds_bad) sum = o = __uint_as_float(0x7fc00000u);
    if (split) {
      float *p = a.part + (((long)b * a.heads + h0 + row) * a.splits + blockIdx.y) * (a.c.dim + 2);
      p[d + 2] = o;
      if (d == 0) p[0] = base, p[1] = sum;
    } else {
      put_at(a.y, b * a.y_stride + (long)(h0 + row) * a.c.dim + d, a.type, sum == 0.0f ? 0.0f : o / sum);
    }
  }
}

template <int NC, int GC, bool TWO>
hipError_t launch_parts4(const Attend4Args &a, hipStream_t s) {
  const int per = a.heads / a.c.heads;
  const dim3 grid(a.c.heads * ((per + 15) / 16), a.splits, a.batch), block(64 * kWaves4);
  return launch_kernel(kv4_attention_parts<NC, GC, TWO>, grid, block, 0, s, a);
}

// Groups of a whole head, of 32 and of 64 (where a head has more than one).
template <int NC, bool TWO>
hipError_t launch_groups4(const Attend4Args &a, hipStream_t s) {
  if constexpr (NC > 1) {
    if (a.c.group == 32) return launch_parts4<NC, 1, TWO>(a, s);
  }
  if constexpr (NC > 2) {
    if (a.c.group == 64) return launch_parts4<NC, 2, TWO>(a, s);
  }
  return launch_parts4<NC, NC, TWO>(a, s);
}

template <bool TWO>
hipError_t launch_attention4(const Attend4Args &a, hipStream_t s) {
  hipError_t e = hipErrorInvalidValue;
  switch (a.c.nc) {
    case 1: e = launch_groups4<1, TWO>(a, s); break;
    case 2: e = launch_groups4<2, TWO>(a, s); break;
    case 3: e = launch_groups4<3, TWO>(a, s); break;
    case 4: e = launch_groups4<4, TWO>(a, s); break;
    case 6: e = launch_groups4<6, TWO>(a, s); break;
    case 8: e = launch_groups4<8, TWO>(a, s); break;
  }
  return e != hipSuccess || a.splits == 1 ? e : launch_kv4_join(a, s);
}

}  // namespace ppocr
