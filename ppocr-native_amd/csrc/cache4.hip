// The paged cache held in 4 bits: appending to it, with the rotation of keys
// and queries on the way (ppocr_hip_kv4_append), and reading tokens back as rows
// (ppocr_hip_kv4_read).
//
//   a group's m = f16(min x), s = f16((max x - m) / 15), n = round((x - m) / s)
//
// A workgroup has the tokens of 16 neighbouring places, so that the chain of
// waits that finds them (text, length, page) is paid for once; a wave takes four
// of them at a time, one of V's blocks, where a code word is four tokens' bytes: a
// lane has eight neighbouring dims of one of them, which are a word of K's codes
// and a byte of each of four words of V's. Those go through a wave's own piece of
// LDS, so that memory sees whole words. The queries have workgroups of their own;
// they are turned at places below 0, too, where there is nothing to append.
//
// Memory bound where there are many tokens: four chunks of prompts (11344 tokens
// of 32 heads of 128, 8 key heads, f16, groups of 32) are appended in 56 us, 247 MB
// at 4.4 TB/s where a copy of as much has 5.2; all 22611 tokens of their texts are
// read in 26 us, 122 MB at 4.6. With a token a text the chain of waits is the
// whole: 64 take 6.5 and 4.5 us. Where a turned half is no multiple of eight values
// a piece is one value: heads of 96 with 24 turned, the same chunks, take 116 us
// for both, with 96 turned 69.
#include <algorithm>

#include "turn.hpp"

namespace ppocr {
namespace {

constexpr int kMostWaves4 = 8;

// Eight values, or `have` of them, of what a kernel that follows reads: as a
// stream, which leaves the caches to what else is written (a read of 22611
// tokens of 8 heads of 128 as f16: 36 us with plain stores, 27 so).
template <class V>
__device__ __forceinline__ void store_past(V *p, int have, const V (&v)[8]) {
  if (have >= 8) {
    stream_out(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (j < have) p[j] = v[j];
  }
}

// The 16 places that workgroup g has, with as many workgroups for each text as
// its rows could touch: text b's begin at (its first row + 30 b) / 16. BELOW: with
// the places below 0 of a text that has fewer tokens than rows.
constexpr int kPlaces = 16;
struct Block16 {
  int b;        // text, or -1
  long row0;    // the row whose place is the first (it may not exist)
  int from, to; // which of the 16 are rows
  long place;   // the first place
  char *chunk;  // its page's chunk of head 0, or NULL
  int slot;     // its number in the page
};

__device__ __forceinline__ long clamped(long v, long most) { return min(max(v, 0L), most); }

template <bool BELOW>
__device__ __forceinline__ Block16 block_of(const Kv4Args &c, const int *starts, long rows, int batch, long g) {
  Block16 o;
  o.b = -1;
  o.chunk = nullptr;
  auto start = [&](int i) { return (clamped(starts ? starts[i] : i, rows) + (2 * kPlaces - 2L) * i) / kPlaces; };
  int b = last_not_past(batch + 1, g, start);
  b = __builtin_amdgcn_readfirstlane(b);
  if (b < 0 || b >= batch) return o;
  long first = b, last = b + 1L;
  if (starts) first = starts[b], last = starts[b + 1];
  const long count = last - first, base = (long)c.lengths[b] - count;  // row first + i has place base + i
  const long begin = max(max(0L, -first), BELOW ? 0L : -base), end = min(count, rows - first);
  if (begin >= end) return o;
  o.place = ((base + begin) & -(long)kPlaces) + kPlaces * (g - start(b));
  if (o.place >= base + end) return o;
  o.b = b;
  o.row0 = first + o.place - base;
  o.from = (int)max(0L, base + begin - o.place);
  o.to = (int)min((long)kPlaces, base + end - o.place);
  o.slot = 0;
  if (o.place < 0) return o;  // (all 16 are)
  const int slot = c.by_page((int)o.place);
  o.slot = (int)(o.place - (long)slot * c.page_size);
  if (slot < c.table_width) {
    const int page = c.table[b * c.table_width + slot];
    if (page >= 0 && page < c.pages) o.chunk = c.data + page * c.page_stride;
  }
  return o;
}

template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, false));
}
// The least and the largest of 4, 8, 16 or 32 neighbouring lanes, in all of them.
__device__ __forceinline__ void lanes_range(float &low, float &high, int lanes) {
  low = fminf(low, dpp_f<0xB1>(low)), high = fmaxf(high, dpp_f<0xB1>(high));  // lane ^ 1
  low = fminf(low, dpp_f<0x4E>(low)), high = fmaxf(high, dpp_f<0x4E>(high));  // lane ^ 2
  if (lanes >= 8) low = fminf(low, dpp_f<0x141>(low)), high = fmaxf(high, dpp_f<0x141>(high));   // of 8, mirrored
  if (lanes >= 16) low = fminf(low, dpp_f<0x140>(low)), high = fmaxf(high, dpp_f<0x140>(high));  // of 16, mirrored
  if (lanes >= 32) low = fminf(low, __shfl_xor(low, 16)), high = fmaxf(high, __shfl_xor(high, 16));
}

// Eight dims' codes as a word, the low bits the first; their group's scale and
// minimum. `lanes`: of a group; `have`: dims that there are (EIGHTS: 0 or 8).
template <bool EIGHTS>
__device__ __forceinline__ uint32_t quantise(float (&x)[8], int have, int lanes, uint16_t &scale, uint16_t &least) {
  constexpr float kMost16 = 65504.0f;
  float low = INFINITY, high = -INFINITY, zero = 0.0f;  // zero: NaN where one is not finite
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const bool on = EIGHTS || j < have;
    zero = on ? fmaf(x[j], 0.0f, zero) : zero;
    x[j] = __builtin_amdgcn_fmed3f(x[j], -kMost16, kMost16);
    low = on ? fminf(low, x[j]) : low;
    high = on ? fmaxf(high, x[j]) : high;
  }
  if (zero != 0.0f) high = INFINITY;
  if (EIGHTS && have == 0) low = INFINITY, high = -INFINITY;
  lanes_range(low, high, lanes);
  const bool none = low == INFINITY && high != INFINITY;  // (a group of padding: no dim of it is there)
  const _Float16 m16 = none ? (_Float16)0.0f : (_Float16)(low + 0.0f);  // (the least of -0 and 0 is either)
  const float m = (float)m16;
  // (The step is rounded to f32 first: an instruction that does both at once would round some the other way.)
  float step = fmaxf((high - m) * (1.0f / 15.0f), 0.0f) + 0.0f;  // (below 0 where m was rounded past all of them)
  asm("" : "+v"(step));
  const _Float16 s16 = none ? (_Float16)0.0f : (_Float16)step;
  const float s = (float)s16, inverse = 1.0f / s;
  const bool off = high == INFINITY || none || s == 0.0f;
  float four[2];  // four codes as one number
#pragma unroll
  for (int j = 7; j >= 0; j--) {
    const float r = __builtin_amdgcn_fmed3f(rintf((x[j] - m) * inverse), 0.0f, 15.0f), n = EIGHTS || j < have ? r : 0.0f;
    four[j / 4] = j % 4 == 3 ? n : fmaf(four[j / 4], 16.0f, n);
  }
  uint32_t word = (uint32_t)four[0] | (uint32_t)four[1] << 16;
  if (off || (EIGHTS && have == 0)) word = 0;
  scale = high == INFINITY ? 0x7e00 : __builtin_bit_cast(uint16_t, s16);
  least = high == INFINITY ? 0 : __builtin_bit_cast(uint16_t, m16);
  return word;
}

// LDS that only this wave uses: what was written is seen after this. (A wave's LDS
// operations are done in order; a fence would wait for its stores to memory, too.)
__device__ __forceinline__ void wave_sync() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

// LP: lanes a head's row has (8 dims each); a wave has four tokens of HEADS heads,
// 64 / LP of these rows a pass.
template <int LP, int F>
struct Split4 {
  static constexpr int PASSES = F * (LP == 32 ? 2 : 1), HEADS = 16 * PASSES / LP;
  static constexpr int WORDS = F * (LP < 32 ? 64 : 128);  // V words of a wave's heads at most
};

// Eight dims of a row of k from d, those that they are turned with, and eight of
// v. EIGHTS: heads and what is turned of them are whole eights (or pairs).
template <class V>
struct Eight {
  V k[8], other[8], v[8];
};
template <bool EIGHTS, class V>
__device__ __forceinline__ Eight<V> load_eight(const V *k, const V *v, int d, int dim, const TurnArgs &t) {
  Eight<V> e;
  const int half = t.rotary / 2;
  auto far = [&](int i) { return t.pairs || i >= t.rotary ? i : i < half ? i + half : i - half; };
  if constexpr (EIGHTS) {
    __builtin_memcpy(e.k, k + d, sizeof e.k);
    __builtin_memcpy(e.other, k + far(d), sizeof e.other);
    __builtin_memcpy(e.v, v + d, sizeof e.v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int i = min(d + j, dim - 1);
      e.k[j] = k[i], e.other[j] = k[far(i)], e.v[j] = v[i];
    }
  }
  return e;
}

// Workgroups blockIdx.y: keys and values, or queries. WHOLE: pieces of 16 bytes
// hold no part of what is turned apart; EIGHTS: as above.
template <int T, int LP, bool WHOLE, bool EIGHTS>
__global__ __launch_bounds__(64 * kMostWaves4, EIGHTS ? 4 : 2) void kv4_append_rows(Append4Args a) {
  typedef num_t<T> V;
  typedef Num<T> F;
  typedef Split4<LP, 1> S;
  constexpr int N = WHOLE ? 16 / sizeof(V) : 1;
  __shared__ v2f cs[kPlaces][128];
  __shared__ uint32_t words[kMostWaves4][S::WORDS];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int threads = blockDim.x, waves = threads / 64;
  const Block16 k16 = block_of<true>(a.c, a.starts, a.rows, a.batch, (long)blockIdx.z * gridDim.x + blockIdx.x);
  if (k16.b < 0) return;
  const TurnArgs &t = a.t;
  const int dim = a.c.dim, half = t.rotary / 2;

  // The queries: a thread has a unit of every token, or where there are two or more
  // teams of threads, of every second or fourth ...; the next token's is on its way.
  struct Q {
    V p[N], r[N];
  };
  const int items = t.heads * a.units, team = threads / a.teams;
  const int of = __builtin_amdgcn_readfirstlane(threadIdx.x / team);
  int item = threadIdx.x - of * team;
  Unit o;
  uint32_t at1, at2;
  auto unit = [&] {
    const int h = a.by_unit(item);
    o = unit_of<N>(item - h * a.units, dim, t.rotary, t.pairs);
    at1 = (uint32_t)(h * dim + o.d1), at2 = (uint32_t)(h * dim + (o.d2 < dim ? o.d2 : o.d1));
  };
  auto load_q = [&](int token) {
    Q q;
    const V *from = (const V *)t.q + (k16.row0 + min(token, k16.to - 1)) * t.q_stride;
    __builtin_memcpy(q.p, from + at1, sizeof q.p);
    __builtin_memcpy(q.r, from + at2, sizeof q.r);
    return q;
  };
  Q q;
  const bool queries = blockIdx.y, some = queries && item < items;
  if (some) unit(), q = load_q(k16.from + of);
  for (int i = threadIdx.x; i < (k16.to - k16.from) * half; i += threads) {
    const int token = k16.from + a.by_half(i), j = i - (token - k16.from) * half;
    const double at = t.positions ? (double)t.positions[k16.row0 + token] : (double)(k16.place + token);
    cs[token][j] = cosine_sine(at * (double)t.freqs[j]);
  }
  __syncthreads();
  if (some) {
    while (true) {
      for (int token = k16.from + of; token < k16.to; token += a.teams) {
        const Q next = load_q(token + a.teams);
        if (o.turned) turn_unit<T, N>(q.p, q.r, cs[token], o, t.rotary, t.pairs);
        V *into = (V *)t.q_out + (k16.row0 + token) * t.q_out_stride;
        stream_out(into + at1, q.p);
        if (o.d2 < dim) stream_out(into + at2, q.r);
        q = next;
      }
      item += team;
      if (item >= items) break;
      unit(), q = load_q(k16.from + of);
    }
  }
  if (queries || !k16.chunk) return;

  // Keys and values: a wave has four tokens (in one pass or more), some heads at
  // a time. With one token a text the waves share the heads.
  const int l = lane % LP, d = 8 * l, have = min(max(dim - d, 0), 8);
  const int nc = a.c.nc, block = l / 4, quarter = l % 4;
  const int lanes = min(a.c.group / 8, LP);  // of a group
  const int group = l / lanes;
  const int four0 = k16.from / 4, fours = (k16.to + 3) / 4 - four0, side = fours > 1 ? kPlaces / 4 : 1;
  const int four = four0 + wave % side, from = max(k16.from - 4 * four, 0), to = min(k16.to - 4 * four, 4);
  if (wave % side >= fours) return;
  const long row0 = k16.row0 + 4 * four;
  for (int h0 = wave / side * S::HEADS; h0 < a.c.heads; h0 += waves / side * S::HEADS) {
    Eight<V> ahead[S::PASSES];
#pragma unroll
    for (int pass = 0; pass < S::PASSES; pass++) {
      const int r = lane / LP + pass * (64 / LP), in = min(h0 + r / 4, a.c.heads - 1) * dim;
      const long row = row0 + min(max(r % 4, from), to - 1);  // (one that there is)
      ahead[pass] = load_eight<EIGHTS>((const V *)a.k + row * a.k_stride + in, (const V *)a.v + row * a.v_stride + in,
                                       EIGHTS ? min(d, dim - 8) : d, dim, t);
    }
    char *chunk0 = k16.chunk + (long)h0 * a.c.chunk;
#pragma unroll
    for (int pass = 0; pass < S::PASSES; pass++) {
      const int row = lane / LP + pass * (64 / LP), token = row % 4, h = h0 + row / 4;
      const bool on = token >= from && token < to && h < a.c.heads;
      const Eight<V> raw = ahead[pass];
      float k[8], v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) k[j] = F::get(raw.k[j]), v[j] = F::get(raw.v[j]);
      if (on) {
        const v2f *turn = cs[4 * four + token];
        if (t.pairs) {
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            if (d + j < t.rotary) {
              const v2f c = turn[d / 2 + j / 2];
              const float x = k[j], y = k[j + 1];
              k[j] = x * c[0] - y * c[1], k[j + 1] = y * c[0] + x * c[1];
            }
        } else if (EIGHTS) {
          if (d < t.rotary) {
            const bool second = d >= half;
            turn += second ? d - half : d;
#pragma unroll
            for (int j = 0; j < 8; j++) {
              const v2f c = turn[j];
              const float other = F::get(raw.other[j]) * c[1];
              k[j] = k[j] * c[0] + (second ? other : -other);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (d + j < t.rotary) {
              const bool second = d + j >= half;
              const v2f c = turn[d + j - (second ? half : 0)];
              const float other = F::get(raw.other[j]) * c[1];
              k[j] = second ? k[j] * c[0] + other : k[j] * c[0] - other;
            }
        }
      }
      // (Lanes without a row go along: their neighbours' ranges are of other rows.)
      uint16_t ks, km, vs, vm;
      const uint32_t kw = quantise<EIGHTS>(k, on ? have : 0, lanes, ks, km), vw = quantise<EIGHTS>(v, on ? have : 0, lanes, vs, vm);
      if (on && block < nc) {
        char *chunk = chunk0 + (long)(row / 4) * a.c.chunk;
        const int slot = k16.slot + 4 * four + token;
        *(uint32_t *)(chunk + (long)slot * 16 * nc + 4 * (nc * quarter + block)) = kw;
        if (l % lanes == 0 && group < a.c.groups) {
          const int at = 2 * (slot * a.c.groups + group);
          *(uint16_t *)(chunk + a.c.at_ks + at) = ks, *(uint16_t *)(chunk + a.c.at_km + at) = km;
          *(uint16_t *)(chunk + a.c.at_vs + at) = vs, *(uint16_t *)(chunk + a.c.at_vm + at) = vm;
        }
        uint8_t *into = (uint8_t *)(words[wave] + row / 4 * 16 * nc);
#pragma unroll
        for (int j = 0; j < 4; j++) into[((4 * quarter + j) * nc + block) * 4 + token] = (uint8_t)(vw >> 8 * j);
      }
    }
    wave_sync();
    for (int i = lane; i < S::HEADS * 16 * nc; i += 64) {
      const int h = h0 + i / (16 * nc), w = i % (16 * nc);
      if (h < a.c.heads) {
        char *into = chunk0 + (long)(i / (16 * nc)) * a.c.chunk + a.c.at_v + (long)(k16.slot / 4 + four) * 64 * nc + 4 * w;
        const uint32_t word = words[wave][i];
        if (from == 0 && to == 4) {
          *(uint32_t *)into = word;
        } else {
          for (int token = from; token < to; token++) into[token] = (char)(word >> 8 * token);
        }
      }
    }
    wave_sync();
  }
}

// What a code stands for, as it is read: 15 of a group that reaches f16's largest
// value can stand for 60 more (15 half steps of a scale), which f16 rounds to
// infinity; it is held at the largest. (NaN stays NaN.)
template <int T>
__device__ __forceinline__ num_t<T> put_held(float v) {
  return Num<T>::put(T == PPOCR_F16 && v > 65504.0f ? 65504.0f : v);
}

// A wave's words of V, its lanes' words of K and their scales are asked for
// together. F4: times the heads that a wave has in the append.
template <int T, int LP, int F4>
__global__ __launch_bounds__(64 * kMostWaves4) void kv4_read_rows(Read4Args a) {
  typedef num_t<T> V;
  typedef Split4<LP, F4> S;
  __shared__ uint32_t words[kMostWaves4][S::WORDS];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64;
  const Block16 k16 = block_of<false>(a.c, a.starts, a.rows, a.batch, (long)blockIdx.z * gridDim.x + blockIdx.x);
  if (k16.b < 0) return;
  const int l = lane % LP, d = 8 * l, dim = a.c.dim, have = min(max(dim - d, 0), 8);
  const int nc = a.c.nc, block = min(l / 4, nc - 1), quarter = l % 4, group = min(d / a.c.group, a.c.groups - 1);
  const char *page = k16.chunk ? k16.chunk : a.c.data;  // (one that there is: then it gives NaN)
  const int slot0 = k16.chunk ? k16.slot : 0;
  const float nan = k16.chunk ? 0.0f : __uint_as_float(0x7fc00000u);
  const int four0 = k16.from / 4, fours = (k16.to + 3) / 4 - four0;
  const int jobs = (a.c.heads + S::HEADS - 1) / S::HEADS * fours;
  struct Held {
    uint32_t v[S::WORDS / 64], k[S::PASSES];
    _Float16 few[S::PASSES][4];
  };
  auto load = [&](int j) {
    Held o;
    const int h0 = j / fours * S::HEADS, slot4 = slot0 + 4 * (four0 + j % fours);
#pragma unroll
    for (int i = 0; i < S::WORDS / 64; i++) {
      const int at = min(lane + 64 * i, S::HEADS * 16 * nc - 1), h = min(h0 + at / (16 * nc), a.c.heads - 1);
      o.v[i] = *(const uint32_t *)(page + (long)h * a.c.chunk + a.c.at_v + slot4 * 16 * nc + 4 * (at % (16 * nc)));
    }
#pragma unroll
    for (int pass = 0; pass < S::PASSES; pass++) {
      const int r = lane / LP + pass * (64 / LP), h = min(h0 + r / 4, a.c.heads - 1), slot = slot4 + r % 4;
      const char *chunk = page + (long)h * a.c.chunk;
      const int at = 2 * (slot * a.c.groups + group);
      o.k[pass] = *(const uint32_t *)(chunk + slot * 16 * nc + 4 * (nc * quarter + block));
      o.few[pass][0] = *(const _Float16 *)(chunk + a.c.at_ks + at), o.few[pass][1] = *(const _Float16 *)(chunk + a.c.at_km + at);
      o.few[pass][2] = *(const _Float16 *)(chunk + a.c.at_vs + at), o.few[pass][3] = *(const _Float16 *)(chunk + a.c.at_vm + at);
    }
    return o;
  };
  int job = wave;
  if (job >= jobs) return;
  for (; job < jobs; job += waves) {
    const int h0 = job / fours * S::HEADS, four = four0 + job % fours;
    const Held held = load(job);
#pragma unroll
    for (int i = 0; i < S::WORDS / 64; i++) words[wave][lane + 64 * i] = held.v[i];
    wave_sync();
#pragma unroll
    for (int pass = 0; pass < S::PASSES; pass++) {
      const int r = lane / LP + pass * (64 / LP), token = 4 * four + r % 4, h = h0 + r / 4;
      if (token < k16.from || token >= k16.to || h >= a.c.heads || have == 0) continue;
      uint32_t w = 0;
      const uint8_t *from = (const uint8_t *)(words[wave] + r / 4 * 16 * nc);
#pragma unroll
      for (int j = 0; j < 4; j++) w |= (uint32_t)from[((4 * quarter + j) * nc + block) * 4 + r % 4] << 8 * j;
      const float ks = (float)held.few[pass][0], km = (float)held.few[pass][1] + nan;
      const float vs = (float)held.few[pass][2], vm = (float)held.few[pass][3] + nan;
      V k[8], v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        k[j] = put_held<T>(fmaf((float)(held.k[pass] >> 4 * j & 15), ks, km));
        v[j] = put_held<T>(fmaf((float)(w >> 4 * j & 15), vs, vm));
      }
      const long row = k16.row0 + token;
      store_past<V>((V *)a.k + row * a.k_stride + (long)h * dim + d, have, k);
      store_past<V>((V *)a.v + row * a.v_stride + (long)h * dim + d, have, v);
    }
    wave_sync();
  }
}

// (A grid's side has fewer than 2^32 threads.)
inline dim3 grid4(long rows, int batch, unsigned roles) {
  const long blocks = (rows + (2 * kPlaces - 2L) * batch) / kPlaces + 1, wide = std::min(blocks, 1L << 20);
  return dim3(unsigned(wide), roles, unsigned((blocks + wide - 1) / wide));
}

// Four waves, or eight where the keys and values of 16 tokens have work for them.
template <int LP, int F>
dim3 threads4(int heads, long rows, int batch) {
  const int jobs = (heads + Split4<LP, F>::HEADS - 1) / Split4<LP, F>::HEADS * (rows > batch ? kPlaces / 4 : 1);
  return dim3(64 * (jobs > 4 ? kMostWaves4 : 4));
}

template <int T, int LP>
hipError_t launch_append4(Append4Args a, hipStream_t s) {
  constexpr int N = 16 / sizeof(num_t<T>);
  const bool whole = whole_pieces(N, a.c.dim, a.t.rotary, a.t.pairs);
  const bool eights = a.c.dim % 8 == 0 && (a.t.pairs || a.t.rotary % 16 == 0);
  a.units = units_of(whole && eights ? N : 1, a.c.dim, a.t.rotary, a.t.pairs);
  a.by_unit = Divide(a.units);
  a.by_half = Divide(std::max(a.t.rotary / 2, 1));
  const dim3 grid = grid4(a.rows, a.batch, a.t.q ? 2 : 1), block = threads4<LP, 1>(a.c.heads, a.rows, a.batch);
  // Teams of whole waves: fewest steps, of which a new unit is half a one.
  const long items = (long)a.t.heads * a.units, tokens = a.rows > a.batch ? kPlaces : 1;
  long least = -1;
  for (int teams = 1; teams <= int(block.x / 64); teams *= 2) {
    const long team = block.x / teams, units = (items + team - 1) / team, steps = units * (2 * ((tokens + teams - 1) / teams) + 1);
    if (least < 0 || steps < least) least = steps, a.teams = teams;
  }
  if (whole && eights) return launch_kernel(kv4_append_rows<T, LP, true, true>, grid, block, 0, s, a);
  if (eights) return launch_kernel(kv4_append_rows<T, LP, false, true>, grid, block, 0, s, a);
  return launch_kernel(kv4_append_rows<T, LP, false, false>, grid, block, 0, s, a);
}

template <int T>
hipError_t launch_append4_of(const Append4Args &a, hipStream_t s) {
  switch (a.c.nc) {
    case 1: return launch_append4<T, 4>(a, s);
    case 2: return launch_append4<T, 8>(a, s);
    case 3:
    case 4: return launch_append4<T, 16>(a, s);
  }
  return launch_append4<T, 32>(a, s);
}

template <int T, int LP>
hipError_t launch_read4(const Read4Args &a, hipStream_t s) {
  // Four times the heads a wave where there is more than a token a text: 22611
  // tokens of 8 heads of 128 as f16 take 26 us instead of 32; 64 texts' newest 5.4
  // instead of 4.3.
  const dim3 grid = grid4(a.rows, a.batch, 1);
  if (a.rows <= a.batch) return launch_kernel(kv4_read_rows<T, LP, 1>, grid, threads4<LP, 1>(a.c.heads, a.rows, a.batch), 0, s, a);
  return launch_kernel(kv4_read_rows<T, LP, 4>, grid, threads4<LP, 4>(a.c.heads, a.rows, a.batch), 0, s, a);
}

template <int T>
hipError_t launch_read4_of(const Read4Args &a, hipStream_t s) {
  switch (a.c.nc) {
    case 1: return launch_read4<T, 4>(a, s);
    case 2: return launch_read4<T, 8>(a, s);
    case 3:
    case 4: return launch_read4<T, 16>(a, s);
  }
  return launch_read4<T, 32>(a, s);
}

}  // namespace

hipError_t launch_kv4_append(const Append4Args &a, int type, hipStream_t s) {
  switch (type) {
    case PPOCR_F32: return launch_append4_of<PPOCR_F32>(a, s);
    case PPOCR_BF16: return launch_append4_of<PPOCR_BF16>(a, s);
    case PPOCR_F16: return launch_append4_of<PPOCR_F16>(a, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_kv4_read(const Read4Args &a, int type, hipStream_t s) {
  switch (type) {
    case PPOCR_F32: return launch_read4_of<PPOCR_F32>(a, s);
    case PPOCR_BF16: return launch_read4_of<PPOCR_BF16>(a, s);
    case PPOCR_F16: return launch_read4_of<PPOCR_F16>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ppocr
