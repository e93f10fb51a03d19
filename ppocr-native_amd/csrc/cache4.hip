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
// LDS, so that memory sees whole words.
#include <algorithm>

#include "turn.hpp"

namespace ppocr {
namespace {

constexpr int kMostWaves4 = 8;

// The 16 places that workgroup g has, with as many workgroups for each text as
// its rows could touch: text b's begin at (its first row + 30 b) / 16.
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
  const long begin = max(max(0L, -first), -base), end = min(count, rows - first);
  if (begin >= end) return o;
  o.place = (base + begin) / kPlaces * kPlaces + kPlaces * (g - start(b));
  if (o.place >= base + end) return o;
  o.b = b;
  o.row0 = first + o.place - base;
  o.from = (int)max(0L, base + begin - o.place);
  o.to = (int)min((long)kPlaces, base + end - o.place);
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
// minimum. `lanes`: of a group; `have`: dims that there are.
__device__ __forceinline__ uint32_t quantise(float (&x)[8], int have, int lanes, uint16_t &scale, uint16_t &least) {
  constexpr float kMost16 = 65504.0f;
  float low = INFINITY, high = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const bool on = j < have;
    bad |= on && !(fabsf(x[j]) < INFINITY);
    x[j] = __builtin_amdgcn_fmed3f(x[j], -kMost16, kMost16);
    low = on ? fminf(low, x[j]) : low;
    high = on ? fmaxf(high, x[j]) : high;
  }
  if (bad) high = INFINITY;
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
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float n = __builtin_amdgcn_fmed3f(rintf((x[j] - m) * inverse), 0.0f, 15.0f);
    word |= (j < have && !off ? (uint32_t)n : 0u) << 4 * j;
  }
  scale = high == INFINITY ? 0x7e00 : __builtin_bit_cast(uint16_t, s16);
  least = high == INFINITY ? 0 : __builtin_bit_cast(uint16_t, m16);
  return word;
}

// Four lanes' worth of LDS that only this wave uses: what was written is seen
// after this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// LP: lanes a head's row has (8 dims each); a wave has 64 / LP rows at once, of
// four tokens of one or more heads, or of two tokens.
template <int LP>
struct Split4 {
  static constexpr int HEADS = LP < 16 ? 16 / LP : 1, PASSES = LP == 32 ? 2 : 1;
  static constexpr int WORDS = LP < 32 ? 64 : 128;  // V words of a wave's heads at most
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

// WHOLE: pieces of 16 bytes hold no part of what is turned apart; EIGHTS: as
// above. Each next unit of the queries, and each next four tokens of a wave's
// heads, are on their way while the ones before are turned.
template <int T, int LP, bool WHOLE, bool EIGHTS>
__global__ __launch_bounds__(64 * kMostWaves4) void kv4_append_rows(Append4Args a) {
  typedef num_t<T> V;
  typedef Num<T> F;
  typedef Split4<LP> S;
  constexpr int N = WHOLE ? 16 / sizeof(V) : 1;
  __shared__ v2f cs[kPlaces][128];
  __shared__ uint32_t words[kMostWaves4][S::WORDS];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int threads = blockDim.x, waves = threads / 64;
  const Block16 k16 = block_of(a.c, a.starts, a.rows, a.batch, blockIdx.x);
  if (k16.b < 0) return;
  const TurnArgs &t = a.t;
  const int dim = a.c.dim, half = t.rotary / 2;

  // The queries' units, token by token.
  struct Q {
    V p[N], r[N];
    int token, h;
    Unit o;
  };
  const int items = t.heads * a.units, last = (k16.to - k16.from) * items - 1;
  auto load_q = [&](int i) {
    Q q;
    i = min(i, last);
    q.token = a.by_items(i);
    i -= q.token * items;
    q.token += k16.from;
    q.h = a.by_unit(i);
    q.o = unit_of<N>(i - q.h * a.units, dim, t.rotary, t.pairs);
    const V *from = (const V *)t.q + (k16.row0 + q.token) * t.q_stride + (long)q.h * dim;
    __builtin_memcpy(q.p, from + q.o.d1, sizeof q.p);
    __builtin_memcpy(q.r, from + (q.o.d2 < dim ? q.o.d2 : q.o.d1), sizeof q.r);
    return q;
  };
  Q q;
  if (t.q) q = load_q(threadIdx.x);
  for (int i = threadIdx.x; i < (k16.to - k16.from) * half; i += threads) {
    const int token = k16.from + a.by_half(i), j = i - (token - k16.from) * half;
    const double at = t.positions ? (double)t.positions[k16.row0 + token] : (double)(k16.place + token);
    cs[token][j] = cosine_sine(at * (double)t.freqs[j]);
  }
  __syncthreads();
  if (t.q) {
    for (int i = threadIdx.x; i <= last; i += threads) {
      const Q next = load_q(i + threads);
      if (q.o.turned) turn_unit<T, N>(q.p, q.r, cs[q.token], q.o, t.rotary, t.pairs);
      V *into = (V *)t.q_out + (k16.row0 + q.token) * t.q_out_stride + (long)q.h * dim;
      __builtin_memcpy(into + q.o.d1, q.p, sizeof q.p);
      if (q.o.d2 < dim) __builtin_memcpy(into + q.o.d2, q.r, sizeof q.r);
      q = next;
    }
  }
  if (!k16.chunk) return;

  // Keys and values: four tokens (or twice two) of some heads a wave at a time.
  const int l = lane % LP, d = 8 * l, have = min(max(dim - d, 0), 8);
  const int nc = a.c.nc, block = l / 4, quarter = l % 4;
  const int lanes = min(a.c.group / 8, LP);  // of a group
  const int group = l / lanes;
  const int four0 = k16.from / 4, fours = (k16.to + 3) / 4 - four0;
  const int jobs = (a.c.heads + S::HEADS - 1) / S::HEADS * fours;  // job j: fours j % fours, heads j / fours
  auto load_kv = [&](int j, int pass) {
    const int r = lane / LP + pass * (64 / LP), h = min(j / fours * S::HEADS + r / 4, a.c.heads - 1);
    const long row = k16.row0 + min(max(4 * (four0 + j % fours) + r % 4, k16.from), k16.to - 1);  // (one that there is)
    return load_eight<EIGHTS>((const V *)a.k + row * a.k_stride + (long)h * dim,
                              (const V *)a.v + row * a.v_stride + (long)h * dim, EIGHTS ? min(d, dim - 8) : d, dim, t);
  };
  int job = wave;
  if (job >= jobs) return;
  Eight<V> ahead[S::PASSES];
#pragma unroll
  for (int pass = 0; pass < S::PASSES; pass++) ahead[pass] = load_kv(job, pass);
  for (; job < jobs; job += waves) {
    const int h0 = job / fours * S::HEADS, four = four0 + job % fours;
    const int from = k16.from - 4 * four, to = k16.to - 4 * four;
#pragma unroll
    for (int pass = 0; pass < S::PASSES; pass++) {
      const int row = lane / LP + pass * (64 / LP), token = row % 4, h = h0 + row / 4;
      const bool on = token >= from && token < to && h < a.c.heads;
      const Eight<V> raw = ahead[pass];
      ahead[pass] = load_kv(min(job + waves, jobs - 1), pass);
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
      const uint32_t kw = quantise(k, on ? have : 0, lanes, ks, km), vw = quantise(v, on ? have : 0, lanes, vs, vm);
      if (on && block < nc) {
        char *chunk = k16.chunk + (long)h * a.c.chunk;
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
        char *into = k16.chunk + (long)h * a.c.chunk + a.c.at_v + (long)(k16.slot / 4 + four) * 64 * nc + 4 * w;
        const uint32_t word = words[wave][i];
        if (from <= 0 && to >= 4) {
          *(uint32_t *)into = word;
        } else {
          for (int token = max(from, 0); token < min(to, 4); token++) into[token] = (char)(word >> 8 * token);
        }
      }
    }
    wave_sync();
  }
}

// A wave's words of V, its lanes' words of K and their scales are asked for
// together, and the next four tokens' before these are written.
template <int T, int LP>
__global__ __launch_bounds__(64 * kMostWaves4) void kv4_read_rows(Read4Args a) {
  typedef num_t<T> V;
  typedef Num<T> F;
  typedef Split4<LP> S;
  __shared__ uint32_t words[kMostWaves4][S::WORDS];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64;
  const Block16 k16 = block_of(a.c, a.starts, a.rows, a.batch, blockIdx.x);
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
  Held held = load(job);
  for (; job < jobs; job += waves) {
    const int h0 = job / fours * S::HEADS, four = four0 + job % fours;
    const Held next = load(min(job + waves, jobs - 1));
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
        k[j] = F::put(fmaf((float)(held.k[pass] >> 4 * j & 15), ks, km));
        v[j] = F::put(fmaf((float)(w >> 4 * j & 15), vs, vm));
      }
      const long row = k16.row0 + token;
      store_n((V *)a.k + row * a.k_stride + (long)h * dim + d, have, k);
      store_n((V *)a.v + row * a.v_stride + (long)h * dim + d, have, v);
    }
    wave_sync();
    held = next;
  }
}

inline unsigned blocks4(long rows, int batch) {
  return unsigned((rows + (2 * kPlaces - 2L) * batch) / kPlaces + 1);
}

// Four waves, or eight where the keys and values of 16 tokens have work for them.
template <int LP>
dim3 threads4(int heads, long rows, int batch) {
  const int jobs = (heads + Split4<LP>::HEADS - 1) / Split4<LP>::HEADS * (rows > batch ? 4 : 1);
  return dim3(64 * (jobs > 4 ? kMostWaves4 : 4));
}

template <int T, int LP>
hipError_t launch_append4(Append4Args a, hipStream_t s) {
  constexpr int N = 16 / sizeof(num_t<T>);
  const bool whole = whole_pieces(N, a.c.dim, a.t.rotary, a.t.pairs);
  const bool eights = a.c.dim % 8 == 0 && (a.t.pairs || a.t.rotary % 16 == 0);
  a.units = units_of(whole && eights ? N : 1, a.c.dim, a.t.rotary, a.t.pairs);
  a.by_unit = Divide(a.units);
  a.by_items = Divide(std::max(a.t.heads * a.units, 1)), a.by_half = Divide(std::max(a.t.rotary / 2, 1));
  const dim3 grid(blocks4(a.rows, a.batch)), block = threads4<LP>(a.c.heads, a.rows, a.batch);
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
  return launch_kernel(kv4_read_rows<T, LP>, dim3(blocks4(a.rows, a.batch)), threads4<LP>(a.c.heads, a.rows, a.batch), 0, s, a);
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
