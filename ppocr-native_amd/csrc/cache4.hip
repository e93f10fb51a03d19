// The paged cache held in 4 bits: appending to it, with the rotation of keys
// and queries on the way (ppocr_hip_kv4_append), and reading tokens back as rows
// (ppocr_hip_kv4_read).
//
//   a group's m = f16(min x), s = f16((max x - m) / 15), n = round((x - m) / s)
//
// A workgroup has four tokens whose places are one of V's blocks, where a code
// word is four tokens' bytes: a lane has eight neighbouring dims of one of them,
// which are a word of K's codes and a byte of each of four words of V's. Those
// go through a wave's own piece of LDS, so that memory sees whole words.
#include <algorithm>

#include "turn.hpp"

namespace ppocr {
namespace {

constexpr int kWaves4 = 4;

// The block of four places that workgroup g has, with as many workgroups for
// each text as its rows could touch blocks: text b's begin at (its first row +
// 6 b) / 4.
struct Block4 {
  int b;        // text, or -1
  long row0;    // the row whose place is the block's first (it may not exist)
  int from, to; // tokens of the block that are rows
  long place;   // the block's first place
  char *chunk;  // its page's chunk of head 0, or NULL
  int slot;     // its first token's number in the page
};

__device__ __forceinline__ long clamped(long v, long most) { return min(max(v, 0L), most); }

__device__ __forceinline__ Block4 block_of(const Kv4Args &c, const int *starts, long rows, int batch, long g) {
  Block4 o;
  o.b = -1;
  o.chunk = nullptr;
  auto start = [&](int i) { return (clamped(starts ? starts[i] : i, rows) + 6L * i) / 4; };
  int b = last_not_past(batch + 1, g, start);
  b = __builtin_amdgcn_readfirstlane(b);
  if (b < 0 || b >= batch) return o;
  long first = b, last = b + 1L;
  if (starts) first = starts[b], last = starts[b + 1];
  const long count = last - first, base = (long)c.lengths[b] - count;  // row first + i has place base + i
  const long begin = max(max(0L, -first), -base), end = min(count, rows - first);
  if (begin >= end) return o;
  o.place = (base + begin) / 4 * 4 + 4 * (g - start(b));
  if (o.place >= base + end) return o;
  o.b = b;
  o.row0 = first + o.place - base;
  o.from = (int)max(0L, base + begin - o.place);
  o.to = (int)min(4L, base + end - o.place);
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

// WHOLE: pieces of 16 bytes hold no part of what is turned apart.
template <int T, int LP, bool WHOLE>
__global__ __launch_bounds__(64 * kWaves4) void kv4_append_rows(Append4Args a) {
  typedef num_t<T> V;
  typedef Num<T> F;
  typedef Split4<LP> S;
  constexpr int N = WHOLE ? 16 / sizeof(V) : 1;
  __shared__ v2f cs[4][128];
  __shared__ uint32_t words[kWaves4][S::WORDS];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const Block4 k4 = block_of(a.c, a.starts, a.rows, a.batch, blockIdx.x);
  if (k4.b < 0) return;
  const TurnArgs &t = a.t;
  const int dim = a.c.dim, half = t.rotary / 2;
  for (int i = threadIdx.x; i < 4 * half; i += 64 * kWaves4) {
    const int token = i / half, j = i - token * half;
    if (token < k4.from || token >= k4.to) continue;
    const double at = t.positions ? (double)t.positions[k4.row0 + token] : (double)(k4.place + token);
    cs[token][j] = cosine_sine(at * (double)t.freqs[j]);
  }
  __syncthreads();

  // The queries.
  if (t.q) {
    const int items = t.heads * a.units;
    for (int token = k4.from; token < k4.to; token++)
      for (int i = threadIdx.x; i < items; i += 64 * kWaves4) {
        const int h = a.by_unit(i);
        const Unit o = unit_of<N>(i - h * a.units, dim, t.rotary, t.pairs);
        const V *from = (const V *)t.q + (k4.row0 + token) * t.q_stride + (long)h * dim;
        V *into = (V *)t.q_out + (k4.row0 + token) * t.q_out_stride + (long)h * dim;
        V p[N], r[N];
        __builtin_memcpy(p, from + o.d1, sizeof p);
        __builtin_memcpy(r, from + (o.d2 < dim ? o.d2 : o.d1), sizeof r);
        if (o.turned) turn_unit<T, N>(p, r, cs[token], o, t.rotary, t.pairs);
        __builtin_memcpy(into + o.d1, p, sizeof p);
        if (o.d2 < dim) __builtin_memcpy(into + o.d2, r, sizeof r);
      }
  }
  if (!k4.chunk) return;

  // Keys and values.
  const int l = lane % LP, d = 8 * l, have = min(max(dim - d, 0), 8);
  const int nc = a.c.nc, block = l / 4, quarter = l % 4;
  const int lanes = min(a.c.group / 8, LP);  // of a group
  const int group = l / lanes;
  for (int h0 = wave * S::HEADS; h0 < a.c.heads; h0 += kWaves4 * S::HEADS) {
#pragma unroll
    for (int pass = 0; pass < S::PASSES; pass++) {
      const int r = lane / LP + pass * (64 / LP), token = r % 4, h = h0 + r / 4;
      const bool on = token >= k4.from && token < k4.to && h < a.c.heads;
      const long row = k4.row0 + token;
      float k[8] = {}, other[8] = {}, v[8] = {};
      if (on && have > 0) {
        const V *kr = (const V *)a.k + row * a.k_stride + (long)h * dim;
        const V *vr = (const V *)a.v + row * a.v_stride + (long)h * dim;
        // The dims that d's are turned with, where those are half a head away.
        const int far = t.pairs || d >= t.rotary ? d : d < half ? d + half : d - half;
        V raw[8], raw2[8], raw3[8];
        if constexpr (WHOLE) {
          if (dim % 8 == 0 && half % 8 == 0) {
            __builtin_memcpy(raw, kr + d, sizeof raw);
            __builtin_memcpy(raw2, kr + far, sizeof raw2);
            __builtin_memcpy(raw3, vr + d, sizeof raw3);
          } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
              const int e = min(d + j, dim - 1);
              raw[j] = kr[e], raw3[j] = vr[e];
              raw2[j] = kr[t.pairs || e >= t.rotary ? e : e < half ? e + half : e - half];
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const int e = min(d + j, dim - 1);
            raw[j] = kr[e], raw3[j] = vr[e];
            raw2[j] = kr[t.pairs || e >= t.rotary ? e : e < half ? e + half : e - half];
          }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) k[j] = F::get(raw[j]), other[j] = F::get(raw2[j]), v[j] = F::get(raw3[j]);
        if (t.pairs) {
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            if (d + j < t.rotary) {
              const v2f c = cs[token][d / 2 + j / 2];
              const float x = k[j], y = k[j + 1];
              k[j] = x * c[0] - y * c[1], k[j + 1] = y * c[0] + x * c[1];
            }
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (d + j < t.rotary) {
              const bool second = d + j >= half;
              const v2f c = cs[token][d + j - (second ? half : 0)];
              k[j] = second ? k[j] * c[0] + other[j] * c[1] : k[j] * c[0] - other[j] * c[1];
            }
        }
      }
      // (Lanes without a row go along: their neighbours' ranges are of other rows.)
      uint16_t ks, km, vs, vm;
      const uint32_t kw = quantise(k, on ? have : 0, lanes, ks, km), vw = quantise(v, on ? have : 0, lanes, vs, vm);
      if (on && block < nc) {
        char *chunk = k4.chunk + (long)h * a.c.chunk;
        const int slot = k4.slot + token;
        *(uint32_t *)(chunk + (long)slot * 16 * nc + 4 * (nc * quarter + block)) = kw;
        if (l % lanes == 0 && group < a.c.groups) {
          const int at = 2 * (slot * a.c.groups + group);
          *(uint16_t *)(chunk + a.c.at_ks + at) = ks, *(uint16_t *)(chunk + a.c.at_km + at) = km;
          *(uint16_t *)(chunk + a.c.at_vs + at) = vs, *(uint16_t *)(chunk + a.c.at_vm + at) = vm;
        }
        uint8_t *into = (uint8_t *)(words[wave] + r / 4 * 16 * nc);
#pragma unroll
        for (int j = 0; j < 4; j++) into[((4 * quarter + j) * nc + block) * 4 + token] = (uint8_t)(vw >> 8 * j);
      }
    }
    wave_sync();
    for (int i = lane; i < S::HEADS * 16 * nc; i += 64) {
      const int h = h0 + i / (16 * nc), w = i % (16 * nc);
      if (h < a.c.heads) {
        char *into = k4.chunk + (long)h * a.c.chunk + a.c.at_v + (long)(k4.slot / 4) * 64 * nc + 4 * w;
        const uint32_t word = words[wave][i];
        if (k4.from == 0 && k4.to == 4) {
          *(uint32_t *)into = word;
        } else {
          for (int token = k4.from; token < k4.to; token++) into[token] = (char)(word >> 8 * token);
        }
      }
    }
    wave_sync();
  }
}

template <int T, int LP>
__global__ __launch_bounds__(64 * kWaves4) void kv4_read_rows(Read4Args a) {
  typedef num_t<T> V;
  typedef Num<T> F;
  typedef Split4<LP> S;
  __shared__ uint32_t words[kWaves4][S::WORDS];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const Block4 k4 = block_of(a.c, a.starts, a.rows, a.batch, blockIdx.x);
  if (k4.b < 0) return;
  const int l = lane % LP, d = 8 * l, dim = a.c.dim, have = min(max(dim - d, 0), 8);
  const int nc = a.c.nc, block = l / 4, quarter = l % 4;
  const int group = min(d / a.c.group, a.c.groups - 1);
  for (int h0 = wave * S::HEADS; h0 < a.c.heads; h0 += kWaves4 * S::HEADS) {
    if (k4.chunk) {
      for (int i = lane; i < S::HEADS * 16 * nc; i += 64) {
        const int h = min(h0 + i / (16 * nc), a.c.heads - 1), w = i % (16 * nc);
        words[wave][i] = *(const uint32_t *)(k4.chunk + (long)h * a.c.chunk + a.c.at_v +
                                             (long)(k4.slot / 4) * 64 * nc + 4 * w);
      }
    }
    wave_sync();
#pragma unroll
    for (int pass = 0; pass < S::PASSES; pass++) {
      const int r = lane / LP + pass * (64 / LP), token = r % 4, h = h0 + r / 4;
      if (token < k4.from || token >= k4.to || h >= a.c.heads || have == 0) continue;
      uint32_t kw = 0, vw = 0;
      float ks, km, vs, vm;
      ks = km = vs = vm = __uint_as_float(0x7fc00000u);  // no page: NaN
      if (k4.chunk) {
        const char *chunk = k4.chunk + (long)h * a.c.chunk;
        const int slot = k4.slot + token, at = 2 * (slot * a.c.groups + group);
        kw = *(const uint32_t *)(chunk + (long)slot * 16 * nc + 4 * (nc * quarter + block));
        ks = (float)*(const _Float16 *)(chunk + a.c.at_ks + at), km = (float)*(const _Float16 *)(chunk + a.c.at_km + at);
        vs = (float)*(const _Float16 *)(chunk + a.c.at_vs + at), vm = (float)*(const _Float16 *)(chunk + a.c.at_vm + at);
        const uint8_t *from = (const uint8_t *)(words[wave] + r / 4 * 16 * nc);
#pragma unroll
        for (int j = 0; j < 4; j++) vw |= (uint32_t)from[((4 * quarter + j) * nc + block) * 4 + token] << 8 * j;
      }
      V k[8], v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        k[j] = F::put(fmaf((float)(kw >> 4 * j & 15), ks, km));
        v[j] = F::put(fmaf((float)(vw >> 4 * j & 15), vs, vm));
      }
      const long row = k4.row0 + token;
      store_n((V *)a.k + row * a.k_stride + (long)h * dim + d, have, k);
      store_n((V *)a.v + row * a.v_stride + (long)h * dim + d, have, v);
    }
    wave_sync();
  }
}

inline unsigned blocks4(long rows, int batch) { return unsigned((rows + 6L * batch) / 4 + 1); }

template <int T, int LP>
hipError_t launch_append4(Append4Args a, hipStream_t s) {
  constexpr int N = 16 / sizeof(num_t<T>);
  const bool whole = whole_pieces(N, a.c.dim, a.t.rotary, a.t.pairs);
  a.units = units_of(whole ? N : 1, a.c.dim, a.t.rotary, a.t.pairs);
  a.by_unit = Divide(a.units);
  const dim3 grid(blocks4(a.rows, a.batch)), block(64 * kWaves4);
  if (whole) return launch_kernel(kv4_append_rows<T, LP, true>, grid, block, 0, s, a);
  return launch_kernel(kv4_append_rows<T, LP, false>, grid, block, 0, s, a);
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

template <int T>
hipError_t launch_read4_of(const Read4Args &a, hipStream_t s) {
  const dim3 grid(blocks4(a.rows, a.batch)), block(64 * kWaves4);
  switch (a.c.nc) {
    case 1: return launch_kernel(kv4_read_rows<T, 4>, grid, block, 0, s, a);
    case 2: return launch_kernel(kv4_read_rows<T, 8>, grid, block, 0, s, a);
    case 3:
    case 4: return launch_kernel(kv4_read_rows<T, 16>, grid, block, 0, s, a);
  }
  return launch_kernel(kv4_read_rows<T, 32>, grid, block, 0, s, a);
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
