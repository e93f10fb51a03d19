// Causal attention of prompts with a sliding window and sinks
// (ppocr_hip_window_attention).
#include "attend.hpp"
#include "kernels.hpp"

namespace ppocr {
namespace {

// A block of queries: which text, and which of its rows. Blocks are counted
// through the texts; there are at most rows_q / size + batch.
struct Block {
  int q0, nq;  // the text's first row of q and its queries
  int k0, nk;
  int first;  // the block's first query in its text
};

// The sum of the lanes' v, each below 2^bits, by its bits.
__device__ __forceinline__ int wave_total(int v, int bits) {
  int s = 0;
  for (int i = 0; i < bits; i++) s += __popcll(__ballot(v >> i & 1)) << i;
  return s;
}

// Finds block `index`; false if there are fewer. Every wave of a workgroup
// walks the starts, 64 texts at a time. Of those, blocks that are far into
// their text come first, as they see most keys, so that the last to run are
// short (14 texts of up to 6971 tokens, one head of 256 in f32, 2.6 ms text by
// text, 2.1 so; 20 of up to 3000, 4 heads of 128 in bf16, 155 and 132 us; but two
// of up to 3000, 12 heads of 96 in f32, 409 and 439). Blocks further in than the
// window see as many keys as one another and come text by text: neighbours share
// most of them. Starts past the rows there are, and such as decrease, leave texts
// of no rows. (The walk is all that short texts by the thousand wait for: 1000 of
// 8 tokens, 8 heads of 64, 87 us, 8000 of 4 2.3 ms.)
__device__ __forceinline__ bool find_block(const PromptArgs &a, int index, int size, Block &out) {
  const int lane = threadIdx.x % 64, far = a.window ? a.window / size + 1 : 1 << 30;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int b = b0 + lane;
    int q0 = 0, nq = 0;
    if (b < a.batch) {
      q0 = min(max(a.starts_q[b], 0), a.rows_q);
      nq = max(min(a.starts_q[b + 1], a.rows_q) - q0, 0);
    }
    const int blocks = (nq + size - 1) / size, near = min(blocks, far);
    int bits = 0;
    while (__any(blocks >> bits)) bits++;
    const int all = wave_total(blocks, bits);
    if (index >= all) {
      index -= all;
      continue;
    }
    int n = 0, at;
    const int beyond = wave_total(blocks - near, bits);
    if (index < beyond) {
      int upto = blocks - near;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o);
        if (lane >= o) upto += v;
      }
      at = __ffsll(__ballot(upto > index)) - 1;
      n = far + __shfl(upto, at) - 1 - index;
    } else {
      // Block number n, the largest of which there are more than `index` blocks
      // with that number or a higher one; `above` have a higher one.
      index -= beyond;
      int above = 0;
      for (int i = bits - 1; i >= 0; i--) {
        const int more = wave_total(max(near - n - (1 << i), 0), bits);
        if (more > index)
          n += 1 << i;
        else
          above = more;
      }
      const unsigned long long has = __ballot(near > n);
      const int before = __popcll(has & ((1ull << lane) - 1));
      at = __ffsll(__ballot(near > n && before == index - above)) - 1;
    }
    out.q0 = __shfl(q0, at);
    out.nq = __shfl(nq, at);
    out.first = n * size;
    const int text = b0 + at;
    out.k0 = min(max(a.starts_k[text], 0), a.rows_k);
    out.nk = max(min(a.starts_k[text + 1], a.rows_k) - out.k0, 0);
    return true;
  }
  return false;
}

// Queries first .. first + count - 1 of a block's text by one wave, one after
// another and every key by itself, so that nothing of an unseen key (an
// infinity or NaN in V) reaches a query: what the fast kernels fall back to
// where they meet one next to a mask. A lane is a key, then a value of dim.
template <int T>
__device__ __forceinline__ void attend_alone(const PromptArgs &a, const Block &bl, int head, int first, int count) {
  typedef num_t<T> V;
  const int lane = threadIdx.x % 64, kv = head / (a.heads / a.kv_heads);
  const V *k = (const V *)a.k + (long)bl.k0 * a.k_stride + (long)kv * a.dim;
  const V *v = (const V *)a.v + (long)bl.k0 * a.v_stride + (long)kv * a.dim;
  for (int i = first; i < min(first + count, bl.nq); i++) {
    const V *q = (const V *)a.q + (long)(bl.q0 + i) * a.q_stride + (long)head * a.dim;
    const int p = bl.nk - bl.nq + i, low = a.window ? max(p - a.window + 1, 0) : 0;
    auto seen = [&](int j) { return j <= p && (j >= low || j < a.sinks); };
    float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
    for (int j0 = 0; j0 <= p; j0 += 64) {
      if (j0 + 63 < low && j0 >= a.sinks) continue;
      const int j = j0 + lane;
      float s = -INFINITY;
      if (seen(j)) {
        s = 0.0f;
        for (int d = 0; d < a.dim; d++) s = fmaf(Num<T>::get(q[d]), Num<T>::get(k[j * a.k_stride + d]), s);
        s *= a.turn ? -a.scale : a.scale;
      }
      float top = s;
#pragma unroll
      for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
      const float now = fmaxf(m, top), base = now == -INFINITY ? 0.0f : now;
      const float shrink = __builtin_amdgcn_exp2f(m - base);
      const float w = seen(j) ? __builtin_amdgcn_exp2f(s - base) : 0.0f;
      m = now;
      l = l * shrink + w;
#pragma unroll
      for (int c = 0; c < 4; c++) o[c] *= shrink;
      for (int u = 0; u < 64; u++) {
        if (!seen(j0 + u)) continue;
        const float wu = __shfl(w, u);
#pragma unroll
        for (int c = 0; c < 4; c++)
          if (lane + 64 * c < a.dim) o[c] = fmaf(wu, Num<T>::get(v[(j0 + u) * a.v_stride + lane + 64 * c]), o[c]);
      }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
    V *y = (V *)a.y + (long)(bl.q0 + i) * a.y_stride + (long)head * a.dim;
#pragma unroll
    for (int c = 0; c < 4; c++)
      if (lane + 64 * c < a.dim) y[lane + 64 * c] = Num<T>::put(l == 0.0f ? 0.0f : o[c] / l);
  }
}

// 16 queries of one head, from the block's query `first` on, by one wave,
// keys and values straight from memory (the caches): any type and dim. Two tiles
// are in registers, of which heads past 64 spill some, and value by value most:
// four texts of up to 1500 tokens, 8 heads of 129 in bf16, take 2.8 ms, where 128
// in tiles take 47 us.
template <int T, int DP, int DIMS>
__device__ __forceinline__ void attend_rows(const PromptArgs &a, const Block &bl, int head, int first) {
  typedef Attend<T, DP, DIMS> A;
  typedef typename A::V V;
  constexpr int K = A::KEYS;
  const int lane = threadIdx.x % 64, col = lane % 16, quarter = lane / 16;
  const int kv = head / (a.heads / a.kv_heads);
  const int rows = min(16, bl.nq - first);
  const int p0 = bl.nk - bl.nq + first;  // the first query's place; the last's is p0 + rows - 1
  const int p = p0 + min(col, rows - 1);
  A at;
  at.start((const V *)a.q + (long)(bl.q0 + first + min(col, rows - 1)) * a.q_stride + (long)head * a.dim, a.dim,
           quarter, a.turn);
  const V *k = (const V *)a.k + (long)bl.k0 * a.k_stride + (long)kv * a.dim;
  const V *v = (const V *)a.v + (long)bl.k0 * a.v_stride + (long)kv * a.dim;
  const int last = p0 + rows - 1;                            // of all rows' keys
  const int low = a.window ? max(p0 - a.window + 1, 0) : 0;  // the first row's window starts here
  const int sinks = min(a.sinks, low);                       // sinks before every window
  const int start = low / K * K, sink_tiles = min((sinks + K - 1) / K, start / K);
  const int tiles = sink_tiles + (last >= start ? (last - start) / K + 1 : 0);
  auto tile_key = [&](int t) { return t < sink_tiles ? t * K : start + (t - sink_tiles) * K; };
  auto load = [&](typename A::Tile &tile, int t) {
    const int k0 = tile_key(t);
    A::load(
        tile, [&](int i) { return k + (long)min(k0 + i, bl.nk - 1) * a.k_stride; },
        [&](int i) { return v + (long)min(k0 + i, bl.nk - 1) * a.v_stride; }, a.dim, lane);
  };
  bool bad = false;
  auto use = [&](typename A::Tile &tile, int t) {
    const int k0 = tile_key(t);
    const bool masked = k0 + K - 1 > p0 || (a.window && k0 <= last - a.window);
    auto seen = [&](int i) {
      const int j = k0 + i;
      return j <= p && (!a.window || j > p - a.window || j < a.sinks);
    };
    auto any = [&](int i) {  // whether some row sees it
      const int j = k0 + i;
      return j <= last && (j >= low || j < a.sinks);
    };
    bad |= at.template use<true>(tile, seen, any, masked, a.dim, a.scale, lane);
  };
  typename A::Tile ta, tb;
  if (tiles > 0) load(ta, 0);
  for (int t = 0; t < tiles; t += 2) {
    if (t + 1 < tiles) load(tb, t + 1);
    use(ta, t);
    if (t + 1 >= tiles) break;
    if (t + 2 < tiles) load(ta, t + 2);
    use(tb, t + 1);
  }
  if (__any(bad)) {
    attend_alone<T>(a, bl, head, first, rows);
    return;
  }
  const float l = at.total();
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  if (col >= rows) return;
  V *y = (V *)a.y + (long)(bl.q0 + first + col) * a.y_stride + (long)head * a.dim;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    V out[A::E];
#pragma unroll
    for (int e = 0; e < A::E; e++) out[e] = Num<T>::put(l == 0.0f ? 0.0f : at.o[e][r] * f);
    const int d = A::E * (4 * quarter + r);
    store_n(y + d, (long)a.dim - d, out);
  }
}

template <int T, int DP, int DIMS>
__global__ __launch_bounds__(256, (DP <= 128 ? 2 : 1)) void window_attention_rows(PromptArgs a) {
  Block bl;
  if (!find_block(a, blockIdx.x / a.heads, 64, bl)) return;
  const int per = a.heads / a.kv_heads, x = blockIdx.x % a.heads;
  const int first = bl.first + threadIdx.x / 64 * 16;
  if (first < bl.nq) attend_rows<T, DP, DIMS>(a, bl, x % a.kv_heads * per + x / a.kv_heads, first);
}

// ------------------------------------------------------------- tiles in LDS

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

constexpr int kTileWaves = 4;
// The running maximum follows where it grew by a factor of 2^kGrow or more, and
// weights are held 2^kUp times as large: up to 2^(kGrow + kUp). F16 has numbers
// from 2^-24 to 65504, with all 11 bits from 2^-14 on, so its weights keep those
// down to 2^-27 of the largest (e^-18.7: far below the one key ahead of all,
// theirs are what counts if its value is near 0) and are off by 2^-38 of it at
// most; following as soon as that takes 2 to 3 % longer (8192 tokens, 32 heads of
// 128: 636 and 651 us). BF16 has f32's range.
template <int T>
constexpr float kGrow = T == PPOCR_F16 ? 2.0f : 8.0f;
template <int T>
constexpr float kUp = T == PPOCR_F16 ? 13.0f : 0.0f;
template <int T>
constexpr int kTileKeys = T == PPOCR_F32 ? 32 : 64;
// 16-byte pieces that a row of a tile has room for.
template <int T, int DP>
constexpr int kPieces = (DP <= 64 ? 8 : DP <= 128 ? 16 : 32) * (T == PPOCR_F32 ? 2 : 1);

// Where a key's row of a tile keeps its 16-byte piece c: place c ^ turn(key),
// so that both the 16 rows that a read of K touches at one piece and the four
// rows of four pieces that a transposing read of V touches lie in different
// banks. C: pieces a row has room for.
template <int C>
__device__ __forceinline__ int turn(int key) {
  return C == 8 ? (key >> 1 & 1) << 2 | (key >> 2 & 3) : (key & 3) << 2 | (key >> 2 & 3);
}

// Whether a dword holds an infinity or NaN.
template <int T>
__device__ __forceinline__ int not_finite2(uint32_t x) {
  if constexpr (T == PPOCR_F32) return (x & 0x7f800000u) == 0x7f800000u;
  constexpr uint32_t lo = T == PPOCR_F16 ? 0x7c00u : 0x7f80u, hi = lo << 16;
  return ((x & lo) == lo ? 1 : 0) + ((x & hi) == hi ? 1 : 0);
}

// Four waves, each 32 queries of one head; `hg` heads of one key head (1, 2 or
// 4) share the workgroup's tiles of 64 keys and values (32 in f32), which go
// straight from memory to LDS, the next tile's while this one's are used. The
// 32 queries are the columns of each product:
//   S^T[key][query] = K Q^T, O^T[d][query] += V^T P^T,
// so that a lane holds one query's numbers: row maxima and sums need one
// exchange between the wave's halves, and P goes from the first product's
// result to the second's operand in its own lane, in 16 bits rounded to T, its
// keys in the order 4 (lane / 32) + {0..3, 8..11}; V is read to match, in 16
// bits transposed on its way out of LDS. In f32 the products take two inner
// values at a time, and V's column d = E (lane % 32) + e is row lane % 32 of
// product e. (With the keys of each wave's 16 queries read from memory in the
// operand's order instead, f32 ran at 60 TFLOP/s: the address unit takes a
// cycle a lane.)
// What bounds it: the matrix cores, which a wave's softmax leaves waiting where
// the other wave of its SIMD has none of its own to do. One text of 8192
// tokens, 32 heads of 128 in bf16: 0.63 ms, 874 TFLOP/s of the seen keys'
// products, where a library product of 8192 x 8192 x 8192 runs at 1124 (f32: 4.3
// ms, 129 of 154); a window of 2048 over two such texts 0.32 to 0.36 ms, 720 to
// 800 TFLOP/s. Eight waves
// a workgroup: 2 to 3 % faster on these, 10 to 16 % slower on heads of 64 and on
// 1115 tokens of 4 heads.
// WHOLE: dim == DP and fills the pieces.
template <int T, int DP, bool WHOLE>
__global__ __launch_bounds__(64 * kTileWaves, DP <= 128 ? 2 : 1) void window_attention_tiles(PromptArgs a, int hg) {
  typedef num_t<T> V;
  constexpr bool F32 = T == PPOCR_F32;
  constexpr int C = kPieces<T, DP>, KEYS = kTileKeys<T>, PN = 16 / sizeof(V);
  constexpr int TILE = KEYS * C * 16;  // bytes
  constexpr int KS = F32 ? DP / 8 : DP / 16, DB = DP / 32, PIECES = KEYS * C / (64 * kTileWaves), SB = KEYS / 32;
  extern __shared__ __attribute__((aligned(1024))) char lds[];  // [2][K, V][TILE]
  // Workgroups in a row are a block's key heads (and the query heads of each,
  // hg at a time): with eight, each XCD has its own, whose keys stay in its L2.
  const int across = a.heads / hg, index = blockIdx.x / across, x = blockIdx.x % across;
  const int size = 32 * kTileWaves / hg;
  Block bl;
  if (!find_block(a, index, size, bl)) return;
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int half = lane / 32, col = lane % 32;
  const int per = a.heads / a.kv_heads, kv = x % a.kv_heads;
  const int head = kv * per + x / a.kv_heads * hg + wave % hg;
  const int w0 = bl.first + wave / hg * 32;  // this wave's first query
  const int p_first = bl.nk - bl.nq + bl.first, p_last = bl.nk - bl.nq + min(bl.first + size, bl.nq) - 1;
  const int query = min(w0 + col, bl.nq - 1), p = bl.nk - bl.nq + query;
  const int pw_first = bl.nk - bl.nq + w0, pw_last = bl.nk - bl.nq + min(w0 + 32, bl.nq) - 1;

  const int p_low = a.window ? p - a.window + 1 : 0;  // this query's window

  // The tiles that the block sees: of sinks, then of the windows.
  const int low = a.window ? max(p_first - a.window + 1, 0) : 0;
  const int sinks = min(a.sinks, low), start = low / KEYS * KEYS;
  const int sink_tiles = min((sinks + KEYS - 1) / KEYS, start / KEYS);
  const int tiles = sink_tiles + (p_last >= start ? (p_last - start) / KEYS + 1 : 0);
  auto tile_key = [&](int t) { return t < sink_tiles ? t * KEYS : start + (t - sink_tiles) * KEYS; };

  const int pieces = a.dim / PN;  // WHOLE: C
  if (!WHOLE) {  // pieces past dim stay zero
    for (int i = tid; i < 4 * TILE / 16; i += 64 * kTileWaves) ((v4u *)lds)[i] = v4u{0, 0, 0, 0};
    __syncthreads();
  }
  const char *k_base = (const char *)((const V *)a.k + (long)bl.k0 * a.k_stride + (long)kv * a.dim);
  const char *v_base = (const char *)((const V *)a.v + (long)bl.k0 * a.v_stride + (long)kv * a.dim);
  auto load = [&](int t, int buffer) {
    const int k0 = tile_key(t);
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
      const int e = (i * kTileWaves + wave) * 64 + lane, row = e / C, piece = (e % C) ^ turn<C>(row);
      const int v_piece = F32 ? e % C : piece;  // (f32 rows of V are read along the row)
      const long key = min(k0 + row, bl.nk - 1);
      char *to = lds + buffer * 2 * TILE + (i * kTileWaves + wave) * 1024;
      if (WHOLE || piece < pieces)
        __builtin_amdgcn_global_load_lds((const void *)(k_base + key * a.k_stride * (long)sizeof(V) + piece * 16),
                                         (lds_void *)to, 16, 0, 0);
      if (WHOLE || v_piece < pieces)
        __builtin_amdgcn_global_load_lds((const void *)(v_base + key * a.v_stride * (long)sizeof(V) + v_piece * 16),
                                         (lds_void *)(to + TILE), 16, 0, 0);
    }
  };

  v4u q[KS];
  {
    const V *row = (const V *)a.q + (long)(bl.q0 + query) * a.q_stride + (long)head * a.dim;
    const uint32_t sign = a.turn ? (F32 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const int d = PN * (2 * s + half);
      q[s] = v4u{0, 0, 0, 0};
      if (d < a.dim) __builtin_memcpy(&q[s], row + d, 16);
#pragma unroll
      for (int i = 0; i < 4; i++) q[s][i] ^= sign;
    }
  }
  v16f o[DB];
#pragma unroll
  for (int b = 0; b < DB; b++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[b][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  int bad = 0;

  if (tiles > 0) load(0, 0);
  for (int t = 0; t < tiles; t++) {
    const int k0 = tile_key(t);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0): this tile is in LDS, the last one read
    ring_barrier();
    const char *kt = lds + (t & 1) * 2 * TILE, *vt = kt + TILE;
    if (t + 1 < tiles) load(t + 1, (t + 1) & 1);
    // Where some query does not see some key of the tile, an infinity or NaN
    // in V would reach it through its weight of 0.
    if (k0 + KEYS - 1 > p_first || (a.window && k0 <= p_last - a.window)) {
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const v4u x = *(const v4u *)(vt + (i * 64 * kTileWaves + tid) * 16);
        bad |= not_finite2<T>(x[0]) + not_finite2<T>(x[1]) + not_finite2<T>(x[2]) + not_finite2<T>(x[3]);
      }
    }
    const bool none = k0 > pw_last || (a.window && k0 + KEYS - 1 <= pw_first - a.window && k0 >= a.sinks);
    if (none || w0 >= bl.nq) continue;
    const bool masked = k0 + KEYS - 1 > pw_first || (a.window && k0 <= pw_last - a.window);

    // The products first where two waves share a SIMD: one's softmax then runs
    // under the other's products (2 to 8 % of the whole).
    __builtin_amdgcn_s_setprio(1);
    v16f s[SB];
#pragma unroll
    for (int b = 0; b < SB; b++) {
#pragma unroll
      for (int i = 0; i < 16; i++) s[b][i] = 0.0f;
      const char *row = kt + (32 * b + col) * C * 16;
#pragma unroll
      for (int c = 0; c < KS; c++) {
        const v4u f = *(const v4u *)(row + ((2 * c + half) ^ turn<C>(col)) * 16);
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < 4; j++)
            s[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(f[j]), __uint_as_float(q[c][j]), s[b], 0, 0, 0);
        } else if constexpr (T == PPOCR_F16)
          s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, f), __builtin_bit_cast(v8h, q[c]), s[b],
                                                        0, 0, 0);
        else
          s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, f), __builtin_bit_cast(v8bf, q[c]),
                                                         s[b], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if (masked) {
      const int here = k0 + 4 * half, last = p - here, from = p_low - here, sunk = a.sinks - here;
#pragma unroll
      for (int b = 0; b < SB; b++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int j = 32 * b + 8 * (i / 4) + i % 4;
          const int hidden = int(j > last) | (int(j < from) & int(j >= sunk));
          s[b][i] = hidden ? -INFINITY : s[b][i];
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int b = 0; b < SB; b++)
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, s[b][i]);
    top = fmaxf(top, __shfl_xor(top, 32));
    // The maximum follows only where it grew much: until then the weights are
    // larger, which costs them no precision.
    if (__any((top - m) * a.scale > kGrow<T>)) {
      const float now = fmaxf(m, top);
      const float shrink = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - now) * a.scale);
      m = now;
      l *= shrink;
#pragma unroll
      for (int b = 0; b < DB; b++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[b][i] *= shrink;
    }
    const float base = m == -INFINITY ? 0.0f : m * a.scale - kUp<T>;
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[0][i], a.scale, -base));
        l += w;
        float f[DB];
        const float *at = (const float *)(vt + (8 * (i / 4) + 4 * half + i % 4) * C * 16) + DB * col;
#pragma unroll
        for (int b = 0; b < DB; b++) f[b] = at[b];
#pragma unroll
        for (int b = 0; b < DB; b++) o[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(f[b], w, o[b], 0, 0, 0);
      }
      continue;
    } else {
      v4u pf[4];
      float part[4] = {0, 0, 0, 0};
#pragma unroll
      for (int b = 0; b < SB; b++)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float x = __builtin_amdgcn_exp2f(fmaf(s[b][i], a.scale, -base));
          const float y = __builtin_amdgcn_exp2f(fmaf(s[b][i + 1], a.scale, -base));
          const uint32_t w = Tile16<T>::pack(x, y);
          part[i / 2 % 4] = Tile16<T>::sum(w, part[i / 2 % 4]);
          pf[2 * b + i / 8][i / 2 % 4] = w;
        }
      l += (part[0] + part[1]) + (part[2] + part[3]);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int b = 0; b < DB; b++) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
          // Lane s of 16 names keys s / 4 of four and values 4 (s % 4) .. + 3 of
          // 16, and gets value s of the four keys.
          v4u f;
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const int key = 16 * c + 8 * g + 4 * half + lane % 16 / 4;
            const int piece = 4 * b + 2 * (lane / 16 % 2) + lane % 4 / 2;
            const char *at = vt + (key * C + (piece ^ turn<C>(key))) * 16 + lane % 2 * 8;
            const v4s r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)at);
            f[2 * g] = __builtin_bit_cast(v2u, r)[0];
            f[2 * g + 1] = __builtin_bit_cast(v2u, r)[1];
          }
          if constexpr (T == PPOCR_F16)
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, f), __builtin_bit_cast(v8h, pf[c]),
                                                          o[b], 0, 0, 0);
          else
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, f), __builtin_bit_cast(v8bf, pf[c]),
                                                           o[b], 0, 0, 0);
        }
      }
    }
  }
  __builtin_amdgcn_s_setprio(0);
  if (__syncthreads_or(bad)) {  // rare: key by key where it matters
    attend_alone<T>(a, bl, head, w0, 32);
    return;
  }
  l += __shfl_xor(l, 32);
  if (w0 + col >= bl.nq) return;
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  V *y = (V *)a.y + (long)(bl.q0 + query) * a.y_stride + (long)head * a.dim;
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < 16; i++) {
      float out[DB];
#pragma unroll
      for (int b = 0; b < DB; b++) out[b] = l == 0.0f ? 0.0f : o[b][i] * f;
      const int d = DB * (8 * (i / 4) + 4 * half + i % 4);
      store_n(y + d, (long)a.dim - d, out);
    }
  } else {
#pragma unroll
    for (int b = 0; b < DB; b++)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * b + 2 * i + 4 * half;
        V out[4];
#pragma unroll
        for (int e = 0; e < 4; e++) out[e] = Num<T>::put(l == 0.0f ? 0.0f : o[b][i + e] * f);
        store_n(y + d, (long)a.dim - d, out);
      }
  }
}

template <int T, int DP, bool WHOLE>
hipError_t launch_tiles_of(const PromptArgs &a, hipStream_t s) {
  const int per = a.heads / a.kv_heads, hg = per % 4 == 0 ? 4 : per % 2 == 0 ? 2 : 1;
  const int size = 32 * kTileWaves / hg;
  constexpr int bytes = 4 * kTileKeys<T> * kPieces<T, DP> * 16;
  const hipError_t e = allow_lds_of<&window_attention_tiles<T, DP, WHOLE>>(bytes);
  if (e != hipSuccess) return e;
  const long blocks = (a.heads / hg) * (a.rows_q / size + (long)a.batch);
  if (blocks >= 1L << 24) return hipErrorInvalidConfiguration;
  return launch_kernel(window_attention_tiles<T, DP, WHOLE>, dim3(unsigned(blocks)), dim3(64 * kTileWaves), bytes, s, a,
                       hg);
}

template <int T, int DP>
hipError_t launch_tiles(const PromptArgs &a, hipStream_t s) {
  if constexpr (DP == 64 || DP == 128 || DP == 256)
    if (a.dim == DP) return launch_tiles_of<T, DP, true>(a, s);
  return launch_tiles_of<T, DP, false>(a, s);
}

template <int T, int DP>
hipError_t launch_rows(const PromptArgs &a, hipStream_t s) {
  const long blocks = a.heads * (a.rows_q / 64 + (long)a.batch);
  if (blocks >= 1L << 24) return hipErrorInvalidConfiguration;
  const dim3 grid{unsigned(blocks)}, block(256);
  if (a.dim == DP) return launch_kernel(window_attention_rows<T, DP, DIMS_WHOLE>, grid, block, 0, s, a);
  if (a.dim % 8 == 0) return launch_kernel(window_attention_rows<T, DP, DIMS_EVEN>, grid, block, 0, s, a);
  return launch_kernel(window_attention_rows<T, DP, DIMS_ANY>, grid, block, 0, s, a);
}

template <int T>
hipError_t launch(const PromptArgs &a, hipStream_t s) {
  // Loads to LDS move 16 aligned bytes.
  constexpr int N = 16 / sizeof(num_t<T>);
  auto a16 = [](const void *p, long stride) { return uintptr_t(p) % 16 == 0 && stride % N == 0; };
  if (a.dim % N == 0 && a.dim > 16 && a16(a.k, a.k_stride) && a16(a.v, a.v_stride)) {
    if (a.dim <= 64) return launch_tiles<T, 64>(a, s);
    if (a.dim <= 96) return launch_tiles<T, 96>(a, s);
    if (a.dim <= 128) return launch_tiles<T, 128>(a, s);
    if (a.dim <= 192) return launch_tiles<T, 192>(a, s);
    return launch_tiles<T, 256>(a, s);
  }
  if (a.dim <= 32) return launch_rows<T, 32>(a, s);
  if (a.dim <= 64) return launch_rows<T, 64>(a, s);
  if (a.dim <= 128) return launch_rows<T, 128>(a, s);
  return launch_rows<T, 256>(a, s);
}

}  // namespace

hipError_t launch_window_attention(const PromptArgs &a, int type, hipStream_t s) {
  switch (type) {
    case PPOCR_F32: return launch<PPOCR_F32>(a, s);
    case PPOCR_BF16: return launch<PPOCR_BF16>(a, s);
    case PPOCR_F16: return launch<PPOCR_F16>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ppocr
