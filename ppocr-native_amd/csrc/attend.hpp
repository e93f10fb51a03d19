// Softmax attention of 16 query rows over keys, a wave's worth, on the matrix
// cores: shared by the decode attention (the 16 are query heads of one key
// head) and the prompt attention of any type and dim (16 queries of a head).
//
// The rows are the columns of every product, so that a lane holds one row's
// numbers throughout (column lane % 16) and its running maximum and sum need
// only two exchanges between the wave's quarters:
//   S^T[key][row] = K Q^T,   O^T[d][row] += V^T P^T.
// A 16-key result leaves quarter p with keys 4 p .. 4 p + 3 of its row, which
// are then what that quarter holds of P^T: the order of the products' inner
// index is free, so V's rows are loaded to match and P stays where it is.
// V comes row by row (each lane DP / 16 neighbouring values of a key's row);
// 16-bit values of two keys are paired by byte permutes.
#pragma once
#include "decoder.hpp"

namespace ppocr {

// How a head's dims fill the DP that the products have.
enum Dims {
  DIMS_WHOLE,  // dim == DP
  DIMS_EVEN,   // a multiple of 8, at most DP
  DIMS_ANY     // at most DP, value by value
};

// N values of a head at d. What lies past dim is some other value of the
// head's: nothing is read behind a branch, which would be waited for.
template <int DIMS, typename V, int N>
__device__ __forceinline__ void load_dims(const V *p, int d, int dim, V (&v)[N]) {
  if constexpr (DIMS == DIMS_WHOLE) {
    __builtin_memcpy(v, p + d, sizeof v);
  } else if constexpr (DIMS == DIMS_EVEN) {
    constexpr int M = N < 8 ? N : 8;
#pragma unroll
    for (int i = 0; i < N; i += M) __builtin_memcpy(v + i, p + (d + i < dim ? d + i : 0), M * sizeof(V));
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = p[min(d + i, dim - 1)];
  }
}

// Zeros for those past dim.
template <int DIMS, typename V, int N>
__device__ __forceinline__ void cut_dims(int d, int dim, V (&v)[N]) {
  if constexpr (DIMS != DIMS_WHOLE) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = d + i < dim ? v[i] : V(0);
  }
}

// 16-bit types: 32 keys a tile, inner index 32.
template <int T>
struct Tile16 {
  static __device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c) {
    if constexpr (T == PPOCR_F16)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0,
                                                    0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0,
                                                     0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    if constexpr (T == PPOCR_F16)
      return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2h));
    else
      return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2bf));
  }
  // Both positive, or 0: rounded down.
  static __device__ __forceinline__ uint32_t pack_down(float a, float b) {
    if constexpr (T == PPOCR_F16)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    else
      return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
  }
  // Adds the two values to a sum.
  static __device__ __forceinline__ float sum(uint32_t p, float to) {
    if constexpr (T == PPOCR_F16)
      return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, p), v2h{(_Float16)1.0f, (_Float16)1.0f}, to, false);
    else
      return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, p), v2bf{(__bf16)1.0f, (__bf16)1.0f}, to, false);
  }
  static __device__ __forceinline__ v2f unpack(uint32_t p) {
    if constexpr (T == PPOCR_F16)
      return __builtin_convertvector(__builtin_bit_cast(v2h, p), v2f);
    else
      return v2f{__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u)};
  }
};

// The state of 16 rows over DP (padded) dims.
template <int T, int DP, int DIMS>
struct Attend {
  typedef num_t<T> V;
  static constexpr bool F32 = T == PPOCR_F32;
  static constexpr int KEYS = F32 ? 16 : 32;        // keys a tile
  static constexpr int H = KEYS / 16;               // 16-key halves
  static constexpr int QC = F32 ? DP / 16 : DP / 32;  // 16-byte pieces of a row a lane has
  static constexpr int QN = F32 ? 4 : 8;            // values in one
  static constexpr int E = DP / 16;                 // values of a V row a lane has
  // Weights (and so their sum) are held 2^UP times as large: F16 ends at 2^-24,
  // and where one key is far ahead of all others, theirs are what counts if its
  // value is near 0. The largest is 2^15 then, below F16's 65504, and a weight
  // is off by 2^-39 of the largest at most.
  static constexpr float UP = T == PPOCR_F16 ? 15.0f : 0.0f;
  V q[QC][QN];
  v4f o[E];  // O^T: this lane's row, d = E (4 quarter + r) + e
  float m, l;  // running maximum of the products and this lane's share of the sum

  // `turn`: the scale is negative, and q turns its sign instead.
  __device__ __forceinline__ void start(const V *qrow, int dim, int quarter, bool turn) {
#pragma unroll
    for (int c = 0; c < QC; c++) {
      load_dims<DIMS>(qrow, QN * (4 * c + quarter), dim, q[c]);
      cut_dims<DIMS>(QN * (4 * c + quarter), dim, q[c]);
      if (turn) {
#pragma unroll
        for (int i = 0; i < QN; i++) q[c][i] = -q[c][i];
      }
    }
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = v4f{0, 0, 0, 0};
    m = -INFINITY;
    l = 0.0f;
  }

  static __device__ __forceinline__ bool finite(V x) {
    if constexpr (F32)
      return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
    else if constexpr (T == PPOCR_BF16)
      return (__builtin_bit_cast(uint16_t, x) & 0x7f80) != 0x7f80;
    else
      return (__builtin_bit_cast(uint16_t, x) & 0x7c00) != 0x7c00;
  }

  // A tile's keys and values in registers.
  struct Tile {
    V k[H][QC][QN], v[H][4][E];
  };

  // k_row(key) and v_row(key) give the rows of the tile's keys 0 .. KEYS - 1,
  // any row that may be read where no row of the 16 sees the key.
  template <class KR, class VR>
  static __device__ __forceinline__ void load(Tile &t, KR k_row, VR v_row, int dim, int lane) {
    const int col = lane % 16, quarter = lane / 16;
#pragma unroll
    for (int h = 0; h < H; h++) {
      const V *p = k_row(16 * h + col);
#pragma unroll
      for (int c = 0; c < QC; c++) load_dims<DIMS>(p, QN * (4 * c + quarter), dim, t.k[h][c]);
    }
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) load_dims<DIMS>(v_row(16 * h + 4 * quarter + r), E * col, dim, t.v[h][r]);
  }

  // Takes a tile in. seen(key) says whether this lane's row sees it, any(key)
  // whether some row does; `masked` (uniform): not every key of the tile is
  // seen by every row. `scale`: of 2-logarithms, positive. RAGGED: the 16 rows
  // do not see the same keys; the result says whether this lane met an
  // infinity or NaN in V in such a tile, which a weight of 0 carries into the
  // rows that do not see it.
  template <bool RAGGED, class Seen, class Any>
  __device__ __forceinline__ bool use(Tile &t, Seen seen, Any any, bool masked, int dim, float scale, int lane) {
    const int quarter = lane / 16;
    auto &k = t.k;
    auto &v = t.v;
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
      for (int c = 0; c < QC; c++) cut_dims<DIMS>(QN * (4 * c + quarter), dim, k[h][c]);
    if (masked) {
#pragma unroll
      for (int h = 0; h < H; h++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const bool on = any(16 * h + 4 * quarter + r);
#pragma unroll
          for (int e = 0; e < E; e++) v[h][r][e] = on ? v[h][r][e] : V(0);
        }
    }
    v4f s[H];
#pragma unroll
    for (int h = 0; h < H; h++) {
      s[h] = v4f{0, 0, 0, 0};
      v4f s2[3] = {};  // F32: four sums, each of a quarter of the roundings
#pragma unroll
      for (int c = 0; c < QC; c++) {
        if constexpr (F32) {
          s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[h][c][0], q[c][0], s[h], 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 3; j++)
            s2[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[h][c][j + 1], q[c][j + 1], s2[j], 0, 0, 0);
        } else {
          v4u a, b;
          __builtin_memcpy(&a, k[h][c], 16);
          __builtin_memcpy(&b, q[c], 16);
          s[h] = Tile16<T>::mfma(a, b, s[h]);
        }
      }
      if constexpr (F32) s[h] = (s[h] + s2[0]) + (s2[1] + s2[2]);
    }
    float top = -INFINITY;
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        if (masked && !seen(16 * h + 4 * quarter + r)) s[h][r] = -INFINITY;
        top = fmaxf(top, s[h][r]);
      }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float now = fmaxf(m, top), base = now == -INFINITY ? 0.0f : now * scale - UP;
    if (__any(now != m)) {
      const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - now) * scale);
      l *= shrink;
#pragma unroll
      for (int e = 0; e < E; e++) o[e] *= shrink;
      m = now;
    }
    float p[H][4];
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[h][r] = __builtin_amdgcn_exp2f(fmaf(s[h][r], scale, -base));
        l += p[h][r];
      }
    bool bad = false;
    if constexpr (RAGGED) {
      if (masked) {
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
          for (int r = 0; r < 4; r++)
#pragma unroll
            for (int e = 0; e < E; e++) bad |= !finite(v[h][r][e]);
      }
    }
    if constexpr (F32) {
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[0][r][e], p[0][r], o[e], 0, 0, 0);
    } else {
      // P as a high and a low part of T: the weights keep 16 bits in BF16 and 22
      // in F16 (down to the parts' last step, 2^-24 of the unit UP makes) where
      // T alone has 8 and 11, at twice the products, which memory hides. Their
      // sum is of the f32 weights. The high part is rounded down and the low one
      // is not 0 where the weight is not, so that an infinity in V times both is
      // that infinity.
      constexpr float least = T == PPOCR_F16 ? 0x1p-24f : 0x1p-126f;
      auto rest = [&](float x, float high) { return __builtin_amdgcn_fmed3f(x - high, least, x); };
      v4u hi, lo;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x = p[i / 2][2 * (i % 2)], y = p[i / 2][2 * (i % 2) + 1];
        hi[i] = Tile16<T>::pack_down(x, y);
        const v2f back = Tile16<T>::unpack(hi[i]);
        lo[i] = Tile16<T>::pack(rest(x, back[0]), rest(y, back[1]));
      }
#pragma unroll
      for (int e = 0; e < E; e++) {
        v4u f;
#pragma unroll
        for (int i = 0; i < 4; i++)
          f[i] = (uint32_t)__builtin_bit_cast(uint16_t, v[i / 2][2 * (i % 2)][e]) |
                 (uint32_t)__builtin_bit_cast(uint16_t, v[i / 2][2 * (i % 2) + 1][e]) << 16;
        o[e] = Tile16<T>::mfma(f, lo, o[e]);
        o[e] = Tile16<T>::mfma(f, hi, o[e]);
      }
    }
    return bad;
  }

  // The row's whole sum, in all four quarters.
  __device__ __forceinline__ float total() const {
    float t = l + __shfl_xor(l, 16);
    return t + __shfl_xor(t, 32);
  }
};

}  // namespace ppocr
