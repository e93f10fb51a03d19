// Products of a few rows with 4-bit weights (ppocr_hip_q4_product).
//
//   y[i][j] = bias[j] + sum_g s[j][g] sum_(k in g) x[i][k] (q[j][k] - z[j][g])
//
// Reading the weights bounds it: at 4.7 TB/s a SIMD of the 1024 gets 512
// weights in 136 cycles, and 512 are what one 16x16x32 matrix product takes,
// in 16 cycles, for up to 16 rows of x. So the products go to the matrix cores
// even for one row, and the vector units, with about 34 instructions in that
// time, only turn nibbles into operands: the four bits are put into the
// mantissa of 16.0, (w << s) & mask | 16.0, which is 16 + q exactly, two
// weights in two instructions. With sum x over the group, from one more
// product whose other operand is ones, in the same lanes as the result,
//   sum x (q - z) = sum x (16 + q) - (16 + z) sum x,
// every term exact in bf16 and f16 but for the f32 sums. f32 rows are split
// into three bf16 parts first (split.hpp), 8-bit rows are exact in bf16.
//
// A wave takes tiles of 16 outputs (NT of them) and every W-th stretch of 128
// inputs, the W waves of a workgroup the same outputs; the parts are summed
// in LDS in the order of the waves. Of a stretch each lane loads 16 bytes of
// one output's row; v_permlane*_swap then exchange dwords between the wave's
// quarters, so that dword j of quarter p holds inputs 32 j + 8 p .. + 7 and
// no product mixes two groups.
#include "decoder.hpp"
#include "split.hpp"

namespace ppocr {
namespace {

constexpr int kWaves = 8;      // most waves of a workgroup
constexpr int kStretch = 128;  // inputs a wave takes at a time

// x in registers as loaded, 8 values, and as matrix operands: dword d holds
// values d (low half) and d + 4, the order the nibbles come in.
template <int X>
struct XRow;
template <>
struct XRow<PPOCR_BF16> {
  typedef uint16_t type;
  static constexpr int parts = 1;
  static __device__ __forceinline__ void operands(const uint16_t (&v)[8], int, v4u (&p)[1]) {
#pragma unroll
    for (int d = 0; d < 4; d++) p[0][d] = (uint32_t)v[d] | (uint32_t)v[d + 4] << 16;
  }
};
template <>
struct XRow<PPOCR_F16> : XRow<PPOCR_BF16> {};
template <>
struct XRow<PPOCR_F32> {
  typedef float type;
  static constexpr int parts = 3;
  static __device__ __forceinline__ void operands(const float (&v)[8], int, v4u (&p)[3]) {
#pragma unroll
    for (int d = 0; d < 4; d++) {
      uint32_t a, b, c;
      split_pair(v[d], v[d + 4], a, b, c);
      p[0][d] = a, p[1][d] = b, p[2][d] = c;
    }
  }
};
template <>
struct XRow<PPOCR_I8> {  // and E4M3
  typedef uint8_t type;
  static constexpr int parts = 1;
  static __device__ __forceinline__ void operands(const uint8_t (&v)[8], int e4m3, v4u (&p)[1]) {
    float f[8];
    if (e4m3) {
      const uint32_t lo = v[0] | v[1] << 8 | v[2] << 16 | (uint32_t)v[3] << 24;
      const uint32_t hi = v[4] | v[5] << 8 | v[6] << 16 | (uint32_t)v[7] << 24;
      const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(lo, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(lo, true);
      const v2f c = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
      f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1], f[4] = c[0], f[5] = c[1], f[6] = d[0], f[7] = d[1];
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = (float)(int8_t)v[i];
    }
    // Exact in bf16: at most 8 significant bits.
#pragma unroll
    for (int d = 0; d < 4; d++)
      p[0][d] = __float_as_uint(f[d]) >> 16 | (__float_as_uint(f[d + 4]) & 0xffff0000u);
  }
};

template <int X>
__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c) {
  if constexpr (X == PPOCR_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0,
                                                   0);
}

// The eight nibbles of w as 16 + q: dword d holds nibbles d and d + 4.
template <int X>
__device__ __forceinline__ v4u weights16(uint32_t w) {
  constexpr int top = X == PPOCR_F16 ? 6 : 3;  // the mantissa's bit of value 1 at 16.0
  constexpr uint32_t mask = 0x000f000fu << top, base = X == PPOCR_F16 ? 0x4c004c00u : 0x41804180u;
  v4u f;
#pragma unroll
  for (int d = 0; d < 4; d++) f[d] = ((4 * d > top ? w >> (4 * d - top) : w << (top - 4 * d)) & mask) | base;
  return f;
}

// Dwords between the wave's quarters (lanes 16 p .. 16 p + 15): before, dword
// j of quarter p is stretch byte 16 p + 4 j; after, 16 j + 4 p.
__device__ __forceinline__ void turn_quarters(uint32_t (&w)[4]) {
  v2u t = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
  w[0] = t[0], w[2] = t[1];
  t = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  w[1] = t[0], w[3] = t[1];
  t = __builtin_amdgcn_permlane16_swap(w[0], w[1], false, false);
  w[0] = t[0], w[1] = t[1];
  t = __builtin_amdgcn_permlane16_swap(w[2], w[3], false, false);
  w[2] = t[0], w[3] = t[1];
}

// What a wave loads for one stretch, a stretch ahead. Where a wave has more
// than 16 rows of x (MT > 1) those are loaded as they are used: a stretch's
// worth would not fit the registers.
template <int X, int MT, int NT, int SG>
struct Stretch {
  uint32_t w[NT][4];
  uint32_t s[NT][SG];  // scales as stored
  uint8_t z[NT][SG];
  typename XRow<X>::type x[MT == 1 ? 1 : 0][4][8];
  float xs[X == PPOCR_I8 ? MT : 1][4][SG];
};

template <int X, int MT, int NT, int GROUP>
__global__ __launch_bounds__(64 * kWaves) void q4_rows(Q4Args a, int e4m3) {
  constexpr int SG = kStretch / GROUP, P = XRow<X>::parts;
  typedef typename XRow<X>::type V;
  __shared__ float red[kWaves][4][256];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
  const int col = lane % 16, quarter = lane / 16;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  const long row_bytes = (a.k + 1L) / 2;
  const int steps = (a.k + kStretch - 1) / kStretch;
  const bool x_grouped = X == PPOCR_I8 && a.x_group;

  auto load_x = [&](int i, int k, V(&v)[8]) {
    const long m = min(m0 + 16 * i + col, a.m - 1);  // rows past m: results not stored
    load_n((const V *)a.x + m * a.x_stride + k, (long)a.k - k, v);
  };
  auto load = [&](Stretch<X, MT, NT, SG> &t, int step) {
    const int k0 = step * kStretch, g0 = k0 / GROUP;
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const long n = min(n0 + 16 * j + col, a.n - 1);
      const long at = k0 / 2 + 16 * quarter;
      uint8_t b[16];
      load_n(a.q + n * row_bytes + at, row_bytes - at, b);
      __builtin_memcpy(t.w[j], b, 16);
      const long g = n * a.groups + g0;
      if (a.scale_type == PPOCR_F32) {
        load_n((const uint32_t *)a.scales + g, a.groups - g0, t.s[j]);
      } else {
        uint16_t h[SG];
        load_n((const uint16_t *)a.scales + g, a.groups - g0, h);
#pragma unroll
        for (int i = 0; i < SG; i++) t.s[j][i] = h[i];
      }
      if (a.zeros) load_n(a.zeros + g, a.groups - g0, t.z[j]);
    }
    if constexpr (MT == 1) {
#pragma unroll
      for (int c = 0; c < 4; c++) load_x(0, k0 + 32 * c + 8 * quarter, t.x[0][c]);
    }
    if constexpr (X == PPOCR_I8) {
      if (x_grouped) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const long m = min(m0 + 16 * i + 4 * quarter + r, a.m - 1);
            load_n(a.x_scales + m * a.x_groups + g0, a.x_groups - g0, t.xs[i][r]);
          }
      }
    }
  };

  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NT; j++) acc[i][j] = v4f{0, 0, 0, 0};

  const v4u ones = X == PPOCR_F16 ? v4u{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u}
                                  : v4u{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  auto compute = [&](Stretch<X, MT, NT, SG> &t, int step) {
#pragma unroll
    for (int j = 0; j < NT; j++) turn_quarters(t.w[j]);
#pragma unroll
    for (int g = 0; g < SG; g++) {
      float s[NT], z[NT];
#pragma unroll
      for (int j = 0; j < NT; j++) {
        if (a.scale_type == PPOCR_F32)
          s[j] = __uint_as_float(t.s[j][g]);
        else if (a.scale_type == PPOCR_BF16)
          s[j] = __uint_as_float(t.s[j][g] << 16);
        else
          s[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)t.s[j][g]);
        z[j] = a.zeros ? 16.0f + (float)t.z[j][g] : 24.0f;
      }
      v4f d[MT][NT][P], sx[MT][P];
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int p = 0; p < P; p++) {
          sx[i][p] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < NT; j++) d[i][j][p] = v4f{0, 0, 0, 0};
        }
#pragma unroll
      for (int c = g * 4 / SG; c < (g + 1) * 4 / SG; c++) {
        v4u wf[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) wf[j] = weights16<X>(t.w[j][c]);
#pragma unroll
        for (int i = 0; i < MT; i++) {
          v4u xf[P];
          if constexpr (MT == 1) {
            XRow<X>::operands(t.x[i][c], e4m3, xf);
          } else {
            V v[8];
            load_x(i, step * kStretch + 32 * c + 8 * quarter, v);
            XRow<X>::operands(v, e4m3, xf);
          }
#pragma unroll
          for (int p = 0; p < P; p++) {
            sx[i][p] = mfma<X>(xf[p], ones, sx[i][p]);
#pragma unroll
            for (int j = 0; j < NT; j++) d[i][j][p] = mfma<X>(xf[p], wf[j], d[i][j][p]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            float v = fmaf(-z[j], sx[i][0][r], d[i][j][0][r]);
            if constexpr (P == 3) {
              const float v2 = fmaf(-z[j], sx[i][1][r], d[i][j][1][r]);
              const float v3 = fmaf(-z[j], sx[i][2][r], d[i][j][2][r]);
              v = fmaf(fmaf(v3, 1.0f / 256.0f, v2), 1.0f / 256.0f, v);
            }
            float f = s[j];
            if constexpr (X == PPOCR_I8)
              if (x_grouped) f *= t.xs[i][r][g];
            acc[i][j][r] = fmaf(f, v, acc[i][j][r]);
          }
    }
  };

  Stretch<X, MT, NT, SG> ta, tb;
  int step = wave;
  if (step < steps) load(ta, step);
  while (step < steps) {
    if (step + waves < steps) load(tb, step + waves);
    compute(ta, step);
    step += waves;
    if (step >= steps) break;
    if (step + waves < steps) load(ta, step + waves);
    compute(tb, step);
    step += waves;
  }

  // The waves' parts, in order, four tiles at a time.
  constexpr int TILES = MT * NT, AT = TILES < 4 ? TILES : 4;
#pragma unroll
  for (int t0 = 0; t0 < TILES; t0 += AT) {
    if (t0) __syncthreads();
#pragma unroll
    for (int t = 0; t < AT; t++)
      *(v4f *)&red[wave][t][4 * lane] = acc[(t0 + t) / NT][(t0 + t) % NT];
    __syncthreads();
    for (int i = threadIdx.x; i < AT * 256; i += blockDim.x) {
      const int t = t0 + i / 256, c = i % 16, r = i / 16 % 16;
      const int n = n0 + 16 * (t % NT) + c, m = m0 + 16 * (t / NT) + r;
      if (m >= a.m || n >= a.n) continue;
      float v = 0.0f;
      for (int w = 0; w < waves; w++) v += red[w][i / 256][4 * (c + 16 * (r / 4)) + r % 4];
      if constexpr (X == PPOCR_I8)
        if (!x_grouped) v *= a.x_scales[m];
      const long at = m * a.y_stride + n;
      if (a.y_type == PPOCR_F32)
        ((float *)a.y)[at] = a.bias ? v + ((const float *)a.bias)[n] : v;
      else if (a.y_type == PPOCR_BF16)
        ((__bf16 *)a.y)[at] = (__bf16)(a.bias ? v + (float)((const __bf16 *)a.bias)[n] : v);
      else
        ((_Float16 *)a.y)[at] = (_Float16)(a.bias ? v + (float)((const _Float16 *)a.bias)[n] : v);
    }
  }
}

template <int X, int MT, int NT>
void launch_tile(const Q4Args &a, int e4m3, hipStream_t s) {
  const int steps = (a.k + kStretch - 1) / kStretch;
  const dim3 grid((a.n + 16 * NT - 1) / (16 * NT), (a.m + 16 * MT - 1) / (16 * MT));
  const dim3 block(64 * (steps < kWaves ? steps : kWaves));
  if (a.group == 32)
    hipLaunchKernelGGL((q4_rows<X, MT, NT, 32>), grid, block, 0, s, a, e4m3);
  else if (a.group == 64)
    hipLaunchKernelGGL((q4_rows<X, MT, NT, 64>), grid, block, 0, s, a, e4m3);
  else
    hipLaunchKernelGGL((q4_rows<X, MT, NT, 128>), grid, block, 0, s, a, e4m3);
}

template <int X>
hipError_t launch(const Q4Args &a, int e4m3, hipStream_t s) {
  if (a.m <= 16)
    launch_tile<X, 1, 1>(a, e4m3, s);
  else if (a.m <= 32)
    launch_tile<X, 2, 1>(a, e4m3, s);
  else
    launch_tile<X, 4, 1>(a, e4m3, s);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_q4_product(const Q4Args &a, int x_type, hipStream_t s) {
  switch (x_type) {
    case PPOCR_F32: return launch<PPOCR_F32>(a, 0, s);
    case PPOCR_BF16: return launch<PPOCR_BF16>(a, 0, s);
    case PPOCR_F16: return launch<PPOCR_F16>(a, 0, s);
    case PPOCR_E4M3: return launch<PPOCR_I8>(a, 1, s);
    case PPOCR_I8: return launch<PPOCR_I8>(a, 0, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ppocr
