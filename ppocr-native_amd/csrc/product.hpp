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
// (16 + q) x passes f32's range before q x does, and f32 values past bf16's
// largest are infinite in the split: an output of f32 or bf16 rows that comes out
// as an infinity or NaN is computed again, in f64 from the formula as it stands,
// where its row of x is finite.
//
// A workgroup takes up to NT tiles of 16 outputs, its waves every W-th stretch
// of 128 inputs of them; the waves' sums are added in LDS in their order. The
// weights of a stretch and tile (1 KB) go straight from memory to the wave's
// own ring in LDS, kRing ahead: with registers in between the compiler waits
// for a load before it copies the register it came to (a ring of four in
// registers took 0.9 us a stretch). Four neighbouring lanes load a row's 64
// bytes: with a row a lane, as the operand has them, the address unit takes a
// cycle a lane and was 95 % busy (35 % so).
//
// x, the scales and the zero points are the same for all of a workgroup's
// waves, or come in rows too short to load well: they go to LDS a chunk of
// stretches at a time, x as finished operands.
//
// 4096 inputs to 28672 outputs (61 to 71 MB): one row of bf16, groups of 128,
// 17.2 us, 3.5 TB/s; 16 rows of f16, groups of 32 with zero points, 22.5 us (25
// in a trace), 3.2 TB/s; 5 rows of f32, groups of 64, 29.6 us; a kernel that only
// reads takes 11 us for 71 MB. What is left is the wait for a chunk at its start,
// the conversion and the launch. Each further 16 rows load and convert all of it
// again: 32 and 64 rows of bf16 41 and 66 us, of f32 86 and 149, of 8 bits 68 (64
// rows). Fetching a chunk's x ahead into registers spilled (60 us for the 22.5);
// tiles of 32 and 64 rows of x were slower than blocks of 16 that share the
// weights through L2 (64 rows of f32: 715 us against 171 at that time).
#include <algorithm>

#include "decoder.hpp"
#include "kernels.hpp"
#include "split.hpp"

namespace ppocr {
namespace {

constexpr int kWaves = kQ4Waves, kStretch = kQ4Stretch;

// Eight values of x as loaded (DW dwords), and as matrix operands: dword d
// holds values d (low half) and d + 4, the order the nibbles come in.
template <int X>
struct XRow {  // BF16, F16
  static constexpr int size = 2, DW = 4, parts = 1;
  static __device__ __forceinline__ void operands(const uint32_t (&v)[4], int, v4u (&p)[1]) {
    p[0] = v4u{__builtin_amdgcn_perm(v[2], v[0], 0x05040100), __builtin_amdgcn_perm(v[2], v[0], 0x07060302),
               __builtin_amdgcn_perm(v[3], v[1], 0x05040100), __builtin_amdgcn_perm(v[3], v[1], 0x07060302)};
  }
};
template <>
struct XRow<PPOCR_F32> {
  static constexpr int size = 4, DW = 8, parts = 3;
  static __device__ __forceinline__ void operands(const uint32_t (&v)[8], int, v4u (&p)[3]) {
#pragma unroll
    for (int d = 0; d < 4; d++) {
      uint32_t a, b, c;
      split_pair(__uint_as_float(v[d]), __uint_as_float(v[d + 4]), a, b, c);
      p[0][d] = a, p[1][d] = b, p[2][d] = c;
    }
  }
};
template <>
struct XRow<PPOCR_I8> {  // and E4M3: exact in bf16, at most 8 significant bits
  static constexpr int size = 1, DW = 2, parts = 1;
  static __device__ __forceinline__ void operands(const uint32_t (&v)[2], int e4m3, v4u (&p)[1]) {
    float f[8];
    if (e4m3) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(v[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(v[i], true);
        f[4 * i] = a[0], f[4 * i + 1] = a[1], f[4 * i + 2] = b[0], f[4 * i + 3] = b[1];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = (float)(int8_t)(v[i / 4] >> 8 * (i % 4));
    }
#pragma unroll
    for (int d = 0; d < 4; d++)
      p[0][d] = __builtin_amdgcn_perm(__float_as_uint(f[d + 4]), __float_as_uint(f[d]), 0x07060302);
  }
};

// N numbers of SIZE bytes at p as dwords, or the first `have` of them and
// zeros.
template <bool TAIL, int SIZE, int N, int D>
__device__ __forceinline__ void load_dwords(const uint8_t *p, int have, uint32_t (&v)[D]) {
  static_assert(N * SIZE <= 4 * D);
  if constexpr (!TAIL) {
    __builtin_memcpy(v, p, N * SIZE);
  } else {
#pragma unroll
    for (int i = 0; i < D; i++) v[i] = 0;
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < have) {
        uint32_t one = 0;
        __builtin_memcpy(&one, p + i * SIZE, SIZE);
        v[i * SIZE / 4] |= one << i * SIZE % 4 * 8;
      }
  }
}

template <int X>
__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c) {
  if constexpr (X == PPOCR_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0,
                                                   0);
}

// The eight nibbles of w as 16 + q: dword d holds nibbles d and d + 4. The mask
// and 16.0 come in registers: as literals they make two instructions of one.
template <int X>
constexpr int kTop = X == PPOCR_F16 ? 6 : 3;  // the mantissa's bit of value 1 at 16.0
template <int X>
__device__ __forceinline__ v4u weights16(uint32_t w, uint32_t mask, uint32_t base) {
  constexpr int top = kTop<X>;
  v4u f;
#pragma unroll
  for (int d = 0; d < 4; d++) f[d] = ((4 * d > top ? w >> (4 * d - top) : w << (top - 4 * d)) & mask) | base;
  return f;
}

constexpr int kRing = 3;

// LDS: the waves' rings; then a chunk of x, for each 32 inputs and part, 4 x
// `rows` 16-byte operand pieces (rows: 1, 2, 4, 8 or 16, not fewer than there
// are), piece (quarter, row) at quarter * rows + (row ^ turn), turn
// = the 8 inputs' number: so that neighbouring pieces of a row, written
// together, lie in different banks; the weights' scales and 16 + zero points,
// [output][group][2]; and 8-bit x's scales a group, [group][row].
struct Chunk {
  int stretches, log_stretches;  // a power of two, not fewer than the waves (one, too)
  int rows;
  int align;  // of the weights' rows: 16, 4 or 1
};

// Whether row m of x has no infinity or NaN: asked by a whole wave.
template <int X>
__device__ __forceinline__ bool row_is_finite(const Q4Args &a, int m, int lane) {
  const num_t<X> *x = (const num_t<X> *)a.x + m * a.x_stride;
#pragma unroll 1
  for (int k0 = 0; k0 < a.k; k0 += 512) {
    const int k = k0 + 8 * lane;
    num_t<X> v[8];
    load_n(x + k, (long)a.k - k, v);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; i++) bad |= !(fabsf(Num<X>::get(v[i])) < INFINITY);
    if (__any(bad)) return false;
  }
  return true;
}

// Output n of row m (the same in all lanes; n: of lane % 16) by one wave, in
// f64, lane / 16's eight inputs of each 32.
template <int X, int GROUP>
__device__ __forceinline__ float q4_alone(const Q4Args &a, int m, int n, int lane) {
  const int row_bytes = (a.k + 1) / 2;
  const num_t<X> *x = (const num_t<X> *)a.x + m * a.x_stride;
  const uint8_t *q = a.q + (long)n * row_bytes;
  const long g0 = (long)n * a.groups;
  double sum = 0.0;
#pragma unroll 1
  for (int k = lane / 16 * 8; k < a.k; k += 32) {
    num_t<X> v[8];
    uint8_t b[4];
    load_n(x + k, (long)a.k - k, v);
    load_n(q + k / 2, (long)row_bytes - k / 2, b);
    const long g = g0 + k / GROUP;
    const float s = a.scale_type == PPOCR_F32    ? ((const float *)a.scales)[g]
                    : a.scale_type == PPOCR_BF16 ? (float)((const __bf16 *)a.scales)[g]
                                                 : (float)((const _Float16 *)a.scales)[g];
    const int z = a.zeros ? a.zeros[g] : 8;
    double part = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) part += double(Num<X>::get(v[i])) * ((b[i / 2] >> i % 2 * 4 & 15) - z);
    sum += part * double(s);
  }
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  return float(sum);
}

template <int X, int NT, int GROUP, int SB>
__global__ __launch_bounds__(64 * kWaves, (X != PPOCR_F32 ? 4 : 2)) void q4_rows(Q4Args a, int e4m3, Chunk ch) {
  constexpr int SG = kStretch / GROUP, P = XRow<X>::parts, DW = XRow<X>::DW, XB = XRow<X>::size, N = 16 * NT;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), waves = threads / 64;
  const int col = lane % 16, quarter = lane / 16;
  // Blocks of 16 rows of x of one tile run on one XCD (blockIdx % 8), near one
  // another: the weights come from its L2 for all but the first.
  const int m_blocks = (a.m + 15) / 16, turn8 = blockIdx.x / 8;
  const int n0 = (turn8 / m_blocks * 8 + blockIdx.x % 8) * N, m0 = turn8 % m_blocks * 16, m_here = min(a.m - m0, 16);
  if (n0 >= a.n) return;
  const int n_here = min(a.n - n0, N);
  const int row_bytes = (a.k + 1) / 2, steps = (a.k + kStretch - 1) / kStretch;
  const bool x_grouped = X == PPOCR_I8 && a.x_group;
  const uint8_t *q0 = a.q + (long)n0 * row_bytes, *x0 = (const uint8_t *)a.x + m0 * a.x_stride * XB;

  const int frag = 4 * ch.rows * 16, a_stretch = 4 * P * frag;  // bytes
  uint8_t *ring = lds + wave * kRing * 1024, *lds_x = lds + waves * kRing * 1024;
  v2f *lds_s = (v2f *)(lds_x + ch.stretches * a_stretch);
  const int s_row = ch.stretches * SG + 1;  // (one more: 16 outputs' scales lie in different banks)
  float *lds_xs = (float *)(lds_s + N * s_row);

  // The ring's loads: the wave's next unit is tile l_tile of stretch l_step.
  // Piece p of row r has place 4 r + (p ^ turn), turn = r / 4 % 4: a read of 16
  // rows' pieces p touches every bank once. (Past a row's end or the last row
  // something else is read, which meets zeros of x or is not stored.)
  int l_step = wave, l_tile = 0, l_slot = 0;
  const int l_at = 16 * ((lane ^ lane >> 4) & 3), tile_bytes = 16 * row_bytes;  // (k is at most 2^24)
  const uint8_t *l_from = q0 + wave * (kStretch / 2);  // of its row 0, in the common case
  const uint32_t l_off = (uint32_t)(lane / 4) * row_bytes + l_at;
  const bool common = ch.align == 16 && n_here == N;
  auto load = [&] {
    const int k2 = l_step * (kStretch / 2);
    uint8_t *to = ring + l_slot * 1024;
    if (common && k2 + kStretch / 2 <= row_bytes) {
      __builtin_amdgcn_global_load_lds((const void *)(l_from + l_off), (lds_void *)to, 16, 0, 0);
    } else if (ch.align == 16) {
      const long row = min(16 * l_tile + lane / 4, n_here - 1);
      __builtin_amdgcn_global_load_lds((const void *)(q0 + row * row_bytes + (k2 + l_at < row_bytes ? k2 + l_at : 0)),
                                       (lds_void *)to, 16, 0, 0);
    } else if (ch.align == 4) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = 4 * i + lane / 16, at = k2 + 16 * ((lane / 4 ^ i) & 3) + 4 * (lane & 3);
        const uint32_t row = min(16 * l_tile + r, n_here - 1);
        __builtin_amdgcn_global_load_lds((const void *)(q0 + (row * row_bytes + (at < row_bytes ? at : 0))),
                                         (lds_void *)(to + 256 * i), 4, 0, 0);
      }
    } else {
      const long row = min(16 * l_tile + lane / 4, n_here - 1);
      uint8_t b[16];
      load_n(q0 + row * row_bytes + k2 + l_at, (long)row_bytes - k2 - l_at, b);
      __builtin_memcpy(to + 16 * lane, b, 16);
    }
    l_slot = l_slot + 1 == kRing ? 0 : l_slot + 1;
    l_from += tile_bytes;
    if (++l_tile == NT) l_tile = 0, l_step += waves, l_from += waves * (kStretch / 2) - (long)NT * tile_bytes;
  };
  // Waits until at most `ahead` later units are on their way.
  auto arrived = [&](int ahead) {
    if (ch.align == 16 && ahead >= kRing - 1)
      ring_wait<kRing - 1>();
    else if (ch.align == 16)
      ring_wait_chunks<1, kRing - 2>(ahead);
    else if (ch.align == 4)
      ring_wait_chunks<4, kRing - 1>(min(ahead, kRing - 1));
    asm volatile("" ::: "memory");
  };

  // Stretches first .. first + ch.stretches - 1 of x, scales and zero points,
  // a batch of a thread's loads of each at a time, none of them behind a
  // branch: a load under one is waited for at its end. The counts are powers
  // of two.
  const uint8_t *zeros = a.zeros ? a.zeros : a.q;  // (read and not used; q has more bytes)
  auto stage = [&](int first) {
    constexpr int BATCH = 4, SBATCH = 4;
    const int log_p = ch.log_stretches + 4, pieces = 1 << log_p, all = m_here << log_p;
    const int log_g = ch.log_stretches + (SG == 4 ? 2 : SG == 2 ? 1 : 0), groups = 1 << log_g, g0 = first * SG;
    const int sums = n_here << log_g;
    auto put = [&](int r, int p, const uint32_t(&v)[DW]) {
      v4u f[P];
      XRow<X>::operands(v, e4m3, f);
#pragma unroll
      for (int c = 0; c < P; c++)
        *(v4u *)(lds_x + (p / 4 * P + c) * frag + (p % 4 * ch.rows + (r ^ (p & (ch.rows - 1)))) * 16) = f[c];
    };
    for (int i0 = tid, j0 = tid; i0 < all || j0 < sums; i0 += BATCH * threads, j0 += SBATCH * threads) {
      uint32_t v[BATCH][DW], s[SBATCH][1], z[SBATCH];
#pragma unroll
      for (int u = 0; u < BATCH; u++) {
        const int i = i0 + u * threads, k = first * kStretch + 8 * (i & (pieces - 1));
        const bool in = i < all && k + 8 <= a.k;  // (else the last whole piece's bytes, of which nothing is kept)
        const uint32_t off = in ? (uint32_t)(i >> log_p) * (uint32_t)a.x_stride + k : 0;
        if (a.k >= 8) load_dwords<false, XB, 8>(x0 + (uint64_t)off * XB, 8, v[u]);
#pragma unroll
        for (int d = 0; d < DW; d++) v[u][d] = in ? v[u][d] : 0;
      }
#pragma unroll
      for (int u = 0; u < SBATCH; u++) {
        const int j = min(j0 + u * threads, sums - 1), g = min(g0 + (j & (groups - 1)), a.groups - 1);
        const long at = (long)(n0 + (j >> log_g)) * a.groups + g;
        load_dwords<false, SB, 1>((const uint8_t *)a.scales + at * SB, 1, s[u]);
        z[u] = zeros[at];
      }
#pragma unroll
      for (int u = 0; u < BATCH; u++) {
        const int i = i0 + u * threads;
        if (i < all) put(i >> log_p, i & (pieces - 1), v[u]);
      }
#pragma unroll
      for (int u = 0; u < SBATCH; u++) {
        const int j = j0 + u * threads, g = j & (groups - 1);
        const uint32_t raw = SB == 2 ? s[u][0] & 0xffff : s[u][0];
        const float f = SB == 4 ? __uint_as_float(raw)
                        : a.scale_type == PPOCR_BF16 ? __uint_as_float(raw << 16)
                                                     : (float)__builtin_bit_cast(_Float16, (uint16_t)raw);
        if (j < sums)
          lds_s[(j >> log_g) * s_row + g] = v2f{g0 + g < a.groups ? f : 0.0f, 16.0f + (float)(a.zeros ? z[u] : 8)};
      }
    }
    const int cut = a.k / 8 - first * 16;  // the piece that x's rows end in
    if (a.k % 8 && cut < pieces) {
      __syncthreads();
      for (int r = tid; r < m_here; r += threads) {
        uint32_t v[DW];
        load_dwords<true, XB, 8>(x0 + (r * a.x_stride + a.k / 8 * 8) * XB, a.k % 8, v);
        put(r, cut, v);
      }
    }
    if (x_grouped)
      for (int i = tid; i < m_here << log_g; i += threads) {
        const int r = i >> log_g, g = i & (groups - 1);
        lds_xs[g * 16 + r] = g0 + g < a.groups ? a.x_scales[(m0 + r) * (long)a.groups + g0 + g] : 0.0f;
      }
  };

  v4f acc[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) acc[j] = v4f{0, 0, 0, 0};

  constexpr uint32_t one = X == PPOCR_F16 ? 0x3c003c00u : 0x3f803f80u;
  const v4u ones{one, one, one, one};
  uint32_t mask = 0x000f000fu << kTop<X>, base = X == PPOCR_F16 ? 0x4c004c00u : 0x41804180u;
  asm volatile("" : "+s"(mask), "+v"(base));
  const int turns = (steps + waves - 1) / waves, each = ch.stretches / waves;
  const int mine = (steps - wave + waves - 1) / waves;  // this wave's stretches
  int units = mine * NT;                             // left to use
  for (int u = 0; u < min(units, kRing); u++) load();
  const uint8_t *my_x = lds_x + (quarter * ch.rows + (min(col, ch.rows - 1) ^ (quarter & (ch.rows - 1)))) * 16;
  const uint8_t *my_w = ring + 64 * col + 4 * quarter;  // + 16 (j ^ col / 4): inputs 32 j + 8 quarter .. + 7
  int slot = 0;

  for (int c0 = 0; c0 < turns; c0 += each) {
    if (c0) __syncthreads();
    stage(c0 * waves);
    __syncthreads();
    for (int t = c0; t < min(c0 + each, mine); t++) {
      const int at = (t - c0) * waves + wave;  // the stretch's place in the chunk
      // Operands of the stretch's four times 32 inputs (piece 4 c + quarter:
      // c only turns rows where there are more than four), and sum x.
      v4u xf[4][P];
      v4f sx[SG][P];
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int p = 0; p < P; p++)
          xf[c][p] = *(const v4u *)(lds + ((uint32_t)(my_x - lds) ^ (4 * c & (ch.rows - 1)) * 16) + at * a_stretch +
                                    (c * P + p) * frag);
#pragma unroll
      for (int g = 0; g < SG; g++)
#pragma unroll
        for (int p = 0; p < P; p++) {
          sx[g][p] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int c = g * 4 / SG; c < (g + 1) * 4 / SG; c++) sx[g][p] = mfma<X>(xf[c][p], ones, sx[g][p]);
        }
#pragma unroll
      for (int j = 0; j < NT; j++) {
        units--;
        arrived(units);
        uint32_t w[4];
#pragma unroll
        for (int c = 0; c < 4; c++) w[c] = *(const uint32_t *)(my_w + slot * 1024 + 16 * (c ^ col >> 2));
        v2f sz[SG];
#pragma unroll
        for (int g = 0; g < SG; g++) sz[g] = lds_s[(16 * j + col) * s_row + at * SG + g];
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the slot has been read
        asm volatile("" ::: "memory");
        slot = slot + 1 == kRing ? 0 : slot + 1;
        if (units >= kRing) load();
#pragma unroll
        for (int g = 0; g < SG; g++) {
          constexpr int CS = 4 / SG;  // products of 32 inputs a group
          v4u wf[CS];
#pragma unroll
          for (int c = 0; c < CS; c++) wf[c] = weights16<X>(w[g * CS + c], mask, base);
          v4f xs{1, 1, 1, 1};
          if constexpr (X == PPOCR_I8)
            if (x_grouped) xs = *(const v4f *)(lds_xs + (at * SG + g) * 16 + 4 * quarter);
          v4f d[P];
#pragma unroll
          for (int p = 0; p < P; p++) {
            d[p] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < CS; c++) d[p] = mfma<X>(xf[g * CS + c][p], wf[c], d[p]);
          }
#pragma unroll
          for (int r = 0; r < 4; r++) {
            float v[P];
#pragma unroll
            for (int p = 0; p < P; p++) v[p] = fmaf(-sz[g][1], sx[g][p][r], d[p][r]);
            if constexpr (P == 3) v[0] = fmaf(fmaf(v[2], 1.0f / 256.0f, v[1]), 1.0f / 256.0f, v[0]);
            acc[j][r] = fmaf(X == PPOCR_I8 ? sz[g][0] * xs[r] : sz[g][0], v[0], acc[j][r]);
          }
        }
        asm volatile("" : "+v"(acc[j]));  // here: or the compiler puts all tiles' last steps off to the loop's end
      }
    }
  }
  __syncthreads();

  // The waves' parts, in order, four tiles at a time (4 KB a wave).
  float (*red)[4][256] = (float (*)[4][256])lds;
  constexpr int AT = NT < 4 ? NT : 4;
#pragma unroll
  for (int t0 = 0; t0 < NT; t0 += AT) {
    if (t0) __syncthreads();
#pragma unroll
    for (int t = 0; t < AT; t++)
      *(v4f *)&red[wave][t][4 * lane] = acc[t0 + t];
    __syncthreads();
    auto row_of = [&](int i) { return m0 + i / 16 % 16; };
    auto col_of = [&](int i) { return n0 + 16 * (t0 + i / 256) + i % 16; };
    auto sum_of = [&](int i) {
      float v = 0.0f;
      for (int w = 0; w < waves; w++) v += red[w][i / 256][4 * (i % 16 + 16 * (i / 64 % 4)) + i / 16 % 4];
      return v;
    };
    auto put = [&](int m, int n, float v) {
      const long at = m * a.y_stride + n;
      if (a.y_type == PPOCR_F32)
        ((float *)a.y)[at] = a.bias ? v + ((const float *)a.bias)[n] : v;
      else if (a.y_type == PPOCR_BF16)
        ((__bf16 *)a.y)[at] = (__bf16)(a.bias ? v + (float)((const __bf16 *)a.bias)[n] : v);
      else
        ((_Float16 *)a.y)[at] = (_Float16)(a.bias ? v + (float)((const _Float16 *)a.bias)[n] : v);
    };
    bool bad = false;
    for (int i = tid; i < AT * 256; i += threads) {
      const int m = row_of(i), n = col_of(i);
      if (m >= a.m || n >= a.n) continue;
      float v = sum_of(i);
      if constexpr (X == PPOCR_I8)
        if (!x_grouped) v *= a.x_scales[m];
      bad |= !(fabsf(v) < INFINITY);
      put(m, n, v);
    }
    if constexpr (X == PPOCR_F32 || X == PPOCR_BF16)
      if (__any(bad)) {  // rare: this wave's rows, 16 outputs at a time
        for (int i0 = 64 * wave; i0 < AT * 256; i0 += threads) {
          const int m = row_of(i0 + lane), n = col_of(i0 + lane);
          const unsigned long long again =
              __ballot(m < a.m && n < a.n && !(fabsf(sum_of(i0 + lane)) < INFINITY));
          for (int r = 0; r < 4; r++) {
            const int row = row_of(i0) + r;
            if (!(again >> 16 * r & 0xffff) || !row_is_finite<X>(a, row, lane)) continue;  // (NaN stays)
            const float v = q4_alone<X, GROUP>(a, row, min(n, a.n - 1), lane);
            if (lane / 16 == r && again >> lane & 1) put(m, n, v);  // (the lane that wrote it)
          }
        }
      }
  }
}

template <int X, int NT, int GROUP, int SB>
hipError_t launch_of(const Q4Args &a, int e4m3, hipStream_t s) {
  const int steps = (a.k + kStretch - 1) / kStretch, row_bytes = (a.k + 1) / 2;
  const int strips = (a.n + 16 * NT - 1) / (16 * NT), m_blocks = (a.m + 15) / 16;
  const dim3 grid((strips + 7) / 8 * 8 * m_blocks);
  Chunk ch;
  ch.align = row_bytes % 16 == 0 && uintptr_t(a.q) % 16 == 0 ? 16 : row_bytes % 4 == 0 && uintptr_t(a.q) % 4 == 0 ? 4 : 1;
  ch.rows = 1;
  while (ch.rows < 16 && ch.rows < a.m) ch.rows *= 2;
  constexpr int SG = kStretch / GROUP;
  const int a_stretch = 4 * XRow<X>::parts * 64 * ch.rows + SG * 16 * NT * 8 + (a.x_group ? SG * 64 : 0);
  constexpr int once = 16 * NT * 8;  // the scales' extra column
  // Each of the workgroups that run on a CU at once has its share of its LDS.
  // At least a stretch a wave.
  int waves = q4_waves(a.k);
  const int on_cu = std::min((strips * (long)m_blocks + 255) / 256, long(q4_at_once(X) / 256 * (kWaves / waves)));
  const int room = 152 * 1024 / on_cu;
  while (waves > 1 && waves * (a_stretch + kRing * 1024) + once > 152 * 1024) waves /= 2;
  ch.stretches = waves;
  while (ch.stretches < steps && waves * kRing * 1024 + 2 * ch.stretches * a_stretch + once <= room) ch.stretches *= 2;
  ch.log_stretches = __builtin_ctz(ch.stretches);
  const hipError_t e = allow_lds_of<&q4_rows<X, NT, GROUP, SB>>(160 * 1024);
  if (e != hipSuccess) return e;
  const int bytes = std::max(waves * kRing * 1024 + ch.stretches * a_stretch + once, waves * 4096);
  return launch_kernel(q4_rows<X, NT, GROUP, SB>, grid, dim3(64 * waves), bytes, s, a, e4m3, ch);
}

template <int X, int NT, int GROUP>
hipError_t launch_rows(const Q4Args &a, int e4m3, hipStream_t s) {
  return a.scale_type == PPOCR_F32 ? launch_of<X, NT, GROUP, 4>(a, e4m3, s)
                                   : launch_of<X, NT, GROUP, 2>(a, e4m3, s);
}

template <int X, int NT>
hipError_t launch_tile(const Q4Args &a, int e4m3, hipStream_t s) {
  if (a.group == 32) return launch_rows<X, NT, 32>(a, e4m3, s);
  if (a.group == 64) return launch_rows<X, NT, 64>(a, e4m3, s);
  return launch_rows<X, NT, 128>(a, e4m3, s);
}

}  // namespace

// One type of x a file (product_*.hip).
hipError_t PPOCR_Q4_LAUNCH(const Q4Args &a, int e4m3, hipStream_t s) {
  constexpr int X = PPOCR_Q4_X;
  switch (q4_tiles(X, a.m, a.n, a.k)) {
    case 1: return launch_tile<X, 1>(a, e4m3, s);
    case 2: return launch_tile<X, 2>(a, e4m3, s);
    case 4: return launch_tile<X, 4>(a, e4m3, s);
  }
  if constexpr (X == PPOCR_F32) return launch_tile<X, 8>(a, e4m3, s);
  return hipErrorInvalidValue;
}

}  // namespace ppocr
