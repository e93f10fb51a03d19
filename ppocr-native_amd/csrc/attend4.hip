// Attention over a cache in 4 bits: the choice of a kernel, the parts of a split
// cache and their join.
#include "parts4.hpp"

namespace ppocr {
namespace {

constexpr int kMostParts4 = 128;

// Joins a row's parts, a workgroup a head of a text: lane i of each wave has
// parts i and i + 64's factors, wave w adds parts w, w + 4, ... of them.
// J: 64s of dim, rounded up to a power of two.
template <int J>
__global__ __launch_bounds__(256) void kv4_attention_join(Attend4Args a, int keys) {
  __shared__ float lds_o[4][256], lds_f[kMostParts4];
  const int head = blockIdx.x, b = blockIdx.y, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const Seen s = seen4(a, b, keys);
  const int each = tiles_a_part(s.tiles, each4(a, keys), a.splits);
  const int parts = max(1, (s.tiles + each - 1) / each), dim = a.c.dim, row = dim + 2, far = lane + 64;
  const float *p = a.part + ((long)b * a.heads + head) * a.splits * row;
  const float b0 = lane < parts ? p[(long)lane * row] : -INFINITY, l0 = lane < parts ? p[(long)lane * row + 1] : 0.0f;
  const float b1 = far < parts ? p[(long)far * row] : -INFINITY, l1 = far < parts ? p[(long)far * row + 1] : 0.0f;
  float base = fmaxf(b0, b1);
#pragma unroll
  for (int o = 32; o; o >>= 1) base = fmaxf(base, __shfl_xor(base, o));
  const float f0 = __builtin_amdgcn_exp2f(b0 - base), f1 = __builtin_amdgcn_exp2f(b1 - base);
  float sum = f0 * l0 + f1 * l1;
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  if (wave == 0) lds_f[lane] = f0, lds_f[far] = f1;
  __syncthreads();
  float o[J] = {};
#pragma unroll 8
  for (int i = wave; i < parts; i += 4) {
    const float f = lds_f[i];
#pragma unroll
    for (int j = 0; j < J; j++)  // (past dim: its last value, not kept)
      o[j] = fmaf(f, p[(long)i * row + 2 + min(lane + 64 * j, dim - 1)], o[j]);
  }
#pragma unroll
  for (int j = 0; j < J; j++) lds_o[wave][lane + 64 * j] = o[j];
  __syncthreads();
  const int d = threadIdx.x;
  if (d < dim) {
    const float v = (lds_o[0][d] + lds_o[1][d]) + (lds_o[2][d] + lds_o[3][d]);
    put_at(a.y, b * a.y_stride + (long)head * dim + d, a.type, sum == 0.0f ? 0.0f : v / sum);
  }
}

}  // namespace

PagedParts kv4_parts(int batch, int heads, int kv_heads, long longest) {
  // At least as long as were 2048 workgroups of it if all texts were the longest, or
  // 4096 where the device makes them longer, by the lengths that it has; but of 512
  // tokens at least, or 128 where that leaves too few for the card. A text of 512 is
  // done without a join.
  const int per = heads / kv_heads, keys = 16 * halves4(copies4(per)), least = 512 / keys, few = 128 / keys;
  const long groups = (long)batch * kv_heads * ((per + 15) / 16), tiles = (longest + keys - 1) / keys + 2;
  const long most = groups <= kShared4 ? 4096 : 2048;
  long each = (tiles * groups + most - 1) / most;
  if (each < least) {
    const long fill = (tiles * groups + 511) / 512;
    each = tiles <= least + 1 ? least + 1 : fill < few ? few : fill < least ? fill : least;
  }
  if (each < (tiles + kMostParts4 - 1) / kMostParts4) each = (tiles + kMostParts4 - 1) / kMostParts4;
  const long splits = (tiles + each - 1) / each;
  return {int(splits < 1 ? 1 : splits), int(each)};
}

hipError_t launch_kv4_attention(Attend4Args a, hipStream_t s) {
  const int copies = copies4(a.heads / a.c.heads);
  const bool two = a.type == PPOCR_F32;
  const hipError_t e = copies == 4   ? (two ? launch_attention4<true, 4>(a, s) : launch_attention4<false, 4>(a, s))
                       : copies == 2 ? (two ? launch_attention4<true, 2>(a, s) : launch_attention4<false, 2>(a, s))
                                     : (two ? launch_attention4<true, 1>(a, s) : launch_attention4<false, 1>(a, s));
  if (e != hipSuccess || a.splits == 1) return e;
  const dim3 grid(a.heads, a.batch), block(256);
  const int keys = 16 * halves4(copies);
  if (a.c.dim <= 64) return launch_kernel(kv4_attention_join<1>, grid, block, 0, s, a, keys);
  if (a.c.dim <= 128) return launch_kernel(kv4_attention_join<2>, grid, block, 0, s, a, keys);
  return launch_kernel(kv4_attention_join<4>, grid, block, 0, s, a, keys);
}

}  // namespace ppocr
