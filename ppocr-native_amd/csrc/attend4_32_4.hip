// Attention over a cache in 4 bits: f32 queries, four columns a query head.
#include "attend4.hpp"

namespace ppocr {
template hipError_t launch_attention4<true, 4>(Attend4Args &, hipStream_t);
}  // namespace ppocr
