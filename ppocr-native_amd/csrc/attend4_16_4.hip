// Attention over a cache in 4 bits: bf16 and f16 queries, four columns a query head.
#include "attend4.hpp"

namespace ppocr {
template hipError_t launch_attention4<false, 4>(Attend4Args &, hipStream_t);
}  // namespace ppocr
