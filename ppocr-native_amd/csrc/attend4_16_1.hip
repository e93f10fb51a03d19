// Attention over a cache in 4 bits: bf16 and f16 queries, one column a query head.
#include "attend4.hpp"

namespace ppocr {
template hipError_t launch_attention4<false, 1>(Attend4Args &, hipStream_t);
}  // namespace ppocr
