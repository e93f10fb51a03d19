// Products with 4-bit weights of rows in bf16 (see product.hpp).
#define PPOCR_Q4_X PPOCR_BF16
#define PPOCR_Q4_LAUNCH launch_q4_bf16
#include "product.hpp"
