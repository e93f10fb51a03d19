// Products with 4-bit weights of rows in f16 (see product.hpp).
#define PPOCR_Q4_X PPOCR_F16
#define PPOCR_Q4_LAUNCH launch_q4_f16
#include "product.hpp"
