// Products with 4-bit weights of rows in 8 bits (both kinds) (see product.hpp).
#define PPOCR_Q4_X PPOCR_I8
#define PPOCR_Q4_LAUNCH launch_q4_i8
#include "product.hpp"
