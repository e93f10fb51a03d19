// Products with 4-bit weights of rows in f32 (see product.hpp).
#define PPOCR_Q4_X PPOCR_F32
#define PPOCR_Q4_LAUNCH launch_q4_f32
#include "product.hpp"
