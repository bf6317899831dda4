// The operands of a linear over 8-bit weights (mt_linear_f8).
#pragma once

#include "f8.hpp"

namespace mt {

// Most values of a row that few_rows_kernel normalises (its blocks' sums of squares stand in LDS, 16 rows
// of 256); mt_quantize_f8 takes 16 times that in the same space.
constexpr uint32_t F8_NORM_K = 32768;

struct F8LinearArgs {
    const void *x;       // codes (xt MT_F8), or rows of the type xt
    const uint8_t *xs;   // their scales, row stride ldxs
    const uint8_t *w, *ws, *w2, *w2s;  // weights [N, K] and their scales, row stride lds
    const uint16_t *bias, *norm;
    float *y;
    uint32_t M, N, K, ldx, ldxs, lds, ldy, flags;
    float eps;
};

}  // namespace mt
