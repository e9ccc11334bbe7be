// What the kernels of a layer of experts share: the operands of a call.
//
//     a token t is sent to experts[t, j] with weights[t, j], j < top: an assignment
//     (g, u)_f = scale1[e, 2 f + (0, 1)] sum_h gate_up[e, 2 f + (0, 1), h] x[t, h];   h[t, j, f] = silu(g) u
//     out[t, n] = residual[t, n] + sum_j weights[t, j] scale2[e, n] sum_f down[e, n, f] h[t, j, f]
// An assignment to no expert (a negative one) counts as nothing, one beyond them too, which is reported.
#pragma once

#include "common.cuh"
#include "status_bits.h"

namespace b200q {

struct ExpertsArgs {
    const void *x;
    int64_t x_stride;
    const int32_t *experts;
    const float *weights;
    const int8_t *gate_up, *down;
    const void *gate_up_scale, *down_scale;
    const void *residual;  // [tokens, residual_stride] of x's type, or null
    void *out;             // [tokens, hidden]
    int64_t residual_stride;
    int tokens, hidden, inner, count, top;
    int scale_type;        // b200q_float_type
    int type;              // of x, residual and out: B200Q_F16 or B200Q_BF16
    unsigned int *status;
};

}  // namespace b200q
