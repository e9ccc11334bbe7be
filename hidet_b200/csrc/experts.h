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

// Few tokens of one launch: 64, or as many as have 1024 assignments.
constexpr int64_t kExpertsTokens = 64, kExpertsAssignments = 1024;
inline int64_t experts_at_once(int64_t tokens, int64_t top) {
    int64_t most = top * kExpertsTokens > kExpertsAssignments ? kExpertsAssignments / top : kExpertsTokens;
    if (most < 1) most = 1;
    return tokens < most ? tokens : most;
}

// Rows and bases in lines of 16 bytes, up to 512 experts.
bool experts_fast(const ExpertsArgs &p);
// Few tokens, those of one launch.
size_t experts_stream_bytes(int64_t tokens, int64_t inner, int64_t top);
int launch_experts_stream(const ExpertsArgs &p, unsigned int *counters, float *scratch, cudaStream_t stream);
// Many, as many as one launch takes.
int64_t experts_many_at_once(int64_t tokens, int64_t hidden, int64_t inner, int64_t count, int64_t top);
size_t experts_many_bytes(int64_t tokens, int64_t hidden, int64_t inner, int64_t count, int64_t top);
int launch_experts_many(const ExpertsArgs &p, unsigned int *counters, void *scratch, cudaStream_t stream);

}  // namespace b200q
