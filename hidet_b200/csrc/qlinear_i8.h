// What the kernels of the int8 x int8 product share: the operands of a call, and what follows the whole-number sum.
//
//     c[m, n] = float(sum_k a[m, k] w[k, n]) * scale[n] * a_scale[m];   + bias[n];   silu(gate) * up of channel pairs;   + residual[m, .]
// The sum is exact: 32 bits hold K = 131071 products of 2^14.  All that follows is float, rounded once to the result's type.
#pragma once

#include "common.cuh"

namespace b200q {

constexpr int64_t kMostInner = 131071;
constexpr int64_t kMostOuter = 0x7fffffffLL - 255;  // of M and N: tiles of up to 256, whose ends are ints too

struct I8Args {
    const int8_t *a, *w;
    const float *a_scale;
    const void *scale;     // [N], scale_type
    const void *bias;      // [N] of the result's type, or null
    const void *residual;  // [M, ldr] of the result's type, or null
    void *c;
    int64_t ldr;
    int M, N, K;
    int scale_type;        // b200q_float_type
    int out_type;          // B200Q_F16 or B200Q_BF16
    bool pairs;            // the channels are (gate_j, up_j)
    bool nk;               // the weight is [N, K]
    bool residual_vec;     // residual rows can be read as 16-byte vectors
    unsigned int *status;
};

// Every alignment and size.
int launch_i8_any(const I8Args &p, cudaStream_t stream);
// 16-byte aligned bases and rows of both operands and the result; tm tokens per tile, a multiple of 32 up to 256; split (1, 2 or 4) pairs that
// share a tile's K: with more than one, all tiles' pairs have to have a place at once.
int launch_i8_pair(const I8Args &p, int tm, int split, cudaStream_t stream);
// tm a multiple of 16 up to 256, a cluster of up to eight CTAs for a tile.
int launch_i8_split(const I8Args &p, int tm, int cluster, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ float i8_scale(const void *p, int type, int64_t i) {
    if (type == B200Q_F16) return __half2float(static_cast<const __half *>(p)[i]);
    if (type == B200Q_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return static_cast<const float *>(p)[i];
}
// a value of the result's type
__device__ __forceinline__ float i8_value(const void *p, int type, int64_t i) {
    return type == B200Q_F16 ? __half2float(static_cast<const __half *>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void i8_store(void *p, int type, int64_t i, float v) {
    if (type == B200Q_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}
#endif

}  // namespace b200q
