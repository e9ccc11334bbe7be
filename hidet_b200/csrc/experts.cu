// A layer of experts on int8 weights: the entry point, and the kernels that take every alignment.
#include "experts.h"
#include "experts_digits.cuh"
#include "serving.cuh"

namespace b200q {
namespace {

constexpr int ANY_WARPS = 8;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A warp a value of h, and a warp a value of out: byte by byte, a weight read again for every token (48 tokens, six of 64 of 2044 x 1404: 1450 us, 103 of 2048 x 1408 where
// rows are aligned; 8 tokens, eight of 600 of 1024 x 512: 81, 33 of 512).  For rows that are not multiples of 16 bytes, bases that are not aligned, and more than 512 experts.
__global__ void __launch_bounds__(32 * ANY_WARPS) experts_any_up_kernel(const ExpertsArgs p, float *h) {
    const int f = blockIdx.x * ANY_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();
    if (f >= p.inner) return;
    for (int64_t a = blockIdx.y; a < (int64_t)p.tokens * p.top; a += gridDim.y) {
        const int e = p.experts[a];
        if (e < 0 || e >= p.count) {
            if (e >= p.count && f == 0 && lane == 0 && p.status != nullptr) atomicOr(p.status, kBadExpert);
            continue;
        }
        const int64_t row = (int64_t)e * 2 * p.inner + 2 * f;
        const int8_t *w = p.gate_up + row * p.hidden;
        float g = 0.0f, u = 0.0f;
        for (int i = lane; i < p.hidden; i += 32) {
            const float x = token_value(p.x, p.type, a / p.top * p.x_stride + i);
            g = fmaf(x, (float)w[i], g);
            u = fmaf(x, (float)w[p.hidden + i], u);
        }
        g = warp_sum(g) * scale_at(p.gate_up_scale, p.scale_type, row);
        u = warp_sum(u) * scale_at(p.gate_up_scale, p.scale_type, row + 1);
        if (lane == 0) h[a * p.inner + f] = silu(g) * u;
    }
}
__global__ void __launch_bounds__(32 * ANY_WARPS) experts_any_down_kernel(const ExpertsArgs p, const float *h) {
    const int n = blockIdx.x * ANY_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();
    if (n >= p.hidden) return;
    for (int t = blockIdx.y; t < p.tokens; t += gridDim.y) {
        float sum = 0.0f;
        for (int j = 0; j < p.top; ++j) {
            const int64_t a = (int64_t)t * p.top + j;
            const int e = p.experts[a];
            if (e < 0 || e >= p.count) continue;
            const int64_t row = (int64_t)e * p.hidden + n;
            float y = 0.0f;
            for (int i = lane; i < p.inner; i += 32) y = fmaf(__ldcg(h + a * p.inner + i), (float)p.down[row * p.inner + i], y);
            sum = fmaf(warp_sum(y) * scale_at(p.down_scale, p.scale_type, row), p.weights[a], sum);
        }
        if (lane == 0) {
            if (p.residual != nullptr) sum += token_value(p.residual, p.type, t * p.residual_stride + n);
            const int64_t at = (int64_t)t * p.hidden + n;
            if (p.type == B200Q_F16) static_cast<__half *>(p.out)[at] = __float2half_rn(sum);
            else static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(sum);
        }
    }
}

int launch_any(const ExpertsArgs &p, float *h, cudaStream_t stream) {
    const int64_t rows = (int64_t)p.tokens * p.top;
    int rc = B200Q_OK;
    if (p.inner > 0 && rows > 0) {
        rc = launch_after("experts_any_up_kernel", experts_any_up_kernel, dim3((unsigned)ceil_div(p.inner, ANY_WARPS), (unsigned)(rows < 65535 ? rows : 65535)),
                          32 * ANY_WARPS, 0, 1, stream, p, h);
    }
    if (rc != B200Q_OK) return rc;
    return launch_after("experts_any_down_kernel", experts_any_down_kernel, dim3((unsigned)ceil_div(p.hidden, ANY_WARPS), (unsigned)(p.tokens < 65535 ? p.tokens : 65535)),
                        32 * ANY_WARPS, 0, 1, stream, p, h);
}

// Whether the tokens are many: made digits of once, for all tiles of the weights (experts_many.cu), or by every tile for itself (experts_stream.cu).  The latter pays by the assignment and tile,
// and at its shared parts by an expert's assignments; the former some microseconds for the kernels in front, between and behind.  us, the latter and the former:
//     8, 16, 32, 64 tokens, 2 of 8 experts of 4096 x 14336   207 206    242 234    276 237    330 248
//     24, 48, 64 tokens, 6 of 64 of 2048 x 1408               95 99     107 104    113 105
//     48, 64 tokens, 8 of 128 of 2048 x 768                  111 113    120 119
//     16, 32 tokens, 2 of 4 of 1024 x 4096                    28 30      37 32
//     16, 32, 64 tokens, 2 of 16 of 2048 x 8192              123 128    140 142    157 143
//     16 tokens, 4 and 8 of 8 of 512 x 1024                   23 23      24 22        8, 16 tokens, 4 of 4 of 2048 x 4096   35.5 36.7    42.5 39
// More than 64 tokens would have the weights read again by the latter (128 tokens, 2 of 8 of 4096 x 14336: 655 270).
bool are_many(int64_t tokens, int64_t hidden, int64_t inner, int64_t count, int64_t top) {
    const double assignments = (double)tokens * (double)top;
    return tokens > kExpertsTokens || assignments / (double)(count > 0 ? count : 1) + 1.5e-8 * assignments * (double)hidden * (double)inner > 16.0;
}

}  // namespace
}  // namespace b200q

extern "C" {

B200Q_API size_t b200q_mixture_of_experts_workspace_bytes(int64_t tokens, int64_t hidden, int64_t inner, int64_t count, int64_t top) {
    using namespace b200q;
    if (tokens <= 0 || hidden <= 0 || inner < 0 || count < 0 || top <= 0) return 0;
    const size_t few = experts_stream_bytes(experts_at_once(tokens, top), inner, top);
    const size_t many = are_many(tokens, hidden, inner, count, top) ? experts_many_bytes(experts_many_at_once(tokens, hidden, inner, count, top), hidden, inner, count, top) : 0;
    return kWorkspaceHead + (few > many ? few : many);
}

B200Q_API int b200q_mixture_of_experts(const void *x, int64_t x_stride, const int32_t *experts, const float *weights, const void *gate_up, const void *gate_up_scale,
                                       const void *down, const void *down_scale, const void *residual, int64_t residual_stride, void *out, int64_t tokens, int64_t hidden,
                                       int64_t inner, int64_t count, int64_t top, int type, int scale_type, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace b200q;
    const char *op = "mixture_of_experts";
    if (tokens < 0 || hidden < 0 || inner < 0 || count < 0 || top < 0 || x_stride < 0 || residual_stride < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative size or stride", op);
    if (type != B200Q_F16 && type != B200Q_BF16) return set_error(B200Q_INVALID_ARGUMENT, "%s: tokens are f16 or bf16, not type %d", op, type);
    if (scale_type < B200Q_F16 || scale_type > B200Q_F32) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown type of the scales %d", op, scale_type);
    if (tokens == 0 || hidden == 0) return B200Q_OK;
    if (tokens > 0xffffff || top > 4096 || hidden > 0x3fffffff || inner > 0x1fffffff || count > 0x3fffffff || tokens * top > 0x3fffffff) {
        return set_error(B200Q_UNSUPPORTED, "%s: %lld tokens of %lld elements, %lld of %lld experts of %lld", op, (long long)tokens, (long long)hidden, (long long)top,
                         (long long)count, (long long)inner);
    }
    if (out == nullptr || x == nullptr || (top > 0 && (experts == nullptr || weights == nullptr)) ||
        (count > 0 && inner > 0 && (gate_up == nullptr || gate_up_scale == nullptr || down == nullptr || down_scale == nullptr))) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    }
    const size_t need = b200q_mixture_of_experts_workspace_bytes(tokens, hidden, inner, count, top);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
        return set_error(B200Q_WORKSPACE_TOO_SMALL, "%s: needs %zu bytes of workspace, got %zu", op, need, workspace == nullptr ? (size_t)0 : workspace_bytes);
    }
    if (!aligned_to(workspace, 16)) return set_error(B200Q_INVALID_ARGUMENT, "%s: the workspace is not 16-byte aligned", op);
    ExpertsArgs p = {};
    p.x = x, p.x_stride = x_stride, p.experts = experts, p.weights = weights, p.gate_up = static_cast<const int8_t *>(gate_up), p.down = static_cast<const int8_t *>(down);
    p.gate_up_scale = gate_up_scale, p.down_scale = down_scale, p.residual = residual, p.out = out, p.residual_stride = residual_stride;
    p.tokens = (int)tokens, p.hidden = (int)hidden, p.inner = (int)inner, p.count = (int)count, p.top = (int)top, p.scale_type = scale_type, p.type = type;
    p.status = device_status_word();
    float *scratch = reinterpret_cast<float *>(static_cast<char *>(workspace) + kWorkspaceHead);
    const bool fast = experts_fast(p), many = fast && are_many(tokens, hidden, inner, count, top);
    const int64_t at_once = many ? experts_many_at_once(tokens, hidden, inner, count, top) : experts_at_once(tokens, top);
    for (int64_t t = 0; t < tokens; t += at_once) {
        ExpertsArgs q = p;
        q.tokens = (int)(tokens - t < at_once ? tokens - t : at_once);
        q.x = static_cast<const uint16_t *>(x) + t * x_stride, q.out = static_cast<uint16_t *>(out) + t * hidden;
        if (top > 0) q.experts = experts + t * top, q.weights = weights + t * top;
        if (residual != nullptr) q.residual = static_cast<const uint16_t *>(residual) + t * residual_stride;
        unsigned int *counters = static_cast<unsigned int *>(workspace);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const int rc = many                                            ? launch_experts_many(q, counters, scratch, s)
                       : fast && at_once * top <= kExpertsAssignments ? launch_experts_stream(q, counters, scratch, s)
                                                                       : launch_any(q, scratch, s);
        if (rc != B200Q_OK) return rc;
    }
    return B200Q_OK;
}

}  // extern "C"
