// The router of a layer of experts: which experts a token goes to, and with which weights.
//
//     l[e] = sum_h x[h] r[e, h];   the `top` largest l, equal ones by index;   weight_j = exp(l_j - m) / sum exp(l - m)
// over the chosen ones or over all, m the largest.  In float.
//
// A cluster of eight CTAs has up to four tokens; each CTA has every eighth expert, and a warp an expert (or, where there are fewer experts than
// warps, a part of one's row).  So a row of the router is read once for four tokens and all of a cluster's logits meet in the first CTA's
// shared memory, where a warp a token puts them in order.  A decode step's router is some KB to MB in L2: what takes the time is
// latency (launch, a row, the cluster's barrier, the choices one after the other).
#include "serving.cuh"

namespace b200q {
namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS, CLUSTER = 8;
constexpr int MOST_EXPERTS = 1024, MOST_TOKENS = 4, MOST_TOP = 32;

struct RouteArgs {
    const void *x, *router;
    int64_t x_stride;
    int32_t *experts;
    float *weights;
    int tokens, width, count, top;
    bool all;           // weights over all experts
    bool vec_x, vec_r;
};

__device__ __forceinline__ uint32_t ordered(float v) {  // NaN is the largest, -0 is 0
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

template <typename T>
__device__ __forceinline__ void load_some(const T *p, int left, bool vec, float (&f)[8]) {
    if (left >= 8 && vec) {
        const Pack8<T> x = load8<T, true>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = Elems<T>::one(x.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < left ? Elems<T>::one(p[i]) : 0.0f;
    }
}

template <typename T, typename R>
__global__ void __launch_bounds__(THREADS) route_kernel(const RouteArgs p) {
    __shared__ float parts[WARPS][MOST_TOKENS];
    __shared__ float logits[MOST_TOKENS][MOST_EXPERTS];  // of the cluster's first CTA: all experts
    const uint32_t rank = cluster_ctarank();
    const int first = (int)(blockIdx.x / CLUSTER) * MOST_TOKENS, tokens = min(MOST_TOKENS, p.tokens - first);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int mine = (p.count - (int)rank + CLUSTER - 1) / CLUSTER;  // experts of this CTA
    // warps that share a row: as many as leave none idle
    const int share = mine > 4 ? 1 : mine > 2 ? 2 : mine > 1 ? 4 : 8;
    const uint32_t logits0 = map_to_rank(smem_u32(&logits[0][0]), 0);
    pdl_launch_dependents();
    pdl_wait();
    cluster_arrive_release();
    cluster_wait_acquire();  // the first CTA is there
    const int at_once = WARPS / share, part = warp % share;
    for (int i0 = 0; i0 < mine; i0 += at_once) {
        const int i = i0 + warp / share, e = (int)rank + CLUSTER * i;
        float sum[MOST_TOKENS] = {};
        if (i < mine) {
            const R *r = static_cast<const R *>(p.router) + (int64_t)e * p.width;
            const T *x = static_cast<const T *>(p.x) + first * p.x_stride;
#pragma unroll 2
            for (int at = (part * 32 + lane) * 8; at < p.width; at += share * 256) {
                const int left = p.width - at;
                float w[8];
                load_some(r + at, left, p.vec_r, w);
#pragma unroll
                for (int t = 0; t < MOST_TOKENS; ++t) {
                    if (t < tokens) {
                        float v[8];
                        load_some(x + t * p.x_stride + at, left, p.vec_x, v);
#pragma unroll
                        for (int j = 0; j < 8; ++j) sum[t] = fmaf(v[j], w[j], sum[t]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < MOST_TOKENS; ++t)
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum[t] += __shfl_xor_sync(0xffffffffu, sum[t], o);
        }
        if (share > 1) {
            if (lane == 0) {
#pragma unroll
                for (int t = 0; t < MOST_TOKENS; ++t) parts[warp][t] = sum[t];
            }
            __syncthreads();
            if (part == 0) {
#pragma unroll
                for (int t = 0; t < MOST_TOKENS; ++t)
                    for (int s = 1; s < share; ++s) sum[t] += parts[warp + s][t];
            }
            __syncthreads();
        }
        if (i < mine && part == 0 && lane == 0) {
#pragma unroll
            for (int t = 0; t < MOST_TOKENS; ++t)
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(logits0 + (uint32_t)(t * MOST_EXPERTS + e) * 4), "f"(sum[t]) : "memory");
        }
    }
    cluster_arrive_release();
    cluster_wait_acquire();
    if (rank != 0 || warp >= tokens) return;
    // ---- a warp a token; lane l has experts l, l + 32, ..: its best of those not yet taken, and the warp's ----
    float *l = logits[warp];
    const int64_t row = (int64_t)(first + warp) * p.top;
    auto best_of_mine = [&](uint32_t &key, int &place) {
        key = 0, place = 0x7fffffff;
        for (int e = lane; e < p.count; e += 32) {
            const uint32_t k = ordered(l[e]);
            if (k > key || place == 0x7fffffff) key = k, place = e;
        }
    };
    uint32_t key, taken = 0;  // taken: bit i of lane's i-th expert
    int place;
    best_of_mine(key, place);
    const bool any = place != 0x7fffffff;
    bool left = any;
    float m = 0.0f, total = 0.0f, chosen = 0.0f;
    for (int j = 0; j < p.top; ++j) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, left ? key : 0u);
        const int e = (int)__reduce_min_sync(0xffffffffu, left && key == top ? (uint32_t)place : 0x7fffffffu);
        const float v = l[e];
        if (j == 0) m = v;
        const float w = expf(v - m);
        total += w;
        if (lane == j) chosen = w;
        if (lane == 0) p.experts[row + j] = e;
        if ((e & 31) == lane) {
            taken |= 1u << (e >> 5);
            left = false;
            for (int i = 0, o = lane; o < p.count; ++i, o += 32) {
                if (taken >> i & 1u) continue;
                const uint32_t k = ordered(l[o]);
                if (!left || k > key) key = k, place = o, left = true;
            }
        }
        __syncwarp();
    }
    if (p.all) {
        total = 0.0f;
        for (int e = lane; e < p.count; e += 32) total += expf(l[e] - m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    } else {
        // a logit that is no number makes its token's weights none, also where it was not chosen
        bool bad = false;
        for (int e = lane; e < p.count; e += 32) bad |= l[e] != l[e];
        if (__any_sync(0xffffffffu, bad)) total = __uint_as_float(0x7fc00000u);
    }
    if (lane < p.top) p.weights[row + lane] = __fdiv_rn(chosen, total);
}

}  // namespace
}  // namespace b200q

extern "C" {

B200Q_API int b200q_route_tokens(const void *x, int64_t x_stride, const void *router, int32_t *experts, float *weights, int64_t tokens, int64_t width, int64_t count,
                                 int64_t top, int over_all, int type, int router_type, void *stream) {
    using namespace b200q;
    const char *op = "route_tokens";
    if (tokens < 0 || width < 0 || count < 0 || top < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative size", op);
    if (type < B200Q_F16 || type > B200Q_F32) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown float type %d", op, type);
    if (router_type != type && router_type != B200Q_F32) return set_error(B200Q_INVALID_ARGUMENT, "%s: the router is of the tokens' type or f32, not type %d", op, router_type);
    if (count > MOST_EXPERTS) return set_error(B200Q_UNSUPPORTED, "%s: %lld experts: up to %d are supported", op, (long long)count, MOST_EXPERTS);
    if (top < 1 || top > count) return set_error(B200Q_INVALID_ARGUMENT, "%s: %lld of %lld experts", op, (long long)top, (long long)count);
    if (top > MOST_TOP) return set_error(B200Q_UNSUPPORTED, "%s: %lld experts a token: up to %d are supported", op, (long long)top, MOST_TOP);
    if (x_stride < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative stride", op);
    if (tokens == 0) return B200Q_OK;
    if (experts == nullptr || weights == nullptr || (width > 0 && (x == nullptr || router == nullptr))) return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    if (tokens > 0x3fffffffLL || width > 0x3fffffffLL) return set_error(B200Q_UNSUPPORTED, "%s: %lld tokens of %lld elements", op, (long long)tokens, (long long)width);
    const int64_t size = type == B200Q_F32 ? 4 : 2, router_size = router_type == B200Q_F32 ? 4 : 2;
    const RouteArgs p = {x, router, x_stride, experts, weights, (int)tokens, (int)width, (int)count, (int)top, over_all != 0,
                         aligned_to(x, 16) && (tokens == 1 || x_stride * size % 16 == 0), aligned_to(router, 16) && (count == 1 || width * router_size % 16 == 0)};
    const dim3 grid((unsigned)(ceil_div(tokens, MOST_TOKENS) * CLUSTER));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const char *name = "route_kernel";
    if (type == B200Q_F32) return launch_after(name, route_kernel<float, float>, grid, THREADS, 0, CLUSTER, s, p);
    if (type == B200Q_F16) {
        return router_type == B200Q_F32 ? launch_after(name, route_kernel<__half, float>, grid, THREADS, 0, CLUSTER, s, p)
                                        : launch_after(name, route_kernel<__half, __half>, grid, THREADS, 0, CLUSTER, s, p);
    }
    return router_type == B200Q_F32 ? launch_after(name, route_kernel<__nv_bfloat16, float>, grid, THREADS, 0, CLUSTER, s, p)
                                    : launch_after(name, route_kernel<__nv_bfloat16, __nv_bfloat16>, grid, THREADS, 0, CLUSTER, s, p);
}

}  // extern "C"
