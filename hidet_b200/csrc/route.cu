// The router of a layer of experts: which experts a token goes to, and with which weights.
//
//     l[e] = sum_h x[h] r[e, h];   the `top` largest l, equal ones by index;   weight_j = exp(l_j - m) / sum exp(l - m)
// over the chosen ones or over all, m the largest.  In float.
//
// A cluster of up to eight CTAs has eight tokens (four, in float or where rows are no whole vectors) and shares the experts; a row of the router is read once for them.  Tokens and router of one
// 16-bit type are multiplied by tensor instructions, whose products are exact and whose sums are float; others by float ones.  All logits meet in the first CTA's shared
// memory, where a warp a token puts them in order, every lane with its experts' keys in registers.  A decode step's router is some KB to MB in L2: what takes the time is
// latency (launch, a row, the cluster's barrier, the choices one after the other), so loads are asked for eight at a time.  One token, 8 experts, rows of 4096:
// 3.3 us; 7 tokens, 64 of 2048: 3.4; 48 tokens, 128 of 2048: 4.0; 64 tokens, 256 of 7168: 12.5; 512 tokens, 64 of 2048: 7.1.  With a float router, or float tokens, on float instructions: 2.7, 5.9, 10.3,
// 61 and 20 to 22.  With more tokens than a cluster has the router is read again by every cluster, which is what the last two are.
#include "serving.cuh"

namespace b200q {
namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS, MOST_CLUSTER = 8;
constexpr int MOST_EXPERTS = 1024, MOST_TOKENS = 4, MOST_TOP = 32;
constexpr int TOKENS_AT_ONCE = WARPS, STEPS = 8;  // of the kernel on tensor instructions: tokens of a cluster, 32 k each

struct RouteArgs {
    const void *x, *router;
    int64_t x_stride;
    int32_t *experts;
    float *weights;
    int tokens, width, count, top, cluster;
    bool all;           // weights over all experts
};

__device__ __forceinline__ uint32_t ordered(float v) {  // NaN is the largest, -0 is 0
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

template <bool VEC, typename T>
__device__ __forceinline__ void load_some(const T *p, int left, float (&f)[8]) {
    if (VEC) {
        const Pack8<T> x = load8<T, true>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = Elems<T>::one(x.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < left ? Elems<T>::one(p[i]) : 0.0f;
    }
}

// The `top` largest of a token's logits, by a warp; lane l has experts l, l + 32, .. and their keys, zero for none and for the ones that are taken.
template <int EACH>
__device__ __forceinline__ void choose(const RouteArgs &p, const float *l, int64_t row, int lane) {
    uint32_t key[EACH];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int e = lane + 32 * i;
        const float v = e < p.count ? l[e] : 0.0f;
        bad |= v != v;
        key[i] = e < p.count ? ordered(v) : 0u;
    }
    int mine = -1;  // lane j: the j-th choice
    for (int j = 0; j < p.top; ++j) {
        uint32_t best = 0, place = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (key[i] > best) best = key[i], place = lane + 32 * i;
        const uint32_t top = __reduce_max_sync(0xffffffffu, best), e = __reduce_min_sync(0xffffffffu, best == top ? place : 0x7fffffffu);
        if (lane == j) mine = (int)e;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (lane + 32 * i == (int)e) key[i] = 0;
    }
    const float v = mine >= 0 ? l[mine] : 0.0f, m = __shfl_sync(0xffffffffu, v, 0);
    const float share = mine >= 0 ? expf(v - m) : 0.0f;
    float total = share;
    if (p.all) {
        total = 0.0f;
        for (int e = lane; e < p.count; e += 32) total += expf(l[e] - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    // a logit that is no number makes its token's weights none, also where it was not chosen
    if (__any_sync(0xffffffffu, bad)) total = __uint_as_float(0x7fc00000u);
    if (mine >= 0) {
        p.experts[row + lane] = mine;
        p.weights[row + lane] = __fdiv_rn(share, total);
    }
}

// VEC: rows of tokens and router are whole vectors of eight elements on 16-byte boundaries.
template <typename T, typename R, bool VEC>
__global__ void __launch_bounds__(THREADS) route_kernel(const RouteArgs p) {
    __shared__ float logits[MOST_TOKENS][MOST_EXPERTS];  // of the cluster's first CTA: all experts
    __shared__ float parts[WARPS][2][MOST_TOKENS];
    const uint32_t rank = cluster_ctarank();
    const int first = (int)(blockIdx.x / p.cluster) * MOST_TOKENS, tokens = min(MOST_TOKENS, p.tokens - first);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t logits0 = p.cluster > 1 ? map_to_rank(smem_u32(&logits[0][0]), 0) : 0u;
    // two experts a warp, or a share of their rows where the CTA has fewer than its warps can take
    const int pairs = (p.count + 2 * p.cluster - 1) / (2 * p.cluster), share = pairs > 4 ? 1 : pairs > 2 ? 2 : pairs > 1 ? 4 : 8, part = warp % share;
    pdl_launch_dependents();
    cluster_arrive_release();  // this CTA is there
    pdl_wait();
    bool met = false;
    for (int pair = 0; pair < pairs; pair += WARPS / share) {
        const int e0 = 2 * ((pair + warp / share) * p.cluster + (int)rank);
        const bool some = pair + warp / share < pairs && e0 < p.count, two = e0 + 1 < p.count;
        float sum[2][MOST_TOKENS] = {};
        if (some) {
            const R *r = static_cast<const R *>(p.router) + (int64_t)e0 * p.width;
            const T *x = static_cast<const T *>(p.x) + first * p.x_stride;
#pragma unroll 4
            for (int at = (part * 32 + lane) * 8; at < p.width; at += share * 256) {
                float w[2][8];
                load_some<VEC>(r + at, p.width - at, w[0]);
                load_some<VEC>(r + (two ? p.width : 0) + at, p.width - at, w[1]);
#pragma unroll
                for (int t = 0; t < MOST_TOKENS; ++t) {
                    if (t < tokens) {
                        float v[8];
                        load_some<VEC>(x + t * p.x_stride + at, p.width - at, v);
#pragma unroll
                        for (int j = 0; j < 8; ++j) sum[0][t] = fmaf(v[j], w[0][j], sum[0][t]), sum[1][t] = fmaf(v[j], w[1][j], sum[1][t]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int t = 0; t < MOST_TOKENS; ++t)
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) sum[i][t] += __shfl_xor_sync(0xffffffffu, sum[i][t], o);
        }
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int t = 0; t < MOST_TOKENS; ++t) parts[warp][i][t] = sum[i][t];
        }
        __syncthreads();
        if (!met) cluster_wait_acquire();  // the first CTA is there
        met = true;
        const int i = lane >> 2, t = lane & 3;
        if (some && part == 0 && lane < 8 && e0 + i < p.count && t < tokens) {
            float l = 0.0f;
            for (int s = 0; s < share; ++s) l += parts[warp + s][i][t];
            if (p.cluster > 1) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(logits0 + (uint32_t)(t * MOST_EXPERTS + e0 + i) * 4), "f"(l) : "memory");
            else logits[t][e0 + i] = l;
        }
        __syncthreads();
    }
    cluster_arrive_release();
    cluster_wait_acquire();
    if (rank != 0 || warp >= tokens) return;
    const int64_t row = (int64_t)(first + warp) * p.top;
    if (p.count <= 32) choose<1>(p, logits[warp], row, lane);
    else if (p.count <= 128) choose<4>(p, logits[warp], row, lane);
    else choose<MOST_EXPERTS / 32>(p, logits[warp], row, lane);
}

// D[16 x 8] += A[16 x 16] * B[16 x 8], experts by tokens.
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    mma_m16n8k16(d, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Tokens and router of one 16-bit type, in whole vectors.  A warp has 16 experts and a share of their rows; a lane's eight neighbouring k of a row, which one load brings, are the same eight of its
// token's, so two instructions take 32 k of 16 experts and eight tokens from three loads, eight steps of which are under way.  The instructions cut their sums where float would round them, always
// towards zero: eight of them in a row, and
// their sums are added as floats (with all of a warp's in a row weights of 1024 tokens, 256 experts of 7168, were 2.0e-6 off, root mean square, 2.5e-7 now).
template <typename T>
__global__ void __launch_bounds__(THREADS, 1) route_mma_kernel(const RouteArgs p) {
    __shared__ float logits[TOKENS_AT_ONCE][MOST_EXPERTS];  // of the cluster's first CTA
    __shared__ float parts[WARPS][16][TOKENS_AT_ONCE];
    const uint32_t rank = cluster_ctarank();
    const int first = (int)(blockIdx.x / p.cluster) * TOKENS_AT_ONCE, tokens = min(TOKENS_AT_ONCE, p.tokens - first);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t logits0 = p.cluster > 1 ? map_to_rank(smem_u32(&logits[0][0]), 0) : 0u;
    const int groups = (p.count + 16 * p.cluster - 1) / (16 * p.cluster), share = groups > 4 ? 1 : groups > 2 ? 2 : groups > 1 ? 4 : 8, part = warp % share;
    pdl_launch_dependents();
    cluster_arrive_release();  // this CTA is there
    pdl_wait();
    bool met = false;
    const T *x = static_cast<const T *>(p.x) + (int64_t)(first + min(g, tokens - 1)) * p.x_stride;
    for (int group = 0; group < groups; group += WARPS / share) {
        const int e0 = 16 * ((group + warp / share) * p.cluster + (int)rank);
        const bool some = group + warp / share < groups && e0 < p.count;
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (some) {
            const T *r0 = static_cast<const T *>(p.router) + (int64_t)min(e0 + g, p.count - 1) * p.width, *r1 = static_cast<const T *>(p.router) + (int64_t)min(e0 + 8 + g, p.count - 1) * p.width;
            for (int k0 = part * 32 * STEPS; k0 < p.width; k0 += share * 32 * STEPS) {
                uint4 a0[STEPS], a1[STEPS], b[STEPS];
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const int k = k0 + 32 * i + 8 * t;
                    a0[i] = a1[i] = b[i] = make_uint4(0, 0, 0, 0);
                    if (k < p.width) {
                        a0[i] = *reinterpret_cast<const uint4 *>(r0 + k), a1[i] = *reinterpret_cast<const uint4 *>(r1 + k);
                        b[i] = *reinterpret_cast<const uint4 *>(x + k);
                    }
                }
                float s[2][4] = {};
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    mma<T>(s[0], a0[i].x, a1[i].x, a0[i].y, a1[i].y, b[i].x, b[i].y);
                    mma<T>(s[1], a0[i].z, a1[i].z, a0[i].w, a1[i].w, b[i].z, b[i].w);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] += s[0][i] + s[1][i];
            }
        }
        // d: experts g and g + 8, tokens 2 t and 2 t + 1
        parts[warp][g][2 * t] = d[0], parts[warp][g][2 * t + 1] = d[1], parts[warp][g + 8][2 * t] = d[2], parts[warp][g + 8][2 * t + 1] = d[3];
        __syncthreads();
        if (!met) cluster_wait_acquire();  // the first CTA is there
        met = true;
        for (int i = threadIdx.x; i < WARPS / share * 16 * TOKENS_AT_ONCE; i += THREADS) {
            const int of = i / (16 * TOKENS_AT_ONCE), e = i / TOKENS_AT_ONCE % 16, token = i % TOKENS_AT_ONCE, expert = 16 * ((group + of) * p.cluster + (int)rank) + e;
            if (group + of >= groups || expert >= p.count || token >= tokens) continue;
            float l = 0.0f;
            for (int s = 0; s < share; ++s) l += parts[of * share + s][e][token];
            if (p.cluster > 1) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(logits0 + (uint32_t)(token * MOST_EXPERTS + expert) * 4), "f"(l) : "memory");
            else logits[token][expert] = l;
        }
        __syncthreads();
    }
    cluster_arrive_release();
    cluster_wait_acquire();
    if (rank != 0 || warp >= tokens) return;
    const int64_t row = (int64_t)(first + warp) * p.top;
    if (p.count <= 32) choose<1>(p, logits[warp], row, lane);
    else if (p.count <= 128) choose<4>(p, logits[warp], row, lane);
    else choose<MOST_EXPERTS / 32>(p, logits[warp], row, lane);
}

template <typename T, typename R>
int launch_typed(const RouteArgs &p, bool vec, cudaStream_t stream) {
    const dim3 grid((unsigned)(ceil_div(p.tokens, MOST_TOKENS) * p.cluster));
    return vec ? launch_after("route_kernel", route_kernel<T, R, true>, grid, THREADS, 0, p.cluster, stream, p)
               : launch_after("route_kernel", route_kernel<T, R, false>, grid, THREADS, 0, p.cluster, stream, p);
}
template <typename T>
int launch_mma(RouteArgs p, cudaStream_t stream) {
    p.cluster = 1;
    while (p.cluster < MOST_CLUSTER && 16 * p.cluster < p.count) p.cluster *= 2;
    return launch_after("route_mma_kernel", route_mma_kernel<T>, dim3((unsigned)(ceil_div(p.tokens, TOKENS_AT_ONCE) * p.cluster)), THREADS, 0, p.cluster, stream, p);
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
    int cluster = 1;
    while (cluster < MOST_CLUSTER && 2 * cluster < count) cluster *= 2;
    const RouteArgs p = {x, router, x_stride, experts, weights, (int)tokens, (int)width, (int)count, (int)top, cluster, over_all != 0};
    const bool vec = width % 8 == 0 && aligned_to(x, 16) && (tokens == 1 || x_stride * size % 16 == 0) && aligned_to(router, 16) && width * router_size % 16 == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (vec && type == router_type && type == B200Q_F16) return launch_mma<__half>(p, s);
    if (vec && type == router_type && type == B200Q_BF16) return launch_mma<__nv_bfloat16>(p, s);
    if (type == B200Q_F32) return launch_typed<float, float>(p, vec, s);
    if (type == B200Q_F16) return router_type == B200Q_F32 ? launch_typed<__half, float>(p, vec, s) : launch_typed<__half, __half>(p, vec, s);
    return router_type == B200Q_F32 ? launch_typed<__nv_bfloat16, float>(p, vec, s) : launch_typed<__nv_bfloat16, __nv_bfloat16>(p, vec, s);
}

}  // extern "C"
