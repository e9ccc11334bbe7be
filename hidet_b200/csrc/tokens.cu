// Tokens -> int8 codes with one float scale each, as they are or behind an RMS norm.
//
//     y = x,  or  y = x * w / sqrt(mean(x^2) + eps);   amax = max |y|,  code = rint(y * (127 / amax)),  scale = amax / 127
// in float.  The factor 1 / sqrt(..) is the same for a whole row, so it cancels out of the codes: they are taken from x * w, and the factor
// stands in the scale alone.  So one round of sums and maxima over the row is enough, and the order of the sum never moves a code.
//
// A row is read once into a CTA's registers, as the bytes it has in memory, and widened twice.  What bounds it is memory: 3 bytes an element of 16 bits.
// Rows beyond 32768 elements are read a second time, from L2.
#include "serving.cuh"

namespace b200q {
namespace {

constexpr int MOST_THREADS = 1024;
constexpr uint32_t kLeastAmax = 0x0d800000u;  // 2^-100: 127 / amax is finite from here on
constexpr uint32_t kInfinity = 0x7f800000u;

struct TokensArgs {
    const void *x;
    int64_t x_stride;
    const void *norm;  // of x's type, or null
    float eps;
    int8_t *codes;
    float *scales;
    int width;
    bool vec_in, vec_norm, vec_out;
};

template <typename T>
__device__ __forceinline__ Pack8<T> load_some(const T *p, int left, bool vec) {
    Pack8<T> x;
    if (left >= 8 && vec) return load8<T, true>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = i < left ? p[i] : Elems<T>::round(0.0f);
    return x;
}

template <typename T, bool NORM>
__device__ __forceinline__ void widen(const Pack8<T> &x, const Pack8<T> &w, float (&y)[8], float &squares) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = Elems<T>::one(x.v[i]);
        if (NORM) {
            squares = fmaf(v, v, squares);
            y[i] = v * Elems<T>::one(w.v[i]);
        } else {
            y[i] = v;
        }
    }
}

// VECS: vectors of eight elements that a thread keeps; 0: a row has more, and is read twice.
template <typename T, bool NORM, int VECS>
__global__ void __launch_bounds__(VECS == 0 || VECS == 4 ? MOST_THREADS : 256) quantize_tokens_kernel(const TokensArgs p) {
    __shared__ float warp_squares[MOST_THREADS / 32];
    __shared__ uint32_t warp_amax[MOST_THREADS / 32];
    constexpr int KEPT = VECS > 0 ? VECS : 1;
    const int64_t row = blockIdx.x;
    const int threads = blockDim.x, warps = threads >> 5, lane = threadIdx.x & 31;
    const int vecs = (p.width + 7) >> 3;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride, *w = static_cast<const T *>(p.norm);
    int8_t *codes = p.codes + row * p.width;
    pdl_launch_dependents();
    pdl_wait();
    Pack8<T> kept[KEPT];
    float squares = 0.0f;
    uint32_t amax = 0;
    // not kept: the second time they come from L1
    auto weights_at = [&](int at) { return NORM ? load_some(w + at, p.width - at, p.vec_norm) : Pack8<T>(); };
    auto look = [&](const Pack8<T> &v, const Pack8<T> &u) {
        float y[8];
        widen<T, NORM>(v, u, y, squares);
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(y[i]) & 0x7fffffffu);  // a NaN is larger than all numbers
    };
    if (VECS > 0) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) {
            const int at = ((int)threadIdx.x + i * threads) * 8, left = p.width - at;
            kept[i] = load_some(x + at, left, p.vec_in);
        }
#pragma unroll
        for (int i = 0; i < KEPT; ++i) look(kept[i], weights_at(((int)threadIdx.x + i * threads) * 8));
    } else {
        for (int v = threadIdx.x; v < vecs; v += threads) {
            kept[0] = load_some(x + v * 8, p.width - v * 8, p.vec_in);
            look(kept[0], weights_at(v * 8));
        }
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if (NORM) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
    }
    if (warps > 1) {
        if (lane == 0) {
            warp_amax[threadIdx.x >> 5] = amax;
            if (NORM) warp_squares[threadIdx.x >> 5] = squares;
        }
        __syncthreads();
        amax = __reduce_max_sync(0xffffffffu, lane < warps ? warp_amax[lane] : 0u);
        if (NORM) {
            squares = lane < warps ? warp_squares[lane] : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
        }
    }
    const bool zeros = amax < kLeastAmax || amax >= kInfinity;
    const float top = __uint_as_float(amax), by = zeros ? 0.0f : __fdiv_rn(127.0f, top);
    if (threadIdx.x == 0) {
        float scale = __fdiv_rn(amax < kLeastAmax ? 0.0f : top, 127.0f);
        if (NORM) {
            const float mean = __fdiv_rn(squares, (float)p.width) + p.eps;
            scale = amax < kLeastAmax ? 0.0f : __fdiv_rn(__fdiv_rn(top, __fsqrt_rn(mean)), 127.0f);
            if (!(mean < INFINITY)) scale = __uint_as_float(0x7fc00000u);  // squares beyond float
        }
        if (amax >= kInfinity) scale = __uint_as_float(0x7fc00000u);
        p.scales[row] = scale;
    }
    auto put = [&](const Pack8<T> &v, const Pack8<T> &u, int at) {
        float y[8], unused = 0.0f;
        widen<T, NORM>(v, u, y, unused);
        uint32_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = zeros ? 0u : (uint32_t)__float2int_rn(y[i] * by);
        const int left = p.width - at;
        if (left >= 8 && p.vec_out) {
            uint2 q;
            q.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
            q.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
            *reinterpret_cast<uint2 *>(codes + at) = q;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) codes[at + i] = (int8_t)c[i];
        }
    };
    if (VECS > 0) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) put(kept[i], weights_at(((int)threadIdx.x + i * threads) * 8), ((int)threadIdx.x + i * threads) * 8);
    } else {
        for (int v = threadIdx.x; v < vecs; v += threads) {
            kept[0] = load_some(x + v * 8, p.width - v * 8, p.vec_in);
            put(kept[0], weights_at(v * 8), v * 8);
        }
    }
}

template <typename T, bool NORM>
int launch_typed(const TokensArgs &p, int64_t rows, cudaStream_t stream) {
    const int vecs = p.width > 0 ? (p.width + 7) / 8 : 1;
    const dim3 grid((unsigned)rows);
    auto threads = [&](int each) { return (int)round_up(ceil_div(vecs, each), 32); };
    const char *name = "quantize_tokens_kernel";
    if (threads(1) <= 256) return launch_after(name, quantize_tokens_kernel<T, NORM, 1>, grid, threads(1), 0, 1, stream, p);
    if (threads(2) <= 256) return launch_after(name, quantize_tokens_kernel<T, NORM, 2>, grid, threads(2), 0, 1, stream, p);
    if (threads(4) <= MOST_THREADS) return launch_after(name, quantize_tokens_kernel<T, NORM, 4>, grid, threads(4), 0, 1, stream, p);
    return launch_after(name, quantize_tokens_kernel<T, NORM, 0>, grid, MOST_THREADS, 0, 1, stream, p);
}

}  // namespace
}  // namespace b200q

extern "C" {

B200Q_API int b200q_quantize_tokens(const void *x, int64_t x_stride, const void *norm, float eps, void *codes, float *scales, int64_t rows, int64_t width, int type,
                                    void *stream) {
    using namespace b200q;
    const char *op = "quantize_tokens";
    if (rows < 0 || width < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative size", op);
    if (type < B200Q_F16 || type > B200Q_F32) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown float type %d", op, type);
    if (!(eps >= 0.0f && eps < INFINITY)) return set_error(B200Q_INVALID_ARGUMENT, "%s: eps must be a number of at least 0, got %g", op, (double)eps);
    if (rows == 0) return B200Q_OK;
    if (width > 0x7fffff00LL || rows > 2147483647LL) return set_error(B200Q_UNSUPPORTED, "%s: %lld rows of %lld elements", op, (long long)rows, (long long)width);
    if (scales == nullptr || (width > 0 && (x == nullptr || codes == nullptr))) return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    if (x_stride < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative stride", op);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t size = type == B200Q_F32 ? 4 : 2;
    TokensArgs p = {x, x_stride, width > 0 ? norm : nullptr, eps, static_cast<int8_t *>(codes), scales, (int)width,
                    aligned_to(x, 16) && (rows == 1 || x_stride * size % 16 == 0), aligned_to(norm, 16), aligned_to(codes, 8) && (rows == 1 || width % 8 == 0)};
    switch (type) {
        case B200Q_F16: return p.norm ? launch_typed<__half, true>(p, rows, s) : launch_typed<__half, false>(p, rows, s);
        case B200Q_BF16: return p.norm ? launch_typed<__nv_bfloat16, true>(p, rows, s) : launch_typed<__nv_bfloat16, false>(p, rows, s);
        default: return p.norm ? launch_typed<float, true>(p, rows, s) : launch_typed<float, false>(p, rows, s);
    }
}

}  // extern "C"
