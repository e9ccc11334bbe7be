// Tokens -> int8 codes with one float scale each, as they are or behind an RMS norm.
//
//     y = x,  or  y = x * w / sqrt(mean(x^2) + eps);   amax = max |y|,  code = rint(y * (127 / amax)),  scale = amax / 127
// in float, each operation rounded: where amax is 127 times a small number, products lie in the middle between whole numbers by the dozen, and only the rounded
// product says so.  The factor 1 / sqrt(..) is the same for a whole row, so it cancels out of the codes: they are taken from x * w, and the factor stands in the scale
// alone.  So one round of sums and maxima over the row is enough, and the order of the sum never moves a code.
//
// A row is read once into registers, of a CTA or (up to 1024 elements) of a warp, as the bytes it has in memory, and widened twice.  Its floor is memory, 3 bytes an element
// of 16 bits; close behind stand the instructions, some 4 an element: maxima are taken of 16-bit pairs, and an addition of 1.5 * 2^23
// rounds to a whole number that then stands in the sum's lowest byte.  Rows beyond 16384 elements are read a second time, from L2.
#include "serving.cuh"

namespace b200q {
namespace {

constexpr int MOST_THREADS = 1024;
constexpr int64_t kMostWidth = 0x7fffffffLL - 8 * MOST_THREADS;  // the step behind a row's last element is an int too
constexpr uint32_t kLeastAmax = 0x0d800000u;  // 2^-100: 127 / amax is finite from here on
constexpr uint32_t kInfinity = 0x7f800000u;
constexpr int ROWS_OF_WARPS = 8;              // rows of a CTA whose warps have one each

struct TokensArgs {
    const void *x;
    int64_t x_stride;
    const void *norm;  // of x's type, or null
    float eps;
    int8_t *codes;
    float *scales;
    int64_t rows;
    int width;
    bool vec_in, vec_norm, vec_out;
};

// Eight elements, zeros behind the last of a row.  Both ways give whole words: where the one by one gave single elements of 16 bits, the other's vector was taken apart to meet
// them (8192 rows of 8192 bf16: 52 us for 32).
template <typename T>
__device__ __forceinline__ Pack8<T> load_some(const T *p, int left, bool vec) {
    union {
        Pack8<T> x;
        uint32_t w[2 * sizeof(T)];
    } u;
    if (left >= 8 && vec) {
        u.x = load8<T, true>(p);
    } else if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) u.w[i % (2 * sizeof(T))] = i < left ? reinterpret_cast<const uint32_t *>(p)[i] : 0u;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = 2 * i < left ? reinterpret_cast<const uint16_t *>(p)[2 * i] : 0u, hi = 2 * i + 1 < left ? reinterpret_cast<const uint16_t *>(p)[2 * i + 1] : 0u;
            u.w[i] = lo | hi << 16;
        }
    }
    return u.x;
}

// The largest magnitude of elements as they are: a running maximum (a NaN stays), and its bits as float's.
__device__ __forceinline__ float max3_abs(float m, float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}
template <typename T>
struct Amax;
template <>
struct Amax<float> {
    float m = 0.0f;
    __device__ __forceinline__ void look(const Pack8<float> &x) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) m = max3_abs(m, x.v[i], x.v[i + 1]);
    }
    __device__ __forceinline__ uint32_t bits() const { return __float_as_uint(m) & 0x7fffffffu; }
};
template <>
struct Amax<__half> {
    __half2 m = __half2half2(__ushort_as_half(0));
    __device__ __forceinline__ void look(const Pack8<__half> &x) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2 *>(&x.v[i])));
    }
    __device__ __forceinline__ uint32_t bits() const { return max(__float_as_uint(__low2float(m)) & 0x7fffffffu, __float_as_uint(__high2float(m)) & 0x7fffffffu); }
};
template <>
struct Amax<__nv_bfloat16> {
    __nv_bfloat162 m = __nv_bfloat162(__ushort_as_bfloat16(0), __ushort_as_bfloat16(0));
    __device__ __forceinline__ void look(const Pack8<__nv_bfloat16> &x) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&x.v[i])));
    }
    __device__ __forceinline__ uint32_t bits() const { return max(__float_as_uint(__low2float(m)) & 0x7fffffffu, __float_as_uint(__high2float(m)) & 0x7fffffffu); }
};

// A row's scale where the mean of its squares and eps is below 2^-100: float's squares lose what is below 2^-75 of such a row.  By one thread, at its end: rows like these come with an
// eps of (next to) nothing only.  That there is such a branch costs 0.7 of 40 us (8192 rows of 8192).
constexpr float kLeastMean = 0x1p-100f;
template <typename T>
__device__ __noinline__ float tiny_scale(const T *x, int width, float eps, float top) {
    double sum = 0.0;
    for (int i = 0; i < width; ++i) {
        const double v = (double)Elems<T>::one(x[i]);
        sum = fma(v, v, sum);
    }
    return (float)((double)top / (sqrt(sum / (double)width + (double)eps) * 127.0));
}

// VECS: vectors of eight elements that a thread keeps; 0: a row has more, and is read twice.  ONE_WARP: a warp has a row of its own.
template <typename T, bool NORM, int VECS, bool ONE_WARP>
__global__ void __launch_bounds__(VECS == 0 ? MOST_THREADS : VECS == 4 ? 512 : 256) quantize_tokens_kernel(const TokensArgs p) {
    __shared__ float warp_squares[MOST_THREADS / 32];
    __shared__ uint32_t warp_amax[MOST_THREADS / 32];
    constexpr int KEPT = VECS > 0 ? VECS : 1;
    const int lane = threadIdx.x & 31;
    const int64_t row = ONE_WARP ? (int64_t)blockIdx.x * ROWS_OF_WARPS + (threadIdx.x >> 5) : blockIdx.x;
    const int threads = ONE_WARP ? 32 : blockDim.x, me = ONE_WARP ? lane : threadIdx.x, warps = threads >> 5;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride, *w = static_cast<const T *>(p.norm);
    int8_t *codes = p.codes + row * p.width;
    pdl_launch_dependents();
    pdl_wait();
    if (ONE_WARP && row >= p.rows) return;
    Pack8<T> kept[KEPT];       // of x,
    f32x2 products[KEPT][4];   // or x * w
    f32x2 squares = pair_of(0.0f, 0.0f);
    Amax<T> plain;    // of x
    float normed = 0.0f;  // of x * w
    auto product = [&](const Pack8<T> &v, int at, f32x2 (&y)[4], bool look) {
        Pairs<T>::widen(v, y);
        if (NORM) {
            f32x2 u[4];
            Pairs<T>::widen(load_some(w + at, p.width - at, p.vec_norm), u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (look) squares = fma2(y[i], y[i], squares);
                y[i] = mul2(y[i], u[i]);
            }
        }
    };
    auto look = [&](const Pack8<T> &v, int at, f32x2 (&y)[4]) {
        if (NORM) {
            product(v, at, y, true);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float lo, hi;
                halves(y[i], lo, hi);
                normed = max3_abs(normed, lo, hi);
            }
        } else {
            plain.look(v);
        }
    };
    if (VECS > 0) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) {
            const int at = (me + i * threads) * 8;
            kept[i] = load_some(x + at, p.width - at, p.vec_in);
        }
#pragma unroll
        for (int i = 0; i < KEPT; ++i) look(kept[i], (me + i * threads) * 8, products[i]);
    } else {
        for (int at = me * 8; at < p.width; at += threads * 8) look(load_some(x + at, p.width - at, p.vec_in), at, products[0]);
    }
    uint32_t amax = __reduce_max_sync(0xffffffffu, NORM ? __float_as_uint(normed) & 0x7fffffffu : plain.bits());  // the bits of a NaN are larger than all numbers'
    float sum = 0.0f;
    if (NORM) {
        float hi;
        halves(squares, sum, hi);
        sum += hi;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (!ONE_WARP && warps > 1) {
        if (lane == 0) {
            warp_amax[threadIdx.x >> 5] = amax;
            if (NORM) warp_squares[threadIdx.x >> 5] = sum;
        }
        __syncthreads();
        amax = __reduce_max_sync(0xffffffffu, lane < warps ? warp_amax[lane] : 0u);
        if (NORM) {
            sum = lane < warps ? warp_squares[lane] : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
    }
    const bool small = amax < kLeastAmax, bad = amax >= kInfinity;
    const float top = __uint_as_float(amax), by = small || bad ? 0.0f : __fdiv_rn(127.0f, top);
    const uint32_t keep = small || bad ? 0u : 0xffffffffu;
    bool tiny = false;
    if (me == 0) {
        float scale = small ? 0.0f : __fdiv_rn(top, 127.0f);
        if (NORM) {
            const float mean = __fdiv_rn(sum, (float)p.width) + p.eps;
            tiny = mean < kLeastMean && !small;
            scale = small ? 0.0f : __fdiv_rn(__fdiv_rn(top, __fsqrt_rn(mean)), 127.0f);
            if (!(mean < INFINITY)) scale = __uint_as_float(0x7fc00000u);  // squares beyond float
        }
        if (bad) scale = __uint_as_float(0x7fc00000u);
        p.scales[row] = scale;
    }
    const f32x2 by2 = pair_of(by, by);
    auto put = [&](const f32x2 (&y)[4], int at) {
        uint32_t c[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo, hi;
            halves(mul2(y[i], by2), lo, hi);
            c[2 * i] = __float_as_uint(__fadd_rn(lo, 12582912.0f)), c[2 * i + 1] = __float_as_uint(__fadd_rn(hi, 12582912.0f));
        }
        uint2 q;
        q.x = keep & __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        q.y = keep & __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
        const int left = p.width - at;
        if (left >= 8 && p.vec_out) {
            *reinterpret_cast<uint2 *>(codes + at) = q;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) codes[at + i] = (int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
        }
    };
    if (VECS > 0) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) {
            if (!NORM) Pairs<T>::widen(kept[i], products[i]);
            put(products[i], (me + i * threads) * 8);
        }
    } else {
        for (int at = me * 8; at < p.width; at += threads * 8) {
            product(load_some(x + at, p.width - at, p.vec_in), at, products[0], false);
            put(products[0], at);
        }
    }
    if (NORM && tiny && !bad) p.scales[row] = tiny_scale(x, p.width, p.eps, top);
}

template <typename T, bool NORM>
int launch_typed(const TokensArgs &p, cudaStream_t stream) {
    const int vecs = p.width > 0 ? (p.width + 7) / 8 : 1;
    auto threads = [&](int each) { return (int)round_up(ceil_div(vecs, each), 32); };
    const char *name = "quantize_tokens_kernel";
    // Rows of up to 1024 elements: a warp each, and no barrier
    const dim3 of_warps((unsigned)ceil_div(p.rows, ROWS_OF_WARPS)), one((unsigned)p.rows);
    if (vecs <= 32) return launch_after(name, quantize_tokens_kernel<T, NORM, 1, true>, of_warps, 32 * ROWS_OF_WARPS, 0, 1, stream, p);
    if (vecs <= 64) return launch_after(name, quantize_tokens_kernel<T, NORM, 2, true>, of_warps, 32 * ROWS_OF_WARPS, 0, 1, stream, p);
    if (vecs <= 128) return launch_after(name, quantize_tokens_kernel<T, NORM, 4, true>, of_warps, 32 * ROWS_OF_WARPS, 0, 1, stream, p);
    if (threads(1) <= 256 && p.rows <= 2 * sm_count()) return launch_after(name, quantize_tokens_kernel<T, NORM, 1, false>, one, threads(1), 0, 1, stream, p);
    if (threads(2) <= 256) return launch_after(name, quantize_tokens_kernel<T, NORM, 2, false>, one, threads(2), 0, 1, stream, p);
    if (threads(4) <= 512) return launch_after(name, quantize_tokens_kernel<T, NORM, 4, false>, one, threads(4), 0, 1, stream, p);
    return launch_after(name, quantize_tokens_kernel<T, NORM, 0, false>, one, MOST_THREADS, 0, 1, stream, p);
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
    if (width > kMostWidth || rows > 2147483647LL) return set_error(B200Q_UNSUPPORTED, "%s: %lld rows of %lld elements", op, (long long)rows, (long long)width);
    if (scales == nullptr || (width > 0 && (x == nullptr || codes == nullptr))) return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    if (x_stride < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative stride", op);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t size = type == B200Q_F32 ? 4 : 2;
    TokensArgs p = {x, x_stride, width > 0 ? norm : nullptr, eps, static_cast<int8_t *>(codes), scales, rows, (int)width,
                    aligned_to(x, 16) && (rows == 1 || x_stride * size % 16 == 0), aligned_to(norm, 16), aligned_to(codes, 8) && (rows == 1 || width % 8 == 0)};
    note_unfinished_codes(s);
    switch (type) {
        case B200Q_F16: return p.norm ? launch_typed<__half, true>(p, s) : launch_typed<__half, false>(p, s);
        case B200Q_BF16: return p.norm ? launch_typed<__nv_bfloat16, true>(p, s) : launch_typed<__nv_bfloat16, false>(p, s);
        default: return p.norm ? launch_typed<float, true>(p, s) : launch_typed<float, false>(p, s);
    }
}

}  // extern "C"
