// Tokens as three digits of 8 bits beside int8 weights: what the kernels of a layer of experts share.
//
// A row is written as whole numbers v = rint(x 2^e), |v| <= 2^22, e by its largest element, and these as v = 65536 d2 + 256 d1 + d0 with d in -128 .. 127: three columns of an
// int8 product, whose sums of 32 bits are exact.  An element is off by at most 2^-22 of the row's largest.
//
// Three, since a fourth would take a third more columns, copies and products, and buys what no rounded result shows but in rows of very unlike elements: with two channels 2^12 times the others
// errors are those of the result's rounding (2.1e-4 of f16, 1.7e-3 of bf16, relative), as with floats; where the weights have zeros at just these channels, 2.8e-4 of f16 with 2^10, 6.5e-4 to 8.9e-4 with
// 2^12, 3.1e-3 with 2^14, and of bf16 1.7e-3 with 2^12, 3.2e-3 to 3.8e-3 with 2^14.
#pragma once

#include "common.cuh"

namespace b200q {

constexpr int DIGITS = 3;
constexpr int kMostExact = 131071;  // products of 2^14 whose sum 32 bits hold

__device__ __forceinline__ float scale_at(const void *p, int type, int64_t i) {
    if (type == B200Q_F16) return __half2float(static_cast<const __half *>(p)[i]);
    if (type == B200Q_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return static_cast<const float *>(p)[i];
}

// The power of two that brings a row's largest magnitude (as bits) to 2^21 .. 2^22, and its inverse.  Rows below 2^-98 are zeros; rows with an infinity or a NaN are NaN.
__device__ __forceinline__ float power_for(uint32_t bits, float &inverse) {
    const int e = 148 - (int)(bits >> 23);  // 127 + 21 - exponent
    const bool zero = e > 119;
    inverse = bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : zero ? 0.0f : __uint_as_float((uint32_t)(127 - e) << 23);
    return zero || bits >= 0x7f800000u ? 0.0f : __uint_as_float((uint32_t)(127 + e) << 23);
}

// Eight neighbouring elements of a token.
struct FromF16 {
    typedef uint4 Raw[1];
    static __device__ __forceinline__ void load(const void *row, int k, Raw &r) { r[0] = *reinterpret_cast<const uint4 *>(static_cast<const __half *>(row) + k); }
    static __device__ __forceinline__ void widen(uint32_t w, float &lo, float &hi) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        lo = f.x, hi = f.y;
    }
    static __device__ __forceinline__ uint32_t largest(uint32_t bits, uint32_t w) {  // as float's
        return max(bits, max(__float_as_uint(__half2float(__ushort_as_half((uint16_t)(w & 0x7fffu)))), __float_as_uint(__half2float(__ushort_as_half((uint16_t)(w >> 16 & 0x7fffu))))));
    }
};
struct FromBF16 {
    typedef uint4 Raw[1];
    static __device__ __forceinline__ void load(const void *row, int k, Raw &r) { FromF16::load(row, k, r); }
    static __device__ __forceinline__ void widen(uint32_t w, float &lo, float &hi) { lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u); }
    static __device__ __forceinline__ uint32_t largest(uint32_t bits, uint32_t w) { return max(bits, max(w << 16 & 0x7fff0000u, w & 0x7fff0000u)); }
};
struct FromF32 {
    typedef uint4 Raw[2];
    static __device__ __forceinline__ void load(const void *row, int k, Raw &r) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const float *>(row) + k);
        r[0] = p[0], r[1] = p[1];
    }
};
template <typename X>
__device__ __forceinline__ void widen4(const typename X::Raw &r, int i, float (&f)[4]) {
    X::widen(i ? r[0].z : r[0].x, f[0], f[1]);
    X::widen(i ? r[0].w : r[0].y, f[2], f[3]);
}
template <>
__device__ __forceinline__ void widen4<FromF32>(const FromF32::Raw &r, int i, float (&f)[4]) {
    f[0] = __uint_as_float(r[i].x), f[1] = __uint_as_float(r[i].y), f[2] = __uint_as_float(r[i].z), f[3] = __uint_as_float(r[i].w);
}

// The digits of four elements, a word each: adding 1.5 * 2^23 rounds to a whole number that stands in the sum's low bits, and with 128 added to each digit they are its bytes.
__device__ __forceinline__ void digits_of(const float (&f)[4], float by, uint32_t (&d)[DIGITS]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(fmaf(f[i], by, 12582912.0f)) + (0x808080u - 0x4b400000u);
    const uint32_t lo = __byte_perm(u[0], u[1], 0x5140), hi = __byte_perm(u[2], u[3], 0x5140);
    d[0] = __byte_perm(lo, hi, 0x5410) ^ 0x80808080u;
    d[1] = __byte_perm(lo, hi, 0x7632) ^ 0x80808080u;
    d[2] = __byte_perm(__byte_perm(u[0], u[1], 0x0062), __byte_perm(u[2], u[3], 0x0062), 0x5410) ^ 0x80808080u;
}

__device__ __forceinline__ float token_value(const void *p, int type, int64_t i) {
    return type == B200Q_F16 ? __half2float(static_cast<const __half *>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

}  // namespace b200q
