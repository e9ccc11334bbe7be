// What the kernels of the decoding operators share: the layout of the quantized key/value cache, loads and stores of eight
// elements in any of the three types, and the launch as a programmatic dependent.
#pragma once

#include <atomic>

#include "common.cuh"
#include "status_bits.h"

namespace b200q {

// ---- the cache ----
// uint8 [pages][kv_heads][page_size / 16][32 D + 128]: a record per 16 positions of a head.  A record holds 16 rows of K
// codes, 16 rows of V codes (D bytes each, code + 128), the 16 float scales of K and the 16 of V.  All records of a page and head
// are one run of bytes, so one bulk copy brings any number of them, codes and scales, into shared memory.
//
// There the rows of a matrix load must lie in different banks without a swizzle on the way, so the 16-byte chunks of row r
// already stand in the order c ^ order(r): the rows that one phase of the load takes together (V: 8 neighbours; K: rows
// {0, 1, 4, 5, 8, 9, 12, 13} and {2, 3, 6, 7, 10, 11, 14, 15}, see cache_attention.cu) have ranks 0 to 7, and the order is as many upper bits of the
// rank as the number of chunks allows.  Rows of 128 and 256 bytes use all three; with rows of 64 and 192 bytes two neighbouring ranks lie in
// different banks by themselves; rows of 96 bytes keep conflicts of degree two.
__host__ __device__ constexpr int record_bytes(int dim) { return 32 * dim + 128; }
__host__ __device__ constexpr int order_shift(int dim) { return dim % 128 == 0 ? 0 : dim % 64 == 0 ? 1 : 2; }
__host__ __device__ constexpr uint32_t k_rank(uint32_t row) { return ((row >> 1) & 6u) | (row & 1u); }
__host__ __device__ constexpr uint32_t v_rank(uint32_t row) { return row & 7u; }
__host__ __device__ constexpr uint32_t k_order(uint32_t row, int dim) { return k_rank(row) >> order_shift(dim); }
__host__ __device__ constexpr uint32_t v_order(uint32_t row, int dim) { return v_rank(row) >> order_shift(dim); }
inline bool cache_dim(int64_t dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 192 || dim == 256; }

// n / d for n below 2^31 as n * by >> shift: by is 2^31+s / d rounded up, 2^s the power of two from d on, off by less than one part in 2^31.  Three instructions for
// the two dozen of a division.
struct Divisor {
    uint32_t by, shift;
};
inline Divisor divisor_of(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return {(uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}

struct CacheShape {
    int64_t slots;  // pages * page_size
    int page_size, kv_heads, dim;
    Divisor by_page;
    int records;      // of a page and head
    int page_records;  // of a page
    int order;        // order_shift(dim)
};
inline CacheShape cache_shape(int64_t pages, int64_t page_size, int64_t kv_heads, int64_t dim) {
    const int records = (int)page_size >> 4;
    return {pages * page_size, (int)page_size, (int)kv_heads, (int)dim, divisor_of((uint32_t)page_size), records, records * (int)kv_heads, order_shift((int)dim)};
}

#ifdef __CUDACC__

__device__ __forceinline__ uint32_t quotient(uint32_t n, Divisor d) { return (uint32_t)((uint64_t)n * d.by >> d.shift); }

// A slot's place: the record, and the row in it.
__device__ __forceinline__ uint8_t *record_of(uint8_t *cache, const CacheShape &c, int64_t slot, int head, uint32_t &row) {
    int64_t record;
    uint32_t in_page;
    if (c.slots <= 0x80000000ll) {
        const uint32_t page = quotient((uint32_t)slot, c.by_page);
        record = (uint64_t)page * (uint32_t)c.page_records;
        in_page = (uint32_t)slot - page * (uint32_t)c.page_size;
    } else {
        const int64_t page = slot / c.page_size;
        record = page * c.page_records;
        in_page = (uint32_t)(slot - page * c.page_size);
    }
    row = in_page & 15u;
    return cache + (record + ((uint32_t)(head * c.records) + (in_page >> 4))) * record_bytes(c.dim);
}

// ---- eight elements <-> float ----
template <typename T>
struct Elems;
template <>
struct Elems<__half> {
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
};
template <>
struct Elems<__nv_bfloat16> {
    static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elems<float> {
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ float round(float v) { return v; }
};

template <typename T>
struct alignas(16) Pack8 {
    T v[8];
};

// VEC: p is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ Pack8<T> load8(const T *p) {
    Pack8<T> x;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(&x)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x.v[i] = p[i];
    }
    return x;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *p, const Pack8<T> &x) {
    if (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(&x)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = x.v[i];
    }
}
// Two floats in a register pair, for the instructions that take two at once.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair_of(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ f32x2 pair_of(uint32_t lo, uint32_t hi) { return pair_of(__uint_as_float(lo), __uint_as_float(hi)); }
__device__ __forceinline__ void halves(f32x2 x, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Eight elements as four pairs of floats, and back.
template <typename T>
struct Pairs;
template <>
struct Pairs<__half> {
    static __device__ __forceinline__ void widen(const Pack8<__half> &x, f32x2 (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&x.v[2 * i]));
            f[i] = pair_of(p.x, p.y);
        }
    }
    static __device__ __forceinline__ Pack8<__half> narrow(const f32x2 (&f)[4]) {
        Pack8<__half> x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo, hi;
            halves(f[i], lo, hi);
            *reinterpret_cast<__half2 *>(&x.v[2 * i]) = __floats2half2_rn(lo, hi);
        }
        return x;
    }
};
template <>
struct Pairs<__nv_bfloat16> {
    static __device__ __forceinline__ void widen(const Pack8<__nv_bfloat16> &x, f32x2 (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = *reinterpret_cast<const uint32_t *>(&x.v[2 * i]);
            f[i] = pair_of(u << 16, u & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ Pack8<__nv_bfloat16> narrow(const f32x2 (&f)[4]) {
        Pack8<__nv_bfloat16> x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo, hi;
            halves(f[i], lo, hi);
            *reinterpret_cast<__nv_bfloat162 *>(&x.v[2 * i]) = __floats2bfloat162_rn(lo, hi);
        }
        return x;
    }
};
template <>
struct Pairs<float> {
    static __device__ __forceinline__ void widen(const Pack8<float> &x, f32x2 (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = pair_of(x.v[2 * i], x.v[2 * i + 1]);
    }
    static __device__ __forceinline__ Pack8<float> narrow(const f32x2 (&f)[4]) {
        Pack8<float> x;
#pragma unroll
        for (int i = 0; i < 4; ++i) halves(f[i], x.v[2 * i], x.v[2 * i + 1]);
        return x;
    }
};
template <typename T>
__device__ __forceinline__ Pack8<T> narrow(const float (&f)[8]) {
    const f32x2 p[4] = {pair_of(f[0], f[1]), pair_of(f[2], f[3]), pair_of(f[4], f[5]), pair_of(f[6], f[7])};
    return Pairs<T>::narrow(p);
}

__device__ __forceinline__ int64_t index_at(const void *p, int bytes, int64_t i) {
    return bytes == 8 ? static_cast<const int64_t *>(p)[i] : (int64_t) static_cast<const int32_t *>(p)[i];
}

// A launch as a programmatic dependent of the kernel in front, in clusters of `cluster` CTAs along x.
template <typename... Params, typename... Args>
inline int launch_after(const char *name, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = (unsigned)cluster;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
    if (err != cudaSuccess) return set_error(B200Q_CUDA_ERROR, "launch of %s failed: %s", name, cudaGetErrorString(err));
    return B200Q_OK;
}

// Lets a kernel have `smem` bytes of dynamic shared memory, once per device.
template <typename Kernel>
inline int allow_smem(std::atomic<bool> (&done)[64], Kernel kernel, int smem) {
    int device = -1;
    B200Q_CUDA_TRY(cudaGetDevice(&device));
    if (device >= 0 && device < 64 && done[device].load(std::memory_order_acquire)) return B200Q_OK;
    B200Q_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (device >= 0 && device < 64) done[device].store(true, std::memory_order_release);
    return B200Q_OK;
}
#endif  // __CUDACC__

inline bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace b200q
