// Rotary positions, and the quantized key/value cache as it is written and read back.
//
// Rotation: pairs (a, b) = (x[i], x[i + R/2]) ("half") or (x[2i], x[2i+1]) ("interleaved"), i < R/2, of every head become
// (a cos - b sin, b cos + a sin) with the cosine and sine of the token's position from a table; the other elements of the
// head are copied.  In float, every product and sum rounded by itself, one rounding to the result's type.
//
// Quantization: a row x of D elements (one token, one head) is stored as code = rint(x * (127 / amax)) and scale = amax / 127,
// amax = max |x|, so that |x - code * scale| <= scale / 2 (1 + 2^-15).  A row whose amax is below 2^-100 is stored as zeros; one with a
// NaN or an infinity has the scale NaN and codes of zero, so that it reads back as NaN and attention that sees it answers NaN.
// Scales are float: as f16 they would add 2^-11 to an error of 2^-8 at worst, for 2 bytes of 2 D + 8.
//
// Each element crosses memory once: the rotation of q and k and the quantization of k and v are one launch, in which a row's lanes hold it in
// registers from load to store.  Measured (64 + 8 heads of 128, 2048 tokens, bf16) 15.8 us for the rotation, 4.9 TB/s of what is read and written, with half of the
// issue slots used and the rest waiting for the loads behind the position's; (32 + 8 + 8 heads of 128, 8192 tokens, bf16) 43 us for the append, 4.4 TB/s, some
// 300 instructions a warp for its four rows; (8 heads of 128, 16384 tokens, f16) 20.9 us for the read, 4.9 TB/s with 60 % of the issue slots.  In float32, where
// bytes count for more, 24.6 us (6.2 TB/s), 59.7 (6.0) and 37.5 (4.5).  A few tokens cost the launch, 4.3 us.
#include "serving.cuh"

namespace b200q {
namespace {

constexpr int kThreads = 256;      // of a block, at most
constexpr float kTinyRow = 7.8886090522101180541e-31f;  // 2^-100

struct HeadRows {
    void *data;
    int64_t token_stride, head_stride;  // elements; the elements of a head are neighbours
};

struct RotaryArgs {
    const void *positions;
    const float *table;
    int64_t table_rows;
    int position_bytes, rotary_dim;
    bool interleaved;
    unsigned int *status;
};

// The table row of a token's position, or nullptr where the position lies outside the table.
__device__ __forceinline__ const float *angles_of(const RotaryArgs &r, uint32_t token) {
    const int64_t p = index_at(r.positions, r.position_bytes, token);
    return p < 0 || p >= r.table_rows ? nullptr : r.table + p * r.rotary_dim;
}

__device__ __forceinline__ void rotate(float &a, float &b, float c, float s) {
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}

template <bool VEC, int N>
__device__ __forceinline__ void load_floats(const float *p, float (&f)[N]) {
    if (VEC) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) reinterpret_cast<float4 *>(f)[i] = reinterpret_cast<const float4 *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = p[i];
    }
}

// The two chunks of eight elements of a head that lane j of its dim / 16 lanes holds, so that neighbouring lanes have neighbouring chunks: partners of a
// rotation (half), or half a head apart.
__device__ __forceinline__ void chunks_of(int j, int dim, const RotaryArgs &r, int &a, int &b) {
    const int pairs = r.interleaved ? 0 : r.rotary_dim >> 4, rest = (dim >> 4) - pairs;
    a = j < pairs ? j : pairs + j;
    b = j < pairs ? j + pairs : pairs + j + rest;
}

// Cosines and sines for a lane's two chunks: of eight pairs of elements, or (interleaved) of four of each chunk.
struct Angles {
    f32x2 c[4], s[4];
};
template <bool VEC>
__device__ __forceinline__ void load_pairs(const float *p, f32x2 &a, f32x2 &b) {
    alignas(16) float x[4];
    load_floats<VEC>(p, x);
    a = pair_of(x[0], x[1]), b = pair_of(x[2], x[3]);
}
template <bool VEC>
__device__ __forceinline__ Angles angles_for(const float *row, const RotaryArgs &r, int ca, int cb) {
    Angles g;
    const int half = r.rotary_dim >> 1;
    const int i = r.interleaved ? min(4 * ca, half - 4) : 8 * ca, j = r.interleaved ? min(4 * cb, half - 4) : 8 * ca + 4;  // a chunk that is not rotated takes any
    load_pairs<VEC>(row + i, g.c[0], g.c[1]);
    load_pairs<VEC>(row + j, g.c[2], g.c[3]);
    load_pairs<VEC>(row + half + i, g.s[0], g.s[1]);
    load_pairs<VEC>(row + half + j, g.s[2], g.s[3]);
    return g;
}
// Whether the chunks are rotated: both of a pair, or (interleaved) each by itself.
struct Turned {
    bool a, b;
};
__device__ __forceinline__ Turned turned(const RotaryArgs &r, int ca, int cb) { return {8 * ca < r.rotary_dim, 8 * cb < r.rotary_dim}; }

// a cos - b sin and b cos + a sin, every product and sum rounded by itself.
__device__ __forceinline__ void rotate_chunks(f32x2 (&a)[4], f32x2 (&b)[4], const Angles &g, bool interleaved, Turned t) {
    if (interleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float c[2], s[2], x, y;
            halves(g.c[e], c[0], c[1]);
            halves(g.s[e], s[0], s[1]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // the two pairs of elements that these angles turn
                f32x2 &pair = e < 2 ? a[2 * e + h] : b[2 * (e - 2) + h];
                if (!(e < 2 ? t.a : t.b)) continue;
                halves(pair, x, y);
                rotate(x, y, c[h], s[h]);
                pair = pair_of(x, y);
            }
        }
    } else if (t.a) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // one by one: a product and a sum of packed pairs become one instruction with one rounding
            float a0, a1, b0, b1, c0, c1, s0, s1;
            halves(a[e], a0, a1), halves(b[e], b0, b1), halves(g.c[e], c0, c1), halves(g.s[e], s0, s1);
            rotate(a0, b0, c0, s0);
            rotate(a1, b1, c1, s1);
            a[e] = pair_of(a0, a1), b[e] = pair_of(b0, b1);
        }
    }
}

__device__ __forceinline__ void zero_turned(f32x2 (&a)[4], f32x2 (&b)[4], Turned t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (t.a) a[e] = 0;
        if (t.b) b[e] = 0;
    }
}

// ---------------------------------------------------------------------------------------------
// rotary_embedding
// ---------------------------------------------------------------------------------------------

// A thread takes two chunks of eight elements of one head of one token (dim / 16 threads a head, threadIdx.x), with everything on its way at once but the angles, which
// wait for the position.  Few registers and many threads: with four heads a thread, which would save the other three's angles, (2048 tokens, 64 + 8 heads
// of 128) took 28.7 us for 21.2 with indexes divided out of one number.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 6) rotary_kernel(const __grid_constant__ HeadRows q, const __grid_constant__ HeadRows k, const __grid_constant__ HeadRows q_out,
                                                              const __grid_constant__ HeadRows k_out, const __grid_constant__ RotaryArgs r, int64_t tokens, int heads, int all_heads,
                                                              int dim) {
    pdl_wait();
    pdl_launch_dependents();
    const int j = threadIdx.x, head = blockIdx.y * blockDim.y + threadIdx.y;
    const uint32_t token = blockIdx.x * blockDim.z + threadIdx.z;  // 32 bits are enough for what the host lets through, rounded up to blocks
    if (token >= tokens || head >= all_heads) return;
    const bool is_q = head < heads;
    const HeadRows &src = is_q ? q : k, &dst = is_q ? q_out : k_out;
    const int h = is_q ? head : head - heads;
    int ca, cb;
    chunks_of(j, dim, r, ca, cb);
    const T *x = static_cast<const T *>(src.data) + token * src.token_stride + h * src.head_stride;
    T *y = static_cast<T *>(dst.data) + token * dst.token_stride + h * dst.head_stride;
    const Turned t = turned(r, ca, cb);
    if (!t.a && !t.b && x == y) return;
    Pack8<T> xa = load8<T, VEC>(x + 8 * ca), xb = load8<T, VEC>(x + 8 * cb);
    if (t.a || t.b) {
        const float *row = angles_of(r, token);
        f32x2 a[4], b[4];
        Pairs<T>::widen(xa, a);
        Pairs<T>::widen(xb, b);
        if (row != nullptr) {
            const Angles g = angles_for<VEC>(row, r, ca, cb);
            rotate_chunks(a, b, g, r.interleaved, t);
        } else {
            zero_turned(a, b, t);
            if (j == 0 && head == 0 && r.status != nullptr) atomicOr(r.status, kBadPosition);
        }
        xa = Pairs<T>::narrow(a);
        xb = Pairs<T>::narrow(b);
    }
    store8<T, VEC>(y + 8 * ca, xa);
    store8<T, VEC>(y + 8 * cb, xb);
}

// Any sizes: a thread per pair, and per element that is only copied.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_generic_kernel(HeadRows q, HeadRows k, HeadRows q_out, HeadRows k_out, RotaryArgs r, int64_t tokens, int heads,
                                                                  int all_heads, int dim) {
    pdl_wait();
    pdl_launch_dependents();
    const int half = r.rotary_dim >> 1, units = dim - half;  // pairs, then single elements
    const int64_t total = tokens * all_heads * units;
    for (int64_t u = (int64_t)blockIdx.x * kThreads + threadIdx.x; u < total; u += (int64_t)gridDim.x * kThreads) {
        const int64_t row = u / units, token = row / all_heads;
        const int i = (int)(u - row * units), head = (int)(row - token * all_heads);
        const bool is_q = head < heads;
        const HeadRows &src = is_q ? q : k, &dst = is_q ? q_out : k_out;
        const int h = is_q ? head : head - heads;
        const T *x = static_cast<const T *>(src.data) + token * src.token_stride + h * src.head_stride;
        T *y = static_cast<T *>(dst.data) + token * dst.token_stride + h * dst.head_stride;
        if (i >= half) {
            y[half + i] = x[half + i];
            continue;
        }
        const int ia = r.interleaved ? 2 * i : i, ib = r.interleaved ? 2 * i + 1 : i + half;
        const float *angles = angles_of(r, (uint32_t)token);
        float a = 0.0f, b = 0.0f;
        if (angles != nullptr) {
            a = Elems<T>::one(x[ia]);
            b = Elems<T>::one(x[ib]);
            rotate(a, b, angles[i], angles[half + i]);
        } else if (i == 0 && head == 0 && r.status != nullptr) {
            atomicOr(r.status, kBadPosition);
        }
        y[ia] = Elems<T>::round(a);
        y[ib] = Elems<T>::round(b);
    }
}

// ---------------------------------------------------------------------------------------------
// quantized_cache_append
// ---------------------------------------------------------------------------------------------

// Codes of eight elements, plus 128, as bytes: adding 1.5 * 2^23 + 128 rounds to the nearest even integer and leaves it in the low byte.
__device__ __forceinline__ uint2 codes_of(const f32x2 (&x)[4], float inv) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float lo, hi;
        halves(x[i], lo, hi);
        u[2 * i] = __float_as_uint(__fadd_rn(__fmul_rn(lo, inv), 12582912.0f + 128.0f));
        u[2 * i + 1] = __float_as_uint(__fadd_rn(__fmul_rn(hi, inv), 12582912.0f + 128.0f));
    }
    return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}
// The largest magnitude of both; NaN stays.
__device__ __forceinline__ float larger(float top, float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(top), "f"(fabsf(x)));
    return r;
}

// Five blocks an SM: for six the registers spill, a fifth slower; four are slower by 4 %.
// GROUP lanes (threadIdx.x, dim / 16 of them active) hold a row: a head of q (rotated and written), of k (rotated and quantized) or of v (quantized).
template <typename T, bool VEC, int GROUP>
__global__ void __launch_bounds__(kThreads, 5) append_kernel(const __grid_constant__ HeadRows q, const __grid_constant__ HeadRows q_out, const __grid_constant__ HeadRows k,
                                                              const __grid_constant__ HeadRows v, uint8_t *cache, const __grid_constant__ CacheShape c, const void *slots, int slot_bytes,
                                                              const __grid_constant__ RotaryArgs r, int64_t tokens, int heads) {
    pdl_wait();
    pdl_launch_dependents();
    const int j = threadIdx.x, row = blockIdx.y * blockDim.y + threadIdx.y, rows = heads + 2 * c.kv_heads;
    const uint32_t token = blockIdx.x * blockDim.z + threadIdx.z;  // 32 bits are enough for what the host lets through, rounded up to blocks
    const bool active = token < tokens && row < rows && 16 * j < c.dim;
    const bool is_q = row < heads, is_v = row >= heads + c.kv_heads;
    const int h = is_q ? row : is_v ? row - heads - c.kv_heads : row - heads;
    const HeadRows &src = is_q ? q : is_v ? v : k;
    int ca, cb;
    chunks_of(j, c.dim, r, ca, cb);
    f32x2 a[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = b[e] = 0;
    int64_t slot = -1;
    if (active) {
        const T *x = static_cast<const T *>(src.data) + token * src.token_stride + h * src.head_stride;
        const Pack8<T> xa = load8<T, VEC>(x + 8 * ca), xb = load8<T, VEC>(x + 8 * cb);
        if (!is_q) slot = index_at(slots, slot_bytes, token);
        const Turned t = turned(r, ca, cb);
        const bool turns = r.rotary_dim > 0 && !is_v && (t.a || t.b);
        const float *angles = turns ? angles_of(r, token) : nullptr;
        Angles g;
        if (angles != nullptr) g = angles_for<VEC>(angles, r, ca, cb);
        Pairs<T>::widen(xa, a);
        Pairs<T>::widen(xb, b);
        if (angles != nullptr) {
            rotate_chunks(a, b, g, r.interleaved, t);
        } else if (turns) {
            zero_turned(a, b, t);
            if (row == 0 && j == 0 && r.status != nullptr) atomicOr(r.status, kBadPosition);
        }
    }
    if (active && is_q) {
        T *y = static_cast<T *>(q_out.data) + token * q_out.token_stride + h * q_out.head_stride;
        store8<T, VEC>(y + 8 * ca, Pairs<T>::narrow(a));
        store8<T, VEC>(y + 8 * cb, Pairs<T>::narrow(b));
    }
    if (!__any_sync(0xffffffffu, active && !is_q)) return;  // nothing to quantize in this warp
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float lo, hi;
        halves(a[e], lo, hi);
        top = larger(larger(top, lo), hi);
        halves(b[e], lo, hi);
        top = larger(larger(top, lo), hi);
    }
#pragma unroll
    for (int d = GROUP / 2; d > 0; d /= 2) top = larger(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (!active || is_q) return;
    if (slot < 0) return;  // padding
    if (slot >= c.slots) {
        if (row == heads && j == 0 && r.status != nullptr) atomicOr(r.status, kBadSlot);
        return;
    }
    const bool fine = top < INFINITY && top >= kTinyRow;
    const float inv = fine ? __fdiv_rn(127.0f, top) : 0.0f;
    if (!fine) {  // 0 * inf is no zero
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = b[e] = 0;
    }
    uint32_t in_record;
    uint8_t *record = record_of(cache, c, slot, h, in_record);
    const uint32_t order = (is_v ? v_rank(in_record) : k_rank(in_record)) >> c.order;
    uint8_t *codes = record + (is_v ? 16 * c.dim : 0) + in_record * c.dim;
    *reinterpret_cast<uint2 *>(codes + 16 * (((uint32_t)ca >> 1) ^ order) + 8 * (ca & 1)) = codes_of(a, inv);
    *reinterpret_cast<uint2 *>(codes + 16 * (((uint32_t)cb >> 1) ^ order) + 8 * (cb & 1)) = codes_of(b, inv);
    if (j == 0) {
        const float scale = fine ? __fdiv_rn(top, 127.0f) : top < INFINITY ? 0.0f : __uint_as_float(0x7fc00000u);
        reinterpret_cast<float *>(record + 32 * c.dim)[(is_v ? 16 : 0) + in_record] = scale;
    }
}

// ---------------------------------------------------------------------------------------------
// quantized_cache_read
// ---------------------------------------------------------------------------------------------

// A thread restores eight elements of a row of K and the same of V.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(const uint8_t *cache, const __grid_constant__ CacheShape c, const void *slots, int slot_bytes, T *k, T *v, int64_t tokens,
                                                            unsigned int *status) {
    pdl_wait();
    pdl_launch_dependents();
    const int j = threadIdx.x, h = blockIdx.y * blockDim.y + threadIdx.y;
    const uint32_t token = blockIdx.x * blockDim.z + threadIdx.z;  // 32 bits are enough for what the host lets through, rounded up to blocks
    if (token >= tokens || h >= c.kv_heads) return;
    const int64_t slot = index_at(slots, slot_bytes, token);
    uint2 x[2] = {make_uint2(0x80808080u, 0x80808080u), make_uint2(0x80808080u, 0x80808080u)};
    float scale[2] = {0.0f, 0.0f};
    if (slot >= 0 && slot < c.slots) {
        uint32_t in_record;
        const uint8_t *record = record_of(const_cast<uint8_t *>(cache), c, slot, h, in_record), *codes = record + in_record * c.dim + 8 * (j & 1);
        x[0] = *reinterpret_cast<const uint2 *>(codes + 16 * (((uint32_t)j >> 1) ^ k_rank(in_record) >> c.order));
        x[1] = *reinterpret_cast<const uint2 *>(codes + 16 * c.dim + 16 * (((uint32_t)j >> 1) ^ v_rank(in_record) >> c.order));
        scale[0] = reinterpret_cast<const float *>(record + 32 * c.dim)[in_record];
        scale[1] = reinterpret_cast<const float *>(record + 32 * c.dim)[16 + in_record];
    } else if (slot >= c.slots && j == 0 && h == 0 && status != nullptr) {
        atomicOr(status, kBadSlot);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f32x2 y[4];
        const f32x2 minus = pair_of(-(8388608.0f + 128.0f), -(8388608.0f + 128.0f)), by = pair_of(scale[i], scale[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // 2^23 + byte, exactly
            const uint32_t w = e < 2 ? x[i].x : x[i].y;
            y[e] = mul2(add2(pair_of(__byte_perm(w, 0x4b000000u, 0x7540u | (2 * e & 3)), __byte_perm(w, 0x4b000000u, 0x7540u | (2 * e + 1 & 3))), minus), by);
        }
        store8<T, true>((i == 0 ? k : v) + ((int64_t)token * c.kv_heads + h) * c.dim + 8 * j, Pairs<T>::narrow(y));
    }
}

// Blocks of lanes x rows x tokens threads, about kThreads of them: the rows of a token in as many equal blocks as they need, or several tokens a block.  `unit`: rows
// come in multiples of it.
void shape(int64_t tokens, int rows, int lanes, int unit, dim3 &block, dim3 &grid) {
    const int room = kThreads / lanes > unit ? kThreads / lanes / unit * unit : unit, parts = (rows + room - 1) / room;
    const int each = ((rows + parts - 1) / parts + unit - 1) / unit * unit;
    int together = parts == 1 && room > each ? room / each : 1;
    const int64_t spread_out = ceil_div(tokens, (int64_t)2 * sm_count());  // a block for every SM, and another, before tokens share one
    if (together > spread_out) together = spread_out > 1 ? (int)spread_out : 1;
    if (together > 64) together = 64;
    block = dim3((unsigned)lanes, (unsigned)each, (unsigned)together);
    grid = dim3((unsigned)ceil_div(tokens, together), (unsigned)((rows + each - 1) / each), 1);
}

bool rows_aligned(const HeadRows &r, size_t item) {
    return aligned_to(r.data, 16) && (r.token_stride * item) % 16 == 0 && (r.head_stride * item) % 16 == 0;
}

HeadRows rows_of(const b200q_heads *h) { return h != nullptr ? HeadRows{h->data, h->token_stride, h->head_stride} : HeadRows{nullptr, 0, 0}; }

int check_rotary(const char *op, const void *positions, const float *table, int64_t table_rows, int64_t rotary_dim, int64_t head_dim, int layout, int position_bytes) {
    if (layout != B200Q_ROTARY_HALF && layout != B200Q_ROTARY_INTERLEAVED) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown rotary layout %d", op, layout);
    if (position_bytes != 4 && position_bytes != 8) return set_error(B200Q_INVALID_ARGUMENT, "%s: positions must be int32 or int64 (4 or 8 bytes), got %d", op, position_bytes);
    if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: %lld rotated elements: an even number of at most the head's %lld is wanted", op, (long long)rotary_dim, (long long)head_dim);
    }
    if (table_rows < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative table size %lld", op, (long long)table_rows);
    if (positions == nullptr || table == nullptr) return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    return B200Q_OK;
}

int check_cache(const char *op, const void *cache, int64_t pages, int64_t page_size, int64_t kv_heads, int64_t head_dim) {
    if (pages < 0 || kv_heads <= 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: a cache of %lld pages and %lld heads", op, (long long)pages, (long long)kv_heads);
    if (page_size <= 0 || page_size % 16 != 0 || page_size > 65536) {
        return set_error(B200Q_UNSUPPORTED, "%s: pages of %lld positions: multiples of 16 up to 65536 are supported", op, (long long)page_size);
    }
    if (!cache_dim(head_dim)) return set_error(B200Q_UNSUPPORTED, "%s: heads of %lld elements: 64, 96, 128, 192 and 256 are supported", op, (long long)head_dim);
    if (kv_heads > 65536) return set_error(B200Q_UNSUPPORTED, "%s: %lld heads", op, (long long)kv_heads);
    if (pages > 1ll << 40) return set_error(B200Q_UNSUPPORTED, "%s: %lld pages", op, (long long)pages);
    if (pages > 0 && (cache == nullptr || !aligned_to(cache, 16))) return set_error(B200Q_INVALID_ARGUMENT, "%s: the cache must be 16-byte aligned, got %p", op, cache);
    return B200Q_OK;
}

template <typename T>
int rotary_typed(const HeadRows &q, const HeadRows &k, const HeadRows &q_out, const HeadRows &k_out, const RotaryArgs &r, int64_t tokens, int heads, int kv_heads, int dim,
                 cudaStream_t stream) {
    const int all = heads + kv_heads;
    if (dim % 16 == 0 && dim <= 16 * 32 && r.rotary_dim % 16 == 0) {
        const size_t s = sizeof(T);
        const bool vec = rows_aligned(q, s) && rows_aligned(q_out, s) && rows_aligned(k, s) && rows_aligned(k_out, s) && aligned_to(r.table, 16);
        dim3 block, grid;
        shape(tokens, all, dim / 16, 1, block, grid);
        auto kernel = vec ? rotary_kernel<T, true> : rotary_kernel<T, false>;
        return launch_after("rotary_kernel", kernel, grid, block, 0, 1, stream, q, k, q_out, k_out, r, tokens, heads, all, dim);
    }
    const int64_t ctas = ceil_div(tokens * all * (dim - r.rotary_dim / 2), kThreads);
    return launch_after("rotary_generic_kernel", rotary_generic_kernel<T>, dim3((unsigned)(ctas < 65536 ? ctas : 65536)), kThreads, 0, 1, stream, q, k, q_out, k_out, r, tokens, heads,
                        all, dim);
}

template <typename T, bool VEC>
int append_sized(const HeadRows &q, const HeadRows &q_out, const HeadRows &k, const HeadRows &v, uint8_t *cache, const CacheShape &c, const void *slots, int slot_bytes,
                 const RotaryArgs &r, int64_t tokens, int heads, cudaStream_t stream) {
    const int group = c.dim <= 64 ? 4 : c.dim <= 128 ? 8 : 16;
    dim3 block, grid;
    shape(tokens, heads + 2 * c.kv_heads, group, 32 / group, block, grid);  // whole warps, for the shuffles
    auto kernel = group == 4 ? append_kernel<T, VEC, 4> : group == 8 ? append_kernel<T, VEC, 8> : append_kernel<T, VEC, 16>;
    return launch_after("append_kernel", kernel, grid, block, 0, 1, stream, q, q_out, k, v, cache, c, slots, slot_bytes, r, tokens, heads);
}

template <typename T>
int append_typed(const HeadRows &q, const HeadRows &q_out, const HeadRows &k, const HeadRows &v, uint8_t *cache, const CacheShape &c, const void *slots, int slot_bytes,
                 const RotaryArgs &r, int64_t tokens, int heads, cudaStream_t stream) {
    const size_t s = sizeof(T);
    const bool vec = rows_aligned(k, s) && rows_aligned(v, s) && rows_aligned(q, s) && rows_aligned(q_out, s) && aligned_to(r.table, 16);
    return vec ? append_sized<T, true>(q, q_out, k, v, cache, c, slots, slot_bytes, r, tokens, heads, stream)
               : append_sized<T, false>(q, q_out, k, v, cache, c, slots, slot_bytes, r, tokens, heads, stream);
}

template <typename T>
int read_typed(const uint8_t *cache, const CacheShape &c, const void *slots, int slot_bytes, void *k, void *v, int64_t tokens, cudaStream_t stream) {
    dim3 block, grid;
    shape(tokens, c.kv_heads, c.dim / 8, 1, block, grid);
    return launch_after("read_kernel", read_kernel<T>, grid, block, 0, 1, stream, cache, c, slots, slot_bytes, static_cast<T *>(k), static_cast<T *>(v), tokens, device_status_word());
}

constexpr int64_t kMostTokens = 2147483647;  // of the grid's first dimension

}  // namespace
}  // namespace b200q

extern "C" {

B200Q_API int b200q_rotary_embedding(const b200q_heads *q, const b200q_heads *k, const b200q_heads *q_out, const b200q_heads *k_out, const void *positions, const float *table,
                                     int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, int64_t table_rows, int layout, int type,
                                     int position_bytes, void *stream) {
    using namespace b200q;
    const char *op = "rotary_embedding";
    if (tokens < 0 || heads < 0 || kv_heads < 0 || head_dim < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative size", op);
    if (type < B200Q_F16 || type > B200Q_F32) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown float type %d", op, type);
    if (tokens == 0 || heads + kv_heads == 0) return B200Q_OK;
    const int rc = check_rotary(op, positions, table, table_rows, rotary_dim, head_dim, layout, position_bytes);
    if (rc != B200Q_OK) return rc;
    if (heads > 65536 || kv_heads > 65536 || head_dim > 65536 || tokens > kMostTokens) return set_error(B200Q_UNSUPPORTED, "%s: %lld tokens of %lld + %lld heads of %lld", op, (long long)tokens, (long long)heads, (long long)kv_heads, (long long)head_dim);
    if ((heads > 0 && (q == nullptr || q_out == nullptr || q->data == nullptr || q_out->data == nullptr)) ||
        (kv_heads > 0 && (k == nullptr || k_out == nullptr || k->data == nullptr || k_out->data == nullptr))) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    }
    const RotaryArgs r = {positions, table, table_rows, position_bytes, (int)rotary_dim, layout == B200Q_ROTARY_INTERLEAVED, device_status_word()};
    const HeadRows none = {nullptr, 0, 0};
    const HeadRows a = heads > 0 ? rows_of(q) : none, b = kv_heads > 0 ? rows_of(k) : none, ao = heads > 0 ? rows_of(q_out) : none, bo = kv_heads > 0 ? rows_of(k_out) : none;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (type) {
        case B200Q_F16: return rotary_typed<__half>(a, b, ao, bo, r, tokens, (int)heads, (int)kv_heads, (int)head_dim, s);
        case B200Q_BF16: return rotary_typed<__nv_bfloat16>(a, b, ao, bo, r, tokens, (int)heads, (int)kv_heads, (int)head_dim, s);
        default: return rotary_typed<float>(a, b, ao, bo, r, tokens, (int)heads, (int)kv_heads, (int)head_dim, s);
    }
}

B200Q_API int b200q_quantized_cache_append(void *cache, int64_t pages, int64_t page_size, const b200q_heads *k, const b200q_heads *v, const b200q_heads *q,
                                           const b200q_heads *q_out, const void *slots, const void *positions, const float *table, int64_t tokens, int64_t heads,
                                           int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, int64_t table_rows, int layout, int type, int slot_bytes, int position_bytes,
                                           void *stream) {
    using namespace b200q;
    const char *op = "quantized_cache_append";
    if (tokens < 0 || heads < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative size", op);
    if (type < B200Q_F16 || type > B200Q_F32) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown float type %d", op, type);
    if (slot_bytes != 4 && slot_bytes != 8) return set_error(B200Q_INVALID_ARGUMENT, "%s: slots must be int32 or int64 (4 or 8 bytes), got %d", op, slot_bytes);
    int rc = check_cache(op, cache, pages, page_size, kv_heads, head_dim);
    if (rc != B200Q_OK) return rc;
    if (tokens == 0) return B200Q_OK;
    if (heads > 65536 || tokens > kMostTokens) return set_error(B200Q_UNSUPPORTED, "%s: %lld tokens of %lld heads", op, (long long)tokens, (long long)heads);
    if (rotary_dim != 0 || heads > 0) {
        rc = check_rotary(op, positions, table, table_rows, rotary_dim, head_dim, layout, position_bytes);
        if (rc != B200Q_OK) return rc;
        if (rotary_dim % 16 != 0) return set_error(B200Q_UNSUPPORTED, "%s: %lld rotated elements: multiples of 16 are supported", op, (long long)rotary_dim);
    }
    if (slots == nullptr || k == nullptr || v == nullptr || k->data == nullptr || v->data == nullptr ||
        (heads > 0 && (q == nullptr || q_out == nullptr || q->data == nullptr || q_out->data == nullptr))) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    }
    const CacheShape c = cache_shape(pages, page_size, kv_heads, head_dim);
    const RotaryArgs r = {positions, table, table_rows, position_bytes, (int)rotary_dim, layout == B200Q_ROTARY_INTERLEAVED, device_status_word()};
    const HeadRows none = {nullptr, 0, 0};
    const HeadRows a = heads > 0 ? rows_of(q) : none, ao = heads > 0 ? rows_of(q_out) : none, kr = rows_of(k), vr = rows_of(v);
    uint8_t *bytes = static_cast<uint8_t *>(cache);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (type) {
        case B200Q_F16: return append_typed<__half>(a, ao, kr, vr, bytes, c, slots, slot_bytes, r, tokens, (int)heads, s);
        case B200Q_BF16: return append_typed<__nv_bfloat16>(a, ao, kr, vr, bytes, c, slots, slot_bytes, r, tokens, (int)heads, s);
        default: return append_typed<float>(a, ao, kr, vr, bytes, c, slots, slot_bytes, r, tokens, (int)heads, s);
    }
}

B200Q_API int b200q_quantized_cache_read(const void *cache, int64_t pages, int64_t page_size, const void *slots, void *k, void *v, int64_t tokens, int64_t kv_heads,
                                         int64_t head_dim, int type, int slot_bytes, void *stream) {
    using namespace b200q;
    const char *op = "quantized_cache_read";
    if (tokens < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative size", op);
    if (type < B200Q_F16 || type > B200Q_F32) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown float type %d", op, type);
    if (slot_bytes != 4 && slot_bytes != 8) return set_error(B200Q_INVALID_ARGUMENT, "%s: slots must be int32 or int64 (4 or 8 bytes), got %d", op, slot_bytes);
    const int rc = check_cache(op, cache, pages, page_size, kv_heads, head_dim);
    if (rc != B200Q_OK) return rc;
    if (tokens == 0) return B200Q_OK;
    if (tokens > kMostTokens) return set_error(B200Q_UNSUPPORTED, "%s: %lld tokens", op, (long long)tokens);
    if (slots == nullptr || k == nullptr || v == nullptr) return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    if (!aligned_to(k, 16) || !aligned_to(v, 16)) return set_error(B200Q_INVALID_ARGUMENT, "%s: k and v must be 16-byte aligned", op);
    const CacheShape c = cache_shape(pages, page_size, kv_heads, head_dim);
    const uint8_t *bytes = static_cast<const uint8_t *>(cache);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (type) {
        case B200Q_F16: return read_typed<__half>(bytes, c, slots, slot_bytes, k, v, tokens, s);
        case B200Q_BF16: return read_typed<__nv_bfloat16>(bytes, c, slots, slot_bytes, k, v, tokens, s);
        default: return read_typed<float>(bytes, c, slots, slot_bytes, k, v, tokens, s);
    }
}

}  // extern "C"
