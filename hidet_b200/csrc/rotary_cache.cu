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
// All of it is bound by memory traffic, and at a few tokens by the launch.  Each element crosses memory once: the rotation of q and k and
// the quantization of k and v are one launch, in which a row's lanes hold it in registers from load to store.
#include "serving.cuh"

namespace b200q {
namespace {

constexpr int kThreads = 256;
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
__device__ __forceinline__ const float *angles_of(const RotaryArgs &r, int64_t token) {
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

// Two chunks of eight elements of one head, whose pairs are (half) across them, from angle i on, or (interleaved) inside them.
template <bool VEC>
__device__ __forceinline__ void rotate_chunks(float (&a)[8], float (&b)[8], const float *angles, int half_dim, int i, bool interleaved) {
    alignas(16) float c[8], s[8];
    load_floats<VEC>(angles + i, c);
    load_floats<VEC>(angles + half_dim + i, s);
    if (interleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            rotate(a[2 * e], a[2 * e + 1], c[e], s[e]);
            rotate(b[2 * e], b[2 * e + 1], c[e + 4], s[e + 4]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) rotate(a[e], b[e], c[e], s[e]);
    }
}

// The two chunks of a head that lane j of its dim / 16 lanes holds: partners of a rotation as long as there are such.
__device__ __forceinline__ void chunks_of(int j, int rotary_dim, bool interleaved, int &a, int &b) {
    const int pairs = rotary_dim >> 4;
    const bool across = !interleaved && j < pairs;
    a = across ? j : 2 * j;
    b = across ? j + pairs : 2 * j + 1;
}

// ---------------------------------------------------------------------------------------------
// rotary_embedding
// ---------------------------------------------------------------------------------------------

// A thread takes two chunks of eight elements of a head (dim / 16 threads a head).  One or a few CTAs a token where tokens are few, and several
// tokens a CTA where they are many, so that a thread has about four such units: (2048 tokens, 64 + 8 heads of 128, bf16).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) rotary_kernel(HeadRows q, HeadRows k, HeadRows q_out, HeadRows k_out, RotaryArgs r, int64_t tokens, int heads, int all_heads,
                                                          int dim, int tokens_per_cta) {
    pdl_wait();
    pdl_launch_dependents();
    const int lanes = dim >> 4, units = all_heads * lanes;
    const int64_t first = (int64_t)blockIdx.x * tokens_per_cta;
    const int n = (int)min((int64_t)tokens_per_cta, tokens - first) * units;
#pragma unroll 2
    for (int u = blockIdx.y * kThreads + threadIdx.x; u < n; u += gridDim.y * kThreads) {
        const int t = u / units, in_token = u - t * units;
        const int head = in_token / lanes, j = in_token - head * lanes;
        const int64_t token = first + t;
        const bool is_q = head < heads;
        const HeadRows &src = is_q ? q : k, &dst = is_q ? q_out : k_out;
        const int h = is_q ? head : head - heads;
        int ca, cb;
        chunks_of(j, r.rotary_dim, r.interleaved, ca, cb);
        const T *x = static_cast<const T *>(src.data) + token * src.token_stride + h * src.head_stride;
        T *y = static_cast<T *>(dst.data) + token * dst.token_stride + h * dst.head_stride;
        const Pack8<T> xa = load8<T, VEC>(x + 8 * ca), xb = load8<T, VEC>(x + 8 * cb);
        if (16 * j < r.rotary_dim) {
            const float *angles = angles_of(r, token);
            float a[8], b[8];
            if (angles != nullptr) {
                widen(xa, a);
                widen(xb, b);
                rotate_chunks<VEC>(a, b, angles, r.rotary_dim >> 1, 8 * j, r.interleaved);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] = b[e] = 0.0f;
                if (in_token == 0 && r.status != nullptr) atomicOr(r.status, kBadPosition);
            }
            store8<T, VEC>(y + 8 * ca, narrow<T>(a));
            store8<T, VEC>(y + 8 * cb, narrow<T>(b));
        } else if (x != y) {
            store8<T, VEC>(y + 8 * ca, xa);
            store8<T, VEC>(y + 8 * cb, xb);
        }
    }
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
        const float *angles = angles_of(r, token);
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
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float inv) {
    uint32_t m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), 12582912.0f + 128.0f));
    uint2 r;
    r.x = __byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410);
    r.y = __byte_perm(__byte_perm(m[4], m[5], 0x0040), __byte_perm(m[6], m[7], 0x0040), 0x5410);
    return r;
}

// GROUP lanes (dim / 16 of them active) hold a row: a head of q (rotated and written), of k (rotated and quantized) or of v (quantized).
template <typename T, bool VEC, int GROUP>
__global__ void __launch_bounds__(kThreads) append_kernel(HeadRows q, HeadRows q_out, HeadRows k, HeadRows v, uint8_t *cache, CacheShape c, const void *slots, int slot_bytes,
                                                          RotaryArgs r, int64_t tokens, int heads, int tokens_per_cta) {
    pdl_wait();
    pdl_launch_dependents();
    const int j = threadIdx.x % GROUP, rows = heads + 2 * c.kv_heads;
    const bool active = 16 * j < c.dim;
    const int64_t first = (int64_t)blockIdx.x * tokens_per_cta;
    const int n = (int)min((int64_t)tokens_per_cta, tokens - first) * rows;
    constexpr int PER_CTA = kThreads / GROUP;
    const bool across = r.rotary_dim > 0;  // 0: nothing is rotated
    // every lane of a warp makes the same number of rounds, for the shuffles
    const int rounds = (n - (int)blockIdx.y * PER_CTA + (int)gridDim.y * PER_CTA - 1) / ((int)gridDim.y * PER_CTA);
    for (int round = 0; round < rounds; ++round) {
        const int u = (round * gridDim.y + blockIdx.y) * PER_CTA + threadIdx.x / GROUP;
        const bool there = u < n;
        const int t = there ? u / rows : 0, in_token = there ? u - t * rows : 0;
        const int64_t token = first + t;
        const bool is_q = in_token < heads, is_v = in_token >= heads + c.kv_heads;
        const int h = is_q ? in_token : is_v ? in_token - heads - c.kv_heads : in_token - heads;
        const HeadRows &src = is_q ? q : is_v ? v : k;
        const bool rotated = across && !is_v && 16 * j < r.rotary_dim;
        int ca = 2 * j, cb = 2 * j + 1;
        if (across && !is_v) chunks_of(j, r.rotary_dim, r.interleaved, ca, cb);
        float a[8], b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = b[e] = 0.0f;
        if (there && active) {
            const T *x = static_cast<const T *>(src.data) + token * src.token_stride + h * src.head_stride;
            const Pack8<T> xa = load8<T, VEC>(x + 8 * ca), xb = load8<T, VEC>(x + 8 * cb);
            const float *angles = rotated ? angles_of(r, token) : nullptr;
            if (rotated && angles == nullptr) {
                if (in_token == 0 && j == 0 && r.status != nullptr) atomicOr(r.status, kBadPosition);
            } else {
                widen(xa, a);
                widen(xb, b);
            }
            if (angles != nullptr) rotate_chunks<VEC>(a, b, angles, r.rotary_dim >> 1, 8 * j, r.interleaved);
        }
        // max |x| as bits: NaNs and infinities are larger than every finite value
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(b[e]) & 0x7fffffffu));
#pragma unroll
        for (int d = GROUP / 2; d > 0; d /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (!there || !active) continue;
        if (is_q) {
            T *y = static_cast<T *>(q_out.data) + token * q_out.token_stride + h * q_out.head_stride;
            store8<T, VEC>(y + 8 * ca, narrow<T>(a));
            store8<T, VEC>(y + 8 * cb, narrow<T>(b));
            continue;
        }
        const int64_t slot = index_at(slots, slot_bytes, token);
        if (slot < 0) continue;  // padding
        if (slot >= c.slots) {
            if (in_token == heads && j == 0 && r.status != nullptr) atomicOr(r.status, kBadSlot);
            continue;
        }
        const float amax = __uint_as_float(top);
        const bool fine = top < 0x7f800000u && amax >= kTinyRow;
        const float inv = fine ? __fdiv_rn(127.0f, amax) : 0.0f;
        if (!fine) {  // 0 * inf is no zero
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = b[e] = 0.0f;
        }
        uint32_t row;
        uint8_t *record = record_of(cache, c, slot, h, row);
        const uint32_t order = is_v ? v_order(row, c.dim) : k_order(row, c.dim);
        uint8_t *codes = record + (is_v ? 16 * c.dim : 0) + row * c.dim;
        const uint2 xa = codes_of(a, inv), xb = codes_of(b, inv);
        if (cb == ca + 1 && (ca & 1) == 0) {
            *reinterpret_cast<uint4 *>(codes + 16 * (((uint32_t)ca >> 1) ^ order)) = make_uint4(xa.x, xa.y, xb.x, xb.y);
        } else {
            *reinterpret_cast<uint2 *>(codes + 16 * (((uint32_t)ca >> 1) ^ order) + 8 * (ca & 1)) = xa;
            *reinterpret_cast<uint2 *>(codes + 16 * (((uint32_t)cb >> 1) ^ order) + 8 * (cb & 1)) = xb;
        }
        if (j == 0) {
            const float scale = fine ? __fdiv_rn(amax, 127.0f) : top < 0x7f800000u ? 0.0f : __uint_as_float(0x7fc00000u);
            reinterpret_cast<float *>(record + 32 * c.dim)[(is_v ? 16 : 0) + row] = scale;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// quantized_cache_read
// ---------------------------------------------------------------------------------------------

// A thread restores one 16-byte chunk of a row; the rows of k and of v of a token are taken by the same CTA.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(const uint8_t *cache, CacheShape c, const void *slots, int slot_bytes, T *k, T *v, int64_t tokens,
                                                        int tokens_per_cta, unsigned int *status) {
    pdl_wait();
    pdl_launch_dependents();
    const int chunks = c.dim >> 4, units = 2 * c.kv_heads * chunks;
    const int64_t first = (int64_t)blockIdx.x * tokens_per_cta;
    const int n = (int)min((int64_t)tokens_per_cta, tokens - first) * units;
#pragma unroll 2
    for (int u = blockIdx.y * kThreads + threadIdx.x; u < n; u += gridDim.y * kThreads) {
        const int t = u / units, in_token = u - t * units;
        const int unit_row = in_token / chunks, chunk = in_token - unit_row * chunks;
        const bool is_v = unit_row >= c.kv_heads;
        const int h = is_v ? unit_row - c.kv_heads : unit_row;
        const int64_t token = first + t, slot = index_at(slots, slot_bytes, token);
        float lo[8], hi[8];
        if (slot < 0 || slot >= c.slots) {
            if (slot >= c.slots && in_token == 0 && status != nullptr) atomicOr(status, kBadSlot);
#pragma unroll
            for (int e = 0; e < 8; ++e) lo[e] = hi[e] = 0.0f;
        } else {
            uint32_t row;
            const uint8_t *record = record_of(const_cast<uint8_t *>(cache), c, slot, h, row);
            const uint32_t order = is_v ? v_order(row, c.dim) : k_order(row, c.dim);
            const uint4 x = *reinterpret_cast<const uint4 *>(record + (is_v ? 16 * c.dim : 0) + row * c.dim + 16 * ((uint32_t)chunk ^ order));
            const float scale = reinterpret_cast<const float *>(record + 32 * c.dim)[(is_v ? 16 : 0) + row];
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 16; ++e) {  // 2^23 + byte, exactly
                const float code = __uint_as_float(__byte_perm(w[e >> 2], 0x4b000000u, 0x7540u | (e & 3))) - (8388608.0f + 128.0f);
                (e < 8 ? lo[e & 7] : hi[e & 7]) = __fmul_rn(code, scale);
            }
        }
        T *y = (is_v ? v : k) + (token * c.kv_heads + h) * c.dim + 16 * chunk;
        store8<T, true>(y, narrow<T>(lo));
        store8<T, true>(y + 8, narrow<T>(hi));
    }
}

// Tokens a CTA takes, and CTAs a token, for `units` threads' work per token: one sweep of a CTA while the whole is less than what
// runs at once, about four beyond.
void spread(int64_t tokens, int64_t units, int &tokens_per_cta, dim3 &grid) {
    const int64_t at_once = (int64_t)sm_count() * 4 * kThreads;
    if (tokens * units <= at_once || units >= 4 * kThreads) {
        tokens_per_cta = 1;
        grid = dim3((unsigned)tokens, (unsigned)ceil_div(units, tokens * units <= at_once ? kThreads : 4 * kThreads), 1);
        return;
    }
    tokens_per_cta = (int)max((int64_t)1, 4 * kThreads / units);
    grid = dim3((unsigned)ceil_div(tokens, tokens_per_cta), 1, 1);
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
    if (pages > 0 && (cache == nullptr || !aligned_to(cache, 16))) return set_error(B200Q_INVALID_ARGUMENT, "%s: the cache must be 16-byte aligned, got %p", op, cache);
    return B200Q_OK;
}

template <typename T>
int rotary_typed(const HeadRows &q, const HeadRows &k, const HeadRows &q_out, const HeadRows &k_out, const RotaryArgs &r, int64_t tokens, int heads, int kv_heads, int dim,
                 cudaStream_t stream) {
    const int all = heads + kv_heads;
    if (dim % 16 == 0 && r.rotary_dim % 16 == 0 && (int64_t)all * dim < (1 << 24)) {
        const size_t s = sizeof(T);
        const bool vec = rows_aligned(q, s) && rows_aligned(q_out, s) && rows_aligned(k, s) && rows_aligned(k_out, s) && aligned_to(r.table, 16);
        int per_cta;
        dim3 grid;
        spread(tokens, (int64_t)all * (dim / 16), per_cta, grid);
        auto kernel = vec ? rotary_kernel<T, true> : rotary_kernel<T, false>;
        return launch_after("rotary_kernel", kernel, grid, kThreads, 0, 1, stream, q, k, q_out, k_out, r, tokens, heads, all, dim, per_cta);
    }
    const int64_t ctas = ceil_div(tokens * all * (dim - r.rotary_dim / 2), kThreads);
    return launch_after("rotary_generic_kernel", rotary_generic_kernel<T>, dim3((unsigned)(ctas < 65536 ? ctas : 65536)), kThreads, 0, 1, stream, q, k, q_out, k_out, r, tokens, heads,
                        all, dim);
}

template <typename T, bool VEC>
int append_sized(const HeadRows &q, const HeadRows &q_out, const HeadRows &k, const HeadRows &v, uint8_t *cache, const CacheShape &c, const void *slots, int slot_bytes,
                 const RotaryArgs &r, int64_t tokens, int heads, cudaStream_t stream) {
    const int group = c.dim <= 64 ? 4 : c.dim <= 128 ? 8 : 16;
    int per_cta;
    dim3 grid;
    spread(tokens, (int64_t)(heads + 2 * c.kv_heads) * group, per_cta, grid);
    auto kernel = group == 4 ? append_kernel<T, VEC, 4> : group == 8 ? append_kernel<T, VEC, 8> : append_kernel<T, VEC, 16>;
    return launch_after("append_kernel", kernel, grid, kThreads, 0, 1, stream, q, q_out, k, v, cache, c, slots, slot_bytes, r, tokens, heads, per_cta);
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
    int per_cta;
    dim3 grid;
    spread(tokens, (int64_t)2 * c.kv_heads * (c.dim / 16), per_cta, grid);
    return launch_after("read_kernel", read_kernel<T>, grid, kThreads, 0, 1, stream, cache, c, slots, slot_bytes, static_cast<T *>(k), static_cast<T *>(v), tokens, per_cta,
                        device_status_word());
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
    const CacheShape c = {pages, pages * page_size, (int)page_size, (int)kv_heads, (int)head_dim};
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
    const CacheShape c = {pages, pages * page_size, (int)page_size, (int)kv_heads, (int)head_dim};
    const uint8_t *bytes = static_cast<const uint8_t *>(cache);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (type) {
        case B200Q_F16: return read_typed<__half>(bytes, c, slots, slot_bytes, k, v, tokens, s);
        case B200Q_BF16: return read_typed<__nv_bfloat16>(bytes, c, slots, slot_bytes, k, v, tokens, s);
        default: return read_typed<float>(bytes, c, slots, slot_bytes, k, v, tokens, s);
    }
}

}  // extern "C"
