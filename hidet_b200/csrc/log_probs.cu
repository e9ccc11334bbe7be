// Log probabilities of given tokens, the entropy of every row and its top alternatives, in one pass over the logits.
//
//     m = max x,  S = sum exp(x - m),  lse = m + log S
//     log p(token) = x[token] - lse,   H = -sum p log p = log S - sum (x - m) exp(x - m) / S
// in float.  The top alternatives are the largest logits, equal ones by their index.  A row with a NaN or +inf, or with nothing above -inf, has no
// distribution: its values are NaN.
//
// A row, or with few or long rows a part of one, is brought into a CTA's shared memory by one bulk copy (the bytes in front of its first and
// behind its last 16-byte boundary by loads) and read from there twice: for the maximum of every thread, and for the sums.  CTAs of a row are a cluster and meet in the shared memory of the first.
//
// Measured: 2047 rows of 32002 bf16 logits with 20 alternatives 41 us, 3.2 TB/s (without alternatives 30); 2476 of 6842 with 5: 21.3; one row 6.0; float32, 1000 rows of 32000: 44.6, 2.9 TB/s.  A copy at
// memory's rate would take 20 us, and the instructions, 12 an element, 22: what is above that is that a row's steps (copy, maxima, bound, sums, alternatives) wait for one another, and with three rows an SM, all that fits its
// shared memory, half of the issue slots stay empty.  More threads a row, parts of half the size (two CTAs a row: 83 us) and candidates sought outside
// the sums' loop (43 to 50 us) are slower.  Five CTAs an SM, where shared memory lets them, want 48 registers, for which loops are unrolled by two and four: with three
// and 78 registers rows of 6842 took 28.5 us and long rows as long as now; with six and 40, 20.4, and long rows 1 to 2 % more.
//
// The maxima of 64 groups of threads bound the alternatives: at least `top` elements are no smaller than the top-th largest of them.  So what the second
// reading passes over is compared with that bound, eight elements at once, and the few that reach it (some 1.2 * top on random rows) are put
// in order by counting.  Where that is too many, mostly equals of the bound, only the first of those are taken; what is left (rows made so, and vocabularies of fewer
// elements than the groups need) has a search for each alternative.
#include <atomic>

#include "serving.cuh"

namespace b200q {
namespace {

constexpr unsigned int kKernelLogProbs = 8;
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int GROUPS = 64;               // four lanes of a warp each
constexpr int MOST_TOP = 32;
constexpr int MOST_CLUSTER = 8;
constexpr int CANDIDATES = 512;
constexpr int kMostPart = 200 * 1024;    // bytes of a row in one CTA
constexpr int kGoodPart = 66 * 1024;     // three CTAs an SM
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// A value as a whole number in its order: NaN is the largest, -0 is 0; none is 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0xffffffffu : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
// A value and the place it stands at as one number: larger values first, then smaller places.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t place) {
    return ((uint64_t)ordered(x) << 32) | (0xffffffffu - place);
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return o == 0xffffffffu ? __uint_as_float(0x7fc00000u) : __uint_as_float((o >> 31) ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint32_t place_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 16 bytes of logits.  pairs: as floats, none below a finite number, whose probability is zero beside a maximum of at least kLeast, so that this times it is zero
// as well; for a maximum of at most kMost its distance, in log2, is finite too.
template <typename T>
struct Vec16;
template <>
struct Vec16<float> {
    static constexpr int N = 4;
    static constexpr float kLeast = -1e29f, kMost = 1e38f;
    static __device__ __forceinline__ void widen(uint4 v, float (&f)[4]) { f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w); }
    static __device__ __forceinline__ void pairs(uint4 v, f32x2 (&p)[2]) {
        float f[4];
        widen(v, f);
        p[0] = pair_of(fmaxf(f[0], -1e30f), fmaxf(f[1], -1e30f)), p[1] = pair_of(fmaxf(f[2], -1e30f), fmaxf(f[3], -1e30f));
    }
    typedef float Top;
    static __device__ __forceinline__ Top all(float x) { return x; }
    static __device__ __forceinline__ Top top(uint4 v) {
        float f[4];
        widen(v, f);
        return max_nan(max_nan(f[0], f[1]), max_nan(f[2], f[3]));
    }
    static __device__ __forceinline__ Top larger(Top a, Top b) { return max_nan(a, b); }
    static __device__ __forceinline__ float value(Top t) { return t; }
    static __device__ __forceinline__ bool below(Top t, Top bound) { return t < bound; }
};
template <>
struct Vec16<__half> {
    static constexpr int N = 8;
    static constexpr float kLeast = -65504.0f + 256.0f, kMost = 65504.0f;
    static __device__ __forceinline__ __half2 h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
    static __device__ __forceinline__ void widen(uint4 v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = __half22float2(h2(w[i]));
            f[2 * i] = p.x, f[2 * i + 1] = p.y;
        }
    }
    static __device__ __forceinline__ void pairs(uint4 v, f32x2 (&p)[4]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(__hmax2(h2(w[i]), __float2half2_rn(-65504.0f)));
            p[i] = pair_of(f.x, f.y);
        }
    }
    typedef __half2 Top;  // of the elements at even and at odd places
    static __device__ __forceinline__ Top all(float x) { return __float2half2_rn(x); }
    static __device__ __forceinline__ Top top(uint4 v) { return __hmax2_nan(__hmax2_nan(h2(v.x), h2(v.y)), __hmax2_nan(h2(v.z), h2(v.w))); }
    static __device__ __forceinline__ Top larger(Top a, Top b) { return __hmax2_nan(a, b); }
    static __device__ __forceinline__ float value(Top t) { return max_nan(__low2float(t), __high2float(t)); }
    static __device__ __forceinline__ bool below(Top t, Top bound) { return __hblt2(t, bound); }  // both
};
template <>
struct Vec16<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr float kLeast = -1e29f, kMost = 1e38f;
    static __device__ __forceinline__ __nv_bfloat162 b2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162 *>(&u); }
    static __device__ __forceinline__ void widen(uint4 v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    static __device__ __forceinline__ void pairs(uint4 v, f32x2 (&p)[4]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __hmax2(b2(w[i]), __float2bfloat162_rn(-1e30f));
            const uint32_t u = *reinterpret_cast<const uint32_t *>(&b);
            p[i] = pair_of(u << 16, u & 0xffff0000u);
        }
    }
    typedef __nv_bfloat162 Top;  // of the elements at even and at odd places
    static __device__ __forceinline__ Top all(float x) { return __float2bfloat162_rn(x); }
    static __device__ __forceinline__ Top top(uint4 v) { return __hmax2_nan(__hmax2_nan(b2(v.x), b2(v.y)), __hmax2_nan(b2(v.z), b2(v.w))); }
    static __device__ __forceinline__ Top larger(Top a, Top b) { return __hmax2_nan(a, b); }
    static __device__ __forceinline__ float value(Top t) { return max_nan(__low2float(t), __high2float(t)); }
    static __device__ __forceinline__ bool below(Top t, Top bound) { return __hblt2(t, bound); }  // both
};
template <typename T>
__device__ __forceinline__ T minus_infinity() { return Elems<T>::round(-INFINITY); }

struct LogProbsArgs {
    const void *logits;
    int64_t row_stride;
    const void *tokens;
    int token_bytes;
    int64_t given;
    float *log_probs, *entropy, *top_log_probs;
    int64_t *top_indices;
    int64_t vocab;
    int64_t part;  // elements of a row that a CTA takes
    int top;
    unsigned int *status;
};

// What a CTA of the cluster tells the first: its maximum, its sums, its best keys.
struct Share {
    float m, sum, weighted;
    uint64_t best[MOST_TOP];
};

struct Block {
    uint64_t bar;
    float m[WARPS], sum[WARPS], weighted[WARPS];
    uint32_t group_top[GROUPS], bound;
    int equals[WARPS];
    uint64_t warp_key[WARPS];
    uint64_t best[MOST_TOP];
    int n_candidates, n_vectors;
    uint16_t vectors[CANDIDATES];  // that hold candidates
    uint64_t candidates[CANDIDATES];
    Share shares[MOST_CLUSTER];
};
static_assert(sizeof(Block) <= 8704 && CANDIDATES >= MOST_CLUSTER * MOST_TOP && THREADS == 4 * GROUPS, "");

// Puts the n keys of `keys` in descending order; the first `top` go to `best` (0 where there are fewer).  All threads.
__device__ __forceinline__ void order_keys(const uint64_t *keys, int n, int top, uint64_t *best) {
    for (int i = threadIdx.x; i < top; i += THREADS)
        if (i >= n) best[i] = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint64_t own = keys[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += keys[j] > own || (keys[j] == own && j < i);
        if (rank < top) best[rank] = own;
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 5) log_probs_kernel(const LogProbsArgs p) {
    constexpr int N = Vec16<T>::N;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Block blk;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cluster_ctarank(), ranks = cluster_nctarank();
    const int64_t row = blockIdx.x / ranks;
    const uint32_t bar = smem_u32(&blk.bar);
    if (threadIdx.x == 0) {
        mbar_init(bar, 1);
        mbar_fence_init();
        blk.n_candidates = blk.n_vectors = 0;
        blk.bound = 0;
    }
    if (ranks > 1) cluster_arrive_release();
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();

    // ---- this CTA's part of the row into shared memory, at the same place between two 16-byte boundaries ----
    const int64_t from = min(rank * p.part, p.vocab);
    const int n = (int)(min(from + p.part, p.vocab) - from);
    const T *src = static_cast<const T *>(p.logits) + row * p.row_stride + from;
    const int lead = (int)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));  // elements between the boundary in front and the first
    const int vecs = (lead + n + N - 1) / N;
    const int whole_first = lead > 0 ? 1 : 0, whole_end = (lead + n) / N;           // vectors that lie in the part entirely
    T *buf = reinterpret_cast<T *>(smem);
    if (threadIdx.x == 0) {
        const int bytes = whole_end > whole_first ? (whole_end - whole_first) * 16 : 0;
        if (bytes > 0) {
            mbar_expect_tx(bar, (uint32_t)bytes);
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem) + whole_first * 16), "l"(src - lead + whole_first * N),
                         "r"(bytes), "r"(bar)
                         : "memory");
        } else {
            mbar_arrive(bar);
        }
    }
    if (threadIdx.x >= 32 && threadIdx.x < 32 + 2 * N) {  // the first and the last vector, if they are not whole
        const int e = threadIdx.x - 32, v = e < N ? 0 : vecs - 1;
        const bool ragged = vecs > 0 && (e < N ? whole_first == 1 : whole_end < vecs && !(v == 0 && whole_first == 1));
        const int i = v * N + e % N - lead;
        if (ragged) buf[v * N + e % N] = i >= 0 && i < n ? src[i] : minus_infinity<T>();
    }
    // the given tokens' logits, by the first CTA
    float own_logit = 0.0f;
    bool inside = true;
    if (rank == 0 && threadIdx.x < p.given) {
        const int64_t token = index_at(p.tokens, p.token_bytes, row * p.given + threadIdx.x);
        inside = token >= 0 && token < p.vocab;
        own_logit = inside ? Elems<T>::one(static_cast<const T *>(p.logits)[row * p.row_stride + token]) : -INFINITY;
    }
    __syncthreads();
    if (!mbar_wait(bar, 0)) {
        if (threadIdx.x == 0) report_timeout(p.status, kKernelLogProbs, 1);
        mbar_wait(bar, 0);
    }
    const uint4 *x = reinterpret_cast<const uint4 *>(smem);

    // ---- the maximum of every thread ----
    using V = Vec16<T>;
    typename V::Top tops = V::all(-INFINITY);
#pragma unroll 4
    for (int v = threadIdx.x; v < vecs; v += THREADS) tops = V::larger(tops, V::top(x[v]));
    float m = V::value(tops);
    uint32_t group = (int)threadIdx.x < vecs ? ordered(m) : 0;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (lane == 0) blk.m[warp] = m;
    if (p.top > 0) {
#pragma unroll
        for (int d = 8; d < 32; d *= 2) group = max(group, __shfl_xor_sync(0xffffffffu, group, d));
        if (lane < 8) blk.group_top[8 * warp + lane] = group;
    }
    __syncthreads();
    m = blk.m[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) m = max_nan(m, blk.m[w]);
    uint32_t bound = 0;
    if (p.top > 0) {  // the top-th largest of the groups': four threads compare one with all
        const int g = threadIdx.x / 4;
        const uint32_t own = blk.group_top[g];
        int before = 0;
#pragma unroll
        for (int i = 0; i < GROUPS / 4; ++i) {
            const int j = 4 * i + threadIdx.x % 4;
            const uint32_t k = blk.group_top[j];
            before += k > own || (k == own && j < g);
        }
        before += __shfl_xor_sync(0xffffffffu, before, 1);
        before += __shfl_xor_sync(0xffffffffu, before, 2);
        if (before == p.top - 1 && threadIdx.x % 4 == 0) blk.bound = own;
        __syncthreads();
        bound = blk.bound;
    }
    // With fewer groups than alternatives there is no bound, and nothing is collected.
    const bool collect = bound != 0;
    const float least = collect ? value_of((uint64_t)bound << 32) : INFINITY;
    const typename V::Top least_of_all = V::all(least);

    // ---- the sums ----
    const float shift = fabsf(m) < INFINITY ? m : 0.0f;
    float sum = 0.0f, weighted = 0.0f;
    // Which of this thread's vectors reach the bound, the last in bit 0: with a branch for each, which few take, the loop's loads and arithmetic could not overlap.
    uint64_t hits = 0;
    static_assert(kMostPart / 16 / THREADS < 63, "");
    if ((m >= V::kLeast && m <= V::kMost) || !(fabsf(m) < INFINITY)) {
        const f32x2 minus = pair_of(-shift, -shift), log2e = pair_of(kLog2e, kLog2e);
        f32x2 sums = 0, products = 0;
#pragma unroll 2
        for (int v = threadIdx.x; v < vecs; v += THREADS) {
            f32x2 f[N / 2];
            const uint4 raw = x[v];
            hits = hits << 1 | (V::below(V::top(raw), least_of_all) ? 0 : 1);  // NaN is a hit too
            Vec16<T>::pairs(raw, f);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                const f32x2 y = mul2(add2(f[e], minus), log2e);  // zero for the largest
                float lo, hi;
                halves(y, lo, hi);
                asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(lo));
                asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(hi));
                const f32x2 z = pair_of(lo, hi);
                sums = add2(sums, z);
                products = fma2(z, y, products);
            }
        }
        float lo, hi;
        halves(sums, lo, hi);
        sum = lo + hi;
        halves(products, lo, hi);
        weighted = lo + hi;
    } else {
        // Nothing but numbers around the type's lowest, which stand for what is not allowed, and -inf: the two differ here.  Or a maximum so large that a distance from
        // it may be -inf.
        for (int v = threadIdx.x; v < vecs; v += THREADS) {
            float f[N];
            const uint4 raw = x[v];
            hits = hits << 1 | (V::below(V::top(raw), least_of_all) ? 0 : 1);
            V::widen(raw, f);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float y = (f[e] - shift) * kLog2e, z = exp2f(y);
                sum += z;
                weighted += z > 0.0f ? z * y : 0.0f;
            }
        }
    }
    if (collect) {
        const int last = (int)threadIdx.x + (vecs - 1 - (int)threadIdx.x) / THREADS * THREADS;  // this thread's, if it has any
        for (; hits != 0; hits &= hits - 1) {
            const int k = atomicAdd(&blk.n_vectors, 1);
            if (k < CANDIDATES) blk.vectors[k] = (uint16_t)(last - (__ffsll((long long)hits) - 1) * THREADS);
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        weighted += __shfl_xor_sync(0xffffffffu, weighted, d);
    }
    if (lane == 0) blk.sum[warp] = sum, blk.weighted[warp] = weighted;

    // ---- this part's best ----
    Share &mine = blk.shares[0];
    __syncthreads();
    if (p.top > 0) {
        // Elements of a vector that pass the bound, or (ties) that are equal to it.
        auto offer = [&](int v, bool ties) {
            float f[N];
            V::widen(x[v], f);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int index = v * N + e - lead;
                if (index < 0 || index >= n || (ties ? ordered(f[e]) != bound : ordered(f[e]) <= bound)) continue;
                const int k = atomicAdd(&blk.n_candidates, 1);
                if (k < CANDIDATES) blk.candidates[k] = key_of(f[e], (uint32_t)(from + index));
            }
        };
        bool listed = collect;
        if (collect && blk.n_vectors <= CANDIDATES) {
            for (int i = threadIdx.x; i < blk.n_vectors * N; i += THREADS) {  // a thread an element
                const int at = blk.vectors[i / N] * N + i % N, index = at - lead;
                const float one = Elems<T>::one(buf[at]);
                if (index < 0 || index >= n || ordered(one) < bound) continue;
                const int k = atomicAdd(&blk.n_candidates, 1);
                if (k < CANDIDATES) blk.candidates[k] = key_of(one, (uint32_t)(from + index));
            }
            __syncthreads();
        } else if (collect) {
            // Too many: mostly equals of the bound (a row of one value, or whose allowed tokens are fewer than the alternatives).  Those above it, and
            // then the first of its equals, as many as are wanted.
            for (int v = threadIdx.x; v < vecs; v += THREADS) offer(v, false);
            __syncthreads();
            const int above = blk.n_candidates;
            for (int base = 0, equals = 0; base < vecs && above < p.top && equals < p.top - above; base += THREADS) {
                const int v = base + threadIdx.x;
                int own = 0;
                if (v < vecs) {
                    float f[N];
                    V::widen(x[v], f);
#pragma unroll
                    for (int e = 0; e < N; ++e) own += v * N + e >= lead && v * N + e - lead < n && ordered(f[e]) == bound;
                }
                int until = own;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int below = __shfl_up_sync(0xffffffffu, until, d);
                    if (lane >= d) until += below;
                }
                if (lane == 31) blk.equals[warp] = until;
                __syncthreads();
                int in_front = equals + until - own, all = 0;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    if (w < warp) in_front += blk.equals[w];
                    all += blk.equals[w];
                }
                if (own > 0 && in_front < p.top - above) offer(v, true);
                equals += all;
                __syncthreads();
            }
        }
        listed = listed && blk.n_candidates <= CANDIDATES;
        if (listed) {
            order_keys(blk.candidates, blk.n_candidates, p.top, mine.best);
        } else {
            uint64_t last = ~0ull;
            for (int k = 0; k < p.top; ++k) {
                uint64_t best = 0;
                for (int v = threadIdx.x; v < vecs; v += THREADS) {
                    float f[N];
                    Vec16<T>::widen(x[v], f);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const int index = v * N + e - lead;
                        const uint64_t key = index >= 0 && index < n ? key_of(f[e], (uint32_t)(from + index)) : 0;
                        if (key < last && key > best) best = key;
                    }
                }
#pragma unroll
                for (int d = 16; d > 0; d /= 2) {
                    const uint64_t other = __shfl_xor_sync(0xffffffffu, best, d);
                    best = other > best ? other : best;
                }
                if (lane == 0) blk.warp_key[warp] = best;
                __syncthreads();
                last = 0;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) last = blk.warp_key[w] > last ? blk.warp_key[w] : last;
                if (threadIdx.x == 0) mine.best[k] = last;
                __syncthreads();
            }
        }
    }
    float part_sum = 0.0f, part_weighted = 0.0f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) part_sum += blk.sum[i], part_weighted += blk.weighted[i];
    if (ranks > 1 && threadIdx.x == 0) {
        mine.m = m;
        mine.sum = part_sum;
        mine.weighted = part_weighted;
    }
    __syncthreads();

    // ---- the parts of a row meet in the first CTA ----
    if (ranks > 1) {
        cluster_wait_acquire();  // every CTA of the cluster runs
        if (rank > 0) {
            constexpr int WORDS = sizeof(Share) / 4;
            const uint32_t dst = map_to_rank(smem_u32(&blk.shares[rank]), 0);
            for (int i = threadIdx.x; i < WORDS; i += THREADS)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + 4 * i), "r"(reinterpret_cast<const uint32_t *>(&mine)[i]) : "memory");
        }
        __syncwarp();
        cluster_arrive_release();
        cluster_wait_acquire();
        if (rank > 0) return;
    }
    float all_m = m, all_sum = part_sum, all_weighted = part_weighted;  // the latter of (x - all_m) log2(e)
    if (ranks > 1) {
        for (uint32_t r = 1; r < ranks; ++r) all_m = max_nan(all_m, blk.shares[r].m);
        all_sum = all_weighted = 0.0f;
        for (uint32_t r = 0; r < ranks; ++r) {
            const Share &s = blk.shares[r];
            if (!(fabsf(s.m) < INFINITY)) continue;  // nothing above -inf in it; +inf and NaN are told by all_m
            const float down = (s.m - all_m) * kLog2e, by = exp2f(down);
            all_sum = fmaf(s.sum, by, all_sum);
            all_weighted = fmaf(fmaf(s.sum, fmaxf(down, -200.0f), s.weighted), by, all_weighted);
        }
    }
    if (!(fabsf(all_m) < INFINITY)) all_sum = __uint_as_float(0x7fc00000u);
    const float log_sum = logf(all_sum), lse = all_m + log_sum;
    if (threadIdx.x == 0) p.entropy[row] = log_sum - all_weighted / all_sum * kLn2;
    for (int64_t i = threadIdx.x; i < p.given; i += THREADS) {
        if (i >= THREADS) {
            const int64_t token = index_at(p.tokens, p.token_bytes, row * p.given + i);
            inside = token >= 0 && token < p.vocab;
            own_logit = inside ? Elems<T>::one(static_cast<const T *>(p.logits)[row * p.row_stride + token]) : -INFINITY;
        }
        if (!inside && p.status != nullptr) atomicOr(p.status, kBadToken);
        p.log_probs[row * p.given + i] = own_logit - lse;
    }
    if (p.top > 0) {
        const uint64_t *best = blk.shares[0].best;
        if (ranks > 1) {
            uint64_t *keys = blk.candidates;
            for (int i = threadIdx.x; i < (int)ranks * p.top; i += THREADS) keys[i] = blk.shares[i / p.top].best[i % p.top];
            __syncthreads();
            order_keys(keys, (int)ranks * p.top, p.top, blk.best);
            __syncthreads();
            best = blk.best;
        }
        if (threadIdx.x < p.top) {
            const uint64_t key = best[threadIdx.x];
            p.top_log_probs[row * p.top + threadIdx.x] = value_of(key) - lse;
            p.top_indices[row * p.top + threadIdx.x] = (int64_t)place_of(key);
        }
    }
}

template <typename T>
int launch_typed(LogProbsArgs p, int64_t rows, cudaStream_t stream) {
    // The fewest CTAs a row whose parts let three of them share an SM; with few rows more, as long as parts have 8 KB and SMs are idle.
    const int64_t bytes = p.vocab * (int64_t)sizeof(T);
    int64_t ranks = ceil_div(bytes, kGoodPart) < MOST_CLUSTER ? ceil_div(bytes, kGoodPart) : MOST_CLUSTER;
    while (2 * ranks <= MOST_CLUSTER && rows * ranks * 2 <= sm_count() && bytes > ranks * 8192) ranks *= 2;
    p.part = round_up(ceil_div(p.vocab, ranks), 64);
    if (p.part * (int64_t)sizeof(T) > kMostPart) {
        return set_error(B200Q_UNSUPPORTED, "token_log_probs: rows of %lld bytes: up to %d are supported", (long long)bytes, MOST_CLUSTER * kMostPart);
    }
    if (rows > 2147483647LL / ranks) return set_error(B200Q_UNSUPPORTED, "token_log_probs: %lld rows", (long long)rows);
    const int smem = (int)(p.part * sizeof(T)) + 32;
    static std::atomic<bool> attr_set[64];
    const int rc = allow_smem(attr_set, log_probs_kernel<T>, kMostPart + 32);
    if (rc != B200Q_OK) return rc;
    return launch_after("log_probs_kernel", log_probs_kernel<T>, dim3((unsigned)(rows * ranks)), THREADS, smem, (int)ranks, stream, p);
}

}  // namespace
}  // namespace b200q

extern "C" {

B200Q_API int b200q_token_log_probs(const void *logits, int64_t row_stride, const void *tokens, float *log_probs, float *entropy, float *top_log_probs, int64_t *top_indices,
                                    int64_t rows, int64_t vocab, int64_t given, int64_t top, int type, int token_bytes, void *stream) {
    using namespace b200q;
    const char *op = "token_log_probs";
    if (rows < 0 || vocab < 0 || given < 0 || top < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative size", op);
    if (type < B200Q_F16 || type > B200Q_F32) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown float type %d", op, type);
    if (token_bytes != 4 && token_bytes != 8) return set_error(B200Q_INVALID_ARGUMENT, "%s: tokens must be int32 or int64 (4 or 8 bytes), got %d", op, token_bytes);
    if (rows == 0) return B200Q_OK;
    if (vocab == 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: a vocabulary of no tokens", op);
    if (top > MOST_TOP) return set_error(B200Q_UNSUPPORTED, "%s: %lld alternatives: up to %d are supported", op, (long long)top, MOST_TOP);
    if (top > vocab) return set_error(B200Q_INVALID_ARGUMENT, "%s: %lld alternatives of %lld tokens", op, (long long)top, (long long)vocab);
    if (row_stride < vocab && rows > 1) return set_error(B200Q_INVALID_ARGUMENT, "%s: rows of %lld elements %lld apart", op, (long long)vocab, (long long)row_stride);
    if (logits == nullptr || entropy == nullptr || (given > 0 && (tokens == nullptr || log_probs == nullptr)) || (top > 0 && (top_log_probs == nullptr || top_indices == nullptr))) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    }
    const LogProbsArgs p = {logits, row_stride, tokens, token_bytes, given, log_probs, entropy, top_log_probs, top_indices, vocab, 0, (int)top, device_status_word()};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (type) {
        case B200Q_F16: return launch_typed<__half>(p, rows, s);
        case B200Q_BF16: return launch_typed<__nv_bfloat16>(p, rows, s);
        default: return launch_typed<float>(p, rows, s);
    }
}

}  // extern "C"
