// A layer of experts over a few tokens as two streams of int8 weights: gate and up, and down.  Inference at batch sizes where the weights of the experts that have
// a token are all there is to read.
//
// Both kernels are the same machine.  Every CTA makes the list of entries, an expert with up to 8 G of its assignments (an expert with more has several), and takes an
// equal, contiguous part of all their units: 32 rows of an entry's weight over all of K (gate and up), or over a part of it (down).  A copying warp streams the
// unit's tiles, 32 rows x 512 k, through a ring; eight warps have 64 k of a tile each:
//     weights  a lane's 16 neighbouring k of a row in one load, int8 -> exact f16, the 16-row operand of mma.sync
//     tokens   a lane's same 16 k of its column's token from global memory (they stay in L1), -> f16, the 8-column operand
//     sums     float, of the eight warps added in shared memory, in their order
// With one to eight tokens an expert the product is a stream, so what tcgen05 would add is not needed and its 128 lanes would stand mostly empty; the conversions take about a
// third of the issue slots at memory's rate.
// Gate and up: h = silu(g) u in float to global memory, and its largest magnitude per assignment.  Down: h is scaled by a power of two from that, so that f16 holds it
// whatever the range (as tokens in bf16 are, by their own largest), and a unit's sums, times scale and weight, are a piece of every assignment's result.  The
// CTA that brings a column tile's last piece adds them up, token by token, assignments and parts of K in their order: the result does not depend on who came when.
//
// Down starts while gate and up run: its CTAs fill their rings with weights and wait there for h.
//
// Waits are bounded: one that runs out is reported and raises a flag, after which nobody in the CTA waits or copies any more; everyone goes through the motions
// to the end, so that no barrier is left alone.
#include "experts.h"
#include "serving.cuh"
#include "umma.cuh"

namespace b200q {
namespace {

constexpr unsigned int kKernelExperts = 11;
constexpr int ROWS = 32;                  // of a unit
constexpr int BOX_K = 128;                // one copy: 32 rows x 128 k, rows of 128 swizzled bytes
constexpr int BOXES = 4, STAGE_K = BOX_K * BOXES;
constexpr int BOX_BYTES = ROWS * BOX_K, STAGE_BYTES = BOX_BYTES * BOXES;
constexpr int MATH_WARPS = 8, MATH_THREADS = 32 * MATH_WARPS, COPY_WARP = MATH_WARPS, FINISH_WARPS = 3;
constexpr int WARP_K = STAGE_K / MATH_WARPS;
constexpr int UP_THREADS = MATH_THREADS + 32, DOWN_THREADS = UP_THREADS + 32 * FINISH_WARPS;
constexpr int MOST_STAGES = 6;
constexpr int MOST_ASSIGNMENTS = 2048;    // of one launch
constexpr int MOST_EXPERTS = 1024;
// what of the workspace's counters is whose
constexpr int COUNTER_TILES = 32768, COUNTER_DONE = COUNTER_TILES, COUNTER_MAX = COUNTER_TILES + 1;

struct StreamArgs {
    ExpertsArgs a;
    float *h;             // [assignments, inner]
    float *pieces;        // [parts][assignments, hidden]
    unsigned int *counters;
    int tiles;            // of 32 rows, of an expert's weight
    int parts, part_k;    // of K (down); part_k a multiple of STAGE_K unless there is one part
    int stages;
};

struct Entry {
    int expert, first, count;  // its assignments are order[first ..]
};

__device__ __forceinline__ float scale_at(const void *p, int type, int64_t i) {
    if (type == B200Q_F16) return __half2float(static_cast<const __half *>(p)[i]);
    if (type == B200Q_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return static_cast<const float *>(p)[i];
}

// The power of two that brings a largest magnitude (as bits) to 2^14 .. 2^15, and its inverse; one for zero, infinity and NaN.
__device__ __forceinline__ float power_for(uint32_t bits, float &inverse) {
    int e = 141 - (int)(bits >> 23);  // 127 + 14 - exponent
    e = bits == 0 || bits >= 0x7f800000u ? 0 : max(-120, min(120, e));
    inverse = __uint_as_float((uint32_t)(127 - e) << 23);
    return __uint_as_float((uint32_t)(127 + e) << 23);
}

// 16 neighbouring elements of a token as eight f16 pairs.
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
struct FromF16 {
    typedef uint4 Raw[2];
    static __device__ __forceinline__ void load(const void *row, int64_t k, Raw &r) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const __half *>(row) + k);
        r[0] = p[0], r[1] = p[1];
    }
    static __device__ __forceinline__ void convert(const Raw &r, float, uint32_t (&b)[8]) {
        b[0] = r[0].x, b[1] = r[0].y, b[2] = r[0].z, b[3] = r[0].w, b[4] = r[1].x, b[5] = r[1].y, b[6] = r[1].z, b[7] = r[1].w;
    }
};
struct FromBF16 {
    typedef uint4 Raw[2];
    static __device__ __forceinline__ void load(const void *row, int64_t k, Raw &r) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(row) + k);
        r[0] = p[0], r[1] = p[1];
    }
    static __device__ __forceinline__ void convert(const Raw &r, float by, uint32_t (&b)[8]) {
        const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[1].x, r[1].y, r[1].z, r[1].w};
        const f32x2 by2 = pair_of(by, by);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float lo, hi;
            halves(mul2(pair_of(w[i] << 16, w[i] & 0xffff0000u), by2), lo, hi);
            b[i] = pack_f16(lo, hi);
        }
    }
};
struct FromF32 {
    typedef float4 Raw[4];
    static __device__ __forceinline__ void load(const void *row, int64_t k, Raw &r) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(row) + k);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = p[i];
    }
    static __device__ __forceinline__ void convert(const Raw &r, float by, uint32_t (&b)[8]) {
        const f32x2 by2 = pair_of(by, by);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo, hi;
            halves(mul2(pair_of(r[i].x, r[i].y), by2), lo, hi);
            b[2 * i] = pack_f16(lo, hi);
            halves(mul2(pair_of(r[i].z, r[i].w), by2), lo, hi);
            b[2 * i + 1] = pack_f16(lo, hi);
        }
    }
};

template <int G>
struct Shared {
    uint64_t full[MOST_STAGES], empty[MOST_STAGES];
    uint64_t ready[2], freed[2];          // (down) a unit's pieces are in memory; its finishing is over
    int abort_flag, entries, last;
    float by[2][8 * G], back[2][8 * G];   // powers of two of the columns' tokens, of this entry and the next
    alignas(16) float sums[MATH_WARPS][ROWS][8 * G + 2];
    int counts[MOST_EXPERTS];
    uint16_t chosen[MOST_ASSIGNMENTS];    // the expert of every assignment, or kNone
    uint16_t order[MOST_ASSIGNMENTS];     // assignments, by expert
    Entry entry[1];                       // as many as there are
};

// The entries of a launch: counts by expert, a scan over the experts, assignments in their places.  Every CTA makes them for itself, so an expert's assignments stand in
// their own order: as they come they would differ from CTA to CTA, and with them who is in which entry of an expert with several.
constexpr uint16_t kNone = 0xffff;
template <int G>
__device__ void make_entries(const ExpertsArgs &a, Shared<G> &s, int threads) {
    const int n = a.tokens * a.top;
    for (int e = threadIdx.x; e < a.count; e += threads) s.counts[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += threads) {
        const int e = __ldcg(a.experts + i);
        const bool there = e >= 0 && e < a.count;
        s.chosen[i] = there ? (uint16_t)e : kNone;
        if (there) atomicAdd(&s.counts[e], 1);
        else if (e >= 0 && blockIdx.x == 0 && a.status != nullptr) atomicOr(a.status, kBadExpert);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        int first = 0, entries = 0;  // assignments and entries of the experts so far
        for (int e0 = 0; e0 < a.count; e0 += 32) {
            const int e = e0 + threadIdx.x, mine = e < a.count ? s.counts[e] : 0, my_entries = (mine + 8 * G - 1) / (8 * G);
            int at = mine, at_entry = my_entries;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, at, o), y = __shfl_up_sync(0xffffffffu, at_entry, o);
                if ((int)threadIdx.x >= o) at += x, at_entry += y;
            }
            for (int i = 0; i < my_entries; ++i) s.entry[entries + at_entry - my_entries + i] = {e, first + at - mine + i * 8 * G, min(8 * G, mine - i * 8 * G)};
            if (e < a.count) s.counts[e] = first + at - mine;
            first += __shfl_sync(0xffffffffu, at, 31), entries += __shfl_sync(0xffffffffu, at_entry, 31);
        }
        if (threadIdx.x == 0) s.entries = entries;
        __syncwarp();
        for (int i0 = 0; i0 < n; i0 += 32) {
            const int i = i0 + threadIdx.x;
            const uint32_t e = i < n ? s.chosen[i] : kNone, same = __match_any_sync(0xffffffffu, e);
            const int place = e != kNone ? s.counts[e] : 0;
            __syncwarp();
            if (e != kNone) {
                s.order[place + __popc(same & ((1u << threadIdx.x) - 1u))] = (uint16_t)i;
                if ((same >> threadIdx.x) == 1u) s.counts[e] = place + __popc(same);  // the last of them
            }
            __syncwarp();
        }
    }
    __syncthreads();
}

__device__ __forceinline__ float token_value(const void *p, int type, int64_t i) {
    return type == B200Q_F16 ? __half2float(static_cast<const __half *>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_result(const ExpertsArgs &a, int t, int n, float v) {
    if (a.residual != nullptr) v += token_value(a.residual, a.type, t * a.residual_stride + n);
    const int64_t at = (int64_t)t * a.hidden + n;
    if (a.type == B200Q_F16) static_cast<__half *>(a.out)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
}

// X: what the tokens are; DOWN: h, else x.
template <int G, bool DOWN, typename X>
__global__ void __launch_bounds__(DOWN ? DOWN_THREADS : UP_THREADS, 1) experts_stream_kernel(const __grid_constant__ CUtensorMap map_w, const StreamArgs p) {
    extern __shared__ unsigned char smem_dyn[];
    const uint32_t ring = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char *ring_gen = smem_dyn + (ring - smem_u32(smem_dyn));
    Shared<G> &s = *reinterpret_cast<Shared<G> *>(ring_gen + p.stages * STAGE_BYTES);
    const ExpertsArgs &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int THREADS = DOWN ? DOWN_THREADS : UP_THREADS;
    constexpr int AHEAD = G < 2 ? G : 2;  // groups of columns whose tokens are on their way
    const uint32_t stages = p.stages;
    const int K = DOWN ? a.inner : a.hidden;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < stages; ++i) {
            mbar_init(smem_u32(&s.full[i]), 1);
            mbar_init(smem_u32(&s.empty[i]), MATH_WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s.ready[i]), MATH_WARPS);
            mbar_init(smem_u32(&s.freed[i]), 1);
        }
        s.abort_flag = 0;
        mbar_fence_init();
    }
    // The experts were chosen in front of gate and up, which waits for that before it lets down start: down may read them, and request weights, without waiting.
    if (!DOWN) pdl_wait();
    make_entries<G>(a, s, THREADS);
    pdl_launch_dependents();
    const int per_entry = p.tiles * p.parts;
    const int64_t units = (int64_t)s.entries * per_entry;
    const int64_t u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;

    auto wait = [&](uint64_t *bar, uint32_t parity, unsigned int site) {
        const uint32_t b = smem_u32(bar);
        for (uint32_t i = 0; i < kSpinLimit; ++i) {
            if (mbar_try_wait(b, parity)) return;
            if ((i & 15u) == 15u && *reinterpret_cast<volatile int *>(&s.abort_flag) != 0) return;
        }
        report_timeout(a.status, kKernelExperts, site);
        atomicExch(&s.abort_flag, 1);
    };
    auto k_of = [&](int64_t u, int &k0, int &k1, int &tile, int &entry) {
        entry = (int)(u / per_entry);
        const int r = (int)(u - (int64_t)entry * per_entry), part = r / p.tiles;
        tile = r - part * p.tiles;
        k0 = part * p.part_k, k1 = min(K, k0 + p.part_k);
    };

    if (warp == COPY_WARP) {
        // ---------------- the stream of weights ----------------
        if (lane == 0) {
            const uint64_t once = l2_policy_evict_first();
            umma::Ring r;
            uint32_t i = 0;
            bool ok = true;
            for (int64_t u = u0; u < u1 && ok; ++u) {
                int k0, k1, tile, entry;
                k_of(u, k0, k1, tile, entry);
                const int row = s.entry[entry].expert * (DOWN ? a.hidden : 2 * a.inner) + tile * ROWS;
                for (int k = k0; k < k1; k += STAGE_K, ++i, r.advance(1, stages)) {
                    if (i >= stages) wait(&s.empty[r.slot], r.phase ^ 1u, 1);
                    if (*reinterpret_cast<volatile int *>(&s.abort_flag) != 0) {
                        ok = false;
                        break;
                    }
                    const int boxes = min(BOXES, (k1 - k + BOX_K - 1) / BOX_K);
                    const uint32_t bar = smem_u32(&s.full[r.slot]), at = ring + r.slot * STAGE_BYTES;
                    mbar_expect_tx(bar, boxes * BOX_BYTES);
                    for (int b = 0; b < boxes; ++b) tma_load_2d_hint(at + b * BOX_BYTES, &map_w, k + b * BOX_K, row, bar, once);
                }
            }
            // every copy armed has landed before the CTA may retire
            for (uint32_t t = 0; t < stages; ++t) {
                if (i <= t) continue;
                const uint32_t j = i - 1 - (i - 1 - t) % stages;
                if (!mbar_wait(smem_u32(&s.full[t]), (j / stages) & 1)) report_timeout(a.status, kKernelExperts, 7);
            }
        }
        __syncwarp();
        if (DOWN) pdl_wait();
    } else if (warp < MATH_WARPS) {
        // ---------------- products ----------------
        if (DOWN) pdl_wait();  // h
        const int g = lane >> 2, t = lane & 3;
        // An eighth of a load's lanes reads two rows' four chunks: they lie in different banks where the rows are four apart (chunk c of row r stands at c ^ (r & 7)).
        const int row = (g >> 1) | ((g & 1) << 2);
        const int chunk = (warp & 1) * 4 + t;
        const uint32_t a_off = (uint32_t)(warp >> 1) * BOX_BYTES + row * BOX_K + ((uint32_t)(chunk ^ row) << 4);
        umma::Ring r;
        int now = -1, which = 0;
        Entry en = {0, 0, 0};
        const void *rows[G];
        float by[G];
        for (int64_t u = u0; u < u1; ++u) {
            int k0, k1, tile, entry;
            k_of(u, k0, k1, tile, entry);
            if (entry != now) {
                // ---- another expert: its tokens' rows, and the powers of two that they are scaled by ----
                now = entry, which ^= 1, en = s.entry[entry];
                for (int c = warp; c < 8 * G; c += MATH_WARPS) {
                    float inverse = 1.0f, power = 1.0f;
                    if (c < en.count) {
                        const int as = s.order[en.first + c];
                        uint32_t bits = 0;
                        if (DOWN) {
                            bits = __ldcg(p.counters + COUNTER_MAX + as);
                            power = power_for(bits, inverse);
                        } else if (a.type == B200Q_BF16) {
                            const uint4 *x = reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(a.x) + (int64_t)(as / a.top) * a.x_stride);
#pragma unroll 4
                            for (int i = lane; i < K / 8; i += 32) {
                                const uint4 v = x[i];
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int j = 0; j < 4; ++j) bits = max(bits, max(w[j] << 16 & 0x7fff0000u, w[j] & 0x7fff0000u));
                            }
                            power = power_for(__reduce_max_sync(0xffffffffu, bits), inverse);
                        }
                    }
                    if (lane == 0) s.by[which][c] = power, s.back[which][c] = inverse;
                }
                asm volatile("bar.sync 1, %0;" ::"n"(MATH_THREADS) : "memory");
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const int c = 8 * i + g, as = c < en.count ? s.order[en.first + c] : 0;
                    by[i] = s.by[which][c];
                    rows[i] = DOWN ? static_cast<const void *>(p.h + (int64_t)as * K) : static_cast<const void *>(static_cast<const uint16_t *>(a.x) + (int64_t)(as / a.top) * a.x_stride);
                }
            }
            float acc[2][G][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int l = 0; l < 4; ++l) acc[i][j][l] = 0.0f;
            for (int k = k0; k < k1; k += STAGE_K, r.advance(1, stages)) {
                const int64_t mine = k + warp * WARP_K + 16 * t;
                const bool some = k + warp * WARP_K < k1, inside = mine < k1;  // K is a multiple of 16
                auto fetch = [&](int i, typename X::Raw &x) {
                    if (inside && 8 * i + g < en.count) X::load(rows[i], mine, x);
                    else memset(x, 0, sizeof(x));
                };
                typename X::Raw raw[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) fetch(i, raw[i]);
                wait(&s.full[r.slot], r.phase, 2);
                if (some) {
                    const unsigned char *at = ring_gen + r.slot * STAGE_BYTES + a_off;
                    uint4 w[4];  // rows + 0, 8, 16, 24
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4 *>(at + i * 8 * BOX_K);
                    uint32_t f[4][8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) umma::cvt_s8x4_to_f16_pairs(v[j], f[i][2 * j], f[i][2 * j + 1]);
                    }
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        if (8 * i < en.count) {
                            uint32_t b[8];
                            X::convert(raw[i % AHEAD], by[i], b);
                            if (i + AHEAD < G && 8 * (i + AHEAD) < en.count) fetch(i + AHEAD, raw[i % AHEAD]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                mma_m16n8k16(acc[0][i], f[0][2 * j], f[1][2 * j], f[0][2 * j + 1], f[1][2 * j + 1], b[2 * j], b[2 * j + 1]);
                                mma_m16n8k16(acc[1][i], f[2][2 * j], f[3][2 * j], f[2][2 * j + 1], f[3][2 * j + 1], b[2 * j], b[2 * j + 1]);
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s.empty[r.slot]));
            }
            // ---- the eight warps' sums ----
            const int groups = (en.count + 7) / 8;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                if (i < groups) {
#pragma unroll
                    for (int l = 0; l < 2; ++l) {
                        *reinterpret_cast<float2 *>(&s.sums[warp][16 * l + row][8 * i + 2 * t]) = make_float2(acc[l][i][0], acc[l][i][1]);
                        *reinterpret_cast<float2 *>(&s.sums[warp][16 * l + 8 + row][8 * i + 2 * t]) = make_float2(acc[l][i][2], acc[l][i][3]);
                    }
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(MATH_THREADS) : "memory");
            if (!DOWN) {
                // thread: pair j of 16, column c
                for (int i = threadIdx.x; i < 128 * groups; i += MATH_THREADS) {
                    const int j = i & 15, c = i >> 4, f = tile * (ROWS / 2) + j;
                    float gate = 0.0f, up = 0.0f;
#pragma unroll
                    for (int w = 0; w < MATH_WARPS; ++w) gate += s.sums[w][2 * j][c], up += s.sums[w][2 * j + 1][c];
                    uint32_t bits = 0;
                    const int as = c < en.count ? s.order[en.first + c] : 0;
                    if (c < en.count && f < a.inner) {
                        const int64_t at = (int64_t)en.expert * 2 * a.inner + 2 * f;
                        const float back = s.back[which][c];
                        gate = gate * back * scale_at(a.gate_up_scale, a.scale_type, at);
                        up = up * back * scale_at(a.gate_up_scale, a.scale_type, at + 1);
                        const float h = silu(gate) * up;
                        p.h[(int64_t)as * a.inner + f] = h;
                        bits = __float_as_uint(h) & 0x7fffffffu;
                    }
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
                    if (j == 0 && c < en.count) atomicMax(p.counters + COUNTER_MAX + as, bits);
                }
                asm volatile("bar.sync 1, %0;" ::"n"(MATH_THREADS) : "memory");  // the sums have been read
            } else {
                const uint32_t nth = (uint32_t)(u - u0);
                const int part = k0 / p.part_k;
                for (int i = threadIdx.x; i < 256 * groups; i += MATH_THREADS) {
                    const int j = i & 31, c = i >> 5, n = tile * ROWS + j;
                    float y = 0.0f;
#pragma unroll
                    for (int w = 0; w < MATH_WARPS; ++w) y += s.sums[w][j][c];
                    if (c < en.count && n < a.hidden) {
                        const int as = s.order[en.first + c];
                        y = y * s.back[which][c] * scale_at(a.down_scale, a.scale_type, (int64_t)en.expert * a.hidden + n) * __ldcg(a.weights + as);
                        __stcg(p.pieces + ((int64_t)part * a.tokens * a.top + as) * a.hidden + n, y);
                    }
                }
                if (nth >= 2) wait(&s.freed[nth & 1], ((nth >> 1) - 1) & 1, 3);
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s.ready[nth & 1]));
                asm volatile("bar.sync 1, %0;" ::"n"(MATH_THREADS) : "memory");
            }
        }
    } else if (DOWN) {
        // ---------------- finishing: who brings a column tile's last piece adds them up ----------------
        pdl_wait();
        const int ft = threadIdx.x - UP_THREADS;
        for (int64_t u = u0; u < u1; ++u) {
            const uint32_t nth = (uint32_t)(u - u0);
            int k0, k1, tile, entry;
            k_of(u, k0, k1, tile, entry);
            wait(&s.ready[nth & 1], (nth >> 1) & 1, 4);
            if (ft == 0) {
                __threadfence();
                const unsigned int pieces = (unsigned int)(s.entries * p.parts);
                const bool last = atomicAdd(p.counters + tile, 1u) == pieces - 1;
                if (last) p.counters[tile] = 0;
                __threadfence();
                s.last = last;
            }
            asm volatile("bar.sync 2, %0;" ::"n"(32 * FINISH_WARPS) : "memory");
            if (s.last) {
                const int n = tile * ROWS + (ft & 7) * 4;  // four columns a thread: hidden is a multiple of 16
                for (int t = ft >> 3; t < a.tokens && n < a.hidden; t += 4 * FINISH_WARPS) {
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int j = 0; j < a.top; ++j) {
                        const int as = t * a.top + j, e = __ldcg(a.experts + as);
                        if (e < 0 || e >= a.count) continue;
#pragma unroll 4
                        for (int q = 0; q < p.parts; ++q) {
                            const float4 v = __ldcg(reinterpret_cast<const float4 *>(p.pieces + ((int64_t)q * a.tokens * a.top + as) * a.hidden + n));
                            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                        }
                    }
                    store_result(a, t, n, sum.x), store_result(a, t, n + 1, sum.y), store_result(a, t, n + 2, sum.z), store_result(a, t, n + 3, sum.w);
                }
            }
            asm volatile("bar.sync 2, %0;" ::"n"(32 * FINISH_WARPS) : "memory");
            if (ft == 0) mbar_arrive(smem_u32(&s.freed[nth & 1]));
        }
    }
    if (DOWN) {
        if (units == 0) {  // nobody is anyone's: the residual, or zeros
            for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < (int64_t)a.tokens * a.hidden; i += (int64_t)gridDim.x * THREADS) store_result(a, (int)(i / a.hidden), (int)(i % a.hidden), 0.0f);
        }
        // the largest magnitudes are zero again when all CTAs have read them
        __syncthreads();
        if (threadIdx.x == 0) {
            __threadfence();
            s.last = atomicAdd(p.counters + COUNTER_DONE, 1u) == gridDim.x - 1;
        }
        __syncthreads();
        if (s.last) {
            for (int i = threadIdx.x; i < a.tokens * a.top; i += THREADS) p.counters[COUNTER_MAX + i] = 0;
            if (threadIdx.x == 0) p.counters[COUNTER_DONE] = 0;
        }
    }
}

template <int G, bool DOWN, typename X>
int launch_stream(const CUtensorMap &map, StreamArgs p, cudaStream_t stream) {
    const ExpertsArgs &a = p.a;
    const int assignments = a.tokens * a.top;
    const int shared = (int)sizeof(Shared<G>) + (int)sizeof(Entry) * assignments;
    // two kernels side by side on an SM where that leaves four stages
    const int most = 113 * 1024 - 1024 - shared >= 4 * STAGE_BYTES ? 113 * 1024 : 225 * 1024;
    const int stages = (most - 1024 - shared) / STAGE_BYTES;
    p.stages = stages < MOST_STAGES ? stages : MOST_STAGES;
    static std::atomic<bool> attr_set[64];
    const int rc = allow_smem(attr_set, experts_stream_kernel<G, DOWN, X>, 225 * 1024);
    if (rc != B200Q_OK) return rc;
    const int grid = sm_count() > 0 ? sm_count() : 148;
    return launch_after("experts_stream_kernel", experts_stream_kernel<G, DOWN, X>, dim3((unsigned)grid), DOWN ? DOWN_THREADS : UP_THREADS,
                        (size_t)(1024 + p.stages * STAGE_BYTES + shared), 1, stream, map, p);
}

template <int G>
int launch_both(const CUtensorMap &up, const CUtensorMap &down, StreamArgs p, cudaStream_t stream) {
    StreamArgs first = p;
    first.tiles = (int)ceil_div(2 * (int64_t)p.a.inner, ROWS), first.parts = 1, first.part_k = p.a.hidden;
    const int rc = p.a.type == B200Q_F16 ? launch_stream<G, false, FromF16>(up, first, stream) : launch_stream<G, false, FromBF16>(up, first, stream);
    return rc != B200Q_OK ? rc : launch_stream<G, true, FromF32>(down, p, stream);
}

// Parts of K of down: units enough for an equal share of every SM, two stages of K each at least.
int parts_of(int64_t tokens, int64_t hidden, int64_t inner, int64_t count, int64_t top, int &part_k) {
    const int64_t experts = count < tokens * top ? count : tokens * top, units = experts * ceil_div(hidden, ROWS);
    int64_t parts = ceil_div(148 * 12, units > 0 ? units : 1);
    const int64_t most = ceil_div(inner, 2 * STAGE_K);
    if (parts > most) parts = most;
    if (parts > 8) parts = 8;
    if (parts < 1) parts = 1;
    part_k = parts == 1 ? (int)inner : (int)round_up(ceil_div(inner, parts), STAGE_K);
    return (int)ceil_div(inner, part_k);
}

}  // namespace

bool experts_stream_supported(const ExpertsArgs &a) {
    return a.hidden % 16 == 0 && a.inner % 16 == 0 && a.inner > 0 && aligned_to(a.x, 16) && (a.tokens == 1 || a.x_stride % 8 == 0) && aligned_to(a.gate_up, 16) && aligned_to(a.down, 16) &&
           a.count > 0 && a.count <= MOST_EXPERTS && a.top > 0 && a.top <= MOST_ASSIGNMENTS / 64 && a.hidden / ROWS < COUNTER_TILES && (int64_t)a.count * 2 * a.inner < 0x7fffff00LL &&
           (int64_t)a.count * a.hidden < 0x7fffff00LL;
}

size_t experts_stream_bytes(int64_t tokens, int64_t hidden, int64_t inner, int64_t count, int64_t top) {
    int64_t most = 0;
    for (int64_t t : {tokens < kExpertsTokens ? tokens : kExpertsTokens, tokens % kExpertsTokens}) {
        int part_k = 0;
        const int64_t bytes = 4 * (round_up(t * top * inner, 64) + (t > 0 && inner > 0 ? parts_of(t, hidden, inner, count, top, part_k) : 0) * t * top * hidden);
        if (bytes > most) most = bytes;
    }
    return (size_t)most;
}

int launch_experts_stream(const ExpertsArgs &all, unsigned int *counters, float *scratch, cudaStream_t stream) {
    CUtensorMap up, down;
    int rc = make_tensor_map_2d(&up, CU_TENSOR_MAP_DATA_TYPE_UINT8, all.gate_up, (uint64_t)all.hidden, (uint64_t)all.count * 2 * all.inner, (uint64_t)all.hidden, BOX_K, ROWS,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != B200Q_OK) return rc;
    rc = make_tensor_map_2d(&down, CU_TENSOR_MAP_DATA_TYPE_UINT8, all.down, (uint64_t)all.inner, (uint64_t)all.count * all.hidden, (uint64_t)all.inner, BOX_K, ROWS,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != B200Q_OK) return rc;
    StreamArgs p = {};
    p.a = all;
    const ExpertsArgs &a = p.a;
    p.h = scratch, p.pieces = scratch + round_up((int64_t)a.tokens * a.top * a.inner, 64), p.counters = counters;
    p.tiles = (int)ceil_div(a.hidden, ROWS);
    p.parts = parts_of(a.tokens, a.hidden, a.inner, a.count, a.top, p.part_k);
    return a.tokens <= 8 ? launch_both<1>(up, down, p, stream) : a.tokens <= 16 ? launch_both<2>(up, down, p, stream) : launch_both<4>(up, down, p, stream);
}

}  // namespace b200q
