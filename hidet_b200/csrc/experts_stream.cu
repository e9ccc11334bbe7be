// A layer of experts over a few tokens as two streams of int8 weights: gate and up, and down.  Inference at batch sizes where the weights of the experts that have
// a token are all there is to read.
//
// The tensor core multiplies the weights as they are, int8 by int8: a token's row is written as whole numbers v = rint(x 2^e), |v| <= 2^22 (e by the row's largest
// element, so that an element is off by at most 2^-22 of that), and these as three digits of 8 bits, v = 65536 d2 + 256 d1 + d0 with d in -128 .. 127.  A tile of 128 rows of the weight is the
// first operand of tcgen05.mma, three columns for each token are the second, sums of 32 bits are exact, and float begins behind them.  So weights are only ever copied,
// and what is computed on them costs no issue slots.  (As f16 by mma.sync, with int8 widened in registers, a tile took 260 instructions of each of eight warps, and the
// stream stood at 3.2 TB/s.)  One token, two of eight experts of 4096 x 14336: 62 us, 5.7 TB/s; 8 tokens 210 us, 6.0 TB/s; 7 tokens, six of 64 of 2048 x 1408: 55 us; one, six of 64 of 608 x 288: 14.  What is not the stream
// is some 5 us at the start of either kernel (launch, entries, first loads) and the meeting of parts at its end.
//
// Every CTA makes the list of entries, an expert with up to C of its assignments (an expert with more has several entries), and takes an equal, contiguous part of
// all stages, 128 rows x 128 k each.  Warps:
//     warp 0      copies the weights' tiles into a ring
//     warp 1      issues the products, into two accumulators in turn
//     warps 4-7   finish: tensor memory -> float -> h, or results
//     the others  digits: four teams take the ring's stages in turn and put the tokens' digits beside the weights' tile
// Gate and up: rows (2 f, 2 f + 1) are neighbouring lanes; h = silu(g) u in float to global memory, and its largest magnitude per assignment, which is what down's
// digits are scaled by.  A unit (an entry's 128 rows) that two or more CTAs share has its whole-number sums added by the one that comes last.
// Down: a column tile's entries follow one another, and what a CTA has of them it adds up in float, times scales and weights, in their order; the CTA that comes last adds the
// CTAs' parts in theirs.  Nothing depends on who comes when.
//
// Down's CTAs start as those of gate and up leave, and fill their rings with weights while they wait for h.
//
// Waits are bounded: one that runs out is reported and raises a flag, after which nobody in the CTA waits or copies any more; everyone goes through the motions
// to the end, so that no barrier is left alone.
#include <type_traits>

#include "experts.h"
#include "experts_digits.cuh"
#include "experts_parts.cuh"
#include "serving.cuh"
#include "umma.cuh"

namespace b200q {
namespace {

constexpr unsigned int kKernelExperts = 11;
constexpr int TN = 128, BK = 128;         // rows and k of a stage
constexpr int W_BYTES = TN * BK;
constexpr int COPY_WARP = 0, MMA_WARP = 1, FINISH_WARP0 = 4, DIGIT_WARP0 = 8, TEAMS = 4;
constexpr int ITEMS = BK / 8;             // of a column in a stage, a thread's eight elements each
constexpr int TEAM = 2;                   // warps
constexpr int THREADS = 32 * (DIGIT_WARP0 + TEAM * TEAMS), WARPS = THREADS / 32;
constexpr int WIDE = 2;                   // columns at a time that results are made of: the code is short, and most of its first run is waiting for it
constexpr int MOST_STAGES = 10;
constexpr int MOST_SMEM = 227 * 1024;
constexpr int MOST_ASSIGNMENTS = kExpertsAssignments;
constexpr int MOST_EXPERTS = 512;
constexpr int FEW_ASSIGNMENTS = 128;
static_assert(FEW_ASSIGNMENTS <= THREADS, "one a thread");
constexpr uint16_t kNone = 0xffff;
// what of the workspace's counters is whose: arrivals at what CTAs share (by the first of them), CTAs that are through, h's largest magnitudes
constexpr int MOST_CTAS = 1024, COUNTER_UP = 0, COUNTER_DOWN = MOST_CTAS, COUNTER_DONE = 2 * MOST_CTAS, COUNTER_MAX = 4 * MOST_CTAS;

constexpr int EARLY_TOKENS = 16;          // whose largest elements are sought before it is known which of them a CTA needs

struct StreamArgs {
    ExpertsArgs a;
    float *h;             // [assignments, inner]
    void *shared;         // gate and up: int32 [CTAs][2][columns][128]; down: float [CTAs][2][tokens][128]
    unsigned int *counters;
    uint32_t tiles;       // of 128 rows, of an expert's weight
    uint32_t k_blocks;
    int most;             // assignments of an entry
    uint32_t tmem_cols;
    int ring_bytes;
};

// What an entry's columns are laid out for: C assignments, whose digits of one rank stand side by side, and 3 C rounded up to 16 columns.
__host__ __device__ constexpr int columns_for(int count) { return count <= 5 ? 5 : count <= 10 ? 10 : count <= 16 ? 16 : count <= 32 ? 32 : 64; }
__host__ __device__ constexpr int sixteens(int c) { return (DIGITS * c + 15) / 16 * 16; }

struct Entry {
    uint16_t expert, first, count;  // its assignments are order[first ..]
};

__device__ __forceinline__ uint32_t idesc_i8(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void ld_columns(uint32_t taddr, int (&v)[2]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(taddr) : "memory");
}

struct alignas(16) Shared {
    uint64_t weights[MOST_STAGES], tokens[MOST_STAGES], empty[MOST_STAGES];  // a stage's two operands are in place; its products are through
    uint64_t acc_full[2], acc_empty[2], drain;
    uint32_t tmem_base;
    int abort_flag, entries, largest, last, to_add;
    int add[2][3];  // (down) what this CTA adds up at the end: tile, first and last CTA
    int duplicates;
    uint32_t bits[EARLY_TOKENS];
};
// Behind it: counts [experts], who [experts] (the tokens of an expert, a bit each), by, back, share [n] (float, of the assignments in their order), entry [n], chosen, order, token [n] (uint16),
// (down) sums [tokens][128] (float)
struct Lists {
    int *counts;
    uint2 *who;
    float *by, *back, *share;
    Entry *entry;
    uint16_t *chosen, *order, *token;
    float *sums;
    __host__ __device__ static constexpr int bytes(int n, int experts, int tokens) { return round16(12 * experts) + round16(12 * n) + round16(6 * n) + round16(6 * n) + tokens * TN * 4; }
    __host__ __device__ static constexpr int round16(int b) { return (b + 15) / 16 * 16; }
    __device__ __forceinline__ Lists(unsigned char *at, int n, int experts) {
        who = reinterpret_cast<uint2 *>(at), counts = reinterpret_cast<int *>(who + experts);
        at += round16(12 * experts);
        by = reinterpret_cast<float *>(at), back = by + n, share = back + n;
        at += round16(12 * n);
        entry = reinterpret_cast<Entry *>(at);
        at += round16(6 * n);
        chosen = reinterpret_cast<uint16_t *>(at), order = chosen + n, token = order + n;
        sums = reinterpret_cast<float *>(at + round16(6 * n));
    }
};

// What make_entries begins with, in front of the wait for the experts.
__device__ __forceinline__ void clear_lists(const ExpertsArgs &a, Shared &s, const Lists &l) {
    if (a.tokens * a.top > FEW_ASSIGNMENTS)
        for (int e = threadIdx.x; e < a.count; e += THREADS) l.counts[e] = 0, l.who[e] = make_uint2(0, 0);
    if (threadIdx.x < EARLY_TOKENS) s.bits[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.duplicates = 0;
    __syncthreads();
}

// The entries of a launch: counts by expert and the tokens that they are of, a sum over the experts, assignments in their places.  Every CTA makes them for itself, so an
// expert's assignments stand in their own order: as they come they would differ from CTA to CTA, and with them whose column is whose.  `meanwhile` runs while the experts are on their way.
// Few assignments have their places by comparing each with all: 1.2 us instead of 2.1.
template <typename F>
__device__ __forceinline__ void make_entries(const ExpertsArgs &a, int columns, Shared &s, const Lists &l, F meanwhile) {
    const int n = a.tokens * a.top;
    if (n <= FEW_ASSIGNMENTS) {
        const int i = threadIdx.x;
        uint16_t mine = kNone;
        const int e = i < n ? __ldcg(a.experts + i) : -1;
        meanwhile();
        if (i < n) {
            if (e >= 0 && e < a.count) mine = (uint16_t)e;
            else if (e >= 0 && blockIdx.x == 0 && a.status != nullptr) atomicOr(a.status, kBadExpert);
            l.chosen[i] = mine;
        }
        __syncthreads();
        int *sizes = reinterpret_cast<int *>(l.by);  // by place: assignments of the entry that begins there
        if (mine != kNone) {
            int less = 0, before = 0, all = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) {
                const uint16_t e = l.chosen[j];
                less += e < mine, all += e == mine, before += e == mine && j < i;
            }
            const int to = less + before;
            l.order[to] = (uint16_t)i, l.token[to] = (uint16_t)(i / a.top);
            sizes[to] = before % columns == 0 ? min(columns, all - before) : 0;
        }
        const int there = __syncthreads_count(mine != kNone);
        if (threadIdx.x < 32) {
            int entries = 0, largest = 0;
            for (int at = (int)threadIdx.x; at - (int)threadIdx.x < there; at += 32) {
                const int size = at < there ? sizes[at] : 0;
                const uint32_t begins = __ballot_sync(0xffffffffu, size > 0);
                if (size > 0) l.entry[entries + __popc(begins & ((1u << threadIdx.x) - 1u))] = {l.chosen[l.order[at]], (uint16_t)at, (uint16_t)size};
                entries += __popc(begins), largest = max(largest, size);
            }
            largest = __reduce_max_sync(0xffffffffu, largest);
            if (threadIdx.x == 0) s.entries = entries, s.largest = largest;
        }
        __syncthreads();
        return;
    }
    meanwhile();
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const int e = __ldcg(a.experts + i), t = i / a.top;
        const bool there = e >= 0 && e < a.count;
        l.chosen[i] = there ? (uint16_t)e : kNone;
        if (there) {
            atomicAdd(&l.counts[e], 1);
            const uint32_t bit = 1u << (t & 31);
            if (atomicOr(t < 32 ? &l.who[e].x : &l.who[e].y, bit) & bit) s.duplicates = 1;
        } else if (e >= 0 && blockIdx.x == 0 && a.status != nullptr) {
            atomicOr(a.status, kBadExpert);
        }
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int each = (a.count + 31) / 32, e0 = threadIdx.x * each, e1 = min(a.count, e0 + each);
        int mine = 0, my_entries = 0, largest = 0;
        for (int e = e0; e < e1; ++e) {
            const int c = l.counts[e];
            mine += c, my_entries += (c + columns - 1) / columns, largest = max(largest, min(c, columns));
        }
        int at = mine, at_entry = my_entries;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, at, o), y = __shfl_up_sync(0xffffffffu, at_entry, o);
            if ((int)threadIdx.x >= o) at += x, at_entry += y;
        }
        if (threadIdx.x == 31) s.entries = at_entry;
        at -= mine, at_entry -= my_entries;
        for (int e = e0; e < e1; ++e) {
            const int c = l.counts[e];
            l.counts[e] = at;
            for (int i = 0; i < c; i += columns) l.entry[at_entry++] = {(uint16_t)e, (uint16_t)(at + i), (uint16_t)min(columns, c - i)};
            at += c;
        }
        largest = __reduce_max_sync(0xffffffffu, largest);
        if (threadIdx.x == 0) s.largest = largest;
        __syncwarp();
        if (s.duplicates) {  // a token that has an expert twice: one assignment after the other
            for (int i0 = 0; i0 < n; i0 += 32) {
                const int i = i0 + threadIdx.x;
                const uint32_t e = i < n ? l.chosen[i] : kNone, same = __match_any_sync(0xffffffffu, e);
                const int place = e != kNone ? l.counts[e] : 0;
                __syncwarp();
                if (e != kNone) {
                    const int to = place + __popc(same & ((1u << threadIdx.x) - 1u));
                    l.order[to] = (uint16_t)i, l.token[to] = (uint16_t)(i / a.top);
                    if ((same >> threadIdx.x) == 1u) l.counts[e] = place + __popc(same);  // the last of them
                }
                __syncwarp();
            }
        }
    }
    __syncthreads();
    if (!s.duplicates) {
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const uint32_t e = l.chosen[i], t = i / a.top;
            if (e == kNone) continue;
            const uint32_t before = (1u << (t & 31)) - 1u;
            const int to = l.counts[e] + (t < 32 ? __popc(l.who[e].x & before) : __popc(l.who[e].x) + __popc(l.who[e].y & before));
            l.order[to] = (uint16_t)i, l.token[to] = (uint16_t)t;
        }
        __syncthreads();
    }
}

// Where a CTA is in its part of the stages.  Gate and up: k fastest, then an entry's tiles, then entries; down: k, then a tile's entries, then tiles.
template <bool DOWN>
struct Place {
    uint32_t entry, tile, k;
    __device__ __forceinline__ Place(uint32_t stage, const StreamArgs &p, uint32_t entries) {
        const uint32_t u = stage / p.k_blocks, inner = DOWN ? max(entries, 1u) : p.tiles, outer = u / inner, in = u - outer * inner;
        k = stage - u * p.k_blocks;
        entry = DOWN ? in : outer, tile = DOWN ? outer : in;
    }
    __device__ __forceinline__ void next_unit(const StreamArgs &p, uint32_t entries) {
        if (DOWN) {
            if (++entry == entries) entry = 0, ++tile;
        } else {
            if (++tile == p.tiles) tile = 0, ++entry;
        }
    }
};

__device__ __forceinline__ void store_result(const ExpertsArgs &a, int t, int n, float v) {
    if (a.residual != nullptr) v += token_value(a.residual, a.type, t * a.residual_stride + n);
    const int64_t at = (int64_t)t * a.hidden + n;
    if (a.type == B200Q_F16) static_cast<__half *>(a.out)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
}

// X: what the tokens are; DOWN: h, else x.
template <bool DOWN, typename X>
__global__ void __launch_bounds__(THREADS, 1) experts_stream_kernel(const __grid_constant__ CUtensorMap map_w, const StreamArgs p) {
    extern __shared__ unsigned char smem_dyn[];
    const uint32_t ring = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char *ring_gen = smem_dyn + (ring - smem_u32(smem_dyn));
    Shared &s = *reinterpret_cast<Shared *>(ring_gen + p.ring_bytes);
    const ExpertsArgs &a = p.a;
    const Lists l(reinterpret_cast<unsigned char *>(&s + 1), a.tokens * a.top, a.count);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int K = DOWN ? a.inner : a.hidden, rows = DOWN ? a.hidden : 2 * a.inner;

    if (threadIdx.x == 0) {
        for (int i = 0; i < MOST_STAGES; ++i) {
            mbar_init(smem_u32(&s.weights[i]), 1);
            mbar_init(smem_u32(&s.tokens[i]), TEAM);
            mbar_init(smem_u32(&s.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s.acc_full[i]), 1);
            mbar_init(smem_u32(&s.acc_empty[i]), 4);
        }
        mbar_init(smem_u32(&s.drain), 1);
        s.abort_flag = 0, s.to_add = 0;
        mbar_fence_init();
    }
    if (warp == MMA_WARP) {
        umma::alloc(smem_u32(&s.tmem_base), p.tmem_cols);
        umma::relinquish();
    }
    clear_lists(a, s, l);
    // The experts were chosen in front of gate and up, which waits for that before it lets down start: down may read them, and request weights, without waiting.
    if (!DOWN) pdl_wait();
    umma::fence_before_sync();
    // The largest magnitudes of a few tokens, a warp 1024 elements at a time, in front of the weights' requests, behind which they would wait.
    make_entries(a, p.most, s, l, [&]() {
        if constexpr (!DOWN) {
            const int pieces = (K + 1023) / 1024;
            for (int i = warp; a.tokens <= EARLY_TOKENS && i < a.tokens * pieces; i += WARPS) {
                const int t = i / pieces, k = (i - t * pieces) * 1024 + lane * 8;
                uint32_t bits = 0;
                uint4 v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = make_uint4(0, 0, 0, 0);
                    if (k + j * 256 < K) v[j] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.x) + t * a.x_stride + k + j * 256);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) bits = X::largest(X::largest(X::largest(X::largest(bits, v[j].x), v[j].y), v[j].z), v[j].w);
                bits = __reduce_max_sync(0xffffffffu, bits);
                if (lane == 0) atomicMax(&s.bits[t], bits);
            }
        }
    });
    umma::fence_after_sync();
    pdl_launch_dependents();
    const uint32_t tmem_base = s.tmem_base;
    const uint32_t entries = s.entries;
    // Stages as large as the largest entry asks for, and as many as there is room for.
    const int C = columns_for(s.largest), columns = sixteens(C);
    const uint32_t stage_bytes = W_BYTES + (uint32_t)columns * BK, stages = min((uint32_t)MOST_STAGES, p.ring_bytes / stage_bytes);
    const Parts parts(entries * p.tiles, p.k_blocks, gridDim.x, !DOWN);
    const uint32_t s0 = parts.first_of(blockIdx.x), s1 = parts.first_of(blockIdx.x + 1);
    const int mine = (int)(s1 - s0);  // stages of this CTA
    const Place<DOWN> start(s0, p, entries);

    auto wait = [&](uint64_t *bar, uint32_t parity, unsigned int site) {
        const uint32_t b = smem_u32(bar);
        for (uint32_t i = 0; i < kSpinLimit; ++i) {
            if (mbar_try_wait(b, parity)) return;
            if ((i & 15u) == 15u && *reinterpret_cast<volatile int *>(&s.abort_flag) != 0) return;
        }
        report_timeout(a.status, kKernelExperts, site);
        atomicExch(&s.abort_flag, 1);
    };

    if (warp == COPY_WARP) {
        // ---------------- the stream of weights ----------------
        if (lane == 0) {
            const uint64_t once = l2_policy_evict_first();
            Place<DOWN> at = start;
            umma::Ring r;
            int i = 0;
            for (; i < mine; ++i, r.advance(1, stages)) {
                if (DOWN && i == (int)stages) pdl_wait();  // the bounded waits do not run against the kernel in front
                if (i >= (int)stages) wait(&s.empty[r.slot], r.phase ^ 1u, 1);
                if (*reinterpret_cast<volatile int *>(&s.abort_flag) != 0) break;
                const uint32_t bar = smem_u32(&s.weights[r.slot]);
                mbar_expect_tx(bar, W_BYTES);
                tma_load_2d_hint(ring + r.slot * stage_bytes, &map_w, at.k * BK, (int)(l.entry[at.entry].expert * (uint32_t)rows + at.tile * TN), bar, once);
                if (++at.k == p.k_blocks) at.k = 0, at.next_unit(p, entries);
            }
            // every copy armed has landed before the CTA may retire
            for (int t = i > (int)stages ? i - (int)stages : 0; t < i; ++t)
                if (!mbar_wait(smem_u32(&s.weights[t % stages]), (t / stages) & 1)) report_timeout(a.status, kKernelExperts, 7);
        }
        __syncwarp();
        if (DOWN) pdl_wait();
    } else if (warp == MMA_WARP) {
        // ---------------- products ----------------
        if (DOWN) pdl_wait();
        if (elect_one()) {
            const uint32_t idesc = idesc_i8(TN, columns);
            umma::Ring r;
            uint32_t k = start.k, unit = 0;
            for (int i = 0; i < mine;) {
                const uint32_t buf = unit & 1;
                if (unit >= 2) wait(&s.acc_empty[buf], ((unit >> 1) - 1) & 1, 3);
                umma::fence_after_sync();
                const uint32_t d = tmem_base + buf * columns;
                for (bool first = true; k < p.k_blocks && i < mine; ++k, ++i, first = false, r.advance(1, stages)) {
                    wait(&s.weights[r.slot], r.phase, 4);
                    wait(&s.tokens[r.slot], r.phase, 5);
                    umma::fence_after_sync();
                    const uint32_t at = ring + r.slot * stage_bytes;
                    const uint64_t w_desc = umma::smem_desc_sw128(at), x_desc = umma::smem_desc_sw128(at + W_BYTES);
#pragma unroll
                    for (int ks = 0; ks < BK / 32; ++ks) mma_i8(d, w_desc + 2 * ks, x_desc + 2 * ks, idesc, !first || ks > 0 ? 1u : 0u);
                    umma::commit(smem_u32(&s.empty[r.slot]));
                }
                umma::commit(smem_u32(&s.acc_full[buf]));
                ++unit, k = 0;
            }
            umma::commit(smem_u32(&s.drain));
            if (!mbar_wait(smem_u32(&s.drain), 0)) report_timeout(a.status, kKernelExperts, 8);
        }
    } else if (warp >= 2) {
        if (DOWN) pdl_wait();  // h
        // ---------------- the powers of two of the rows that this CTA's entries have ----------------
        if (mine > 0) {
            if (DOWN) {
                const Entry last = l.entry[entries - 1];
                for (int i = threadIdx.x - 64; i < last.first + last.count; i += THREADS - 64) {
                    const int as = l.order[i];
                    l.by[i] = power_for(__ldcg(p.counters + COUNTER_MAX + as), l.back[i]);
                    l.share[i] = __ldcg(a.weights + as);
                }
            } else {
                const Place<DOWN> end(s1 - 1, p, entries);
                const Entry last = l.entry[end.entry];
                if (a.tokens <= EARLY_TOKENS) {
                    for (int i = l.entry[start.entry].first + threadIdx.x - 64; i < last.first + last.count; i += THREADS - 64) l.by[i] = power_for(s.bits[l.token[i]], l.back[i]);
                } else {
                    for (int i = l.entry[start.entry].first + warp - 2; i < last.first + last.count; i += WARPS - 2) {
                        const uint4 *x = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.x) + (int64_t)l.token[i] * a.x_stride);
                        uint32_t bits = 0;
#pragma unroll 8
                        for (int j = lane; j < K / 8; j += 32) {
                            const uint4 v = x[j];
                            if constexpr (!DOWN) bits = X::largest(X::largest(X::largest(X::largest(bits, v.x), v.y), v.z), v.w);
                        }
                        bits = __reduce_max_sync(0xffffffffu, bits);
                        if (lane == 0) l.by[i] = power_for(bits, l.back[i]);
                    }
                }
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(THREADS - 64) : "memory");
        if (DOWN && warp == 2) {  // the largest magnitudes are zero again when all CTAs have read them
            int last = 0;
            if (lane == 0) {
                __threadfence();
                last = atomicAdd(p.counters + COUNTER_DONE, 1u) == gridDim.x - 1;
            }
            if (__shfl_sync(0xffffffffu, last, 0)) {
                for (int i = lane; i < a.tokens * a.top; i += 32) p.counters[COUNTER_MAX + i] = 0;
                if (lane == 0) p.counters[COUNTER_DONE] = 0;
            }
        }
        if (warp >= DIGIT_WARP0) {
            // ---------------- digits ----------------
            // Teams of two warps take stages in turn.  No more teams than stages: a wait tells a phase from its neighbours only, and a team that has written its last stage
            // knows that the one two rounds of the ring in front of its next has been read.
            const int team = (warp - DIGIT_WARP0) / TEAM, me = (warp - DIGIT_WARP0) % TEAM * 32 + lane;
            Place<DOWN> at(s0 + team, p, entries);
            auto fetch = [&](const Entry &en, uint32_t k_block, int j, typename X::Raw &raw, float &by) {  // eight k of a column
                const int c = j / ITEMS, k = (int)k_block * BK + j % ITEMS * 8;
                by = 0.0f;
                memset(raw, 0, sizeof(raw));
                if (c < en.count && k < K) {
                    const void *row = DOWN ? static_cast<const void *>(p.h + (int64_t)l.order[en.first + c] * K)
                                           : static_cast<const void *>(static_cast<const uint16_t *>(a.x) + (int64_t)l.token[en.first + c] * a.x_stride);
                    X::load(row, k, raw);
                    by = l.by[en.first + c];
                }
            };
            // What a stage needs first is asked for a stage of the team ahead.
            typename X::Raw raw, next;
            float by = 0.0f, next_by = 0.0f;
            Entry en = {0, 0, 0};
            if (team < mine) {
                en = l.entry[at.entry];
                fetch(en, at.k, me, raw, by);
            }
            for (int i = team; i < mine; i += TEAMS) {
                const uint32_t slot = (uint32_t)i % stages, use = (uint32_t)i / stages, k_block = at.k;
                const Entry here = en;
                unsigned char *tile = ring_gen + slot * stage_bytes + W_BYTES;
                for (at.k += TEAMS; at.k >= p.k_blocks; at.k -= p.k_blocks) at.next_unit(p, entries);
                if (i + TEAMS < mine) en = l.entry[at.entry];
                if (use > 0) wait(&s.empty[slot], (use - 1) & 1, 2);
                for (int j = me; j < here.count * ITEMS; j += 32 * TEAM) {
                    const bool more_here = j + 32 * TEAM < here.count * ITEMS;
                    if (more_here) fetch(here, k_block, j + 32 * TEAM, next, next_by);
                    else if (i + TEAMS < mine) fetch(en, at.k, me, next, next_by);
                    const int c = j / ITEMS, place = j % ITEMS;
                    uint32_t d[2][DIGITS];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float f[4];
                        widen4<X>(raw, q, f);
                        digits_of(f, by, d[q]);
                    }
#pragma unroll
                    for (int g = 0; g < DIGITS; ++g) {
                        const int row = g * C + c;
                        *reinterpret_cast<uint2 *>(tile + row * BK + (((place >> 1) ^ (row & 7)) << 4) + (place & 1) * 8) = make_uint2(d[0][g], d[1][g]);
                    }
                    memcpy(raw, next, sizeof(raw));
                    by = next_by;
                }
                if (me >= here.count * ITEMS && i + TEAMS < mine) fetch(en, at.k, me, raw, by);  // nothing here, perhaps something there
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s.tokens[slot]));
            }
        } else if (warp >= FINISH_WARP0) {
            // ---------------- results ----------------
            const int q = warp - FINISH_WARP0, row = 32 * q + lane;
            const uint32_t lane_addr = tmem_base + ((uint32_t)(32 * q) << 16);
            auto meet = [&]() { asm volatile("bar.sync 2, 128;" ::: "memory"); };
            // Who came to `counter` last of n: what all threads stored in front of it is seen by the last one's loads behind it.
            auto came_last = [&](unsigned int *counter, int n) {
                meet();
                if (row == 0) {
                    unsigned int before;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
                    const bool last = before == (unsigned int)(n - 1);
                    if (last) *counter = 0;
                    s.last = last;
                }
                meet();
                return s.last != 0;
            };
            Place<DOWN> at = start;
            uint32_t unit = 0;
            for (int i = 0; i < mine; ++unit) {
                const uint32_t buf = unit & 1;
                const uint32_t first_k = at.k;
                const int steps = min((int)(p.k_blocks - at.k), mine - i);
                const Entry en = l.entry[at.entry];
                const int n = at.tile * TN + row;
                const bool there = n < rows;
                const float scale = there ? scale_at(DOWN ? a.down_scale : a.gate_up_scale, a.scale_type, (int64_t)en.expert * rows + n) : 0.0f;
                if (DOWN && (i == 0 || (at.entry == 0 && at.k == 0))) {
                    for (int t = 0; t < a.tokens; ++t) l.sums[t * TN + row] = 0.0f;
                }
                wait(&s.acc_full[buf], (unit >> 1) & 1, 6);
                umma::fence_after_sync();
                const uint32_t acc = lane_addr + buf * columns;
                uint32_t c0 = blockIdx.x, c1 = blockIdx.x;
                bool finish = true;
                if (!DOWN && steps < (int)p.k_blocks) {
                    // a unit of several CTAs: this one's sums to the others, and whoever comes last adds them
                    const uint32_t u0 = s0 + i - first_k;
                    c0 = parts.cta_of(u0), c1 = parts.cta_of(u0 + p.k_blocks - 1);
                    int *to = static_cast<int *>(p.shared) + ((int64_t)blockIdx.x * 2 + parts.second_place(blockIdx.x, u0)) * columns * TN + row;
#pragma unroll 1
                    for (int c = 0; c < en.count; c += WIDE) {
                        int v[DIGITS][WIDE];
#pragma unroll
                        for (int g = 0; g < DIGITS; ++g) ld_columns(acc + g * C + c, v[g]);
                        umma::ld_wait();
#pragma unroll
                        for (int g = 0; g < DIGITS; ++g)
#pragma unroll
                            for (int j = 0; j < WIDE; ++j)
                                if (c + j < en.count) __stcg(to + (g * C + c + j) * TN, v[g][j]);
                    }
                    finish = came_last(p.counters + COUNTER_UP + c0, (int)(c1 - c0 + 1));
                }
#pragma unroll 1
                for (int c = 0; finish && c < en.count; c += WIDE) {
                    int v[DIGITS][WIDE];
#pragma unroll
                    for (int g = 0; g < DIGITS; ++g) ld_columns(acc + g * C + c, v[g]);
                    umma::ld_wait();
                    if (!DOWN) {
                        for (uint32_t other = c0; other <= c1; ++other) {
                            if (other == blockIdx.x) continue;
                            // the first of them has this unit last, the others first
                            const int *from = static_cast<const int *>(p.shared) + ((int64_t)other * 2 + parts.second_place(other, s0 + i - first_k)) * columns * TN + row;
#pragma unroll
                            for (int g = 0; g < DIGITS; ++g)
#pragma unroll
                                for (int j = 0; j < WIDE; ++j)
                                    if (c + j < en.count) v[g][j] += __ldcg(from + (g * C + c + j) * TN);
                        }
                    }
                    float y[WIDE];
#pragma unroll
                    for (int j = 0; j < WIDE; ++j) {
                        y[j] = fmaf((float)v[2][j], 65536.0f, fmaf((float)v[1][j], 256.0f, (float)v[0][j]));
                        y[j] *= scale;  // first: it and the power of two may be small together
                        if (c + j < en.count) y[j] *= l.back[en.first + c + j];
                    }
                    if (DOWN) {
#pragma unroll
                        for (int j = 0; j < WIDE; ++j) {
                            if (c + j < en.count) l.sums[l.token[en.first + c + j] * TN + row] += y[j] * l.share[en.first + c + j];
                        }
                    } else {
                        // even lanes have gates, odd ones what they multiply; of two columns each lane of a pair finishes one
                        const bool odd = lane & 1;
#pragma unroll
                        for (int j = 0; j < WIDE; j += 2) {
                            const float other = __shfl_xor_sync(0xffffffffu, odd ? y[j] : y[j + 1], 1);
                            const int col = c + j + (odd ? 1 : 0);
                            const float h = silu(odd ? other : y[j]) * (odd ? y[j + 1] : other);
                            uint32_t bits = 0;
                            int as = 0;
                            if (col < en.count) {
                                as = l.order[en.first + col];
                                if (there) {
                                    p.h[(int64_t)as * a.inner + (n >> 1)] = h;
                                    bits = __float_as_uint(h) & 0x7fffffffu;
                                }
                            }
                            const uint32_t even_most = __reduce_max_sync(0xffffffffu, odd ? 0u : bits), odd_most = __reduce_max_sync(0xffffffffu, odd ? bits : 0u);
                            if (lane < 2 && col < en.count) atomicMax(p.counters + COUNTER_MAX + as, odd ? odd_most : even_most);
                        }
                    }
                }
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s.acc_empty[buf]));
                i += steps;
                if (DOWN && (i == mine || (at.entry == entries - 1 && first_k + (uint32_t)steps == p.k_blocks))) {
                    // the tile's last stage, or this CTA's
                    const uint32_t t0 = at.tile * entries * p.k_blocks, t1 = t0 + entries * p.k_blocks;
                    if (t0 >= s0 && t1 <= s1) {
                        for (int t = 0; t < a.tokens && there; ++t) store_result(a, t, n, l.sums[t * TN + row]);
                    } else {
                        c0 = parts.cta_of(t0), c1 = parts.cta_of(t1 - 1);
                        float *to = static_cast<float *>(p.shared) + ((int64_t)blockIdx.x * 2 + parts.second_place(blockIdx.x, t0)) * a.tokens * TN + row;
                        for (int t = 0; t < a.tokens; ++t) __stcg(to + t * TN, l.sums[t * TN + row]);
                        if (came_last(p.counters + COUNTER_DOWN + c0, (int)(c1 - c0 + 1)) && row == 0) {
                            int *add = s.add[s.to_add];
                            add[0] = (int)at.tile, add[1] = (int)c0, add[2] = (int)c1;
                            ++s.to_add;
                        }
                    }
                }
                at.k = 0;
                at.next_unit(p, entries);
            }
        }
    }
    // ---------------- the end ----------------
    umma::fence_before_sync();
    __syncthreads();
    if (warp == MMA_WARP) {
        umma::fence_after_sync();
        umma::dealloc(tmem_base, p.tmem_cols);
    }
    if (DOWN) {
        // tiles of several CTAs whose last this one was: all warps, a token each, four columns a lane
        for (int i = 0; i < s.to_add; ++i) {
            const int tile = s.add[i][0], n = tile * TN + lane * 4;
            const uint32_t t0 = (uint32_t)tile * entries * p.k_blocks;
            // ROWS tokens of a warp, and ABREAST CTAs' parts of each, are asked for at once
            auto add_up = [&](auto rows_at_once, auto abreast) {
                constexpr int ROWS = decltype(rows_at_once)::value, ABREAST = decltype(abreast)::value;
                for (int t = warp; t < a.tokens && n < a.hidden; t += ROWS * WARPS) {  // hidden is a multiple of 16
                    float4 sum[ROWS];
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) sum[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
                    for (int c = s.add[i][1]; c <= s.add[i][2]; c += ABREAST) {
                        float4 v[ABREAST][ROWS];
#pragma unroll
                        for (int j = 0; j < ABREAST; ++j) {
                            const bool second = parts.second_place(c + j, t0);
                            const float *from = static_cast<const float *>(p.shared) + ((int64_t)(c + j) * 2 + second) * a.tokens * TN + lane * 4;
#pragma unroll
                            for (int r = 0; r < ROWS; ++r) {
                                v[j][r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                if (c + j <= s.add[i][2] && t + r * WARPS < a.tokens) v[j][r] = __ldcg(reinterpret_cast<const float4 *>(from + (t + r * WARPS) * TN));
                            }
                        }
#pragma unroll
                        for (int j = 0; j < ABREAST; ++j)
#pragma unroll
                            for (int r = 0; r < ROWS; ++r) sum[r].x += v[j][r].x, sum[r].y += v[j][r].y, sum[r].z += v[j][r].z, sum[r].w += v[j][r].w;
                    }
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        const int row = t + r * WARPS;
                        if (row < a.tokens) store_result(a, row, n, sum[r].x), store_result(a, row, n + 1, sum[r].y), store_result(a, row, n + 2, sum[r].z), store_result(a, row, n + 3, sum[r].w);
                    }
                }
            };
            if (a.tokens <= WARPS) add_up(std::integral_constant<int, 1>(), std::integral_constant<int, 12>());
            else add_up(std::integral_constant<int, 3>(), std::integral_constant<int, 4>());
        }
        if (parts.total == 0) {  // nobody is anyone's: the residual, or zeros
            for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < (int64_t)a.tokens * a.hidden; i += (int64_t)gridDim.x * THREADS) store_result(a, (int)(i / a.hidden), (int)(i % a.hidden), 0.0f);
        }
    }
}

int grid_of() {
    const int sms = sm_count() > 0 ? sm_count() : 148;
    return sms < MOST_CTAS ? sms : MOST_CTAS;
}

template <bool DOWN, typename X>
int launch_stream(const CUtensorMap &map, StreamArgs p, cudaStream_t stream) {
    const ExpertsArgs &a = p.a;
    const int rows = DOWN ? a.hidden : 2 * a.inner, K = DOWN ? a.inner : a.hidden;
    p.tiles = (uint32_t)ceil_div(rows, TN), p.k_blocks = (uint32_t)ceil_div(K, BK);
    const int shared = (int)sizeof(Shared) + Lists::bytes(a.tokens * a.top, a.count, DOWN ? a.tokens : 0);
    p.ring_bytes = (MOST_SMEM - 1024 - shared) / 1024 * 1024;
    static_assert((MOST_SMEM - 2048 - (int)sizeof(Shared) - Lists::bytes(MOST_ASSIGNMENTS, MOST_EXPERTS, kExpertsTokens)) / (W_BYTES + sixteens(columns_for(kExpertsTokens)) * BK) >= TEAMS,
                  "a stage for every team, whatever the sizes");
    static std::atomic<bool> attr_set[64];
    const int rc = allow_smem(attr_set, experts_stream_kernel<DOWN, X>, MOST_SMEM);
    if (rc != B200Q_OK) return rc;
    return launch_after("experts_stream_kernel", experts_stream_kernel<DOWN, X>, dim3((unsigned)grid_of()), THREADS, (size_t)(1024 + p.ring_bytes + shared), 1, stream, map, p);
}

}  // namespace

bool experts_fast(const ExpertsArgs &a) {
    return a.hidden % 16 == 0 && a.inner % 16 == 0 && a.inner > 0 && aligned_to(a.x, 16) && (a.tokens == 1 || a.x_stride % 8 == 0) && aligned_to(a.gate_up, 16) && aligned_to(a.down, 16) &&
           a.count > 0 && a.count <= MOST_EXPERTS && a.top > 0 && a.hidden <= kMostExact && a.inner <= kMostExact && (int64_t)a.count * 2 * a.inner < 0x7fffff00LL &&
           (int64_t)a.count * a.hidden < 0x7fffff00LL;
}

size_t experts_stream_bytes(int64_t tokens, int64_t inner, int64_t top) {
    const int64_t sums = sixteens(columns_for((int)tokens)), results = tokens;
    return (size_t)(4 * (round_up(tokens * top * inner, 64) + (int64_t)grid_of() * 2 * TN * (sums > results ? sums : results)));
}

int launch_experts_stream(const ExpertsArgs &a, unsigned int *counters, float *scratch, cudaStream_t stream) {
    CUtensorMap up, down;
    int rc = make_tensor_map_2d(&up, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.gate_up, (uint64_t)a.hidden, (uint64_t)a.count * 2 * a.inner, (uint64_t)a.hidden, BK, TN,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != B200Q_OK) return rc;
    rc = make_tensor_map_2d(&down, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.down, (uint64_t)a.inner, (uint64_t)a.count * a.hidden, (uint64_t)a.inner, BK, TN, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != B200Q_OK) return rc;
    StreamArgs p = {};
    p.a = a;
    p.h = scratch, p.shared = scratch + round_up((int64_t)a.tokens * a.top * a.inner, 64), p.counters = counters;
    p.most = columns_for(a.tokens);
    p.tmem_cols = 32;
    while ((int)p.tmem_cols < 2 * sixteens(p.most) + WIDE) p.tmem_cols *= 2;  // some columns are read behind the last
    rc = a.type == B200Q_F16 ? launch_stream<false, FromF16>(up, p, stream) : launch_stream<false, FromBF16>(up, p, stream);
    return rc != B200Q_OK ? rc : launch_stream<true, FromF32>(down, p, stream);
}

}  // namespace b200q
