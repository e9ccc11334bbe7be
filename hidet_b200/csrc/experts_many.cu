// A layer of experts over many tokens, on int8 weights: prompts, and batches with dozens of tokens an expert.
//
// The products are those of experts_stream.cu, three digits of 8 bits for an element of a token beside weights that are only copied, but time goes to the products here, and a
// token's digits are wanted by a hundred tiles of the weight.  So they are made once, as an image in memory: the rows of an expert's assignments side by side, digits of one rank
// together, which a tile's copies fetch as they are.  In order:
//     plan     one CTA sorts the assignments by expert into entries, up to MOST of one expert each, and gives every assignment a slot
//     image    x -> digits, a CTA a slot
//     product  gate and up: h = silu(g) u in float by slots, and its rows' largest magnitudes
//     image    h -> digits, in the same memory
//     product  down: its rows in float by slots, in h's memory
//     join     out[t] = residual[t] + sum_j weights[t, j] of the rows of its slots, in the order of j
// An assignment's sums do not depend on its place, so neither does the result.
//
// The products run on pairs of SMs as in qlinear_i8_pair.cu: a pair owns 256 rows of the weight x the columns of an entry, three for each of its slots, 128 k a stage.  Entries of an expert
// are neighbours in a round of all pairs, so that a tile of its weight comes from memory once (a contiguous part of the tiles for every pair instead: down of 512 tokens 230 us for 142).
// Bounded waits and their ends are as there.
//
// What bounds it, two of eight experts of 4096 x 14336: with 64 tokens (235 to 247 us) the weights' way from memory, 215 us; with 512 (487 to 530 us: 270 + 145 us by themselves, the rest small kernels and
// the clock under the power cap) and 2048 (1.93 to 2.1 ms, up to 2.2 POP/s) an SM's copies, some 40 bytes a clock of which 16 KB a stage are weights, whatever the entry's columns.  A copy of the
// image is one box: in boxes of 16 rows 512 tokens took 733 us, 576 in one then.  Rows' largest magnitudes are stored by warp and not gathered with atomics: gate and up 332 us with them, 274 without.
// With few k (1000 tokens, four of 32 of 1024 x 512: 72 us, 50 of them the products) results take the time: four groups of warps make them, two take 88 us.
#include <cstddef>
#include <type_traits>

#include "experts.h"
#include "experts_digits.cuh"
#include "experts_parts.cuh"
#include "serving.cuh"
#include "umma.cuh"
#include "umma_i8_pair.cuh"

namespace b200q {
namespace {

using i8pair::commit_to;
using i8pair::idesc_i8;
using i8pair::load_pair;
using i8pair::mma_pair_i8;

constexpr unsigned int kKernelExpertsMany = 13;
constexpr int MOST = kEntryMost, SLOTS = kEntrySlots;
constexpr int MOST_EXPERTS = 512, MOST_ASSIGNMENTS = 8192, MOST_ENTRIES = MOST_EXPERTS + MOST_ASSIGNMENTS / MOST + 1;
constexpr int MOST_SLOTS = MOST_ASSIGNMENTS + (SLOTS - 1) * MOST_ENTRIES;
constexpr int MOST_PAIRS = 512;               // which have some of the workspace's counters each: arrivals at a unit that pairs share, at the first of them, by CTA and group
static_assert(MOST_SLOTS < 65536 && 8 * MOST_PAIRS <= kWorkspaceCounters, "slots' numbers have 16 bits");

constexpr int TN = 128;                       // rows of the weight per CTA; a pair's tile has twice as many
constexpr int BK = 128;
constexpr int W_BYTES = BK * TN;
constexpr int MOST_COLUMNS = 256;
constexpr int STAGES = 6;
constexpr int STAGE_BYTES = W_BYTES + MOST_COLUMNS / 2 * BK;
constexpr int EPI_GROUPS = 4, LOAD_WARP = 4 * EPI_GROUPS, MMA_WARP = LOAD_WARP + 1, THREADS = 32 * (MMA_WARP + 1);
constexpr int TMEM_COLS = 512;

struct Group {  // an expert that has a token
    uint16_t expert, first, entries, none;
};
struct Entry {
    uint16_t slot, count, slots, none;
};
struct Slot {
    int assignment;       // or -1
    int row, stride;      // its digit g is row + g * stride of the image
};
struct alignas(16) Plan {
    int groups, entries, slots, largest;  // largest: slots of an entry
    Group group[MOST_EXPERTS];
    Entry entry[MOST_ENTRIES];
};
static_assert(sizeof(Group) == 8 && sizeof(Entry) == 8 && offsetof(Plan, group) == 16 && offsetof(Plan, entry) % 8 == 0, "read as vectors");
constexpr int LISTS_BYTES = (int)(sizeof(Group) * MOST_EXPERTS + sizeof(Entry) * MOST_ENTRIES);
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + (LISTS_BYTES + 15) / 16 * 16 + 1024;
static_assert(SMEM_BYTES <= 226 * 1024, "beside what is declared in the kernel");

// An entry's columns, a multiple of 32: three for each slot, and what lies behind them.
__host__ __device__ constexpr int columns_of(int slots) { return (DIGITS * slots + 31) / 32 * 32; }
static_assert(columns_of(MOST) <= MOST_COLUMNS, "two accumulators");

struct ManyArgs {
    ExpertsArgs a;
    Plan *plan;
    Slot *slot;           // [slots]
    float *back;          // [slots] what a slot's sums are multiplied by
    int *slot_of;         // [assignments], or -1
    uint32_t *largest;    // [slots, maxima]: largest magnitudes of h, as bits, of a warp's rows of the weight each
    int maxima;
    float *rows;          // [slots, max(inner, hidden)]: h, then down's rows
    int8_t *image;        // [3 slots, K]
    int *parts;           // [CTAs][most_columns][128]: sums of units that pairs share
    int most_columns;
    unsigned int *counters;
    int most_slots;
};

// ---------------- plan ----------------
constexpr int PLAN_THREADS = 1024;

__global__ void __launch_bounds__(PLAN_THREADS) experts_plan_kernel(const ManyArgs p) {
    __shared__ int counts[MOST_EXPERTS], taken[MOST_EXPERTS], first_slot[MOST_EXPERTS];
    const ExpertsArgs &a = p.a;
    const int n = a.tokens * a.top;
    pdl_launch_dependents();
    for (int e = threadIdx.x; e < a.count; e += PLAN_THREADS) counts[e] = 0, taken[e] = 0;
    __syncthreads();
    pdl_wait();
    constexpr int MINE = MOST_ASSIGNMENTS / PLAN_THREADS;
    int mine[MINE];
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        const int i = j * PLAN_THREADS + (int)threadIdx.x;
        mine[j] = i < n ? a.experts[i] : -1;
    }
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        if (mine[j] >= 0 && mine[j] < a.count) atomicAdd(&counts[mine[j]], 1);
        else if (mine[j] >= 0 && a.status != nullptr) atomicOr(a.status, kBadExpert);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int of_lane = (a.count + 31) / 32, e0 = min(a.count, (int)threadIdx.x * of_lane), e1 = min(a.count, e0 + of_lane);
        int my[3] = {0, 0, 0}, largest = 0;  // groups, entries, slots
        for (int e = e0; e < e1; ++e) {
            const EntrySizes its(counts[e]);
            if (counts[e] == 0) continue;
            largest = max(largest, its.room(0));
            my[0] += 1, my[1] += its.entries, my[2] += its.slots();
        }
        int at[3] = {my[0], my[1], my[2]};
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const int x = __shfl_up_sync(0xffffffffu, at[i], o);
                if ((int)threadIdx.x >= o) at[i] += x;
            }
        }
        largest = __reduce_max_sync(0xffffffffu, largest);
        if (threadIdx.x == 31) {
            p.plan->largest = largest;
            p.plan->groups = at[0], p.plan->entries = at[1], p.plan->slots = at[2];
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) at[i] -= my[i];
        for (int e = e0; e < e1; ++e) {
            const EntrySizes its(counts[e]);
            first_slot[e] = at[2];
            if (counts[e] == 0) continue;
            p.plan->group[at[0]++] = {(uint16_t)e, (uint16_t)at[1], (uint16_t)its.entries, 0};
            for (int i = 0; i < its.entries; ++i) {
                p.plan->entry[at[1]++] = {(uint16_t)at[2], (uint16_t)its.assignments(i), (uint16_t)its.room(i), 0};
                at[2] += its.room(i);
            }
        }
    } else {
        for (int s = threadIdx.x - 32; s < p.most_slots; s += PLAN_THREADS - 32) p.slot[s] = {-1, 0, 0};  // nobody's, until the others have theirs
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        const int i = j * PLAN_THREADS + (int)threadIdx.x, e = mine[j];
        if (i >= n) break;
        int slot = -1;
        if (e >= 0 && e < a.count) {
            const EntrySizes its(counts[e]);
            const int place = atomicAdd(&taken[e], 1), entry = place / its.size, in = place - entry * its.size;
            const int start = first_slot[e] + entry * EntrySizes::rounded(its.size);
            slot = start + in;
            p.slot[slot] = {i, DIGITS * start + in, its.room(entry)};
        }
        p.slot_of[i] = slot;
    }
}

// ---------------- image ----------------
constexpr int IMAGE_THREADS = 256;

// A slot's row is shared by the CTAs of a column of the grid, each of which looks for the largest of all of it.
template <typename X, bool OF_H>
__global__ void __launch_bounds__(IMAGE_THREADS) experts_image_kernel(const ManyArgs p) {
    __shared__ uint32_t largest;
    const int s = blockIdx.x, K = OF_H ? p.a.inner : p.a.hidden;
    if (threadIdx.x == 0) largest = 0;
    pdl_wait();
    pdl_launch_dependents();  // behind the wait: the product reads the plan without waiting for more
    if (s >= p.plan->slots) return;
    const Slot slot = p.slot[s];
    if (slot.assignment < 0) return;
    const void *row = OF_H ? static_cast<const void *>(p.rows + (int64_t)s * K) : static_cast<const void *>(static_cast<const uint16_t *>(p.a.x) + (int64_t)(slot.assignment / p.a.top) * p.a.x_stride);
    uint32_t bits = 0;
    if constexpr (OF_H) {
        for (int i = threadIdx.x; i < p.maxima; i += IMAGE_THREADS) bits = max(bits, p.largest[(int64_t)s * p.maxima + i]);
    } else {
#pragma unroll 2
        for (int k = threadIdx.x * 8; k < K; k += IMAGE_THREADS * 8) {
            typename X::Raw raw;
            X::load(row, k, raw);
            bits = X::largest(X::largest(X::largest(X::largest(bits, raw[0].x), raw[0].y), raw[0].z), raw[0].w);
        }
    }
    bits = __reduce_max_sync(0xffffffffu, bits);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) atomicMax(&largest, bits);
    __syncthreads();
    bits = largest;
    float back;
    const float by = power_for(bits, back);
    if (threadIdx.x == 0 && blockIdx.y == 0) p.back[s] = back;
    int8_t *to = p.image + (int64_t)slot.row * K;
    const int64_t apart = (int64_t)slot.stride * K;
#pragma unroll 2
    for (int k = (blockIdx.y * IMAGE_THREADS + threadIdx.x) * 8; k < K; k += gridDim.y * IMAGE_THREADS * 8) {
        typename X::Raw raw;
        X::load(row, k, raw);
        uint32_t d[2][DIGITS];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float f[4];
            widen4<X>(raw, q, f);
            digits_of(f, by, d[q]);
        }
#pragma unroll
        for (int g = 0; g < DIGITS; ++g) *reinterpret_cast<uint2 *>(to + g * apart + k) = make_uint2(d[0][g], d[1][g]);
    }
}

// ---------------- product ----------------
__device__ __forceinline__ void ld_columns(uint32_t taddr, int (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
}

// Which entry and tile of the weight a unit is (an entry's 256 rows); units are asked for in ascending order.
struct Units {
    const Group *group;
    int g, tiles;
    __device__ __forceinline__ Units(const Group *groups, int tiles_) : group(groups), g(0), tiles(tiles_) {}
    __device__ __forceinline__ void find(int u, int &expert, int &tile, int &entry) {
        while (u >= tiles * (group[g].first + group[g].entries)) ++g;
        const Group at = group[g];
        const int r = u - tiles * at.first;
        tile = r / at.entries, entry = at.first + (r - tile * at.entries), expert = at.expert;
    }
};

// A map of the image for each number of slots, by the columns that a CTA copies.
struct ImageMaps {
    CUtensorMap of[MOST / SLOTS];
};

template <bool DOWN>
__global__ void __launch_bounds__(THREADS, 1) experts_product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ ImageMaps map_x, const ManyArgs p) {
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) uint64_t full[STAGES];        // (first CTA) both CTAs' tiles of the stage have landed
    __shared__ __align__(8) uint64_t empty[STAGES];       // the MMAs that read it have completed
    __shared__ __align__(8) uint64_t acc_full[2];         // an accumulator holds a finished tile
    __shared__ __align__(8) uint64_t acc_empty[2];        // (first CTA) both CTAs' epilogue warps have read it out
    __shared__ __align__(8) uint64_t drain_bar;           // every MMA issued has completed
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag, came_last[EPI_GROUPS];

    const ExpertsArgs &a = p.a;
    const int rows = DOWN ? a.hidden : 2 * a.inner, K = DOWN ? a.inner : a.hidden;
    const uint32_t smem_base = (smem_u32(smem_dyn) + 1023u) & ~1023u;  // the same in both CTAs
    unsigned char *lists = smem_dyn + (smem_base - smem_u32(smem_dyn)) + STAGES * STAGE_BYTES;
    Group *group = reinterpret_cast<Group *>(lists);
    Entry *entry = reinterpret_cast<Entry *>(group + MOST_EXPERTS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int tiles = (rows + 2 * TN - 1) / (2 * TN), k_blocks = (K + BK - 1) / BK;
    const int pair = (int)blockIdx.x / 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&acc_full[b]), 1);
            mbar_init(smem_u32(&acc_empty[b]), 2 * 4 * EPI_GROUPS);
        }
        mbar_init(smem_u32(&drain_bar), 1);
        abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == MMA_WARP) {
        umma::alloc_pair(smem_u32(&tmem_base_slot), TMEM_COLS);
        umma::relinquish_pair();
    }
    // The plan is complete: the kernel in front waited for it, or for one that did, before it let this one start.  It comes from L2: ahead of its own wait this kernel has no promise that the SM's
    // first-level cache does not hold the plan of an earlier layer, which stood in the same place.
    const int4 sizes = __ldcg(reinterpret_cast<const int4 *>(p.plan));  // groups, entries, slots, largest
    const int groups = sizes.x, entries = sizes.y;
    const Rounds mine(tiles * entries, k_blocks, (int)gridDim.x / 2, pair, sizes.w);
    for (int i = threadIdx.x; i < groups; i += THREADS) *reinterpret_cast<uint2 *>(&group[i]) = __ldcg(reinterpret_cast<const uint2 *>(&p.plan->group[i]));
    for (int i = threadIdx.x; i < entries; i += THREADS) *reinterpret_cast<uint2 *>(&entry[i]) = __ldcg(reinterpret_cast<const uint2 *>(&p.plan->entry[i]));
    umma::fence_before_sync();
    __syncthreads();
    cluster_arrive_release();
    cluster_wait_acquire();  // both CTAs' barriers are set up and both have their tensor memory
    umma::fence_after_sync();
    pdl_launch_dependents();
    const uint32_t tmem_base = tmem_base_slot;

    auto wait = [&](uint32_t bar, uint32_t parity, unsigned int site) -> bool {
        bool ok = mbar_wait(bar, parity, umma::kFastPolls);
        if (__all_sync(0xffffffffu, ok)) return true;
        if (!ok) ok = umma::wait_or_abort<kKernelExpertsMany>(bar, parity, site, &abort_flag, a.status);
        return __all_sync(0xffffffffu, ok);
    };
    auto wait_one = [&](uint32_t bar, uint32_t parity, unsigned int site) -> bool {
        return mbar_wait(bar, parity, umma::kFastPolls) || umma::wait_or_abort<kKernelExpertsMany>(bar, parity, site, &abort_flag, a.status);
    };
    Units at(group, tiles);
    if (warp != LOAD_WARP) pdl_wait();  // no bounded wait runs against the kernel in front

    if (warp == LOAD_WARP) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            const uint64_t keep = l2_policy_evict_last(), once = l2_policy_evict_first();
            const uint32_t full0 = map_to_rank(smem_u32(&full[0]), 0);
            uint32_t i = 0, ahead = 0;
            umma::Ring r;
            bool ok = true;
            for (int t = 0; t < mine.count() && ok; ++t) {
                const int kb0 = mine.first_k(t), kb1 = mine.last_k(t);
                int expert, tile, which;
                at.find(mine.unit(t), expert, tile, which);
                const Entry en = entry[which];
                const CUtensorMap *image = &map_x.of[en.slots / SLOTS - 1];
                const int half = columns_of(en.slots) / 2, row = expert * rows + tile * 2 * TN + (int)rank * TN, x_row = DIGITS * en.slot + (int)rank * half;
                const uint64_t policy = group[at.g].entries > 1 ? keep : once;
                auto load_w = [&](uint32_t slot, int kb) {
                    if (rank == 0) mbar_expect_tx(smem_u32(&full[slot]), 2 * (W_BYTES + half * BK));
                    load_pair(smem_base + slot * STAGE_BYTES, &map_w, kb * BK, row, full0 + 8 * slot, policy);
                };
                auto load_x = [&](uint32_t slot, int kb) { load_pair(smem_base + slot * STAGE_BYTES + W_BYTES, image, kb * BK, x_row, full0 + 8 * slot, keep); };
                if (t == 0) {  // the first weights are requested before the image is complete
                    ahead = (uint32_t)min(kb1 - kb0, STAGES);
                    for (uint32_t j = 0; j < ahead; ++j) load_w(j, kb0 + (int)j);
                    pdl_wait();
                    for (uint32_t j = 0; j < ahead; ++j) load_x(j, kb0 + (int)j);
                }
                for (int kb = kb0; kb < kb1; ++kb, ++i, r.advance(1, STAGES)) {
                    if (i < ahead) continue;
                    if (i >= STAGES && !wait_one(smem_u32(&empty[r.slot]), r.phase ^ 1u, 1)) {
                        ok = false;
                        break;
                    }
                    load_w(r.slot, kb);
                    load_x(r.slot, kb);
                }
            }
            // Every copy armed must have landed before a CTA may retire; what counts them is the first CTA's barriers, and the second CTA waits for the first at the
            // cluster barrier below.  Slot s was last used for the largest j < i with j % STAGES == s.
            for (uint32_t s = 0; rank == 0 && s < STAGES; ++s) {
                if (i <= s) continue;
                const uint32_t j = i - 1 - (i - 1 - s) % STAGES;
                if (!mbar_wait(smem_u32(&full[s]), (j / STAGES) & 1)) report_timeout(a.status, kKernelExpertsMany, 7);
            }
        }
    } else if (warp == MMA_WARP) {
        // ---------------- products ----------------
        if (rank == 0 && elect_one()) {
            umma::Ring r;
            bool ok = true, here = false;
            for (int t = 0; t < mine.count() && ok; ++t) {
                const int kb0 = mine.first_k(t), kb1 = mine.last_k(t);
                int expert, tile, which;
                at.find(mine.unit(t), expert, tile, which);
                const uint32_t idesc = idesc_i8(2 * TN, columns_of(entry[which].slots), false);
                const uint32_t buf = t & 1, acc_use = (uint32_t)t >> 1;
                if (acc_use >= 1 && !wait_one(smem_u32(&acc_empty[buf]), (acc_use - 1) & 1, 3)) break;
                umma::fence_after_sync();
                const uint32_t d_addr = tmem_base + buf * MOST_COLUMNS;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!here && !wait_one(smem_u32(&full[r.slot]), r.phase, 4)) {
                        ok = false;
                        break;
                    }
                    umma::fence_after_sync();
                    const uint32_t from = smem_base + r.slot * STAGE_BYTES;
                    const uint64_t w_desc = umma::smem_desc_sw128(from), x_desc = umma::smem_desc_sw128(from + W_BYTES);
#pragma unroll
                    for (int ks = 0; ks < BK / 32; ++ks) mma_pair_i8(d_addr, w_desc + 2 * ks, x_desc + 2 * ks, idesc, (kb > kb0 || ks > 0) ? 1u : 0u);
                    commit_to(smem_u32(&empty[r.slot]), (uint16_t)3);
                    r.advance(1, STAGES);
                    here = mbar_test(smem_u32(&full[r.slot]), r.phase);
                }
                if (ok) commit_to(smem_u32(&acc_full[buf]), (uint16_t)3);
            }
            // No MMA may still be running when tensor memory is given back or the peer retires.
            umma::commit_pair_self(smem_u32(&drain_bar));
            if (!mbar_wait(smem_u32(&drain_bar), 0)) report_timeout(a.status, kKernelExpertsMany, 8);
        }
    } else {
        // ---------------- results: a lane a row of the weight, eight assignments at a time, the groups in turn ----------------
        const int eg = warp >> 2, q = warp & 3;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(32 * q) << 16);
        auto group_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + eg) : "memory"); };
        // A unit's scale is asked for a unit ahead, the powers of two eight slots ahead: with few k, results take longer than products.
        int next_tile = 0, next_which = 0;
        float next_scale = 0.0f;
        auto ask = [&](int t) {
            if (t >= mine.count()) return;
            int expert;
            at.find(mine.unit(t), expert, next_tile, next_which);
            const int n = next_tile * 2 * TN + (int)rank * TN + 32 * q + lane;
            next_scale = n < rows ? scale_at(DOWN ? a.down_scale : a.gate_up_scale, a.scale_type, (int64_t)expert * rows + n) : 0.0f;
        };
        ask(0);
        for (int t = 0; t < mine.count(); ++t) {
            const int tile = next_tile;
            const Entry en = entry[next_which];
            const float scale = next_scale;
            ask(t + 1);
            const int n = tile * 2 * TN + (int)rank * TN + 32 * q + lane;
            const bool there = n < rows;
            float4 b0, b1;
            auto ask_back = [&](int c) {
                if (c >= en.slots) return;
                b0 = __ldcg(reinterpret_cast<const float4 *>(p.back + en.slot + c)), b1 = __ldcg(reinterpret_cast<const float4 *>(p.back + en.slot + c) + 1);
            };
            ask_back(8 * eg);
            const uint32_t buf = t & 1, acc = lane_addr + buf * MOST_COLUMNS;
            if (!all_of_128(1 + eg, wait(smem_u32(&acc_full[buf]), ((uint32_t)t >> 1) & 1, 10))) break;  // the group stays or leaves as one
            umma::fence_after_sync();
            auto is_read = [&]() {
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(map_to_rank(smem_u32(&acc_empty[buf]), 0));
            };
            if (8 * eg >= en.count) {
                is_read();
                continue;
            }
            int p0 = pair, p1 = pair;
            if (mine.shared(t)) {
                // this pair's sums to the others, and whoever comes last adds them
                p0 = pair / mine.split * mine.split, p1 = p0 + mine.split - 1;
                int *to = p.parts + (int64_t)blockIdx.x * p.most_columns * TN + 32 * q + lane;
#pragma unroll 1
                for (int c = 8 * eg; c < en.count; c += 8 * EPI_GROUPS) {
                    int v[DIGITS][8];
#pragma unroll
                    for (int g = 0; g < DIGITS; ++g) ld_columns(acc + g * en.slots + c, v[g]);
                    umma::ld_wait();
#pragma unroll
                    for (int g = 0; g < DIGITS; ++g)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (c + j < en.count) __stcg(to + (g * en.count + c + j) * TN, v[g][j]);
                }
                group_sync();
                if ((threadIdx.x & 127) == 0) {
                    unsigned int *counter = p.counters + (2 * p0 + (int)rank) * EPI_GROUPS + eg, before;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
                    const bool last = before == (unsigned int)(p1 - p0);
                    if (last) *counter = 0;
                    came_last[eg] = last;
                }
                group_sync();
                if (!came_last[eg]) {
                    is_read();
                    continue;
                }
            }
#pragma unroll 1
            for (int c = 8 * eg; c < en.count; c += 8 * EPI_GROUPS) {
                int v[DIGITS][8];
#pragma unroll
                for (int g = 0; g < DIGITS; ++g) ld_columns(acc + g * en.slots + c, v[g]);
                umma::ld_wait();
                if (c + 8 * EPI_GROUPS >= en.count) is_read();
                for (int other = p0; other <= p1; ++other) {
                    if (other == pair) continue;
                    const int *from = p.parts + (int64_t)(2 * other + (int)rank) * p.most_columns * TN + 32 * q + lane;
#pragma unroll
                    for (int g = 0; g < DIGITS; ++g)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (c + j < en.count) v[g][j] += __ldcg(from + (g * en.count + c + j) * TN);
                }
                const int slot = en.slot + c;
                const float back[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
                ask_back(c + 8 * EPI_GROUPS);
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = fmaf((float)v[2][j], 65536.0f, fmaf((float)v[1][j], 256.0f, (float)v[0][j])) * scale * back[j];  // the scale first: it and the power of two may be small together
                if (DOWN) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (there && c + j < en.count) p.rows[(int64_t)(slot + j) * rows + n] = y[j];
                } else {
                    // even lanes have gates, odd ones what they multiply; of two columns each lane of a pair finishes one
                    const bool odd = lane & 1;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float other = __shfl_xor_sync(0xffffffffu, odd ? y[j] : y[j + 1], 1);
                        const int mine = j + (odd ? 1 : 0);
                        const float h = silu(odd ? other : y[j]) * (odd ? y[j + 1] : other);
                        uint32_t bits = 0;
                        if (there && c + mine < en.count) {
                            p.rows[(int64_t)(slot + mine) * a.inner + (n >> 1)] = h;
                            bits = __float_as_uint(h) & 0x7fffffffu;
                        }
                        const uint32_t even_most = __reduce_max_sync(0xffffffffu, odd ? 0u : bits), odd_most = __reduce_max_sync(0xffffffffu, odd ? bits : 0u);
                        if (lane < 2 && c + mine < en.count) p.largest[(int64_t)(slot + mine) * p.maxima + 8 * tile + 4 * rank + q] = odd ? odd_most : even_most;
                    }
                }
            }
        }
    }
    // ---------------- both CTAs are done with each other's shared and tensor memory ----------------
    __syncwarp();
    umma::fence_before_sync();
    cluster_arrive_release();
    cluster_wait_acquire();
    if (warp == MMA_WARP) {
        umma::fence_after_sync();
        umma::dealloc_pair(tmem_base, TMEM_COLS);
    }
}

// ---------------- join ----------------
constexpr int JOIN_THREADS = 256;

// Four columns a thread; hidden is a multiple of 16.  VEC: the result and the residual in lines of eight bytes.
template <bool VEC, bool BF16>
__global__ void __launch_bounds__(JOIN_THREADS) experts_join_kernel(const ManyArgs p) {
    const ExpertsArgs &a = p.a;
    const int t = blockIdx.x, n = (blockIdx.y * JOIN_THREADS + threadIdx.x) * 4;
    pdl_launch_dependents();
    pdl_wait();
    if (n >= a.hidden) return;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int j = 0; j < a.top; ++j) {
        const int slot = p.slot_of[(int64_t)t * a.top + j];
        if (slot < 0) continue;
        const float w = a.weights[(int64_t)t * a.top + j];
        const float4 y = __ldcg(reinterpret_cast<const float4 *>(p.rows + (int64_t)slot * a.hidden + n));
        sum[0] = fmaf(y.x, w, sum[0]), sum[1] = fmaf(y.y, w, sum[1]), sum[2] = fmaf(y.z, w, sum[2]), sum[3] = fmaf(y.w, w, sum[3]);
    }
    const int64_t from = (int64_t)t * a.residual_stride + n, to = (int64_t)t * a.hidden + n;
    union {
        uint2 v;
        uint16_t e[4];
    } r;
    if (a.residual != nullptr) {
        if (VEC) {
            r.v = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.residual) + from);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) r.e[i] = static_cast<const uint16_t *>(a.residual)[from + i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += BF16 ? __bfloat162float(__ushort_as_bfloat16(r.e[i])) : __half2float(__ushort_as_half(r.e[i]));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) r.e[i] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(sum[i])) : __half_as_ushort(__float2half_rn(sum[i]));
    if (VEC) {
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + to) = r.v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) static_cast<uint16_t *>(a.out)[to + i] = r.e[i];
    }
}

// ---------------- launches ----------------
int64_t slots_for(int64_t assignments, int64_t count) {
    const int64_t entries = (assignments < count ? assignments : count) + assignments / MOST;
    return assignments + (SLOTS - 1) * entries;
}
int pairs_of() {
    const int pairs = (sm_count() > 0 ? sm_count() : 148) / 2;
    return pairs < MOST_PAIRS ? pairs : MOST_PAIRS;
}
struct Places {
    size_t slot, back, slot_of, largest, rows, image, parts, bytes;
    int most_columns, maxima;
};
Places places_for(int64_t assignments, int64_t hidden, int64_t inner, int64_t count) {
    const int64_t slots = round_up(slots_for(assignments, count), SLOTS), widest = hidden > inner ? hidden : inner;
    Places p = {};
    size_t at = (size_t)round_up((int64_t)sizeof(Plan), 256);
    auto take = [&](int64_t bytes) {
        const size_t here = at;
        at += (size_t)round_up(bytes, 256);
        return here;
    };
    p.slot = take(slots * (int64_t)sizeof(Slot)), p.back = take(slots * 4), p.slot_of = take(assignments * 4);
    p.maxima = 8 * (int)ceil_div(2 * inner, 2 * TN);
    p.largest = take(slots * p.maxima * 4);
    p.rows = take(slots * widest * 4), p.image = take(slots * widest * DIGITS);
    p.most_columns = DIGITS * (int)(assignments < MOST ? assignments : MOST);
    p.parts = take((int64_t)2 * pairs_of() * p.most_columns * TN * 4);
    p.bytes = at;
    return p;
}
constexpr size_t kMostBytes = (size_t)511 << 20;  // with the workspace's head half a gigabyte.  Half of it: 2048 tokens, two of eight experts of 4096 x 14336, in four parts, 2.3 ms for 2.0

template <bool DOWN>
int launch_product(const ManyArgs &p, cudaStream_t stream) {
    const ExpertsArgs &a = p.a;
    const int64_t rows = DOWN ? a.hidden : 2 * (int64_t)a.inner, K = DOWN ? a.inner : a.hidden;
    CUtensorMap map_w;
    ImageMaps map_x;
    int rc = make_tensor_map_2d(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, DOWN ? a.down : a.gate_up, (uint64_t)K, (uint64_t)(a.count * rows), (uint64_t)K, BK, TN, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != B200Q_OK) return rc;
    for (int i = 0; i < MOST / SLOTS; ++i) {
        rc = make_tensor_map_2d(&map_x.of[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, p.image, (uint64_t)K, (uint64_t)(DIGITS * (int64_t)p.most_slots), (uint64_t)K, BK,
                                (uint32_t)columns_of((i + 1) * SLOTS) / 2, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
        if (rc != B200Q_OK) return rc;
    }
    static std::atomic<bool> attr_set[64];
    rc = allow_smem(attr_set, experts_product_kernel<DOWN>, SMEM_BYTES);
    if (rc != B200Q_OK) return rc;
    return launch_after("experts_product_kernel", experts_product_kernel<DOWN>, dim3((unsigned)(2 * pairs_of())), THREADS, (size_t)SMEM_BYTES, 2, stream, map_w, map_x, p);
}

template <typename X, bool OF_H>
int launch_image(const ManyArgs &p, cudaStream_t stream) {
    // few slots: a CTA 2048 elements, as long as all CTAs run at once (64 rows of 14336: 6.5 us for 10)
    const int64_t pieces = ceil_div(OF_H ? p.a.inner : p.a.hidden, IMAGE_THREADS * 8), room = 8 * 148 / p.most_slots;
    const int64_t share = room < 1 ? 1 : room < pieces ? room : pieces;
    return launch_after("experts_image_kernel", experts_image_kernel<X, OF_H>, dim3((unsigned)p.most_slots, (unsigned)share), IMAGE_THREADS, 0, 1, stream, p);
}

}  // namespace

int64_t experts_many_at_once(int64_t tokens, int64_t hidden, int64_t inner, int64_t count, int64_t top) {
    int64_t most = (int64_t)kMostBytes / ((4 + DIGITS) * (hidden > inner ? hidden : inner));  // assignments
    if (most > MOST_ASSIGNMENTS) most = MOST_ASSIGNMENTS;
    while (most > SLOTS && places_for(most, hidden, inner, count).bytes > kMostBytes) most -= most / 16 > 0 ? most / 16 : 1;
    most = most / top > 1 ? most / top : 1;
    return ceil_div(tokens, ceil_div(tokens, most));  // parts of one size
}

size_t experts_many_bytes(int64_t tokens, int64_t hidden, int64_t inner, int64_t count, int64_t top) { return places_for(tokens * top, hidden, inner, count).bytes; }

int launch_experts_many(const ExpertsArgs &a, unsigned int *counters, void *scratch, cudaStream_t stream) {
    const Places at = places_for((int64_t)a.tokens * a.top, a.hidden, a.inner, a.count);
    char *base = static_cast<char *>(scratch);
    ManyArgs p = {};
    p.a = a, p.counters = counters, p.plan = reinterpret_cast<Plan *>(base), p.slot = reinterpret_cast<Slot *>(base + at.slot), p.back = reinterpret_cast<float *>(base + at.back);
    p.slot_of = reinterpret_cast<int *>(base + at.slot_of), p.rows = reinterpret_cast<float *>(base + at.rows), p.image = reinterpret_cast<int8_t *>(base + at.image);
    p.largest = reinterpret_cast<uint32_t *>(base + at.largest), p.maxima = at.maxima, p.parts = reinterpret_cast<int *>(base + at.parts), p.most_columns = at.most_columns;
    p.most_slots = (int)round_up(slots_for((int64_t)a.tokens * a.top, a.count), SLOTS);
    int rc = launch_after("experts_plan_kernel", experts_plan_kernel, dim3(1), PLAN_THREADS, 0, 1, stream, p);
    if (rc == B200Q_OK) rc = a.type == B200Q_F16 ? launch_image<FromF16, false>(p, stream) : launch_image<FromBF16, false>(p, stream);
    if (rc == B200Q_OK) rc = launch_product<false>(p, stream);
    if (rc == B200Q_OK) rc = launch_image<FromF32, true>(p, stream);
    if (rc == B200Q_OK) rc = launch_product<true>(p, stream);
    if (rc != B200Q_OK) return rc;
    const bool vec = aligned_to(a.out, 8) && (a.residual == nullptr || (aligned_to(a.residual, 8) && (a.tokens == 1 || a.residual_stride % 4 == 0)));
    const dim3 grid((unsigned)a.tokens, (unsigned)ceil_div(a.hidden, JOIN_THREADS * 4));
    if (a.type == B200Q_F16) return vec ? launch_after("experts_join_kernel", experts_join_kernel<true, false>, grid, JOIN_THREADS, 0, 1, stream, p) : launch_after("experts_join_kernel", experts_join_kernel<false, false>, grid, JOIN_THREADS, 0, 1, stream, p);
    return vec ? launch_after("experts_join_kernel", experts_join_kernel<true, true>, grid, JOIN_THREADS, 0, 1, stream, p) : launch_after("experts_join_kernel", experts_join_kernel<false, true>, grid, JOIN_THREADS, 0, 1, stream, p);
}

}  // namespace b200q
