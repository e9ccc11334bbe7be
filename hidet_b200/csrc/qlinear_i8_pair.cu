// The int8 x int8 product for many tokens, on pairs of SMs: tcgen05.mma kind::i8 with cta_group::2.
//
// Computed transposed, D[n, m] = sum_k w[k, n] a[m, k], sums of 32 bits in tensor memory: a pair owns 256 channels x tm tokens (tm a multiple of 32, at most
// 256), of which each CTA fetches its own 128 channels and half of the tokens, 128 k a stage, straight into the form that the tensor core reads; nothing is
// converted.  Tokens are the columns because their number is what comes in odd sizes: tm follows it in steps of 32, where lanes go by 256.  A weight [N, K] is a
// K-major operand, one [K, N] an MN-major one.
//
// One persistent CTA per SM, ten warps:
//   warps 0-7  epilogue, two groups that take the 32-token blocks of a tile in turn: tensor memory -> float, the two scales, bias, gate / up pairing, residual ->
//              16 bits, transposed through a staging buffer (two per group, taken in turn) by matrix stores, 16-byte stores of whole output rows
//   warp 8     TMA producer; both CTAs' copies count on the first CTA's barrier
//   warp 9     MMA issuer (first CTA of the pair only), one thread for the whole loop
// Two accumulators, so that a tile's epilogue runs beside the next one's products.  With few k the epilogue is what takes the time (4096 x 1024 x 4096: 20 us, 11 without it), and what it reads
// is asked for ahead: scales a tile, the residual a tile (into L2) and a block, tokens' scales a block (2048 x 512 x 8192 with a residual: 34 us without, 29 with).  Four groups
// instead of two have registers for too little of that (26 us for 20).
//
// Where tiles are few, K is shared by the two or four pairs of a cluster, a tile each cluster and no second one.  Sums are whole numbers: when all have theirs, every pair
// hands the others the 32-token blocks that they finish (its fragments as they come out of tensor memory, into the ring, which is no longer in use) and adds what it gets.
//
// Every wait is bounded: a wait that runs out records where and raises a CTA-wide flag, all roles leave, the first CTA waits for what was armed and issued, and the
// two CTAs meet at a cluster barrier before either gives back tensor memory or retires.
#include <atomic>
#include <type_traits>

#include "qlinear_i8.h"
#include "umma.cuh"
#include "umma_i8_pair.cuh"

namespace b200q {
namespace i8pair {

constexpr unsigned int kKernelI8Pair = 12;
constexpr int TN = 128;                      // channels per CTA; a pair's tile has twice as many
constexpr int BK = 128;                      // k per stage = four MMAs of K = 32
constexpr int W_BYTES = BK * TN;
constexpr int MAX_STAGES = 10;
constexpr int EPI_GROUPS = 2;
constexpr int LOAD_WARP = 4 * EPI_GROUPS, MMA_WARP = LOAD_WARP + 1;
constexpr int THREADS = 32 * (MMA_WARP + 1);
constexpr int TMEM_COLS = 512;
constexpr int ROW_BYTES = TN * 2 + 16;       // one output row in the staging buffer, padded: matrix stores touch every bank once
constexpr int STAGING_BYTES = 32 * ROW_BYTES;
constexpr int FRAGMENT_BYTES = 32 * 32 * 4;  // a warp's part of a block's sums
constexpr int RING_BYTES = 188 * 1024;
constexpr int SMEM_BYTES = RING_BYTES + EPI_GROUPS * 2 * STAGING_BYTES + 1024;  // + alignment slack

struct Params {
    I8Args a;
    int tm;                    // tokens per tile
    int n_tiles, m_tiles;
    int band;                  // token tiles that are walked together, channel tile by channel tile
    int k_blocks;
    int stages;
    int split;                 // pairs of a cluster, which share K
};

__device__ __forceinline__ void tile_of(const Params &p, int u, int &n0, int &m0) {
    const int band_tiles = p.band * p.n_tiles;
    const int b = u / band_tiles, r = u - b * band_tiles;
    const int rows = min(p.band, p.m_tiles - b * p.band);
    const int n = r / rows;
    n0 = n * 2 * TN;
    m0 = (b * p.band + (r - n * rows)) * p.tm;
}

// A tile of [k][128 channels] in rows of 128 swizzled bytes: 8-row groups 1024 bytes apart, both strides (there is one group of channels, so that one of them is not used).
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | (64ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
template <bool BF16>
__device__ __forceinline__ float value_at(const void *p, int64_t i) {
    return BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]) : __half2float(static_cast<const __half *>(p)[i]);
}

// NK: the weight is [N, K].  PAIRS: channels (2j, 2j + 1) = (gate, up).
template <bool NK, bool BF16, bool PAIRS>
__global__ void __launch_bounds__(THREADS, 1)
    i8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const Params p) {
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) uint64_t full[MAX_STAGES];    // (first CTA) both CTAs' tiles of the stage have landed
    __shared__ __align__(8) uint64_t empty[MAX_STAGES];   // the MMAs that read it have completed
    __shared__ __align__(8) uint64_t acc_full[2];         // an accumulator holds a finished tile
    __shared__ __align__(8) uint64_t acc_empty[2];        // (first CTA) both CTAs' epilogue warps have read it out
    __shared__ __align__(8) uint64_t drain_bar;           // every MMA issued has completed (teardown)
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;

    const uint32_t smem_base = (smem_u32(smem_dyn) + 1023u) & ~1023u;  // swizzled operands; the same in both CTAs
    unsigned char *smem_gen = smem_dyn + (smem_base - smem_u32(smem_dyn));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cluster_rank = cluster_ctarank(), rank = cluster_rank & 1u, lead = cluster_rank & ~1u;  // in the pair; the pair's first CTA
    const int units = p.n_tiles * p.m_tiles, share = (int)(cluster_rank >> 1);
    const int first = blockIdx.x / (2 * p.split), step = gridDim.x / (2 * p.split);
    const int kb0 = p.k_blocks * share / p.split, kb1 = p.k_blocks * (share + 1) / p.split;
    const uint32_t stages = p.stages, stage_bytes = W_BYTES + (uint32_t)p.tm * (BK / 2);
    constexpr int STAGING_OFF = RING_BYTES;

    if (threadIdx.x == 0) {
        for (int s = 0; s < MAX_STAGES; ++s) {
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
    umma::fence_before_sync();
    __syncthreads();
    cluster_arrive_release();
    cluster_wait_acquire();  // both CTAs' barriers are set up and both have their tensor memory
    umma::fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    if (lane == 0 && warp == LOAD_WARP) {
        tma_prefetch_desc(&map_w);
        tma_prefetch_desc(&map_a);
    }
    if (warp != LOAD_WARP) pdl_wait();  // every other role: none of their bounded waits runs against the kernel in front

    auto wait = [&](uint32_t bar, uint32_t parity, unsigned int site) -> bool {
        bool ok = mbar_wait(bar, parity, umma::kFastPolls);
        if (__all_sync(0xffffffffu, ok)) return true;
        if (!ok) ok = umma::wait_or_abort<kKernelI8Pair>(bar, parity, site, &abort_flag, p.a.status);
        return __all_sync(0xffffffffu, ok);
    };
    auto wait_one = [&](uint32_t bar, uint32_t parity, unsigned int site) -> bool {
        return mbar_wait(bar, parity, umma::kFastPolls) || umma::wait_or_abort<kKernelI8Pair>(bar, parity, site, &abort_flag, p.a.status);
    };

    // Where pairs share K, all threads of their cluster meet twice: when the sums are complete, and when they have been handed over.
    auto meet = [&]() {
        if (p.split == 1) return;
        __syncwarp();
        cluster_arrive_release();
        cluster_wait_acquire();
    };

    if (warp == LOAD_WARP) {
        // ---------------- TMA producer ----------------
        pdl_launch_dependents();  // tensor memory is allocated: a kernel that is placed as this one's CTAs leave cannot take it away
        if (lane == 0) {
            const uint64_t keep = l2_policy_evict_last();  // both operands are read again by other tiles
            const uint32_t full0 = map_to_rank(smem_u32(&full[0]), lead);
            auto load_w = [&](uint32_t slot, int n, int kb) {
                if (rank == 0) mbar_expect_tx(smem_u32(&full[slot]), 2 * stage_bytes);
                load_pair(smem_base + slot * stage_bytes, &map_w, NK ? kb * BK : n, NK ? n : kb * BK, full0 + 8 * slot, keep);
            };
            auto load_a = [&](uint32_t slot, int m, int kb) { load_pair(smem_base + slot * stage_bytes + W_BYTES, &map_a, kb * BK, m, full0 + 8 * slot, keep); };
            // The first tile's weights are asked for into L2 before the kernel in front has finished, which may be the one that writes them; they come from there behind it, with the tokens.
            int n, m;
            tile_of(p, first, n, m);
            n += (int)rank * TN;
            m += (int)rank * (p.tm / 2);
            const int ahead = min(kb1 - kb0, (int)stages);
            for (int j = 0; j < ahead; ++j) tma_prefetch_2d(&map_w, NK ? (kb0 + j) * BK : n, NK ? n : (kb0 + j) * BK);
            pdl_wait();
            for (int j = 0; j < ahead; ++j) load_w(j, n, kb0 + j), load_a(j, m, kb0 + j);
            uint32_t i = 0;
            umma::Ring r;
            bool ok = true;
            for (int u = first; u < units && ok; u += step) {
                tile_of(p, u, n, m);
                n += (int)rank * TN;
                m += (int)rank * (p.tm / 2);
                for (int kb = kb0; kb < kb1; ++kb, ++i, r.advance(1, stages)) {
                    if (i < (uint32_t)ahead) continue;
                    if (i >= stages && !wait_one(smem_u32(&empty[r.slot]), r.phase ^ 1u, 1)) {
                        ok = false;
                        break;
                    }
                    load_w(r.slot, n, kb);
                    load_a(r.slot, m, kb);
                }
            }
            // Teardown: every copy armed must have landed before a CTA may retire; what counts them is the first CTA's barriers, and the second CTA
            // waits for the first at the cluster barrier below.  Slot s was last used for the largest j < i with j % stages == s.
            for (uint32_t s = 0; rank == 0 && s < stages; ++s) {
                if (i <= s) continue;
                const uint32_t j = i - 1 - (i - 1 - s) % stages;
                if (!mbar_wait(smem_u32(&full[s]), (j / stages) & 1)) report_timeout(p.a.status, kKernelI8Pair, 7);
            }
        }
        meet();
        meet();
    } else if (warp == MMA_WARP) {
        // ---------------- MMA issuer ----------------
        if (rank == 0 && elect_one()) {
            const uint32_t idesc = idesc_i8(2 * TN, p.tm, !NK);
            const uint16_t both = (uint16_t)(3u << lead);
            constexpr uint32_t W_STEP = NK ? 32 / 16 : 32 * TN / 16;  // of the weight's descriptor, 32 k on
            uint32_t t_iter = 0;
            umma::Ring r;
            bool ok = true, here = false;
            for (int u = first; u < units && ok; u += step, ++t_iter) {
                const uint32_t buf = t_iter & 1, acc_use = t_iter >> 1;
                if (acc_use >= 1 && !wait_one(smem_u32(&acc_empty[buf]), (acc_use - 1) & 1, 3)) break;
                umma::fence_after_sync();
                const uint32_t d_addr = tmem_base + buf * p.tm;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!here && !wait_one(smem_u32(&full[r.slot]), r.phase, 4)) {
                        ok = false;
                        break;
                    }
                    umma::fence_after_sync();
                    const uint32_t at = smem_base + r.slot * stage_bytes;
                    const uint64_t w_desc = NK ? umma::smem_desc_sw128(at) : smem_desc_mn(at), a_desc = umma::smem_desc_sw128(at + W_BYTES);
#pragma unroll
                    for (int ks = 0; ks < BK / 32; ++ks) mma_pair_i8(d_addr, w_desc + W_STEP * ks, a_desc + 2 * ks, idesc, (kb > kb0 || ks > 0) ? 1u : 0u);
                    commit_to(smem_u32(&empty[r.slot]), both);
                    r.advance(1, stages);
                    here = mbar_test(smem_u32(&full[r.slot]), r.phase);
                }
                if (ok) commit_to(smem_u32(&acc_full[buf]), both);
            }
            // Teardown: no MMA may still be running when tensor memory is given back or the peer retires.
            umma::commit_pair_self(smem_u32(&drain_bar));
            if (!mbar_wait(smem_u32(&drain_bar), 0)) report_timeout(p.a.status, kKernelI8Pair, 8);
        }
        meet();
        meet();
    } else {
        // ---------------- epilogue ----------------
        const int eg = warp >> 2;               // takes blocks eg, eg + EPI_GROUPS, ...
        const int q = warp & 3;                 // tensor-memory lanes 32 q .. 32 q + 31
        const int et = 32 * q + lane;           // 0 .. 127
        auto group_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + eg) : "memory"); };
        const int g = lane >> 2, tq = lane & 3; // fragment coordinates: channel g of 8, tokens 2 tq, 2 tq + 1 of 8
        const int M = p.a.M, N = p.a.N;
        const void *res = p.a.residual;
        const bool res_vec = !PAIRS && p.a.residual_vec;
        const int out_n = PAIRS ? N >> 1 : N;
        constexpr int ROW_CHUNKS_LOG2 = PAIRS ? 3 : 4;         // 16-byte pieces of a tile's output row
        const int chunk = et & ((1 << ROW_CHUNKS_LOG2) - 1);
        const int row_in_pass = et >> ROW_CHUNKS_LOG2;
        constexpr int PASS_ROWS = 128 >> ROW_CHUNKS_LOG2;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(32 * q) << 16);
        uint32_t t_iter = 0, block = 0;         // block: the group's 32-token blocks so far, staging buffers in turn
        // A tile's residual comes to L2 a tile ahead, a row a thread: a block of it on its way is not enough for its way from memory.
        auto prefetch_residual = [&](int u) {
            if (PAIRS || res == nullptr || u >= units) return;
            int n, m;
            tile_of(p, u, n, m);
            n += (int)rank * TN;
            const int width = min(TN, N - n);
            for (int r = 128 * eg + et; r < min(M - m, p.tm); r += 128 * EPI_GROUPS) {
                const char *row = static_cast<const char *>(res) + ((int64_t)(m + r) * p.a.ldr + n) * 2;
                for (int i = 0; i < width; i += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + 2 * i));
            }
        };
        float next_sc[2][2], next_bias[2][2];  // [16-channel block][8-channel half]: channel 16 h + 8 e + g of this warp's 32
        auto ask_scales = [&](int u) {
            if (u >= units) return;
            int n0, m0;
            tile_of(p, u, n0, m0);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int n = n0 + (int)rank * TN + 32 * q + 16 * h + 8 * e + g;
                    next_sc[h][e] = n < N ? i8_scale(p.a.scale, p.a.scale_type, n) : 0.0f;
                    next_bias[h][e] = n < N && p.a.bias != nullptr ? value_at<BF16>(p.a.bias, n) : 0.0f;
                }
        };
        ask_scales(first);
        prefetch_residual(first);
        for (int u = first; u < units; u += step, ++t_iter) {
            int n0, m0;
            tile_of(p, u, n0, m0);
            n0 += (int)rank * TN;
            prefetch_residual(u + step);
            const uint32_t buf = t_iter & 1, acc_use = t_iter >> 1;
            const int m_left = min(M - m0, p.tm);
            const int blocks = (m_left + 31) / 32;
            const uint32_t acc = lane_addr + buf * p.tm;
            float sc[2][2], bias[2][2];
            memcpy(sc, next_sc, sizeof(sc)), memcpy(bias, next_bias, sizeof(bias));
            ask_scales(u + step);
            const int out_n0 = PAIRS ? n0 >> 1 : n0;
            const bool cols_ok = out_n0 + chunk * 8 < out_n;  // widths are multiples of 8: eight channels are in or out together
            // What a block needs from memory is asked for a block ahead: with few k it is what takes the time.
            uint4 next_res[4];
            float next_sa[4][2];  // token 8 j + 2 tq + i
            auto ask = [&](int cb) {
#pragma unroll
                for (int pass = 0; res_vec && pass < 4; ++pass) {
                    const int m = cb * 32 + pass * 8 + row_in_pass;
                    next_res[pass] = make_uint4(0, 0, 0, 0);
                    if (m < m_left && cols_ok) next_res[pass] = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(res) + (size_t)(m0 + m) * p.a.ldr + out_n0 + chunk * 8));
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int m = cb * 32 + 8 * j + 2 * tq + i;
                        next_sa[j][i] = m < m_left ? p.a.a_scale[m0 + m] : 0.0f;
                    }
            };
            ask(share + p.split * eg);
            const bool ok = all_of_128(1 + eg, wait(smem_u32(&acc_full[buf]), acc_use & 1, 10));  // the group stays or leaves as one
            if (!ok && p.split == 1) break;
            umma::fence_after_sync();
            if (p.split > 1) {
                // Block cb is finished by pair cb % split, as the (cb / split)-th of its blocks.
                meet();
                const int of_each = (blocks + p.split - 1) / p.split;
                for (int cb = 0; ok && cb < blocks; ++cb) {
                    const int owner = cb % p.split, nth = cb / p.split;
                    if (owner == share || nth % EPI_GROUPS != eg) continue;
                    uint32_t v[2][16];
                    umma::ld_16x256b_x4(acc + cb * 32, v[0]);
                    umma::ld_16x256b_x4(acc + (16u << 16) + cb * 32, v[1]);
                    umma::ld_wait();
                    const uint32_t to = map_to_rank(smem_base + (uint32_t)((share * of_each + nth) * 4 + q) * FRAGMENT_BYTES + lane * 16, 2 * owner + rank);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + i * 512), "r"(v[i >> 2][4 * (i & 3)]), "r"(v[i >> 2][4 * (i & 3) + 1]),
                                     "r"(v[i >> 2][4 * (i & 3) + 2]), "r"(v[i >> 2][4 * (i & 3) + 3])
                                     : "memory");
                }
                meet();
                if (!ok) break;
            }
            const size_t out_off = (size_t)m0 * out_n + out_n0 + chunk * 8;
            if (p.split == 1 && eg >= blocks) {  // a tile of a single block: nothing for this group
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(map_to_rank(smem_u32(&acc_empty[buf]), lead));
            }
#pragma unroll 1
            for (int cb = share + p.split * eg; cb < blocks; cb += p.split * EPI_GROUPS, ++block) {
                unsigned char *staging = smem_gen + STAGING_OFF + (2 * eg + (block & 1)) * STAGING_BYTES;
                const uint32_t staging_a = smem_base + STAGING_OFF + (2 * eg + (block & 1)) * STAGING_BYTES;
                float sa[4][2];
                memcpy(sa, next_sa, sizeof(sa));
                if (res_vec) {
                    // the residual's block goes through the staging buffer into the fragments' layout
#pragma unroll
                    for (int pass = 0; pass < 4; ++pass) *reinterpret_cast<uint4 *>(staging + (pass * 8 + row_in_pass) * ROW_BYTES + chunk * 16) = next_res[pass];
                    group_sync();
                }
                ask(cb + p.split * EPI_GROUPS);
                uint32_t v[2][16];
                umma::ld_16x256b_x4(acc + cb * 32, v[0]);
                umma::ld_16x256b_x4(acc + (16u << 16) + cb * 32, v[1]);
                umma::ld_wait();
                if (p.split > 1) {
                    const int of_each = (blocks + p.split - 1) / p.split;
                    for (int from = 0; from < p.split; ++from) {
                        if (from == share) continue;
                        const unsigned char *at = smem_gen + ((from * of_each + cb / p.split) * 4 + q) * FRAGMENT_BYTES + lane * 16;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint4 w = *reinterpret_cast<const uint4 *>(at + i * 512);
                            v[i >> 2][4 * (i & 3)] += w.x, v[i >> 2][4 * (i & 3) + 1] += w.y, v[i >> 2][4 * (i & 3) + 2] += w.z, v[i >> 2][4 * (i & 3) + 3] += w.w;
                        }
                    }
                } else if (cb + EPI_GROUPS >= blocks) {  // the group's part of the accumulator is in registers
                    umma::fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_remote(map_to_rank(smem_u32(&acc_empty[buf]), lead));
                }
                // v[h][4 j + 2 e + i]: channel 16 h + 8 e + g, token 8 j + 2 tq + i
                auto sum_of = [&](int h, int j, int e, int i) { return fmaf((float)(int)v[h][4 * j + 2 * e + i] * sc[h][e], sa[j][i], bias[h][e]); };
                if (PAIRS) {
                    // Lanes with even g hold gates, the lanes with g + 1 what they multiply; of the two 8-channel halves each lane of such a pair finishes one,
                    // for its two tokens.
                    const bool odd = g & 1;
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        float z[2][2][2];  // [token block j, j + 1][channel block h][token]
#pragma unroll
                        for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    const float y0 = sum_of(h, j + jj, 0, i), y1 = sum_of(h, j + jj, 1, i);
                                    const float other = __shfl_xor_sync(0xffffffffu, odd ? y0 : y1, 4);
                                    z[jj][h][i] = silu(odd ? other : y0) * (odd ? y1 : other);
                                }
                        if (res != nullptr) {
#pragma unroll
                            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
#pragma unroll
                                    for (int i = 0; i < 2; ++i) {
                                        const int oc = out_n0 + 16 * q + 8 * h + (odd ? 4 : 0) + (g >> 1), m = cb * 32 + 8 * (j + jj) + 2 * tq + i;
                                        if (oc < out_n && m < m_left) z[jj][h][i] += value_at<BF16>(res, (int64_t)(m0 + m) * p.a.ldr + oc);
                                    }
                        }
                        uint32_t pk[4];
#pragma unroll
                        for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                            for (int h = 0; h < 2; ++h) pk[2 * jj + h] = pack2<BF16>(z[jj][h][0], z[jj][h][1]);
                        // result channel g / 2 (even g) or 4 + g / 2 (odd g) of each 8: stored in the order of g, put right on the way out
                        const int mi = lane >> 3;
                        umma::stmatrix_x4_trans(staging_a + (8 * (j + (mi >> 1)) + (lane & 7)) * ROW_BYTES + (16 * q + 8 * (mi & 1)) * 2, pk);
                    }
                } else {
                    // RESIDUAL: none, vectors in the staging buffer, elements.  Apart, since a branch inside would keep one value's instructions from another's.
                    auto finish = [&](auto residual) {
                        constexpr int RESIDUAL = decltype(residual)::value;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t place = staging_a + (8 * j + (lane & 7)) * ROW_BYTES + (32 * q + 8 * (lane >> 3)) * 2;
                            uint32_t rs[4], pk[4];
                            if (RESIDUAL == 1) umma::ldmatrix_x4_trans(rs, place);
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    float y[2] = {sum_of(h, j, e, 0), sum_of(h, j, e, 1)};
                                    if (RESIDUAL == 1) {
                                        const float2 r2 = unpack2<BF16>(rs[2 * h + e]);
                                        y[0] += r2.x;
                                        y[1] += r2.y;
                                    } else if (RESIDUAL == 2) {
                                        const int n = n0 + 32 * q + 16 * h + 8 * e + g;
#pragma unroll
                                        for (int i = 0; i < 2; ++i) {
                                            const int m = cb * 32 + 8 * j + 2 * tq + i;
                                            if (n < N && m < m_left) y[i] += value_at<BF16>(res, (int64_t)(m0 + m) * p.a.ldr + n);
                                        }
                                    }
                                    pk[2 * h + e] = pack2<BF16>(y[0], y[1]);
                                }
                            umma::stmatrix_x4_trans(place, pk);
                        }
                    };
                    if (res == nullptr) finish(std::integral_constant<int, 0>());
                    else if (res_vec) finish(std::integral_constant<int, 1>());
                    else finish(std::integral_constant<int, 2>());
                }
                group_sync();  // the four warps: block complete; the other buffer is free
#pragma unroll 4
                for (int r = row_in_pass; r < 32; r += PASS_ROWS) {
                    const int m = cb * 32 + r;
                    if (m < m_left && cols_ok) {
                        uint4 val = *reinterpret_cast<const uint4 *>(staging + r * ROW_BYTES + chunk * 16);
                        if (PAIRS) {  // channels stand in the order 0 4 1 5 2 6 3 7
                            val = make_uint4(__byte_perm(val.x, val.y, 0x5410), __byte_perm(val.z, val.w, 0x5410), __byte_perm(val.x, val.y, 0x7632),
                                             __byte_perm(val.z, val.w, 0x7632));
                        }
                        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.a.c) + out_off + (size_t)m * out_n) = val;
                    }
                }
            }
        }
    }

    // ---------------- teardown: both CTAs are done with each other's shared and tensor memory ----------------
    __syncwarp();
    umma::fence_before_sync();
    cluster_arrive_release();
    cluster_wait_acquire();
    if (warp == MMA_WARP) {
        umma::fence_after_sync();
        umma::dealloc_pair(tmem_base, TMEM_COLS);
    }
}

template <bool NK, bool BF16, bool PAIRS>
int launch_as(const CUtensorMap &map_w, const CUtensorMap &map_a, const Params &p, unsigned grid, cudaStream_t stream) {
    static std::atomic<bool> attr_set[64];  // per device; a repeated set by a racing thread is harmless
    int dev = 0;
    B200Q_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
        B200Q_CUDA_TRY(cudaFuncSetAttribute(i8_pair_kernel<NK, BF16, PAIRS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = 2 * (unsigned)p.split;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    B200Q_CUDA_TRY(cudaLaunchKernelEx(&cfg, i8_pair_kernel<NK, BF16, PAIRS>, map_w, map_a, p));
    return B200Q_OK;
}

}  // namespace i8pair

int launch_i8_pair(const I8Args &a, int tm, int split, cudaStream_t stream) {
    using namespace i8pair;
    CUtensorMap map_w, map_a;
    int rc = a.nk ? make_tensor_map_2d(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, (uint64_t)a.K, (uint64_t)a.N, (uint64_t)a.K, BK, TN, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B)
                  : make_tensor_map_2d(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, (uint64_t)a.N, (uint64_t)a.K, (uint64_t)a.N, TN, BK, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != B200Q_OK) return rc;
    rc = make_tensor_map_2d(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.a, (uint64_t)a.K, (uint64_t)a.M, (uint64_t)a.K, BK, (uint32_t)(tm / 2), CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != B200Q_OK) return rc;
    Params p = {};
    p.a = a;
    p.tm = tm;
    p.n_tiles = (int)ceil_div(a.N, 2 * TN);
    p.m_tiles = (int)ceil_div(a.M, tm);
    // as many token tiles in a band as leave the band's codes well inside L2
    int64_t band = ((int64_t)48 << 20) / ((int64_t)tm * a.K);
    if (band < 1) band = 1;
    p.band = (int)(band < p.m_tiles ? band : p.m_tiles);
    p.k_blocks = (int)ceil_div(a.K, BK);
    const int stages = RING_BYTES / (W_BYTES + tm * (BK / 2));
    p.stages = stages < MAX_STAGES ? stages : MAX_STAGES;
    const int64_t units = (int64_t)p.n_tiles * p.m_tiles;
    if (units * 2 > 2147483647LL) return set_error(B200Q_UNSUPPORTED, "qlinear_i8_i8: problem too large for the tile counter");
    int sms = sm_count();
    if (sms <= 0) sms = 148;
    if (split > p.k_blocks) split = 1;  // each has a part
    p.split = split;
    const int64_t pairs_at_once = sms / 2;
    const unsigned grid = split > 1 ? 2u * (unsigned)(units * split) : 2u * (unsigned)(units < pairs_at_once ? units : pairs_at_once);
    const int form = (a.nk ? 4 : 0) + (a.out_type == B200Q_BF16 ? 2 : 0) + (a.pairs ? 1 : 0);
    switch (form) {
        case 0: return launch_as<false, false, false>(map_w, map_a, p, grid, stream);
        case 1: return launch_as<false, false, true>(map_w, map_a, p, grid, stream);
        case 2: return launch_as<false, true, false>(map_w, map_a, p, grid, stream);
        case 3: return launch_as<false, true, true>(map_w, map_a, p, grid, stream);
        case 4: return launch_as<true, false, false>(map_w, map_a, p, grid, stream);
        case 5: return launch_as<true, false, true>(map_w, map_a, p, grid, stream);
        case 6: return launch_as<true, true, false>(map_w, map_a, p, grid, stream);
        default: return launch_as<true, true, true>(map_w, map_a, p, grid, stream);
    }
}

}  // namespace b200q
