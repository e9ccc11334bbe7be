// The int8 x int8 product where a tile's K is shared by a cluster: few tokens, where the stream of the weight is all the time, and few tiles.
//
// Computed transposed as on pairs of SMs (qlinear_i8_pair.cu): 128 channels are the lanes of a CTA's accumulator, tm tokens (a multiple of 16, at most 256) its columns, which is what
// makes tcgen05 the right instruction even for one token: nothing but copies goes into the operands, so a CTA's only work is to keep bytes on their way.  The CTAs
// of a cluster have a part of K each.  Their sums are whole numbers, so that nothing depends on the order in which they meet: every CTA gets the sums
// of its share of the tokens from all of them, through distributed shared memory in the place where the operands' ring was, adds them and finishes them.
//
// Two CTAs an SM where their ring lets them (up to 96 KB), so that one's start and end pass while the other's bytes come in.
//   warp 0  TMA producer.  The first weight tiles are asked for before the kernel in front has finished, but into L2 only: it may be the one that writes them (quantize_tokens lets this
//           kernel start long before its codes are there).  Behind it they come from there.  Quantization and product of one token, 4096 x 4096:
//           7.0 us; 6.7 with the tiles read at once, which took such a weight's codes before they were written, 8.6 where quantize_tokens let nothing start before its end.
//   warp 1  MMA issuer
//   all     sums to their shares, shares to results
// Waits are bounded as on pairs of SMs; a CTA that gives up still meets its cluster's barriers.
#include <atomic>

#include "qlinear_i8.h"
#include "serving.cuh"
#include "umma.cuh"

namespace b200q {
namespace i8split {

constexpr unsigned int kKernelI8Split = 10;
constexpr int TN = 128, BK = 128;
constexpr int W_BYTES = TN * BK;
constexpr int MAX_STAGES = 12;
constexpr int THREADS = 256;
constexpr int LOAD_WARP = 0, MMA_WARP = 1;

struct Params {
    I8Args a;
    int tm, n_tiles;
    int k_blocks;
    int stages;
    int cluster, share;  // CTAs of a tile, tokens of a CTA's share
    uint32_t tmem_cols;
    uint32_t sums_at;    // where the sums lie in shared memory
};

__device__ __forceinline__ uint32_t idesc_i8(int m, int n, bool a_mn_major) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn_major << 15) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | (64ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void ld_32x32b_x16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                   "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr)
                 : "memory");
}

template <bool NK, bool BF16, bool PAIRS>
__global__ void __launch_bounds__(THREADS) i8_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const Params p) {
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) uint64_t full[MAX_STAGES], empty[MAX_STAGES], done;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;

    const uint32_t smem_base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char *smem_gen = smem_dyn + (smem_base - smem_u32(smem_dyn));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int tile = blockIdx.x / p.cluster;
    const int n0 = tile % p.n_tiles * TN, m0 = tile / p.n_tiles * p.tm;
    const int kb0 = (int)((int64_t)p.k_blocks * (int)rank / p.cluster), kb1 = (int)((int64_t)p.k_blocks * ((int)rank + 1) / p.cluster), blocks = kb1 - kb0;
    const uint32_t stages = p.stages, a_bytes = (uint32_t)p.tm * BK, stage_bytes = W_BYTES + a_bytes;

    if (threadIdx.x == 0) {
        for (int s = 0; s < MAX_STAGES; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        mbar_init(smem_u32(&done), 1);
        abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == MMA_WARP) {
        umma::alloc(smem_u32(&tmem_base_slot), p.tmem_cols);
        umma::relinquish();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    pdl_launch_dependents();
    if (p.cluster > 1 && p.sums_at != 0) cluster_arrive_release();  // this CTA is there, for the others' stores

    auto wait_one = [&](uint32_t bar, uint32_t parity, unsigned int site) -> bool {
        return mbar_wait(bar, parity, umma::kFastPolls) || umma::wait_or_abort<kKernelI8Split>(bar, parity, site, &abort_flag, p.a.status);
    };

    if (warp == LOAD_WARP && lane == 0) {
        const uint64_t once = l2_policy_evict_first(), keep = l2_policy_evict_last();
        const bool one_pass = (int)(gridDim.x / p.cluster) == p.n_tiles;  // no other tile reads the weight again
        auto load_w = [&](int i) {
            const uint32_t s = (uint32_t)i % stages, bar = smem_u32(&full[s]);
            const int k = (kb0 + i) * BK;
            mbar_expect_tx(bar, stage_bytes);
            tma_load_2d_hint(smem_base + s * stage_bytes, &map_w, NK ? k : n0, NK ? n0 : k, bar, one_pass ? once : keep);
        };
        auto load_a = [&](int i) {
            const uint32_t s = (uint32_t)i % stages;
            tma_load_2d_hint(smem_base + s * stage_bytes + W_BYTES, &map_a, (kb0 + i) * BK, m0, smem_u32(&full[s]), keep);
        };
        const int ahead = min(blocks, (int)stages);
        for (int i = 0; i < ahead; ++i) tma_prefetch_2d(&map_w, NK ? (kb0 + i) * BK : n0, NK ? n0 : (kb0 + i) * BK);
        pdl_wait();
        for (int i = 0; i < ahead; ++i) load_w(i), load_a(i);
        int i = ahead;
        for (; i < blocks; ++i) {
            if (!wait_one(smem_u32(&empty[(uint32_t)i % stages]), ((uint32_t)i / stages - 1) & 1, 1)) break;
            load_w(i);
            load_a(i);
        }
        // every copy armed has landed before the ring is given to the sums, or the CTA retires
        for (int j = max(0, i - (int)stages); j < i; ++j)
            if (!mbar_wait(smem_u32(&full[(uint32_t)j % stages]), ((uint32_t)j / stages) & 1)) report_timeout(p.a.status, kKernelI8Split, 7);
    } else if (warp == MMA_WARP && elect_one()) {
        pdl_wait();  // the bounded waits do not run against the kernel in front
        const uint32_t idesc = idesc_i8(TN, p.tm, !NK);
        constexpr uint32_t W_STEP = NK ? 32 / 16 : 32 * TN / 16;
        for (int i = 0; i < blocks; ++i) {
            const uint32_t s = (uint32_t)i % stages;
            if (!wait_one(smem_u32(&full[s]), ((uint32_t)i / stages) & 1, 4)) break;
            umma::fence_after_sync();
            const uint32_t at = smem_base + s * stage_bytes;
            const uint64_t w_desc = NK ? umma::smem_desc_sw128(at) : smem_desc_mn(at), a_desc = umma::smem_desc_sw128(at + W_BYTES);
#pragma unroll
            for (int ks = 0; ks < BK / 32; ++ks) mma_i8(tmem_base, w_desc + W_STEP * ks, a_desc + 2 * ks, idesc, (i > 0 || ks > 0) ? 1u : 0u);
            umma::commit(smem_u32(&empty[s]));
        }
        umma::commit(smem_u32(&done));
    }
    __syncwarp();
    pdl_wait();
    bool ok = wait_one(smem_u32(&done), 0, 5);
    ok = __syncthreads_and(ok) && abort_flag == 0;
    umma::fence_after_sync();
    if (p.cluster > 1 && p.sums_at == 0) {
        cluster_arrive_release();
        cluster_wait_acquire();  // nobody's ring is in use any more
    }
    if (p.cluster > 1 && p.sums_at != 0) cluster_wait_acquire();
    // ---- sums: [rank that made them][token of the share][128 channels] in the ring of the CTA that has the share ----
    if (ok && warp < 4) {
        const uint32_t lane_addr = tmem_base + ((uint32_t)(32 * warp) << 16);
        const uint32_t mine = smem_base + p.sums_at + (rank * p.share * TN + 32 * warp + lane) * 4;
        uint32_t target = 0, place = 0, base = map_to_rank(mine, 0);
        for (int c = 0; c < p.tm; c += 16) {
            uint32_t v[16];
            ld_32x32b_x16(lane_addr + c, v);
            umma::ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(base + place * TN * 4), "r"(v[i]) : "memory");
                if (++place == (uint32_t)p.share) {
                    place = 0;
                    if (++target < (uint32_t)p.cluster) base = map_to_rank(mine, target);
                }
            }
        }
    }
    umma::fence_before_sync();
    if (p.cluster > 1) {
        cluster_arrive_release();
        cluster_wait_acquire();
    } else {
        __syncthreads();
    }
    if (warp == MMA_WARP) {
        umma::fence_after_sync();
        umma::dealloc(tmem_base, p.tmem_cols);
    }
    if (!ok) return;
    // ---- two channels a thread ----
    const int t0 = (int)rank * p.share, tokens = min(min(p.share, p.tm - t0), p.a.M - m0 - t0);
    const int ch = (threadIdx.x & 63) * 2, n = n0 + ch;
    const bool in0 = n < p.a.N, in1 = n + 1 < p.a.N;
    if (!in0) return;
    const float s0 = i8_scale(p.a.scale, p.a.scale_type, n), s1 = in1 ? i8_scale(p.a.scale, p.a.scale_type, n + 1) : 0.0f;
    const float b0 = p.a.bias != nullptr ? i8_value(p.a.bias, p.a.out_type, n) : 0.0f, b1 = p.a.bias != nullptr && in1 ? i8_value(p.a.bias, p.a.out_type, n + 1) : 0.0f;
    const int out_n = PAIRS ? p.a.N / 2 : p.a.N, out_at = PAIRS ? n / 2 : n;
    for (int t = threadIdx.x >> 6; t < tokens; t += THREADS / 64) {
        const int64_t m = m0 + t0 + t;
        int x = 0, y = 0;
        for (int r = 0; r < p.cluster; ++r) {
            const int2 v = *reinterpret_cast<const int2 *>(smem_gen + p.sums_at + (((r * p.share + t) * TN + ch) << 2));
            x += v.x, y += v.y;
        }
        const float a_scale = p.a.a_scale[m];
        float y0 = fmaf((float)x * s0, a_scale, b0), y1 = fmaf((float)y * s1, a_scale, b1);
        if (PAIRS) {
            y0 = silu(y0) * y1;
            if (p.a.residual != nullptr) y0 += i8_value(p.a.residual, p.a.out_type, m * p.a.ldr + out_at);
            i8_store(p.a.c, p.a.out_type, m * out_n + out_at, y0);
        } else {
            if (p.a.residual != nullptr) {
                y0 += i8_value(p.a.residual, p.a.out_type, m * p.a.ldr + out_at);
                if (in1) y1 += i8_value(p.a.residual, p.a.out_type, m * p.a.ldr + out_at + 1);
            }
            const int64_t at = m * out_n + out_at;  // widths are even: two channels are in or out together
            if (BF16) {
                *reinterpret_cast<__nv_bfloat162 *>(static_cast<__nv_bfloat16 *>(p.a.c) + at) = __floats2bfloat162_rn(y0, y1);
            } else {
                *reinterpret_cast<__half2 *>(static_cast<__half *>(p.a.c) + at) = __floats2half2_rn(y0, y1);
            }
        }
    }
}

template <bool NK, bool BF16, bool PAIRS>
int launch_as(const CUtensorMap &map_w, const CUtensorMap &map_a, const Params &p, unsigned grid, int smem, cudaStream_t stream) {
    static std::atomic<bool> attr_set[64];
    const int rc = allow_smem(attr_set, i8_split_kernel<NK, BF16, PAIRS>, 224 * 1024);
    if (rc != B200Q_OK) return rc;
    return launch_after("i8_split_kernel", i8_split_kernel<NK, BF16, PAIRS>, dim3(grid), THREADS, (size_t)smem, p.cluster, stream, map_w, map_a, p);
}

}  // namespace i8split

int launch_i8_split(const I8Args &a, int tm, int cluster, cudaStream_t stream) {
    using namespace i8split;
    CUtensorMap map_w, map_a;
    int rc = a.nk ? make_tensor_map_2d(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, (uint64_t)a.K, (uint64_t)a.N, (uint64_t)a.K, BK, TN, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B)
                  : make_tensor_map_2d(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, (uint64_t)a.N, (uint64_t)a.K, (uint64_t)a.N, TN, BK, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != B200Q_OK) return rc;
    rc = make_tensor_map_2d(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.a, (uint64_t)a.K, (uint64_t)a.M, (uint64_t)a.K, BK, (uint32_t)tm, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (rc != B200Q_OK) return rc;
    Params p = {};
    p.a = a;
    p.tm = tm;
    p.n_tiles = (int)ceil_div(a.N, TN);
    p.k_blocks = (int)ceil_div(a.K, BK);
    if (cluster > p.k_blocks) cluster = p.k_blocks;  // each has a part
    p.cluster = cluster;
    p.share = (int)ceil_div(tm, cluster);
    p.tmem_cols = 32;
    while ((int)p.tmem_cols < tm) p.tmem_cols *= 2;
    const int stage = W_BYTES + tm * BK, sums = cluster * p.share * TN * 4;
    // As many stages as a CTA has work for, in what leaves room for a second CTA, or with larger ones (more than 64 tokens) for one.
    int stages = (tm <= 64 ? 96 * 1024 : 192 * 1024) / stage;
    const int work = (int)ceil_div(p.k_blocks, cluster);
    if (stages > work) stages = work;
    if (stages > MAX_STAGES) stages = MAX_STAGES;
    p.stages = stages;
    // Sums of few tokens have a place of their own, which saves the cluster a meeting in front of them.
    p.sums_at = cluster > 1 && tm <= 32 ? (uint32_t)(stages * stage) : 0u;
    const int ring = p.sums_at != 0 ? stages * stage + sums : stages * stage > sums ? stages * stage : sums;
    const int64_t grid = (int64_t)p.n_tiles * ceil_div(a.M, tm) * cluster;
    if (grid > 2147483647LL) return set_error(B200Q_UNSUPPORTED, "qlinear_i8_i8: problem too large for the tile counter");
    const int smem = ring + 1024, form = (a.nk ? 4 : 0) + (a.out_type == B200Q_BF16 ? 2 : 0) + (a.pairs ? 1 : 0);
    const unsigned g = (unsigned)grid;
    switch (form) {
        case 0: return launch_as<false, false, false>(map_w, map_a, p, g, smem, stream);
        case 1: return launch_as<false, false, true>(map_w, map_a, p, g, smem, stream);
        case 2: return launch_as<false, true, false>(map_w, map_a, p, g, smem, stream);
        case 3: return launch_as<false, true, true>(map_w, map_a, p, g, smem, stream);
        case 4: return launch_as<true, false, false>(map_w, map_a, p, g, smem, stream);
        case 5: return launch_as<true, false, true>(map_w, map_a, p, g, smem, stream);
        case 6: return launch_as<true, true, false>(map_w, map_a, p, g, smem, stream);
        default: return launch_as<true, true, true>(map_w, map_a, p, g, smem, stream);
    }
}

}  // namespace b200q
