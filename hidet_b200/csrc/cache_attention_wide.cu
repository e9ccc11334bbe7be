// Attention over the quantized cache where many query rows share a key/value head (trees of drafted tokens, grouped heads, short prompts): the products
// on tcgen05, 128 rows at a time.
//
// As in cache_attention.cu the tiles of all items stand in one line that is cut into equal pieces, one a CTA, one CTA an SM.  Inside a CTA:
//   one warp plans and copies records (codes and scales) into a ring;
//   four warps convert a tile's codes to f16, each one record: K as it lies, [position][element], V through transposing matrix loads as
//       [element][position], both in the 128-byte swizzle, so that both are K-major operands;
//   one thread issues S = Q K^T (128 x 64) and O += P V (128 x D), sums in tensor memory;
//   two groups of four warps turn scores into probabilities, a thread a row, alternate tiles: each group has its own S, P, O, maxima and sums, which
//       meet at the end of the item.
// The probabilities go back into tensor memory, in the place of their scores, as the first operand of the second product.  A thread has a whole row of 64 scores, so maximum and sum
// need no exchange.  A row's unit is 2^u: u is its running maximum (in log2) plus the exponent of the largest value scale that it has seen so far, so that the products with
// value scales fit f16 and sums of probabilities and of values are in the same unit.  (So an exponential's argument has the exponent in it: where value scales are
// near 2^-16, or 2^16, it is off by 2^-20 and the denominator's logarithm by up to 3e-6.  The result is not: its sums have the same errors above and below.)
//
// Bound by the two softmax groups.  A tile takes one 3400 clocks, 600 for the bound on its scores and 2800 for the probabilities (an item's first, whose maximum is
// looked for, 1800 and 2000), so 64 positions of 128 rows pass every 1700, in which the tensor cores work for 256 (15 % of the time by the counters); the groups
// issue in 37 % of the slots and wait for tensor memory, for scales (four bytes a clock, whoever asks for them) and for instructions.  The codes' conversion, 950
// clocks a tile, keeps out of the way.  An item has about 8000 clocks that no tile hides: its queries, its first scores, the last product and the result.
//
// Measured with 128 elements a head, f16 (and in the kernel for few rows), us: 8 sequences of 4096 positions, 64 tokens, 64 heads over 8: 142 (524), 484 TFLOP/s counting
// all positions; 8 of 820 to 4096, 64 tokens, 32 over 8: 59 (190); 16 of 600, 48 tokens, 32 over 8: 41 (91); 50 of 90, 11 tokens, 128 over 32, where it is the
// items' cost above all: 79 (109).
// Slower: one reading of the scores with all 64 in registers (spills, and code beyond the instruction caches), two groups that convert, the
// next item's queries loaded in front of the last product (registers spill: 88 us where it was 82 then).
#include <stddef.h>

#include "cache_attention.cuh"

namespace b200q {
namespace cache_attention {
namespace {

constexpr unsigned int kKernelCacheAttentionWide = 9;

constexpr int ROWS = 128;
constexpr int GROUP_WARPS = 4;                  // of a group that turns scores into probabilities
constexpr int SOFTMAX_THREADS = 2 * 32 * GROUP_WARPS;
constexpr int CONVERT_WARP0 = 8, PRODUCER_WARP = 12, MMA_WARP = 13;
constexpr int THREADS = 32 * 14;
constexpr int kItemUnits = 8;                   // what an item costs besides its tiles, in tiles
constexpr int ITEMS = 2;                        // that the other roles may know of
constexpr int RAW_STAGES = 3, KV_STAGES = 4;
constexpr int AHEAD = 2;                        // tiles whose scores are asked for in front of the probabilities of another
// Items of which the first of several pieces is a CTA's, behind the pieces in the workspace.
__device__ __forceinline__ Item *split_items(const AttentionArgs &p) { return reinterpret_cast<Item *>(p.partial + p.partial_floats); }
static_assert(sizeof(Item) <= 64, "");
constexpr uint32_t TMEM_COLS = 512;
// Columns of a group's scores, two tiles of them (the probabilities take the place of their scores), and of its sums.
__device__ __forceinline__ constexpr uint32_t s_col(int group, int buffer) { return 64 * (2 * group + buffer); }
__device__ __forceinline__ constexpr uint32_t o_col(int group) { return 256 + 128 * group; }
constexpr float kLeastUnit = -90.0f;            // exponents of value scales below are not followed: sums in that unit stay in float's range

template <int D>
struct Layout {
    // Pieces in the workspace: four elements of all rows, the next four, ..., then the rows' units (log2) and sums of probabilities.
    static constexpr int Q = ROWS * D * 2;
    static constexpr int K = TILE * D * 2, V = D * TILE * 2, KV = K + V;
    static constexpr int RAW = RECORDS * record_bytes(D);
    static constexpr int KV_AT = Q, RAW_AT = Q + KV_STAGES * KV;
    static constexpr int SMEM = RAW_AT + RAW_STAGES * RAW + 1024;  // 1024: the operands begin at a multiple of it
};

// The position of a record that stands in place j of it (below eight: the first two of every four, above: the others).
__device__ __forceinline__ constexpr uint32_t position_of(uint32_t j) { return 4 * ((j & 7) >> 1) + (j & 1) + 2 * (j >> 3); }
__device__ __forceinline__ constexpr uint32_t position_of32(uint32_t j) { return (j & 16) + position_of(j & 15); }  // of two records

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Four scales, read where this stands: ahead of their use they would take as many registers as the scores.
__device__ __forceinline__ void scales_at(uint32_t addr, f32x2 &a, f32x2 &b) { asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(addr)); }

// The largest value scale of what a row sees of a tile (the others may be larger by any factor), or another with its exponent: records that it sees entirely by their
// largest, and others only if one in them would change the exponent.  Seldom called, and what it costs is the way of its instructions into the caches: a function of its
// own adds 0 to 3 % to calls with a few tiles a CTA (inline 1 to 6, as loops that stay loops 1 to 6, with a load for each position 44).
__device__ __noinline__ float seen_v_top(const float *scales, const float *tops, uint64_t seen, float v_limit) {
    const float4 of = *reinterpret_cast<const float4 *>(tops);
    auto bits = [&](int w) { return (uint32_t)(seen >> (16 * w)) & 0xffffu; };
    float top = fmaxf(fmaxf(bits(0) == 0xffffu ? of.x : 0.0f, bits(1) == 0xffffu ? of.y : 0.0f), fmaxf(bits(2) == 0xffffu ? of.z : 0.0f, bits(3) == 0xffffu ? of.w : 0.0f));
    const float enough = fmaxf(v_limit, __uint_as_float((__float_as_uint(top) & 0x7f800000u) + 0x00800000u));
    if (seen == 0 || fmaxf(fmaxf(of.x, of.y), fmaxf(of.z, of.w)) < enough) return top;
#pragma unroll 1
    for (int w = 0; w < RECORDS; ++w) {
        const uint32_t own = bits(w);
        if (own == 0 || tops[w] < enough) continue;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(scales + 16 * w + j);
            top = fmaxf(top, fmaxf(fmaxf(own >> position_of(j) & 1u ? v.x : 0.0f, own >> position_of(j + 1) & 1u ? v.y : 0.0f),
                                   fmaxf(own >> position_of(j + 2) & 1u ? v.z : 0.0f, own >> position_of(j + 3) & 1u ? v.w : 0.0f)));
        }
    }
    return top;
}

struct Control {
    uint64_t raw_full[RAW_STAGES], raw_empty[RAW_STAGES], kv_full[KV_STAGES], kv_empty[KV_STAGES], item_full[ITEMS], item_empty[ITEMS];
    uint64_t q_full, s_full[2][2], p_full[2][2], pv_done[2], item_done, drained;  // [group][buffer]
    alignas(16) float k_scale[KV_STAGES][TILE];  // read four at a time
    alignas(16) float v_scale[KV_STAGES][TILE];
    alignas(16) float k_top[KV_STAGES][RECORDS];
    alignas(16) float v_top[KV_STAGES][RECORDS];
    int key0[RAW_STAGES], length[RAW_STAGES];  // length -1: no more tiles
    Item items[ITEMS];
    float top[2][ROWS], unit[2][ROWS], sum[2][ROWS];
    int abort, last;
    uint32_t tmem;
};
static_assert(offsetof(Control, k_scale) % 16 == 0 && offsetof(Control, v_scale) % 16 == 0 && alignof(Control) % 16 == 0, "");

template <int D, typename T>
__global__ void __launch_bounds__(THREADS, 1) cache_attention_wide_kernel(const __grid_constant__ AttentionArgs p) {
    using L = Layout<D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Control ctl;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem - smem_u32(smem_raw));

    if (threadIdx.x == 0) {
        for (int i = 0; i < RAW_STAGES; ++i) mbar_init(smem_u32(&ctl.raw_full[i]), 1), mbar_init(smem_u32(&ctl.raw_empty[i]), RECORDS);
        for (int i = 0; i < KV_STAGES; ++i) mbar_init(smem_u32(&ctl.kv_full[i]), RECORDS), mbar_init(smem_u32(&ctl.kv_empty[i]), 1);
        for (int i = 0; i < ITEMS; ++i) mbar_init(smem_u32(&ctl.item_full[i]), 1), mbar_init(smem_u32(&ctl.item_empty[i]), 2 * GROUP_WARPS + 1);
        for (int i = 0; i < 2; ++i) {
            for (int j = 0; j < 2; ++j) mbar_init(smem_u32(&ctl.s_full[i][j]), 1), mbar_init(smem_u32(&ctl.p_full[i][j]), GROUP_WARPS);
            mbar_init(smem_u32(&ctl.pv_done[i]), 1);
        }
        mbar_init(smem_u32(&ctl.q_full), 2 * GROUP_WARPS);
        mbar_init(smem_u32(&ctl.item_done), 1);
        mbar_init(smem_u32(&ctl.drained), 1);
        ctl.abort = 0;
        mbar_fence_init();
    }
    // Tensor memory is taken when the kernel in front is over (its CTAs that have yet to begin may need it) and before any kernel behind may begin.
    pdl_wait();
    if (warp == MMA_WARP) {
        umma::alloc(smem_u32(&ctl.tmem), TMEM_COLS);
        umma::relinquish();
        umma::fence_before_sync();
    }
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = ctl.tmem;

    auto wait_one = [&](uint64_t &barrier, uint32_t parity, unsigned int site) -> bool {  // one thread's
        const uint32_t bar = smem_u32(&barrier);
        return mbar_wait(bar, parity, umma::kFastPolls) || umma::wait_or_abort<kKernelCacheAttentionWide>(bar, parity, site, &ctl.abort, p.status);
    };
    auto wait = [&](uint64_t &barrier, uint32_t parity, unsigned int site) -> bool { return __all_sync(0xffffffffu, wait_one(barrier, parity, site)); };

    if (warp == PRODUCER_WARP) {
        // ---------------- plan and copies ----------------
        pdl_launch_dependents();
        Line<ROWS, 4, kItemUnits> line(p, lane);
        Item item;
        const int32_t *table;
        int n_items = 0, it = 0, slot = 0;
        uint32_t parity = 0;
        bool ok = true;
        auto publish = [&]() {
            const int at = n_items % ITEMS;
            if (n_items >= ITEMS) ok = wait(ctl.item_empty[at], (n_items / ITEMS - 1) & 1, 1);
            if (ok && lane == 0) {
                ctl.items[at] = item;
                mbar_arrive(smem_u32(&ctl.item_full[at]));
            }
            ++n_items;
        };
        Item *split = split_items(p) + blockIdx.x;  // the item whose first piece of several is here, for the kernel behind
        if (lane == 0) split->rows = -1;
        while (ok && line.next(item, table)) {
            if (lane == 0 && item.first_cta == (int)blockIdx.x && item.last_cta > (int)blockIdx.x) *split = item;
            Pages pages(p, item, lane, table);
            publish();
            for (int i = 0; ok && i < item.tiles; ++i) {
                const int key0 = (item.tile0 + i) * TILE;
                if (it >= RAW_STAGES) ok = wait(ctl.raw_empty[slot], parity ^ 1u, 2);
                if (!ok) break;
                const uint32_t bar = smem_u32(&ctl.raw_full[slot]);
                if (lane == 0) {
                    const int keys = copied_keys(item, key0);
                    ctl.key0[slot] = key0;
                    ctl.length[slot] = item.length;
                    if (keys > 0) mbar_expect_tx(bar, (uint32_t)(keys >> 4) * record_bytes(D));
                    else mbar_arrive(bar);
                }
                __syncwarp();
                copy_tile<D>(p, item, pages, lane, key0, smem + L::RAW_AT + slot * L::RAW, bar);
                ++it;
                if (++slot == RAW_STAGES) slot = 0, parity ^= 1u;
            }
        }
        item.rows = -1;
        if (ok) publish();
        if (ok && it >= RAW_STAGES) ok = wait(ctl.raw_empty[slot], parity ^ 1u, 3);
        if (ok && lane == 0) {
            ctl.length[slot] = -1;
            mbar_arrive(smem_u32(&ctl.raw_full[slot]));
        }
        __syncwarp();
        write_unowned<D>(p, line.placed, lane);
        // Nothing may be on its way when the CTA ends, whoever's wait has run out.  (Where the end was told, a stage was empty for that.)
        for (int back = 1; back <= RAW_STAGES - (ok ? 1 : 0) && back <= it; ++back) {
            const int at = it - back;
            mbar_wait(smem_u32(&ctl.raw_full[at % RAW_STAGES]), (at / RAW_STAGES) & 1, 1u << 16);
        }
    } else if (warp == MMA_WARP) {
        // ---------------- products ----------------
        if (elect_one()) {
            const uint32_t qk_desc = umma::instr_desc_f16(ROWS, TILE), pv_desc = umma::instr_desc_f16(ROWS, D);
            // Products are carried out in the order they are issued, so the second product of a tile frees the place of its scores for a later
            // tile's without a wait.
            uint32_t n[2] = {0, 0};  // tiles of the groups, of the items in front
            int kv = 0;              // of both
            bool ok = true;
            for (int n_items = 0; ok; ++n_items) {
                ok = wait_one(ctl.item_full[n_items % ITEMS], (n_items / ITEMS) & 1, 4);
                if (!ok) break;
                const int rows = ctl.items[n_items % ITEMS].rows, tiles = ctl.items[n_items % ITEMS].tiles;
                mbar_arrive(smem_u32(&ctl.item_empty[n_items % ITEMS]));
                if (rows < 0) break;
                ok = wait_one(ctl.q_full, n_items & 1, 5);
                for (int i = 0, asked = 0; ok && i < tiles; ++i) {
                    for (; ok && asked < min(tiles, i + AHEAD + 1); ++asked) {
                        const int g = asked & 1, buf = (kv + asked) % KV_STAGES;
                        const uint32_t at = n[g] + (asked >> 1);
                        ok = wait_one(ctl.kv_full[buf], ((kv + asked) / KV_STAGES) & 1, 6);
                        if (!ok) break;
                        umma::fence_after_sync();
                        const uint64_t a = umma::smem_desc_sw128(smem), b = umma::smem_desc_sw128(smem + L::KV_AT + buf * L::KV);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const int half = k / 4, to = 2 * (k % 4);  // 16-byte units
                            umma::mma_ss(tmem + s_col(g, at & 1), a + half * (ROWS * 128 / 16) + to, b + half * (TILE * 128 / 16) + to, qk_desc, k > 0);
                        }
                        umma::commit(smem_u32(&ctl.s_full[g][at & 1]));
                    }
                    if (!ok) break;
                    const int g = i & 1, buf = (kv + i) % KV_STAGES;
                    const uint32_t at = n[g] + (i >> 1);
                    ok = wait_one(ctl.p_full[g][at & 1], (at >> 1) & 1, 8);
                    if (!ok) break;
                    umma::fence_after_sync();
                    const uint64_t b = umma::smem_desc_sw128(smem + L::KV_AT + buf * L::KV + L::K);
#pragma unroll
                    for (int k = 0; k < TILE / 16; ++k) umma::mma_ts(tmem + o_col(g), tmem + s_col(g, at & 1) + 8 * k, b + 2 * k, pv_desc, i > 1 || k > 0);
                    umma::commit(smem_u32(&ctl.pv_done[g]));
                    umma::commit(smem_u32(&ctl.kv_empty[buf]));
                }
                if (!ok) break;
                umma::commit(smem_u32(&ctl.item_done));
                kv += tiles;
                n[0] += (tiles + 1) >> 1;
                n[1] += tiles >> 1;
            }
            umma::commit(smem_u32(&ctl.drained));  // tensor memory is given back when nothing is on its way
            if (!mbar_wait(smem_u32(&ctl.drained), 0)) report_timeout(p.status, kKernelCacheAttentionWide, 9);
        }
        __syncwarp();
    } else if (warp >= CONVERT_WARP0) {
        // ---------------- codes to f16 ----------------
        const int w = warp - CONVERT_WARP0;
        // Matrix stores take the halves of what a transposing load of V leaves in a register (positions 4t .. 4t + 3) apart, so place j of a
        // record holds position position_of(j), in K, V and the scales alike.  The same order gives eight lanes' rows of K different banks.
        const uint32_t place = lane & 15, row = position_of(place), sw = k_order(row, D), v_sw = v_order(place, D);
        const uint32_t k_at = (2 * w + (place >> 3)) * 1024 + (place & 7) * 128;                    // of this lane's row of K
        const uint32_t v_at = (lane >> 4) * 1024 + (lane & 7) * 128 + (((2 * w + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);  // of its row of a matrix store
        for (int it = 0;; ++it) {
            const int slot = it % RAW_STAGES, buf = it % KV_STAGES;
            if (!wait(ctl.raw_full[slot], (it / RAW_STAGES) & 1, 10)) break;
            const int key0 = ctl.key0[slot] + 16 * w, length = ctl.length[slot];
            if (length < 0) break;
            const uint32_t rec = smem + L::RAW_AT + slot * L::RAW + w * record_bytes(D);
            uint32_t x[4], v[4];
            auto load = [&](int i) {  // a chunk of 16 codes of a row of K, and two 16 x 16 blocks of V
                const uint32_t c = 2 * i + (lane >> 4);
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(rec + row * D + ((c ^ sw) << 4)));
                umma::ldmatrix_x2_trans_b8(v, rec + 16 * D + place * D + ((c ^ v_sw) << 4));
            };
            load(0);
            const float *scales = reinterpret_cast<const float *>(smem_gen + L::RAW_AT + slot * L::RAW + w * record_bytes(D) + 32 * D);
            const bool there = key0 + (int)row < length;  // behind the end, and in records that were not copied, is anything
            const float ks = there ? scales[row] : 0.0f, vs = there ? scales[16 + row] : 0.0f;
            // the largest of each (they are not negative)
            const uint32_t k_top = __reduce_max_sync(0xffffffffu, ks == ks ? __float_as_uint(ks) : 0u), v_top = __reduce_max_sync(0xffffffffu, vs == vs ? __float_as_uint(vs) : 0u);
            if (it >= KV_STAGES && !wait(ctl.kv_empty[buf], (it / KV_STAGES - 1) & 1, 11)) break;
            const uint32_t k_dst = smem + L::KV_AT + buf * L::KV + k_at, v_dst = smem + L::KV_AT + buf * L::KV + L::K + v_at;
            if (lane < 16) ctl.k_scale[buf][16 * w + lane] = ks, ctl.v_scale[buf][16 * w + lane] = vs;
            if (lane == 0) ctl.k_top[buf][w] = __uint_as_float(k_top), ctl.v_top[buf][w] = __uint_as_float(v_top);
            // A loop that stays a loop: the roles' code together has to stay in the instruction caches nearest to the schedulers.  Where all was unrolled,
            // warps waited for instructions more than for anything else (2.8 of 13 clocks an instruction).
#pragma unroll 1
            for (int i = 0; i < D / 32; ++i) {
                const uint32_t c = 2 * i + (lane >> 4), at = (c & 3) * 2;  // the chunk's 16-byte places in a row of 128
                uint32_t y[8], z[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) codes_to_f16(x[e], y[2 * e], y[2 * e + 1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) codes_to_f16(v[e], z[2 * e], z[2 * e + 1]);
                if (i + 1 < D / 32) load(i + 1);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(k_dst + (c >> 2) * (TILE * 128) + (((at + e) ^ (place & 7)) << 4)), "r"(y[4 * e]), "r"(y[4 * e + 1]),
                                 "r"(y[4 * e + 2]), "r"(y[4 * e + 3])
                                 : "memory");
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // elements 32 i + 16 h .. + 15 of V: two blocks of eight, two halves of the record's positions each
                    const uint32_t block[4] = {z[4 * h], z[4 * h + 1], z[4 * h + 2], z[4 * h + 3]};
                    umma::stmatrix_x4(v_dst + (4 * i + 2 * h) * 1024, block);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&ctl.kv_full[buf]));
                mbar_arrive(smem_u32(&ctl.raw_empty[slot]));
            }
        }
    } else {
        // ---------------- scores to probabilities ----------------
        const int grp = warp / GROUP_WARPS, quarter = warp % GROUP_WARPS, r = 32 * quarter + lane;  // this thread's row
        const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
        const uint32_t o_addr = tmem + lanes + o_col(grp);
        uint32_t n = 0;  // tiles of this group
        int kv = 0;      // of both
        bool alive = true, met = false;  // as in the other kernel
        for (int n_items = 0;; ++n_items) {
            alive = wait(ctl.item_full[n_items % ITEMS], (n_items / ITEMS) & 1, 12);
            if (!alive) break;
            const Item item = ctl.items[n_items % ITEMS];
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[n_items % ITEMS]));
            if (item.rows < 0) break;
            const int token = token_of(p, item.row0 + r), hidden = first_hidden(p, item);
            const bool busy = 32 * quarter < item.rows;  // this warp has rows

            // ---- the queries: group 0 brings the first half of a row, group 1 the second ----
            float qs = p.scale_log2;
            {
                // Of the warp's 32 rows, D / 2 elements each: LANES lanes take a row, 16 bytes each, so that what a load brings lies together.
                constexpr int LANES = D / 16, STEP = 32 / LANES;
                uint4 x[LANES];
#pragma unroll
                for (int i = 0; i < LANES; ++i) {
                    const int own = 32 * quarter + STEP * i + lane / LANES, row = item.row0 + own, tok = token_of(p, row);
                    const T *src = static_cast<const T *>(p.q) + (int64_t)(item.token0 + tok) * p.q_token + (int64_t)(item.head * p.group + row - tok * p.group) * p.q_head;
                    x[i] = own < item.rows ? *reinterpret_cast<const uint4 *>(src + grp * (D / 2) + 8 * (lane % LANES)) : make_uint4(0, 0, 0, 0);
                }
                constexpr bool kScaled = std::is_same<T, __nv_bfloat16>::value;
                if (kScaled) {
#pragma unroll
                    for (int i = 0; i < LANES; ++i) {
                        const T *v = reinterpret_cast<const T *>(&x[i]);
                        float top = 0.0f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(Elems<T>::one(v[e])));
#pragma unroll
                        for (int d = 1; d < LANES; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        if (lane % LANES == 0) ctl.top[grp][32 * quarter + STEP * i + lane / LANES] = top;
                    }
                }
                if (!all_of<SOFTMAX_THREADS>(true)) {  // behind it no thread reads or writes anything of the item in front
                    met = true;
                    break;
                }
                auto exponent_of = [&](int row) { return min(max(__float_as_uint(fmaxf(ctl.top[0][row], ctl.top[1][row])) >> 23, 1u), 253u); };
                if (kScaled) qs = fmaxf(qs * __uint_as_float(exponent_of(r) << 23), kLeastNormal);  // not zero, which makes NaN of a hidden position's -inf
#pragma unroll
                for (int i = 0; i < LANES; ++i) {
                    const int own = 32 * quarter + STEP * i + lane / LANES;
                    if (kScaled) {
                        const float down = __uint_as_float((254u - exponent_of(own)) << 23);
                        const T *v = reinterpret_cast<const T *>(&x[i]);
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = pack_f16(Elems<T>::one(v[2 * e]) * down, Elems<T>::one(v[2 * e + 1]) * down);
                        x[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    const int c = grp * LANES + lane % LANES;  // 16-byte chunk of the row
                    *reinterpret_cast<uint4 *>(smem_gen + (c >> 3) * (ROWS * 128) + (own >> 3) * 1024 + (own & 7) * 128 + (((c & 7) ^ (own & 7)) << 4)) = x[i];
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl.q_full));
            }
            const float rise = fminf(kRise / qs, 1e38f);
            float m = -INFINITY, shift = 0.0f, sum = 0.0f;  // shift: m, or 0 as long as nothing was seen
            // Of the value scales that the row has seen, and the first scale that is too large for it (none as long as it has seen nothing: its first score raises the maximum).
            float exponent = 0.0f, v_limit = INFINITY;

            for (int i = grp; i < item.tiles; i += 2) {
                const int buf = (kv + i) % KV_STAGES, key0 = (item.tile0 + i) * TILE;
                const uint32_t s_addr = tmem + lanes + s_col(grp, n & 1);
                alive = wait(ctl.s_full[grp][n & 1], (n >> 1) & 1, 13) && wait(ctl.kv_full[buf], ((kv + i) / KV_STAGES) & 1, 14);  // the latter for the scales
                if (!alive) break;
                umma::fence_after_sync();
                if (busy) {
                    // Two passes over the scores, 32 at a time, rather than one with all in registers.
                    const bool partly = key0 + TILE > hidden;
                    const uint32_t ks = smem_u32(ctl.k_scale[buf]), vs = smem_u32(ctl.v_scale[buf]);
                    uint64_t seen = ~0ull;
                    if (partly) seen = seen_of_64(p, item, r, token, key0);
                    auto scores = [&](int h, f32x2 (&s)[16]) {
                        uint32_t raw[32];
                        umma::ld_32x32b_x32(s_addr + 32 * h, raw);
                        umma::ld_wait();
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            f32x2 k0, k1;
                            scales_at(ks + 128 * h + 16 * j, k0, k1);
                            s[2 * j] = mul2(pair_of(raw[4 * j], raw[4 * j + 1]), k0);
                            s[2 * j + 1] = mul2(pair_of(raw[4 * j + 2], raw[4 * j + 3]), k1);
                        }
                        if (partly) {
                            const uint32_t bits = (uint32_t)(seen >> (32 * h));
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                float lo, hi;
                                halves(s[j], lo, hi);
                                s[j] = pair_of(bits >> position_of32(2 * j) & 1u ? lo : -INFINITY, bits >> position_of32(2 * j + 1) & 1u ? hi : -INFINITY);
                            }
                        }
                    };
                    // Whether a score can pass the maximum so far by too much: first by the largest product and the largest scale.  (Scales are read from
                    // shared memory by all lanes at once, four bytes a clock; most tiles need those of K once so.)
                    float top = 0.0f, other = 0.0f;
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        uint32_t raw[32];
                        umma::ld_32x32b_x32(s_addr + 32 * h, raw);
                        umma::ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            top = max3(top, __uint_as_float(raw[j]), __uint_as_float(raw[j + 1]));
                            other = max3(other, __uint_as_float(raw[j + 2]), __uint_as_float(raw[j + 3]));
                        }
                    }
                    const float4 k_tops = *reinterpret_cast<const float4 *>(ctl.k_top[buf]), v_tops = *reinterpret_cast<const float4 *>(ctl.v_top[buf]);
                    const float k_top = max3(fmaxf(k_tops.x, k_tops.y), k_tops.z, k_tops.w);
                    float v_top = max3(fmaxf(v_tops.x, v_tops.y), v_tops.z, v_tops.w);
                    bool raised = false;
                    if (__any_sync(0xffffffffu, fmaxf(top, other) * k_top > m + rise)) {
                        top = other = -INFINITY;
#pragma unroll 1
                        for (int h = 0; h < 2; ++h) {
                            f32x2 s[16];
                            scores(h, s);
#pragma unroll
                            for (int j = 0; j < 16; j += 2) {
                                float lo, hi;
                                halves(s[j], lo, hi);
                                top = max3(top, lo, hi);
                                halves(s[j + 1], lo, hi);
                                other = max3(other, lo, hi);
                            }
                        }
                        top = fmaxf(top, other);
                        raised = top > m + rise;
                    }
                    // The bound counts what lies behind the end too, in records that were not copied whatever the ring held.  So a maximum is taken
                    // over only where one of the warp's rows passes its own by too much: results do not depend on what ran before.
                    if (!__any_sync(0xffffffffu, raised)) top = m;
                    if (__any_sync(0xffffffffu, raised || v_top >= v_limit)) {
                        const float was = exponent;
                        if (v_limit == INFINITY && seen != 0) v_limit = kLeastNormal;
                        if (partly) v_top = seen_v_top(ctl.v_scale[buf], ctl.v_top[buf], seen, v_limit);
                        if (v_top >= v_limit) {
                            exponent = fmaxf((float)((int)(__float_as_uint(v_top) >> 23) - 127), kLeastUnit);
                            v_limit = __uint_as_float((uint32_t)((int)exponent + 128) << 23);
                        }
                        __syncwarp();
                        const float higher = fmaxf(m, top);
                        // in two steps: with value scales of very unlike sizes the whole may leave float's range where its product with the sum does not
                        const float by = higher == -INFINITY ? 1.0f : ex2(0.5f * ((m - higher) * qs + (was - exponent)));
                        m = higher;
                        shift = higher == -INFINITY ? 0.0f : higher;
                        sum = sum * by * by;
                        if (i > grp) {
                            // O is this thread's when the group's product in front is over.  (The one in front of that is: this tile's scores were issued behind it.)
                            alive = wait(ctl.pv_done[grp], (n - 1) & 1, 15);
                            if (!alive) break;
                            umma::fence_after_sync();
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                uint32_t o[32];
                                umma::ld_32x32b_x32(o_addr + c, o);
                                umma::ld_wait();
#pragma unroll
                                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * by * by);
                                umma::st_32x32b_x32(o_addr + c, o);
                            }
                        }
                    }
                    const f32x2 minus = pair_of(-shift, -shift), scale2 = pair_of(qs, qs), bias = pair_of(kBias - exponent, kBias - exponent);
                    f32x2 sums[2] = {0, 0};
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        f32x2 s[16];
                        scores(h, s);
                        uint32_t packed[16];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            f32x2 v[2];
                            scales_at(vs + 128 * h + 16 * j, v[0], v[1]);
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float lo, hi;
                                halves(fma2(add2(s[2 * j + e], minus), scale2, bias), lo, hi);
                                const f32x2 x = pair_of(ex2(lo), ex2(hi));
                                sums[e] = add2(sums[e], x);
                                halves(mul2(x, v[e]), lo, hi);
                                packed[2 * j + e] = pack_f16(lo, hi);
                            }
                        }
                        if (partly) {  // nothing, whatever the scale of a position that is not seen
                            const uint32_t bits = (uint32_t)(seen >> (32 * h));
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                if (!(bits >> position_of32(2 * j) & 1u)) packed[j] &= 0xffff0000u;
                                if (!(bits >> position_of32(2 * j + 1) & 1u)) packed[j] &= 0x0000ffffu;
                            }
                        }
                        umma::st_32x32b_x16(s_addr + 16 * h, packed);
                    }
                    float lo, hi;
                    halves(add2(sums[0], sums[1]), lo, hi);
                    sum += lo + hi;
                    umma::st_wait();
                }
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl.p_full[grp][n & 1]));
                ++n;
            }
            if (!alive) break;
            kv += item.tiles;

            // ---- the two groups' sums meet ----
            // (Not by pv_done: two of its phases may be under way, and a wait tells a phase only from its neighbours.)
            alive = wait(ctl.item_done, n_items & 1, 16);
            if (!alive) break;
            ctl.unit[grp][r] = m == -INFINITY ? -INFINITY : m * qs + exponent;
            ctl.sum[grp][r] = sum;
            umma::fence_before_sync();
            if (!all_of<SOFTMAX_THREADS>(true)) {
                met = true;
                break;
            }
            umma::fence_after_sync();
            const bool whole = item.first_cta == item.last_cta;
            if (busy) {
                const float u0 = ctl.unit[0][r], u1 = ctl.unit[1][r], unit = fmaxf(u0, u1);
                const float f0 = u0 == -INFINITY ? 1.0f : ex2(0.5f * (u0 - unit)), f1 = u1 == -INFINITY ? 1.0f : ex2(0.5f * (u1 - unit));
                const float total = ctl.sum[0][r] * f0 * f0 + ctl.sum[1][r] * f1 * f1;
                float *piece = p.partial + (int64_t)item.slot * kPieceFloats<D, ROWS>;
#pragma unroll
                for (int c0 = 0; c0 < D / 2; c0 += 32) {  // group 0 takes the first half of the elements, group 1 the second
                    const int c = grp * (D / 2) + c0;
                    uint32_t a[32], b[32];
                    umma::ld_32x32b_x32(tmem + lanes + o_col(0) + c, a);
                    umma::ld_32x32b_x32(tmem + lanes + o_col(1) + c, b);
                    umma::ld_wait();
                    if (r < item.rows) {
                        float v[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) {  // the second sum begins with the item's second tile
                            v[j] = __uint_as_float(a[j]) * f0 * f0;
                            if (item.tiles > 1) v[j] = fmaf(__uint_as_float(b[j]) * f1, f1, v[j]);
                        }
                        if (whole) {
                            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
                            const int row = item.row0 + r, head = item.head * p.group + row - token * p.group;
                            const int64_t at = (int64_t)(item.token0 + token) * p.kv_heads * p.group + head;
#pragma unroll
                            for (int j = 0; j < 32; j += 8) {
                                const float y[8] = {v[j] * inv, v[j + 1] * inv, v[j + 2] * inv, v[j + 3] * inv, v[j + 4] * inv, v[j + 5] * inv, v[j + 6] * inv, v[j + 7] * inv};
                                store8<T, true>(static_cast<T *>(p.out) + at * D + c + j, narrow<T>(y));
                            }
                            if (c == 0) write_lse(p, at, total, unit);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; j += 4) __stcg(reinterpret_cast<float4 *>(piece) + (c + j) / 4 * ROWS + r, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
                            if (c == 0) __stcg(piece + ROWS * D + r, unit), __stcg(piece + ROWS * (D + 1) + r, total);
                        }
                    }
                }
                umma::fence_before_sync();
            }
        }
        if (!met) all_of<SOFTMAX_THREADS>(alive);
    }
    __syncwarp();
    __syncthreads();
    if (warp == MMA_WARP) {
        umma::fence_after_sync();
        umma::dealloc(tmem, TMEM_COLS);
    }
}

// Adds the pieces of the items that are in several: a CTA takes ADD_ROWS rows of one, a thread four elements of a row at a time.  (In the CTA that is
// last with its piece, as the kernel for few rows does it, 128 rows would take 13 us; here they are spread over the device.)
constexpr int ADD_ROWS = 16, ADD_THREADS = 256;
template <int D, typename T>
__global__ void __launch_bounds__(ADD_THREADS) add_pieces_kernel(const __grid_constant__ AttentionArgs p) {
    pdl_wait();
    pdl_launch_dependents();
    const Item item = split_items(p)[blockIdx.x];
    const int row0 = blockIdx.y * ADD_ROWS;
    if (row0 >= item.rows) return;
    const int parts = item.last_cta - item.first_cta + 1;
    for (int i = threadIdx.x; i < ADD_ROWS * D / 4; i += ADD_THREADS) {
        const int r = row0 + i % ADD_ROWS, d = 4 * (i / ADD_ROWS);
        if (r >= item.rows) continue;
        const float *first = p.partial + (2 * item.first_cta + 1) * kPieceFloats<D, ROWS>, *others = p.partial + 2 * (item.first_cta + 1) * kPieceFloats<D, ROWS>;
        auto piece = [&](int j) { return j == 0 ? first : others + (j - 1) * 2 * kPieceFloats<D, ROWS>; };
        float top = -INFINITY;
#pragma unroll 8
        for (int j = 0; j < parts; ++j) top = fmaxf(top, __ldcg(piece(j) + ROWS * D + r));
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
#pragma unroll 4
        for (int j = 0; j < parts; ++j) {
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(piece(j)) + d / 4 * ROWS + r);
            const float own = __ldcg(piece(j) + ROWS * D + r), s = __ldcg(piece(j) + ROWS * (D + 1) + r);
            // in two steps: units may lie so far apart that the whole factor leaves float's range where the products do not
            const float by = own == -INFINITY ? 1.0f : ex2(0.5f * (own - top));
            sum = fmaf(s * by, by, sum);
            v.x = fmaf(x.x * by, by, v.x), v.y = fmaf(x.y * by, by, v.y), v.z = fmaf(x.z * by, by, v.z), v.w = fmaf(x.w * by, by, v.w);
        }
        write_out<D, T>(p, item, r, d, v, sum, top);
    }
}

template <int D, typename T>
int launch_sized(const AttentionArgs &p, cudaStream_t stream) {
    using L = Layout<D>;
    auto kernel = cache_attention_wide_kernel<D, T>;
    static std::atomic<bool> attr_set[64];
    const int rc = allow_smem(attr_set, kernel, L::SMEM);
    if (rc != B200Q_OK) return rc;
    const int64_t tiles = most_tiles(p, ROWS), at_once = sm_count();
    if (tiles > (1ll << 29)) return set_error(B200Q_UNSUPPORTED, "quantized_cache_attention: up to %lld tiles of %d rows and %d positions", (long long)tiles, ROWS, TILE);
    int64_t grid = tiles < at_once ? tiles : at_once;
    if (grid > kMostWideCtas) grid = kMostWideCtas;
    const int status = launch_after("cache_attention_wide_kernel", kernel, dim3((unsigned)grid), THREADS, L::SMEM, 1, stream, p);
    if (status != B200Q_OK || grid == 1) return status;
    return launch_after("add_pieces_kernel", add_pieces_kernel<D, T>, dim3((unsigned)grid, ROWS / ADD_ROWS), ADD_THREADS, 0, 1, stream, p);
}

}  // namespace

int launch_wide(const AttentionArgs &p, int dim, bool bf16, cudaStream_t stream) {
    if (dim == 64) return bf16 ? launch_sized<64, __nv_bfloat16>(p, stream) : launch_sized<64, __half>(p, stream);
    return bf16 ? launch_sized<128, __nv_bfloat16>(p, stream) : launch_sized<128, __half>(p, stream);
}

}  // namespace cache_attention
}  // namespace b200q
