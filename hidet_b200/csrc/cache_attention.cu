// Attention of new tokens (one a sequence, several, or a tree of drafted ones) over the quantized, paged key/value cache: the entry point, and the kernel
// for few query rows a key/value head, decoding above all.  (cache_attention_wide.cu: for many.)
//
// For query row i (a token and one of the `group` heads that share a key/value head) and position j:
//     s_ij = scale * (q_i . kcode_j) * kscale_j,     o_i = sum_j exp(s_ij - m_i) * vscale_j * vcode_j / sum_j exp(s_ij - m_i)
// over the positions that the row may see, with the running maximum m_i and sum of one pass over the cache.  Codes are exact in f16, so
// the products q . kcode run on f16 tensor-core instructions with float sums; bf16 queries go through f16 too, scaled row by row by a power of
// two (their eight bits fit; what is 2^-24 of the row's largest element is lost).  Probabilities, times vscale_j over the power of two below the largest vscale that the row has seen so far (so
// that they cannot leave f16's range whatever the values' size), are rounded to f16 for the second product, an error of 2^-12 of each, at random; the sums
// that divide are float.
//
// A row's maximum follows its scores only where one passes it by 2^8, an idea published with recent attention kernels: between such steps nothing is rescaled.
//
// The work is in tiles of positions for one (sequence, key/value head, 8 * NT query rows).  The tiles of all sequences stand in
// one line, with a gap in front of every item for what that costs besides where pieces are long, and the line is cut into equal pieces, one a CTA, whatever the sequences' lengths are (the host does not know them: they
// are on the device, so that a captured step can be replayed as they grow).  A CTA's piece may end one item and begin others; items in
// several pieces leave partial sums in the workspace, and the CTA that arrives last adds them in the order of the pieces.
//
// One warp copies whole records (codes and scales, one bulk copy per run of a page) into a ring of shared memory; each of
// the other warps takes one record of 16 positions of a tile: it loads K with plain and V with transposing matrix loads, converts two codes an
// instruction and multiplies, with the codes as the 16-row operand (positions of K, elements of V) and eight query rows as columns.  With the positions
// (and not the rows) shared out among the warps, each code is converted once per CTA.
//
// Bound by the cache's bytes where sequences are long: pieces stream at 5.9 TB/s, and 8 us are the launch, the plan, the first tile and the additions.  Measured with
// 128 elements a head, 64 heads over 8: 32 sequences of 90 to 8000 positions 58 us, one of 131071 57 us, 4.7 TB/s each.  Where they are short it is
// latency: 5.0 us for one tile, 7.0 for two pieces and their sum, 10.4 for 577 positions of 32 heads.  (Code that the instruction caches hold already, by an
// item without rows in front, and all of the queries' loads on their way at once change nothing there.)
#include <atomic>

#include "cache_attention.cuh"

namespace b200q {
namespace cache_attention {
namespace {

constexpr unsigned int kKernelCacheAttention = 7;

struct Tile {
    int key0;  // first position
    int last;  // of the item, in this CTA
};

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ float lds32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
// 8 x 8 elements of 16 bits: from lane (g, t) holding (row g, columns 2t, 2t + 1) to it holding (rows 2t, 2t + 1, column g).
__device__ __forceinline__ uint32_t transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
constexpr int MOST_STAGES = 6;
constexpr int kItemUnits = 2;           // what an item costs besides its tiles, in tiles
constexpr int WARPS = 4;                // that multiply
constexpr int CONSUMERS = 32 * WARPS;
constexpr int THREADS = CONSUMERS + 32;
static_assert(WARPS == RECORDS, "");

template <int D, int NT>
struct Layout {
    static constexpr int ROWS = 8 * NT;
    static constexpr int RECORD = record_bytes(D);
    static constexpr int STAGE = WARPS * RECORD;
    static constexpr int PITCH = D + 4;  // floats between rows of a merge buffer: what a warp stores at once lies in 32 banks
    static constexpr int MERGE = ROWS * PITCH * 4;
    static constexpr int BUFFERS = WARPS / 2;
    static constexpr int PER_SM = NT * D <= 128 ? 3 : NT * D <= 256 ? 2 : 1;
    static constexpr int Q = ROWS * D * 2;
    static constexpr int FIXED = Q + BUFFERS * MERGE;
    static constexpr int ROOM = (PER_SM == 3 ? 75 : PER_SM == 2 ? 113 : 226) * 1024 - 3 * 1024 - FIXED;  // 3 KB: Control, and what an SM keeps for itself
    static constexpr int STAGES = ROOM / STAGE > MOST_STAGES ? MOST_STAGES : ROOM / STAGE;
    static constexpr int SMEM = FIXED + STAGES * STAGE;
    static constexpr bool Q_IN_REGISTERS = NT * D <= 128;
    static_assert(STAGES >= 2, "");
};

constexpr int ITEMS = 2;  // of which the consumers may know
struct Control {
    uint64_t full[MOST_STAGES], empty[MOST_STAGES], item_full[ITEMS], item_empty[ITEMS];
    Tile tiles[MOST_STAGES];
    Item items[ITEMS];
    float m[WARPS][16], l[WARPS][16], q_scale[16];
    int abort, last;
};
static_assert(sizeof(Control) <= 2048, "");

template <typename T>
__device__ __forceinline__ void load_q4(const T *p, float (&f)[4]) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    const T *v = reinterpret_cast<const T *>(&x);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = Elems<T>::one(v[i]);
}

// The reciprocal of a power of two.
__device__ __forceinline__ float power_over(float power) { return __uint_as_float(0x7f000000u - __float_as_uint(power)); }

// A row's maximum as long as it has seen nothing: finite, so that differences from it are numbers.  Hidden positions have -inf.
constexpr float kNothing = -3.4028234663852886e38f;

// The largest of the warps' maxima of a row.
__device__ __forceinline__ float row_top(const Control &ctl, int r) {
    float n = kNothing;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) n = fmaxf(n, ctl.m[w][r]);
    return n;
}

// What becomes of an item whose sums stand in the merge buffers: the result, or a piece of it.  All consumers.
template <int D, int NT, typename T>
__device__ __forceinline__ void finish_item(const AttentionArgs &p, Control &ctl, float *merge, const Item &item) {
    using L = Layout<D, NT>;
    constexpr int ROWS = L::ROWS;
    const bool whole = item.first_cta == item.last_cta;
    float *piece = p.partial + (int64_t)item.slot * kPieceFloats<D, ROWS>;
    for (int i = threadIdx.x; i < item.rows * (D / 4); i += CONSUMERS) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));
        const float top = row_top(ctl, r), scale = ctl.q_scale[r];
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) sum += ctl.l[w][r] * ex2((ctl.m[w][r] - top) * scale);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < L::BUFFERS; ++k) {
            const float4 x = *reinterpret_cast<const float4 *>(merge + k * (L::MERGE / 4) + r * L::PITCH + d);
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        if (whole) write_out<D, T>(p, item, r, d, v, sum, top * scale);
        else write_piece<D, ROWS>(piece, r, d, v, sum, top * scale);
    }
    static_assert(L::BUFFERS * L::MERGE >= 2 * FAN * ROWS * 4, "");
    if (!whole) meet<D, ROWS, CONSUMERS, T>(p, item, threadIdx.x, merge, &ctl.last);  // whose first barrier frees the merge buffers
}

template <int D, int NT, typename T>
__global__ void __launch_bounds__(THREADS, Layout<D, NT>::PER_SM) cache_attention_kernel(const __grid_constant__ AttentionArgs p) {
    using L = Layout<D, NT>;
    constexpr int ROWS = L::ROWS, STAGES = L::STAGES;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Control ctl;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t stages = smem_u32(smem), q_frag = stages + STAGES * L::STAGE;
    float *merge = reinterpret_cast<float *>(smem + STAGES * L::STAGE + L::Q);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&ctl.full[s]), 1);
            mbar_init(smem_u32(&ctl.empty[s]), WARPS);
        }
        for (int s = 0; s < ITEMS; ++s) {
            mbar_init(smem_u32(&ctl.item_full[s]), 1);
            mbar_init(smem_u32(&ctl.item_empty[s]), WARPS);
        }
        ctl.abort = 0;
        mbar_fence_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();

    if (warp == WARPS) {
        // ---------------- producer ----------------
        bool dead = false;
        auto wait_for = [&](uint64_t &barrier, uint32_t parity) {
            const uint32_t bar = smem_u32(&barrier);
            bool ok = false;
            for (uint32_t i = 0; i < umma::kFastPolls && !ok; ++i) ok = mbar_try_wait(bar, parity);
            if (!ok) ok = umma::wait_or_abort<kKernelCacheAttention>(bar, parity, 1, &ctl.abort, p.status);
            dead = !__all_sync(0xffffffffu, ok);
        };
        int n_items = 0;
        auto publish = [&](const Item &item) {
            const int slot = n_items % ITEMS;
            if (n_items >= ITEMS) wait_for(ctl.item_empty[slot], (n_items / ITEMS - 1) & 1);
            if (!dead && lane == 0) {
                ctl.items[slot] = item;
                mbar_arrive(smem_u32(&ctl.item_full[slot]));
            }
            ++n_items;
        };

        Line<ROWS, FAN, kItemUnits> line(p, lane);
        Item item;
        const int32_t *table;
        int slot = 0, it = 0;
        uint32_t parity = 0;
        while (!dead && line.next(item, table)) {
            Pages pages(p, item, lane, table);
            publish(item);
            for (int i = 0; i < item.tiles && !dead; ++i) {
                const int key0 = (item.tile0 + i) * TILE;
                if (it >= STAGES) wait_for(ctl.empty[slot], parity ^ 1u);
                if (dead) break;
                const uint32_t bar = smem_u32(&ctl.full[slot]);
                if (lane == 0) {
                    const int keys = copied_keys(item, key0);
                    ctl.tiles[slot] = {key0, i == item.tiles - 1};
                    if (keys > 0) mbar_expect_tx(bar, (uint32_t)(keys >> 4) * L::RECORD);
                    else mbar_arrive(bar);
                }
                __syncwarp();
                copy_tile<D>(p, item, pages, lane, key0, stages + slot * L::STAGE, bar);
                ++it;
                if (++slot == STAGES) slot = 0, parity ^= 1u;
            }
        }
        item.rows = -1;
        if (!dead) publish(item);
        write_unowned<D>(p, line.placed, lane);
        // Nothing may be on its way when the CTA ends, whoever's wait has run out.
        for (int back = 1; back <= STAGES && back <= it; ++back) {
            const int at = it - back;
            mbar_wait(smem_u32(&ctl.full[at % STAGES]), (at / STAGES) & 1, 1u << 16);
        }
        return;
    }

    // ---------------- consumers ----------------
    const int g = lane >> 2, t = lane & 3;
    // K: lane l addresses row 4 (c / 2) + c % 2 + 2 (l / 8 % 2) of its record, c = l % 8, and of a pair of chunks the (l / 16)-th.  So MMA
    // row g is position 4 (g / 2) + g % 2 and row g + 8 the one two further on: after the transposition of the probabilities
    // lane (g, t) has positions 4t .. 4t + 3 of query row g, the four whose codes a transposing load of V leaves in one register.  Inside a
    // chunk a lane holds elements 4t .. 4t + 3; the query's fragments follow that.
    const uint32_t k_row = 4 * ((lane & 7) >> 1) + (lane & 1) + 2 * ((lane >> 3) & 1);
    const uint32_t k_off = k_row * D, k_sw = k_order(k_row, D), k_chunk = lane >> 4;
    const uint32_t v_row = lane & 15;
    const uint32_t v_off = 16 * D + v_row * D, v_sw = v_order(v_row, D), v_chunk = lane >> 4;
    const int key_of_lane = 4 * (g >> 1) + (g & 1);  // of the scores in [0] and [1]; those in [2] and [3] are two positions further on
    // A warp whose wait runs out brings `false` to the next barrier of all consumers, where all of them leave: one by one, it would
    // leave the others waiting there.  `met`: this warp has been at that barrier.
    bool alive = true, met = false;
    int slot = 0, parity = 0;
    auto wait_for = [&](uint64_t &barrier, uint32_t phase) {
        const uint32_t bar = smem_u32(&barrier);
        bool ok = false;
        for (uint32_t i = 0; i < umma::kFastPolls && !ok; ++i) ok = mbar_try_wait(bar, phase);
        if (!ok) ok = umma::wait_or_abort<kKernelCacheAttention>(bar, phase, 2, &ctl.abort, p.status);
        alive = __all_sync(0xffffffffu, ok);
    };
    for (int n_item = 0;; ++n_item) {
        wait_for(ctl.item_full[n_item % ITEMS], (n_item / ITEMS) & 1);
        if (!alive) break;
        const Item item = ctl.items[n_item % ITEMS];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[n_item % ITEMS]));
        if (item.rows < 0) break;
        const int length = item.length, hidden = first_hidden(p, item);
        float o[NT][D / 16][4];  // elements 16 i + g (0, 1) and + 8 (2, 3) of query rows 2t (0, 2) and 2t + 1 (1, 3)
        float m[NT][2], l[NT][2], qs[NT][2], limit[NT][2];  // limit: a score beyond it is too large for m
        // A row's values are counted in a power of two: its reciprocal, and the first scale that is too large for one of this thread's rows.  Each row has its own,
        // since what one row sees may be larger by any factor than what another does.
        float v_inv[NT][2], v_limit = INFINITY;
        uint2 q_reg[L::Q_IN_REGISTERS ? NT * D / 16 : 1];
        {
            // the queries, as MMA fragments: for chunk c and row g lane (g, t) has elements 16 c + 4t .. + 3
            if (!all_of<CONSUMERS>(true)) {
                met = true;
                break;
            }
#pragma unroll
            for (int r0 = 0; r0 < ROWS; r0 += WARPS) {
                const int r = r0 + warp;
                const int row = item.row0 + r, token = token_of(p, row);
                const T *src = static_cast<const T *>(p.q) + (int64_t)(item.token0 + token) * p.q_token + (int64_t)(item.head * p.group + row - token * p.group) * p.q_head;
                float f[(D + 127) / 128][4];
                float top = 0.0f;
#pragma unroll
                for (int j = 0; j < (D + 127) / 128; ++j) {
                    const int d = 4 * lane + 128 * j;
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[j][e] = 0.0f;
                    if (r < item.rows && d < D) load_q4(src + d, f[j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(f[j][e]));
                }
                float up = 1.0f, down = 1.0f;
                if (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
                    for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
                    if (top > 0.0f) down = __uint_as_float((254u - e) << 23), up = __uint_as_float(e << 23);
                }
                if (lane == 0) ctl.q_scale[r] = fmaxf(up * p.scale_log2, kLeastNormal);  // not zero, which makes NaN of a hidden position's -inf
#pragma unroll
                for (int j = 0; j < (D + 127) / 128; ++j) {
                    const int d = 4 * lane + 128 * j;
                    if (d < D) {
                        const uint32_t at = (((r >> 3) * (D / 16) + (d >> 4)) * 32 + ((r & 7) << 2) + ((d >> 2) & 3)) * 8;
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(q_frag + at), "r"(pack_f16(f[j][0] * down, f[j][1] * down)), "r"(pack_f16(f[j][2] * down, f[j][3] * down)) : "memory");
                    }
                }
            }
            sync_of<CONSUMERS>();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int n = 0; n < D / 16; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][n][e] = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    m[nt][h] = kNothing;
                    limit[nt][h] = -INFINITY;
                    l[nt][h] = 0.0f;
                    qs[nt][h] = ctl.q_scale[8 * nt + 2 * t + h];
                    v_inv[nt][h] = power_over(kLeastNormal);
                }
            }
            if (L::Q_IN_REGISTERS) {
#pragma unroll
                for (int i = 0; i < NT * D / 16; ++i) q_reg[L::Q_IN_REGISTERS ? i : 0] = lds64(q_frag + (i * 32 + lane) * 8);
            }
        }
        for (;;) {
            wait_for(ctl.full[slot], parity);
            if (!alive) break;
            const Tile tile = ctl.tiles[slot];
            const int key0 = tile.key0 + 16 * warp;
            if (key0 < length) {
                const uint32_t rec = stages + slot * L::STAGE + warp * L::RECORD;
                const uint32_t scales = rec + 32 * D + 4 * key_of_lane;
                const float ks[2] = {lds32(scales), lds32(scales + 8)};
                float vs[2] = {lds32(scales + 64), lds32(scales + 72)};
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nt][e] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < D / 32; ++kk) {
                    uint32_t r[4];
                    umma::ldmatrix_x4(r, rec + k_off + (((2 * kk + k_chunk) ^ k_sw) << 4));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t a[4];
                        codes_to_f16(r[2 * i], a[0], a[2]);
                        codes_to_f16(r[2 * i + 1], a[1], a[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const int at = nt * (D / 16) + 2 * kk + i;
                            const uint2 b = L::Q_IN_REGISTERS ? q_reg[L::Q_IN_REGISTERS ? at : 0] : lds64(q_frag + (at * 32 + lane) * 8);
                            mma_m16n8k16(s[nt], a[0], a[1], a[2], a[3], b.x, b.y);
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nt][e] *= ks[e >> 1];
                const bool partly = key0 + 16 > hidden;
                if (partly) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        bool seen[4];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int r = 8 * nt + 2 * t + e, token = token_of(p, item.row0 + r);
#pragma unroll
                            for (int h = 0; h < 2; ++h) seen[2 * h + e] = may_see(p, item, r, token, key0 + key_of_lane + 2 * h);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!seen[e]) s[nt][e] = -INFINITY;
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (key0 + key_of_lane + 2 * h >= length) vs[h] = 0.0f;
                }
                bool up = fmaxf(vs[0], vs[1]) >= v_limit;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) up |= fmaxf(s[nt][h], s[nt][2 + h]) > limit[nt][h];
                if (__any_sync(0xffffffffu, up)) {  // then each row by what it sees itself, whatever the others do
                    v_limit = INFINITY;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float by[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float n = fmaxf(s[nt][h], s[nt][2 + h]), v = fmaxf(s[nt][h] == -INFINITY ? 0.0f : vs[0], s[nt][2 + h] == -INFINITY ? 0.0f : vs[1]);
#pragma unroll
                            for (int d = 4; d < 32; d *= 2) {
                                n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, d));
                                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
                            }
                            float alpha = 1.0f;
                            if (n > limit[nt][h]) {
                                alpha = ex2((m[nt][h] - n) * qs[nt][h]);
                                m[nt][h] = n;
                                float rise;
                                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rise) : "f"(qs[nt][h]));
                                limit[nt][h] = n + fminf(kRise * rise, 1e38f);
                            }
                            const float v_ref = power_over(v_inv[nt][h]), v_new = __uint_as_float(__float_as_uint(fmaxf(v, v_ref)) & 0x7f800000u), beta = v_ref * power_over(v_new);
                            v_inv[nt][h] = power_over(v_new);
                            if (m[nt][h] > kNothing) v_limit = fminf(v_limit, 2.0f * v_new);  // else its first position will pass the other limit
                            l[nt][h] *= alpha;
                            by[h] = alpha * beta;
                        }
#pragma unroll
                        for (int n = 0; n < D / 16; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[nt][n][e] *= by[e & 1];
                    }
                    __syncwarp();
                }
                uint32_t b[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = ex2(fmaf(s[nt][e] - m[nt][e & 1], qs[nt][e & 1], kBias));
                        l[nt][e & 1] += x[e];
                        x[e] *= vs[e >> 1] * v_inv[nt][e & 1];
                        if (partly && s[nt][e] == -INFINITY) x[e] = 0.0f;  // whatever the scale of a position that is not seen
                    }
                    b[nt][0] = transpose(pack_f16(x[0], x[1]));
                    b[nt][1] = transpose(pack_f16(x[2], x[3]));
                }
#pragma unroll
                for (int dd = 0; dd < D / 32; ++dd) {
                    uint32_t r[4];
                    umma::ldmatrix_x2_trans_b8(r, rec + v_off + (((2 * dd + v_chunk) ^ v_sw) << 4));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t a[4];
                        codes_to_f16(r[2 * i], a[0], a[2]);
                        codes_to_f16(r[2 * i + 1], a[1], a[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_m16n8k16(o[nt][2 * dd + i], a[0], a[1], a[2], a[3], b[nt][0], b[nt][1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl.empty[slot]));
            if (++slot == STAGES) slot = 0, parity ^= 1;
            if (tile.last) break;
        }
        if (!alive) break;

        // ---- the warps' sums meet ----
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int d = 4; d < 32; d *= 2) l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], d);
                if (g == 0) {
                    ctl.m[warp][8 * nt + 2 * t + h] = m[nt][h];
                    ctl.l[warp][8 * nt + 2 * t + h] = l[nt][h];
                }
            }
        if (!all_of<CONSUMERS>(true)) {
            met = true;
            break;
        }
        float factor[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) factor[nt][h] = ex2((m[nt][h] - row_top(ctl, 8 * nt + 2 * t + h)) * qs[nt][h]) * power_over(v_inv[nt][h]);
        float *mine = merge + (warp % L::BUFFERS) * (L::MERGE / 4) + 2 * t * L::PITCH + g;
        if (warp >= L::BUFFERS) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int n = 0; n < D / 16; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mine[(8 * nt + (e & 1)) * L::PITCH + 16 * n + 8 * (e >> 1)] = o[nt][n][e] * factor[nt][e & 1];
        }
        sync_of<CONSUMERS>();
        if (warp < L::BUFFERS) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int n = 0; n < D / 16; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float *at = mine + (8 * nt + (e & 1)) * L::PITCH + 16 * n + 8 * (e >> 1);
                        *at = fmaf(o[nt][n][e], factor[nt][e & 1], *at);
                    }
        }
        sync_of<CONSUMERS>();
        finish_item<D, NT, T>(p, ctl, merge, item);
        // the merge buffers and statistics are written again only behind the barrier in front of the next item's queries
    }
    if (!met) all_of<CONSUMERS>(alive);
}

template <int D, int NT, typename T>
int launch_sized(AttentionArgs p, cudaStream_t stream) {
    using L = Layout<D, NT>;
    auto kernel = cache_attention_kernel<D, NT, T>;
    static std::atomic<bool> attr_set[64];
    const int rc = allow_smem(attr_set, kernel, L::SMEM);
    if (rc != B200Q_OK) return rc;
    const int64_t tiles = most_tiles(p, L::ROWS), at_once = L::PER_SM * (int64_t)sm_count();
    if (tiles > (1ll << 29)) return set_error(B200Q_UNSUPPORTED, "quantized_cache_attention: up to %lld tiles of %d rows and %d positions", (long long)tiles, L::ROWS, TILE);
    int64_t grid = tiles < at_once ? tiles : at_once;
    if (grid > kMaxCtas) grid = kMaxCtas;
    if (grid < 1) grid = 1;  // no sequences, whose rows are written all the same
    return launch_after("cache_attention_kernel", kernel, dim3((unsigned)grid), THREADS, L::SMEM, 1, stream, p);
}

// Items of 8 query rows, and of 16 where more than 8 share a key/value head and there is much work: these read the cache once for twice the rows, but a tile, an item's ends
// and the additions take them half as long again, and fewer fit an SM.  Measured (8 / 16 rows, us; tiles as in is_wide): 1 sequence of 512 positions, 8 heads of
// 128, 16 rows (72 tiles) 9.2 / 12.7; of 16384 (2056) 21.7 / 28.9; 16 of 4096 (8320) 49.7 / 51.5; 24 of 4000 (12288) 67.3 / 66.3, with 64 elements 49.2 / 41.4, 96: 60.9 / 55.7,
// 192: 99.5 / 86.4, 256: 138 / 125; 1 of 131071 (16392) 92 / 83.
template <typename T>
int launch_typed(const AttentionArgs &p, int dim, cudaStream_t stream) {
    const bool sixteen = p.batch > 0 && p.tokens * p.group > 8 * (int64_t)p.batch && tiles_of_16(p) > 10000;
    switch (dim) {
        case 64: return sixteen ? launch_sized<64, 2, T>(p, stream) : launch_sized<64, 1, T>(p, stream);
        case 96: return sixteen ? launch_sized<96, 2, T>(p, stream) : launch_sized<96, 1, T>(p, stream);
        case 128: return sixteen ? launch_sized<128, 2, T>(p, stream) : launch_sized<128, 1, T>(p, stream);
        case 192: return sixteen ? launch_sized<192, 2, T>(p, stream) : launch_sized<192, 1, T>(p, stream);
        default: return sixteen ? launch_sized<256, 2, T>(p, stream) : launch_sized<256, 1, T>(p, stream);
    }
}

}  // namespace
}  // namespace cache_attention
}  // namespace b200q

extern "C" {

B200Q_API size_t b200q_quantized_cache_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim) {
    using namespace b200q;
    using namespace b200q::cache_attention;
    if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || !cache_dim(head_dim)) return 0;
    const int64_t few = (int64_t)2 * kMaxCtas * 16 * (head_dim + 2) * 4;
    const int64_t many = may_be_wide(tokens, heads / kv_heads, batch, head_dim) ? (int64_t)2 * kMostWideCtas * 128 * (head_dim + 2) * 4 + kMostWideCtas * 64 : 0;  // 64: an item's description
    return kWorkspaceHead + (size_t)(few > many ? few : many);
}

B200Q_API int b200q_quantized_cache_attention(const b200q_heads *q, void *out, float *lse, const void *cache, int64_t pages, int64_t page_size, const int32_t *page_table,
                                              int64_t table_width, int64_t table_stride, const int32_t *lengths, const int32_t *starts, const void *mask, int64_t mask_width,
                                              int64_t mask_stride, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, int type,
                                              void *workspace, size_t workspace_bytes, void *stream) {
    using namespace b200q;
    using namespace b200q::cache_attention;
    const char *op = "quantized_cache_attention";
    if (batch < 0 || tokens < 0 || table_width < 0 || mask_width < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative size", op);
    if (type != B200Q_F16 && type != B200Q_BF16) return set_error(B200Q_UNSUPPORTED, "%s: float type %d: float16 and bfloat16 are supported", op, type);
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: %lld heads over %lld key/value heads", op, (long long)heads, (long long)kv_heads);
    }
    if (page_size <= 0 || page_size % 16 != 0 || page_size > 65536) {
        return set_error(B200Q_UNSUPPORTED, "%s: pages of %lld positions: multiples of 16 up to 65536 are supported", op, (long long)page_size);
    }
    if (!cache_dim(head_dim)) return set_error(B200Q_UNSUPPORTED, "%s: heads of %lld elements: 64, 96, 128, 192 and 256 are supported", op, (long long)head_dim);
    if (!(scale > 0.0f) || scale > 1e30f || scale < 1e-20f) return set_error(B200Q_INVALID_ARGUMENT, "%s: the scale must be a positive number, got %g", op, (double)scale);
    if (tokens == 0) return B200Q_OK;
    if (starts == nullptr && batch > 0 && tokens % batch != 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: %lld tokens of %lld sequences need starts", op, (long long)tokens, (long long)batch);
    if (batch > 1 << 20 || kv_heads > 65536 || tokens > (1ll << 31) / 4 / heads) return set_error(B200Q_UNSUPPORTED, "%s: %lld sequences, %lld tokens of %lld heads", op, (long long)batch, (long long)tokens, (long long)heads);
    if (q == nullptr || q->data == nullptr || out == nullptr || (batch > 0 && (lengths == nullptr || (table_width > 0 && page_table == nullptr))) || (pages > 0 && cache == nullptr)) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    }
    if (batch > 0 && pages <= 0 && table_width > 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: a cache of %lld pages", op, (long long)pages);
    if (!aligned_to(cache, 16) || !aligned_to(q->data, 16) || !aligned_to(out, 16) || q->token_stride % 8 != 0 || q->head_stride % 8 != 0) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: 16-byte aligned cache, q and out and strides of 8 elements are wanted", op);
    }
    const size_t need = b200q_quantized_cache_attention_workspace_bytes(batch, tokens, heads, kv_heads, head_dim);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return set_error(B200Q_WORKSPACE_TOO_SMALL, "%s: a workspace of %zu bytes is needed, got %zu", op, need, workspace_bytes);
    if (!aligned_to(workspace, 16)) return set_error(B200Q_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", op);
    AttentionArgs p = {};
    p.q = q->data;
    p.q_token = q->token_stride;
    p.q_head = q->head_stride;
    p.out = out;
    p.lse = lse;
    p.cache = static_cast<const uint8_t *>(cache);
    p.pages = pages;
    p.page_size = (int)page_size;
    p.table = page_table;
    p.table_stride = table_stride;
    const int64_t most = (1ll << 31) - 65536 * 2;  // positions are counted in 32 bits, past the end of a tile
    p.capacity = table_width < most / page_size ? table_width * page_size : most;
    p.lengths = lengths;
    p.starts = starts;
    p.tokens = tokens;
    p.per_sequence = starts == nullptr && batch > 0 ? (int)(tokens / batch) : 0;
    p.mask = static_cast<const uint8_t *>(mask);
    p.mask_stride = mask_stride;
    p.mask_width = mask == nullptr ? 0 : (int)(mask_width < (1 << 30) ? mask_width : 1 << 30);  // what lies inside the width is read
    p.batch = (int)batch;
    p.kv_heads = (int)kv_heads;
    p.group = (int)(heads / kv_heads);
    p.by_group = divisor_of((uint32_t)p.group);
    p.scale_log2 = scale * kLog2e;
    p.counters = static_cast<unsigned int *>(workspace);
    p.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kWorkspaceHead);
    p.partial_floats = (int64_t)2 * kMostWideCtas * 128 * (head_dim + 2);  // of the kernel for many rows
    p.status = device_status_word();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (is_wide(p, head_dim)) return launch_wide(p, (int)head_dim, type == B200Q_BF16, s);
    return type == B200Q_F16 ? launch_typed<__half>(p, (int)head_dim, s) : launch_typed<__nv_bfloat16>(p, (int)head_dim, s);
}

}  // extern "C"
