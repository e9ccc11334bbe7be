// Attention of new tokens (one a sequence, several, or a tree of drafted ones) over the quantized, paged key/value cache.
//
// For query row i (a token and one of the `group` heads that share a key/value head) and position j:
//     s_ij = scale * (q_i . kcode_j) * kscale_j,     o_i = sum_j exp(s_ij - m_i) * vscale_j * vcode_j / sum_j exp(s_ij - m_i)
// over the positions that the row may see, with the running maximum m_i and sum of one pass over the cache.  Codes are exact in f16, so
// the products q . kcode run on f16 tensor-core instructions with float sums; bf16 queries go through f16 too, scaled row by row by a power of
// two (their eight bits fit; what is 2^-24 of the row's largest element is lost).  Probabilities, times vscale_j over the power of two below the largest vscale so far (so that
// they cannot leave f16's range whatever the values' size), are rounded to f16 for the second product, an error of 2^-12 of each, at random; the sums
// that divide are float.
//
// A unit of work is a tile of positions for one (sequence, key/value head, 16 * MT query rows).  The tiles of all sequences stand in
// one line, which is cut into equal pieces, one a CTA, whatever the sequences' lengths are (the host does not know them: they
// are on the device, so that a captured step can be replayed as they grow).  A CTA's piece may end one item and begin others; items in
// several pieces leave partial sums in the workspace, and the CTA that arrives last adds them in the order of the pieces.
//
// One warp copies whole records (codes and scales, one bulk copy per run of a page) into a ring of shared memory; each of
// the other warps takes one record of 16 positions of a tile: it loads K fragments with plain and V fragments with transposing matrix loads, converts
// two codes an instruction and multiplies.  With the positions (and not the rows) shared out among the warps, each code is converted
// once per CTA.
#include <atomic>
#include <type_traits>

#include "serving.cuh"
#include "umma.cuh"

namespace b200q {
namespace {

constexpr unsigned int kKernelCacheAttention = 7;
constexpr int kMaxCtas = 2 * 148;         // of a launch; the workspace is made for them
constexpr int kCounterBytes = 65536 * 4;  // arrival counters in front of the workspace, zero between calls
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are kept 2^6 times as large, and a row's maximum is raised when a score passes it by 2^8 (rarely, behind its first
// positions): with a value's scale below 2 that is at most 2^15 of f16's 2^16, and a probability of 2^-31 is still there, so that a long tail of
// small ones is not lost.
constexpr float kBias = 6.0f, kRise = 8.0f;
constexpr float kLeastNormal = 1.1754943508222875e-38f;

struct AttentionArgs {
    const void *q;
    int64_t q_token, q_head;
    void *out;
    float *lse;
    const uint8_t *cache;
    int64_t pages;
    int page_size;
    const int32_t *table;
    int64_t table_stride;
    int64_t capacity;  // positions that a row of the table covers
    const int32_t *lengths, *starts;
    int64_t tokens;    // all rows of q
    int per_sequence;  // tokens of every sequence where starts is null
    const uint8_t *mask;
    int64_t mask_stride;
    int mask_width;
    int batch, kv_heads, group;
    float scale_log2;
    float *partial;
    unsigned int *counters;
    unsigned int *status;
};

// What a consumer has to know of a tile.
struct Step {
    int head, row0, rows;  // key/value head; first query row (token * group + head in group) and rows of this item
    int key0, length, fresh;  // first position of the tile; cached positions; of them those of the new tokens
    int token0;
    int flags;
    int first_cta, last_cta, slot;  // of an item in several pieces: who holds them, and where this CTA's goes
    int first_slot;
};
constexpr int kFirst = 1, kLast = 2, kEnd = 4;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Four bytes of code + 128 -> f16 pairs of codes (0x6400 | u is 1024 + u).
__device__ __forceinline__ void codes_to_f16(uint32_t u, uint32_t &p01, uint32_t &p23) {
    const uint32_t bias = 0x64806480u;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(p01) : "r"(__byte_perm(u, 0x64646464u, 0x4140)), "r"(bias));
    asm("sub.f16x2 %0, %1, %2;" : "=r"(p23) : "r"(__byte_perm(u, 0x64646464u, 0x4342)), "r"(bias));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

constexpr int MOST_STAGES = 6;

template <int D, int MT, int WARPS>
struct Layout {
    static constexpr int TILE = 16 * WARPS;  // positions
    static constexpr int ROWS = 16 * MT;
    static constexpr int RECORD = record_bytes(D);
    static constexpr int STAGE = WARPS * RECORD;
    static constexpr int PITCH = D + 8;  // floats between rows of a merge buffer: eight rows of float2 in different banks
    static constexpr int MERGE = ROWS * PITCH * 4;
    static constexpr int BUFFERS = WARPS / 2;
    static constexpr int THREADS = 32 * WARPS + 32;
    static constexpr int PER_SM = WARPS == 4 ? 2 : 1;
    static constexpr int Q = ROWS * D * 2;
    static constexpr int FIXED = Q + BUFFERS * MERGE;
    static constexpr int ROOM = (PER_SM == 2 ? 113 : 226) * 1024 - 4096 - FIXED;  // 4096: Control, and what an SM keeps for itself
    static constexpr int STAGES = ROOM / STAGE > MOST_STAGES ? MOST_STAGES : ROOM / STAGE;
    static constexpr int SMEM = FIXED + STAGES * STAGE;
    static_assert(STAGES >= 2, "");
};

// One answer for the N threads that meet at named barrier 1: true where all of them bring true.
template <int N>
__device__ __forceinline__ bool all_of(bool ok) {
    uint32_t all;
    __syncwarp();
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.u32 p, %2, 0;\n\t"
        "bar.red.and.pred q, 1, %1, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t"
        "}\n"
        : "=r"(all)
        : "n"(N), "r"((uint32_t)ok)
        : "memory");
    return all != 0;
}

struct Control {
    uint64_t full[MOST_STAGES], empty[MOST_STAGES];
    Step steps[MOST_STAGES];
    float m[8][32], l[8][32], vref[8];  // at most 8 warps, 32 rows
    float q_scale[32];
    int64_t scan[16];
    int64_t begin_offset;
    int begin_sequence, abort, last;
};
static_assert(sizeof(Control) <= 3072, "");

template <typename T>
__device__ __forceinline__ void load_q4(const T *p, float (&f)[4]) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    const T *v = reinterpret_cast<const T *>(&x);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = Elems<T>::one(v[i]);
}

struct Sequence {
    int length, fresh, token0;
    int tiles;     // of one item
    int row_tiles; // items of a key/value head
};
template <int TILE, int ROWS>
__device__ __forceinline__ Sequence sequence_of(const AttentionArgs &p, int b) {
    Sequence s;
    int64_t n = p.lengths[b];
    if (n > p.capacity) {
        n = p.capacity;
        if (p.status != nullptr) atomicOr(p.status, kBadPage);
    }
    s.length = n < 0 ? 0 : (int)n;
    if (p.starts != nullptr) {
        const int64_t first = min(max((int64_t)p.starts[b], (int64_t)0), p.tokens), end = min(max((int64_t)p.starts[b + 1], first), p.tokens);
        s.token0 = (int)first;
        s.fresh = (int)(end - first);
    } else {
        s.token0 = b * p.per_sequence;
        s.fresh = p.per_sequence;
    }
    s.tiles = max(1, (s.length + TILE - 1) / TILE);  // an empty sequence has a tile too: its rows are written
    s.row_tiles = (int)(((int64_t)s.fresh * p.group + ROWS - 1) / ROWS);
    return s;
}

template <int D, int MT, int WARPS, typename T>
__global__ void __launch_bounds__(32 * WARPS + 32, WARPS == 4 ? 2 : 1) cache_attention_kernel(const AttentionArgs p) {
    using L = Layout<D, MT, WARPS>;
    constexpr int TILE = L::TILE, ROWS = L::ROWS, CONSUMERS = 32 * WARPS, STAGES = L::STAGES;
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
        ctl.abort = 0;
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();

    // ---- this CTA's piece of the line of tiles ----
    int64_t sum = 0;
    for (int b = threadIdx.x; b < p.batch; b += L::THREADS) {
        const Sequence s = sequence_of<TILE, ROWS>(p, b);
        sum += (int64_t)s.tiles * s.row_tiles;
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) ctl.scan[warp] = sum;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < WARPS + 1; ++w) total += ctl.scan[w];
    total *= p.kv_heads;
    const int64_t ctas = min((int64_t)gridDim.x, total);
    if (blockIdx.x >= ctas) return;
    const int64_t begin = blockIdx.x * total / ctas, end = (blockIdx.x + 1) * total / ctas;
    // the sequence that `begin` lies in
    int64_t base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += L::THREADS) {
        const int b = b0 + threadIdx.x;
        int64_t own = 0;
        if (b < p.batch) {
            const Sequence s = sequence_of<TILE, ROWS>(p, b);
            own = (int64_t)s.tiles * s.row_tiles * p.kv_heads;
        }
        int64_t incl = own;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int64_t below = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += below;
        }
        __syncthreads();
        if (lane == 31) ctl.scan[warp] = incl;
        __syncthreads();
        int64_t before = base, all = 0;
#pragma unroll
        for (int w = 0; w < WARPS + 1; ++w) {
            if (w < warp) before += ctl.scan[w];
            all += ctl.scan[w];
        }
        const int64_t from = before + incl - own;
        if (from <= begin && begin < from + own) {
            ctl.begin_sequence = b;
            ctl.begin_offset = begin - from;
        }
        base += all;
        if (base > begin) break;
    }
    __syncthreads();

    if (warp == WARPS) {
        // ---------------- producer ----------------
        int b = ctl.begin_sequence;
        int64_t offset = ctl.begin_offset, cur = begin;
        const int records_per_page = p.page_size >> 4;
        int slot = 0, it = 0;
        uint32_t parity = 0;
        bool dead = false;
        auto next_stage = [&]() {
            if (it >= STAGES) {
                const uint32_t bar = smem_u32(&ctl.empty[slot]);
                bool ok = false;
                for (uint32_t i = 0; i < umma::kFastPolls && !ok; ++i) ok = mbar_try_wait(bar, parity ^ 1u);
                if (!ok) ok = umma::wait_or_abort<kKernelCacheAttention>(bar, parity ^ 1u, 1, &ctl.abort, p.status);
                dead = !__all_sync(0xffffffffu, ok);
            }
        };
        while (cur < end && !dead) {
            const Sequence s = sequence_of<TILE, ROWS>(p, b);
            if (s.row_tiles == 0) {
                ++b;
                continue;
            }
            const int64_t item = offset / s.tiles;
            const int tile0 = (int)(offset - item * s.tiles);
            const int head = (int)(item / s.row_tiles), rt = (int)(item - (int64_t)head * s.row_tiles);
            const int n = (int)min((int64_t)(s.tiles - tile0), end - cur);
            const int64_t item_begin = cur - tile0, item_end = item_begin + s.tiles;
            const int first_cta = (int)(((item_begin + 1) * ctas - 1) / total), last_cta = (int)((item_end * ctas - 1) / total);
            const int first_slot = first_cta * total / ctas == item_begin ? 0 : 1;
            const int32_t *pages = p.table + (int64_t)b * p.table_stride;
            // lane i < 8 brings the i-th page that the tile touches; its number is asked for one tile ahead
            auto page_of = [&](int tile) {
                const int page = tile * TILE / p.page_size + lane;
                return tile < tile0 + n && lane <= WARPS && (int64_t)page * p.page_size < s.length ? pages[page] : 0;
            };
            int page = page_of(tile0);
            for (int i = 0; i < n && !dead; ++i) {
                const int tile = tile0 + i, key0 = tile * TILE;
                const int next = page_of(tile + 1);
                next_stage();
                if (dead) break;
                const int keys = min(TILE, (s.length - key0 + 15) & ~15);  // 0 where the sequence is empty
                const uint32_t bar = smem_u32(&ctl.full[slot]);
                if (lane == 0) {
                    Step &st = ctl.steps[slot];
                    st.head = head;
                    st.row0 = rt * ROWS;
                    st.rows = min(ROWS, s.fresh * p.group - rt * ROWS);
                    st.key0 = key0;
                    st.length = s.length;
                    st.fresh = s.fresh;
                    st.token0 = s.token0;
                    st.flags = (i == 0 ? kFirst : 0) | (i == n - 1 ? kLast : 0);
                    st.first_cta = first_cta;
                    st.last_cta = last_cta;
                    st.first_slot = first_slot;
                    st.slot = 2 * blockIdx.x + (cur == begin ? 0 : 1);
                    if (keys > 0) mbar_expect_tx(bar, (uint32_t)(keys >> 4) * L::RECORD);
                    else mbar_arrive(bar);
                }
                __syncwarp();
                const int at = (key0 / p.page_size + lane) * p.page_size;  // first position of this lane's page
                const int from = max(at, key0), to = min(at + p.page_size, key0 + keys);
                if (lane <= WARPS && from < to) {
                    if (page < 0 || page >= p.pages) {
                        page = 0;
                        if (p.status != nullptr) atomicOr(p.status, kBadPage);
                    }
                    const uint8_t *src = p.cache + (((int64_t)page * p.kv_heads + head) * records_per_page + ((from - at) >> 4)) * L::RECORD;
                    bulk_load(stages + slot * L::STAGE + ((from - key0) >> 4) * L::RECORD, src, (uint32_t)((to - from) >> 4) * L::RECORD, bar);
                }
                page = next;
                ++it;
                if (++slot == STAGES) slot = 0, parity ^= 1u;
            }
            cur += n;
            offset += n;
            if (offset == (int64_t)s.tiles * s.row_tiles * p.kv_heads) ++b, offset = 0;
        }
        if (!dead) {
            next_stage();
            if (!dead && lane == 0) {
                ctl.steps[slot].flags = kEnd;
                mbar_arrive(smem_u32(&ctl.full[slot]));
            }
        }
        if (dead) {  // nothing may be on its way when the CTA ends
            for (int back = 1; back <= STAGES && back <= it; ++back) {
                const int s = (it - back) % STAGES;
                mbar_wait(smem_u32(&ctl.full[s]), ((it - back) / STAGES) & 1, 1u << 16);
            }
        }
        return;
    }

    // ---------------- consumers ----------------
    const int g = lane >> 2, t = lane & 3;
    // K: lane l addresses row 4 (c / 2) + c % 2 + 2 (l / 16) of its record, c = l % 8, and of a pair of chunks the (l / 8 % 2)-th.  So MMA
    // columns 2t, 2t + 1 of the first matrix are positions 4t, 4t + 1 and of the second 4t + 2, 4t + 3: the four whose codes a transposing
    // load of V leaves in one register of this lane.  Inside a chunk a lane holds elements 4t .. 4t + 3; the query's fragments follow that.
    const uint32_t k_row = 4 * ((lane & 7) >> 1) + (lane & 1) + 2 * (lane >> 4);
    const uint32_t k_off = k_row * D, k_sw = k_order(k_row, D), k_chunk = (lane >> 3) & 1;
    const uint32_t v_row = lane & 15;
    const uint32_t v_off = 16 * D + v_row * D, v_sw = v_order(v_row, D), v_chunk = lane >> 4;
    float o[MT][D / 8][4];
    float m[MT][2], l[MT][2], shift[MT][2], qs[MT][2], rise[MT][2];  // shift: m, or 0 as long as nothing was seen
    float vref = 0.0f, v_inv = 0.0f, v_limit = kLeastNormal;  // a power of two, its reciprocal, and the first scale that is too large for it
    // A warp whose wait runs out brings `false` to the next barrier of all consumers, where all of them leave: one by one, it would
    // leave the others waiting there.  `met`: this warp has been at that barrier.
    bool alive = true, met = false;
    for (int slot = 0, parity = 0;;) {
        {
            const uint32_t bar = smem_u32(&ctl.full[slot]);
            bool ok = false;
            for (uint32_t i = 0; i < umma::kFastPolls && !ok; ++i) ok = mbar_try_wait(bar, parity);
            if (!ok) ok = umma::wait_or_abort<kKernelCacheAttention>(bar, parity, 2, &ctl.abort, p.status);
            alive = __all_sync(0xffffffffu, ok);
        }
        if (!alive) break;
        const Step st = ctl.steps[slot];
        if (st.flags & kEnd) break;
        if (st.flags & kFirst) {
            // the queries, as MMA fragments: for chunk c and rows g, g + 8 lane (g, t) has elements 16 c + 4t .. + 3 of both
            if (!all_of<CONSUMERS>(true)) {
                met = true;
                break;
            }
#pragma unroll
            for (int r0 = 0; r0 < ROWS; r0 += WARPS) {
                const int r = r0 + warp;
                const int row = st.row0 + r, token = row / p.group;
                const T *src = static_cast<const T *>(p.q) + (int64_t)(st.token0 + token) * p.q_token + (int64_t)(st.head * p.group + row - token * p.group) * p.q_head;
                float f[(D + 127) / 128][4];
                float top = 0.0f;
#pragma unroll
                for (int j = 0; j < (D + 127) / 128; ++j) {
                    const int d = 4 * lane + 128 * j;
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[j][e] = 0.0f;
                    if (r < st.rows && d < D) load_q4(src + d, f[j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(f[j][e]));
                }
                float up = 1.0f, down = 1.0f;
                if (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
                    for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const uint32_t e = min(max(__float_as_uint(top) >> 23, 64u), 253u);
                    if (top > 0.0f) down = __uint_as_float((254u - e) << 23), up = __uint_as_float(e << 23);
                }
                if (lane == 0) ctl.q_scale[r] = up * p.scale_log2;
#pragma unroll
                for (int j = 0; j < (D + 127) / 128; ++j) {
                    const int d = 4 * lane + 128 * j;
                    if (d < D) {
                        const uint32_t at = (((r >> 4) * (D / 16) + (d >> 4)) * 32 + ((r & 7) << 2) + ((d >> 2) & 3)) * 16 + ((r >> 3) & 1) * 4;
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(q_frag + at), "r"(pack_f16(f[j][0] * down, f[j][1] * down)) : "memory");
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(q_frag + at + 8), "r"(pack_f16(f[j][2] * down, f[j][3] * down)) : "memory");
                    }
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    m[mt][h] = -INFINITY;
                    l[mt][h] = shift[mt][h] = 0.0f;
                    qs[mt][h] = ctl.q_scale[16 * mt + 8 * h + g];
                    rise[mt][h] = fminf(kRise / qs[mt][h], 1e38f);
                }
            }
            vref = v_inv = 0.0f;
            v_limit = kLeastNormal;
        }
        const int key0 = st.key0 + 16 * warp;
        if (key0 < st.length) {
            const uint32_t rec = stages + slot * L::STAGE + warp * L::RECORD;
            const uint4 ks4 = lds128(rec + 32 * D + 16 * t), vs4 = lds128(rec + 32 * D + 64 + 16 * t);
            const float ks[4] = {__uint_as_float(ks4.x), __uint_as_float(ks4.y), __uint_as_float(ks4.z), __uint_as_float(ks4.w)};
            float vs[4] = {__uint_as_float(vs4.x), __uint_as_float(vs4.y), __uint_as_float(vs4.z), __uint_as_float(vs4.w)};
            float c[MT][2][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[mt][j][e] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) {
                uint32_t r[4];
                umma::ldmatrix_x4(r, rec + k_off + (((2 * kk + k_chunk) ^ k_sw) << 4));
                uint32_t b[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) codes_to_f16(r[i], b[i][0], b[i][1]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 a = lds128(q_frag + ((mt * (D / 16) + 2 * kk + i) * 32 + lane) * 16);
                        mma_m16n8k16(c[mt][0], a.x, a.y, a.z, a.w, b[i][0], b[i][1]);
                        mma_m16n8k16(c[mt][1], a.x, a.y, a.z, a.w, b[2 + i][0], b[2 + i][1]);
                    }
            }
            // scores, four positions of each of the lane's rows
            float s[MT][2][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[mt][h][e] = c[mt][e >> 1][2 * h + (e & 1)] * ks[e];
            const int old = st.length - st.fresh;  // positions in front of the new tokens
            const bool partly = key0 + 16 > (p.mask != nullptr ? old : min(old + 1, st.length));
            if (partly) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (key0 + 4 * t + e >= st.length) vs[e] = 0.0f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = 16 * mt + 8 * h + g, token = (st.row0 + r) / p.group;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int pos = key0 + 4 * t + e, drafted = pos - old;
                            bool seen = pos < st.length && r < st.rows;
                            if (seen && drafted >= 0) {
                                seen = p.mask == nullptr ? drafted <= token : drafted < p.mask_width && p.mask[(int64_t)(st.token0 + token) * p.mask_stride + drafted] != 0;
                            }
                            if (!seen) s[mt][h][e] = -INFINITY;
                        }
                    }
            }
            bool up = false;
            const float v_top = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
            up = v_top >= v_limit;
            float top[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[mt][h] = fmaxf(fmaxf(s[mt][h][0], s[mt][h][1]), fmaxf(s[mt][h][2], s[mt][h][3]));
                    up |= top[mt][h] > m[mt][h] + rise[mt][h];
                }
            if (__any_sync(0xffffffffu, up)) {
                float v_new = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, 1));
                v_new = fmaxf(fmaxf(v_new, __shfl_xor_sync(0xffffffffu, v_new, 2)), vref);
                const uint32_t power = __float_as_uint(v_new) & 0x7f800000u;
                const float beta = power != 0 ? vref * __uint_as_float(0x7f000000u - power) : 1.0f;
                vref = __uint_as_float(power);
                v_inv = power != 0 ? __uint_as_float(0x7f000000u - power) : 0.0f;
                v_limit = power != 0 ? 2.0f * vref : kLeastNormal;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float by[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float n = fmaxf(top[mt][h], __shfl_xor_sync(0xffffffffu, top[mt][h], 1));
                        n = fmaxf(fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 2)), m[mt][h]);
                        const float alpha = n == -INFINITY ? 1.0f : ex2((m[mt][h] - n) * qs[mt][h]);
                        m[mt][h] = n;
                        shift[mt][h] = n == -INFINITY ? 0.0f : n;
                        l[mt][h] *= alpha;
                        by[h] = alpha * beta;
                    }
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) {
                        o[mt][n][0] *= by[0];
                        o[mt][n][1] *= by[0];
                        o[mt][n][2] *= by[1];
                        o[mt][n][3] *= by[1];
                    }
                }
            }
            uint32_t a[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = ex2(fmaf(s[mt][h][e] - shift[mt][h], qs[mt][h], kBias));
                        l[mt][h] += x;
                        w[e] = x * (vs[e] * v_inv);
                        if (partly && s[mt][h][e] == -INFINITY) w[e] = 0.0f;  // whatever the scale of a position that is not seen
                    }
                    a[mt][h] = pack_f16(w[0], w[1]);
                    a[mt][2 + h] = pack_f16(w[2], w[3]);
                }
#pragma unroll
            for (int dd = 0; dd < D / 32; ++dd) {
                uint32_t r[4];
                umma::ldmatrix_x2_trans_b8(r, rec + v_off + (((2 * dd + v_chunk) ^ v_sw) << 4));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t b0, b1;
                    codes_to_f16(r[i], b0, b1);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) mma_m16n8k16(o[mt][4 * dd + i], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b0, b1);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.empty[slot]));
        if (++slot == STAGES) slot = 0, parity ^= 1;
        if (!(st.flags & kLast)) continue;

        // ---- the warps' sums meet ----
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 1);
                l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 2);
                if (t == 0) {
                    ctl.m[warp][16 * mt + 8 * h + g] = m[mt][h];
                    ctl.l[warp][16 * mt + 8 * h + g] = l[mt][h];
                }
            }
        if (!all_of<CONSUMERS>(true)) {
            met = true;
            break;
        }
        auto row_top = [&](int r) {
            float n = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) n = fmaxf(n, ctl.m[w][r]);
            return n;
        };
        float factor[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) factor[mt][h] = m[mt][h] == -INFINITY ? vref : ex2((m[mt][h] - row_top(16 * mt + 8 * h + g)) * qs[mt][h]) * vref;
        float *mine = merge + (warp % L::BUFFERS) * (L::MERGE / 4) + g * L::PITCH + 2 * t;
        if (warp >= L::BUFFERS) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        *reinterpret_cast<float2 *>(mine + (16 * mt + 8 * h) * L::PITCH + 8 * n) = make_float2(o[mt][n][2 * h] * factor[mt][h], o[mt][n][2 * h + 1] * factor[mt][h]);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
        if (warp < L::BUFFERS) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float2 *at = reinterpret_cast<float2 *>(mine + (16 * mt + 8 * h) * L::PITCH + 8 * n);
                        const float2 other = *at;
                        *at = make_float2(fmaf(o[mt][n][2 * h], factor[mt][h], other.x), fmaf(o[mt][n][2 * h + 1], factor[mt][h], other.y));
                    }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
        const bool whole = st.first_cta == st.last_cta;
        float *part = p.partial + (int64_t)st.slot * ROWS * (D + 2);
        constexpr int VECS = ROWS * D / 4;
        auto write_out = [&](int r, int d, float4 v, float total_l, float top_log2) {
            const int row = st.row0 + r, token = row / p.group, head = st.head * p.group + row - token * p.group;
            const int64_t at = (int64_t)(st.token0 + token) * p.kv_heads * p.group + head;
            const float inv = total_l == 0.0f ? 0.0f : 1.0f / total_l;
            T y[4] = {Elems<T>::round(v.x * inv), Elems<T>::round(v.y * inv), Elems<T>::round(v.z * inv), Elems<T>::round(v.w * inv)};
            *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + at * D + d) = *reinterpret_cast<const uint2 *>(y);
            if (d == 0 && p.lse != nullptr) p.lse[at] = total_l == 0.0f ? -INFINITY : (top_log2 - kBias + __log2f(total_l)) * kLn2;
        };
        for (int i = threadIdx.x; i < VECS; i += CONSUMERS) {
            const int r = i / (D / 4), d = 4 * (i % (D / 4));
            if (r >= st.rows) break;
            const float top = row_top(r), scale = ctl.q_scale[r];
            float sum_l = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum_l += ctl.m[w][r] == -INFINITY ? ctl.l[w][r] : ctl.l[w][r] * ex2((ctl.m[w][r] - top) * scale);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < L::BUFFERS; ++k) {
                const float4 x = *reinterpret_cast<const float4 *>(merge + k * (L::MERGE / 4) + r * L::PITCH + d);
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
            const float top_log2 = top * scale;
            if (whole) {
                write_out(r, d, v, sum_l, top_log2);
            } else {
                __stcg(reinterpret_cast<float4 *>(part + r * D + d), v);
                if (d == 0) {
                    __stcg(part + ROWS * D + r, top_log2);
                    __stcg(part + ROWS * (D + 1) + r, sum_l);
                }
            }
        }
        if (!whole) {
            __threadfence();
            asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
            const int parts = st.last_cta - st.first_cta + 1;
            if (threadIdx.x == 0) {
                const unsigned int before = atomicAdd(p.counters + st.first_cta, 1u);
                ctl.last = before == (unsigned int)(parts - 1);
                if (ctl.last) p.counters[st.first_cta] = 0;
                __threadfence();
            }
            asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
            if (ctl.last) {
                __threadfence();
                auto part_of = [&](int k) { return p.partial + (int64_t)(2 * (st.first_cta + k) + (k == 0 ? st.first_slot : 0)) * ROWS * (D + 2); };
                for (int i = threadIdx.x; i < VECS; i += CONSUMERS) {
                    const int r = i / (D / 4), d = 4 * (i % (D / 4));
                    if (r >= st.rows) break;
                    float top = -INFINITY, sum_l = 0.0f;
#pragma unroll 8
                    for (int k = 0; k < parts; ++k) top = fmaxf(top, __ldcg(part_of(k) + ROWS * D + r));
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                    for (int k = 0; k < parts; ++k) {
                        const float *from = part_of(k);
                        const float4 x = __ldcg(reinterpret_cast<const float4 *>(from + r * D + d));
                        const float own = __ldcg(from + ROWS * D + r), part_l = __ldcg(from + ROWS * (D + 1) + r);
                        const float by = own == -INFINITY ? 1.0f : ex2(own - top);
                        sum_l = fmaf(part_l, by, sum_l);
                        v.x = fmaf(x.x, by, v.x), v.y = fmaf(x.y, by, v.y), v.z = fmaf(x.z, by, v.z), v.w = fmaf(x.w, by, v.w);
                    }
                    write_out(r, d, v, sum_l, top);
                }
            }
        }
        // the merge buffers and statistics are written again only behind the barrier in front of the next item's queries
    }
    if (!met) all_of<CONSUMERS>(alive);
}

template <int D, int MT, int WARPS, typename T>
int launch_sized(AttentionArgs p, int64_t most_tiles, cudaStream_t stream) {
    using L = Layout<D, MT, WARPS>;
    auto kernel = cache_attention_kernel<D, MT, WARPS, T>;
    static std::atomic<bool> attr_set[64];  // per device; a repeated set by a racing thread is harmless
    const int rc = allow_smem(attr_set, kernel, L::SMEM);
    if (rc != B200Q_OK) return rc;
    const int64_t at_once = L::PER_SM * (int64_t)sm_count();
    int64_t grid = most_tiles < at_once ? most_tiles : at_once;
    if (grid > kMaxCtas) grid = kMaxCtas;
    return launch_after("cache_attention_kernel", kernel, dim3((unsigned)grid), L::THREADS, L::SMEM, 1, stream, p);
}

// Rows of the query that share a key/value head, on average: up to 16 in 16-row items, two CTAs an SM; more in 32-row items, each code
// converted for twice as many products, one CTA of eight warps an SM (its sums need the registers).
template <typename T>
int launch_typed(const AttentionArgs &p, int dim, cudaStream_t stream) {
    const bool wide = dim <= 128 && p.tokens * p.group > 16 * (int64_t)p.batch;
    const int rows = wide ? 32 : 16, tile = wide ? 128 : 64;
    const int64_t tiles = p.kv_heads * (p.tokens * p.group / rows + p.batch) * (p.capacity / tile + 1);
    switch (dim) {
        case 64: return wide ? launch_sized<64, 2, 8, T>(p, tiles, stream) : launch_sized<64, 1, 4, T>(p, tiles, stream);
        case 96: return wide ? launch_sized<96, 2, 8, T>(p, tiles, stream) : launch_sized<96, 1, 4, T>(p, tiles, stream);
        case 128: return wide ? launch_sized<128, 2, 8, T>(p, tiles, stream) : launch_sized<128, 1, 4, T>(p, tiles, stream);
        case 192: return launch_sized<192, 1, 4, T>(p, tiles, stream);
        default: return launch_sized<256, 1, 4, T>(p, tiles, stream);
    }
}

}  // namespace
}  // namespace b200q

extern "C" {

B200Q_API size_t b200q_quantized_cache_attention_workspace_bytes(int64_t head_dim) {
    using namespace b200q;
    if (!cache_dim(head_dim)) return 0;
    const int64_t rows = head_dim <= 128 ? 32 : 16;
    return (size_t)(kCounterBytes + (int64_t)2 * kMaxCtas * rows * (head_dim + 2) * 4);
}

B200Q_API int b200q_quantized_cache_attention(const b200q_heads *q, void *out, float *lse, const void *cache, int64_t pages, int64_t page_size, const int32_t *page_table,
                                              int64_t table_width, int64_t table_stride, const int32_t *lengths, const int32_t *starts, const void *mask, int64_t mask_width,
                                              int64_t mask_stride, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, int type,
                                              void *workspace, size_t workspace_bytes, void *stream) {
    using namespace b200q;
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
    if (batch == 0 || tokens == 0) return B200Q_OK;
    if (starts == nullptr && tokens % batch != 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: %lld tokens of %lld sequences need starts", op, (long long)tokens, (long long)batch);
    if (batch > 1 << 20 || kv_heads > 65536 || tokens > (1ll << 31) / 4 / heads) return set_error(B200Q_UNSUPPORTED, "%s: %lld sequences, %lld tokens of %lld heads", op, (long long)batch, (long long)tokens, (long long)heads);
    if (q == nullptr || q->data == nullptr || out == nullptr || lengths == nullptr || (table_width > 0 && page_table == nullptr) || (pages > 0 && cache == nullptr)) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    }
    if (pages <= 0 && table_width > 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: a cache of %lld pages", op, (long long)pages);
    if (!aligned_to(cache, 16) || !aligned_to(q->data, 8) || !aligned_to(out, 8) || q->token_stride % 4 != 0 || q->head_stride % 4 != 0) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: a 16-byte aligned cache, 8-byte aligned q and out and strides of 4 elements are wanted", op);
    }
    const size_t need = b200q_quantized_cache_attention_workspace_bytes(head_dim);
    if (workspace == nullptr || workspace_bytes < need) return set_error(B200Q_WORKSPACE_TOO_SMALL, "%s: a workspace of %zu bytes is needed, got %zu", op, need, workspace_bytes);
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
    p.per_sequence = starts == nullptr ? (int)(tokens / batch) : 0;
    p.mask = static_cast<const uint8_t *>(mask);
    p.mask_stride = mask_stride;
    p.mask_width = (int)(mask_width < (1 << 30) ? mask_width : 1 << 30);
    p.batch = (int)batch;
    p.kv_heads = (int)kv_heads;
    p.group = (int)(heads / kv_heads);
    p.scale_log2 = scale * kLog2e;
    p.counters = static_cast<unsigned int *>(workspace);
    p.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kCounterBytes);
    p.status = device_status_word();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return type == B200Q_F16 ? launch_typed<__half>(p, (int)head_dim, s) : launch_typed<__nv_bfloat16>(p, (int)head_dim, s);
}

}  // extern "C"
