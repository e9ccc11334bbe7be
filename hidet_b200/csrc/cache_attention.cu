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
// The work is in tiles of positions for one (sequence, key/value head, 8 * NT query rows).  The tiles of all sequences stand in
// one line, with a gap in front of every item for what that costs besides where pieces are long, and the line is cut into equal pieces, one a CTA, whatever the sequences' lengths are (the host does not know them: they
// are on the device, so that a captured step can be replayed as they grow).  A CTA's piece may end one item and begin others; items in
// several pieces leave partial sums in the workspace, and the CTA that arrives last adds them in the order of the pieces.
//
// One warp copies whole records (codes and scales, one bulk copy per run of a page) into a ring of shared memory; each of
// the other warps takes one record of 16 positions of a tile: it loads K with plain and V with transposing matrix loads, converts two codes an
// instruction and multiplies, with the codes as the 16-row operand (positions of K, elements of V) and eight query rows as columns.  With the positions
// (and not the rows) shared out among the warps, each code is converted once per CTA.
#include <atomic>
#include <type_traits>

#include "serving.cuh"
#include "umma.cuh"

namespace b200q {
namespace {

constexpr unsigned int kKernelCacheAttention = 7;
constexpr int kMaxCtas = 3 * 148;         // of a launch; the workspace is made for them
constexpr int kCounterBytes = 65536 * 4;  // arrival counters in front of the workspace, zero between calls: kMaxCtas a level
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

// A key/value head of a sequence with some of its query rows, and the pieces that it is in.
struct Item {
    int head, row0, rows, token0;       // key/value head; first query row (token * group + head in group) and how many, -1: no more items; the sequence's first row of q
    int length, fresh;                  // cached positions; of them those of the new tokens
    int first_cta, last_cta, slot;      // who holds the pieces; the place of this CTA's
};
struct Tile {
    int key0;  // first position
    int last;  // of the item, in this CTA
};

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
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

constexpr int MOST_STAGES = 6;
constexpr int kItemUnits = 2;           // what an item costs besides its tiles, in tiles
constexpr int FAN = 8;                  // pieces of an item that are added at once
constexpr int WARPS = 4;                // that multiply
constexpr int CONSUMERS = 32 * WARPS;
constexpr int THREADS = CONSUMERS + 32;
constexpr int TILE = 16 * WARPS;        // positions

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
    static constexpr int ROOM = (PER_SM == 3 ? 75 : PER_SM == 2 ? 113 : 226) * 1024 - 3072 - FIXED;  // 3072: Control, and what an SM keeps for itself
    static constexpr int STAGES = ROOM / STAGE > MOST_STAGES ? MOST_STAGES : ROOM / STAGE;
    static constexpr int SMEM = FIXED + STAGES * STAGE;
    static constexpr bool Q_IN_REGISTERS = NT * D <= 128;
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

struct Sequence {
    int length, fresh, token0;
    int tiles;     // of one item
    int row_tiles; // items of a key/value head
};
template <int ROWS>
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
    s.row_tiles = (s.fresh * p.group + ROWS - 1) / ROWS;
    return s;
}

// The largest of the warps' maxima of a row.
__device__ __forceinline__ float row_top(const Control &ctl, int r) {
    float n = -INFINITY;
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
    float *part = p.partial + (int64_t)item.slot * ROWS * (D + 2);
    constexpr int VECS = ROWS * D / 4;
    auto write_out = [&](int r, int d, float4 v, float total_l, float top_log2) {
        const int row = item.row0 + r, token = row / p.group, head = item.head * p.group + row - token * p.group;
        const int64_t at = (int64_t)(item.token0 + token) * p.kv_heads * p.group + head;
        const float inv = total_l == 0.0f ? 0.0f : 1.0f / total_l;
        T y[4] = {Elems<T>::round(v.x * inv), Elems<T>::round(v.y * inv), Elems<T>::round(v.z * inv), Elems<T>::round(v.w * inv)};
        *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + at * D + d) = *reinterpret_cast<const uint2 *>(y);
        if (d == 0 && p.lse != nullptr) p.lse[at] = total_l == 0.0f ? -INFINITY : (top_log2 - kBias + __log2f(total_l)) * kLn2;
    };
    for (int i = threadIdx.x; i < VECS; i += CONSUMERS) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));
        if (r >= item.rows) break;
        const float top = row_top(ctl, r), scale = ctl.q_scale[r];
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
    // ---- the pieces of an item meet: FAN neighbours at a time, in the CTA that arrives last of them, then FAN of those ----
    if (!whole) {
        int k = blockIdx.x - item.first_cta, n = item.last_cta - item.first_cta + 1, stride = 1;
        auto part_of = [&](int i) { return p.partial + (int64_t)(2 * (item.first_cta + i) + (i == 0 ? 1 : 0)) * ROWS * (D + 2); };
        float (*part_m)[16] = reinterpret_cast<float (*)[16]>(merge), (*part_l)[16] = part_m + FAN;  // the merge buffers are free behind the next barrier
        static_assert(L::BUFFERS * L::MERGE >= 2 * FAN * 16 * 4, "");
        for (unsigned int *counters = p.counters;; counters += kMaxCtas, k /= FAN, n = (n + FAN - 1) / FAN, stride *= FAN) {
            const int first = k / FAN * FAN, some = min(FAN, n - first);
            // The last piece by itself is its own sum.  (It has no counter either: where it starts another item may have its first.)
            if (some == 1) continue;
            asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
            if (threadIdx.x == 0) {
                unsigned int *counter = counters + item.first_cta + first * stride;
                unsigned int before;  // releases what the barrier put in front, the stores of all threads of the CTA
                asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
                ctl.last = before == (unsigned int)(some - 1);
                if (ctl.last) *counter = 0;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
            if (!ctl.last) break;
            for (int i = threadIdx.x; i < some * ROWS; i += CONSUMERS) {
                const float *from = part_of((first + i / ROWS) * stride) + ROWS * D + i % ROWS;
                const bool there = i % ROWS < item.rows;
                part_m[i / ROWS][i % ROWS] = there ? __ldcg(from) : -INFINITY;
                part_l[i / ROWS][i % ROWS] = there ? __ldcg(from + ROWS) : 0.0f;
            }
            const bool done = n <= FAN;
            for (int i0 = 0; i0 < item.rows * (D / 4); i0 += CONSUMERS) {
                const int i = i0 + threadIdx.x, r = i / (D / 4), d = 4 * (i % (D / 4));
                float4 x[FAN];
#pragma unroll
                for (int j = 0; j < FAN; ++j)
                    if (j < some && r < item.rows) x[j] = __ldcg(reinterpret_cast<const float4 *>(part_of((first + j) * stride) + r * D + d));
                if (i0 == 0) asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
                if (r >= item.rows) continue;
                float top = -INFINITY, sum_l = 0.0f;
#pragma unroll
                for (int j = 0; j < FAN; ++j)
                    if (j < some) top = fmaxf(top, part_m[j][r]);
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < FAN; ++j)
                    if (j < some) {
                        const float by = part_m[j][r] == -INFINITY ? 1.0f : ex2(part_m[j][r] - top);
                        sum_l = fmaf(part_l[j][r], by, sum_l);
                        v.x = fmaf(x[j].x, by, v.x), v.y = fmaf(x[j].y, by, v.y), v.z = fmaf(x[j].z, by, v.z), v.w = fmaf(x[j].w, by, v.w);
                    }
                if (done) {
                    write_out(r, d, v, sum_l, top);
                } else {  // into the place of the first of them, whose statistics are in shared memory by now
                    float *to = part_of(first * stride);
                    __stcg(reinterpret_cast<float4 *>(to + r * D + d), v);
                    if (d == 0) {
                        __stcg(to + ROWS * D + r, top);
                        __stcg(to + ROWS * (D + 1) + r, sum_l);
                    }
                }
            }
            if (done) break;
        }
    }
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

        // ---- this CTA's piece of the line ----
        int items = 0, tiles = 0;
        for (int b = lane; b < p.batch; b += 32) {
            const Sequence s = sequence_of<ROWS>(p, b);
            items += s.row_tiles;
            tiles += s.row_tiles * s.tiles;
        }
#pragma unroll
        for (int d = 16; d > 0; d /= 2) {
            items += __shfl_xor_sync(0xffffffffu, items, d);
            tiles += __shfl_xor_sync(0xffffffffu, tiles, d);
        }
        items *= p.kv_heads;
        tiles *= p.kv_heads;
        // No more pieces of an item than are added at once, as long as the wait for another round of additions, about two tiles, would be longer
        // than what shorter pieces save.
        int ctas = min((int)gridDim.x, tiles);
        if (ctas > FAN * items && tiles / (FAN * max(1, items)) - tiles / ctas <= 2) ctas = FAN * items;
        // Where pieces are long, a gap in front of every item stands for what it costs besides its tiles.
        const int gap = tiles >= 8 * ctas ? kItemUnits : 0, units = tiles + items * gap;
        const int each = units / max(1, ctas), more = units - each * ctas;  // the first `more` pieces have one unit more
        auto piece = [&](int c) { return c * each + min(c, more); };
        auto cta_of = [&](int unit) { return unit < more * (each + 1) ? unit / (each + 1) : more + (unit - more * (each + 1)) / each; };
        int cur = 0, end = 0, b = 0, offset = 0;  // units; the sequence that cur lies in, and where in its items
        if ((int)blockIdx.x < ctas && items > 0) {
            cur = piece(blockIdx.x);
            end = piece(blockIdx.x + 1);
            for (int base = 0, b0 = 0;; b0 += 32) {
                int own = 0;
                if (b0 + lane < p.batch) {
                    const Sequence s = sequence_of<ROWS>(p, b0 + lane);
                    own = (s.tiles + gap) * s.row_tiles * p.kv_heads;
                }
                int until = own;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int below = __shfl_up_sync(0xffffffffu, until, d);
                    if (lane >= d) until += below;
                }
                const uint32_t behind = __ballot_sync(0xffffffffu, base + until > cur);
                if (behind != 0) {
                    const int l = __ffs(behind) - 1;
                    b = b0 + l;
                    offset = cur - base - __shfl_sync(0xffffffffu, until - own, l);
                    break;
                }
                base += __shfl_sync(0xffffffffu, until, 31);
            }
        }
        const int begin = cur, records_per_page = p.page_size >> 4;
        int slot = 0, it = 0;
        uint32_t parity = 0;
        while (cur < end && !dead) {
            const Sequence s = sequence_of<ROWS>(p, b);
            const int per = s.tiles + gap;
            if (s.row_tiles == 0) {
                ++b;
                continue;
            }
            const int index = offset / per, head = index / s.row_tiles, rt = index - head * s.row_tiles;
            const int item_begin = cur - (offset - index * per), tiles_begin = item_begin + gap, item_end = item_begin + per;
            const int to = min(end, item_end), tile0 = max(cur, tiles_begin) - tiles_begin, n = to - tiles_begin - tile0;
            const int32_t *pages = p.table + (int64_t)b * p.table_stride;
            offset += to - cur;
            cur = to;
            if (offset == per * s.row_tiles * p.kv_heads) ++b, offset = 0;
            if (n <= 0) continue;  // its tiles are another CTA's
            // lane i brings the i-th page that the tile touches; its number is asked for one tile ahead
            auto page_of = [&](int tile) {
                const int page = tile * TILE / p.page_size + lane;
                return tile < tile0 + n && lane <= WARPS && (int64_t)page * p.page_size < s.length ? pages[page] : 0;
            };
            int page = page_of(tile0);
            publish({head, rt * ROWS, min(ROWS, s.fresh * p.group - rt * ROWS), s.token0, s.length, s.fresh, cta_of(tiles_begin), cta_of(item_end - 1),
                     2 * (int)blockIdx.x + (tiles_begin >= begin ? 1 : 0)});
            for (int i = 0; i < n && !dead; ++i) {
                const int tile = tile0 + i, key0 = tile * TILE;
                const int next = page_of(tile + 1);
                if (it >= STAGES) wait_for(ctl.empty[slot], parity ^ 1u);
                if (dead) break;
                const int keys = min(TILE, (s.length - key0 + 15) & ~15);  // 0 where the sequence is empty
                const uint32_t bar = smem_u32(&ctl.full[slot]);
                if (lane == 0) {
                    ctl.tiles[slot] = {key0, i == n - 1};
                    if (keys > 0) mbar_expect_tx(bar, (uint32_t)(keys >> 4) * L::RECORD);
                    else mbar_arrive(bar);
                }
                __syncwarp();
                const int at = (key0 / p.page_size + lane) * p.page_size;  // first position of this lane's page
                const int from = max(at, key0), until = min(at + p.page_size, key0 + keys);
                if (lane <= WARPS && from < until) {
                    if (page < 0 || page >= p.pages) {
                        page = 0;
                        if (p.status != nullptr) atomicOr(p.status, kBadPage);
                    }
                    const uint8_t *src = p.cache + (((int64_t)page * p.kv_heads + head) * records_per_page + ((from - at) >> 4)) * L::RECORD;
                    bulk_load(stages + slot * L::STAGE + ((from - key0) >> 4) * L::RECORD, src, (uint32_t)((until - from) >> 4) * L::RECORD, bar);
                }
                page = next;
                ++it;
                if (++slot == STAGES) slot = 0, parity ^= 1u;
            }
        }
        if (!dead) publish({0, 0, -1, 0, 0, 0, 0, 0, 0});
        if (dead) {  // nothing may be on its way when the CTA ends
            for (int back = 1; back <= STAGES && back <= it; ++back) {
                const int at = it - back;
                mbar_wait(smem_u32(&ctl.full[at % STAGES]), (at / STAGES) & 1, 1u << 16);
            }
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
        const int length = item.length, fresh = item.fresh;
        float o[NT][D / 16][4];  // elements 16 i + g (0, 1) and + 8 (2, 3) of query rows 2t (0, 2) and 2t + 1 (1, 3)
        float m[NT][2], l[NT][2], shift[NT][2], qs[NT][2], rise[NT][2];  // shift: m, or 0 as long as nothing was seen
        float vref = 0.0f, v_inv = 0.0f, v_limit = kLeastNormal;  // a power of two, its reciprocal, and the first scale that is too large for it
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
                const int row = item.row0 + r, token = row / p.group;
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
                    const uint32_t e = min(max(__float_as_uint(top) >> 23, 64u), 253u);
                    if (top > 0.0f) down = __uint_as_float((254u - e) << 23), up = __uint_as_float(e << 23);
                }
                if (lane == 0) ctl.q_scale[r] = up * p.scale_log2;
#pragma unroll
                for (int j = 0; j < (D + 127) / 128; ++j) {
                    const int d = 4 * lane + 128 * j;
                    if (d < D) {
                        const uint32_t at = (((r >> 3) * (D / 16) + (d >> 4)) * 32 + ((r & 7) << 2) + ((d >> 2) & 3)) * 8;
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(q_frag + at), "r"(pack_f16(f[j][0] * down, f[j][1] * down)), "r"(pack_f16(f[j][2] * down, f[j][3] * down)) : "memory");
                    }
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int n = 0; n < D / 16; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][n][e] = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    m[nt][h] = -INFINITY;
                    l[nt][h] = shift[nt][h] = 0.0f;
                    qs[nt][h] = ctl.q_scale[8 * nt + 2 * t + h];
                    rise[nt][h] = fminf(kRise / qs[nt][h], 1e38f);
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
                const int old = length - fresh;  // positions in front of the new tokens
                const bool partly = key0 + 16 > (p.mask != nullptr ? old : min(old + 1, length));
                if (partly) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int pos = key0 + key_of_lane + 2 * h, drafted = pos - old;
                        if (pos >= length) vs[h] = 0.0f;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int r = 8 * nt + 2 * t + e, token = (item.row0 + r) / p.group;
                                bool seen = pos < length && r < item.rows;
                                if (seen && drafted >= 0) {
                                    seen = p.mask == nullptr ? drafted <= token : drafted < p.mask_width && p.mask[(int64_t)(item.token0 + token) * p.mask_stride + drafted] != 0;
                                }
                                if (!seen) s[nt][2 * h + e] = -INFINITY;
                            }
                    }
                }
                const float v_top = fmaxf(vs[0], vs[1]);
                bool up = v_top >= v_limit;
                float top[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        top[nt][h] = fmaxf(s[nt][h], s[nt][2 + h]);
                        up |= top[nt][h] > m[nt][h] + rise[nt][h];
                    }
                if (__any_sync(0xffffffffu, up)) {
                    float v_new = v_top;
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) v_new = fmaxf(v_new, __shfl_xor_sync(0xffffffffu, v_new, d));
                    v_new = fmaxf(v_new, vref);
                    const uint32_t power = __float_as_uint(v_new) & 0x7f800000u;
                    const float beta = power != 0 ? vref * __uint_as_float(0x7f000000u - power) : 1.0f;
                    vref = __uint_as_float(power);
                    v_inv = power != 0 ? __uint_as_float(0x7f000000u - power) : 0.0f;
                    v_limit = power != 0 ? 2.0f * vref : kLeastNormal;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float by[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float n = top[nt][h];
#pragma unroll
                            for (int d = 4; d < 32; d *= 2) n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, d));
                            n = fmaxf(n, m[nt][h]);
                            const float alpha = n == -INFINITY ? 1.0f : ex2((m[nt][h] - n) * qs[nt][h]);
                            m[nt][h] = n;
                            shift[nt][h] = n == -INFINITY ? 0.0f : n;
                            l[nt][h] *= alpha;
                            by[h] = alpha * beta;
                        }
#pragma unroll
                        for (int n = 0; n < D / 16; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[nt][n][e] *= by[e & 1];
                    }
                }
                const float w[2] = {vs[0] * v_inv, vs[1] * v_inv};
                uint32_t b[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = ex2(fmaf(s[nt][e] - shift[nt][e & 1], qs[nt][e & 1], kBias));
                        l[nt][e & 1] += x[e];
                        x[e] *= w[e >> 1];
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
            for (int h = 0; h < 2; ++h) factor[nt][h] = m[nt][h] == -INFINITY ? vref : ex2((m[nt][h] - row_top(ctl, 8 * nt + 2 * t + h)) * qs[nt][h]) * vref;
        float *mine = merge + (warp % L::BUFFERS) * (L::MERGE / 4) + 2 * t * L::PITCH + g;
        if (warp >= L::BUFFERS) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int n = 0; n < D / 16; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mine[(8 * nt + (e & 1)) * L::PITCH + 16 * n + 8 * (e >> 1)] = o[nt][n][e] * factor[nt][e & 1];
        }
        asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
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
        asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
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
    const int64_t tiles = p.kv_heads * (p.tokens * p.group / L::ROWS + p.batch) * (p.capacity / TILE + 1), at_once = L::PER_SM * (int64_t)sm_count();
    if (tiles > (1ll << 29)) return set_error(B200Q_UNSUPPORTED, "quantized_cache_attention: up to %lld tiles of %d rows and %d positions", (long long)tiles, L::ROWS, TILE);
    int64_t grid = tiles < at_once ? tiles : at_once;
    if (grid > kMaxCtas) grid = kMaxCtas;
    return launch_after("cache_attention_kernel", kernel, dim3((unsigned)grid), THREADS, L::SMEM, 1, stream, p);
}

// Rows of the query that share a key/value head, on average: up to 8 in 8-row items, more in 16-row items.
template <typename T>
int launch_typed(const AttentionArgs &p, int dim, cudaStream_t stream) {
    const bool wide = p.tokens * p.group > 8 * (int64_t)p.batch;
    switch (dim) {
        case 64: return wide ? launch_sized<64, 2, T>(p, stream) : launch_sized<64, 1, T>(p, stream);
        case 96: return wide ? launch_sized<96, 2, T>(p, stream) : launch_sized<96, 1, T>(p, stream);
        case 128: return wide ? launch_sized<128, 2, T>(p, stream) : launch_sized<128, 1, T>(p, stream);
        case 192: return wide ? launch_sized<192, 2, T>(p, stream) : launch_sized<192, 1, T>(p, stream);
        default: return wide ? launch_sized<256, 2, T>(p, stream) : launch_sized<256, 1, T>(p, stream);
    }
}

}  // namespace
}  // namespace b200q

extern "C" {

B200Q_API size_t b200q_quantized_cache_attention_workspace_bytes(int64_t head_dim) {
    using namespace b200q;
    if (!cache_dim(head_dim)) return 0;
    return (size_t)(kCounterBytes + (int64_t)2 * kMaxCtas * 16 * (head_dim + 2) * 4);
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
