// What the two kernels of attention over the quantized cache share: their arguments, the copies of a tile's records, and the sum of an item's
// pieces.  (cache_plan.cuh: the line of tiles and its pieces.)
#pragma once

#include <type_traits>

#include "cache_plan.cuh"
#include "serving.cuh"
#include "umma.cuh"

namespace b200q {
namespace cache_attention {

constexpr int kMaxCtas = 3 * 148;         // of a launch; the workspace is made for them
constexpr int kMostWideCtas = 148;        // of the kernel for many rows
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are kept 2^6 times as large, and a row's maximum is raised when a score passes it by 2^8 (rarely, behind its first
// positions): with a value's scale below 2 that is at most 2^15 of f16's 2^16, and a probability of 2^-31 is still there, so that a long tail of
// small ones is not lost.
constexpr float kBias = 6.0f, kRise = 8.0f;
constexpr float kLeastNormal = 1.1754943508222875e-38f;

constexpr int RECORDS = 4;     // of a tile
constexpr int FAN = 8;         // pieces of an item that are added at once
// Three rounds of additions, each with a counter for every CTA in the workspace's head.
static_assert(FAN * FAN * FAN >= kMaxCtas && 3 * kMaxCtas <= kWorkspaceCounters, "");

struct AttentionArgs : PlanArgs {
    const void *q;
    int64_t q_token, q_head;
    void *out;
    float *lse;
    const uint8_t *cache;
    int64_t pages;
    int page_size;
    const uint8_t *mask;
    int64_t mask_stride;
    int mask_width;
    Divisor by_group;
    float scale_log2;
    float *partial;
    int64_t partial_floats;  // of all pieces of the kernel for many rows
    unsigned int *counters;
};

// At most this many tiles of `rows` query rows.
inline int64_t most_tiles(const AttentionArgs &p, int rows) { return p.kv_heads * (p.tokens * p.group / rows + p.batch) * (p.capacity / TILE + 1); }
// The kernel for many rows (cache_attention_wide.cu) takes heads of 64 and 128 elements; its workspace is asked for from 17 query rows a key/value head on.
inline bool may_be_wide(int64_t tokens, int64_t group, int64_t batch, int64_t dim) { return (dim == 64 || dim == 128) && tokens * group > 16 * batch; }
// Tiles of 64 positions and 16 rows, by what the page table could hold.
inline int64_t tiles_of_16(const AttentionArgs &p) { return p.batch * (int64_t)p.kv_heads * (p.capacity / TILE + 1) * ((p.tokens * p.group / p.batch + 15) / 16); }  // batch > 0
// It takes the calls with more than 4200 of them; its fixed costs are 6 us higher.  Measured
// (few / many rows, us) with 8 key/value heads of 128 elements, pages of 64: 1 sequence of 4096 positions, 96 rows (3120 tiles) 24.2 / 40.1; 4 of 4096, 32 rows (4160) 28.9 / 33.3;
// 16 of 600, 48 rows (4224) 31.0 / 27.3; 16 of 300, 96 rows (4608) 34.9 / 24.6; 4 of 4096, 64 rows (8320) 47.4 / 34.1; 8 of 8000, 48 rows (24192) 107 / 76.5.  It is wrong for
// some calls of few rows: 8 of 4096, 24 rows (8320) 39.0 / 46.0.
inline bool is_wide(const AttentionArgs &p, int64_t dim) { return p.batch > 0 && may_be_wide(p.tokens, p.group, p.batch, dim) && tiles_of_16(p) > 4200; }
int launch_wide(const AttentionArgs &p, int dim, bool bf16, cudaStream_t stream);

#ifdef __CUDACC__

// Of a query row, token * group + head in group.
__device__ __forceinline__ int token_of(const AttentionArgs &p, int row) { return (int)quotient((uint32_t)row, p.by_group); }

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
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
template <int N>
__device__ __forceinline__ void sync_of() {
    asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}
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

// The pages of an item's tiles: lane i < 5 has the number of the i-th page that a tile touches, asked for one tile ahead.
struct Pages {
    const int32_t *pages;
    int end, page;  // behind the item's last tile here; of the next tile
    __device__ __forceinline__ int of(const AttentionArgs &p, const Item &item, int lane, int tile) const {
        const int i = tile * TILE / p.page_size + lane;
        return tile < end && lane <= RECORDS && (int64_t)i * p.page_size < item.length ? pages[i] : 0;
    }
    __device__ __forceinline__ Pages(const AttentionArgs &p, const Item &item, int lane, const int32_t *table) : pages(table), end(item.tile0 + item.tiles) { page = of(p, item, lane, item.tile0); }
};
// Positions of a tile that are copied, whole records; 0 where the sequence is empty.
__device__ __forceinline__ int copied_keys(const Item &item, int key0) { return min(TILE, (item.length - key0 + 15) & ~15); }
// Brings a tile's records, one bulk copy for each page.
template <int D>
__device__ __forceinline__ void copy_tile(const AttentionArgs &p, const Item &item, Pages &pages, int lane, int key0, uint32_t dst, uint32_t bar) {
    int page = pages.page;
    pages.page = pages.of(p, item, lane, key0 / TILE + 1);
    const int at = (key0 / p.page_size + lane) * p.page_size;  // first position of this lane's page
    const int from = max(at, key0), until = min(at + p.page_size, key0 + copied_keys(item, key0));
    if (lane <= RECORDS && from < until) {
        if (page < 0 || page >= p.pages) {
            page = 0;
            if (p.status != nullptr) atomicOr(p.status, kBadPage);
        }
        const uint8_t *src = p.cache + (((int64_t)page * p.kv_heads + item.head) * (p.page_size >> 4) + ((from - at) >> 4)) * record_bytes(D);
        bulk_load(dst + ((from - key0) >> 4) * record_bytes(D), src, (uint32_t)((until - from) >> 4) * record_bytes(D), bar);
    }
}

// Whether query row r of the item may see a position.  (Without a return in between: several of these have their loads on their way together.)
__device__ __forceinline__ bool may_see(const AttentionArgs &p, const Item &item, int r, int token, int pos) {
    const int drafted = pos - (item.length - item.fresh);
    const bool there = pos < item.length && r < item.rows;
    uint8_t seen = drafted < 0 || (p.mask == nullptr && drafted <= token);
    if (there && drafted >= 0 && drafted < p.mask_width) seen = p.mask[(int64_t)(item.token0 + token) * p.mask_stride + drafted];
    return there && seen != 0;
}
// The same for the 64 positions from key0 on, as bits.
__device__ __forceinline__ uint64_t seen_of_64(const AttentionArgs &p, const Item &item, int r, int token, int key0) {
    if (r >= item.rows) return 0;
    const int old = item.length - item.fresh;
    const int sure = p.mask == nullptr ? min(item.length, old + token + 1) - key0 : old - key0;  // positions in front of this one
    uint64_t seen = sure >= 64 ? ~0ull : sure > 0 ? (1ull << sure) - 1 : 0;
    if (p.mask != nullptr) {
        const uint8_t *row = p.mask + (int64_t)(item.token0 + token) * p.mask_stride + (key0 - old);
        const int from = old - key0, until = from + min(item.fresh, p.mask_width);
#pragma unroll 1
        for (int h = 0; h < 64; h += 32) {
            uint32_t bits = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j)  // all loads on their way together
                if (h + j >= from && h + j < until && row[h + j] != 0) bits |= 1u << j;
            seen |= (uint64_t)bits << h;
        }
    }
    return seen;
}
// Positions from here on may be hidden from a row.
__device__ __forceinline__ int first_hidden(const AttentionArgs &p, const Item &item) {
    const int old = item.length - item.fresh;
    return p.mask != nullptr ? old : min(old + 1, item.length);
}

__device__ __forceinline__ void write_lse(const AttentionArgs &p, int64_t at, float sum, float top) {
    if (p.lse != nullptr) p.lse[at] = sum == 0.0f ? -INFINITY : (top - kBias + __log2f(sum)) * kLn2;
}
// Zeros, and -inf for their softmax's denominators, in the place of the results of rows of q that no sequence has: those in front of the first one's and behind the
// last one's (a captured step has a fixed number of rows, often with fewer in use); all where the sequences' rows are not `placed`.  One warp of every
// CTA, with nothing waiting for it.
template <int D>
__device__ __forceinline__ void write_unowned(const AttentionArgs &p, bool placed, int lane) {
    if (p.starts == nullptr && p.batch > 0) return;  // tokens / batch each: all rows
    const bool any = p.batch > 0 && placed;
    const int64_t from = any ? min(max((int64_t)p.starts[0], (int64_t)0), p.tokens) : 0, to = any ? min(max((int64_t)p.starts[p.batch], from), p.tokens) : 0;
    const int heads = p.kv_heads * p.group;
    for (int64_t i = blockIdx.x; i < p.tokens - (to - from); i += gridDim.x) {
        const int64_t row = (i < from ? i : i + (to - from)) * heads;
        uint4 *out = reinterpret_cast<uint4 *>(p.out) + row * (D / 8);
        for (int j = lane; j < heads * (D / 8); j += 32) out[j] = make_uint4(0, 0, 0, 0);
        if (p.lse != nullptr)
            for (int j = lane; j < heads; j += 32) p.lse[row + j] = -INFINITY;
    }
}
// Four elements of a query row's result, from the sum of its values and of its probabilities, both in units of 2^top.
template <int D, typename T>
__device__ __forceinline__ void write_out(const AttentionArgs &p, const Item &item, int r, int d, float4 v, float sum, float top) {
    const int row = item.row0 + r, token = token_of(p, row), head = item.head * p.group + row - token * p.group;
    const int64_t at = (int64_t)(item.token0 + token) * p.kv_heads * p.group + head;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T y[4] = {Elems<T>::round(v.x * inv), Elems<T>::round(v.y * inv), Elems<T>::round(v.z * inv), Elems<T>::round(v.w * inv)};
    *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + at * D + d) = *reinterpret_cast<const uint2 *>(y);
    if (d == 0) write_lse(p, at, sum, top);
}

// A piece in the workspace: [ROWS][D] sums of values, then the rows' units (log2) and sums of probabilities.
template <int D, int ROWS>
constexpr int kPieceFloats = ROWS * (D + 2);
template <int D, int ROWS>
__device__ __forceinline__ void write_piece(float *piece, int r, int d, float4 v, float sum, float top) {
    __stcg(reinterpret_cast<float4 *>(piece + r * D + d), v);
    if (d == 0) {
        __stcg(piece + ROWS * D + r, top);
        __stcg(piece + ROWS * (D + 1) + r, sum);
    }
}

// The sum of `some` pieces, four elements of a row a thread at a time.  tops, sums: of the pieces' rows, [FAN][ROWS], filled by all threads in front of
// the barrier behind the first loads.
template <int D, int ROWS, int N, typename T, typename PieceOf>
__device__ __forceinline__ void add_pieces(const AttentionArgs &p, const Item &item, const float *tops, const float *sums, int tid, int some, bool done, PieceOf piece_of) {
    bool waited = false;
    for (int i = tid; i < item.rows * (D / 4) || !waited; i += N) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));
        float4 x[FAN];
#pragma unroll
        for (int j = 0; j < FAN; ++j)
            if (j < some && r < item.rows) x[j] = __ldcg(reinterpret_cast<const float4 *>(p.partial + (piece_of(j) + r * D + d)));
        if (!waited) sync_of<N>();
        waited = true;
        if (r >= item.rows) continue;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int j = 0; j < FAN; ++j)
            if (j < some) top = fmaxf(top, tops[j * ROWS + r]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < FAN; ++j)
            if (j < some) {
                // in two steps: units may lie so far apart that the whole factor leaves float's range where the products do not
                const float own = tops[j * ROWS + r], by = own == -INFINITY ? 1.0f : ex2(0.5f * (own - top));
                sum = fmaf(sums[j * ROWS + r] * by, by, sum);
                v.x = fmaf(x[j].x * by, by, v.x), v.y = fmaf(x[j].y * by, by, v.y), v.z = fmaf(x[j].z * by, by, v.z), v.w = fmaf(x[j].w * by, by, v.w);
            }
        if (done) write_out<D, T>(p, item, r, d, v, sum, top);
        else write_piece<D, ROWS>(p.partial + piece_of(0), r, d, v, sum, top);  // into the place of the first of them, whose rows' units and sums are in shared memory by now
    }
}

// The pieces of an item meet: FAN neighbours at a time, in the CTA that arrives last of them, then FAN of those.  N threads, which have written this
// CTA's piece; scratch: 2 * FAN * ROWS floats.
template <int D, int ROWS, int N, typename T>
__device__ __forceinline__ void meet(const AttentionArgs &p, const Item &item, int tid, float *scratch, int *last) {
    int k = blockIdx.x - item.first_cta, n = item.last_cta - item.first_cta + 1, stride = 1;
    auto place = [&](int i) { return (2 * (item.first_cta + i) + (i == 0 ? 1 : 0)) * kPieceFloats<D, ROWS>; };  // 32 bits are enough for the workspace
    float *tops = scratch, *sums = scratch + FAN * ROWS;
    for (unsigned int *counters = p.counters;; counters += kMaxCtas, k /= FAN, n = (n + FAN - 1) / FAN, stride *= FAN) {
        const int first = k / FAN * FAN, some = min(FAN, n - first);
        // The last piece by itself is its own sum.  (It has no counter either: where it starts another item may have its first.)
        if (some == 1) continue;
        sync_of<N>();
        if (tid == 0) {
            unsigned int *counter = counters + item.first_cta + first * stride;
            unsigned int before;  // releases what the barrier put in front, the stores of all threads of the CTA
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
            *last = before == (unsigned int)(some - 1);
            if (*last) *counter = 0;
        }
        sync_of<N>();
        if (!*last) break;
        auto piece_of = [&](int j) { return place((first + j) * stride); };
        for (int i = tid; i < some * ROWS; i += N) {
            const int j = i / ROWS, r = i % ROWS;
            const float *from = p.partial + piece_of(j) + ROWS * D + r;
            tops[i] = r < item.rows ? __ldcg(from) : -INFINITY;
            sums[i] = r < item.rows ? __ldcg(from + ROWS) : 0.0f;
        }
        const bool done = n <= FAN;
        add_pieces<D, ROWS, N, T>(p, item, tops, sums, tid, some, done, piece_of);
        if (done) break;
    }
}

#endif  // __CUDACC__

}  // namespace cache_attention
}  // namespace b200q
