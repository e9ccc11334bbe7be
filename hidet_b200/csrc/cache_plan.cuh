// The plan of attention over the quantized cache: the line of tiles of all sequences, and the piece of it that a CTA takes.
//
// No header of CUDA's is included, so that the plan runs on the host as well (tests/host/cache_plan.cpp, which brings the names that nvcc knows by itself).
#pragma once

#include <stdint.h>

#include "status_bits.h"

namespace b200q {
namespace cache_attention {

constexpr int TILE = 64;  // positions

struct PlanArgs {
    const int32_t *table;
    int64_t table_stride;
    int64_t capacity;  // positions that a row of the table covers
    const int32_t *lengths, *starts;
    int64_t tokens;    // all rows of q
    int per_sequence;  // tokens of every sequence where starts is null
    int batch, kv_heads, group;
    unsigned int *status;
};

// A key/value head of a sequence with some of its query rows, and the pieces that it is in.
struct Item {
    int head, row0, rows, token0;   // key/value head; first query row (token * group + head in group) and how many, -1: no more items; the sequence's first row of q
    int length, fresh;              // cached positions; of them those of the new tokens
    int first_cta, last_cta, slot;  // who holds the pieces; the place of this CTA's
    int tile0, tiles;               // of this piece
};

struct Sequence {
    int length, fresh, token0;
    bool placed;    // its rows lie inside, and do not end in front of where they begin
    int tiles;      // of one item
    int row_tiles;  // items of a key/value head
};
template <int ROWS>
__device__ __forceinline__ Sequence sequence_of(const PlanArgs &p, int b) {
    Sequence s;
    int64_t n = p.lengths[b];
    if (n > p.capacity) {
        n = p.capacity;
        if (p.status != nullptr) atomicOr(p.status, kBadPage);
    }
    s.length = n < 0 ? 0 : (int)n;
    if (p.starts != nullptr) {
        const int first = p.starts[b], end = p.starts[b + 1];
        s.placed = first >= 0 && end >= first && end <= p.tokens;
        s.token0 = s.placed ? first : 0;
        s.fresh = s.placed ? end - first : 0;
    } else {
        s.placed = true;
        s.token0 = b * p.per_sequence;
        s.fresh = p.per_sequence;
    }
    s.tiles = max(1, (s.length + TILE - 1) / TILE);  // an empty sequence has a tile too: its rows are written
    s.row_tiles = (s.fresh * p.group + ROWS - 1) / ROWS;
    return s;
}

// This CTA's piece of the line of tiles: a sequence's items one behind the other, head by head, and the sequences behind one another.  One warp.
template <int ROWS, int ROUND, int UNITS>  // ROUND: pieces of an item that are added at once; UNITS: what an item costs besides its tiles, in tiles
struct Line {
    const PlanArgs &p;
    const int lane;
    int each = 0, more = 0, gap = 0;            // units of a piece; the first `more` pieces have one more; units in front of an item's tiles
    int begin = 0, cur = 0, end = 0;            // units
    int b = 0, offset = 0;                      // the sequence that cur lies in, and where in its items
    bool placed = true;                         // all sequences are: no row is in two of them, so that the tiles of all are as few as the host allows

    __device__ __forceinline__ int piece(int c) const { return c * each + min(c, more); }
    __device__ __forceinline__ int cta_of(int unit) const {
        const int longer = more * (each + 1);
        return unit < longer ? (int)((uint32_t)unit / (uint32_t)(each + 1)) : more + (int)((uint32_t)(unit - longer) / (uint32_t)each);
    }

    __device__ __forceinline__ Line(const PlanArgs &args, int lane_) : p(args), lane(lane_) {
        // The plan is in front of everything else, alone: few sums and divisions, and no sequence looked up twice that need not be.
        Sequence mine = {};
        if (lane < p.batch) mine = sequence_of<ROWS>(p, lane), placed = mine.placed;
        int items = mine.row_tiles, tiles = mine.row_tiles * mine.tiles;
        for (int s0 = lane + 32; s0 < p.batch; s0 += 32) {
            const Sequence s = sequence_of<ROWS>(p, s0);
            items += s.row_tiles;
            tiles += s.row_tiles * s.tiles;
            placed &= s.placed;
        }
        if (p.starts != nullptr && !__all_sync(0xffffffffu, placed)) {  // then these are sums of anything, beyond 32 bits too
            placed = false;
            if (lane == 0 && p.status != nullptr) atomicOr(p.status, kBadStarts);
            return;
        }
        items = __reduce_add_sync(0xffffffffu, items) * p.kv_heads;
        tiles = __reduce_add_sync(0xffffffffu, tiles) * p.kv_heads;
        // No more pieces of an item than are added at once, as long as the wait for another round of additions, about two tiles, would be longer
        // than what shorter pieces save.
        int ctas = min((int)gridDim.x, tiles);
        if (ctas > ROUND * items && tiles / (ROUND * max(1, items)) - tiles / ctas <= 2) ctas = ROUND * items;
        if ((int)blockIdx.x >= ctas) return;
        // Where pieces are long, a gap in front of every item stands for what it costs besides its tiles.
        gap = tiles >= 8 * ctas ? UNITS : 0;
        const int units = tiles + items * gap;
        each = (int)((uint32_t)units / (uint32_t)ctas);
        more = units - each * ctas;
        begin = cur = piece(blockIdx.x);
        end = piece(blockIdx.x + 1);
        for (int base = 0, b0 = 0; b0 < p.batch; b0 += 32) {
            if (b0 > 0) mine = b0 + lane < p.batch ? sequence_of<ROWS>(p, b0 + lane) : Sequence{};
            const int own = (mine.tiles + gap) * mine.row_tiles * p.kv_heads;
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
                return;
            }
            base += __shfl_sync(0xffffffffu, until, 31);
        }
        end = cur;  // lengths that have become less since they were counted
    }

    // The next item with tiles in this piece, and its sequence's pages; false behind the last.
    __device__ __forceinline__ bool next(Item &item, const int32_t *&pages) {
        while (cur < end && b < p.batch) {
            const Sequence s = sequence_of<ROWS>(p, b);
            if (s.row_tiles == 0) {
                ++b;
                continue;
            }
            const int per = s.tiles + gap, index = (int)((uint32_t)offset / (uint32_t)per);
            const int item_begin = cur - (offset - index * per), tiles_begin = item_begin + gap, item_end = item_begin + per, to = min(end, item_end);
            item.head = s.row_tiles == 1 ? index : (int)((uint32_t)index / (uint32_t)s.row_tiles);
            item.row0 = (index - item.head * s.row_tiles) * ROWS;
            item.rows = min(ROWS, s.fresh * p.group - item.row0);
            item.token0 = s.token0;
            item.length = s.length;
            item.fresh = s.fresh;
            item.first_cta = tiles_begin >= begin ? blockIdx.x : cta_of(tiles_begin);
            item.last_cta = item_end <= end ? blockIdx.x : cta_of(item_end - 1);
            item.slot = 2 * (int)blockIdx.x + (tiles_begin >= begin ? 1 : 0);  // only its first piece can begin in this CTA, and only the first item here have begun before
            item.tile0 = max(cur, tiles_begin) - tiles_begin;
            item.tiles = to - tiles_begin - item.tile0;
            pages = p.table + (int64_t)b * p.table_stride;
            offset += to - cur;
            cur = to;
            if (offset == per * s.row_tiles * p.kv_heads) ++b, offset = 0;
            if (item.tiles > 0) return true;  // else they are another CTA's
        }
        item.rows = -1;
        return false;
    }
};

}  // namespace cache_attention
}  // namespace b200q
