// hidet_b200/csrc/cache_plan.cuh on the host: the pieces of a line of tiles, for every CTA of a grid.  A warp is 32 contexts that take turns at its
// collective operations.  What a call puts on the device ends where a page that cannot be read begins.
//
// Reads: rows grid batch kv_heads group tokens capacity per_sequence with_starts, the starts, the lengths.  Writes a line for each piece, then the status word.
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <sys/mman.h>
#include <ucontext.h>
#include <unistd.h>

#include <algorithm>

#define __device__
#define __forceinline__ inline
using std::max;
using std::min;

struct Dim {
    unsigned x;
} blockIdx, gridDim;

namespace {

constexpr int LANES = 32;
ucontext_t main_context, contexts[LANES];
char stacks[LANES][1 << 16];
int current, turns[LANES];
uint32_t brought[2][LANES];  // of a collective operation and the one behind it
bool over[LANES];

// Brings this lane's word and waits for the others'.
uint32_t *meet(uint32_t word) {
    uint32_t *all = brought[turns[current]++ & 1];
    all[current] = word;
    swapcontext(&contexts[current], &main_context);
    return all;
}

}  // namespace

int __reduce_add_sync(unsigned, int x) {
    const uint32_t *all = meet((uint32_t)x);
    uint32_t sum = 0;
    for (int i = 0; i < LANES; ++i) sum += all[i];
    return (int)sum;
}
int __shfl_sync(unsigned, int x, int lane) { return (int)meet((uint32_t)x)[lane]; }
int __shfl_up_sync(unsigned, int x, int d) {
    const int own = current;
    const uint32_t *all = meet((uint32_t)x);
    return (int)all[own >= d ? own - d : own];
}
uint32_t __ballot_sync(unsigned, bool x) {
    const uint32_t *all = meet(x);
    uint32_t bits = 0;
    for (int i = 0; i < LANES; ++i) bits |= all[i] << i;
    return bits;
}
bool __all_sync(unsigned mask, bool x) { return __ballot_sync(mask, x) == 0xffffffffu; }
int __ffs(uint32_t x) { return __builtin_ffs((int)x); }
void atomicOr(unsigned int *p, unsigned int x) { *p |= x; }

#include "../../hidet_b200/csrc/cache_plan.cuh"

using namespace b200q::cache_attention;

namespace {

PlanArgs args;
int rows;

template <int ROWS, int ROUND, int UNITS>
void pieces(int lane) {
    Line<ROWS, ROUND, UNITS> line(args, lane);
    Item item;
    const int32_t *pages;
    for (int n = 0; line.next(item, pages); ++n) {
        if (lane == 0)
            printf("%u %lld %d %d %d %d %d %d %d %d %d %d %d\n", blockIdx.x, (long long)(pages - args.table), item.head, item.row0, item.rows, item.token0, item.length, item.fresh,
                   item.first_cta, item.last_cta, item.slot, item.tile0, item.tiles);
        if (n > 1000000) exit(3);
    }
}

void lane_of_warp(int lane) {
    rows == 8 ? pieces<8, 8, 2>(lane) : rows == 16 ? pieces<16, 8, 2>(lane) : pieces<128, 4, 8>(lane);  // as the kernels have them
    over[lane] = true;
}

int32_t *guarded(long n) {
    const long page = sysconf(_SC_PAGESIZE), bytes = (n * 4 + page - 1) / page * page;
    char *p = (char *)mmap(nullptr, bytes + page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    if (p == (char *)MAP_FAILED || mprotect(p + bytes, page, PROT_NONE) != 0) exit(2);
    int32_t *x = (int32_t *)(p + bytes) - n;
    for (long i = 0; i < n; ++i)
        if (scanf("%d", &x[i]) != 1) exit(2);
    return x;
}

}  // namespace

int main() {
    long long tokens, capacity;
    int with_starts;
    static unsigned int status;
    if (scanf("%d %u %d %d %d %lld %lld %d %d", &rows, &gridDim.x, &args.batch, &args.kv_heads, &args.group, &tokens, &capacity, &args.per_sequence, &with_starts) != 9) return 2;
    args.tokens = tokens, args.capacity = capacity, args.status = &status, args.table_stride = 1;
    args.starts = with_starts ? guarded(args.batch + 1) : nullptr;
    args.lengths = guarded(args.batch);
    for (blockIdx.x = 0; blockIdx.x < gridDim.x; ++blockIdx.x) {
        for (int i = 0; i < LANES; ++i) {
            getcontext(&contexts[i]);
            contexts[i].uc_stack.ss_sp = stacks[i];
            contexts[i].uc_stack.ss_size = sizeof(stacks[i]);
            contexts[i].uc_link = &main_context;
            over[i] = false, turns[i] = 0;
            makecontext(&contexts[i], (void (*)())lane_of_warp, 1, i);
        }
        for (bool any = true; any;) {
            any = false;
            for (current = 0; current < LANES; ++current)
                if (!over[current]) swapcontext(&main_context, &contexts[current]), any |= !over[current];
        }
    }
    printf("status %u\n", status);
    return 0;
}
