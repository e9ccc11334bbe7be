// What a CTA of the kernels of experts_stream.cu takes of a line of stages, and where its pieces lie when a unit has several CTAs; how experts_many.cu cuts an expert's assignments into entries, and
// which units, and which part of their k, a pair has.
//
// No header of CUDA's is included, so that it runs on the host as well (tests/host/experts_parts.cpp).
#pragma once

#include <stdint.h>

namespace b200q {

// The line: units (an entry's tile of rows) of k_blocks stages each.  CTA c takes stages first_of(c) .. first_of(c + 1) - 1: `each` pieces of `step` stages, and one of the `more` that are left.
// Divisions are of 32 bits: those of 64 took 2 us of a kernel's start, and more at its end.
struct Parts {
    uint32_t total, step, each, more;
    // may_be_whole: units need not be cut where the CTA with the most has hardly more than an equal part; bringing a cut one together takes the time of some ten stages.
    __host__ __device__ __forceinline__ Parts(uint32_t units, uint32_t k_blocks, uint32_t ctas, bool may_be_whole) {
        total = units * k_blocks;
        const bool whole = may_be_whole && (units + ctas - 1) / ctas * k_blocks <= total / ctas + 10;
        const uint32_t pieces = whole ? units : total;
        step = whole ? k_blocks : 1, each = pieces / ctas, more = pieces - each * ctas;
    }
    __host__ __device__ __forceinline__ uint32_t first_of(uint32_t cta) const { return (cta * each + (cta < more ? cta : more)) * step; }
    // Who has a stage; where units are cut.
    __host__ __device__ __forceinline__ uint32_t cta_of(uint32_t stage) const {
        const uint32_t large = more * (each + 1);
        return stage < large || each == 0 ? stage / (each + 1) : more + (stage - large) / each;
    }
    // A CTA has at most two places for what it holds of something shared: the first for what its part begins with, the second for what it ends with.
    __host__ __device__ __forceinline__ bool second_place(uint32_t cta, uint32_t first_stage) const { return first_of(cta) < first_stage; }
};

// An expert's assignments in entries of one size but the last, each with slots for a multiple of kEntrySlots.
constexpr int kEntryMost = 80;   // 240 columns
constexpr int kEntrySlots = 16;
struct EntrySizes {
    int count, entries, size;
    __host__ __device__ __forceinline__ EntrySizes(int count_) : count(count_) {
        entries = (count + kEntryMost - 1) / kEntryMost;
        size = count > 0 ? (count + entries - 1) / entries : 1;
    }
    __host__ __device__ static __forceinline__ int rounded(int n) { return (n + kEntrySlots - 1) / kEntrySlots * kEntrySlots; }
    __host__ __device__ __forceinline__ int assignments(int entry) const { return entry + 1 < entries ? size : count - entry * size; }  // of the last: at least one, up to 8192 in all
    __host__ __device__ __forceinline__ int room(int entry) const { return rounded(assignments(entry)); }
    __host__ __device__ __forceinline__ int slots() const { return (entries - 1) * rounded(size) + room(entries - 1); }
};

constexpr int kMostSplit = 8;
// The units of a pair: whole rounds of all pairs, neighbours at a time, and of the units that are left each is shared by `split` pairs, a part of K each.  Bringing a unit together costs the
// time of some stages, and of some more for each pair and ten slots.
struct Rounds {
    int rounds, split, rest, pairs, pair, k_blocks;
    __host__ __device__ __forceinline__ Rounds(int units, int k_blocks_, int pairs_, int pair_, int slots) : pairs(pairs_), pair(pair_), k_blocks(k_blocks_) {
        rounds = units / pairs, rest = units - rounds * pairs, split = 1;
        int least = k_blocks;
        for (int s = 2; s <= kMostSplit && rest * s <= pairs && s <= k_blocks; ++s) {
            const int cost = (k_blocks + s - 1) / s + 4 + (s - 1) * slots / 10;
            if (cost < least) least = cost, split = s;
        }
    }
    __host__ __device__ __forceinline__ int count() const { return rounds + (pair < rest * split ? 1 : 0); }
    __host__ __device__ __forceinline__ bool shared(int i) const { return i == rounds && split > 1; }
    __host__ __device__ __forceinline__ int unit(int i) const { return i < rounds ? i * pairs + pair : rounds * pairs + pair / split; }
    __host__ __device__ __forceinline__ int first_k(int i) const { return i < rounds ? 0 : k_blocks * (pair % split) / split; }
    __host__ __device__ __forceinline__ int last_k(int i) const { return i < rounds ? k_blocks : k_blocks * (pair % split + 1) / split; }
};

}  // namespace b200q
