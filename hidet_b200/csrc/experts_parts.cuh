// What a CTA of the kernels of experts_stream.cu takes of a line of stages, and where its pieces lie when a unit has several CTAs.
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

}  // namespace b200q
