// hidet_b200/csrc/experts_parts.cuh and qlinear_i8_plan.h on the host.
//
// Reads lines "parts units k_blocks ctas may_be_whole" and "plan M N K sms"; writes total step and all first stages, or pair tm split.
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#define __host__
#define __device__
#define __forceinline__ inline

#include "../../hidet_b200/csrc/experts_parts.cuh"
#include "../../hidet_b200/csrc/qlinear_i8_plan.h"

int main() {
    char what[16];
    long long a, b, c, d;
    while (scanf("%15s %lld %lld %lld %lld", what, &a, &b, &c, &d) == 5) {
        if (strcmp(what, "plan") == 0) {
            const b200q::I8Plan p = b200q::plan_i8(a, b, c, (int)d);
            printf("%d %d %d\n", (int)p.pair, p.tm, p.split);
            continue;
        }
        const b200q::Parts p((uint32_t)a, (uint32_t)b, (uint32_t)c, d != 0);
        printf("%u %u", p.total, p.step);
        for (uint32_t i = 0; i <= (uint32_t)c; ++i) printf(" %u", p.first_of(i));
        if (p.step == 1 && p.total < 4096)
            for (uint32_t i = 0; i < p.total; ++i) printf(" %u", p.cta_of(i));
        printf("\n");
    }
}
