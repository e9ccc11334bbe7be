// hidet_b200/csrc/experts_parts.cuh and qlinear_i8_plan.h on the host.
//
// Reads lines "parts units k_blocks ctas may_be_whole", "plan M N K sms", "rounds units k_blocks pairs slots" and "entries count 0 0 0"; writes total step and all first stages; pair tm split; of every
// pair the number of its units and, of each, unit, first and last k block and who shares it; or the slots, the size and of every entry assignments and room.
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
        if (strcmp(what, "rounds") == 0) {
            printf("%lld", c);
            for (int pair = 0; pair < (int)c; ++pair) {
                const b200q::Rounds r((int)a, (int)b, (int)c, pair, (int)d);
                printf(" %d", r.count());
                for (int i = 0; i < r.count(); ++i) printf(" %d %d %d %d", r.unit(i), r.first_k(i), r.last_k(i), r.shared(i) ? r.split : 1);
            }
            printf("\n");
            continue;
        }
        if (strcmp(what, "entries") == 0) {
            const b200q::EntrySizes e((int)a);
            printf("%d %d", e.slots(), e.size);
            for (int i = 0; i < e.entries; ++i) printf(" %d %d", e.assignments(i), e.room(i));
            printf("\n");
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
