// The choice between the kernels of the int8 x int8 product.  Plain C++: it runs on the host alone (tests/host/experts_parts.cpp has it too).
#pragma once

#include <stdint.h>

namespace b200q {

inline int64_t i8_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Which kernel takes a product whose operands and result lie in lines of 16 bytes, in tiles of how many tokens, and how many CTAs (pairs of them) share a tile's K.
struct I8Plan {
    bool pair = false;
    int tm = 0, split = 1;
};

// Estimated microseconds, the least of all forms.  A stage (128 k) takes an SM what its bytes take at some 50 a clock, copies from L2 and memory alike, and a round of CTAs at least what its
// weights take from memory, or, on pairs of SMs, what making a tile's results takes, beside which the next one's products run; to that come a start and an end, the meeting where K is shared, and for the single CTAs' kernel, whose sums pass through shared memory, some per
// token.  Of 39 sizes of 1 to 8000 tokens, every form timed, the choice is the fastest or within 5 % of it at 31, within 14 % at 38, 18 % off at (33, 2048, 8192).  What it is between, us:
//     64 x 4096 x 4096      single CTAs, tiles of 32, four a tile 8.6    pairs 9.7
//     512 x 4096 x 4096     pairs, tiles of 128 12.9                     two pairs a tile 14.5, single CTAs 22.2
//     512 x 11008 x 4096    two pairs a tile, tiles of 256 22.6          one 26.1
//     1000 x 16384 x 512    four pairs a tile, tiles of 192 17.3         two 21.7
//     2219 x 128 x 11360    pairs, tiles of 256 25.9                     tiles of 128 32.2 (the results' 1.2 us a tile and 10 ns a token)
inline I8Plan plan_i8(int64_t M, int64_t N, int64_t K, int sms) {
    const int64_t k_blocks = i8_ceil(K, 128);
    // `ctas` with a part of K each, `places` at once: rounds take what an SM's copies or products take, or the weight's way from memory
    auto stream_us = [&](int64_t ctas, int64_t places, int64_t split, double stage, double results) {
        const double products = (double)i8_ceil(k_blocks, split) * stage / 1900.0, own = products > results ? products : results, weight = (double)K * N / 6.5e6;
        const int64_t full = ctas / places, rest = ctas - full * places;
        const double round = weight * places / ctas, last = weight * rest / ctas;
        return full * (own > round ? own : round) + (rest == 0 ? 0.0 : own > last ? own : last);
    };
    I8Plan best;
    double least = 1e300;
    // single CTAs: tiles of 128 channels, K shared by up to eight; two an SM up to 64 tokens
    for (int64_t parts = i8_ceil(M, 256); parts <= i8_ceil(M, 256) + 3 && M <= 1024; ++parts) {
        const int64_t tm = i8_ceil(i8_ceil(M, parts), 16) * 16, tiles = i8_ceil(N, 128) * i8_ceil(M, tm), places = (tm <= 64 ? 2 : 1) * (int64_t)sms;
        for (int split = 1; split <= 8 && split <= k_blocks; split *= 2) {  // clusters of seven found fewer places (128 x 8192 x 1280: 14.6 us for 9.5)
            const int64_t ctas = tiles * split;
            const bool two = ctas > sms && tm <= 64;
            const double us = 4.3 + 0.032 * tm + 4.0 * (i8_ceil(ctas, places) - 1) + stream_us(ctas, places, split, (16384 + 128 * tm) * (two ? 2.0 / 60.0 : 1.0 / 46.0), 0.0);
            if (us < least) least = us, best.pair = false, best.tm = (int)tm, best.split = split;
        }
    }
    // pairs: tiles of 256 channels
    for (int tm = 32; tm <= 256 && tm < M + 32; tm += 32) {
        const int64_t tiles = i8_ceil(N, 256) * i8_ceil(M, tm);
        double stage = (16384 + 64 * tm) / (55.0 - (tm > 128 ? 0.05 * (tm - 128) : 0.0));
        if (stage < 390.0) stage = 390.0;
        for (int split = 1; split <= 4 && split <= k_blocks; split *= 2) {
            // clusters of eight CTAs lie within a group of SMs, of which some are left over
            if (split > 1 && tiles * split > (split == 4 ? sms * 3 / 8 : sms / 2)) break;
            const double us = 4.1 + 0.008 * tm + (split > 1 ? 0.006 * tm + (split > 2 ? 3.0 : 2.0) : 0.0) + stream_us(tiles * split, sms / 2, split, stage, split > 1 || tiles <= sms / 2 ? 0.0 : 1.2 + 0.0097 * tm);
            if (us < least) least = us, best.pair = true, best.tm = tm, best.split = split;
        }
    }
    return best;
}

}  // namespace b200q
