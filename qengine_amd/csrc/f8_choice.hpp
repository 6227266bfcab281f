// Which kernel a grouped 8-bit product takes (f8.hpp), from what the host knows of it: totals, not the segments' lengths.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>

// -> rows of a block: 16 (f8_dec), 64 or 128 (f8_ring, 128 columns) or, where its offsets reach (`gemm`), 256 (f8_gemm).
//
// us of a call by rounds of blocks: segments of ragged lengths end in a block that is half empty on average, and have one at least. An XCD
// takes an eighth of the rows of blocks, whole ones, with all their columns, and its busiest CU its share of these rounded up, `fit` at once. A block alone takes `alone` us for each 128 k and `start` to begin and end;
// several at once `each`, and 0.6 of `start`, as the one's start hides behind the other's products. Weights and y come and go at 5 TB/s at
// most. Fitted to 200 measured products (1 to 512 matrices of 256 to 8192 x 256 to 8192, 200 to 80000 rows), and on 240 others the
// choice is 0.6 % slower than the fastest on average, 26 % at most; by work alone, without rounds, it was 20 % and 256 %: 1024 rows of
// 8 matrices of 256 x 4096 took 49 us in 256 x 256 tiles on eight CUs, 15 in blocks of 64. 512 matrices of 1024 x 2048, us by 64 / 128 /
// 256 rows: 4096 rows 183 / 235 / 281, 40960 271 / 285 / 325, 81920 423 / 418 / 366.
inline int f8_grouped_rows(int64_t r, int64_t n, int64_t k, int experts, int cus, bool gemm) {
    if (r / experts < 8) return 16;
    struct Shape {
        int bt, bw, fit;
        double alone, each, start;
    };
    static constexpr Shape kShapes[] = {{64, 128, 2, .37, .34, 4.7}, {128, 128, 2, .78, .56, 6.9}, {256, 256, 1, 1.22, 0., 14.}};
    const double steps = (double)((k + 127) / 128), moved = (double)experts * n * k + 2.0 * r * n;
    int best = 0;
    double least = 1e30;
    for (const Shape& s : kShapes) {
        if (s.bt == 256 && !gemm) continue;
        const double rows = std::max((double)r / s.bt + 0.5 * experts, (double)experts), blocks = std::ceil(rows / 8) * (double)((n + s.bw - 1) / s.bw);
        const double most = std::ceil(blocks * 8 / cus), full = std::floor(most / s.fit), rest = most - full * s.fit;
        auto at_once = [&](double m) { return m > 0 ? std::max(steps * s.alone + s.start, m * (steps * s.each + 0.6 * s.start)) : 0.0; };
        const double us = std::max(full * at_once(s.fit) + at_once(rest), moved / 5.0e6);
        if (us < least) least = us, best = s.bt;
    }
    return best;
}
