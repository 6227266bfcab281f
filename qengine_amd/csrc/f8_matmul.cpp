// The 8-bit products' checks and the choice of their kernel (f8.hpp).
#include "f8.hpp"
#include "f8_choice.hpp"

#include <algorithm>

namespace {
struct Choice {
    int bt = 0, bw = 0, parts = 1;  // bt 256: f8_gemm, else f8_ring
    double us = 1e30;
};

// us of a product of up to 64 rows by rounds of blocks, one a CU (MI355X): a block takes its stages' bytes at 40 bytes/ns and 4 us to start
// and end; the weights come at 5.4 TB/s at most. K ranges cost a launch (4 us) and the sums written and read again at 5 TB/s. Measured /
// modelled: 48 rows of 34816 x 5120: 192 columns a block 36 / 37, 128 48 / 53, 64 44 / 53; of 5120 x 17408: 64 columns in 3 ranges
// 20 / 27, 128 in 6 21 / 26. Small matrices it splits for nothing: 1024 x 2048 10.8, by blocks of 32 x 64 unsplit 7.9.
Choice choose_few(const F8Mat& a) {
    const int cus = qe_num_cus(), blocks = (a.k + 127) / 128, bt = a.r <= 32 ? 32 : 64;
    Choice best;
    for (int bw : {64, 128, 192}) {
        const int64_t tiles = (a.n + bw - 1) / bw;
        for (int p = 1; p <= 16 && p <= blocks && (p == 1 || tiles * p <= cus); p++) {
            const double rounds = (double)((tiles * p + cus - 1) / cus), steps = (blocks + p - 1) / p;
            double us = std::max(rounds * steps * (bt + bw) * 128 / 40e3, (double)a.n * a.k / 5.4e6) + 4;
            if (p > 1) us += 4 + 2.0 * tiles * p * bt * bw * 4 / 5e6;
            if (us < best.us) best = {bt, bw, p, us};
        }
    }
    return best;
}

// More rows: blocks of every shape but 32 x 192, `fit` of them a CU at once, whose step of 128 k takes `alone` us or `each` for each of
// several; fitted to 2500 measured products of 12 matrices (512 to 34816 rows of 1024 to 17408) with 100 to 2500 rows, blocks and
// ranges of all shapes. Measured, the choice is 1 % slower than the fastest of them on average and 19 % at most (14336 x 4096, 512 rows:
// 51 us, by 128 x 128 43); with blocks of 128 or 256 rows only, by the model above, it was 12 %, 74 % at most. 400 rows of 2048 x 6144: 24.1 ->
// 15.3 us (blocks of 64 x 64, none of them split); 160 of 10240 x 5120: 38.7 -> 22.3; 1000 of 5120 x 17408: 256 x 256 in 3 ranges, 100.
Choice choose(const F8Mat& a) {
    if (a.r <= 64) return choose_few(a);
    struct Shape {
        int bt, bw, fit;
        double alone, each;
    };
    static constexpr Shape kShapes[] = {{32, 64, 3, .10, .156}, {32, 128, 2, .21, .25}, {64, 64, 2, .10, .223}, {64, 128, 2, .33, .33}, {64, 192, 1, .50, .364},
                                        {128, 64, 2, .34, .36}, {128, 128, 2, .40, .75}, {128, 192, 1, .40, 1.0}, {256, 256, 1, 1.05, 1.32}};
    const int cus = qe_num_cus(), blocks = (a.k + 127) / 128;
    Choice best;
    for (const Shape& s : kShapes) {
        const int64_t tiles = (int64_t)((a.r + s.bt - 1) / s.bt) * ((a.n + s.bw - 1) / s.bw);
        for (int p = 1; p <= 16 && p <= blocks && (p == 1 || tiles * p <= cus); p++) {
            const int64_t most = (tiles * p + cus - 1) / cus, rest = most % s.fit;  // blocks of a CU
            const double steps = (blocks + p - 1) / p;
            double us = steps * ((most / s.fit) * std::max(s.alone, s.fit * s.each) + (rest ? std::max(s.alone, rest * s.each) : 0)) + 1.1 * most / s.fit;
            us = std::max(us, (double)a.n * a.k / 6.3e6) + 4.2;
            if (p > 1) us += 3.5 + 2.0 * tiles * p * s.bt * s.bw * 4 / 5.2e6;
            if (us < best.us) best = {s.bt, s.bw, p, us};
        }
    }
    return best;
}
}  // namespace

static void check(const F8Mat& a) {
    CHECK(a.n > 0 && a.n <= kF8MaxDim && a.k > 0 && a.k <= kF8MaxDim && a.k % 16 == 0, "matmul_f8: n = %d, k = %d", a.n, a.k);
    CHECK(a.r > 0 && a.r <= kF8MaxRows && a.t >= 0 && a.t <= kF8MaxRows && (a.off || a.t == a.r), "matmul_f8: %d rows of x, %d of y", a.t, a.r);
    CHECK(a.experts > 0 && a.experts <= kF8MaxExperts && (a.off || (a.experts == 1 && !a.rows)), "matmul_f8: %d matrices", a.experts);
    CHECK((int64_t)a.r * a.n <= (int64_t)1 << 34, "matmul_f8: %d rows of %d are too many for a call", a.r, a.n);
    CHECK(a.q && a.s && a.y && (a.t == 0 || (a.x && a.xs)), "matmul_f8: a tensor is missing");
    CHECK(((uintptr_t)a.q & 15) == 0 && ((uintptr_t)a.x & 15) == 0 && a.ldx % 16 == 0 && a.ldx >= 0 && a.ldx < kF8MaxRowBytes,
          "matmul_f8: x and its rows are 16-byte aligned, rows less than %d bytes apart", kF8MaxRowBytes);
    CHECK(a.t < 2 || (a.xs_row >= 0 && a.xs_row < kF8MaxScaleStride), "matmul_f8: scales of rows are less than %d elements apart", kF8MaxScaleStride);
}

static void grouped(const F8Mat& call, int bt, hipStream_t st) {
    F8Mat a = call;
    if (a.t == 0) {  // every index is outside x: rows that are read and not used
        a.x = a.q;
        a.xs = a.s;
        a.ldx = a.xs_row = 0;
        a.xs_group = 1;
    }
    if (bt == 16) f8_dec(a, st);
    else if (bt == 256) f8_gemm(a, 1, st);
    else f8_ring(a, bt, 128, 1, st);
}

void f8_matmul(const F8Mat& a, hipStream_t st) {
    check(a);
    if (a.off) return grouped(a, f8_grouped_rows(a.r, a.n, a.k, a.experts, qe_num_cus(), f8_gemm_takes(a)), st);
    // 16 rows of 34816 x 5120 36 us by f8_dec, of 5120 x 17408 19
    if (a.r <= 16) return f8_dec(a, st);
    const Choice c = choose(a);
    if (c.bt == 256) f8_gemm(a, c.parts, st);
    else f8_ring(a, c.bt, c.bw, c.parts, st);
}

void f8_matmul_choice(const F8Mat& a, int bt, int bw, int parts, hipStream_t st) {
    check(a);
    CHECK(!a.off && parts >= 1 && parts <= 16 && parts <= (a.k + 127) / 128, "matmul_f8: %d K ranges of %d", parts, a.k);
    if (bt == 16) return f8_dec(a, st);
    if (bt == 256) return f8_gemm(a, parts, st);
    CHECK((bt == 32 || bt == 64 || bt == 128) && (bw == 64 || bw == 128 || bw == 192), "matmul_f8: blocks of %d x %d", bt, bw);
    f8_ring(a, bt, bw, parts, st);
}

void f8_grouped_choice(const F8Mat& a, int bt, hipStream_t st) {
    check(a);
    CHECK(a.off && (bt == 16 || bt == 64 || bt == 128 || (bt == 256 && f8_gemm_takes(a))), "matmul_f8_grouped: blocks of %d rows", bt);
    grouped(a, bt, st);
}
