// Which rows belong to a sequence of a packed batch. Plain functions of numbers, the same on the host (where
// tests/test_seq_rows.py runs them) and in the kernels.
#pragma once
#include <hip/hip_runtime.h>

struct RowRange {
    int first, n;
};
// The rows of a sequence that starts at c0 and ends at c1, of t rows. The starts are device memory that nothing has checked:
// both are moved into 0 .. t before they are subtracted (c1 near -2^31 less a start past 0 would wrap to a large length).
__host__ __device__ inline RowRange rows_of(int c0, int c1, int t) {
    const int a = c0 < 0 ? 0 : c0 < t ? c0 : t, e = c1 < 0 ? 0 : c1 < t ? c1 : t;
    return {a, e > a ? e - a : 0};
}
