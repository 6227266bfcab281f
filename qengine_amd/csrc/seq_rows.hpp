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

// Blocks of rows of all sequences in the order of their index in their sequence, the highest first.
//
// kMostBlocks is above the blocks of any batch whose sequences do not overlap (2^30 rows in blocks of at least 64, and one more
// for each of 4096 sequences). Starts that do not ascend can name more, so a lane's sums stop there: the total over 64 lanes
// stays below 2^31, and the sums still fall with the level by at most what the level has, so the search below ends on a block
// that exists.
constexpr int kMostBlocks = (1 << 24) + (1 << 13);
// n and the blocks of a sequence from index `level` on
__host__ __device__ inline int add_blocks(int n, int blocks, int level) {
    const int more = blocks > level ? blocks - level : 0;
    return n + more < kMostBlocks ? n + more : kMostBlocks;
}
struct BlockPlace {
    int level, rank;  // the block's index, and how many sequences with a block of that index come before its own
};
// Where the slot-th block is. count(level): all sequences' blocks from index `level` on; false: there are not so many blocks
template <class Count>
__host__ __device__ inline bool place_of(int slot, Count count, BlockPlace& p) {
    if (slot >= count(0)) return false;
    int lo = 0, hi = 1;  // the largest level with more than `slot` blocks from it on is in [lo, hi)
    while (hi < kMostBlocks && count(hi) > slot) {
        lo = hi;
        hi *= 2;
    }
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (count(mid) > slot) lo = mid;
        else hi = mid;
    }
    p.level = lo;
    p.rank = slot - count(lo + 1);
    return true;
}
