// Functions of qengine_amd/csrc/seq_rows.hpp on the host. Lines "rows c0 c1 t" print "first n"; lines "place slot n b0 .. " (the
// blocks of n sequences) print the level and rank of the slot-th block, as 64 lanes find it, or "none".
#include <cstdio>
#include <cstring>
#include <vector>

#include "../qengine_amd/csrc/seq_rows.hpp"

int main() {
    char what[8];
    while (scanf("%7s", what) == 1) {
        if (!strcmp(what, "rows")) {
            int c0, c1, t;
            if (scanf("%d %d %d", &c0, &c1, &t) != 3) return 1;
            const RowRange r = rows_of(c0, c1, t);
            printf("%d %d\n", r.first, r.n);
        } else {
            int slot, n;
            if (scanf("%d %d", &slot, &n) != 2) return 1;
            std::vector<int> blocks(n);
            for (int& b : blocks)
                if (scanf("%d", &b) != 1) return 1;
            BlockPlace p;
            const bool ok = place_of(slot, [&](int level) {
                int sum = 0;  // over the lanes
                for (int lane = 0; lane < 64; lane++) {
                    int x = 0;
                    for (int i = lane; i < n; i += 64) x = add_blocks(x, blocks[i], level);
                    sum += x;
                }
                return sum;
            }, p);
            if (ok) printf("%d %d\n", p.level, p.rank);
            else printf("none\n");
        }
    }
    return 0;
}
