// rows_of of qengine_amd/csrc/seq_rows.hpp on the host: reads "c0 c1 t" lines, prints "first n".
#include <cstdio>

#include "../qengine_amd/csrc/seq_rows.hpp"

int main() {
    int c0, c1, t;
    while (scanf("%d %d %d", &c0, &c1, &t) == 3) {
        const RowRange r = rows_of(c0, c1, t);
        printf("%d %d\n", r.first, r.n);
    }
    return 0;
}
