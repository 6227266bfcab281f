// reads lines "rows n k experts cus gemm", prints the rows of a block that a grouped 8-bit product takes
#include <cstdio>

#include "../qengine_amd/csrc/f8_choice.hpp"

int main() {
    long long r, n, k;
    int experts, cus, gemm;
    while (scanf("%lld %lld %lld %d %d %d", &r, &n, &k, &experts, &cus, &gemm) == 6) printf("%d\n", f8_grouped_rows(r, n, k, experts, cus, gemm != 0));
    return 0;
}
