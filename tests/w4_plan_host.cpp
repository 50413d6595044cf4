// Prints the configuration that a 4-bit product runs on, one line per "total_rows experts N cu_count" of
// the input. Host code, compiled from the plan's own header by tests/test_w4_plan.py.
#include <cstdio>

#include "../teamredbench_amd/csrc/gemm_w4_plan.hpp"

int main() {
    long long rows, n;
    int experts, cus;
    while (std::scanf("%lld %d %lld %d", &rows, &experts, &n, &cus) == 4)
        std::printf("%d\n", mb::w4_config(rows, experts, n, cus));
    return 0;
}
