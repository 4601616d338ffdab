// Host-side checks of the grouped product's plans that keep it from waiting for
// good (csrc/tinym_grouped.cuh: grouped_plan).  Built with nvcc and run on the
// CPU by tests/test_grouped_safety.py; no GPU is touched.
//
//  * A CTA of a pair plan takes all of its SM's shared memory, whatever K is:
//    it is alone on its SM, so nothing contends for tensor memory there.
#include <cstdio>

#include "tinym_grouped.cuh"

int main() {
    const uint32_t limit = 232448;
    long checks = 0, failures = 0, pairs = 0;
    for (int64_t rows : {65, 130, 700, 8192})
        for (int64_t experts : {1, 2, 8, 1024})
            for (int64_t n : {1, 300, 5120})
                for (int64_t k_bytes = 16; k_bytes <= 8192; k_bytes += k_bytes < 2048 ? 16 : 512)
                    for (int fp4 = 0; fp4 < 2; ++fp4) {
                        tinym::GroupedPlan g;
                        ++checks;
                        if (tinym::grouped_plan(fp4, rows, experts, n, k_bytes, 148, limit, &g)) {
                            ++failures;
                            continue;
                        }
                        if (!g.pair) continue;
                        ++pairs;
                        if (g.smem != limit && ++failures <= 10)
                            std::printf("FAIL pair plan of %u bytes (rows %ld, K bytes %ld)\n", g.smem,
                                        static_cast<long>(rows), static_cast<long>(k_bytes));
                    }
    if (failures || !pairs) {
        std::printf("%ld of %ld checks failed, %ld pair plans\n", failures, checks, pairs);
        return 1;
    }
    std::printf("grouped safety checks ok (%ld checks)\n", checks);
    return 0;
}
