// How products of rows with 4-bit matrices are divided (w4_rules.h).
#include <stdio.h>
#include <stdlib.h>

#include "w4_rules.h"

using namespace mphip;

static void expect(bool ok, const char* what, long a = 0, long b = 0) {
    if (ok) return;
    fprintf(stderr, "%s (%ld, %ld)\n", what, a, b);
    exit(1);
}

static void few() {
    const int sizes[] = {1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 200, 511, 576, 960, 1000, 1536, 4095, 4096, 12288, 16384, 49152, 1 << 20};
    const int depths[] = {32, 64, 128, 160, 512, 576, 1024, 1536, 4096, 12288, 16384, 1 << 20};
    for (int rows : sizes)
        for (int n : sizes)
            for (int depth : depths)
                for (int gated = 0; gated < 2; ++gated)
                    for (int pairs = 0; pairs < (n % 32 ? 1 : 2); ++pairs) {
                        const W4Plan p = w4_few_plan(rows, n, depth, gated, pairs);
                        expect(p.column_tiles == 1 || p.column_tiles == 2 || p.column_tiles == 4, "column tiles", rows, n);
                        expect(p.row_tiles == 1 || p.row_tiles == 2 || p.row_tiles == 4, "row tiles", rows, n);
                        expect(!pairs || p.column_tiles % 2 == 0, "groups of 32 results lie in one block", rows, n);
                        expect(p.waves >= 1 && p.waves <= 8, "wavefronts", rows, n);
                        expect(p.waves == 1 || p.waves <= w4_steps(depth), "a step for every wavefront", rows, depth);
                        expect(p.waves * p.column_tiles * p.row_tiles * (gated + 1) <= 64, "partial results in 64 KB", rows, n);
                        const int64_t columns = w4_ceil(w4_tiles(n), p.column_tiles), blocks = w4_ceil(w4_tiles(rows), p.row_tiles);
                        expect(columns * p.column_tiles * 16 >= n && blocks * p.row_tiles * 16 >= rows, "all covered", rows, n);
                        expect(w4_groups(p, rows, n) == columns * blocks, "groups", rows, n);
                    }
}

static void sizes() {
    expect(w4_code_bytes(16, 128) == 1024 && w4_code_bytes(17, 129) == 4096, "codes");
    expect(w4_scale_bytes(16, 512) == 256 && w4_scale_bytes(17, 513) == 1024, "scales");
    expect(w4_code_bytes(kW4MostMatrixRows, kW4MostDepth) == (size_t)1 << 43, "no overflow");
}

int main() {
    few();
    sizes();
    puts("ok");
}
