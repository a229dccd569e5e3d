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
                        expect(p.side == 16 ? p.row_tiles == 1 && (p.column_tiles == 1 || p.column_tiles == 2 || p.column_tiles == 4)
                                            : p.side == 32 && (p.row_tiles == 1 || p.row_tiles == 2) &&
                                                  (p.column_tiles == 1 || p.column_tiles == 2),
                               "a kernel for every plan", rows, n);
                        expect(!gated || p.side == 16 || p.row_tiles * p.column_tiles < 4, "a gated kernel, too", rows, n);
                        expect(!pairs || p.side * p.column_tiles % 32 == 0, "groups of 32 results lie in one block", rows, n);
                        expect(p.waves >= 1 && p.waves <= 8, "wavefronts", rows, n);
                        expect(p.waves == 1 || p.waves <= w4_ceil(depth, p.side == 16 ? 128 : 64), "work for every wavefront", rows, depth);
                        expect(w4_few_shared(p, gated) <= 65536, "partial results in 64 KB", rows, n);
                        const int64_t columns = w4_ceil(n, p.side * p.column_tiles), blocks = w4_ceil(rows, p.side * p.row_tiles);
                        expect(columns * p.column_tiles * p.side >= n && blocks * p.row_tiles * p.side >= rows, "all covered", rows, n);
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
