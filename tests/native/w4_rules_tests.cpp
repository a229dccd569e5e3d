// How products of rows with 4-bit matrices are divided (w4_rules.h).
#include <stdio.h>
#include <stdlib.h>

#include <initializer_list>

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
                        for (int parts = 1; parts <= 3; ++parts) {
                            const W4Plan p = w4_few_plan(rows, n, depth, parts, gated, pairs);
                            expect(p.side == 16 ? p.column_tiles == 1 || p.column_tiles == 2 || p.column_tiles == 4
                                                : p.side == 32 && (p.column_tiles == 1 || p.column_tiles == 2),
                                   "a kernel for every plan", rows, n);
                            expect(!pairs || p.side * p.column_tiles % 32 == 0, "groups of 32 results lie in one block", rows, n);
                            expect(p.waves >= 1 && p.waves <= 8, "wavefronts", rows, n);
                            expect(p.waves == 1 || p.waves <= w4_ceil(depth, p.side == 16 ? 128 : 64), "work for every wavefront", rows, depth);
                            expect(w4_few_shared(p, rows, parts, gated) <= 65536, "LDS", rows, n);
                            const int64_t columns = w4_ceil(n, p.side * p.column_tiles), blocks = w4_ceil(rows, p.side);
                            expect(columns * p.column_tiles * p.side >= n && blocks * p.side >= rows, "all covered", rows, n);
                            expect(w4_groups(p, rows, n) == columns * blocks, "groups", rows, n);
                        }
                    }
}

static void sizes() {
    expect(w4_code_bytes(16, 128) == 1024 && w4_code_bytes(17, 129) == 4096, "codes");
    expect(w4_scale_bytes(16, 512) == 256 && w4_scale_bytes(17, 513) == 1024, "scales");
    expect(w4_code_bytes(kW4MostMatrixRows, kW4MostDepth) == (size_t)1 << 43, "no overflow");
}

// The kernel's places in LDS: every row of every run has one of its own, inside the wavefront's share.
static void places() {
    for (int rows = 1; rows <= 32; ++rows)
        for (int side = rows <= 16 ? 16 : 32; side <= 32; side += 16) {
            const int runs = side == 16 ? 16 : 8, places = w4_places(rows), mask = places - 1;
            expect(places >= rows && (places & mask) == 0, "places", rows);
            bool taken[16 * 32] = {};
            for (int e = 0; e < runs; ++e)
                for (int r = 0; r < places; ++r) {
                    const int at = e * places + (r ^ (e & mask));
                    expect(at >= 0 && at < runs * places && !taken[at], "a place of its own", rows, at);
                    taken[at] = true;
                    expect(((r ^ e) & mask) == (r ^ (e & mask)), "the reader's place", rows, r);
                }
        }
}

// A way is kept as rows grow: a workspace for more rows is enough for fewer.
static void ways() {
    for (int n : {1, 96, 960, 4096, 12288, 49152})
        for (int gated = 0; gated < 2; ++gated) {
            bool large = false;
            for (int rows = 1; rows < 5000; rows += rows < 300 ? 1 : 37) {
                const bool now = w4_way(rows, n, gated) == kW4LargeTiles;
                expect(now || !large, "large tiles for more rows, too", rows, n);
                large = now;
            }
        }
    expect(w4_planes_bytes(129, 65) == (size_t)4 * 12288 + 2 * 1024 && kPlanesBlock == 12288, "planes");
}

int main() {
    few();
    places();
    ways();
    sizes();
    puts("ok");
}
