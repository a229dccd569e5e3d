// Prints how products are divided. With rows, columns, depth, parts of an element,
// gated and 8-bit results (1 or 0) as arguments: the way, and for few rows the side
// of a tile, a wavefront's tiles of columns and the wavefronts. Without any: every
// way that sizes can lead to, a line each, with gated and 8-bit results before it.
#include "w4_rules.h"

#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include <set>
#include <tuple>

using namespace mphip;

int main(int argc, char** argv) {
    if (argc == 7) {
        int n[7];
        for (int i = 1; i < 7; ++i) n[i] = std::atoi(argv[i]);
        const W4Way way = w4_way(n[1], n[2], n[5]);
        std::printf("%d", (int)way);
        if (way == kW4Few) {
            const W4Plan p = w4_few_plan(n[1], n[2], n[3], n[4], n[5], n[6]);
            std::printf(" %d %d %d", p.side, p.column_tiles, p.waves);
        }
        std::printf("\n");
        return 0;
    }
    if (argc != 1) return 1;
    std::set<std::tuple<int, int, int, int, int>> seen;
    for (int rows = 1; rows < 5000; rows += rows < 520 ? 1 : 61)
        for (int n = 32; n <= kW4MostMatrixRows; n = n < 4096 ? n + 32 : n + n / 64 / 32 * 32)
            for (int gated : {0, 1})
                for (int eight : {0, 1}) {
                    const W4Way way = w4_way(rows, n, gated);
                    W4Plan p{0, 0, 0};
                    if (way == kW4Few) p = w4_few_plan(rows, n, 576, 1, gated, eight);
                    seen.insert({gated, eight, (int)way, p.side, p.column_tiles});
                }
    for (const auto& [gated, eight, way, side, tiles] : seen) {
        std::printf("%d %d %d", gated, eight, way);
        if (way == kW4Few) std::printf(" %d %d", side, tiles);
        std::printf("\n");
    }
    return 0;
}
