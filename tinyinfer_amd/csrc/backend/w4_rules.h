// Sizes of 4-bit matrices and 8-bit rows and how products are divided among
// work-groups: plain functions (no HIP), so that they can be checked without a
// GPU.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace mphip {

constexpr int kW4Group = 32;   // elements of a scale
constexpr int kW4Step = 128;   // columns of a tile, one matrix instruction deep
constexpr int kW4Rows = 16;    // rows of a tile
constexpr int kW4Word = 4;     // tiles whose scales share a word
constexpr int kW4MostRows = 1 << 20, kW4MostDepth = 1 << 20, kW4MostMatrixRows = 1 << 24;

constexpr int64_t w4_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int64_t w4_tiles(int64_t rows) { return w4_ceil(rows, kW4Rows); }
constexpr int64_t w4_steps(int64_t depth) { return w4_ceil(depth, kW4Step); }
constexpr int64_t w4_words(int64_t depth) { return w4_ceil(depth, kW4Step * kW4Word); }
constexpr size_t w4_code_bytes(int64_t rows, int64_t depth) { return (size_t)(w4_tiles(rows) * w4_steps(depth)) * 1024; }
constexpr size_t w4_scale_bytes(int64_t rows, int64_t depth) { return (size_t)(w4_tiles(rows) * w4_words(depth)) * 256; }

// Elements of a call on rows alone (norm, conversion): 2^30 threads of 8.
constexpr int64_t kRowsMostElements = (int64_t)1 << 33;

// Runs of 16 bytes from which on a read takes 8 rows a thread: 34 us instead of 47
// for 49,152 FP32 rows of 576 in order, to three buffers in turn (7 million runs).
// Rows out of order have no lines in common: 37.2 instead of 36.2 for as many, 15.4
// instead of 14.4 for 16,000 (2 million), 4.3 instead of 2.8 for 64.
constexpr int64_t kW4ReadRuns = 1 << 22;

// A product by wavefronts that share a block of columns and deal the depth
// among themselves: `column_tiles` tiles of `side` columns and rows a wavefront,
// `waves` of them a work-group.
struct W4Plan {
    int side, column_tiles, waves;
};

constexpr int64_t w4_groups(const W4Plan& p, int rows, int n) {
    return w4_ceil(n, p.side * p.column_tiles) * w4_ceil(rows, p.side);
}
// Places that a tile's rows take in LDS: a power of two, and all 8 runs of a
// tile of 32 rows have one of their own.
constexpr int w4_places(int rows) { return rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32; }
// Bytes of LDS: a wavefront's rows as operands (`parts` BF16 numbers an element),
// at the end the sums that meet.
constexpr size_t w4_few_shared(const W4Plan& p, int rows, int parts, bool gated) {
    const int side = p.side, inside = rows < side ? rows : side;
    const size_t operands = (size_t)p.waves * parts * (side == 16 ? 16 : 8) * w4_places(inside) * 16;
    const size_t sums = (size_t)p.waves * p.column_tiles * (gated ? 2 : 1) * side * side * 4;
    return operands > sums ? operands : sums;
}

constexpr int64_t kW4MostGroups = 1 << 22;  // 2^31 threads of 512

// Tiles of 32 from 17 rows on; as many columns a wavefront as leave a work-group
// for every CU: with 512 instead of 256 of them 1,000 FP32 rows of 576 by 960 take
// 13.1 us instead of 9.9, 64 BF16 rows of 4,096 by 12,288 20.9 instead of 19.0, 512
// FP32 rows through a gated pair of 576 by 1,536 13.0 instead of 14.2; with 1,024
// 16 rows of 576 by 49,152 12.8 instead of 10.3; with 128 one row of 4,096 by 4,096
// 7.3 instead of 6.1.
inline W4Plan w4_few_plan(int rows, int n, int depth, int parts, bool gated, bool eight) {
    W4Plan p{rows <= 16 ? 16 : 32, rows <= 16 ? 4 : 2, 8};
    // 8-bit results: a row's group of 32 lies in one block.
    const int least = eight && p.side == 16 ? 2 : 1;
    while (p.column_tiles > least && w4_groups(p, rows, n) < 256) p.column_tiles /= 2;
    const int64_t blocks = w4_ceil(depth, p.side == 16 ? 128 : 64);
    while (p.waves > 1 && (p.waves > blocks || w4_few_shared(p, rows, parts, gated) > 65536)) p.waves /= 2;
    return p;
}

// More rows, by tiles that work-groups bring their rows to LDS for: 128 rows by
// 256 columns (128 of each matrix of a gated pair), or 64 by 128, 64 columns of
// depth at a time. For the large ones 8-bit rows are laid out before, in blocks of
// 128 rows and 64 columns: two planes of 24 bytes a lane, and their scales.
constexpr int kTileRows = 128, kTileColumns = 256, kTileDepth = 64;
constexpr int kSmallTileRows = 64, kSmallTileColumns = 128;
constexpr int kPlaneBytes = 64 * 24, kPlanesBlock = 4 * 2 * kPlaneBytes;  // of 32 and of 128 rows

enum W4Way { kW4Few, kW4SmallTiles, kW4LargeTiles };

constexpr int64_t w4_tile_groups(int64_t rows, int64_t n, bool gated, bool large) {
    return large ? w4_ceil(rows, kTileRows) * w4_ceil(n, gated ? kTileColumns / 2 : kTileColumns)
                 : w4_ceil(rows, kSmallTileRows) * w4_ceil(n, gated ? kSmallTileColumns / 2 : kSmallTileColumns);
}
// Tiles where there is one for every CU, the largest that leave that. Small ones
// from 128 work-groups on would take 256 BF16 rows of 4,096 by 4,096 from 20.3 us to
// 35.6, from 512 on only 64 FP32 rows of 576 by 49,152 from 20.0 to 22.6; large ones
// from 100 on 1,024 BF16 rows of 4,096 by 4,096 from 43.9 to 71.4 and 2,048 FP16 rows
// of 1,024 by 2,048 from 23.3 to 39.3, from 512 on only 2,048 8-bit rows of 4,096 by
// 4,096 from 58.1 to 93.6. The rule does not look at columns that a tile has in vain:
// for 32,768 BF16 rows of 576 by 64 small tiles would take 12.3 us instead of 18.6.
constexpr W4Way w4_way(int rows, int n, bool gated) {
    return rows > 64 && w4_tile_groups(rows, n, gated, true) >= 256 ? kW4LargeTiles
           : rows > 32 && w4_tile_groups(rows, n, gated, false) >= 256 ? kW4SmallTiles
                                                                      : kW4Few;
}

constexpr int64_t w4_planes_blocks(int64_t rows, int64_t depth) {
    return w4_ceil(rows, kTileRows) * w4_ceil(depth, kTileDepth);
}
constexpr size_t w4_planes_bytes(int64_t rows, int64_t depth) {
    return (size_t)w4_planes_blocks(rows, depth) * kPlanesBlock +
           (size_t)(w4_ceil(rows, kTileRows) * w4_steps(depth)) * kTileRows * 8;
}

}  // namespace mphip
