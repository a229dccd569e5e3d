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

// A product by wavefronts that share a block of columns and deal the depth
// among themselves: `column_tiles` and `row_tiles` of 16 a wavefront, `waves`
// of them a work-group.
struct W4Plan {
    int column_tiles, row_tiles, waves;
};

constexpr int64_t w4_groups(const W4Plan& p, int rows, int n) {
    return w4_ceil(w4_tiles(n), p.column_tiles) * w4_ceil(w4_tiles(rows), p.row_tiles);
}

constexpr int64_t kW4MostGroups = 1 << 22;  // 2^31 threads of 512

inline W4Plan w4_few_plan(int rows, int n, int depth, bool gated, bool pairs) {
    const int row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    W4Plan p{4, row_tiles, 8};
    while (p.column_tiles > (pairs ? 2 : 1) && w4_groups(p, rows, n) < 512) p.column_tiles /= 2;
    const int64_t steps = w4_steps(depth);
    // Partial results of all wavefronts fit 64 KB.
    const int tiles = p.column_tiles * p.row_tiles * (gated ? 2 : 1);
    while (p.waves > 1 && (p.waves > steps || p.waves * tiles > 64)) p.waves /= 2;
    return p;
}

// Many rows: work-groups of 128 rows by 256 columns (128 of each matrix of a
// gated pair), the rows laid out before in blocks of 128 rows and 64 columns:
// 8-bit rows as two planes of E2M3 numbers, 24 bytes a lane each, and their
// scales; float rows as 1 to 3 parts of 16 KB.
constexpr int kW4FewRows = 64, kTileRows = 128, kTileColumns = 256, kTileDepth = 64;
constexpr int kPlaneBytes = 64 * 24, kEightTile = 2 * kPlaneBytes + 256;  // of 32 rows
constexpr int kEightBlock = 4 * kEightTile, kPartBlock = kTileRows * kTileDepth * 2;

constexpr int w4_block_bytes(int type) {
    return type == 3 ? kEightBlock : kPartBlock * (type == 0 ? 3 : type == 2 ? 2 : 1);  // MP_TYPE_*
}
constexpr size_t w4_tiles_workspace(int64_t rows, int64_t depth, int type) {
    return (size_t)(w4_ceil(rows, kTileRows) * w4_ceil(depth, kTileDepth)) * w4_block_bytes(type);
}
constexpr int64_t w4_tiles_groups(int64_t rows, int64_t n, bool gated) {
    return w4_ceil(rows, kTileRows) * w4_ceil(n, gated ? kTileColumns / 2 : kTileColumns);
}
// Where tiles pay.
constexpr bool w4_tiled(int rows, int n, bool gated) {
    return rows > kW4FewRows && w4_tiles_groups(rows, n, gated) >= 128;
}

}  // namespace mphip
