// What a call on the 8-bit cache touches and how it is divided among
// work-groups: plain functions (no HIP; the kernels call the constexpr ones),
// so that they can be checked without a GPU.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace mphip {

constexpr int kTile = 16;  // tokens of a tile
constexpr int kKv8MaxRows = 1 << 20, kKv8MaxHeads = 1024, kKv8MaxGroup = 16, kKv8MaxLength = 1 << 30;

// Rows times query heads of an attention call: 2^31 threads at most.
constexpr int64_t kKv8MostColumns = 1 << 22;

// Rows start .. next-1 of a sequence inside 0 .. rows-1, whatever the two are.
struct Kv8Span {
    int row0, count;
};
constexpr Kv8Span kv8_span(int start, int next, int rows) {
    const int row0 = start < 0 ? 0 : start > rows ? rows : start;
    const int row1 = next < row0 ? row0 : next > rows ? rows : next;
    return {row0, row1 - row0};
}

// Pages that `count` (at least 1) tokens from position `used` on touch; none
// for a position that no sequence has.
constexpr int kv8_pages(int count, int used, int page_shift) {
    const int bt = 1 << page_shift;
    return used < 0 || used > kKv8MaxLength ? 0 : ((used & (bt - 1)) + count + bt - 1) >> page_shift;
}
// The `index`-th of those pages: its number in the table, its slots that the
// tokens take and the token (of `count`) that takes the first of them.
struct Kv8Page {
    int page, first, last, token;
};
constexpr Kv8Page kv8_page(int count, int used, int index, int page_shift) {
    const int page = (used >> page_shift) + index, begin = page << page_shift, end = used + count - begin;
    const int first = used > begin ? used - begin : 0, bt = 1 << page_shift;
    return {page, first, end < bt ? end : bt, begin + first - used};
}
// Pages that `rows` rows of `sequences` sequences touch at most: all but the
// first and last of a sequence are filled, and each has a row at least.
constexpr int64_t kv8_most_pages(int rows, int sequences, int bt) {
    const int64_t by_pages = ((int64_t)rows + (int64_t)sequences * (2 * bt - 2)) / bt;
    return by_pages < rows ? by_pages : rows;
}
constexpr int64_t kv8_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A table's page `page` if it is one of the pool's, else -1.
constexpr int kv8_block(const int32_t* table, int stride, int page, int blocks) {
    if (page < 0 || page >= stride) return -1;
    const int block = table[page];
    return block >= 0 && block < blocks ? block : -1;
}

// A work-group takes 16 * column_tiles columns (a column is one row's query
// head) of a KV head and `chunk` of their tokens; its 1, 4 or 8 `waves` deal
// the chunk's pairs of 16-token tiles among themselves. With more than one
// chunk the results meet in a second launch.
struct Kv8Plan {
    int column_tiles, waves, chunk, splits;
};

constexpr int kKv8Pair = 32;         // tokens of two tiles, a step of a wavefront
constexpr int kKv8MostWaves = 8;     // of a work-group
constexpr int kKv8MostGroups = 512;  // work-groups that splitting over tokens aims at
constexpr int kKv8LeastChunk = 128;  // tokens

// Divides `items` work-groups of up to max_length tokens.
//
// Alone with its columns, a work-group takes about 5.5 us and 3.9 for every
// 1,000 tokens; splitting the tokens takes a second launch (3 to 4 us) and the
// chip's memory rate. One row of 3 KV heads of 64, alone and split: 7.6 and
// 9.6 us at 500 tokens, 11 and 9.9 at 1,500, 17 and 10.3 at 3,000, 119 and 13
// at 30,000; 48 heads of rows 10.8 and 11.7 at 1,500, 15 and 12.8 at 3,000; 192
// 17 and 20.5 at 3,000, 32 and 35 at 8,000. Half as many chunks for very few
// work-groups: 13 instead of 16 us for the row of 30,000, but 39 instead of 32
// for 16 of them.
// Eight wavefronts where the work-groups leave the chip idle and each has
// enough to join for: 17.0 instead of 18.7 us for 192 heads of 3,000 tokens,
// 8.4 instead of 7.9 at 500; 27 instead of 25.6 for 384 heads of 3,000; dims of
// 128 take four up to 2,048 tokens (13.9 and 13.5 at 1,500, 21.6 and 23.6 at
// 4,096).
inline void kv8_split(Kv8Plan* p, int64_t items, int dim, int max_length) {
    const int64_t length = max_length > 0 ? max_length : 1;
    int64_t splits = 1;
    if (items < kKv8MostGroups && length > 1024 + 40 * items) {
        p->waves = 4;
        splits = kv8_ceil(items < 16 ? kKv8MostGroups / 2 : kKv8MostGroups, items);
    } else if (p->waves == 4 && items < 256 && length > (dim == 64 ? 1024 : 2048)) {
        p->waves = 8;
    }
    const int64_t step = (int64_t)kKv8Pair * p->waves;
    int64_t chunk = kv8_ceil(kv8_ceil(length, splits), step) * step;
    if (chunk < kKv8LeastChunk) chunk = kKv8LeastChunk;
    p->chunk = (int)chunk;
    p->splits = (int)kv8_ceil(length, chunk);
}

inline Kv8Plan kv8_decode_plan(int rows, int kv_heads, int dim, int max_length) {
    Kv8Plan p{1, 4, 0, 0};
    kv8_split(&p, (int64_t)rows * kv_heads, dim, max_length);
    return p;
}

// Work-groups of `column_tiles` that the sequences' columns take: every
// sequence's last one may be part empty.
inline int64_t kv8_items(int rows, int sequences, int group, int column_tiles) {
    const int64_t columns = 16 * column_tiles, by_tiles = (int64_t)rows * group / columns + sequences;
    return by_tiles < rows * (int64_t)group ? by_tiles : rows * (int64_t)group;
}

// Two column tiles share a conversion of the codes, where that leaves
// work-groups enough (1 and 2 tiles, us; 3 heads of 64, then 8 of 128): 18.6
// and 20.2 for 512 rows at 1,500 tokens, 57 and 52 for 16 x 256, 445 and 365
// at 16,000; 34 and 30 for 512 rows at 1,500, 176 and 137 for 16 x 256, 35.5
// and 36.4 for prompts of 256. dims of 256 have no registers for two.
// One wavefront a work-group saves the joining where there is work for the
// chip without dealing tokens (1 and 4 wavefronts, us): 15 and 20 for 16 x 256
// rows of prompts, 36 and 79 for the wide heads, 272 and 483 for 16.8k rows of
// prompts of up to 2,000, but 152 and 109 for 16 x 256 rows at 4,000.
inline Kv8Plan kv8_prefill_plan(int rows, int sequences, int kv_heads, int group, int dim, int max_length) {
    Kv8Plan p{1, 4, 0, 0};
    if (dim <= 128 && max_length > 512 &&
        kv8_items(rows, sequences, group, 1) * kv_heads * (int64_t)max_length >= 3 << 19)
        p.column_tiles = 2;
    const int64_t items = kv8_items(rows, sequences, group, p.column_tiles) * kv_heads;
    if (items >= 4096 || max_length <= 64 || (max_length <= 512 && items >= kKv8MostGroups)) p.waves = 1;
    kv8_split(&p, items, dim, max_length);
    return p;
}

// Floats that a plan's partial results take.
inline size_t kv8_partial_floats(const Kv8Plan& p, int rows, int heads, int dim) {
    return p.splits > 1 ? (size_t)rows * heads * p.splits * (dim + 2) : 0;
}

// Floats that hold the partial results of any call of up to these sizes:
// items * splits < 2 * kKv8MostGroups while there is more than one split.
inline size_t kv8_workspace_floats(int rows, int sequences, int heads, int kv_heads, int dim, int max_length) {
    (void)sequences;
    const int64_t splits = kv8_ceil(max_length > 0 ? max_length : 1, kKv8LeastChunk);
    if (splits <= 1) return 0;
    const int64_t columns = 16 * 2;  // of the largest work-group
    const int64_t by_rows = (int64_t)rows * heads * splits, by_groups = 2ll * kKv8MostGroups * columns;
    return (size_t)(by_rows < by_groups ? by_rows : by_groups) * (dim + 2);
}

}  // namespace mphip
