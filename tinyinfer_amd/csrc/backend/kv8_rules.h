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
// Alone with its columns, a work-group of four wavefronts takes about 5 us and
// 4 for every 1,000 tokens; splitting the tokens takes a second launch (2 to 3
// us) and then the chip's memory rate. One row of 3 KV heads of 64, alone and
// split: 6.9 and 8.5 us at 500 tokens, 10.1 and 8.8 at 1,500, 14.4 and 9.2 at
// 3,000, 90 and 12 at 30,000; 48 heads of rows 10.1 and 10.7 at 1,500, 14.6 and
// 11.7 at 3,000; 192 16.0 and 19.8 at 3,000, 31.5 and 35.5 at 8,000. Half as many
// chunks for very few work-groups: 12 instead of 15 us for the row of 30,000,
// but 39 instead of 31 for 16 of them.
// Eight wavefronts where the work-groups leave the chip idle and each has
// enough to join for: 16.0 instead of 18.1 us for 192 heads of 3,000 tokens,
// 7.4 instead of 7.2 at 500; 26.6 instead of 25.0 for 384 heads of 3,000; dims of
// 128 take four up to 2,048 tokens (13.7 and 13.6 at 1,500, 25.4 and 23.0 at
// 4,096).
// What it does not see is which rows are long: from kKv8MostGroups work-groups
// on, and below 1,024 + 40 x work-groups tokens, a row that is far longer than
// the others is walked by one work-group a head. One of 8,000 tokens among 64
// rows, the others of 300: 29 us with 3 heads of 64, 53 with 8 of 128, where the
// long row alone takes 11 and 12; one of 32,000 among 64 rows of 8 heads 178,
// alone 20.
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
// work-groups enough: from 1.5 million (3 << 19) work-groups of one tile times
// tokens on, six thousand a CU, between 0.6 and 2 million where both sides were
// measured (1 and 2 tiles, us; 3 heads of 64 in FP32, then 8 of 128 in BF16):
// 17.3 and 18.0 for 512 rows at 1,500 tokens (0.6 million), 57 and 49 for 16 x
// 256 (4 million), 460 and 378 at 16,000; 37 and 34 for 512 rows at 1,500 (2
// million), 219 and 174 for 16 x 256. Up to 512 tokens there is no more than
// the one walk to share: 38.6 and 39.4 for prompts of 256 (2 million). dims of
// 256 have no registers for two.
// One wavefront a work-group saves the joining where there is work for the chip
// without dealing tokens: from 4,096 work-groups on (four a SIMD), from 512 on
// (two a CU) up to 512 tokens (16 steps), and where there are two steps to deal (1
// and 4 wavefronts, us): 15 and 18.5 for 16 x 256 rows of prompts, 39 and 71 for
// the wide heads, 174 and 201 for those at 1,500, but 149 and 107 for 16 x 256
// rows of 3 heads at 4,000 (1,200 work-groups).
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
// items * splits < 2 * kKv8MostGroups while there is more than one split, for
// any number of sequences (more of them are more items and fewer splits).
inline size_t kv8_workspace_floats(int rows, int sequences, int heads, int kv_heads, int dim, int max_length) {
    (void)sequences;
    const int64_t splits = kv8_ceil(max_length > 0 ? max_length : 1, kKv8LeastChunk);
    if (splits <= 1) return 0;
    const int64_t columns = 16 * 2;  // of the largest work-group
    const int64_t by_rows = (int64_t)rows * heads * splits, by_groups = 2ll * kKv8MostGroups * columns;
    return (size_t)(by_rows < by_groups ? by_rows : by_groups) * (dim + 2);
}

}  // namespace mphip
