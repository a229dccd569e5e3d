// kv8_rules.h: which rows, pages and slots a call on the 8-bit cache touches,
// for metadata of every kind, and how its attention is divided.
#include "kv8_rules.h"

#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

using namespace mphip;

#define REQUIRE(x)                                                         \
    do {                                                                   \
        if (!(x)) {                                                        \
            std::fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #x);   \
            std::exit(1);                                                  \
        }                                                                  \
    } while (0)

namespace {

// Every row of well-formed metadata is one slot of one page item, in order;
// the items are no more than the launch has.
void covers_every_row_once() {
    std::mt19937 rng(1);
    for (int trial = 0; trial < 3000; ++trial) {
        const int shift = 4 + (int)(rng() % 4), bt = 1 << shift, n = 1 + (int)(rng() % 6);
        std::vector<int> starts = {(int)(rng() % 3)}, used;
        for (int s = 0; s < n; ++s) {
            starts.push_back(starts.back() + (int)(rng() % (rng() % 3 ? 4 : 300)));
            used.push_back((int)(rng() % (rng() % 2 ? 40 : 100000)));
        }
        const int rows = starts.back() + (int)(rng() % 3);
        std::vector<int> seen(rows, 0);
        int64_t items = 0;
        for (int s = 0; s < n; ++s) {
            const Kv8Span span = kv8_span(starts[s], starts[s + 1], rows);
            REQUIRE(span.row0 == starts[s] && span.count == starts[s + 1] - starts[s]);
            const int pages = span.count ? kv8_pages(span.count, used[s], shift) : 0;
            items += pages;
            for (int i = 0; i < pages; ++i) {
                const Kv8Page p = kv8_page(span.count, used[s], i, shift);
                REQUIRE(p.first >= 0 && p.first < p.last && p.last <= bt);
                REQUIRE(i == 0 || p.first == 0);
                for (int slot = p.first; slot < p.last; ++slot) {
                    const int token = p.token + slot - p.first;
                    REQUIRE(token >= 0 && token < span.count);
                    REQUIRE((p.page << shift) + slot == used[s] + token);
                    ++seen[span.row0 + token];
                }
            }
        }
        for (int r = 0; r < rows; ++r) REQUIRE(seen[r] == (r >= starts[0] && r < starts[n]));
        REQUIRE(items <= kv8_most_pages(rows, n, bt));
    }
}

// Whatever the arrays hold, rows stay inside the matrices, slots inside pages
// and pages inside the table and the pool.
void stays_inside() {
    std::mt19937 rng(2);
    const int extremes[] = {0, 1, -1, 15, 16, 17, 100, 1 << 20, 1 << 30, (1 << 30) + 1, 2147483647, -2147483647 - 1};
    const auto any = [&] { return rng() % 2 ? extremes[rng() % 12] : (int)rng(); };
    for (int trial = 0; trial < 200000; ++trial) {
        const int rows = (int)(rng() % 200), shift = 4 + (int)(rng() % 4);
        const Kv8Span span = kv8_span(any(), any(), rows);
        REQUIRE(span.row0 >= 0 && span.count >= 0 && span.row0 + span.count <= rows);
        if (!span.count) continue;
        const int used = any(), pages = kv8_pages(span.count, used, shift);
        REQUIRE(pages >= 0 && pages <= span.count + 1);
        for (int i = 0; i < pages; ++i) {
            const Kv8Page p = kv8_page(span.count, used, i, shift);
            REQUIRE(p.page >= 0 && p.first >= 0 && p.first < p.last && p.last <= 1 << shift);
            REQUIRE(p.token >= 0 && p.token + (p.last - p.first) <= span.count);
        }
    }
    const int32_t table[] = {0, 4, 5, -1, 2147483647, -2147483647 - 1, 3};
    const int want[] = {0, 4, -1, -1, -1, -1, 3};
    for (int page = 0; page < 7; ++page) REQUIRE(kv8_block(table, 7, page, 5) == want[page]);
    for (int page : {-1, 7, 8, 2147483647}) REQUIRE(kv8_block(table, 7, page, 5) == -1);
}

// The chunks of a plan cover the longest row, its launch fits the grid's
// limits, and a workspace for the largest sizes serves every smaller call.
void plans() {
    std::mt19937 rng(3);
    const auto upto = [&](int most) {  // spread over the logarithm
        int v = 1;
        while (v < most && rng() % 3) v = v * 2 + (int)(rng() % 2);
        return v < most ? v : most;
    };
    for (int trial = 0; trial < 100000; ++trial) {
        const int group = 1 + (int)(rng() % 16), kv_heads = upto(64), dim = 64 << rng() % 3;
        const int rows = upto(1 << 20), sequences = upto(rows), length = (int)(rng() % 8) ? upto(1 << 22) : 0;
        const int heads = group * kv_heads;
        const Kv8Plan d = kv8_decode_plan(rows, kv_heads, dim, length);
        const Kv8Plan f = kv8_prefill_plan(rows, sequences, kv_heads, group, dim, length);
        for (const Kv8Plan& p : {d, f}) {
            REQUIRE(p.column_tiles == 1 || (p.column_tiles == 2 && dim <= 128));
            REQUIRE((p.waves == 1 || p.waves == 4 || p.waves == kKv8MostWaves) && p.splits >= 1 && p.splits <= 65535);
            REQUIRE(p.chunk % kKv8Pair == 0 && (int64_t)p.chunk * p.splits >= length);
        }
        REQUIRE(d.column_tiles == 1);
        const int64_t items = kv8_items(rows, sequences, group, f.column_tiles);
        if ((int64_t)rows * heads <= kKv8MostColumns)
            REQUIRE(items * kv_heads * 64 * f.waves < 1ll << 32 && (int64_t)rows * kv_heads * 64 * d.waves < 1ll << 32);
        // Smaller calls on the same workspace.
        const size_t space = kv8_workspace_floats(rows, sequences, heads, kv_heads, dim, length);
        const int fewer = 1 + (int)(rng() % rows), shorter = length ? (int)(rng() % (length + 1)) : 0;
        const int some = 1 + (int)(rng() % (fewer < sequences ? fewer : sequences));
        for (int r : {rows, fewer})
            for (int n : {length, shorter}) {
                REQUIRE(kv8_partial_floats(kv8_decode_plan(r, kv_heads, dim, n), r, heads, dim) <= space);
                REQUIRE(kv8_partial_floats(kv8_prefill_plan(r, some, kv_heads, group, dim, n), r, heads, dim) <= space);
            }
    }
}

}  // namespace

int main() {
    covers_every_row_once();
    stays_inside();
    plans();
    std::puts("ok");
    return 0;
}
