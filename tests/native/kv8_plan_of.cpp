// Prints the plan of an attention call: decode (1 or 0), rows, sequences, KV
// heads, query heads each, dim, max_length.
#include "kv8_rules.h"

#include <cstdio>
#include <cstdlib>

int main(int argc, char** argv) {
    using namespace mphip;
    if (argc != 8) return 1;
    int n[8];
    for (int i = 1; i < 8; ++i) n[i] = std::atoi(argv[i]);
    const Kv8Plan p = n[1] ? kv8_decode_plan(n[2], n[4], n[6], n[7])
                           : kv8_prefill_plan(n[2], n[3], n[4], n[5], n[6], n[7]);
    std::printf("%d %d %d %d\n", p.column_tiles, p.waves, p.splits, p.chunk);
    return 0;
}
