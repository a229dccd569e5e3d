// The paged K/V cache in 8 bits: its device view, elements of the caller's
// types, the search for a work item's sequence and what the C entries share.
//
// Order of a (block, layer, KV head)'s bytes: tiles of 16 tokens, 16 dim
// bytes each, that are the A operands of v_mfma_f32_16x16x32_f16 as they lie.
// That operand's lane l = (c = l%16, g = l/16) holds row c at 8 consecutive
// steps of the contraction, and which dim or token a step is may be chosen as
// long as the other operand agrees:
// - keys (rows: the tile's tokens; contraction: dims) are
//   [dim/16][slot][16 dims]: load j of a lane is the 16 bytes at 1024 j + 16 l,
//   token c's dims 64j + 16g ..+15, two steps of 8;
// - values (rows: 16 dims; contraction: the 32 tokens of two tiles) are
//   [dim/64][slot/4][dim%16][dim%64/16][slot%4]: load j is the 16 bytes at
//   1024 j + 16 l, tokens 4g..+3 of dims 64j + 16n + c for n = 0..3. Tokens
//   4g..+3 of both tiles are the 8 steps of group g, which are the tokens whose
//   scores the lane got from the product with the keys: the probabilities
//   go from one product to the other in their registers.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include "../../../include/mp_hip.h"
#include "elements.h"
#include "entry.h"
#include "kv8_rules.h"
#include "lanes.h"

namespace mphip {

// One layer of a cache on the device.
struct Kv8Layer {
    uint8_t* keys;
    uint8_t* values;
    float2* scales;  // {keys, values}
    int blocks, layers, layer, kv_heads, dim;
    int page_shift;  // log2(block_tokens)
};

// Index of (block, head) in `scales`; its bytes follow from there.
__device__ __forceinline__ size_t kv8_head(const Kv8Layer& kv, int block, int head) {
    return ((size_t)block * kv.layers + kv.layer) * kv.kv_heads + head;
}

// ---- across a wavefront, without a way through LDS -----------------------------

// The sum over the lanes up to this one: within rows of 16, then the rows'
// totals (row_shr 1, 2, 4, 8; row_bcast 15 and 31).
__device__ __forceinline__ int wave_prefix(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}

// Packed rows of sequences (mp_hip.h).
struct Kv8Rows {
    const int32_t* tables;
    const int32_t* starts;
    const int32_t* used;
    int table_stride, sequences, rows;
};

// Where the work item of a wavefront lies: `index` of the sequence's items.
struct Kv8Item {
    int sequence, index, row0, count, used;
};

// Finds item `item` of all sequences' items, `items(count, used)` each, in
// their order; false behind the last one. Every wavefront searches for
// itself, 64 sequences at a step. Rows are clamped to 0..rows, whatever
// `starts` holds.
template <typename Items>
__device__ __forceinline__ bool kv8_find(const Kv8Rows& r, int item, Items items, Kv8Item* out) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < r.sequences; base += 64) {
        const int s = base + lane;
        int row0 = 0, count = 0, used = 0, n = 0;
        if (s < r.sequences) {
            const Kv8Span span = kv8_span(r.starts[s], r.starts[s + 1], r.rows);
            row0 = span.row0;
            count = span.count;
            used = r.used[s];
            if (count > 0) n = items(count, used);
        }
        const int sum = wave_prefix(n);
        const uint64_t past = __builtin_amdgcn_ballot_w64(sum > item - before);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int first = __builtin_amdgcn_readlane(sum - n, l);
            out->sequence = base + l;
            out->index = item - before - first;
            out->row0 = __builtin_amdgcn_readlane(row0, l);
            out->count = __builtin_amdgcn_readlane(count, l);
            out->used = __builtin_amdgcn_readlane(used, l);
            return out->index >= 0;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// ---- host side of the entries ---------------------------------------------

// Whether rows at `p` with this stride can be read and written by fours.
inline bool kv8_wide(const void* p, int64_t stride, int type) {
    const size_t four = 4 * element_bytes(type);
    return reinterpret_cast<uintptr_t>(p) % four == 0 && stride % 4 == 0;
}

// nullptr, or what is wrong with a cache and a layer of it.
inline const char* kv8_wrong_cache(const mp_kv8_cache* c, int layer) {
    if (!c || !c->keys || !c->values || !c->scales) return "8-bit cache: a pool is missing";
    if (reinterpret_cast<uintptr_t>(c->keys) % 16 || reinterpret_cast<uintptr_t>(c->values) % 16 ||
        reinterpret_cast<uintptr_t>(c->scales) % 8)
        return "8-bit cache: keys and values must be 16-byte aligned, scales 8-byte";
    if (c->block_tokens != 16 && c->block_tokens != 32 && c->block_tokens != 64 && c->block_tokens != 128)
        return "8-bit cache: block_tokens must be 16, 32, 64 or 128";
    if (c->dim != 64 && c->dim != 128 && c->dim != 256) return "8-bit cache: dim must be 64, 128 or 256";
    if (c->format != MP_KV8_INT8 && c->format != MP_KV8_E4M3) return "8-bit cache: unknown format";
    if (c->blocks < 1 || c->layers < 1 || c->kv_heads < 1 || c->kv_heads > kKv8MaxHeads)
        return "8-bit cache: blocks, layers and kv_heads must be positive (kv_heads at most 1024)";
    if ((int64_t)c->layers * c->kv_heads * c->block_tokens * c->dim >= (int64_t)1 << 31)
        return "8-bit cache: a block's keys must be smaller than 2 GiB";
    if ((int64_t)c->blocks * c->layers >= ((int64_t)1 << 29) / c->kv_heads)  // 512 GiB of keys at the least
        return "8-bit cache: blocks * layers * kv_heads must be smaller than 2^29";
    if (layer < 0 || layer >= c->layers) return "8-bit cache: no such layer";
    return nullptr;
}
inline const char* kv8_wrong_matrix(const void* p, int64_t stride, int64_t width, int type) {
    if (type != MP_TYPE_F32 && type != MP_TYPE_BF16 && type != MP_TYPE_F16) return "8-bit cache: unknown element type";
    if (!p || reinterpret_cast<uintptr_t>(p) % element_bytes(type)) return "8-bit cache: a row matrix is missing or misaligned";
    if (stride < width || stride > (int64_t)1 << 40) return "8-bit cache: a row stride is smaller than the row";
    return nullptr;
}
inline const char* kv8_wrong_rows(const int32_t* tables, int table_stride, int sequences, int rows) {
    if (!tables || reinterpret_cast<uintptr_t>(tables) % 4) return "8-bit cache: page tables are missing or misaligned";
    if (table_stride < 1) return "8-bit cache: table_stride must be positive";
    if (sequences < 0 || sequences > kKv8MaxRows || rows < 0 || rows > kKv8MaxRows)
        return "8-bit cache: sequences and rows must be 0 to 1,048,576";
    return nullptr;
}
inline bool kv8_bad_ints(const int32_t* p) { return !p || reinterpret_cast<uintptr_t>(p) % 4; }

inline Kv8Layer kv8_layer(const mp_kv8_cache& c, int layer) {
    return Kv8Layer{c.keys, c.values, reinterpret_cast<float2*>(c.scales), c.blocks, c.layers, layer, c.kv_heads,
                    c.dim, __builtin_ctz((unsigned)c.block_tokens)};
}

}  // namespace mphip
