// Appending to and reading from the 8-bit paged K/V cache.
//
// A page's bytes share one scale, so the unit of an append is everything that
// a call writes to one (page, KV head, K or V): its new tokens' largest
// magnitude decides the scale, and where the scale grows the tokens held
// before are rounded again. One wavefront per 16-token tile of a unit, lane
// (c, g) = (l%16, l/16) owning the 16 bytes at 16 l of each 1 KB of the tile
// (kv8.h): for keys 16 dims of slot c, for values 4 slots of dims 16 apart.
// The maximum of a unit meets in LDS where its page has several tiles.
// Queries are rotated by wavefronts of their own, one row each. Every
// wavefront finds its rows from the device's metadata by itself (kv8_find).
//
// Bound by memory: bytes in and out (378 MB in 101 us for 16.8k BF16 rows of 32
// query and 8 KV heads of 128, 3.7 TB/s, where a large copy reaches 4.7), and
// for few rows by the launch and one chain of loads: metadata, table, rows
// (4.4 us for one row of 9 and 3 heads of 64). The values' elements are read
// one by one, 16 lanes a run, since a lane's bytes are of dims 16 apart: the
// page's order suits the attention that reads it a thousand times.
//
// Arithmetic (every operation rounded on its own, so that the codes are a
// function of the inputs alone): a' = a cos - b sin, b' = b cos + a sin; code =
// rint(x * (1/s)), exact but for the rint since s is a power of two; E4M3
// codes by v_cvt_pk_fp8_f32 (nearest even).
#include <type_traits>

#include "kernels.h"
#include "kv8.h"

namespace mphip {
namespace {

constexpr int kThreads = 256;

struct RopeView {
    const float* cos;
    const float* sin;
    int positions, half;
    bool interleaved;
};

struct AppendArgs {
    Kv8Layer kv;
    Kv8Rows rows;
    RopeView rope;
    const void* x[2];  // k, v
    int64_t x_stride[2];
    const void* q;
    void* q_out;
    int64_t q_stride, q_out_stride;
    int heads, type, format;
    bool k_wide;  // the keys' rows by 16 bytes (8 of 16-bit types); values are taken one by one
    bool q_by_16;  // rows, strides and the turning dims are whole 16 bytes
    int kv_groups;  // work-groups before those of the queries
};

__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7FC00000u); }

// The smallest power of two s >= 2^-126 with amax <= top * s, top = 127 (INT8)
// or 448; NaN where amax (its bits) is an infinity or NaN.
__device__ __forceinline__ float scale_for(uint32_t amax, int format) {
    if (amax >= 0x7F800000u) return quiet_nan();
    // top = (1 + part) * 2^bits: 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8.
    const int bits = format == MP_KV8_INT8 ? 6 : 8;
    const uint32_t part = format == MP_KV8_INT8 ? 0x7E0000u : 0x600000u;
    const int e = (int)(amax >> 23) - bits + ((amax & 0x7FFFFFu) > part);  // biased
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

__device__ __forceinline__ uint32_t encode(float x, int format) {
    if (format == MP_KV8_INT8) return (uint32_t)((int)__builtin_rintf(x) + 128) & 0xFF;
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xFF;
}
__device__ __forceinline__ float decode(uint32_t byte, int format) {
    if (format == MP_KV8_INT8) return (float)((int)byte - 128);
    return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
}

// x[0..15] = dims d0..d0+15 of the head whose row starts at `at`, rotated to
// position `pos`.
__device__ __forceinline__ void load_rotated(const void* p, int type, bool wide, int64_t at, int d0, int pos,
                                             const RopeView& rope, float (&x)[16]) {
    load_row<16>(p, type, wide, at + d0, x);
    const int turned = 2 * rope.half;
    if (d0 >= turned) return;
    const float* cos = rope.cos + (size_t)pos * rope.half;
    const float* sin = rope.sin + (size_t)pos * rope.half;
    if (rope.interleaved) {
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
            const int d = d0 + k;
            if (d < turned) {
                const float c = cos[d >> 1], s = sin[d >> 1], a = x[k], b = x[k + 1];
                x[k] = a * c - b * s;
                x[k + 1] = b * c + a * s;
            }
        }
        return;
    }
    if (rope.half % 16 == 0) {  // the partners are 16 dims in a row, all on one side
        const bool low = d0 < rope.half;
        float y[16];
        load_row<16>(p, type, wide, at + (low ? d0 + rope.half : d0 - rope.half), y);
        const int i = low ? d0 : d0 - rope.half;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float own = x[k] * cos[i + k], other = y[k] * sin[i + k];
            x[k] = low ? own - other : own + other;
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int d = d0 + k;
        if (d < turned) {
            const bool low = d < rope.half;
            const int i = low ? d : d - rope.half;
            const float own = x[k] * cos[i];
            const float other = load_one(p, type, at + (low ? d + rope.half : i)) * sin[i];
            x[k] = low ? own - other : own + other;
        }
    }
}

// The bytes of one dword, low first.
__device__ __forceinline__ uint32_t byte_of(uint32_t w, int i) { return w >> (8 * i) & 0xFF; }

// A unit's tile: its page, and which of its slots are new.
struct Tile {
    bool found;       // there is such an item
    int block;        // -1: no valid page
    int first, last;  // the new slots [first, last), counted from the tile's slot 0
    int row0;         // row of slot `first`
    int pos0;         // position of the tile's slot 0
    bool kept;        // the page keeps slots before `first`
};

__device__ __forceinline__ Tile find_tile(const Kv8Layer& kv, const Kv8Rows& rows, int item, int tile) {
    const int shift = kv.page_shift;
    Tile t;
    Kv8Item at;
    t.found = kv8_find(rows, item, [=](int count, int used) { return kv8_pages(count, used, shift); }, &at);
    t.block = -1;
    t.first = t.last = t.row0 = t.pos0 = 0;
    t.kept = false;
    if (!t.found) return t;
    const Kv8Page page = kv8_page(at.count, at.used, at.index, shift);
    t.block = kv8_block(rows.tables + (size_t)at.sequence * rows.table_stride, rows.table_stride, page.page, kv.blocks);
    t.first = page.first - tile * kTile;
    t.last = page.last - tile * kTile;
    t.row0 = at.row0 + page.token;
    t.pos0 = (page.page << shift) + tile * kTile;
    t.kept = page.first > 0;
    return t;
}

// Units of a work-group of `blockDim.x` threads: (item, head, K or V), each
// the page's tiles in adjacent wavefronts.
struct Unit {
    int item, head, kind, tile, first_wave, tiles;
};
__device__ __forceinline__ Unit unit_of(const Kv8Layer& kv) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Unit u;
    u.tiles = 1 << (kv.page_shift - 4);
    const int unit = blockIdx.x * ((blockDim.x >> 6) / u.tiles) + wave / u.tiles;
    u.item = unit / (2 * kv.kv_heads);
    u.head = unit % (2 * kv.kv_heads) >> 1;
    u.kind = unit & 1;
    u.tile = wave % u.tiles;
    u.first_wave = wave - u.tile;
    return u;
}

// `t`: the wavefront's tile of unit `u`.
template <int DIM>
__device__ __forceinline__ void append_unit(const AppendArgs& a, const Unit& u, const Tile& t, uint32_t* amax_s) {
    constexpr int kLoads = DIM / 64;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int head = u.head, kind = u.kind;
    const void* const src = kind ? a.x[1] : a.x[0];
    const int64_t stride = kind ? a.x_stride[1] : a.x_stride[0];
    float x[kLoads][16];
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k) x[j][k] = 0.0f;
    // The rows do not wait for the table, only the held scale does.
    if (t.found && kind == 0) {
        if (c >= t.first && c < t.last) {
            const int64_t at = (t.row0 + c - t.first) * stride + (int64_t)head * DIM;
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
                load_rotated(src, a.type, a.k_wide, at, 64 * j + 16 * g, t.pos0 + c, a.rope, x[j]);
        }
    } else if (t.found) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int slot = 4 * g + i;
            if (slot < t.first || slot >= t.last) continue;
            const int64_t at = (t.row0 + slot - t.first) * stride + (int64_t)head * DIM + c;
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
#pragma unroll
                for (int n = 0; n < 4; ++n) x[j][4 * n + i] = load_one(src, a.type, at + 64 * j + 16 * n);
        }
    }
    const size_t index = kv8_head(a.kv, max(t.block, 0), head);
    const float held = t.kept && t.block >= 0 ? reinterpret_cast<const float*>(a.kv.scales + index)[kind] : 0.0f;
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k) amax = max(amax, __float_as_uint(x[j][k]) & 0x7FFFFFFFu);
    amax = wave_max(amax);
    if (u.tiles > 1) {  // the same in the whole launch
        if (lane == 0) amax_s[threadIdx.x >> 6] = amax;
        __syncthreads();  // also: every tile has read `held` before one changes it
        for (int w = 0; w < u.tiles; ++w) amax = max(amax, amax_s[u.first_wave + w]);
    }
    if (t.block < 0 || t.first >= t.last) return;  // no page, or nothing new before the rotation tables end
    const float wanted = scale_for(amax, a.format);
    const float scale = held >= wanted || held != held ? held : wanted;
    const bool grew = t.kept && scale != held && scale == scale;  // kept codes move
    const float inverse = 1.0f / scale, ratio = held * inverse;
    uint8_t* const bytes = (kind ? a.kv.values : a.kv.keys) + index * ((size_t)DIM << a.kv.page_shift) +
                           u.tile * kTile * DIM + 16 * lane;
    if (u.tile == 0 && lane == 0) reinterpret_cast<float*>(a.kv.scales + index)[kind] = scale;
    if (!grew && (t.first >= kTile || t.last <= 0)) return;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        uint4* const at = reinterpret_cast<uint4*>(bytes + 1024 * j);
        uint32_t w[4];
        if (kind == 0) {
            const bool fresh = c >= t.first && c < t.last;
            if (!fresh && !(grew && c < t.first)) continue;
            if (!fresh) {
                const uint4 was = *at;
                w[0] = was.x, w[1] = was.y, w[2] = was.z, w[3] = was.w;
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                uint32_t out = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    out |= encode(fresh ? x[j][4 * n + i] * inverse : decode(byte_of(w[n], i), a.format) * ratio,
                                  a.format)
                           << (8 * i);
                w[n] = out;
            }
        } else {
            if (4 * g >= t.last || (!grew && 4 * g + 4 <= t.first)) continue;
            const uint4 was = *at;
            w[0] = was.x, w[1] = was.y, w[2] = was.z, w[3] = was.w;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                uint32_t out = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int slot = 4 * g + i;
                    uint32_t b = byte_of(w[n], i);
                    if (slot < t.first) {
                        if (grew) b = encode(decode(b, a.format) * ratio, a.format);
                    } else if (slot < t.last) {
                        b = encode(x[j][4 * n + i] * inverse, a.format);
                    }
                    out |= b << (8 * i);
                }
                w[n] = out;
            }
        }
        *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// 16 bytes as E elements (4 FP32, 8 of a 16-bit type), and back.
template <int E>
__device__ __forceinline__ void unpack(uint4 v, int type, float (&x)[E]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint32_t two = w[i * 4 / E];
        if (E == 4) x[i] = __uint_as_float(two);
        else if (type == MP_TYPE_BF16) x[i] = __uint_as_float(i % 2 ? two & 0xFFFF0000u : two << 16);
        else x[i] = from_f16(i % 2 ? two >> 16 : two & 0xFFFF);
    }
}
template <int E>
__device__ __forceinline__ uint4 pack(const float (&x)[E], int type) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (E == 4) {
            w[i] = __float_as_uint(x[i]);
        } else {
            const float lo = x[2 * i % E], hi = x[(2 * i + 1) % E];
            w[i] = type == MP_TYPE_BF16 ? to_bf16(lo) | (uint32_t)to_bf16(hi) << 16
                                        : to_f16(lo) | (uint32_t)to_f16(hi) << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A row's queries by 16 bytes. A lane has one place in every head it sees:
// E pairs (i, i + half), or E elements of adjacent pairs, or E dims that pass.
// It reads its cosines and sines once, and four heads at a time.
template <int E>
__device__ __forceinline__ void rotate_wide(const AppendArgs& a, int64_t row, int64_t pos, bool bad) {
    const int lane = threadIdx.x & 63, dim = a.kv.dim, half = a.rope.half;
    const bool pairs_apart = !a.rope.interleaved;
    const int turning = pairs_apart ? half / E : 2 * half / E, places = turning + (dim - 2 * half) / E;
    const int lanes = places <= 8 ? 8 : places <= 16 ? 16 : places <= 32 ? 32 : 64;  // dim / E is at most 64
    const int place = lane % lanes, step = 64 / lanes;
    if (place >= places) return;
    const bool turns = place < turning, two = turns && pairs_apart;
    const int d0 = turns || !pairs_apart ? place * E : 2 * half + (place - turning) * E, d1 = two ? d0 + half : d0;
    const int64_t size = E == 4 ? 4 : 2;
    const char* const from = static_cast<const char*>(a.q) + row * a.q_stride * size;
    char* const to = static_cast<char*>(a.q_out) + row * a.q_out_stride * size;
    // Cosine and sine of the lane's pairs; a row without any is NaN, turned or not.
    float cos[E], sin[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int pair = two ? d0 + i : (d0 + i) / 2;
        cos[i] = turns && !bad ? a.rope.cos[pos * half + pair] : bad ? quiet_nan() : 1.0f;
        sin[i] = turns && !bad ? a.rope.sin[pos * half + pair] : 0.0f;
    }
    for (int h0 = lane / lanes; h0 < a.heads; h0 += 4 * step) {
        uint4 u[4], v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int h = h0 + k * step;
            if (h < a.heads) {
                u[k] = *reinterpret_cast<const uint4*>(from + ((int64_t)h * dim + d0) * size);
                if (two) v[k] = *reinterpret_cast<const uint4*>(from + ((int64_t)h * dim + d1) * size);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int h = h0 + k * step;
            if (h >= a.heads) continue;
            float x[E], y[E], lo[E], hi[E];
            unpack<E>(u[k], a.type, x);
            if (two) {
                unpack<E>(v[k], a.type, y);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    lo[i] = x[i] * cos[i] - y[i] * sin[i];
                    hi[i] = y[i] * cos[i] + x[i] * sin[i];
                }
                *reinterpret_cast<uint4*>(to + ((int64_t)h * dim + d1) * size) = pack<E>(hi, a.type);
            } else {
#pragma unroll
                for (int i = 0; i < E; i += 2) {
                    lo[i] = turns ? x[i] * cos[i] - x[i + 1] * sin[i] : bad ? cos[i] : x[i];
                    lo[i + 1] = turns ? x[i + 1] * cos[i] + x[i] * sin[i] : bad ? cos[i] : x[i + 1];
                }
            }
            *reinterpret_cast<uint4*>(to + ((int64_t)h * dim + d0) * size) = pack<E>(lo, a.type);
        }
    }
}

// The queries of row `r` at position `pos`, rotated, by one wavefront.
__device__ __forceinline__ void rotate_row(const AppendArgs& a, int64_t r, int64_t pos, bool bad) {
    const int lane = threadIdx.x & 63, dim = a.kv.dim, half = a.rope.half, turned = 2 * half;
    if (a.q_by_16) {
        if (a.type == MP_TYPE_F32) rotate_wide<4>(a, r, pos, bad);
        else rotate_wide<8>(a, r, pos, bad);
        return;
    }
    // One pair, or one dim that passes, at a time.
    const int64_t from = r * a.q_stride, to = r * a.q_out_stride;
    const int per_head = half + dim - turned;
    for (int i = lane; i < a.heads * per_head; i += 64) {
        const int head = i / per_head, p = i % per_head;
        const int64_t src = from + (int64_t)head * dim, dst = to + (int64_t)head * dim;
        if (p >= half) {
            const int d = turned + p - half;
            const float x = load_one(a.q, a.type, src + d);
            store_one(a.q_out, a.type, dst + d, bad ? quiet_nan() : x);
            continue;
        }
        const int d0 = a.rope.interleaved ? 2 * p : p, d1 = a.rope.interleaved ? 2 * p + 1 : p + half;
        const float c = bad ? quiet_nan() : a.rope.cos[pos * half + p], s = bad ? quiet_nan() : a.rope.sin[pos * half + p];
        const float x = load_one(a.q, a.type, src + d0), y = load_one(a.q, a.type, src + d1);
        store_one(a.q_out, a.type, dst + d0, x * c - y * s);
        store_one(a.q_out, a.type, dst + d1, y * c + x * s);
    }
}

// The query row of a wavefront of work-group `group`; rows as items, behind
// those before starts[0].
__device__ __forceinline__ void rotate_rows(const AppendArgs& a, int group) {
    Kv8Item at;
    const int row = group * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= a.rows.rows || !kv8_find(a.rows, row, [](int count, int) { return count; }, &at)) return;
    const int64_t pos = (int64_t)at.used + at.index;
    rotate_row(a, at.row0 + at.index, pos, a.rope.half && (at.used < 0 || pos >= a.rope.positions));
}

// Type and format are constants of a kernel: loads of elements under a branch
// on either are each waited for before the next (237 us instead of 67 for the
// keys and values of 16.8k BF16 rows of 8 heads of 128). The queries' rows go
// beside the keys and values in one launch: 136 instead of 147 us in two for
// those rows and their 32 query heads, read back, and 8.0 instead of 10.5 for
// one row of 9 heads of 64. What it waits for is memory: with registers for six
// wavefronts a SIMD instead of four 127 us instead of 136, for eight (spilled)
// 160.
template <int TYPE, int FORMAT, int DIM>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(DIM <= 128 ? 6 : 4))) void kv8_append_kernel(
    AppendArgs a) {
    __shared__ uint32_t amax_s[8];
    a.type = TYPE;
    a.format = FORMAT;
    if ((int)blockIdx.x < a.kv_groups) {
        const Unit u = unit_of(a.kv);
        Tile t = find_tile(a.kv, a.rows, u.item, u.tile);
        if (a.rope.half) t.last = min(t.last, a.rope.positions - t.pos0);
        append_unit<DIM>(a, u, t, amax_s);
    } else {
        rotate_rows(a, blockIdx.x - a.kv_groups);
    }
}

struct ReadArgs {
    Kv8Layer kv;
    Kv8Rows rows;
    void* x[2];
    int64_t x_stride[2];
    int type, format;
    bool k_wide;
};

template <int TYPE, int FORMAT, int DIM>
__global__ __launch_bounds__(512) void kv8_read_kernel(ReadArgs a) {
    a.type = TYPE;
    a.format = FORMAT;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const Unit u = unit_of(a.kv);
    const Tile t = find_tile(a.kv, a.rows, u.item, u.tile);
    if (!t.found || t.first >= kTile || t.last <= 0) return;
    const int first = max(t.first, 0);  // row0 is that of slot t.first
    const int head = u.head, kind = u.kind;
    void* const dst = kind ? a.x[1] : a.x[0];
    const int64_t stride = kind ? a.x_stride[1] : a.x_stride[0];
    const size_t index = kv8_head(a.kv, max(t.block, 0), head);
    const float scale =
        t.block >= 0 ? reinterpret_cast<const float*>(a.kv.scales + index)[kind] : quiet_nan();
    const uint8_t* const bytes = (kind ? a.kv.values : a.kv.keys) + index * ((size_t)DIM << a.kv.page_shift) +
                                 u.tile * kTile * DIM + 16 * lane;
#pragma unroll
    for (int j = 0; j < DIM / 64; ++j) {
        const uint4 v = *reinterpret_cast<const uint4*>(bytes + 1024 * j);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if (kind == 0) {
            if (c < first || c >= t.last) continue;
            const int64_t at = (t.row0 + c - t.first) * stride + (int64_t)head * DIM + 64 * j + 16 * g;
#pragma unroll
            for (int n = 0; n < 4; ++n)
                store_four(dst, a.type, a.k_wide, at + 4 * n, decode(byte_of(w[n], 0), a.format) * scale,
                           decode(byte_of(w[n], 1), a.format) * scale, decode(byte_of(w[n], 2), a.format) * scale,
                           decode(byte_of(w[n], 3), a.format) * scale);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int slot = 4 * g + i;
                if (slot < first || slot >= t.last) continue;
                const int64_t at = (t.row0 + slot - t.first) * stride + (int64_t)head * DIM + 64 * j + c;
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    store_one(dst, a.type, at + 16 * n, decode(byte_of(w[n], i), a.format) * scale);
            }
        }
    }
}

// Calls f(type, format, dim) with the call's as constants.
template <typename F, int TYPE, int FORMAT>
hipError_t with_dim(int dim, const F& f) {
    using Type = std::integral_constant<int, TYPE>;
    using Format = std::integral_constant<int, FORMAT>;
    if (dim == 64) return f(Type(), Format(), std::integral_constant<int, 64>());
    if (dim == 128) return f(Type(), Format(), std::integral_constant<int, 128>());
    return f(Type(), Format(), std::integral_constant<int, 256>());
}
template <typename F, int TYPE>
hipError_t with_format(int format, int dim, const F& f) {
    return format == MP_KV8_INT8 ? with_dim<F, TYPE, MP_KV8_INT8>(dim, f) : with_dim<F, TYPE, MP_KV8_E4M3>(dim, f);
}
template <typename F>
hipError_t with_constants(int type, int format, int dim, const F& f) {
    if (type == MP_TYPE_F32) return with_format<F, MP_TYPE_F32>(format, dim, f);
    if (type == MP_TYPE_BF16) return with_format<F, MP_TYPE_BF16>(format, dim, f);
    return with_format<F, MP_TYPE_F16>(format, dim, f);
}

int threads_for(int bt) { return bt == 128 ? 512 : kThreads; }

int too_large() { return kv8_refuse("8-bit cache: rows times heads are too many for one call"); }
constexpr int64_t kMaxGroups = 1 << 22;  // 2^31 threads of 512

}  // namespace
}  // namespace mphip

extern "C" int mp_hip_kv8_append(const mp_kv8_cache* cache, int32_t layer, const void* k, int64_t k_stride,
                                 const void* v, int64_t v_stride, const void* q, int64_t q_stride, void* q_out,
                                 int64_t q_out_stride, int32_t heads, int32_t type, const mp_rope* rope,
                                 const int32_t* tables, int32_t table_stride, const int32_t* starts,
                                 const int32_t* used, int32_t sequences, int32_t rows, void* stream) {
    using namespace mphip;
    return kv8_entry([&]() -> int {
        const char* wrong = kv8_wrong_cache(cache, layer);
        if (!wrong) wrong = kv8_wrong_rows(tables, table_stride, sequences, rows);
        if (wrong) return kv8_refuse(wrong);
        const int64_t width = (int64_t)cache->kv_heads * cache->dim;
        wrong = kv8_wrong_matrix(k, k_stride, width, type);
        if (!wrong) wrong = kv8_wrong_matrix(v, v_stride, width, type);
        if (wrong) return kv8_refuse(wrong);
        if (kv8_bad_ints(starts) || kv8_bad_ints(used))
            return kv8_refuse("8-bit cache: starts or used are missing or misaligned");
        if (q) {
            if (heads < 1 || heads > kKv8MaxHeads) return kv8_refuse("8-bit cache: heads must be 1 to 1,024");
            wrong = kv8_wrong_matrix(q, q_stride, (int64_t)heads * cache->dim, type);
            if (!wrong) wrong = kv8_wrong_matrix(q_out, q_out_stride, (int64_t)heads * cache->dim, type);
            if (wrong) return kv8_refuse(wrong);
            if (q == q_out && q_stride != q_out_stride)
                return kv8_refuse("8-bit cache: queries rotated in place need one stride");
        }
        RopeView view{nullptr, nullptr, 0, 0, false};
        if (rope && rope->dims != 0) {
            if (rope->dims < 0 || rope->dims % 2 || rope->dims > cache->dim)
                return kv8_refuse("8-bit cache: rotated dims must be even and at most dim");
            if (!rope->cos || !rope->sin || reinterpret_cast<uintptr_t>(rope->cos) % 4 ||
                reinterpret_cast<uintptr_t>(rope->sin) % 4 || rope->positions < 1)
                return kv8_refuse("8-bit cache: rotation tables are missing, misaligned or empty");
            view = RopeView{rope->cos, rope->sin, rope->positions, rope->dims / 2, rope->interleaved != 0};
        }
        if (rows == 0 || sequences == 0) return MP_OK;
        const int bt = cache->block_tokens, threads = threads_for(bt), waves = threads / 64;
        const int64_t units = kv8_most_pages(rows, sequences, bt) * cache->kv_heads * 2, per_group = waves / (bt / kTile);
        const int64_t kv_groups = kv8_ceil(units, per_group), q_groups = q ? kv8_ceil(rows, waves) : 0;
        if (kv_groups + q_groups > kMaxGroups) return too_large();
        AppendArgs a{};
        a.kv = kv8_layer(*cache, layer);
        a.rows = Kv8Rows{tables, starts, used, table_stride, sequences, rows};
        a.rope = view;
        a.x[0] = k, a.x[1] = v;
        a.x_stride[0] = k_stride, a.x_stride[1] = v_stride;
        a.q = q, a.q_out = q_out;
        a.q_stride = q_stride, a.q_out_stride = q_out_stride;
        a.heads = heads, a.type = type, a.format = cache->format;
        a.k_wide = kv8_wide(k, k_stride, type);
        const int per16 = 16 / (int)kv8_element(type);
        a.q_by_16 = q && reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(q_out) % 16 == 0 &&
                    q_stride % per16 == 0 && q_out_stride % per16 == 0 &&
                    (view.interleaved ? 2 * view.half : view.half) % per16 == 0;
        a.kv_groups = (int)kv_groups;
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return kv8_done(device.status, "8-bit append: device of the stream");
        const hipError_t e = with_constants(type, cache->format, cache->dim, [&](auto t, auto f, auto d) {
            kv8_append_kernel<decltype(t)::value, decltype(f)::value, decltype(d)::value>
                <<<(unsigned)(kv_groups + q_groups), threads, 0, s>>>(a);
            return hipGetLastError();
        });
        return kv8_done(e, "8-bit append launch");
    });
}

extern "C" int mp_hip_kv8_read(const mp_kv8_cache* cache, int32_t layer, const int32_t* tables, int32_t table_stride,
                               const int32_t* starts, const int32_t* used, int32_t sequences, int32_t rows,
                               int32_t type, void* k, int64_t k_stride, void* v, int64_t v_stride, void* stream) {
    using namespace mphip;
    return kv8_entry([&]() -> int {
        const char* wrong = kv8_wrong_cache(cache, layer);
        if (!wrong) wrong = kv8_wrong_rows(tables, table_stride, sequences, rows);
        if (wrong) return kv8_refuse(wrong);
        const int64_t width = (int64_t)cache->kv_heads * cache->dim;
        wrong = kv8_wrong_matrix(k, k_stride, width, type);
        if (!wrong) wrong = kv8_wrong_matrix(v, v_stride, width, type);
        if (wrong) return kv8_refuse(wrong);
        if (kv8_bad_ints(starts) || kv8_bad_ints(used))
            return kv8_refuse("8-bit cache: starts or used are missing or misaligned");
        if (rows == 0 || sequences == 0) return MP_OK;
        const int bt = cache->block_tokens, threads = threads_for(bt), waves = threads / 64;
        const int64_t units = kv8_most_pages(rows, sequences, bt) * cache->kv_heads * 2, per_group = waves / (bt / kTile);
        const int64_t groups = kv8_ceil(units, per_group);
        if (groups > kMaxGroups) return too_large();
        ReadArgs a{};
        a.kv = kv8_layer(*cache, layer);
        a.rows = Kv8Rows{tables, starts, used, table_stride, sequences, rows};
        a.x[0] = k, a.x[1] = v;
        a.x_stride[0] = k_stride, a.x_stride[1] = v_stride;
        a.type = type, a.format = cache->format;
        a.k_wide = kv8_wide(k, k_stride, type);
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return kv8_done(device.status, "8-bit read: device of the stream");
        const hipError_t e = with_constants(type, cache->format, cache->dim, [&](auto t, auto f, auto d) {
            kv8_read_kernel<decltype(t)::value, decltype(f)::value, decltype(d)::value>
                <<<(unsigned)groups, threads, 0, s>>>(a);
            return hipGetLastError();
        });
        return kv8_done(e, "8-bit read launch");
    });
}
