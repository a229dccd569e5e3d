// Appending to and reading from the 8-bit paged K/V cache.
//
// A page's bytes share one scale, so the unit of an append is everything that
// a call writes to one (page, KV head, K or V): its new tokens' largest
// magnitude decides the scale, and where the scale grows the tokens held
// before are rounded again. One wavefront per 16-token tile of a unit, lane
// (c, g) = (l%16, l/16) owning the 16 bytes at 16 l of each 1 KB of the tile
// (kv8.h): for keys 16 dims of slot c, for values 4 slots of dims 16 apart.
// The maximum of a unit meets in LDS where its page has several tiles.
// Queries are rotated by wavefronts of their own, one row each.
//
// Arithmetic (every operation rounded on its own, so that the codes are a
// function of the inputs alone): a' = a cos - b sin, b' = b cos + a sin; code =
// rint(x * (1/s)), exact but for the rint since s is a power of two; E4M3
// codes by v_cvt_pk_fp8_f32 (nearest even).
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
    bool wide[2], q_wide;
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
    const int wave = threadIdx.x >> 6;
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

template <int DIM>
__device__ __forceinline__ void append_unit(const AppendArgs& a, uint32_t* amax_s) {
    constexpr int kLoads = DIM / 64;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const Unit u = unit_of(a.kv);
    Tile t = find_tile(a.kv, a.rows, u.item, u.tile);
    if (a.rope.half) t.last = min(t.last, a.rope.positions - t.pos0);
    const void* const src = u.kind ? a.x[1] : a.x[0];
    const int64_t stride = u.kind ? a.x_stride[1] : a.x_stride[0];
    const bool wide = u.kind ? a.wide[1] : a.wide[0];
    float x[kLoads][16];
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k) x[j][k] = 0.0f;
    uint32_t amax = 0;
    float held = 0.0f;
    size_t index = 0;
    if (t.block >= 0) {
        index = kv8_head(a.kv, t.block, u.head);
        if (t.kept) held = reinterpret_cast<const float*>(a.kv.scales + index)[u.kind];
        if (u.kind == 0) {
            if (c >= t.first && c < t.last) {
                const int64_t at = (t.row0 + c - t.first) * stride + (int64_t)u.head * DIM;
#pragma unroll
                for (int j = 0; j < kLoads; ++j)
                    load_rotated(src, a.type, wide, at, 64 * j + 16 * g, t.pos0 + c, a.rope, x[j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int slot = 4 * g + i;
                if (slot < t.first || slot >= t.last) continue;
                const int64_t at = (t.row0 + slot - t.first) * stride + (int64_t)u.head * DIM + c;
#pragma unroll
                for (int j = 0; j < kLoads; ++j)
#pragma unroll
                    for (int n = 0; n < 4; ++n) x[j][4 * n + i] = load_one(src, a.type, at + 64 * j + 16 * n);
            }
        }
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) amax = max(amax, __float_as_uint(x[j][k]) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
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
    uint8_t* const bytes = (u.kind ? a.kv.values : a.kv.keys) + index * ((size_t)DIM << a.kv.page_shift) +
                           u.tile * kTile * DIM + 16 * lane;
    if (u.tile == 0 && lane == 0) reinterpret_cast<float*>(a.kv.scales + index)[u.kind] = scale;
    if (!grew && (t.first >= kTile || t.last <= 0)) return;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        uint4* const at = reinterpret_cast<uint4*>(bytes + 1024 * j);
        uint32_t w[4];
        if (u.kind == 0) {
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

// Row `row`'s queries, rotated, by one wavefront.
__device__ __forceinline__ void rotate_row(const AppendArgs& a, int row) {
    const int lane = threadIdx.x & 63, dim = a.kv.dim, half = a.rope.half, turned = 2 * half;
    // The row's sequence: rows as items, behind those before starts[0].
    Kv8Item at;
    if (row >= a.rows.rows || !kv8_find(a.rows, row, [](int count, int) { return count; }, &at)) return;
    const int64_t r = at.row0 + at.index;
    const int64_t pos = (int64_t)at.used + at.index;
    const int64_t from = r * a.q_stride, to = r * a.q_out_stride;
    const bool bad = half && (at.used < 0 || pos >= a.rope.positions);
    const float* const cos = a.rope.cos + (bad ? 0 : pos) * half;
    const float* const sin = a.rope.sin + (bad ? 0 : pos) * half;
    const float poison = bad ? quiet_nan() : 0.0f;
    const int step = a.q_wide && half % 4 == 0 ? 4 : 1;
    // Per head: the pairs, `step` of them at a time (interleaved: two steps'
    // worth of elements), then the dims that pass.
    const int pairs = half / step, rest = (dim - turned) / step, per_head = pairs + rest;
    for (int i = lane; i < a.heads * per_head; i += 64) {
        const int head = i / per_head, p = i % per_head;
        const int64_t src = from + (int64_t)head * dim, dst = to + (int64_t)head * dim;
        if (p >= pairs) {
            const int d = turned + (p - pairs) * step;
            if (step == 4) {
                float x[4];
                load_row<4>(a.q, a.type, true, src + d, x);
                store_four(a.q_out, a.type, true, dst + d, bad ? poison : x[0], bad ? poison : x[1],
                           bad ? poison : x[2], bad ? poison : x[3]);
            } else {
                const float x = load_one(a.q, a.type, src + d);
                store_one(a.q_out, a.type, dst + d, bad ? poison : x);
            }
            continue;
        }
        const int k = p * step;  // first pair
        const int d0 = a.rope.interleaved ? 2 * k : k, d1 = a.rope.interleaved ? 2 * k + step : k + half;
        if (step == 4) {
            float u[4], v[4], lo[4], hi[4];
            load_row<4>(a.q, a.type, true, src + d0, u);
            load_row<4>(a.q, a.type, true, src + d1, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float c = bad ? poison : cos[k + e], s = bad ? poison : sin[k + e];
                const float x = a.rope.interleaved ? (e < 2 ? u[2 * (e & 1)] : v[2 * (e & 1)]) : u[e];
                const float y = a.rope.interleaved ? (e < 2 ? u[2 * (e & 1) + 1] : v[2 * (e & 1) + 1]) : v[e];
                lo[e] = x * c - y * s;
                hi[e] = y * c + x * s;
            }
            if (a.rope.interleaved) {
                store_four(a.q_out, a.type, true, dst + d0, lo[0], hi[0], lo[1], hi[1]);
                store_four(a.q_out, a.type, true, dst + d1, lo[2], hi[2], lo[3], hi[3]);
            } else {
                store_four(a.q_out, a.type, true, dst + d0, lo[0], lo[1], lo[2], lo[3]);
                store_four(a.q_out, a.type, true, dst + d1, hi[0], hi[1], hi[2], hi[3]);
            }
        } else {
            const float c = bad ? poison : cos[k], s = bad ? poison : sin[k];
            const float x = load_one(a.q, a.type, src + d0), y = load_one(a.q, a.type, src + d1);
            store_one(a.q_out, a.type, dst + d0, x * c - y * s);
            store_one(a.q_out, a.type, dst + d1, y * c + x * s);
        }
    }
}

template <int DIM>
__global__ __launch_bounds__(512) void kv8_append_kernel(AppendArgs a) {
    __shared__ uint32_t amax_s[8];
    if ((int)blockIdx.x < a.kv_groups) append_unit<DIM>(a, amax_s);
    else rotate_row(a, (blockIdx.x - a.kv_groups) * (blockDim.x >> 6) + (threadIdx.x >> 6));
}

struct ReadArgs {
    Kv8Layer kv;
    Kv8Rows rows;
    void* x[2];
    int64_t x_stride[2];
    int type, format;
    bool wide[2];
};

template <int DIM>
__global__ __launch_bounds__(512) void kv8_read_kernel(ReadArgs a) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const Unit u = unit_of(a.kv);
    const Tile t = find_tile(a.kv, a.rows, u.item, u.tile);
    if (!t.found || t.first >= kTile || t.last <= 0) return;
    const int first = max(t.first, 0);  // row0 is that of slot t.first
    void* const dst = u.kind ? a.x[1] : a.x[0];
    const int64_t stride = u.kind ? a.x_stride[1] : a.x_stride[0];
    const bool wide = u.kind ? a.wide[1] : a.wide[0];
    const size_t index = kv8_head(a.kv, max(t.block, 0), u.head);
    const float scale =
        t.block >= 0 ? reinterpret_cast<const float*>(a.kv.scales + index)[u.kind] : quiet_nan();
    const uint8_t* const bytes = (u.kind ? a.kv.values : a.kv.keys) + index * ((size_t)DIM << a.kv.page_shift) +
                                 u.tile * kTile * DIM + 16 * lane;
#pragma unroll
    for (int j = 0; j < DIM / 64; ++j) {
        const uint4 v = *reinterpret_cast<const uint4*>(bytes + 1024 * j);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if (u.kind == 0) {
            if (c < first || c >= t.last) continue;
            const int64_t at = (t.row0 + c - t.first) * stride + (int64_t)u.head * DIM + 64 * j + 16 * g;
#pragma unroll
            for (int n = 0; n < 4; ++n)
                store_four(dst, a.type, wide, at + 4 * n, decode(byte_of(w[n], 0), a.format) * scale,
                           decode(byte_of(w[n], 1), a.format) * scale, decode(byte_of(w[n], 2), a.format) * scale,
                           decode(byte_of(w[n], 3), a.format) * scale);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int slot = 4 * g + i;
                if (slot < first || slot >= t.last) continue;
                const int64_t at = (t.row0 + slot - t.first) * stride + (int64_t)u.head * DIM + 64 * j + c;
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    store_one(dst, a.type, at + 16 * n, decode(byte_of(w[n], i), a.format) * scale);
            }
        }
    }
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
        const int64_t kv_groups = (units + per_group - 1) / per_group, q_groups = q ? (rows + waves - 1) / waves : 0;
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
        a.wide[0] = kv8_wide(k, k_stride, type), a.wide[1] = kv8_wide(v, v_stride, type);
        a.q_wide = q && kv8_wide(q, q_stride, type) && kv8_wide(q_out, q_out_stride, type);
        a.kv_groups = (int)kv_groups;
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return kv8_done(device.status, "8-bit append: device of the stream");
        const dim3 grid((unsigned)(kv_groups + q_groups));
        if (cache->dim == 64) kv8_append_kernel<64><<<grid, threads, 0, s>>>(a);
        else if (cache->dim == 128) kv8_append_kernel<128><<<grid, threads, 0, s>>>(a);
        else kv8_append_kernel<256><<<grid, threads, 0, s>>>(a);
        return kv8_done(hipGetLastError(), "8-bit append launch");
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
        const int64_t groups = (units + per_group - 1) / per_group;
        if (groups > kMaxGroups) return too_large();
        ReadArgs a{};
        a.kv = kv8_layer(*cache, layer);
        a.rows = Kv8Rows{tables, starts, used, table_stride, sequences, rows};
        a.x[0] = k, a.x[1] = v;
        a.x_stride[0] = k_stride, a.x_stride[1] = v_stride;
        a.type = type, a.format = cache->format;
        a.wide[0] = kv8_wide(k, k_stride, type), a.wide[1] = kv8_wide(v, v_stride, type);
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return kv8_done(device.status, "8-bit read: device of the stream");
        const dim3 grid((unsigned)groups);
        if (cache->dim == 64) kv8_read_kernel<64><<<grid, threads, 0, s>>>(a);
        else if (cache->dim == 128) kv8_read_kernel<128><<<grid, threads, 0, s>>>(a);
        else kv8_read_kernel<256><<<grid, threads, 0, s>>>(a);
        return kv8_done(hipGetLastError(), "8-bit read launch");
    });
}
