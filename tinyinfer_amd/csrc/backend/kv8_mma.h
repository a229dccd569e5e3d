// What the attention kernels of the 8-bit cache share: arguments, operands of
// the matrix cores from bytes and queries, and where tiles lie.
#pragma once
#include "kv8.h"

namespace mphip {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

enum Kv8Mode { kPacked, kTwo, kOne };

constexpr float kShift = 11.0f;  // probabilities are held times 2^11 ...
constexpr float kRaise = 15.0f;  // ... and below 2^15: past it the reference is raised

struct Kv8Attention {
    Kv8Layer kv;
    Kv8Rows rows;          // decode: starts null, used = lengths
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int heads, group, type, max_length, chunk, splits;
    float scale;           // times log2(e)
    bool q_wide, out_wide;
    float* partial_out;    // [row][head][split][dim]
    float2* partial_ml;    // [row][head][split]: reference (log2), sum
};

__device__ __forceinline__ float infinity() { return __builtin_inff(); }
__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7FC00000u); }

// v plus its value 8 columns on.
__device__ __forceinline__ float add_across(float v) {
    return v + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, true));
}

// Four codes times a power of two as FP16. INT8: a byte b under 0x64 is the
// FP16 number 1024 + b; less 1152 it is the code, exactly. E4M3: the
// conversion takes the power of two.
template <int FORMAT>
struct Convert;
template <>
struct Convert<MP_KV8_INT8> {
    h2 times, less;
    explicit __device__ __forceinline__ Convert(float power) {
        const _Float16 p = (_Float16)power;
        times = h2{p, p};
        less = h2{(_Float16)-1152, (_Float16)-1152} * times;
    }
    __device__ __forceinline__ void operator()(uint32_t w, h2* lo, h2* hi) const {
        const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u));
        const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u));
        *lo = __builtin_elementwise_fma(a, times, less);
        *hi = __builtin_elementwise_fma(b, times, less);
    }
    // Power 1.
    static __device__ __forceinline__ void plain(uint32_t w, h2* lo, h2* hi) {
        const h2 less = {(_Float16)-1152, (_Float16)-1152};
        *lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + less;
        *hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + less;
    }
};
template <>
struct Convert<MP_KV8_E4M3> {
    float power;
    explicit __device__ __forceinline__ Convert(float p) : power(p) {}
    __device__ __forceinline__ void operator()(uint32_t w, h2* lo, h2* hi) const {
        *lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, power, false);
        *hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, power, true);
    }
    static __device__ __forceinline__ void plain(uint32_t w, h2* lo, h2* hi) {
        *lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        *hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    }
};

union Half8 {
    h8 all;
    h2 two[4];
    _Float16 one[8];
};

// A load through the scalar cache, at byte `offset` of an array that no kernel
// beside this one writes; uniform over the wavefront.
__device__ __forceinline__ int scalar_int(const void* p, uint32_t offset) {
    return *(const __attribute__((address_space(4))) int32_t*)((uintptr_t)p + offset);
}
// In asm, as are the two below (the compiler makes two or three instructions of
// them, 32 more a step). It puts no waits around asm: what these read comes
// from ordinary vector instructions, exponentials by way of the conversion to
// `half`, never straight from an exponential or a matrix instruction.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// x - (float)half of the low or high half, times `factor`: factor * half + x.
__device__ __forceinline__ float mix_low(h2 half, float factor, float x) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(half), "v"(factor), "v"(x));
    return r;
}
__device__ __forceinline__ float mix_high(h2 half, float factor, float x) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(half), "v"(factor), "v"(x));
    return r;
}

// The queries of a lane's columns as they are in memory: for column tile t
// and j the 16 elements of dims 64j + 16g .. +15 (the last two registers are
// unused for 16-bit types). All loads before any use.
template <int DIM, int NT>
__device__ __forceinline__ void load_queries(const Kv8Attention& a, bool f32, const int64_t (&at)[NT], int g,
                                             u4 (&raw)[NT][DIM / 64][4]) {
    const auto each = [&](auto get) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < DIM / 64; ++j) get(raw[t][j], at[t] + 64 * j + 16 * g);
    };
    if (f32) {
        const float* const from = static_cast<const float*>(a.q);
        if (a.q_wide)
            each([&](u4 (&to)[4], int64_t i) {
#pragma unroll
                for (int k = 0; k < 4; ++k) to[k] = *reinterpret_cast<const u4*>(from + i + 4 * k);
            });
        else
            each([&](u4 (&to)[4], int64_t i) {
#pragma unroll
                for (int k = 0; k < 16; ++k) to[k / 4][k % 4] = __float_as_uint(from[i + k]);
            });
    } else {
        typedef u4 u4_by_8 __attribute__((aligned(8)));
        const uint16_t* const from = static_cast<const uint16_t*>(a.q);
        if (a.q_wide)
            each([&](u4 (&to)[4], int64_t i) {
                to[0] = *reinterpret_cast<const u4_by_8*>(from + i);
                to[1] = *reinterpret_cast<const u4_by_8*>(from + i + 8);
            });
        else
            each([&](u4 (&to)[4], int64_t i) {
#pragma unroll
                for (int k = 0; k < 16; k += 2)
                    to[k / 8][k / 2 % 4] = from[i + k] | (uint32_t)from[i + k + 1] << 16;
            });
    }
}

// Those queries as operands: part, column tile, step 2j + h of dims 64j + 16g
// + 8h .. +7; and the factor of a column's scores, the softmax scale over the
// query's power of two (NaN for a row that is not finite, longer than the
// caller allowed for or with pages that the table has not).
template <int DIM, int NT, int MODE, int PARTS>
__device__ __forceinline__ void split_queries(const Kv8Attention& a, bool f32, const u4 (&raw)[NT][DIM / 64][4],
                                              const int (&qpos)[NT], int c, Half8 (&q)[PARTS][NT][DIM / 32],
                                              float (&factor)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float x[DIM / 64][16];
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < DIM / 64; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t two = raw[t][j][i / 8][i / 2 % 4];
                x[j][i] = f32                      ? __uint_as_float(raw[t][j][i / 4][i % 4])
                          : a.type == MP_TYPE_BF16 ? __uint_as_float(i % 2 ? two & 0xFFFF0000u : two << 16)
                                                   : from_f16(i % 2 ? two >> 16 : two & 0xFFFF);
                amax = max(amax, __float_as_uint(x[j][i]) & 0x7FFFFFFFu);
            }
        amax = column_max(amax);
        const int power = min(127 + 14 - (int)(amax >> 23), 126);  // at least -113
        const float up = __uint_as_float((uint32_t)(127 + power) << 23);
        const bool lost = amax >= 0x7F800000u || qpos[t] >= a.max_length ||
                          qpos[t] >> a.kv.page_shift >= a.rows.table_stride;
        factor[t] = lost ? quiet_nan() : a.scale * __uint_as_float((uint32_t)(127 - power) << 23);
#pragma unroll
        for (int j = 0; j < DIM / 64; ++j)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float u = x[j][i] * up, v = x[j][i + 1] * up;
                const h2 high = {(_Float16)u, (_Float16)v};
                const h2 low = {(_Float16)(u - (float)high[0]), (_Float16)(v - (float)high[1])};
                h2& first = q[0][t][2 * j + i / 8].two[i % 8 / 2];
                if (MODE == kPacked) first = c & 8 ? low : high;
                else first = high;
                if (MODE == kTwo) q[PARTS - 1][t][2 * j + i / 8].two[i % 8 / 2] = low;
            }
    }
}

// Where tiles lie and their scales, worked out by the lanes. A step has EACH
// tiles, tile0 + n * stride .. of step n; lane l holds tile l % EACH of the
// steps whose number is l / EACH modulo kSteps, and a step reads what it needs
// from a lane. Every kSteps/2 steps half the lanes go on to the steps kSteps
// on, whose scales were fetched half a round and whose table entries a round
// before. A page that is none reads page 0 and has NaN scales; a tile behind
// the last reads page 0 and has scales 0.
template <int DIM, int EACH>
struct Kv8Tiles {
    static constexpr int kSteps = 64 / EACH, kHalf = kSteps / 2;
    struct Found {
        uint64_t base;
        float2 bits;
        uint32_t none, present;  // bits of NaN or 0; all bits or 0
    };
    const int32_t* table;
    const float2* scales;
    uint32_t block_scales, block_bytes, head_bytes;
    int stride, blocks, shift, tile0, step, tile_end, steps, lane;
    uint32_t at_low, at_high, at_k, at_v;  // this lane's tile: where, and its scales' bits
    Found soon;                            // of the steps kSteps on
    int found;                             // their successors' table entry

    __device__ __forceinline__ int tile_of(int n) const { return tile0 + n * step + lane % EACH; }
    __device__ __forceinline__ int find_block(int n) const {
        return table[min(tile_of(n) >> (shift - 4), stride - 1)];
    }
    __device__ __forceinline__ Found find(int n, int block) const {
        const int tile = tile_of(n);
        const bool is = (unsigned)block < (unsigned)blocks;
        const uint32_t at = is && tile < tile_end ? block : 0;
        Found t;
        t.none = is ? 0u : 0x7FC00000u;
        t.present = tile < tile_end ? ~0u : 0u;
        t.base = (uint64_t)at * block_bytes + (head_bytes + (tile & ((1 << (shift - 4)) - 1)) * (kTile * DIM));
        t.bits = scales[(size_t)at * block_scales];
        return t;
    }
    __device__ __forceinline__ void take_places(const Found& t) {
        at_low = (uint32_t)t.base;
        at_high = (uint32_t)(t.base >> 32);
    }
    __device__ __forceinline__ void take_scales(const Found& t) {
        at_k = (__float_as_uint(t.bits.x) | t.none) & t.present;
        at_v = (__float_as_uint(t.bits.y) | t.none) & t.present;
    }
    // The table's entries of the first steps.
    __device__ __forceinline__ int begin(const Kv8Attention& a, int sequence, int head, int first_tile, int tiles_on,
                                         int l) {
        table = a.rows.tables + (size_t)sequence * a.rows.table_stride;
        stride = a.rows.table_stride;
        blocks = a.kv.blocks;
        shift = a.kv.page_shift;
        block_scales = (uint32_t)a.kv.layers * a.kv.kv_heads;  // heads of a block
        block_bytes = block_scales * DIM << shift;
        head_bytes = (uint32_t)(a.kv.layer * a.kv.kv_heads + head) * DIM << shift;
        scales = a.kv.scales + (a.kv.layer * a.kv.kv_heads + head);
        tile0 = first_tile;
        step = tiles_on;
        lane = l;
        return find_block(lane / EACH);
    }
    // The tiles end at `end`, and this wavefront has `count` steps.
    __device__ __forceinline__ void until(int end, int count) {
        tile_end = end;
        steps = count;
    }
    // After the first steps' tiles have been taken.
    __device__ __forceinline__ void look_ahead() {
        if (steps <= kSteps) return;
        soon = find(kSteps + lane / EACH % kHalf, find_block(kSteps + lane / EACH % kHalf));
        found = find_block(kSteps + kHalf + lane / EACH % kHalf);
    }
    // Before step n is looked for.
    __device__ __forceinline__ void go_on(int n) {
        if (n % kHalf || n < kSteps || n >= steps) return;
        if (lane / (32) == (n / kHalf) % 2) {
            take_places(soon);
            take_scales(soon);
        }
        soon = find(n + kHalf + lane / EACH % kHalf, found);
        found = find_block(n + kSteps + lane / EACH % kHalf);
    }
    __device__ __forceinline__ uint64_t base(int n, int tile) const {
        const int from = EACH * (n % kSteps) + tile;
        return (uint32_t)__builtin_amdgcn_readlane(at_low, from) |
               (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_high, from) << 32;
    }
    __device__ __forceinline__ uint32_t k_bits(int n, int tile) const {
        return __builtin_amdgcn_readlane(at_k, EACH * (n % kSteps) + tile);
    }
    __device__ __forceinline__ uint32_t v_bits(int n, int tile) const {
        return __builtin_amdgcn_readlane(at_v, EACH * (n % kSteps) + tile);
    }
};

// A lane's 16 bytes of each 1 KB of a tile; no bytes where size is 0.
template <int DIM>
__device__ __forceinline__ void load_tile(uint8_t* pool, uint64_t base, int size, int lane, u4 (&raw)[DIM / 64]) {
    const auto tile = __builtin_amdgcn_make_buffer_rsrc(pool + base, 0, size, 0x27000);
#pragma unroll
    for (int j = 0; j < DIM / 64; ++j) raw[j] = __builtin_amdgcn_raw_buffer_load_b128(tile, 16 * lane + 1024 * j, 0, 0);
}

// Value bytes of slots past the last row's position may be anything; as bytes
// they are made 0 where an E4M3 NaN could be (INT8 codes are finite, and their
// probability is 0). `left`: slots from the lane's first on that are inside.
template <int DIM>
__device__ __forceinline__ void clear_past(int left, u4 (&raw)[DIM / 64]) {
    const uint32_t keep = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
#pragma unroll
    for (int j = 0; j < DIM / 64; ++j) raw[j] &= keep;
}

// 0x80 in the bytes that are E4M3 NaNs (0x7F and 0xFF), 0 in the others.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// Makes the NaN bytes of a lane's values 0, whose product with the probability
// of 0 of a token that a column does not see is 0; nonzero where there were any.
template <int DIM>
__device__ __forceinline__ uint32_t clear_nan(u4 (&raw)[2][DIM / 64]) {
    uint32_t met = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < DIM / 16; ++n) {
            const uint32_t is = nan_bytes(raw[h][n / 4][n % 4]);
            raw[h][n / 4][n % 4] &= ~((is >> 7) * 0xFFu);
            met |= is;
        }
    return met;
}

// o becomes NaN in the dims of the columns that see a NaN byte among the
// values of a pair of tiles; `token`: the lane's first of the first tile's.
// Which ones do is a product as well, of marks where bytes are NaN with marks
// where columns see tokens.
template <int DIM, int NT>
__device__ __forceinline__ void spread_nan(int token, const int (&qpos)[NT], uint8_t* pool, const uint64_t (&base)[2],
                                           int lane, f4 (&o)[NT][DIM / 16]) {
    Half8 seen[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) seen[t].one[4 * h + i] = token + kTile * h + i <= qpos[t] ? 1 : 0;
#pragma unroll
    for (int j = 0; j < DIM / 64; ++j) {
        u4 raw[2][1];
#pragma unroll
        for (int h = 0; h < 2; ++h) load_tile<64>(pool, base[h] + 1024 * j, kTile * 64, lane, raw[h]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            Half8 marks;
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // 0x80 as the FP16 number 0x2000, 2^-7
                const uint32_t is = nan_bytes(raw[h][0][k]) >> 2;
                marks.two[2 * h] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0u, is, 0x010C000Cu));
                marks.two[2 * h + 1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0u, is, 0x030C020Cu));
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const f4 none = {0.f, 0.f, 0.f, 0.f};
                const f4 met = __builtin_amdgcn_mfma_f32_16x16x32_f16(marks.all, seen[t].all, none, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (met[i] != 0.0f) o[t][4 * j + k][i] = quiet_nan();
            }
        }
    }
}

// Powers of two between the value scales of a pair of tiles up to which the
// first is converted to the second's scale: exact in FP16 (E4M3's smallest code
// is 2^-9, FP16's smallest number 2^-24).
constexpr uint32_t kApart = 8;

// A value scale as a power of two of the largest its columns see. Codes are
// exact down to 2^-24 of it (E4M3: 2^-15), below that rounded to 2^-25 of it,
// 2^-31 (2^-33) of its page's largest value; 2^-40 of it is nothing.
__device__ __forceinline__ float value_power(uint32_t bits, uint32_t top) {
    return __uint_as_float((uint32_t)max((int)(bits - top) + (127 << 23), (127 - 40) << 23));
}

}  // namespace mphip
