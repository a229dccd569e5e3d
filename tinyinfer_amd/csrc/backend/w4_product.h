// What the kernels of products with 4-bit matrices share: arguments and results.
#pragma once
#include "w4.h"

namespace mphip {

typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

struct ProductArgs {
    W4View m[2];  // the matrix, the gate
    int n, depth, rows;
    RowsView x, out;
    bool out_wide;
    int column_blocks, row_blocks;
};

// 8 weights, an eighth of a lane's 128 columns, times their scale: E2M1 numbers
// times a power of two are BF16 numbers, one conversion for two.
__device__ __forceinline__ b8 weights8(uint32_t codes, float power) {
    b2 w[4];
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 0);
    w[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 1);
    w[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 2);
    w[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 3);
    return b8{w[0][0], w[0][1], w[1][0], w[1][1], w[2][0], w[2][1], w[3][0], w[3][1]};
}

// The upper halves of two numbers: each cut to a BF16 number.
__device__ __forceinline__ uint32_t upper_halves(float u, float v) {
    return __builtin_amdgcn_perm(__float_as_uint(v), __float_as_uint(u), 0x07060302u);
}
// A float row's elements as sums of this many BF16 numbers, each the next 8
// bits: exactly, but for FP32 elements below 2^-110, of which BF16 numbers, multiples
// of 2^-133, hold no more than those. 8-bit rows are BF16 numbers as they are.
constexpr int parts_of(int kind) { return kind == MP_TYPE_F32 ? 3 : kind == MP_TYPE_F16 ? 2 : 1; }

// silu(gate) * up. From -88.7 down exp(-gate) is infinite, while the product with
// `up` can be any number. Below -80 silu is gate * exp(gate) far beyond the last bit,
// and exp(gate) four equal factors: every number on the way is larger than the
// result, so that only the last is rounded below the normal numbers. One branch for
// all of a lane's results takes no time (4,096 8-bit rows through a pair of 4,096 by
// 12,288: 451 us with it and without), one for each result 2 %.
template <typename V>
__device__ __forceinline__ V gated(const V& gate, const V& up) {
    constexpr int N = sizeof(V) / sizeof(float);
    V y;
    float least = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        y[i] = gate[i] / (1.0f + expf(-gate[i])) * up[i];
        least = fminf(least, gate[i]);
    }
    if (least < -80.0f) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float quarter = expf(0.25f * gate[i]);
            const float far = gate[i] * quarter * up[i] * quarter * quarter * quarter;
            y[i] = gate[i] < -80.0f ? far : y[i];
        }
    }
    return y;
}

// Results of `row`, columns n ..+3 of a tile.
__device__ __forceinline__ void store_result(const ProductArgs& a, int64_t row, int n, const f4& v) {
    const int64_t at = row * a.out.stride + n;
    if (n + 3 < a.n) {
        store_four(a.out.data, a.out.type, a.out_wide, at, v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.n) store_one(a.out.data, a.out.type, at + i, v[i]);
    }
}

// Results of `row`, columns n ..+31, as 8 bits: lane (c, g) has columns n + 16t +
// 4g ..+3 of two tiles t of 16 columns (SIDE 16), or n + 8q + 4g ..+3 for q = 0..3
// of one of 32 columns. All lanes of a row come together.
template <int SIDE, int N>
__device__ __forceinline__ void store_result8(const ProductArgs& a, int64_t row, int n, int g, const f4 (&v)[N],
                                              bool there) {
    static_assert(N == (SIDE == 32 ? 4 : 2));
    uint32_t amax = 0;
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = max(amax, magnitude(v[t][i]));
    if constexpr (SIDE == 32) {
        const auto both = __builtin_amdgcn_permlane32_swap(amax, amax, false, false);
        amax = max((uint32_t)both[0], (uint32_t)both[1]);
    } else {
        amax = column_max(amax);
    }
    if (!there) return;
    const uint32_t byte = scale_byte8(amax);
    const float inverse = scale_inverse(byte);
    uint8_t* const codes = static_cast<uint8_t*>(a.out.data) + row * a.out.stride + n + 4 * g;
#pragma unroll
    for (int t = 0; t < N; ++t)
        *reinterpret_cast<uint32_t*>(codes + 32 / N * t) = to_codes8(v[t][0], v[t][1], v[t][2], v[t][3], inverse);
    if (g == 0) a.out.scales[row * a.out.scale_stride + n / kW4Group] = (uint8_t)byte;
}

// 8 columns of a row, as they lie and as the BF16 numbers whose sums they are.
// Loads are of 16 bytes wherever a row begins: the memory takes any alignment of
// the elements, and aligned rows are as fast.
template <int KIND>
struct Run8 {
    static constexpr int BYTES = 8 * (KIND == MP_TYPE_I8 ? 1 : KIND == MP_TYPE_F32 ? 4 : 2), WORDS = BYTES / 4;
    uint32_t raw[WORDS];
    float scale;
    // A row behind the end is the last again.
    struct Row {
        const uint8_t* data;
        const uint8_t* scales;
        __device__ __forceinline__ void begin(const ProductArgs& a, int64_t row) {
            row = min(row, (int64_t)a.rows - 1);
            data = static_cast<const uint8_t*>(a.x.data) + row * a.x.stride * (BYTES / 8);
            if constexpr (KIND == MP_TYPE_I8) scales = a.x.scales + row * a.x.scale_stride;
        }
    };
    // `column` is one of the row's: where a block's columns end behind the depth, the
    // row's last ones stand in for them, times weights that are zeros.
    __device__ __forceinline__ void load(const Row& row, uint32_t column) {
        typedef uint32_t w4 __attribute__((ext_vector_type(4), aligned(2)));
        const uint8_t* const from = row.data + column * (BYTES / 8);
        if constexpr (KIND == MP_TYPE_I8) {
            const uint2 v = *reinterpret_cast<const uint2*>(from);
            raw[0] = v.x, raw[1] = v.y;
            scale = scale_number(row.scales[column / kW4Group]);
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const w4 v = reinterpret_cast<const w4*>(from)[i / 4];
                raw[i] = v[0], raw[i + 1] = v[1], raw[i + 2] = v[2], raw[i + 3] = v[3];
            }
        }
    }
    __device__ __forceinline__ void split(u4 (&part)[parts_of(KIND)]) const {
        if constexpr (KIND == MP_TYPE_BF16) {
            part[0] = u4{raw[0], raw[1], raw[2], raw[3]};
        } else if constexpr (KIND == MP_TYPE_I8) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f4 x = from_codes8(raw[k], scale);
                part[0][2 * k] = upper_halves(x[0], x[1]);
                part[0][2 * k + 1] = upper_halves(x[2], x[3]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float u, v;
                if constexpr (KIND == MP_TYPE_F32) {
                    u = __uint_as_float(raw[2 * k]), v = __uint_as_float(raw[2 * k + 1]);
                } else {
                    u = from_f16(raw[k] & 0xFFFF), v = from_f16(raw[k] >> 16);
                }
#pragma unroll
                for (int p = 0; p < parts_of(KIND); ++p) {
                    part[p][k] = upper_halves(u, v);
                    u -= __uint_as_float(__float_as_uint(u) & 0xFFFF0000u);
                    v -= __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
                }
            }
        }
    }
};

// Products of more rows, by tiles: 256 columns by 128 rows (`large`; 8-bit rows are
// laid out in the workspace before) or 128 by 64.
void w4_tiles(const ProductArgs& a, int kind, bool gate, bool large, void* workspace, hipStream_t s);

}  // namespace mphip
