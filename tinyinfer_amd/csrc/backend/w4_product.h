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
    bool x_wide, out_wide;
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
// bits: exactly. 8-bit rows are BF16 numbers as they are.
constexpr int parts_of(int kind) { return kind == MP_TYPE_F32 ? 3 : kind == MP_TYPE_F16 ? 2 : 1; }

__device__ __forceinline__ float gated(float gate, float up) { return gate / (1.0f + expf(-gate)) * up; }

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

// Products of many rows: rows laid out for the matrix cores in the workspace,
// then tiles of 256 columns and 128 rows.
void w4_tiles(const ProductArgs& a, int kind, bool gate, void* workspace, hipStream_t s);

}  // namespace mphip
