// Products of rows with 4-bit matrices: wavefronts that share columns and deal
// the depth among themselves.
#include "w4_product.h"

namespace mphip {
namespace {

// The rows' operand of 128 columns: lane (c, g) has row c at columns 32g ..+31.
template <int KIND>
struct Operand {
    static constexpr int PARTS = parts_of(KIND);
    u4 part[4][PARTS];  // 8 columns each
    __device__ __forceinline__ void load(const ProductArgs& a, int64_t row, int step, int g) {
        const int column = step * kW4Step + 32 * g;
        const int64_t at = row * a.x.stride + column;
        if (column >= a.depth) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int p = 0; p < PARTS; ++p) part[s][p] = u4{0, 0, 0, 0};
            return;
        }
        if constexpr (KIND == MP_TYPE_I8) {
            const u4* const from = reinterpret_cast<const u4*>(static_cast<const uint8_t*>(a.x.data) + at);
            const float scale = scale_number(a.x.scales[row * a.x.scale_stride + column / kW4Group]);
            const u4 codes[2] = {from[0], from[1]};
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    const f4 x = from_codes8(codes[s / 2][s % 2 * 2 + k / 2], scale);
                    part[s][0][k] = upper_halves(x[0], x[1]);
                    part[s][0][k + 1] = upper_halves(x[2], x[3]);
                }
        } else if constexpr (KIND == MP_TYPE_BF16) {
            const uint16_t* const from = static_cast<const uint16_t*>(a.x.data) + at;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (a.x_wide) {
                    part[s][0] = *reinterpret_cast<const u4*>(from + 8 * s);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        part[s][0][k] = from[8 * s + 2 * k] | (uint32_t)from[8 * s + 2 * k + 1] << 16;
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                float x[8];
                load_row(a.x.data, KIND, a.x_wide, at + 8 * s, x);
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    float u = x[k], v = x[k + 1];
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        part[s][p][k / 2] = upper_halves(u, v);
                        u -= __uint_as_float(__float_as_uint(u) & 0xFFFF0000u);
                        v -= __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
                    }
                }
            }
        }
    }
};

// Adds a tile's 128 columns of `codes` (lane (c, g): row c of the matrix,
// columns 32g ..+31) times the rows' operand.
template <int KIND>
__device__ __forceinline__ void multiply(const u4& codes, uint32_t scale, const Operand<KIND>& x, f4* sum) {
    const float power = scale_power(scale & 0xFF);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const b8 w = weights8(codes[s], power);
#pragma unroll
        for (int p = 0; p < Operand<KIND>::PARTS; ++p)
            *sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, __builtin_bit_cast(b8, x.part[s][p]), *sum, 0, 0, 0);
    }
}

// Results of `row`, columns n ..+3 and n + 16 ..+3, as 8 bits; n + 16's group of
// 32 begins at this tile. The four lanes of a column have a row's group.
__device__ __forceinline__ void store_result8(const ProductArgs& a, int64_t row, int n, int g, const f4& v, const f4& w,
                                              bool there) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) amax = max(amax, max(magnitude(v[i]), magnitude(w[i])));
    const uint32_t byte = scale_byte8(column_max(amax));
    if (!there) return;
    const float inverse = scale_inverse(byte);
    uint8_t* const codes = static_cast<uint8_t*>(a.out.data) + row * a.out.stride + n;
    *reinterpret_cast<uint32_t*>(codes) = to_codes8(v[0], v[1], v[2], v[3], inverse);
    *reinterpret_cast<uint32_t*>(codes + 16) = to_codes8(w[0], w[1], w[2], w[3], inverse);
    if (g == 0) a.out.scales[row * a.out.scale_stride + n / kW4Group] = (uint8_t)byte;
}

// A work-group has 16 NT columns of 16 RT rows; its wavefronts deal the depth
// among themselves, each with all of the block's sums, which meet in LDS at the
// end, in the wavefronts' order.
template <int KIND, int NT, int RT, bool GATED>
__global__ void __launch_bounds__(512) w4_few_kernel(ProductArgs a) {
    constexpr int M = GATED ? 2 : 1, TILES = M * NT * RT;
    extern __shared__ f4 parts_s[];  // [wavefront][tile][lane]
    const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int column_block = blockIdx.x / a.row_blocks, row_block = blockIdx.x % a.row_blocks;
    const int tiles = (int)w4_tiles(a.n), steps = (int)w4_steps(a.depth), words = (int)w4_words(a.depth);
    // Tiles and rows behind the end are those at the end again, and not stored.
    int64_t tile[NT], row[RT];
#pragma unroll
    for (int i = 0; i < NT; ++i) tile[i] = min(column_block * NT + i, tiles - 1);
#pragma unroll
    for (int j = 0; j < RT; ++j) row[j] = min((row_block * RT + j) * kW4Rows + c, a.rows - 1);
    f4 sum[M][NT][RT];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < RT; ++j) sum[m][i][j] = f4{0.f, 0.f, 0.f, 0.f};
    const int first = steps * wave / waves, last = steps * (wave + 1) / waves;
    for (int step = first; step < last; ++step) {
        u4 codes[M][NT];
        uint32_t scale[M][NT];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                codes[m][i] = a.m[m].codes[(tile[i] * steps + step) * 64 + lane];
                scale[m][i] = a.m[m].scales[(tile[i] * words + step / kW4Word) * 64 + lane] >> (8 * (step % kW4Word));
            }
        Operand<KIND> x[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) x[j].load(a, row[j], step, g);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j) multiply<KIND>(codes[m][i], scale[m][i], x[j], &sum[m][i][j]);
    }
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < RT; ++j) parts_s[(wave * TILES + (m * NT + i) * RT + j) * 64 + lane] = sum[m][i][j];
    __syncthreads();
    auto joined = [&](int i, int j) {
        f4 v[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            v[m] = f4{0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < waves; ++w) v[m] += parts_s[(w * TILES + (m * NT + i) * RT + j) * 64 + lane];
        }
        if constexpr (GATED) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[0][k] = gated(v[1][k], v[0][k]);
        }
        return v[0];
    };
    if (a.out.type == MP_TYPE_I8) {
        if constexpr (NT % 2 == 0) {
            for (int unit = wave; unit < NT / 2 * RT; unit += waves) {
                const int i = unit / RT * 2, j = unit % RT, r = (row_block * RT + j) * kW4Rows + c;
                const int n = (column_block * NT + i) * kW4Rows + 4 * g;
                const f4 v = joined(i, j), w = joined(i + 1, j);
                store_result8(a, r, n, g, v, w, r < a.rows && n < a.n);
            }
        }
    } else {
        for (int unit = wave; unit < NT * RT; unit += waves) {
            const int i = unit / RT, j = unit % RT, r = (row_block * RT + j) * kW4Rows + c;
            const int n = (column_block * NT + i) * kW4Rows + 4 * g;
            const f4 v = joined(i, j);
            if (r < a.rows && n < a.n) store_result(a, r, n, v);
        }
    }
}

template <int KIND, int NT, int RT>
void few(const ProductArgs& a, const W4Plan& p, bool gate, hipStream_t s) {
    const unsigned groups = (unsigned)(a.column_blocks * (int64_t)a.row_blocks);
    const size_t shared = (size_t)p.waves * NT * RT * (gate ? 2 : 1) * 64 * sizeof(f4);
    if (gate) w4_few_kernel<KIND, NT, RT, true><<<groups, 64 * p.waves, shared, s>>>(a);
    else w4_few_kernel<KIND, NT, RT, false><<<groups, 64 * p.waves, shared, s>>>(a);
}
template <int KIND, int NT>
void few_rows(const ProductArgs& a, const W4Plan& p, bool gate, hipStream_t s) {
    if (p.row_tiles == 1) few<KIND, NT, 1>(a, p, gate, s);
    else if (p.row_tiles == 2) few<KIND, NT, 2>(a, p, gate, s);
    else few<KIND, NT, 4>(a, p, gate, s);
}
template <int KIND>
void few_columns(const ProductArgs& a, const W4Plan& p, bool gate, hipStream_t s) {
    if (p.column_tiles == 1) few_rows<KIND, 1>(a, p, gate, s);
    else if (p.column_tiles == 2) few_rows<KIND, 2>(a, p, gate, s);
    else few_rows<KIND, 4>(a, p, gate, s);
}

W4View view(const mp_w4_matrix& m) {
    return W4View{reinterpret_cast<const u4*>(m.codes), reinterpret_cast<const uint32_t*>(m.scales)};
}

}  // namespace
}  // namespace mphip

extern "C" int mp_hip_w4_product_workspace(const mp_w4_matrix* w, int32_t type, int32_t rows, int32_t gated,
                                           size_t* bytes) {
    using namespace mphip;
    return c_entry([&]() -> int {
        if (!bytes) return refuse_call("4-bit product: no place for the workspace's size");
        const char* wrong = w ? w4_wrong_size(w->rows, w->depth) : "4-bit matrix: codes or scales are missing";
        if (wrong) return refuse_call(wrong);
        if (type < MP_TYPE_F32 || type > MP_TYPE_I8) return refuse_call("rows: element type unknown or not taken here");
        if (rows < 0 || rows > kW4MostRows) return refuse_call("4-bit product: 0 to 1,048,576 rows a call");
        *bytes = rows > kW4FewRows ? w4_tiles_workspace(rows, w->depth, type) : 0;
        return MP_OK;
    });
}

extern "C" int mp_hip_w4_product(const mp_w4_matrix* w, const mp_w4_matrix* gate, const mp_rows* x, int32_t rows,
                                 const mp_rows* out, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace mphip;
    return c_entry([&]() -> int {
        const char* wrong = w4_wrong_matrix(w);
        if (!wrong && gate) wrong = w4_wrong_matrix(gate);
        if (!wrong) wrong = rows_wrong(x, w->depth, true);
        if (!wrong) wrong = rows_wrong(out, w->rows, true);
        if (wrong) return refuse_call(wrong);
        if (gate && (gate->rows != w->rows || gate->depth != w->depth))
            return refuse_call("4-bit product: the gate is of another size");
        if (rows < 0 || rows > kW4MostRows) return refuse_call("4-bit product: 0 to 1,048,576 rows a call");
        if (x->data == out->data) return refuse_call("4-bit product: no result in place of the rows");
        if (rows == 0) return MP_OK;
        const bool pairs = out->type == MP_TYPE_I8, tiled = w4_tiled(rows, w->rows, gate != nullptr);
        const size_t need = tiled ? w4_tiles_workspace(rows, w->depth, x->type) : 0;
        if (need > workspace_bytes || (need && !workspace))
            return refuse_call("4-bit product: the workspace is smaller than mp_hip_w4_product_workspace says");
        if (need && reinterpret_cast<uintptr_t>(workspace) % 16)
            return refuse_call("4-bit product: the workspace must be 16-byte aligned");
        const W4Plan p = w4_few_plan(rows, w->rows, w->depth, gate != nullptr, pairs);
        if (tiled ? w4_tiles_groups(rows, w->rows, gate != nullptr) > kW4MostGroups ||
                        w4_ceil(rows, kTileRows) * w4_ceil(w->depth, kTileDepth) > kW4MostGroups
                  : w4_groups(p, rows, w->rows) > kW4MostGroups)
            return refuse_call("4-bit product: too large for one call");
        ProductArgs a{};
        a.m[0] = view(*w);
        if (gate) a.m[1] = view(*gate);
        a.n = w->rows, a.depth = w->depth, a.rows = rows;
        a.x = rows_view(*x), a.out = rows_view(*out);
        a.x_wide = rows_wide(*x), a.out_wide = rows_wide(*out);
        a.column_blocks = (int)w4_ceil(w4_tiles(a.n), p.column_tiles);
        a.row_blocks = (int)w4_ceil(w4_tiles(rows), p.row_tiles);
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return call_done(device.status, "4-bit product: device of the stream");
        if (tiled) w4_tiles(a, x->type, gate != nullptr, workspace, s);
        else if (x->type == MP_TYPE_F32) few_columns<MP_TYPE_F32>(a, p, gate != nullptr, s);
        else if (x->type == MP_TYPE_BF16) few_columns<MP_TYPE_BF16>(a, p, gate != nullptr, s);
        else if (x->type == MP_TYPE_F16) few_columns<MP_TYPE_F16>(a, p, gate != nullptr, s);
        else few_columns<MP_TYPE_I8>(a, p, gate != nullptr, s);
        return call_done(hipGetLastError(), "4-bit product launch");
    });
}
