// Products of rows with 4-bit matrices: wavefronts that share columns and deal
// the depth among themselves.
#include "w4_product.h"

namespace mphip {
namespace {

// Tiles of 16 by 16 (128 columns of depth a step, lane (c, g) of a tile with row
// c at columns 32g ..+31), and of 32 by 32 (64 columns, lane (r, h) with row r at
// columns 32h ..+31), which take less time an operation: 1.87 PFLOP/s instead of
// 1.29 from registers alone.
template <int SIDE>
struct Tile;
template <>
struct Tile<16> {
    typedef f4 Sum;
    static constexpr int QUADS = 1, DEPTH = 128;
    static __device__ __forceinline__ void add(const b8& w, const b8& x, Sum* s) {
        *s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, *s, 0, 0, 0);
    }
    static __device__ __forceinline__ f4 quad(const Sum& s, int) { return s; }
};
template <>
struct Tile<32> {
    typedef float Sum __attribute__((ext_vector_type(16)));
    static constexpr int QUADS = 4, DEPTH = 64;
    static __device__ __forceinline__ void add(const b8& w, const b8& x, Sum* s) {
        *s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, x, *s, 0, 0, 0);
    }
    static __device__ __forceinline__ f4 quad(const Sum& s, int q) {
        return f4{s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
    }
};

// A work-group has NT tiles of columns and one of rows; its wavefronts deal the
// depth among themselves, each with all of the block's sums, which meet in LDS at
// the end, in the wavefronts' order.
//
// A wavefront reads its rows along their columns, whole lines of memory at a time
// (16 bytes of 64 rows take four times as long), and turns them into operands on
// the way through LDS of its own, so that wavefronts do not wait for each other.
// Of a tile that is not full only the rows that are there are kept. What the next
// block of depth needs is on its way while this one is multiplied.
//
// A single row reads the weights once. The gated pair of 4,096 by 12,288, with four
// tiles of a wavefront on their way, is bounded by those bytes: 14.5 us for 53.5 MB,
// 3.7 TB/s (a large copy 5.1). Square and deep matrices leave a wavefront one tile, a
// kilobyte on its way, and are bounded by latency: 9.6 us for 12,288 by 4,096 (2.8
// TB/s), 6.1 for 4,096 by 4,096 (1.5). Small ones are one chain of latencies, 4.3 us
// for FP32, 1,536 by 576. With more rows every work-group reads and turns round all of
// its rows for 32 or 64 columns, and splitting FP32 into BF16 numbers takes the vector
// unit as long as the products: 24 us for 64 rows of 4,096 by 4,096, 16 for 8 bits.
template <int KIND, int SIDE, int NT, bool GATED>
__global__ void __launch_bounds__(512) w4_few_kernel(ProductArgs a) {
    typedef Tile<SIDE> T;
    constexpr int M = GATED ? 2 : 1, Q = T::QUADS, UNITS = M * NT * Q, PARTS = parts_of(KIND);
    constexpr int RUNS = T::DEPTH / 8, EACH = SIDE * RUNS / 64, ROWS_EACH = 64 / RUNS;
    extern __shared__ u4 shared_s[];  // [wavefront][part][run][row]; at the end [wavefront][matrix][tile][quad][lane]
    const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane % SIDE, g = lane / SIDE;
    const int column_block = blockIdx.x / a.row_blocks, row_block = blockIdx.x % a.row_blocks;
    const int tiles = (int)w4_tiles(a.n), steps = (int)w4_steps(a.depth), words = (int)w4_words(a.depth);
    // Columns behind the end are those at the end again, and not stored.
    const u4* codes_at[M][NT];
    const uint32_t* scales_at[M][NT];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int64_t tile = min((column_block * NT + i) * (SIDE / 16) + c / 16, tiles - 1);
            codes_at[m][i] = a.m[m].codes + tile * steps * 64 + g * 16 + c % 16;
            scales_at[m][i] = a.m[m].scales + tile * words * 64 + g * 16 + c % 16;
        }
    typename T::Sum sum[M][NT] = {};
    // Blocks of DEPTH columns: halves of a step with tiles of 32.
    constexpr int HALVES = kW4Step / T::DEPTH;
    const int blocks = (int)w4_ceil(a.depth, T::DEPTH);
    const int first = blocks * wave / waves, last = blocks * (wave + 1) / waves;
    // Rows of this tile, and the power of two that their places in LDS take:
    // row r of run e lies at r ^ e, so that neither rows nor runs share banks.
    const int rows = min(a.rows - row_block * SIDE, SIDE), places = w4_places(rows), mask = places - 1;
    u4* const mine = shared_s + wave * (PARTS * RUNS) * places;
    const int run_of = lane % RUNS, row_of = lane / RUNS;
    u4 codes[M][NT];
    uint32_t scale[M][NT];
    Run8<KIND> run[EACH];
    typename Run8<KIND>::Row row_at[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) row_at[i].begin(a, (int64_t)row_block * SIDE + i * ROWS_EACH + row_of);
    auto load = [&](int block) {
        const int step = block / HALVES, half = block % HALVES;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                codes[m][i] = codes_at[m][i][step * 64 + half * 32];
                scale[m][i] = scales_at[m][i][step / kW4Word * 64 + half * 32];
            }
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (i * ROWS_EACH < rows)
                run[i].load(row_at[i], min(block * T::DEPTH + 8 * run_of, a.depth - 8));
    };
    if (first < last) load(first);
    for (int block = first; block < last; ++block) {
        wave_sync();
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int r = i * ROWS_EACH + row_of;
            if (i * ROWS_EACH < rows && r < places) {
                u4 part[PARTS];
                run[i].split(part);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) mine[(p * RUNS + run_of) * places + (r ^ (run_of & mask))] = part[p];
            }
        }
        wave_sync();
        u4 now[M][NT];
        float power[M][NT];
        const int shift = 8 * (block / HALVES % kW4Word);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                now[m][i] = codes[m][i];
                power[m][i] = scale_power(scale[m][i] >> shift & 0xFF);
            }
        if (block + 1 < last) load(block + 1);
        __builtin_amdgcn_sched_barrier(0);  // the loads go out before the products
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            b8 x[PARTS];
            const int e = 4 * g + d;
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                x[p] = __builtin_bit_cast(b8, mine[(p * RUNS + e) * places + ((c ^ e) & mask)]);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const b8 w = weights8(now[m][i][d], power[m][i]);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) T::add(w, x[p], &sum[m][i]);
                }
        }
    }
    f4* const parts_s = reinterpret_cast<f4*>(shared_s);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int q = 0; q < Q; ++q)
                parts_s[(wave * UNITS + (m * NT + i) * Q + q) * 64 + lane] = T::quad(sum[m][i], q);
    __syncthreads();
    auto joined = [&](int i, int q) {
        f4 v[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            v[m] = f4{0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < waves; ++w) v[m] += parts_s[(w * UNITS + (m * NT + i) * Q + q) * 64 + lane];
        }
        if constexpr (GATED) v[0] = gated(v[1], v[0]);
        return v[0];
    };
    const int64_t row = (int64_t)row_block * SIDE + c;
    if (a.out.type == MP_TYPE_I8) {
        // A row's group of 32: two tiles of 16 columns, or one of 32.
        if constexpr (SIDE == 32) {
            for (int i = wave; i < NT; i += waves) {
                const int n = (column_block * NT + i) * SIDE;
                f4 v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = joined(i, q);
                store_result8<32>(a, row, n, g, v, c < rows && n < a.n);
            }
        } else if constexpr (NT % 2 == 0) {
            for (int i = 2 * wave; i < NT; i += 2 * waves) {
                const int n = (column_block * NT + i) * SIDE;
                const f4 v[2] = {joined(i, 0), joined(i + 1, 0)};
                store_result8<16>(a, row, n, g, v, c < rows && n < a.n);
            }
        }
    } else {
        for (int unit = wave; unit < NT * Q; unit += waves) {
            const int n = (column_block * NT + unit / Q) * SIDE + 8 * (unit % Q) + 4 * g;
            const f4 v = joined(unit / Q, unit % Q);
            if (c < rows && n < a.n) store_result(a, row, n, v);
        }
    }
}

template <int KIND, int SIDE, int NT>
void few(const ProductArgs& a, const W4Plan& p, bool gate, hipStream_t s) {
    const unsigned groups = (unsigned)(a.column_blocks * (int64_t)a.row_blocks);
    const size_t shared = w4_few_shared(p, a.rows, parts_of(KIND), gate);
    if (gate) w4_few_kernel<KIND, SIDE, NT, true><<<groups, 64 * p.waves, shared, s>>>(a);
    else w4_few_kernel<KIND, SIDE, NT, false><<<groups, 64 * p.waves, shared, s>>>(a);
}
template <int KIND>
void few_tiles(const ProductArgs& a, const W4Plan& p, bool gate, hipStream_t s) {
    if (p.side == 32) {
        if (p.column_tiles == 1) few<KIND, 32, 1>(a, p, gate, s);
        else few<KIND, 32, 2>(a, p, gate, s);
    } else {
        if (p.column_tiles == 1) few<KIND, 16, 1>(a, p, gate, s);
        else if (p.column_tiles == 2) few<KIND, 16, 2>(a, p, gate, s);
        else few<KIND, 16, 4>(a, p, gate, s);
    }
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
        *bytes = type == MP_TYPE_I8 && w4_way(rows, w->rows, gated != 0) == kW4LargeTiles ? w4_planes_bytes(rows, w->depth) : 0;
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
        const W4Way way = w4_way(rows, w->rows, gate != nullptr);
        const bool planes = way == kW4LargeTiles && x->type == MP_TYPE_I8;
        const size_t need = planes ? w4_planes_bytes(rows, w->depth) : 0;
        if (need > workspace_bytes || (need && !workspace))
            return refuse_call("4-bit product: the workspace is smaller than mp_hip_w4_product_workspace says");
        if (need && reinterpret_cast<uintptr_t>(workspace) % 16)
            return refuse_call("4-bit product: the workspace must be 16-byte aligned");
        const W4Plan p = w4_few_plan(rows, w->rows, w->depth, parts_of(x->type), gate != nullptr, out->type == MP_TYPE_I8);
        const int64_t groups = way == kW4Few ? w4_groups(p, rows, w->rows)
                                             : w4_tile_groups(rows, w->rows, gate != nullptr, way == kW4LargeTiles);
        if (groups > kW4MostGroups || (planes && w4_planes_blocks(rows, w->depth) > kW4MostGroups))
            return refuse_call("4-bit product: too large for one call");
        ProductArgs a{};
        a.m[0] = view(*w);
        if (gate) a.m[1] = view(*gate);
        a.n = w->rows, a.depth = w->depth, a.rows = rows;
        a.x = rows_view(*x), a.out = rows_view(*out);
        a.out_wide = rows_wide(*out);
        a.column_blocks = (int)w4_ceil(a.n, p.side * p.column_tiles);
        a.row_blocks = (int)w4_ceil(rows, p.side);
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return call_done(device.status, "4-bit product: device of the stream");
        if (way != kW4Few) w4_tiles(a, x->type, gate != nullptr, way == kW4LargeTiles, workspace, s);
        else if (x->type == MP_TYPE_F32) few_tiles<MP_TYPE_F32>(a, p, gate != nullptr, s);
        else if (x->type == MP_TYPE_BF16) few_tiles<MP_TYPE_BF16>(a, p, gate != nullptr, s);
        else if (x->type == MP_TYPE_F16) few_tiles<MP_TYPE_F16>(a, p, gate != nullptr, s);
        else few_tiles<MP_TYPE_I8>(a, p, gate != nullptr, s);
        return call_done(hipGetLastError(), "4-bit product launch");
    });
}
