// Products of many rows with 4-bit matrices: tiles on the matrix cores.
#include <type_traits>

#include "w4_product.h"

namespace mphip {
namespace {

typedef int v8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;

// ---- what the work-groups share ------------------------------------------------------

// Work-groups that an XCD runs together share columns and rows: each XCD has a
// run of blocks that goes down 8 blocks of rows before the next columns.
__device__ __forceinline__ void find_block(const ProductArgs& a, int* row_block, int* column_block) {
    const int all = gridDim.x, xcd = blockIdx.x % 8, inside = blockIdx.x / 8;
    const int index = xcd * (all / 8) + min(xcd, all % 8) + inside;
    const int band = index / (8 * a.column_blocks), in_band = index % (8 * a.column_blocks);
    const int band_rows = min(8, a.row_blocks - 8 * band);
    *row_block = 8 * band + in_band % band_rows, *column_block = in_band / band_rows;
}

// A wavefront's N tiles of 32 columns from `first` on: of the matrix, or half of
// them of it and the same of the gate. Codes come from memory to the registers as
// they lie, lane (c, h) with row c at columns 32h ..+31 of a block of 64. Places are
// a uniform address and 32 bits of a lane's own.
template <int N, bool GATED>
struct Weights {
    static constexpr int EACH = GATED ? N / 2 : N, M = GATED ? 2 : 1;
    struct Block {
        u4 codes[N];
        uint32_t scale[N];
    };
    const uint8_t* codes_at[M];
    const uint8_t* scales_at[M];
    uint32_t code_place[EACH], scale_place[EACH];
    __device__ __forceinline__ void begin(const ProductArgs& a, int first) {
        const int lane = threadIdx.x & 63, last = (int)w4_tiles(a.n) - 1, tile0 = min(first / kW4Rows, last);
        const int steps = (int)w4_steps(a.depth), words = (int)w4_words(a.depth);
#pragma unroll
        for (int m = 0; m < M; ++m) {
            codes_at[m] = reinterpret_cast<const uint8_t*>(a.m[m].codes) + (int64_t)tile0 * steps * 1024;
            scales_at[m] = reinterpret_cast<const uint8_t*>(a.m[m].scales) + (int64_t)tile0 * words * 256;
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            // Columns behind the end are those at the end again, and not stored.
            const uint32_t tile = min((first + i * 32) / kW4Rows + lane % 32 / 16, last) - tile0;
            code_place[i] = tile * steps * 1024 + (lane / 32 * 16 + lane % 16) * 16;
            scale_place[i] = tile * words * 256 + (lane / 32 * 16 + lane % 16) * 4;
        }
    }
    __device__ __forceinline__ void load(int block, Block* to) const {
        const int step = block >> 1, half = block & 1;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const uint8_t* const codes = codes_at[m] + step * 1024 + half * 512;
            const uint8_t* const scales = scales_at[m] + (step >> 2) * 256 + half * 128 + (step & 3);
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                to->codes[m * EACH + i] = *reinterpret_cast<const u4*>(codes + code_place[i]);
                to->scale[m * EACH + i] = scales[scale_place[i]];
            }
        }
    }
};

// Results of 32 rows by 32 columns: lane (r, h) has row r at columns 8q + 4h ..+3.
__device__ __forceinline__ void store_tile(const ProductArgs& a, int64_t row, int n, int h, const f16v& v) {
    f4 quad[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) quad[q] = f4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
    if (a.out.type == MP_TYPE_I8) {
        store_result8<32>(a, row, n, h, quad, row < a.rows && n < a.n);
    } else if (row < a.rows) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (n + 8 * q + 4 * h < a.n) store_result(a, row, n + 8 * q + 4 * h, quad[q]);
    }
}

template <int N, int RT, bool GATED>
__device__ __forceinline__ void store_tiles(const ProductArgs& a, int64_t first_row, int first_column,
                                            const f16v (&sum)[N][RT]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
        for (int i = 0; i < Weights<N, GATED>::EACH; ++i) {
            f16v v = sum[i][j];
            if constexpr (GATED) v = gated(sum[i + N / 2][j], v);
            store_tile(a, first_row + j * 32 + lane % 32, first_column + i * 32, lane / 32, v);
        }
}

// ---- rows as BF16 numbers --------------------------------------------------------------

// A work-group of WN x WR wavefronts has 32 N WN columns (half of them of each
// matrix of a gated pair) by 32 RT WR rows. It brings 64 columns of its rows to
// LDS, as the BF16 numbers whose sums they are, while the columns before are
// multiplied. 4,096 rows of 4,096 by 4,096: 124 us in BF16 (1.11 PFLOP/s; a large
// library product of this card 1.41), 205 in FP16, 305 in FP32 (two and three BF16
// numbers each: 1.34 and 1.35). 64 FP32 rows of 576 by 49,152, the small tiles' case,
// take 18 to 20 us: 1.5 work-groups a CU, each 9 blocks long.
template <int KIND, bool GATED, int N, int RT, int WN, int WR>
__global__ void __launch_bounds__(64 * WN * WR, 2) w4_tiles_kernel(ProductArgs a) {
    constexpr int PARTS = parts_of(KIND), THREADS = 64 * WN * WR, TILES = RT * WR, ROWS = 32 * TILES;
    constexpr int EACH = ROWS * 8 / THREADS;  // runs of 8 columns a thread
    constexpr int SIZE = PARTS * TILES * 256, BUFFERS = 2 * SIZE * 16 <= 65536 ? 2 : 1;
    __shared__ u4 rows_s[BUFFERS][SIZE];  // [part][tile][run of 8 columns][row]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane / 32;
    const int wave_columns = wave / WR, wave_rows = wave % WR;
    int row_block, column_block;
    find_block(a, &row_block, &column_block);
    constexpr int COLUMNS = Weights<N, GATED>::EACH * 32;  // of a wavefront
    const int first_column = (column_block * WN + wave_columns) * COLUMNS;
    const int64_t first_row = (int64_t)row_block * ROWS;
    Weights<N, GATED> w;
    w.begin(a, first_column);
    const int blocks = (int)w4_ceil(a.depth, kTileDepth);
    f16v sum[N][RT] = {};

    // Run i of a thread: columns 8e ..+7 of the block of a row, so that neighbours
    // read a line of memory. In LDS row r of run e lies at r ^ e: neither rows nor
    // runs share banks.
    const int e = threadIdx.x % 8, r0 = threadIdx.x / 8;
    Run8<KIND> run[EACH];
    typename Run8<KIND>::Row row[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) row[i].begin(a, first_row + r0 + i * (THREADS / 8));
    auto load_rows = [&](int block) {
        const uint32_t column = min(block * kTileDepth + 8 * e, a.depth - 8);
#pragma unroll
        for (int i = 0; i < EACH; ++i) run[i].load(row[i], column);
    };
    auto keep_rows = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int r = r0 + i * (THREADS / 8);
            u4 part[PARTS];
            run[i].split(part);
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                rows_s[buffer][((p * TILES + r / 32) * 8 + e) * 32 + (r % 32 ^ e)] = part[p];
        }
    };
    // A block from the buffer and the registers that have it, while the next one's
    // rows go from the registers to the other buffer and those behind it come from
    // memory: what is waited for was asked for a block's products before. With one
    // buffer the next rows are asked for here and kept behind the products.
    typename Weights<N, GATED>::Block even, odd;
    auto step = [&](int block, int buffer, const auto& now, auto* next) {
        const int behind = min(block + 1, blocks - 1);  // the last again, behind it
        if constexpr (BUFFERS == 2) {
            keep_rows(buffer ^ 1);
            load_rows(min(block + 2, blocks - 1));
        } else {
            load_rows(behind);
        }
        w.load(behind, next);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            b8 c[N];
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = weights8(now.codes[i][d], scale_power(now.scale[i]));
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const b8 x = __builtin_bit_cast(
                        b8, rows_s[buffer][((p * TILES + wave_rows * RT + j) * 8 + h * 4 + d) * 32 + (lane % 32 ^ (h * 4 + d))]);
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(c[i], x, sum[i][j], 0, 0, 0);
                }
        }
        if constexpr (BUFFERS == 1) {
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
            keep_rows(0);
        }
        __syncthreads();
    };
    load_rows(0);
    w.load(0, &even);
    keep_rows(0);
    if (BUFFERS == 2) load_rows(min(1, blocks - 1));
    __syncthreads();
    for (int block = 0; block < blocks; block += 2) {
        step(block, 0, even, &odd);
        if (block + 1 < blocks) step(block + 1, BUFFERS - 1, odd, &even);
    }
    store_tiles<N, RT, GATED>(a, first_row + wave_rows * RT * 32, first_column, sum);
}

// ---- 8-bit rows as planes of 6-bit numbers ------------------------------------------------

// Lays rows out in blocks of 128 rows and 64 columns, [rows/128][columns/64][block]:
// a lane (r = l%32, h = l/32) of a tile of 32 rows has row r at columns 32h ..+31.
// A whole number up to 127 (or -128) is 16 times one up to 15 plus another, and
// whole numbers up to 15 times 1/8 are E2M3 numbers whose code is that number: two
// planes of 6-bit codes, both with the element's sign. The matrix cores take E2M3
// times E2M1 at twice the rate of 8-bit formats and sum such products exactly
// before they join the FP32 sum, where 8-bit formats lose what lies 2^-13 below the
// largest of eight products. Per tile: the low plane ([lane][16 bytes], [lane][8
// bytes]) and the high one. Behind all blocks the scale bytes of both planes, [rows/
// 128][columns/128][tile][lane], a word a lane for the two halves of 128 columns.
__global__ void __launch_bounds__(kThreads) w4_planes_layout_kernel(ProductArgs a, uint8_t* laid) {
    const int tile = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int blocks = (int)w4_ceil(a.depth, kTileDepth);
    const int64_t row = (int64_t)(blockIdx.x / blocks) * kTileRows + tile * 32 + r;
    const int column = blockIdx.x % blocks * kTileDepth + 32 * h;
    u4 codes[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    uint32_t scale = 127;
    if (row < a.rows && column < a.depth) {
        const u4* const from =
            reinterpret_cast<const u4*>(static_cast<const uint8_t*>(a.x.data) + row * a.x.stride + column);
        codes[0] = from[0], codes[1] = from[1];
        scale = a.x.scales[row * a.x.scale_stride + column / kW4Group];
    }
    uint64_t low[3] = {0, 0, 0}, high[3] = {0, 0, 0};
#pragma unroll
    for (int k = 0; k < 32; ++k) {
        const int x = (int8_t)(codes[k / 16][k % 16 / 4] >> (8 * (k % 4)));
        const uint32_t m = (uint32_t)(x < 0 ? -x : x), sign = x < 0 ? 32u : 0u;
        const uint64_t l = sign | (m & 15), u = sign | (m >> 4);
        const int bit = 6 * k, word = bit / 64, shift = bit % 64;
        low[word] |= l << shift, high[word] |= u << shift;
        if (shift > 58) low[word + 1] |= l >> (64 - shift), high[word + 1] |= u >> (64 - shift);
    }
    uint8_t* const to = laid + (size_t)blockIdx.x * kPlanesBlock + tile * 2 * kPlaneBytes;
    reinterpret_cast<ulonglong2*>(to)[lane] = make_ulonglong2(low[0], low[1]);
    reinterpret_cast<uint64_t*>(to + 1024)[lane] = low[2];
    reinterpret_cast<ulonglong2*>(to + kPlaneBytes)[lane] = make_ulonglong2(high[0], high[1]);
    reinterpret_cast<uint64_t*>(to + kPlaneBytes + 1024)[lane] = high[2];
    uint16_t* const scales = reinterpret_cast<uint16_t*>(laid + (size_t)gridDim.x * kPlanesBlock);
    const int64_t step = (int64_t)(blockIdx.x / blocks) * w4_steps(a.depth) + blockIdx.x % blocks / 2;
    scales[((step * 4 + tile) * 64 + lane) * 2 + blockIdx.x % blocks % 2] =
        scale > kMostScale ? 0xFFFF : (uint16_t)((scale + 3) | (scale + 7) << 8);
}

// 16 bytes a lane from memory to LDS, at `to` and on, without registers.
__device__ __forceinline__ void bring(const uint8_t* from, void* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// A work-group of 2 x 2 wavefronts: 256 columns (of a gated pair 128 of each
// matrix) by 128 rows. A wavefront has 4 tiles of columns and 2 of rows. The
// work-group brings 64 columns of its rows and weights to LDS at a time. While a
// block is multiplied from the registers, the next comes to them from LDS and the
// one behind it from memory to LDS, so that a wavefront only ever waits for what
// was asked for a whole block's products before.
//
// 4,096 rows through a gated pair of 4,096 by 12,288 take 414 to 506 us, 1.6 to 2.0
// PFLOP/s; the products alone, from registers, take 290 to 330 (the card lowers its
// clock). The matrix cores are busy for 0.48 of the cycles: at the barrier of every 64
// columns all loads are waited for, and half of the wavefronts' cycles go by waiting to
// issue. Rows through registers and weights straight from memory by both their readers
// took 506 to 574: of that 82 went with the rows' loads left out, 70 with the weights',
// 213 with both, the L1's 64 bytes a cycle being shared by the two.
template <bool GATED>
__global__ void __launch_bounds__(kThreads, 2) w4_planes_kernel(ProductArgs a, const uint8_t* laid_rows) {
    constexpr int TILE = 1024;  // bytes of 32 columns of the matrix
    constexpr int BLOCK = 8 * TILE + kPlanesBlock, ROW_PIECES = kPlanesBlock / 1024 / 4;
    constexpr int EACH = GATED ? 2 : 4;
    __shared__ u4 block_s[2][BLOCK / 16];  // [columns' tile][16 rows of it][lane], then the rows' block
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wave_columns = wave >> 1, wave_rows = wave & 1;
    int row_block, column_block;
    find_block(a, &row_block, &column_block);
    const int blocks = (int)w4_ceil(a.depth, kTileDepth), steps = (int)w4_steps(a.depth), words = (int)w4_words(a.depth);
    const int last_tile = (int)w4_tiles(a.n) - 1;
    // What this wavefront brings: two tiles of columns (tile `slot` of 4 for each half of
    // the work-group; columns behind the end are those at the end again, and not
    // stored) and three pieces of the rows.
    const int tile0 = min(column_block * 2 * EACH * 2, last_tile);
    uint32_t code_place[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int slot = wave % 2 * 2 + k, column = (column_block * 2 + wave / 2) * EACH * 32 + slot % EACH * 32;
        code_place[k] = (min(column / kW4Rows + lane / 32, last_tile) - tile0) * steps * 1024 + lane % 32 * 16;
    }
    const uint8_t* const codes_at =
        reinterpret_cast<const uint8_t*>(a.m[GATED ? wave % 2 : 0].codes) + (int64_t)tile0 * steps * 1024;
    const uint8_t* const rows_at = laid_rows + (size_t)row_block * blocks * kPlanesBlock + wave * 1024;
    auto bring_block = [&](int block, int buffer) {
        uint8_t* const to = reinterpret_cast<uint8_t*>(block_s[buffer]);
#pragma unroll
        for (int k = 0; k < 2; ++k) bring(codes_at + block * 512 + code_place[k], to + (wave * 2 + k) * TILE);
#pragma unroll
        for (int k = 0; k < ROW_PIECES; ++k)
            bring(rows_at + (size_t)block * kPlanesBlock + k * 4096 + (uint32_t)lane * 16,
                  to + 8 * TILE + (k * 4 + wave) * 1024);
    };
    // The scales: a word for 8 blocks of a tile of columns and a half of 128 columns,
    // and one for both planes and halves of a tile of rows.
    const int first_column = (column_block * 2 + wave_columns) * EACH * 32;
    uint32_t scale_place[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        scale_place[i] = (min((first_column + i * 32) / kW4Rows + lane % 32 / 16, last_tile) - tile0) * words * 256 +
                         (lane / 32 * 16 + lane % 16) * 4;
    uint32_t scale[2][4], scale_next[2][4];
    auto load_scales = [&](int word) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t* const from =
                reinterpret_cast<const uint8_t*>(a.m[i / EACH].scales) + ((int64_t)tile0 * words + min(word, words - 1)) * 256;
#pragma unroll
            for (int half = 0; half < 2; ++half)
                scale_next[half][i] = *reinterpret_cast<const uint32_t*>(from + scale_place[i % EACH] + half * 128);
        }
    };
    const uint8_t* const powers_at = laid_rows + (size_t)a.row_blocks * blocks * kPlanesBlock +
                                     ((size_t)row_block * steps * 4 + wave_rows * 2) * 256;
    int power[2], power_next[2];
    auto load_powers = [&](int step) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
            power_next[j] = *reinterpret_cast<const int*>(powers_at + (size_t)min(step, steps - 1) * 1024 + j * 256 + (uint32_t)lane * 4);
    };
    struct Operands {
        u4 codes[4], rows[2][2];
        uint2 rest[2][2];
    } even, odd;
    auto take = [&](int buffer, Operands* to) {
        const uint8_t* const from = reinterpret_cast<const uint8_t*>(block_s[buffer]);
        const uint8_t* const columns = from + wave_columns * 4 * TILE + lane % 32 / 16 * 512 + (lane / 32 * 16 + lane % 16) * 16;
        const uint8_t* const rows = from + 8 * TILE + wave_rows * 4 * kPlaneBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) to->codes[i] = *reinterpret_cast<const u4*>(columns + i * TILE);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                to->rows[j][p] = *reinterpret_cast<const u4*>(rows + (j * 2 + p) * kPlaneBytes + lane * 16);
                to->rest[j][p] = *reinterpret_cast<const uint2*>(rows + (j * 2 + p) * kPlaneBytes + 1024 + lane * 8);
            }
    };
    f16v sum[4][2] = {};
    // Multiplies a block from `now`, as the HALF of a step of 128 columns, while the next is taken.
    auto step = [&](int block, auto half, const Operands& now, Operands* next) {
        constexpr int HALF = decltype(half)::value;
        const int shift = 8 * (block / 2 % kW4Word);
        uint32_t s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = scale[HALF][i] >> shift;
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's part of the next block is in LDS
        __syncthreads();                     // and everybody's, and nobody reads this one any more
        take(HALF ^ 1, next);
        bring_block(min(block + 2, blocks - 1), HALF);
        if constexpr (HALF == 0) load_powers(block / 2 + 1);
        if (HALF == 1 && block % 8 == 7) load_scales(block / 8 + 1);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const u4& x = now.rows[j][p];
                const v8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)now.rest[j][p].x, (int)now.rest[j][p].y, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u4& q = now.codes[i];
                    const v8 c = {(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
                    // Formats 4 and 2: E2M1 and E2M3; a byte of the words of scales.
                    sum[i][j] = p == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(c, b, sum[i][j], 4, 2, 0, (int)s[i],
                                                                                         2 * HALF, power[j])
                                       : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(c, b, sum[i][j], 4, 2, 0, (int)s[i],
                                                                                         2 * HALF + 1, power[j]);
                }
            }
    };
    bring_block(0, 0);
    load_scales(0);
    load_powers(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    take(0, &even);
    bring_block(min(1, blocks - 1), 1);
    for (int block = 0; block < blocks; block += 2) {
        if (block % 8 == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) scale[0][i] = scale_next[0][i], scale[1][i] = scale_next[1][i];
        }
        power[0] = power_next[0], power[1] = power_next[1];
        step(block, std::integral_constant<int, 0>(), even, &odd);
        if (block + 1 < blocks) step(block + 1, std::integral_constant<int, 1>(), odd, &even);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // nothing is on its way to LDS when the work-group gives it up
    store_tiles<4, 2, GATED>(a, (int64_t)row_block * kTileRows + wave_rows * 64, first_column, sum);
}

void blocks_of(ProductArgs* a, int rows, int columns) {
    a->row_blocks = (int)w4_ceil(a->rows, rows);
    a->column_blocks = (int)w4_ceil(a->n, columns);
}

template <int KIND, bool GATED>
void tiles(ProductArgs a, bool large, hipStream_t s) {
    blocks_of(&a, large ? kTileRows : kSmallTileRows, (large ? kTileColumns : kSmallTileColumns) / (GATED ? 2 : 1));
    const unsigned groups = (unsigned)(a.row_blocks * (int64_t)a.column_blocks);
    if constexpr (KIND != MP_TYPE_I8) {  // whose large tiles have planes
        if (large) return w4_tiles_kernel<KIND, GATED, 4, 2, 2, 2><<<groups, 256, 0, s>>>(a);
    }
    w4_tiles_kernel<KIND, GATED, 2, 1, 2, 2><<<groups, 256, 0, s>>>(a);
}
template <int KIND>
void tiles(const ProductArgs& a, bool gate, bool large, hipStream_t s) {
    if (gate) tiles<KIND, true>(a, large, s);
    else tiles<KIND, false>(a, large, s);
}
template <bool GATED>
void planes(ProductArgs a, uint8_t* laid, hipStream_t s) {
    blocks_of(&a, kTileRows, kTileColumns / (GATED ? 2 : 1));
    w4_planes_layout_kernel<<<(unsigned)w4_planes_blocks(a.rows, a.depth), kThreads, 0, s>>>(a, laid);
    w4_planes_kernel<GATED><<<(unsigned)(a.row_blocks * (int64_t)a.column_blocks), kThreads, 0, s>>>(a, laid);
}

}  // namespace

void w4_tiles(const ProductArgs& a, int kind, bool gate, bool large, void* workspace, hipStream_t s) {
    uint8_t* const laid = static_cast<uint8_t*>(workspace);
    if (kind == MP_TYPE_F32) tiles<MP_TYPE_F32>(a, gate, large, s);
    else if (kind == MP_TYPE_BF16) tiles<MP_TYPE_BF16>(a, gate, large, s);
    else if (kind == MP_TYPE_F16) tiles<MP_TYPE_F16>(a, gate, large, s);
    else if (!large) tiles<MP_TYPE_I8>(a, gate, false, s);
    else if (gate) planes<true>(a, laid, s);
    else planes<false>(a, laid, s);
}

}  // namespace mphip
