// Attention over the 8-bit paged K/V cache on the FP16 matrix cores
// (v_mfma_f32_16x16x32_f16), decode and prefill.
//
// out = sum_t p_t v_t / sum_t p_t, p_t = exp(scale q.k_t - m), over the
// tokens a row may see, in one pass with a running reference m per row and
// head (flash attention). A "column" is one (row, query head) of a KV head;
// the products are taken transposed, so that a column's scores and
// probabilities stay in the lanes that made them (kv8.h has the layouts):
//   S^T[token][column] = K Q^T,   O^T[dim][column] += V^T P^T.
//
// Exactness. Codes of 8 bits are exact in FP16, and their products with FP16
// numbers exact in FP32. An FP32 query, scaled by a power of two so that its
// largest element lies in [2^14, 2^15), is the sum of two FP16 numbers to
// 2^-23 of an element (2^-39 of the largest); so is a probability, which is
// kept below 2^15. Two matrix products, of the high and the low parts, into
// one FP32 sum then give FP32 accuracy at half the FP16 rate, 8 times the
// FP32 matrix rate. How the two parts are arranged is the kernel's mode:
// - kPacked: up to 8 query heads a KV head, one row: columns 0..7 hold the
//   high and columns 8..15 the low parts of the same heads, so the second
//   product costs nothing;
// - kTwo: two products into the same sums;
// - kOne: FP16 and BF16 rows: a query element is one FP16 number (2^-12 for
//   FP16's and BF16's own bits: exact, but for elements below 2^-29 of the
//   largest), a probability is rounded to FP16 (2^-12 of its size, a
//   sixteenth of a BF16 output's step).
// The key scale multiplies the score with the softmax scale; the value scale,
// as a power of two relative to the largest met so far, is applied with the
// conversion of the value codes, where it is exact.
#include "kernels.h"
#include "kv8.h"

// The summation order is the kernels' own: multiply-adds may be fused.
#pragma clang fp contract(fast)

namespace mphip {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

enum Mode { kPacked, kTwo, kOne };

constexpr float kShift = 11.0f;  // probabilities are held times 2^11 ...
constexpr float kRaise = 15.0f;  // ... and below 2^15: past it the reference is raised

struct AttentionArgs {
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

// Of the four lanes (c, 0..3) of a column.
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
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

// One tile's bytes as a lane holds them, and its scales' bits (uniform).
template <int DIM>
struct RawTile {
    u4 k[DIM / 64], v[DIM / 64];
    uint32_t k_scale, v_scale;
};

template <int DIM>
__device__ __forceinline__ void load_tile(const Kv8Layer& kv, int head, int block, int tile, int lane,
                                          RawTile<DIM>* out) {
    const size_t index = kv8_head(kv, max(block, 0), head);
    const size_t base = index * ((size_t)DIM << kv.page_shift) +
                        (tile & ((1 << (kv.page_shift - 4)) - 1)) * (kTile * DIM) + 16 * lane;
#pragma unroll
    for (int j = 0; j < DIM / 64; ++j) {
        out->k[j] = *reinterpret_cast<const u4*>(kv.keys + base + 1024 * j);
        out->v[j] = *reinterpret_cast<const u4*>(kv.values + base + 1024 * j);
    }
    const float2 s = kv.scales[index];
    const uint32_t bad = 0x7FC00000u;  // NaN for a page that is none
    out->k_scale = __builtin_amdgcn_readfirstlane(block < 0 ? bad : __float_as_uint(s.x));
    out->v_scale = __builtin_amdgcn_readfirstlane(block < 0 ? bad : __float_as_uint(s.y));
}

// DECODE: one row a sequence, its columns the KV head's query heads; else
// columns are those of a sequence's rows, row major.
template <int FORMAT, int DIM, int NT, int MODE, bool DECODE>
__global__ __launch_bounds__(512, 2) void kv8_attention_kernel(AttentionArgs a) {
    constexpr int kSteps = DIM / 32;             // of the contraction over dims
    constexpr int kDims = DIM / 16;              // 16-dim tiles of the output
    constexpr int kParts = MODE == kTwo ? 2 : 1;  // operands of a query or probability
    constexpr int kColumns = MODE == kPacked ? 8 : 16;
    static_assert(MODE != kPacked || (NT == 1 && DECODE), "one row's heads");
    __shared__ f4 o_s[8][NT][64];
    __shared__ float2 ml_s[8][NT][16];
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int head = blockIdx.y, split = blockIdx.z;

    // The work-group's columns, all of one sequence: rows row0.. and the
    // position of the first, `first` columns into the sequence's.
    int sequence, row0, count, used, first;
    if (DECODE) {
        sequence = row0 = blockIdx.x;
        count = 1;
        const int length = a.rows.used[sequence];
        used = min(length, a.max_length + 1) - 1;
        first = 0;
        if (length <= 0) {  // nothing to see: zeros
            if (split) return;
            for (int i = threadIdx.x; i < a.group * DIM; i += blockDim.x)
                store_one(a.out, a.type, row0 * a.out_stride + (int64_t)head * a.group * DIM + i, 0.0f);
            return;
        }
    } else {
        Kv8Item at;
        const int group = a.group;
        if (!kv8_find(a.rows, blockIdx.x, [=](int n, int) { return (n * group + 16 * NT - 1) / (16 * NT); }, &at))
            return;
        sequence = at.sequence;
        row0 = at.row0;
        count = at.count;
        used = at.used;
        // The last columns see the most tokens: they start first.
        first = ((count * group - 1) / (16 * NT) - at.index) * (16 * NT);
    }
    const int columns = count * a.group;
    const int last = used + (min(first + kColumns * NT, columns) - 1) / a.group;  // position of the last row
    if (used < 0 || used >= a.max_length || last >= a.max_length) {  // more than the caller allowed for
        if (split) return;
        for (int i = threadIdx.x; i < kColumns * NT * DIM; i += blockDim.x) {
            const int column = first + i / DIM;
            if (column < columns)
                store_one(a.out, a.type,
                          (row0 + column / a.group) * a.out_stride +
                              ((int64_t)head * a.group + column % a.group) * DIM + i % DIM,
                          quiet_nan());
        }
        return;
    }
    const int begin = split * a.chunk, end = min(begin + a.chunk, last + 1);  // tokens of this work-group
    if (begin >= end) return;
    const bool alone = last < a.chunk;  // the columns' tokens are one chunk

    // This lane's column in each column tile.
    int qpos[NT];
    int64_t q_at[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int column = min(first + 16 * t + (MODE == kPacked ? c & 7 : c), columns - 1);
        const int row = column / a.group;
        qpos[t] = used + row;
        q_at[t] = (row0 + row) * a.q_stride + ((int64_t)head * a.group + column % a.group) * DIM;
    }

    // Pairs of tiles: first + wave, + waves, ... of the chunk's.
    const int32_t* const table = a.rows.tables + (size_t)sequence * a.rows.table_stride;
    const int tile_end = (end + kTile - 1) / kTile;
    const int pair_end = (tile_end + 1) / 2;
    int pair = begin / kKv8Pair + wave;
    RawTile<DIM> next[2];
    int block[2];
    const auto find_blocks = [&](int p) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            block[h] = __builtin_amdgcn_readfirstlane(
                kv8_block(table, a.rows.table_stride, min(2 * p + h, tile_end - 1) >> (a.kv.page_shift - 4),
                          a.kv.blocks));
    };
    const auto load_pair = [&](int p) {
#pragma unroll
        for (int h = 0; h < 2; ++h) load_tile<DIM>(a.kv, head, block[h], min(2 * p + h, tile_end - 1), lane, &next[h]);
    };
    if (pair < pair_end) {
        find_blocks(pair);
        load_pair(pair);
        find_blocks(min(pair + waves, pair_end - 1));
    }

    // Queries: part, column tile, step (j, h): dims 64j + 16g + 8h .. +7.
    Half8 q[kParts][NT][kSteps];
    float factor[NT];  // of a score: softmax scale / the query's power of two
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float x[DIM / 64][16];
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < DIM / 64; ++j) {
            load_row<16>(a.q, a.type, a.q_wide, q_at[t] + 64 * j + 16 * g, x[j]);
#pragma unroll
            for (int i = 0; i < 16; ++i) amax = max(amax, __float_as_uint(x[j][i]) & 0x7FFFFFFFu);
        }
        amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16));
        amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
        const int power = min(127 + 14 - (int)(amax >> 23), 126);  // at least -113
        const float up = __uint_as_float((uint32_t)(127 + power) << 23);
        factor[t] = amax >= 0x7F800000u ? quiet_nan() : a.scale * __uint_as_float((uint32_t)(127 - power) << 23);
#pragma unroll
        for (int j = 0; j < DIM / 64; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float v = x[j][i] * up;
                const _Float16 high = (_Float16)v, low = (_Float16)(v - (float)high);
                if (MODE == kPacked) q[0][t][2 * j + i / 8].one[i % 8] = c & 8 ? low : high;
                else q[0][t][2 * j + i / 8].one[i % 8] = high;
                if (MODE == kTwo) q[kParts - 1][t][2 * j + i / 8].one[i % 8] = low;
            }
    }

    f4 o[NT][kDims];
    float ref[NT], sum[NT];  // reference less kShift, this lane's share of the sum
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        ref[t] = -infinity();
        sum[t] = 0.0f;
#pragma unroll
        for (int n = 0; n < kDims; ++n) o[t][n] = f4{0.f, 0.f, 0.f, 0.f};
    }
    uint32_t v_top = 0;  // bits of the value scale that o is held in

    for (; pair < pair_end; pair += waves) {
        RawTile<DIM> now[2] = {next[0], next[1]};
        if (pair + waves < pair_end) {
            load_pair(pair + waves);
            find_blocks(min(pair + 2 * waves, pair_end - 1));
        }
        f4 s[NT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][h] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                Half8 k;
                Convert<FORMAT>::plain(now[h].k[i / 2][2 * (i % 2)], &k.two[0], &k.two[1]);
                Convert<FORMAT>::plain(now[h].k[i / 2][2 * (i % 2) + 1], &k.two[2], &k.two[3]);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int part = 0; part < kParts; ++part)
                        s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.all, q[part][t][i].all, s[t][h], 0, 0, 0);
            }
        }
        if (MODE == kPacked) {  // the low parts' scores are 8 columns on
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[0][h][i] += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
                        0, __float_as_int(s[0][h][i]), 0x128, 0xF, 0xF, true));
        }
        const int token0 = pair * kKv8Pair;
        const bool masked = token0 + kKv8Pair - 1 > (DECODE ? last : used + first / a.group);
        const float k_scale[2] = {__uint_as_float(now[0].k_scale), __uint_as_float(now[1].k_scale)};
        // Scores in powers of two less the reference; the reference is
        // raised only where one is past kRaise.
        bool need = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float f[2] = {factor[t] * k_scale[0], factor[t] * k_scale[1]};
            float top = -infinity();
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[t][h][i] *= f[h];
                    if (masked && token0 + kTile * h + 4 * g + i > qpos[t]) s[t][h][i] = -infinity();
                    top = fmaxf(top, s[t][h][i]);
                }
            need |= top > ref[t] + kRaise;
        }
        if (__builtin_amdgcn_ballot_w64(need)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float top = -infinity();
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][h][i]);
                top = column_max(top);
                if (top > ref[t] + kRaise) {
                    const float to = top - kShift;
                    const float keep = __builtin_amdgcn_exp2f(ref[t] - to);  // 0 from -inf
                    ref[t] = to;
                    sum[t] *= keep;
#pragma unroll
                    for (int n = 0; n < kDims; ++n) o[t][n] *= keep;
                }
            }
        }
        // The value scale: o is held in the largest met so far.
        const uint32_t v_now = max(now[0].v_scale, now[1].v_scale);
        if (v_now > v_top) {
            if (v_top) {
                const float keep = __uint_as_float(v_top) / __uint_as_float(v_now);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int n = 0; n < kDims; ++n) o[t][n] *= keep;
            }
            v_top = v_now;
        }
        Half8 p[kParts][NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float base = ref[t] == -infinity() ? 0.0f : ref[t];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(s[t][h][i] - base);
                    sum[t] += e;
                    const _Float16 high = (_Float16)e;
                    const _Float16 low = (_Float16)(e - (float)high);
                    if (MODE == kPacked) p[0][t].one[4 * h + i] = c & 8 ? low : high;
                    else p[0][t].one[4 * h + i] = high;
                    if (MODE == kTwo) p[kParts - 1][t].one[4 * h + i] = low;
                }
        }
        // Powers of two of the tiles' values; 2^-40 of the top one is nothing.
        const auto power = [&](uint32_t v) {
            return __uint_as_float((uint32_t)max((int)(v - v_top) + (127 << 23), (127 - 40) << 23));
        };
        const Convert<FORMAT> convert0(power(now[0].v_scale)), convert1(power(now[1].v_scale));
        // Slots past the last row's position may hold anything: as bytes they
        // are made 0 where an E4M3 NaN could be (INT8 codes are finite, and
        // their probability is 0).
        uint32_t keep0 = ~0u, keep1 = ~0u;
        if (FORMAT == MP_KV8_E4M3 && token0 + kKv8Pair - 1 > last) {
            const int left0 = last + 1 - token0 - 4 * g, left1 = left0 - kTile;
            keep0 = left0 >= 4 ? ~0u : left0 <= 0 ? 0u : (1u << (8 * left0)) - 1;
            keep1 = left1 >= 4 ? ~0u : left1 <= 0 ? 0u : (1u << (8 * left1)) - 1;
        }
#pragma unroll
        for (int n = 0; n < kDims; ++n) {
            Half8 v;
            convert0(now[0].v[n / 4][n % 4] & keep0, &v.two[0], &v.two[1]);
            convert1(now[1].v[n / 4][n % 4] & keep1, &v.two[2], &v.two[3]);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int part = 0; part < kParts; ++part)
                    o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v.all, p[part][t].all, o[t][n], 0, 0, 0);
        }
    }

    // Each wavefront's result as values: o / sum in the value scale.
    float weight[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        sum[t] = column_sum(sum[t]);
        if (MODE == kPacked) {
#pragma unroll
            for (int n = 0; n < kDims; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][n][i] += __shfl_xor(o[t][n][i], 8);
        }
        weight[t] = sum[t] == 0.0f ? 0.0f : __uint_as_float(v_top) / sum[t];
    }
    float best[NT], total[NT];
    if (waves > 1) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
            if (g == 0) ml_s[wave][t][c] = make_float2(ref[t], sum[t]);
        __syncthreads();
    }
    // Reference and sum over the wavefronts, and this one's share.
    float share[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        best[t] = ref[t];
        total[t] = sum[t];
        share[t] = sum[t];
        if (waves > 1) {
            best[t] = -infinity();
            for (int w = 0; w < waves; ++w) best[t] = fmaxf(best[t], ml_s[w][t][c].x);
            total[t] = 0.0f;
            for (int w = 0; w < waves; ++w) {
                const float2 ml = ml_s[w][t][c];
                if (ml.y != 0.0f) total[t] += ml.y * __builtin_amdgcn_exp2f(ml.x - best[t]);
            }
            share[t] = sum[t] == 0.0f ? 0.0f : sum[t] * __builtin_amdgcn_exp2f(ref[t] - best[t]);
        }
        weight[t] = share[t] == 0.0f ? 0.0f : weight[t] * (share[t] / total[t]);
    }
    const auto store = [&](int t, int n, f4 x) {
        const int column = first + 16 * t + c;
        if ((MODE == kPacked && c >= a.group) || column >= columns) return;
        const int row = row0 + column / a.group, at_head = head * a.group + column % a.group;
        const int d = 16 * n + 4 * g;
        if (alone) {
            store_four(a.out, a.type, a.out_wide, row * a.out_stride + (int64_t)at_head * DIM + d, x[0], x[1], x[2],
                       x[3]);
        } else {
            const size_t at = ((size_t)row * a.heads + at_head) * a.splits + split;
            *reinterpret_cast<float2*>(a.partial_out + at * DIM + d) = make_float2(x[0], x[1]);
            *reinterpret_cast<float2*>(a.partial_out + at * DIM + d + 2) = make_float2(x[2], x[3]);
            if (n == 0 && g == 0) a.partial_ml[at] = make_float2(best[t], total[t]);
        }
    };
    if (waves == 1) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int n = 0; n < kDims; ++n) store(t, n, o[t][n] * weight[t]);
        return;
    }
#pragma unroll
    for (int n = 0; n < kDims; ++n) {
#pragma unroll
        for (int t = 0; t < NT; ++t) o_s[wave][t][lane] = o[t][n] * weight[t];
        __syncthreads();
        for (int t = wave; t < NT; t += waves) {
            f4 x = o_s[0][t][lane];
            for (int w = 1; w < waves; ++w) x += o_s[w][t][lane];
#pragma unroll
            for (int u = 0; u < NT; ++u)
                if (u == t) store(u, n, x);
        }
        __syncthreads();
    }
}

// Joins the chunks of rows that have several: one wavefront a (row, head),
// lanes over dims. `columns_tile`: columns of an attention work-group.
template <bool DECODE>
__global__ __launch_bounds__(256) void kv8_merge_kernel(AttentionArgs a, int columns_tile) {
    const int lane = threadIdx.x & 63, dim = a.kv.dim;
    const int index = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = index % a.heads;
    int row = index / a.heads, last;
    if (row >= a.rows.rows) return;
    if (DECODE) {
        last = a.rows.used[row] - 1;
    } else {
        Kv8Item at;
        if (!kv8_find(a.rows, row, [](int n, int) { return n; }, &at)) return;
        row = at.row0 + at.index;
        if (at.used < 0 || at.used >= a.max_length) return;
        const int column = at.index * a.group + head % a.group;
        const int end = min((column / columns_tile + 1) * columns_tile, at.count * a.group);
        last = at.used + (end - 1) / a.group;  // of the work-group that had this column
    }
    // One chunk (or none) was stored by its work-group, as were NaN rows.
    if (last < a.chunk || last >= a.max_length) return;
    const int chunks = last / a.chunk + 1;
    const size_t at = ((size_t)row * a.heads + head) * a.splits;
    float best = -infinity();
    for (int b = lane; b < chunks; b += 64) best = fmaxf(best, a.partial_ml[at + b].x);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) best = fmaxf(best, __shfl_xor(best, d));
    float total = 0.0f, out[4] = {0.f, 0.f, 0.f, 0.f};
    for (int b = 0; b < chunks; b += 64) {
        float w = 0.0f;
        if (b + lane < chunks) {
            const float2 ml = a.partial_ml[at + b + lane];
            if (ml.y != 0.0f) w = ml.y * __builtin_amdgcn_exp2f(ml.x - best);
        }
        const int n = min(64, chunks - b);
        for (int i = 0; i < n; ++i) {
            const float wi = __shfl(w, i);
            total += wi;
            const float* part = a.partial_out + (at + b + i) * dim + lane;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (64 * k < dim) out[k] += wi * part[64 * k];
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (64 * k < dim)
            store_one(a.out, a.type, row * a.out_stride + (int64_t)head * dim + 64 * k + lane, out[k] / total);
}

// Column tiles that a prefill wavefront holds in its registers.
constexpr int most_tiles(int dim, int mode) {
    return dim == 64 ? 4 : dim == 128 ? (mode == kTwo ? 2 : 4) : (mode == kTwo ? 1 : 2);
}

template <int FORMAT, int DIM, int NT, int MODE, bool DECODE>
void launch(hipStream_t s, const Kv8Plan& p, int64_t items, const AttentionArgs& a) {
    const dim3 grid((unsigned)items, (unsigned)a.kv.kv_heads, (unsigned)p.splits);
    kv8_attention_kernel<FORMAT, DIM, NT, MODE, DECODE><<<grid, 64 * p.waves, 0, s>>>(a);
}
template <int FORMAT, int DIM>
void launch_decode(hipStream_t s, const Kv8Plan& p, const AttentionArgs& a) {
    if (a.group <= 8) launch<FORMAT, DIM, 1, kPacked, true>(s, p, a.rows.rows, a);
    else launch<FORMAT, DIM, 1, kTwo, true>(s, p, a.rows.rows, a);
}
template <int FORMAT, int DIM, int MODE>
void launch_prefill(hipStream_t s, const Kv8Plan& p, const AttentionArgs& a) {
    const int64_t items = kv8_items(a.rows.rows, a.rows.sequences, a.group, p.column_tiles);
    constexpr int kMost = most_tiles(DIM, MODE);
    if (p.column_tiles == 4) {
        if constexpr (kMost >= 4) launch<FORMAT, DIM, 4, MODE, false>(s, p, items, a);
    } else if (p.column_tiles == 2) {
        if constexpr (kMost >= 2) launch<FORMAT, DIM, 2, MODE, false>(s, p, items, a);
    } else {
        launch<FORMAT, DIM, 1, MODE, false>(s, p, items, a);
    }
}
template <int FORMAT, int DIM>
void launch_attention(hipStream_t s, const Kv8Plan& p, const AttentionArgs& a, bool decode) {
    if (decode) launch_decode<FORMAT, DIM>(s, p, a);
    else if (a.type == MP_TYPE_F32) launch_prefill<FORMAT, DIM, kTwo>(s, p, a);
    else launch_prefill<FORMAT, DIM, kOne>(s, p, a);
}
template <int FORMAT>
void launch_format(hipStream_t s, const Kv8Plan& p, const AttentionArgs& a, bool decode) {
    if (a.kv.dim == 64) launch_attention<FORMAT, 64>(s, p, a, decode);
    else if (a.kv.dim == 128) launch_attention<FORMAT, 128>(s, p, a, decode);
    else launch_attention<FORMAT, 256>(s, p, a, decode);
}

const char* wrong_attention(const mp_kv8_cache* c, int layer, int heads, int max_length) {
    if (const char* wrong = kv8_wrong_cache(c, layer)) return wrong;
    if (heads < 1 || heads > kKv8MaxHeads || heads % c->kv_heads || heads / c->kv_heads > kKv8MaxGroup)
        return "8-bit attention: heads must be a multiple of kv_heads, at most 16 of them each and 1,024 in all";
    if (max_length < 0 || max_length > kKv8MaxLength) return "8-bit attention: max_length must be 0 to 2^30";
    return nullptr;
}

// Both entries; starts is null for decode, whose `used` are the lengths.
int attention(const mp_kv8_cache* cache, int layer, const void* q, int64_t q_stride, int type, const int32_t* tables,
              int table_stride, const int32_t* starts, const int32_t* used, int sequences, int rows, int heads,
              int max_length, float scale, void* out, int64_t out_stride, void* workspace, size_t workspace_bytes,
              void* stream, bool decode) {
    const char* wrong = wrong_attention(cache, layer, heads, max_length);
    if (!wrong) wrong = kv8_wrong_rows(tables, table_stride, sequences, rows);
    if (!wrong) wrong = kv8_wrong_matrix(q, q_stride, (int64_t)heads * cache->dim, type);
    if (!wrong) wrong = kv8_wrong_matrix(out, out_stride, (int64_t)heads * cache->dim, type);
    if (wrong) return kv8_refuse(wrong);
    if (kv8_bad_ints(used) || (!decode && kv8_bad_ints(starts)))
        return kv8_refuse("8-bit attention: lengths, starts or used are missing or misaligned");
    if (!isfinite(scale) || scale < 0) return kv8_refuse("8-bit attention: scale must be finite and not negative");
    if (rows == 0 || sequences == 0) return MP_OK;
    const int group = heads / cache->kv_heads;
    const Kv8Plan p = decode ? kv8_decode_plan(rows, cache->kv_heads, max_length)
                             : kv8_prefill_plan(rows, sequences, cache->kv_heads, group,
                                                most_tiles(cache->dim, type == MP_TYPE_F32 ? kTwo : kOne), max_length);
    const size_t need = kv8_partial_floats(p, rows, heads, cache->dim) * sizeof(float);
    if (need > workspace_bytes || (need && !workspace))
        return kv8_refuse("8-bit attention: the workspace is smaller than mp_hip_kv8_attention_workspace says");
    if (need && reinterpret_cast<uintptr_t>(workspace) % 16)
        return kv8_refuse("8-bit attention: the workspace must be 16-byte aligned");
    AttentionArgs a{};
    a.kv = kv8_layer(*cache, layer);
    a.rows = Kv8Rows{tables, starts, used, table_stride, sequences, rows};
    a.q = q, a.out = out;
    a.q_stride = q_stride, a.out_stride = out_stride;
    a.heads = heads, a.group = group, a.type = type, a.max_length = max_length;
    a.chunk = p.chunk, a.splits = p.splits;
    a.scale = (float)(scale * 1.4426950408889634074);
    a.q_wide = kv8_wide(q, q_stride, type), a.out_wide = kv8_wide(out, out_stride, type);
    a.partial_out = static_cast<float*>(workspace);
    a.partial_ml = reinterpret_cast<float2*>(a.partial_out + (need ? (size_t)rows * heads * p.splits * cache->dim : 0));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const StreamDevice device(s);
    if (device.status != hipSuccess) return kv8_done(device.status, "8-bit attention: device of the stream");
    if (cache->format == MP_KV8_INT8) launch_format<MP_KV8_INT8>(s, p, a, decode);
    else launch_format<MP_KV8_E4M3>(s, p, a, decode);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && p.splits > 1) {
        const unsigned groups = (unsigned)(((int64_t)rows * heads + 3) / 4);
        if (decode) kv8_merge_kernel<true><<<groups, 256, 0, s>>>(a, 16);
        else kv8_merge_kernel<false><<<groups, 256, 0, s>>>(a, 16 * p.column_tiles);
        e = hipGetLastError();
    }
    return kv8_done(e, "8-bit attention launch");
}

}  // namespace
}  // namespace mphip

extern "C" int mp_hip_kv8_attention_workspace(const mp_kv8_cache* cache, int32_t rows, int32_t sequences,
                                              int32_t heads, int32_t max_length, size_t* bytes) {
    using namespace mphip;
    return kv8_entry([&]() -> int {
        if (!bytes) return kv8_refuse("8-bit attention: no place for the workspace's size");
        if (const char* wrong = wrong_attention(cache, 0, heads, max_length)) return kv8_refuse(wrong);
        if (sequences < 0 || sequences > kKv8MaxRows || rows < 0 || rows > kKv8MaxRows)
            return kv8_refuse("8-bit cache: sequences and rows must be 0 to 1,048,576");
        *bytes = kv8_workspace_floats(rows, sequences, heads, cache->kv_heads, cache->dim, max_length) * sizeof(float);
        return MP_OK;
    });
}

extern "C" int mp_hip_kv8_attention_decode(const mp_kv8_cache* cache, int32_t layer, const void* q, int64_t q_stride,
                                           int32_t type, const int32_t* tables, int32_t table_stride,
                                           const int32_t* lengths, int32_t rows, int32_t heads, int32_t max_length,
                                           float scale, void* out, int64_t out_stride, void* workspace,
                                           size_t workspace_bytes, void* stream) {
    using namespace mphip;
    return kv8_entry([&]() -> int {
        return attention(cache, layer, q, q_stride, type, tables, table_stride, nullptr, lengths, rows, rows, heads,
                         max_length, scale, out, out_stride, workspace, workspace_bytes, stream, true);
    });
}

extern "C" int mp_hip_kv8_attention_prefill(const mp_kv8_cache* cache, int32_t layer, const void* q, int64_t q_stride,
                                            int32_t type, const int32_t* tables, int32_t table_stride,
                                            const int32_t* starts, const int32_t* used, int32_t sequences,
                                            int32_t rows, int32_t heads, int32_t max_length, float scale, void* out,
                                            int64_t out_stride, void* workspace, size_t workspace_bytes,
                                            void* stream) {
    using namespace mphip;
    return kv8_entry([&]() -> int {
        return attention(cache, layer, q, q_stride, type, tables, table_stride, starts, used, sequences, rows, heads,
                         max_length, scale, out, out_stride, workspace, workspace_bytes, stream, false);
    });
}
