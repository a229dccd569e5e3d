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
// - kOne: FP16 and BF16 rows: a query element is one FP16 number (FP16's and
//   BF16's own bits: exact down to 2^-39 of the largest), so the scores take
//   one product; a probability is two, as for FP32 rows. In one FP16 number it
//   is off by up to 2^-11 of its size, as much as an FP16 result is rounded by,
//   and more than that where values cancel: 331-339 instead of 269-280 us for
//   16.8k BF16 rows of prompts keep a row as exact as the decode of it.
// The key scale multiplies the score with the softmax scale; the value scale,
// as a power of two relative to the largest met so far, is applied with the
// conversion of the value codes, where it is exact (value_power; a column's
// sums keep the largest scale that it has seen itself).
//
// What bounds it. Decode: memory, 5.3 TB/s over 256 rows of about 1,050 tokens,
// 8 heads of 128 in E4M3 (558 MB in 105 us, 564 MB by the counters); rows of a
// few hundred tokens the chain of launch, table, first tiles and joining (6.9 us
// for one of 503).
// Prefill: the vector unit beside the matrix cores, 0.76 and 0.46 of a SIMD's
// cycles for 8 x 512 FP32 rows at 8,192 (186-210 us, 0.8 PFLOP/s of products
// counting both parts; a large FP16 matrix product reaches 1.15 here), 0.68 and
// 0.46 for 16.8k BF16 rows of prompts (331-339 us, 0.84 PFLOP/s). Of about 150
// vector instructions a step of 32 tokens and 32 columns, 64 convert codes, 16
// scale scores, 16 are exponentials (four cycles each) and 32 split probabilities.
// Hence: sums of probabilities by a matrix instruction (an operand of ones), the
// reference raised only past 2^15, masks under a branch, one test a pair of
// tiles, tile lookups by the lanes for 32 pairs at once instead of 90 scalar
// instructions a pair (decode of 64 rows 14.7 -> 13.2 us).
#include <type_traits>

#include "kernels.h"
#include "kv8_mma.h"

// The summation order is the kernels' own: multiply-adds may be fused.
#pragma clang fp contract(fast)

namespace mphip {
namespace {

// 16-dim tiles of every wavefront that meet in LDS at a time, in 32 KB of it
// where that holds one: 1 KB a tile, wavefront and column tile.
constexpr int join_dims(int waves, int column_tiles, int dims) {
    const int fit = 32 / (waves * column_tiles);
    return fit < 1 ? 1 : fit < dims ? fit : dims;
}
constexpr size_t join_bytes(int waves, int column_tiles, int dims) {
    return waves == 1 ? 0 : (size_t)waves * column_tiles * join_dims(waves, column_tiles, dims) * 1024;
}

// Wavefronts a SIMD that the registers are kept to.
constexpr int least_waves(int dim, int column_tiles, bool decode) {
    return !decode && dim == 64 && column_tiles == 2 ? 3 : 2;
}

// DECODE: one row a sequence, its columns the KV head's query heads; else
// columns are those of a sequence's rows, row major.
template <int FORMAT, int DIM, int NT, int MODE, bool DECODE>
__global__ __launch_bounds__(64 * kKv8MostWaves) __attribute__((amdgpu_waves_per_eu(least_waves(DIM, NT, DECODE)))) void
kv8_attention_kernel(Kv8Attention a) {
    constexpr int kDepth = DECODE && DIM < 256 ? 2 : 1;
    constexpr int kSteps = DIM / 32;             // of the contraction over dims
    constexpr int kDims = DIM / 16;              // 16-dim tiles of the output
    constexpr int kQueryParts = MODE == kTwo ? 2 : 1, kParts = MODE == kPacked ? 1 : 2;  // of a query, of a probability
    constexpr int kColumns = MODE == kPacked ? 8 : 16;
    static_assert(MODE != kPacked || (NT == 1 && DECODE), "one row's heads");
    extern __shared__ f4 shared_s[];  // join_bytes
    f4(*const o_s)[64] = reinterpret_cast<f4(*)[64]>(shared_s);
    float2(*const ml_s)[NT][16] = reinterpret_cast<float2(*)[NT][16]>(shared_s);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    // Neighbouring work-groups, on different XCDs, have different heads.
    const int head = blockIdx.x % a.kv.kv_heads, item = blockIdx.x / a.kv.kv_heads, split = blockIdx.z;

    // The work-group's columns, all of one sequence: rows row0.. and the
    // position of the first, `first` columns into the sequence's.
    int sequence = item, row0 = item, count = 1, used = 0, first = 0;
    if (!DECODE) {
        Kv8Item at;
        const int group = a.group;
        if (!kv8_find(a.rows, item, [=](int n, int) { return (n * group + 16 * NT - 1) / (16 * NT); }, &at)) return;
        sequence = at.sequence;
        row0 = at.row0;
        count = at.count;
        used = at.used;
        // The last columns see the most tokens: they start first.
        first = ((count * group - 1) / (16 * NT) - at.index) * (16 * NT);
    }
    const int columns = count * a.group, begin = split * a.chunk;
    // This wavefront's pairs of tiles: pair0, + waves, ... of the chunk's.
    const int pair0 = begin / kKv8Pair + wave;
    int row_of[NT];  // of this lane's column in each column tile
    int64_t q_at[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int column = min(first + 16 * t + (MODE == kPacked ? c & 7 : c), columns - 1);
        row_of[t] = column / a.group;
        q_at[t] = (row0 + row_of[t]) * a.q_stride + ((int64_t)head * a.group + column % a.group) * DIM;
    }
    // The table's first entries and the queries. A decode row's are on their
    // way while its length is (13.2 instead of 13.5 us for 64 ragged rows).
    const bool f32 = DECODE ? a.type == MP_TYPE_F32 : MODE == kTwo;
    Kv8Tiles<DIM, 2> tiles;
    int first_block;
    u4 raw_q[NT][DIM / 64][4];
    const auto first_loads = [&]() {
        first_block = tiles.begin(a, sequence, head, 2 * pair0, 2 * waves, lane);
        load_queries<DIM, NT>(a, f32, q_at, g, raw_q);
    };
    if (DECODE) {
        first_loads();
        const int length = scalar_int(a.rows.used, (uint32_t)sequence * 4u);
        used = min(length, a.max_length + 1) - 1;
        if (length <= 0) {  // nothing to see: zeros
            if (split) return;
            for (int i = threadIdx.x; i < a.group * DIM; i += blockDim.x)
                store_one(a.out, a.type, row0 * a.out_stride + (int64_t)head * a.group * DIM + i, 0.0f);
            return;
        }
    }
    // Position of the last row, of those within what the caller allowed for.
    const int last = min(used + (min(first + kColumns * NT, columns) - 1) / a.group, a.max_length - 1);
    if (used < 0 || used >= a.max_length) {  // none is
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
    const int end = min(begin + a.chunk, last + 1);  // of the tokens of this work-group
    if (begin >= end) return;
    const bool alone = last < a.chunk;  // the columns' tokens are one chunk
    if (!DECODE) first_loads();
    int qpos[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) qpos[t] = used + row_of[t];
    const int tile_end = (end + kTile - 1) / kTile;
    const int pairs = max((tile_end + 1) / 2 - pair0 + waves - 1, 0) / waves;
    tiles.until(tile_end, pairs);

    // The loop runs on pairs in two strands that do not wait for each other:
    // the scores of pair n+1 are multiplied while the probabilities of pair n
    // are formed and multiplied with its values. Keys are loaded kDepth + 1
    // and values kDepth pairs ahead, into the registers just used up; the
    // number of loads is the same at every step, and so is what a step waits for.
    // Behind the last pair the loads are of no bytes.
    u4 raw_k[kDepth][2][DIM / 64], raw_v[kDepth][2][DIM / 64];
    uint64_t base[2], base_v[2];  // of the newest pair; of the one before
    int size, size_v;
    const auto find_pair = [&](int n) {
        base[0] = tiles.base(n, 0);
        base[1] = tiles.base(n, 1);
        size = n < pairs ? kTile * DIM : 0;
    };
    const auto load = [&](uint8_t* pool, const uint64_t (&at)[2], int bytes, u4 (&raw)[2][DIM / 64]) {
        load_tile<DIM>(pool, at[0], bytes, lane, raw[0]);
        load_tile<DIM>(pool, at[1], bytes, lane, raw[1]);
    };
    {
        const auto t = tiles.find(lane / 2, first_block);
        tiles.take_places(t);
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            find_pair(d);
            load(a.kv.keys, base, size, raw_k[d]);
            load(a.kv.values, base, size, raw_v[d]);
        }
        tiles.take_scales(t);
    }
    tiles.look_ahead();
    Half8 q[kQueryParts][NT][kSteps];
    float factor[NT];
    split_queries<DIM, NT, MODE, kQueryParts>(a, f32, raw_q, qpos, c, q, factor);

    // o, and the sum of the probabilities as one more row of the product with
    // the values (a matrix of ones), whose four registers are the same.
    f4 o[NT][kDims], l[NT];
    float ref[NT], limit[NT];  // reference less kShift; a score above the limit raises it
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        ref[t] = 0.0f;
        limit[t] = -infinity();  // the first score that is seen
        l[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < kDims; ++n) o[t][n] = f4{0.f, 0.f, 0.f, 0.f};
    }
    uint32_t v_top = 0;  // bits of the largest value scale met
    float v_held[NT];    // the scale that o is held in: the largest that the column has seen
#pragma unroll
    for (int t = 0; t < NT; ++t) v_held[t] = 0.0f;
    uint64_t nan_met = 0;  // NaN bytes among values that some columns see and others do not
    const h8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
    const float part_factor = MODE == kPacked && !(c & 8) ? 0.0f : -1.0f;

    const auto scores = [&](const u4 (&raw)[2][DIM / 64], f4 (&to)[NT][2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int t = 0; t < NT; ++t) to[t][h] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                Half8 k;
                Convert<FORMAT>::plain(raw[h][i / 2][2 * (i % 2)], &k.two[0], &k.two[1]);
                Convert<FORMAT>::plain(raw[h][i / 2][2 * (i % 2) + 1], &k.two[2], &k.two[3]);
#pragma unroll
                for (int part = 0; part < kQueryParts; ++part)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        to[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.all, q[part][t][i].all, to[t][h], 0, 0, 0);
            }
        }
    };
    f4 s[NT][2];
    scores(raw_k[0], s);
    find_pair(kDepth);
    load(a.kv.keys, base, size, raw_k[0]);

    // `k_next`: the next pair's keys, `v`: this one's values.
    const auto step = [&](int n, u4 (&k_next)[2][DIM / 64], u4 (&v)[2][DIM / 64]) {
        const uint32_t k_bits[2] = {tiles.k_bits(n, 0), tiles.k_bits(n, 1)};
        uint32_t v_bits[2] = {tiles.v_bits(n, 0), tiles.v_bits(n, 1)};
        if (MODE == kPacked) {  // the low parts' scores are 8 columns on
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[0][h][i] = add_across(s[0][h][i]);
        }
        const int token0 = (pair0 + n * waves) * kKv8Pair;
        // Scores in powers of two less the reference.
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float f = factor[t] * __uint_as_float(k_bits[h]);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][h][i] = __builtin_fmaf(s[t][h][i], f, -ref[t]);
            }
        if (token0 + kKv8Pair - 1 > (DECODE ? last : used + first / a.group)) {  // past some row's position
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (token0 + kTile * h + 4 * g + i > qpos[t]) s[t][h][i] = -infinity();
            if (FORMAT == MP_KV8_E4M3 && token0 + kKv8Pair - 1 > last) {
                clear_past<DIM>(last + 1 - token0 - 4 * g, v[0]);
                clear_past<DIM>(last + 1 - token0 - kTile - 4 * g, v[1]);
            }
        }
        // A block of its own: in the one above dims of 256 spill 15 registers.
        if (FORMAT == MP_KV8_E4M3 && !DECODE && token0 + kKv8Pair - 1 > used + first / a.group)
            nan_met |= __builtin_amdgcn_ballot_w64(clear_nan<DIM>(v));
        // The reference is raised only where a score is past the limit.
        bool need = false;
        float top[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            top[t] = max3(max3(s[t][0][0], s[t][0][1], s[t][0][2]), max3(s[t][0][3], s[t][1][0], s[t][1][1]),
                          fmaxf(s[t][1][2], s[t][1][3]));
            need |= top[t] > limit[t];
        }
        if (__builtin_amdgcn_ballot_w64(need)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float most = column_max(top[t]);
                if (most > limit[t]) {
                    const float by = most - kShift;
                    const float keep = limit[t] == -infinity() ? 0.0f : __builtin_amdgcn_exp2f(-by);
                    ref[t] += by;
                    limit[t] = kRaise;
                    l[t] *= keep;
#pragma unroll
                    for (int n = 0; n < kDims; ++n) o[t][n] *= keep;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[t][h][i] -= by;
                }
            }
        }
        // Values that are NaN: so are the columns that see the tile, and only
        // they, since the tile's place is taken by zeros.
        if (max(v_bits[0], v_bits[1]) >= 0x7F800000u) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (v_bits[h] >= 0x7F800000u) {
                    v_bits[h] = 0;
#pragma unroll
                    for (int j = 0; j < DIM / 64; ++j) v[h][j] = u4{0, 0, 0, 0};
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        if (token0 + kTile * h <= qpos[t]) l[t] = f4{1.f, 1.f, 1.f, 1.f} * quiet_nan();
                }
        }
        // The value scale: o is held in the largest that its column has seen.
        // Columns that end before a larger one keep theirs: they take nothing
        // of what is converted for the others. Where the pair's second tile is
        // far larger, the first one's codes stay as they are for the columns
        // that end with it, and for the others its probabilities are reduced
        // (but not in their sum).
        uint32_t v_first = max(v_bits[0], v_top);  // what the first tile is converted to
        const uint32_t v_now = max(v_first, v_bits[1]);
        if (v_now > v_top) {
            const bool apart = !DECODE && v_first && v_now - v_first > kApart << 23;
            if (!apart) v_first = v_now;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const bool both = DECODE || token0 + kTile <= qpos[t];
                if (apart) {
                    const float less = both ? (float)((v_now - v_first) >> 23) : 0.0f;
                    float taken = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float reduced = s[t][0][i] - less;
                        taken += __builtin_amdgcn_exp2f(s[t][0][i]) - __builtin_amdgcn_exp2f(reduced);
                        s[t][0][i] = reduced;
                    }
                    taken = column_sum(taken);
                    l[t] += f4{taken, taken, taken, taken};
                }
                if (DECODE || token0 <= qpos[t]) {
                    const float to = __uint_as_float(both ? v_now : v_first);
                    if (v_top) {
                        const float keep = v_held[t] / to;
#pragma unroll
                        for (int n = 0; n < kDims; ++n) o[t][n] *= keep;
                    }
                    v_held[t] = to;
                }
            }
            v_top = v_now;
        } else {
            v_first = v_top;
        }
        const Convert<FORMAT> convert0(value_power(v_bits[0], v_first)), convert1(value_power(v_bits[1], v_top));
        base_v[0] = base[0], base_v[1] = base[1], size_v = size;
        find_pair(n + kDepth + 1);
        f4 s_next[NT][2];
        scores(k_next, s_next);
        load(a.kv.keys, base, size, k_next);
        Half8 p[kParts][NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float x = __builtin_amdgcn_exp2f(s[t][h][i]), y = __builtin_amdgcn_exp2f(s[t][h][i + 1]);
                    const h2 high = {(_Float16)x, (_Float16)y};
                    if (MODE != kPacked) p[0][t].two[2 * h + i / 2] = high;
                    p[kParts - 1][t].two[2 * h + i / 2] =
                        h2{(_Float16)mix_low(high, part_factor, x), (_Float16)mix_high(high, part_factor, y)};
                }
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int t = 0; t < NT; ++t)
                l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[part][t].all, l[t], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < kDims; ++n) {
            Half8 w;
            convert0(v[0][n / 4][n % 4], &w.two[0], &w.two[1]);
            convert1(v[1][n / 4][n % 4], &w.two[2], &w.two[3]);
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.all, p[part][t].all, o[t][n], 0, 0, 0);
        }
        load(a.kv.values, base_v, size_v, v);
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][0] = s_next[t][0], s[t][1] = s_next[t][1];
    };
    for (int n = 0; n < pairs;) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            tiles.go_on(n + kDepth + 1);
            step(n, raw_k[(d + 1) % kDepth], raw_v[d]);
            if (++n >= pairs && d + 1 < kDepth) break;
        }
    }

    // NaN bytes among the values: where all columns see a pair the products did
    // it; the others are of the last 16 NT tokens, two pairs at most.
    if (FORMAT == MP_KV8_E4M3 && !DECODE && nan_met) {
        for (int n = max(pairs - 2, 0); n < pairs; ++n) {
            const uint64_t at[2] = {tiles.base(n, 0), tiles.base(n, 1)};
            spread_nan<DIM, NT>((pair0 + n * waves) * kKv8Pair + 4 * g, qpos, a.kv.values, at, lane, o);
        }
    }

    // Each wavefront's reference and sum (-inf and 0 where it saw nothing).
    float sum[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        sum[t] = l[t][0];
        if (limit[t] == -infinity() && sum[t] == sum[t]) ref[t] = -infinity();
        if (MODE == kPacked) {
            sum[t] = add_across(sum[t]);
#pragma unroll
            for (int n = 0; n < kDims; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][n][i] = add_across(o[t][n][i]);
        }
    }
    // Reference and sum over the wavefronts; what turns this one's o into its
    // share of the result. The values' scale comes after it: their product is
    // below the normal numbers for scales near the smallest, the result is not.
    float best[NT], total[NT], weight[NT];
    const auto weigh = [&](int t, float scaled) { weight[t] = sum[t] == 0.0f ? 0.0f : scaled / total[t]; };
    const auto share = [&](int t, int n) { return o[t][n] * weight[t] * v_held[t]; };
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
        for (int t = 0; t < NT; ++t) {
            best[t] = ref[t];
            total[t] = sum[t];
            weigh(t, 1.0f);
#pragma unroll
            for (int n = 0; n < kDims; ++n) store(t, n, share(t, n));
        }
        return;
    }
    // Four or eight wavefronts meet in LDS: first their references and sums,
    // then their shares, join_dims tiles of 16 dims at a time; output tiles are
    // dealt to the wavefronts. As many reads in flight as there are wavefronts.
    const auto join = [&](auto count) {
        constexpr int kCount = decltype(count)::value, kAt = join_dims(kCount, NT, kDims);
#pragma unroll
        for (int t = 0; t < NT; ++t)
            if (g == 0) ml_s[wave][t][c] = make_float2(ref[t], sum[t]);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float2 ml[kCount];
#pragma unroll
            for (int w = 0; w < kCount; ++w) ml[w] = ml_s[w][t][c];
            best[t] = ml[0].x;
#pragma unroll
            for (int w = 1; w < kCount; ++w) best[t] = fmaxf(best[t], ml[w].x);
            total[t] = 0.0f;
#pragma unroll
            for (int w = 0; w < kCount; ++w)
                total[t] += ml[w].y != 0.0f ? ml[w].y * __builtin_amdgcn_exp2f(ml[w].x - best[t]) : 0.0f;
            weigh(t, __builtin_amdgcn_exp2f(ref[t] - best[t]));
        }
        __syncthreads();  // the shares lie where the references did
#pragma unroll
        for (int n0 = 0; n0 < kDims; n0 += kAt) {
            if (n0) __syncthreads();
#pragma unroll
            for (int n = 0; n < kAt; ++n)
#pragma unroll
                for (int t = 0; t < NT; ++t) o_s[(wave * kAt + n) * NT + t][lane] = share(t, n0 + n);
            __syncthreads();
            for (int i = wave; i < kAt * NT; i += kCount) {
                f4 x[kCount];
#pragma unroll
                for (int w = 0; w < kCount; ++w) x[w] = o_s[w * kAt * NT + i][lane];
#pragma unroll
                for (int w = 1; w < kCount; ++w) x[0] += x[w];
#pragma unroll
                for (int u = 0; u < NT; ++u)
                    if (u == i % NT) store(u, n0 + i / NT, x[0]);
            }
        }
    };
    if (waves == 4) join(std::integral_constant<int, 4>());
    else join(std::integral_constant<int, kKv8MostWaves>());
}

// Joins the chunks of rows that have several: WAVES wavefronts a (row, head),
// four (row, head) or one a work-group. `columns_tile`: columns of an
// attention work-group.
template <bool DECODE, int WAVES>
__global__ __launch_bounds__(256) void kv8_merge_kernel(Kv8Attention a, int columns_tile) {
    __shared__ f4 out_s[WAVES][64];
    const int lane = threadIdx.x & 63, dim = a.kv.dim;
    const int in_group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int index = WAVES > 1 ? blockIdx.x : blockIdx.x * 4 + in_group, wave = WAVES > 1 ? in_group : 0;
    const int head = index % a.heads;
    int row = index / a.heads, last;
    if (row >= a.rows.rows) return;
    if (DECODE) {
        const int length = a.rows.used[row];
        if (length <= a.chunk || length > a.max_length) return;
        last = length - 1;
    } else {
        Kv8Item at;
        if (!kv8_find(a.rows, row, [](int n, int) { return n; }, &at)) return;
        row = at.row0 + at.index;
        if (at.used < 0 || at.used >= a.max_length) return;
        const int column = at.index * a.group + head % a.group;
        const int end = min((column / columns_tile + 1) * columns_tile, at.count * a.group);
        last = min(at.used + (end - 1) / a.group, a.max_length - 1);  // of the work-group that had this column
    }
    // One chunk (or none) was stored by its work-group, as were NaN rows.
    if (last < a.chunk) return;
    const int chunks = last / a.chunk + 1;
    const size_t at = ((size_t)row * a.heads + head) * a.splits;
    // Every wavefront finds the reference and the weights' sum, and joins its
    // share of the chunks: dim/4 lanes a chunk.
    float best = -infinity();
    for (int b = lane; b < chunks; b += 64) best = fmaxf(best, a.partial_ml[at + b].x);
    best = wave_max(best);
    float total = 0.0f;
    for (int b = lane; b < chunks; b += 64) {
        const float2 ml = a.partial_ml[at + b];
        if (ml.y != 0.0f) total += ml.y * __builtin_amdgcn_exp2f(ml.x - best);
    }
    total = wave_sum(total);
    const int lanes = dim / 4, each = 64 / lanes, d4 = lane % lanes;
    f4 out = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int b = wave * each + lane / lanes; b < chunks; b += WAVES * each) {
        const float2 ml = a.partial_ml[at + b];
        const float w = ml.y != 0.0f ? ml.y * __builtin_amdgcn_exp2f(ml.x - best) / total : 0.0f;
        const float2* const part = reinterpret_cast<const float2*>(a.partial_out + (at + b) * dim + 4 * d4);
        const float2 x = part[0], y = part[1];
        out += f4{x.x, x.y, y.x, y.y} * w;
    }
    for (int d = lanes; d < 64; d *= 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] += __shfl_xor(out[i], d);
    if (WAVES > 1) {
        out_s[wave][lane] = out;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) out += out_s[w][lane];
    }
    if (lane < lanes)
        store_four(a.out, a.type, a.out_wide, row * a.out_stride + (int64_t)head * dim + 4 * d4, out[0], out[1], out[2],
                   out[3]);
}

template <int FORMAT, int DIM, int NT, int MODE, bool DECODE>
void launch(hipStream_t s, const Kv8Plan& p, int64_t items, const Kv8Attention& a) {
    const dim3 grid((unsigned)(items * a.kv.kv_heads), 1, (unsigned)p.splits);
    const size_t shared = join_bytes(p.waves, NT, DIM / 16);
    kv8_attention_kernel<FORMAT, DIM, NT, MODE, DECODE><<<grid, 64 * p.waves, shared, s>>>(a);
}
template <int FORMAT, int DIM>
void launch_decode(hipStream_t s, const Kv8Plan& p, const Kv8Attention& a) {
    if (a.group <= 8) launch<FORMAT, DIM, 1, kPacked, true>(s, p, a.rows.rows, a);
    else launch<FORMAT, DIM, 1, kTwo, true>(s, p, a.rows.rows, a);
}
template <int FORMAT, int DIM, int MODE>
void launch_prefill(hipStream_t s, const Kv8Plan& p, const Kv8Attention& a) {
    const int64_t items = kv8_items(a.rows.rows, a.rows.sequences, a.group, p.column_tiles);
    if constexpr (DIM <= 128) {
        if (p.column_tiles == 2) return launch<FORMAT, DIM, 2, MODE, false>(s, p, items, a);
    }
    launch<FORMAT, DIM, 1, MODE, false>(s, p, items, a);
}
template <int FORMAT, int DIM>
void launch_attention(hipStream_t s, const Kv8Plan& p, const Kv8Attention& a, bool decode) {
    if (decode) launch_decode<FORMAT, DIM>(s, p, a);
    else if (a.type == MP_TYPE_F32) launch_prefill<FORMAT, DIM, kTwo>(s, p, a);
    else launch_prefill<FORMAT, DIM, kOne>(s, p, a);
}
template <int FORMAT>
void launch_format(hipStream_t s, const Kv8Plan& p, const Kv8Attention& a, bool decode) {
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
    if (q == out && q_stride != out_stride && rows > 1)
        return kv8_refuse("8-bit attention: a result in place of the queries needs one stride");
    if (kv8_bad_ints(used) || (!decode && kv8_bad_ints(starts)))
        return kv8_refuse("8-bit attention: lengths, starts or used are missing or misaligned");
    if (!(scale >= 0) || !isfinite((float)(scale * 1.4426950408889634074)))
        return kv8_refuse("8-bit attention: scale must be finite (to 2.3e38) and not negative");
    if ((int64_t)rows * heads > kKv8MostColumns)
        return kv8_refuse("8-bit attention: rows times heads are too many for one call");
    if (rows == 0 || sequences == 0) return MP_OK;
    const int group = heads / cache->kv_heads;
    const Kv8Plan p = decode ? kv8_decode_plan(rows, cache->kv_heads, cache->dim, max_length)
                             : kv8_prefill_plan(rows, sequences, cache->kv_heads, group, cache->dim,
                                                max_length);
    const size_t need = kv8_partial_floats(p, rows, heads, cache->dim) * sizeof(float);
    if (need > workspace_bytes || (need && !workspace))
        return kv8_refuse("8-bit attention: the workspace is smaller than mp_hip_kv8_attention_workspace says");
    if (need && reinterpret_cast<uintptr_t>(workspace) % 16)
        return kv8_refuse("8-bit attention: the workspace must be 16-byte aligned");
    Kv8Attention a{};
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
        const int64_t outputs = (int64_t)rows * heads;
        const int columns = 16 * p.column_tiles;
        if (p.splits > 8) {
            const unsigned groups = (unsigned)outputs;
            if (decode) kv8_merge_kernel<true, 4><<<groups, 256, 0, s>>>(a, columns);
            else kv8_merge_kernel<false, 4><<<groups, 256, 0, s>>>(a, columns);
        } else {
            const unsigned groups = (unsigned)((outputs + 3) / 4);
            if (decode) kv8_merge_kernel<true, 1><<<groups, 256, 0, s>>>(a, columns);
            else kv8_merge_kernel<false, 1><<<groups, 256, 0, s>>>(a, columns);
        }
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
