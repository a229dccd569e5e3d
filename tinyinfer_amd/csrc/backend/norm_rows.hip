// Rows from one type to another, and the root-mean-square norm of rows.
#include <type_traits>

#include "w4.h"

namespace mphip {
namespace {

constexpr int kThreads = 256;
constexpr int kEach = 8;  // consecutive elements of a lane

// A row's elements dealt to lanes. Wide rows: 8 consecutive elements a lane, 16
// bytes or two times 16 a load, the 4 lanes of a quad a group of an 8-bit row.
// Others (odd widths, rows that do not start at 16 bytes): single elements, 32
// consecutive lanes a group, so that a load still takes neighbouring elements.
template <bool WIDE>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    v = max(v, dpp_u<kDppQuadXor1>(v));
    v = max(v, dpp_u<kDppQuadXor2>(v));
    if (WIDE) return v;
    v = max(v, dpp_u<kDppRowRor4>(v));
    v = max(v, dpp_u<kDppRowRor8>(v));
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}

// One element; for 8 bits all lanes of its group come together.
template <int TYPE>
__device__ __forceinline__ float load_element(const RowsView& r, int64_t row, int i) {
    if constexpr (TYPE == MP_TYPE_I8) {
        const uint32_t code = static_cast<const uint8_t*>(r.data)[row * r.stride + i];
        return (float)(int8_t)code * scale_number(r.scales[row * r.scale_stride + i / kW4Group]);
    } else {
        return load_one(r.data, TYPE, row * r.stride + i);
    }
}
template <int TYPE>
__device__ __forceinline__ void store_element(const RowsView& r, int64_t row, int i, float x) {
    if constexpr (TYPE == MP_TYPE_I8) {
        const uint32_t byte = scale_byte8(group_max<false>(magnitude(x)));
        const uint32_t code = to_code8(x, scale_inverse(byte));
        static_cast<uint8_t*>(r.data)[row * r.stride + i] = (uint8_t)code;
        if (i % kW4Group == 0) r.scales[row * r.scale_stride + i / kW4Group] = (uint8_t)byte;
    } else {
        store_one(r.data, TYPE, row * r.stride + i, x);
    }
}

// 8 consecutive elements of a wide row, from a multiple of 8 on.
template <int TYPE>
__device__ __forceinline__ void load_eight(const RowsView& r, int64_t row, int i, float (&x)[kEach]) {
    if constexpr (TYPE == MP_TYPE_I8) {
        const float scale = scale_number(r.scales[row * r.scale_stride + i / kW4Group]);
        const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(r.data) + row * r.stride + i);
        const f4 lo = from_codes8(c.x, scale), hi = from_codes8(c.y, scale);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = lo[k], x[4 + k] = hi[k];
    } else {
        load_row(r.data, TYPE, true, row * r.stride + i, x);
    }
}
template <int TYPE>
__device__ __forceinline__ void store_eight(const RowsView& r, int64_t row, int i, const float (&x)[kEach]) {
    const int64_t at = row * r.stride + i;
    if constexpr (TYPE == MP_TYPE_I8) {
        uint32_t amax = 0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) amax = max(amax, magnitude(x[k]));
        const uint32_t byte = scale_byte8(group_max<true>(amax));
        const float inverse = scale_inverse(byte);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(r.data) + at) =
            make_uint2(to_codes8(x[0], x[1], x[2], x[3], inverse), to_codes8(x[4], x[5], x[6], x[7], inverse));
        if (i % kW4Group == 0) r.scales[row * r.scale_stride + i / kW4Group] = (uint8_t)byte;
    } else if constexpr (TYPE == MP_TYPE_F32) {
        const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
        store_row<TYPE, 4>(r.data, true, at, lo);
        store_row<TYPE, 4>(r.data, true, at + 4, hi);
    } else {
        store_row<TYPE, 8>(r.data, true, at, x);
    }
}

// A lane's 8 elements of a row: i + 0..7 (wide), else i + step * 0..7 as far as
// they are below `end`.
template <int TYPE, bool WIDE>
__device__ __forceinline__ void load_each(const RowsView& r, int64_t row, int i, int step, int end, float (&x)[kEach]) {
    if constexpr (WIDE) {
        load_eight<TYPE>(r, row, i, x);
    } else {
#pragma unroll
        for (int k = 0; k < kEach; ++k) x[k] = i + k * step < end ? load_element<TYPE>(r, row, i + k * step) : 0.0f;
    }
}
template <int TYPE, bool WIDE>
__device__ __forceinline__ void store_each(const RowsView& r, int64_t row, int i, int step, int end,
                                           const float (&x)[kEach]) {
    if constexpr (WIDE) {
        store_eight<TYPE>(r, row, i, x);
    } else {
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (i + k * step < end) store_element<TYPE>(r, row, i + k * step, x[k]);
    }
}

// ---- conversion ---------------------------------------------------------------------

struct ConvertArgs {
    RowsView x, out;
    int rows, width;
};

// The elements of all rows in one line, dealt to threads: what it reads and
// writes is what bounds it (4,096 x 4,096 from BF16 to 8 bits 10.6 us, 4.8 TB/s, to
// FP32 from 8 bits 16, 5.2 TB/s).
template <int FROM, int TO, bool WIDE>
__global__ void __launch_bounds__(kThreads) convert_kernel(ConvertArgs a) {
    if constexpr (WIDE) {
        const uint32_t chunks = a.width / kEach, item = blockIdx.x * kThreads + threadIdx.x;
        const uint32_t row = item / chunks;
        const int column = (int)(item - row * chunks) * kEach;
        if (row >= (uint32_t)a.rows) return;  // whole quads, where a row has groups
        float x[kEach];
        load_eight<FROM>(a.x, row, column, x);
        store_eight<TO>(a.out, row, column, x);
    } else {
        // One element a lane; a group's 32 lanes are all there or none.
        const int64_t all = (int64_t)a.rows * a.width;
        for (int k = 0; k < kEach; ++k) {
            const int64_t item = ((int64_t)blockIdx.x * kEach + k) * kThreads + threadIdx.x;
            if (item >= all) return;
            const int64_t row = item / a.width;
            const int column = (int)(item - row * a.width);
            store_element<TO>(a.out, row, column, load_element<FROM>(a.x, row, column));
        }
    }
}

template <int FROM, int TO>
hipError_t convert(const ConvertArgs& a, bool wide, hipStream_t s) {
    const int64_t all = (int64_t)a.rows * a.width;
    const unsigned groups = (unsigned)w4_ceil(all, kThreads * kEach);
    if (wide) convert_kernel<FROM, TO, true><<<groups, kThreads, 0, s>>>(a);
    else convert_kernel<FROM, TO, false><<<groups, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

// ---- norm ------------------------------------------------------------------------------

struct NormArgs {
    RowsView x, residual, sum, out;
    const float* weight;
    float epsilon;
    int rows, width;
    double share;  // 1 / width
};

// The sum over a wavefront's lanes, in every lane.
__device__ __forceinline__ double wave_sum(double v) {
    auto add = [](double v, uint32_t lo, uint32_t hi) {
        return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    auto halves = [](double v, uint32_t* lo, uint32_t* hi) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        *lo = (uint32_t)b, *hi = (uint32_t)(b >> 32);
    };
    uint32_t lo, hi;
    halves(v, &lo, &hi);
    v = add(v, dpp_u<kDppQuadXor1>(lo), dpp_u<kDppQuadXor1>(hi));
    halves(v, &lo, &hi);
    v = add(v, dpp_u<kDppQuadXor2>(lo), dpp_u<kDppQuadXor2>(hi));
    halves(v, &lo, &hi);
    v = add(v, dpp_u<kDppRowRor4>(lo), dpp_u<kDppRowRor4>(hi));
    halves(v, &lo, &hi);
    v = add(v, dpp_u<kDppRowRor8>(lo), dpp_u<kDppRowRor8>(hi));
    halves(v, &lo, &hi);
    auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    v = add(__builtin_bit_cast(double, (uint64_t)h[0] << 32 | l[0]), l[1], h[1]);
    halves(v, &lo, &hi);
    l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    return add(__builtin_bit_cast(double, (uint64_t)h[0] << 32 | l[0]), l[1], h[1]);
}

// y in FP32 so that rounding it further, to 16 or 8 bits, gives what rounding y
// itself gives: the first BITS bits of its mantissa, the last of them set if anything
// follows. Numbers of BITS - 1 bits, and the borders between numbers of BITS - 2, stay
// on their side.
template <int BITS>
__device__ __forceinline__ float to_odd(double y) {
    constexpr uint32_t below = (1u << (20 - BITS)) - 1;
    const uint64_t b = __builtin_bit_cast(uint64_t, y);
    const uint32_t hi = (uint32_t)(b >> 32), rest = min((hi & below) | (uint32_t)b, below + 1);
    return (float)__builtin_bit_cast(double, (uint64_t)((hi | (rest + below)) & ~below) << 32);
}
template <int TYPE, int BITS>
__device__ __forceinline__ float to_type(double y) {
    return TYPE == MP_TYPE_F32 ? (float)y : to_odd<BITS>(y);
}
// BF16 has numbers down to 2^-133 and borders to 2^-134, where FP32 holds no 20 bits
// any more, but 10. That takes three instructions an element more, a check for small
// results with a branch as many and registers (131,072 rows of 128 41 us, with the
// check 42.5, with 20 bits 39.6). The sum of two BF16 numbers has nothing below 2^-133.
template <int TYPE>
constexpr int kBits = TYPE == MP_TYPE_BF16 ? 10 : 20;

// 1 / sqrt(v) to the last bit or two: an estimate of half the bits and two steps of
// Newton's method, a fourth of the instructions of a root and a division. Infinity
// gives 0.
__device__ __forceinline__ double inverse_root(double v) {
    const double estimate = __builtin_amdgcn_rsq(v);
    double y = estimate;
#pragma unroll
    for (int i = 0; i < 2; ++i) y = __builtin_fma(0.5 * y, __builtin_fma(-v * y, y, 1.0), y);
    return v == __builtin_inf() ? estimate : y;
}

// A row by `waves` wavefronts (a work-group, or one of a work-group's
// wavefronts), C chunks of 8 elements a lane in registers between the sum of
// squares and the result; longer rows are read a second time.
//
// Sums, the root and the products are FP64, a single rounding an element: an
// 8-bit code next to the border of two would go either way by the order of an
// FP32 sum. The FP64 unit is as wide as the FP32 one: 4,096 x 4,096 BF16 rows with a
// residual, to 8 bits, take 32 us, 3.7 TB/s in five streams, with the vector unit
// busy for half of it. One row of 576 takes 2.3 us (3.0 with one wavefront of two
// chunks), a chain of latencies. Rows that do not begin at 16 bytes are read by
// elements: with a residual 777 FP16 rows of 2,047 take 9.0 us, of 2,048 5.7. Rows
// of fewer than 512 elements leave lanes idle: 131,072 BF16 rows of 64 take 42 us (a
// copy's 7), as many of 128 41 (13), 65,536 of 256 23 (13), 32,768 of 512 15 (13).
template <int TYPE, int OUT, bool RESIDUAL, bool WIDE, int C>
__global__ void __launch_bounds__(1024) rms_norm_kernel(NormArgs a, int waves) {
    __shared__ double sums[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const bool alone = waves == 1;
    const int row = alone ? blockIdx.x * (blockDim.x >> 6) + wave : blockIdx.x;
    if (row >= a.rows) return;  // with one wavefront a row nothing waits; else there is no such row
    const int lanes = alone ? 64 : blockDim.x, me = alone ? lane : threadIdx.x;
    const int block = lanes * kEach * C;  // elements that the row's wavefronts hold
    // Chunk c of this lane from `base` on: where it begins, and the step between its elements.
    const int step = WIDE ? 1 : lanes;
    auto place = [&](int base, int c) { return base + c * lanes * kEach + (WIDE ? me * kEach : me); };
    double t[C][kEach];
    float w[C][kEach];
    auto load = [&](int base) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = place(base, c);
            float x[kEach] = {}, r[kEach] = {};
            if (i < a.width) {
                load_each<TYPE, WIDE>(a.x, row, i, step, a.width, x);
                if constexpr (RESIDUAL) load_each<TYPE, WIDE>(a.residual, row, i, step, a.width, r);
            }
#pragma unroll
            for (int k = 0; k < kEach; ++k) t[c][k] = RESIDUAL ? (double)x[k] + (double)r[k] : (double)x[k];
        }
    };
    // On their way while the row's sums meet.
    auto load_weight = [&](int base) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = place(base, c);
            if constexpr (WIDE) {
                if (i < a.width) load_row(a.weight, MP_TYPE_F32, true, i, w[c]);
            } else {
#pragma unroll
                for (int k = 0; k < kEach; ++k) w[c][k] = i + k * step < a.width ? a.weight[i + k * step] : 0.0f;
            }
        }
    };
    double squares = 0.0;
    for (int base = 0; base < a.width; base += block) {
        load(base);
        if (block >= a.width) load_weight(base);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < kEach; ++k) squares = __builtin_fma(t[c][k], t[c][k], squares);
    }
    squares = wave_sum(squares);
    if (!alone) {
        if (lane == 0) sums[wave] = squares;
        __syncthreads();
        squares = 0.0;
        for (int w = 0; w < waves; ++w) squares += sums[w];
    }
    const double inverse = inverse_root(__builtin_fma(squares, a.share, (double)a.epsilon));
    for (int base = 0; base < a.width; base += block) {
        if (block < a.width) {
            load(base);
            load_weight(base);
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = place(base, c);
            // A quad or 32 lanes whose group is there stay together.
            float y[kEach] = {};
            if (i < a.width) {
                if constexpr (RESIDUAL) {
                    if (a.sum.data) {
#pragma unroll
                        for (int k = 0; k < kEach; ++k) y[k] = to_type<TYPE, 20>(t[c][k]);
                        store_each<TYPE, WIDE>(a.sum, row, i, step, a.width, y);
                    }
                }
#pragma unroll
                for (int k = 0; k < kEach; ++k) y[k] = to_type<OUT, kBits<OUT>>(t[c][k] * inverse * (double)w[c][k]);
                store_each<OUT, WIDE>(a.out, row, i, step, a.width, y);
            }
        }
    }
}

template <int TYPE, int OUT, bool RESIDUAL, bool WIDE>
hipError_t norm(const NormArgs& a, hipStream_t s) {
    // A wavefront for 512 elements, up to 16 of them; short rows four a work-group.
    const int waves = (int)w4_ceil(a.width, 64 * kEach);
    if (waves == 1) rms_norm_kernel<TYPE, OUT, RESIDUAL, WIDE, 1><<<(a.rows + 3) / 4, 256, 0, s>>>(a, 1);
    else if (waves <= 16) rms_norm_kernel<TYPE, OUT, RESIDUAL, WIDE, 1><<<a.rows, 64 * waves, 0, s>>>(a, waves);
    else rms_norm_kernel<TYPE, OUT, RESIDUAL, WIDE, 2><<<a.rows, 1024, 0, s>>>(a, 16);
    return hipGetLastError();
}

// f with the type as a constant.
template <typename F>
hipError_t with_type(int type, const F& f) {
    if (type == MP_TYPE_F32) return f(std::integral_constant<int, MP_TYPE_F32>());
    if (type == MP_TYPE_BF16) return f(std::integral_constant<int, MP_TYPE_BF16>());
    if (type == MP_TYPE_F16) return f(std::integral_constant<int, MP_TYPE_F16>());
    return f(std::integral_constant<int, MP_TYPE_I8>());
}
template <typename F>
hipError_t with_float_type(int type, const F& f) {
    if (type == MP_TYPE_F32) return f(std::integral_constant<int, MP_TYPE_F32>());
    if (type == MP_TYPE_BF16) return f(std::integral_constant<int, MP_TYPE_BF16>());
    return f(std::integral_constant<int, MP_TYPE_F16>());
}

const char* wrong_sizes(int rows, int width) {
    if (rows < 0 || rows > kW4MostRows) return "rows: 0 to 1,048,576 rows a call";
    if (width < 1 || width > kW4MostDepth) return "rows: width must be 1 to 2^20";
    if ((int64_t)rows * width > kRowsMostElements) return "rows: too many elements for one call";
    return nullptr;
}

}  // namespace
}  // namespace mphip

extern "C" int mp_hip_convert_rows(const mp_rows* x, int32_t rows, int32_t width, const mp_rows* out, void* stream) {
    using namespace mphip;
    return c_entry([&]() -> int {
        const char* wrong = wrong_sizes(rows, width);
        if (!wrong) wrong = rows_wrong(x, width, true);
        if (!wrong) wrong = rows_wrong(out, width, true);
        if (wrong) return refuse_call(wrong);
        if (rows_clash(*x, *out)) return refuse_call("rows: a result in place must be the same rows");
        if (rows == 0) return MP_OK;
        ConvertArgs a{rows_view(*x), rows_view(*out), rows, width};
        const bool wide = rows_wide(*x) && rows_wide(*out) && width % kEach == 0;
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return call_done(device.status, "conversion of rows: device of the stream");
        const hipError_t e = with_type(x->type, [&](auto from) {
            return with_type(out->type, [&](auto to) {
                return convert<decltype(from)::value, decltype(to)::value>(a, wide, s);
            });
        });
        return call_done(e, "conversion of rows");
    });
}

extern "C" int mp_hip_rms_norm(const mp_rows* x, const mp_rows* residual, const mp_rows* sum, const float* weight,
                               float epsilon, int32_t rows, int32_t width, const mp_rows* out, void* stream) {
    using namespace mphip;
    return c_entry([&]() -> int {
        const char* wrong = wrong_sizes(rows, width);
        if (!wrong) wrong = rows_wrong(x, width, false);
        if (!wrong) wrong = rows_wrong(out, width, true);
        if (!wrong && residual) wrong = rows_wrong(residual, width, false);
        if (!wrong && sum) wrong = rows_wrong(sum, width, false);
        if (wrong) return refuse_call(wrong);
        if (!weight || reinterpret_cast<uintptr_t>(weight) % 4) return refuse_call("norm: the weight is missing or misaligned");
        if (!(epsilon >= 0) || !isfinite(epsilon)) return refuse_call("norm: epsilon must be finite and not negative");
        if (sum && !residual) return refuse_call("norm: a sum without a residual");
        if ((residual && residual->type != x->type) || (sum && sum->type != x->type))
            return refuse_call("norm: x, residual and sum have one type");
        if (rows_clash(*x, *out) || (residual && residual->data == out->data) || (sum && sum->data == out->data) ||
            (sum && (rows_clash(*x, *sum) || rows_clash(*residual, *sum))))
            return refuse_call("norm: a result in place must be the same rows, and out none but x");
        if (rows == 0) return MP_OK;
        NormArgs a{};
        a.x = rows_view(*x), a.out = rows_view(*out);
        if (residual) a.residual = rows_view(*residual);
        if (sum) a.sum = rows_view(*sum);
        a.weight = weight, a.epsilon = epsilon, a.rows = rows, a.width = width, a.share = 1.0 / width;
        const bool wide = width % kEach == 0 && rows_wide(*x) && rows_wide(*out) && (!residual || rows_wide(*residual)) &&
                          (!sum || rows_wide(*sum)) && reinterpret_cast<uintptr_t>(weight) % 16 == 0;
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return call_done(device.status, "norm: device of the stream");
        const hipError_t e = with_float_type(x->type, [&](auto type) {
            return with_type(out->type, [&](auto to) {
                constexpr int TYPE = decltype(type)::value, OUT = decltype(to)::value;
                if (residual) return wide ? norm<TYPE, OUT, true, true>(a, s) : norm<TYPE, OUT, true, false>(a, s);
                return wide ? norm<TYPE, OUT, false, true>(a, s) : norm<TYPE, OUT, false, false>(a, s);
            });
        });
        return call_done(e, "norm launch");
    });
}
