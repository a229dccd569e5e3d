// Weights to 4 bits, and rows of a 4-bit matrix as floats.
#include "w4.h"

namespace mphip {
namespace {

constexpr int kThreads = 256;

// ---- packing --------------------------------------------------------------------

struct PackArgs {
    const void* x;
    int64_t x_stride;
    u4* codes;
    uint32_t* scales;
    int first, count, rows, depth;  // rows first .. first+count-1 of the matrix's `rows`
    bool wide;
};

// A wavefront takes a tile, 16 rows by 128 columns. It reads each row's groups by
// 16 bytes a lane (8 lanes a group in FP32, 4 in 16 bits; whole lines of memory),
// and turns the codes round through LDS: there a lane of the result finds the 16
// bytes of its row and group.
//
// Reads 4 (or 2) bytes an element and writes 17/32, which bounds it: 49,152 x 576 in
// FP32 32.5 us (3.9 TB/s), 12,288 x 4,096 in BF16 31 (4.1).
template <int TYPE>
__global__ void __launch_bounds__(kThreads) w4_pack_kernel(PackArgs a) {
    constexpr int V = TYPE == MP_TYPE_F32 ? 4 : 8, L = kW4Group / V, RPI = 64 / L;  // elements, lanes a group, rows a load
    __shared__ u4 codes_s[kThreads / 64][64];
    __shared__ uint8_t scales_s[kThreads / 64][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15;
    const int words = (int)w4_words(a.depth), steps = (int)w4_steps(a.depth);
    const int64_t item = (int64_t)blockIdx.x * (kThreads / 64) + wave;
    const int tile = (int)(item / steps) + a.first / kW4Rows, step = (int)(item % steps);
    const int last = a.first + a.count;
    if (tile * kW4Rows >= last) return;  // a wavefront behind the end: nothing here waits for it
    uint8_t* const code_bytes = reinterpret_cast<uint8_t*>(codes_s[wave]);
    float x[4][kW4Rows / RPI][V];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int h = 0; h < kW4Rows / RPI; ++h) {
            const int r = tile * kW4Rows + h * RPI + lane / L, column = step * kW4Step + b * kW4Group;
#pragma unroll
            for (int i = 0; i < V; ++i) x[b][h][i] = 0.0f;
            if (r >= a.first && r < last && column < a.depth)
                load_row(a.x, TYPE, a.wide, (r - a.first) * a.x_stride + column + V * (lane % L), x[b][h]);
        }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int h = 0; h < kW4Rows / RPI; ++h) {
            const int inside = h * RPI + lane / L;
            uint32_t amax = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) amax = max(amax, magnitude(x[b][h][i]));
            amax = max(amax, dpp_u<kDppQuadXor1>(amax));
            amax = max(amax, dpp_u<kDppQuadXor2>(amax));
            if (L == 8) amax = max(amax, dpp_u<kDppHalfMirror>(amax));
            const uint32_t byte = scale_byte4(amax);
            const float scale = scale_power(byte);
            uint32_t code = 0;
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[b][h][0], x[b][h][1], scale, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[b][h][2], x[b][h][3], scale, 1);
            uint8_t* const to = code_bytes + (b * 16 + inside) * 16 + (lane % L) * (V / 2);
            if constexpr (V == 8) {
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[b][h][4], x[b][h][5], scale, 2);
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[b][h][6], x[b][h][7], scale, 3);
                *reinterpret_cast<uint32_t*>(to) = code;
            } else {
                *reinterpret_cast<uint16_t*>(to) = (uint16_t)code;
            }
            // Rows and columns that fill a tile up have scales of 0, as their codes are.
            const bool there = step * kW4Step + b * kW4Group < a.depth && tile * kW4Rows + inside < last;
            if (lane % L == 0) scales_s[wave][b * 16 + inside] = there ? (uint8_t)byte : 0;
        }
    wave_sync();
    // Rows that fill the last tile up are written with the matrix's last row.
    const int row = tile * kW4Rows + c;
    if (row < a.first || (row >= last && last != a.rows)) return;
    a.codes[((int64_t)tile * steps + step) * 64 + lane] = codes_s[wave][lane];
    uint8_t* const scale =
        reinterpret_cast<uint8_t*>(a.scales + ((int64_t)tile * words + step / kW4Word) * 64 + lane) + step % kW4Word;
    *scale = scales_s[wave][lane];
    if (step == steps - 1)  // the rest of the last word
        for (int t = 1; t < kW4Word - step % kW4Word; ++t) scale[t] = 0;
}

// ---- reading -----------------------------------------------------------------------

struct ReadArgs {
    W4View m;
    const int32_t* ids;
    int rows, depth, count;
    RowsView out;
    bool wide;
};

// V consecutive columns of R rows a thread, 16 bytes of result each: the stores,
// several times the codes' bytes, are what bounds it (49,152 x 576 in FP32 27.8 us,
// 4.6 TB/s). Several rows share the arithmetic of the places, where there are enough
// of them.
template <int TYPE, int R>
__global__ void __launch_bounds__(kThreads) w4_read_kernel(ReadArgs a) {
    constexpr int V = TYPE == MP_TYPE_F32 ? 4 : 8;
    const uint32_t chunks = a.depth / V, item = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t group = item / chunks, column = (item - group * chunks) * V;
    const int64_t steps = w4_steps(a.depth), words = w4_words(a.depth);
    const uint32_t step = column / kW4Step, g = column % kW4Step / kW4Group;
    const uint8_t* const codes = reinterpret_cast<const uint8_t*>(a.m.codes) + step * 1024 + g * 256 + column % kW4Group / 2;
    const uint8_t* const scales =
        reinterpret_cast<const uint8_t*>(a.m.scales) + step / kW4Word * 256 + g * 64 + step % kW4Word;
    int id[R];
    uint32_t code[R], scale[R];
#pragma unroll
    for (int k = 0; k < R; ++k) id[k] = group * R + k < (uint32_t)a.count ? a.ids[group * R + k] : -1;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const bool there = id[k] >= 0 && id[k] < a.rows;
        const int64_t tile = there ? id[k] / kW4Rows : 0, row = there ? id[k] % kW4Rows : 0;
        const uint8_t* const from = codes + tile * steps * 1024 + row * 16;
        if constexpr (V == 8) code[k] = *reinterpret_cast<const uint32_t*>(from);
        else code[k] = *reinterpret_cast<const uint16_t*>(from);
        scale[k] = there ? scales[tile * words * 256 + row * 4] : kNanScale;
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
        if (group * R + k >= (uint32_t)a.count) return;
        const float power = scale_power(scale[k]);
        float x[V];
        auto two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[k], power, 0);
        x[0] = two[0], x[1] = two[1];
        two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[k], power, 1);
        x[2] = two[0], x[3] = two[1];
        if constexpr (V == 8) {
            two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[k], power, 2);
            x[4] = two[0], x[5] = two[1];
            two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[k], power, 3);
            x[6] = two[0], x[7] = two[1];
        }
        store_row<TYPE, V>(a.out.data, a.wide, (group * R + k) * a.out.stride + column, x);
    }
}

template <int TYPE>
void read(const ReadArgs& a, hipStream_t s) {
    const int64_t runs = a.depth / (TYPE == MP_TYPE_F32 ? 4 : 8), items = a.count * runs;
    if (items >= kW4ReadRuns) {
        const int64_t groups = w4_ceil(w4_ceil(a.count, 8) * runs, kThreads);
        w4_read_kernel<TYPE, 8><<<(unsigned)groups, kThreads, 0, s>>>(a);
    } else {
        w4_read_kernel<TYPE, 1><<<(unsigned)w4_ceil(items, kThreads), kThreads, 0, s>>>(a);
    }
}

}  // namespace
}  // namespace mphip

extern "C" int mp_hip_w4_sizes(int32_t rows, int32_t depth, size_t* code_bytes, size_t* scale_bytes) {
    using namespace mphip;
    return c_entry([&]() -> int {
        if (!code_bytes || !scale_bytes) return refuse_call("4-bit matrix: no place for its sizes");
        if (const char* wrong = w4_wrong_size(rows, depth)) return refuse_call(wrong);
        *code_bytes = w4_code_bytes(rows, depth);
        *scale_bytes = w4_scale_bytes(rows, depth);
        return MP_OK;
    });
}

extern "C" int mp_hip_w4_pack(const mp_w4_matrix* w, int32_t first, const mp_rows* x, int32_t rows, void* stream) {
    using namespace mphip;
    return c_entry([&]() -> int {
        const char* wrong = w4_wrong_matrix(w);
        if (!wrong) wrong = rows_wrong(x, w->depth, false);
        if (wrong) return refuse_call(wrong);
        if (first < 0 || rows < 0 || first > w->rows || rows > w->rows - first)
            return refuse_call("4-bit matrix: no such rows");
        if (rows == 0) return MP_OK;
        const int64_t tiles = w4_tiles(first + rows) - first / kW4Rows, items = tiles * w4_steps(w->depth);
        const int64_t groups = w4_ceil(items, kThreads / 64);
        if (groups > kW4MostGroups) return refuse_call("4-bit matrix: too many rows for one call");
        PackArgs a{};
        a.x = x->data, a.x_stride = x->stride;
        a.codes = reinterpret_cast<u4*>(w->codes), a.scales = reinterpret_cast<uint32_t*>(w->scales);
        a.first = first, a.count = rows, a.rows = w->rows, a.depth = w->depth;
        a.wide = rows_wide(*x);
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return call_done(device.status, "4-bit packing: device of the stream");
        if (x->type == MP_TYPE_F32) w4_pack_kernel<MP_TYPE_F32><<<(unsigned)groups, kThreads, 0, s>>>(a);
        else if (x->type == MP_TYPE_BF16) w4_pack_kernel<MP_TYPE_BF16><<<(unsigned)groups, kThreads, 0, s>>>(a);
        else w4_pack_kernel<MP_TYPE_F16><<<(unsigned)groups, kThreads, 0, s>>>(a);
        return call_done(hipGetLastError(), "4-bit packing launch");
    });
}

extern "C" int mp_hip_w4_read(const mp_w4_matrix* w, const int32_t* ids, int32_t count, const mp_rows* out,
                              void* stream) {
    using namespace mphip;
    return c_entry([&]() -> int {
        const char* wrong = w4_wrong_matrix(w);
        if (!wrong) wrong = rows_wrong(out, w->depth, false);
        if (wrong) return refuse_call(wrong);
        if (!ids || reinterpret_cast<uintptr_t>(ids) % 4) return refuse_call("4-bit matrix: ids are missing or misaligned");
        if (count < 0 || count > kW4MostRows) return refuse_call("4-bit matrix: 0 to 1,048,576 rows a call");
        if ((int64_t)count * w->depth > kRowsMostElements)
            return refuse_call("4-bit matrix: too many elements for one call");
        if (count == 0) return MP_OK;
        ReadArgs a{};
        a.m = W4View{reinterpret_cast<const u4*>(w->codes), reinterpret_cast<const uint32_t*>(w->scales)};
        a.ids = ids, a.rows = w->rows, a.depth = w->depth, a.count = count;
        a.out = rows_view(*out);
        a.wide = rows_wide(*out);
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const StreamDevice device(s);
        if (device.status != hipSuccess) return call_done(device.status, "4-bit read: device of the stream");
        if (out->type == MP_TYPE_F32) read<MP_TYPE_F32>(a, s);
        else if (out->type == MP_TYPE_BF16) read<MP_TYPE_BF16>(a, s);
        else read<MP_TYPE_F16>(a, s);
        return call_done(hipGetLastError(), "4-bit read launch");
    });
}
