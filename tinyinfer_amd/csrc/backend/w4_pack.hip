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

// A wavefront takes 16 rows by 512 columns, four tiles and the words of their
// scales. It reads each row's groups by 16 bytes a lane (8 lanes a group in
// FP32, 4 in 16 bits; whole lines of memory), and turns the codes round through
// LDS: there a lane of the result finds the 16 bytes of its row and group.
//
// Reads 4 (or 2) bytes an element and writes 17/32, which bounds it.
template <int TYPE>
__global__ void __launch_bounds__(kThreads) w4_pack_kernel(PackArgs a) {
    constexpr int V = TYPE == MP_TYPE_F32 ? 4 : 8, L = kW4Group / V, RPI = 64 / L;  // elements, lanes a group, rows a load
    __shared__ u4 codes_s[kThreads / 64][64];
    __shared__ uint32_t scales_s[kThreads / 64][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15;
    const int words = (int)w4_words(a.depth), steps = (int)w4_steps(a.depth);
    const int64_t item = (int64_t)blockIdx.x * (kThreads / 64) + wave;
    const int tile = (int)(item / words) + a.first / kW4Rows, word = (int)(item % words);
    const int last = a.first + a.count;
    if (tile * kW4Rows >= last) return;  // a wavefront behind the end: nothing here waits for it
    uint8_t* const code_bytes = reinterpret_cast<uint8_t*>(codes_s[wave]);
    uint8_t* const scale_bytes = reinterpret_cast<uint8_t*>(scales_s[wave]);
    // Rows that fill the last tile up are written with the matrix's last row, as zeros.
    const int row = tile * kW4Rows + c;
    const bool writes = row >= a.first && (row < last || last == a.rows);
    scales_s[wave][lane] = 0;
    wave_sync();
    for (int t = 0; t < kW4Word && word * kW4Word + t < steps; ++t) {
        const int step = word * kW4Word + t;
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
                const int column = step * kW4Step + b * kW4Group;
                if (lane % L == 0 && column < a.depth && tile * kW4Rows + inside < last)
                    scale_bytes[(b * 16 + inside) * 4 + t] = (uint8_t)byte;
            }
        wave_sync();
        if (writes) a.codes[((int64_t)tile * steps + step) * 64 + lane] = codes_s[wave][lane];
        wave_sync();
    }
    if (writes) a.scales[((int64_t)tile * words + word) * 64 + lane] = scales_s[wave][lane];
}

// ---- reading -----------------------------------------------------------------------

struct ReadArgs {
    W4View m;
    const int32_t* ids;
    int rows, depth, count;
    RowsView out;
    bool wide;
};

// V consecutive columns a thread, 16 bytes of result: the stores, several times
// the codes' bytes, are what bounds it.
template <int TYPE>
__global__ void __launch_bounds__(kThreads) w4_read_kernel(ReadArgs a) {
    constexpr int V = TYPE == MP_TYPE_F32 ? 4 : 8;
    const uint32_t chunks = a.depth / V;
    const uint32_t item = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t r = item / chunks, column = (item - r * chunks) * V;
    if (r >= (uint32_t)a.count) return;
    const int id = a.ids[r];
    float x[V];
    if (id < 0 || id >= a.rows) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = __builtin_nanf("");
    } else {
        const int64_t tile = id / kW4Rows, step = column / kW4Step;
        const int lane = column % kW4Step / kW4Group * 16 + id % kW4Rows;
        const uint8_t* const from = reinterpret_cast<const uint8_t*>(a.m.codes) +
                                    (((tile * w4_steps(a.depth)) + step) * 64 + lane) * 16 + column % kW4Group / 2;
        const uint32_t word = a.m.scales[(tile * w4_words(a.depth) + step / kW4Word) * 64 + lane];
        const float scale = scale_power(word >> (8 * (step % kW4Word)) & 0xFF);
        uint32_t codes;
        if constexpr (V == 8) codes = *reinterpret_cast<const uint32_t*>(from);
        else codes = *reinterpret_cast<const uint16_t*>(from);
        auto two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
        x[0] = two[0], x[1] = two[1];
        two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
        x[2] = two[0], x[3] = two[1];
        if constexpr (V == 8) {
            two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
            x[4] = two[0], x[5] = two[1];
            two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
            x[6] = two[0], x[7] = two[1];
        }
    }
    store_row<TYPE, V>(a.out.data, a.wide, r * a.out.stride + column, x);
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
        const int64_t tiles = w4_tiles(first + rows) - first / kW4Rows, items = tiles * w4_words(w->depth);
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
        const int64_t items = (int64_t)count * (w->depth / (out->type == MP_TYPE_F32 ? 4 : 8));
        const unsigned groups = (unsigned)w4_ceil(items, kThreads);
        if (out->type == MP_TYPE_F32) w4_read_kernel<MP_TYPE_F32><<<groups, kThreads, 0, s>>>(a);
        else if (out->type == MP_TYPE_BF16) w4_read_kernel<MP_TYPE_BF16><<<groups, kThreads, 0, s>>>(a);
        else w4_read_kernel<MP_TYPE_F16><<<groups, kThreads, 0, s>>>(a);
        return call_done(hipGetLastError(), "4-bit read launch");
    });
}
