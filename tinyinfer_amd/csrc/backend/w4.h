// Matrices of 4-bit weights and rows of 8 bits: their formats on the device,
// and what their C entries check.
//
// A weight is an E2M1 number (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives)
// times the power of two of its group of 32 along the row; an element of an
// 8-bit row a whole number times that of its group. A scale byte b stands for
// 2^(b - 127), 0xFF for NaN. The matrix cores take such weights with their scales
// (v_mfma_scale_f32_*_f8f6f4), and one instruction makes two BF16 numbers of two
// weights and their scale, exactly.
//
// Order of a matrix: that instruction's operand for 16 rows and 128 columns as it
// lies. Lane l = (c = l%16, g = l/16) holds row c at columns 32g ..+31, 16 bytes,
// and the scale of that group. Codes are [rows/16][columns/128][64 lanes][16
// bytes], even columns in the low halves; scales are [rows/16][columns/512]
// [64 lanes][4 tiles], so that a lane's word has its scales of four tiles. 8-bit
// rows lie as they come.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include "../../../include/mp_hip.h"
#include "elements.h"
#include "entry.h"
#include "lanes.h"
#include "w4_rules.h"

namespace mphip {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// A 4-bit matrix on the device.
struct W4View {
    const u4* codes;
    const uint32_t* scales;
};

// ---- scales and codes ----------------------------------------------------------

// Scales go down to 2^-100: what is smaller is rounded on that grid, and codes times
// scales and the scales' inverses are normal numbers. They go up to 2^120, so that
// 127 times one is finite and the planes' scales, up to 2^7 more, have a byte.
// Products of two small elements may be smaller than FP32's numbers: they vanish, as
// in any FP32 sum.
constexpr uint32_t kLeastScale = 27, kMostScale = 247, kNanScale = 255;

// The scale byte of a group by the bits of its largest magnitude: the smallest
// power of two s with amax <= (1 + top / 2^23) * 2^exponent * s. Bits order as
// magnitudes do, with infinity and NaN at the end: a group with either has the
// scale NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax, uint32_t exponent, uint32_t top) {
    const int e = (int)(amax >> 23) - (int)exponent + ((amax & 0x7FFFFFu) > top ? 1 : 0);
    return e > (int)kMostScale ? kNanScale : (uint32_t)max(e, (int)kLeastScale);
}
__device__ __forceinline__ uint32_t scale_byte8(uint32_t amax) { return scale_byte(amax, 6, 0x7E0000u); }  // 127
__device__ __forceinline__ uint32_t scale_byte4(uint32_t amax) { return scale_byte(amax, 2, 0x400000u); }  // 6

// The scale as a number. NaN's exponent makes the conversions of 4-bit codes
// give NaN; products with it need the number.
__device__ __forceinline__ float scale_power(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float scale_number(uint32_t byte) {
    return byte == kNanScale ? __builtin_nanf("") : scale_power(byte);
}
// 1 / scale.
__device__ __forceinline__ float scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// A number over its group's scale in the low byte, rounded to nearest, ties to
// even: next to 1.5 * 2^23 an FP32 number's last bit is 1. What a group whose scale
// is NaN holds does not matter.
__device__ __forceinline__ uint32_t to_code8(float x, float inverse) {
    return __float_as_uint(__builtin_fmaf(x, inverse, 12582912.0f));
}
__device__ __forceinline__ uint32_t to_codes8(float a, float b, float c, float d, float inverse) {
    const uint32_t lo = __builtin_amdgcn_perm(to_code8(b, inverse), to_code8(a, inverse), 0x0C0C0400u);
    const uint32_t hi = __builtin_amdgcn_perm(to_code8(d, inverse), to_code8(c, inverse), 0x04000C0Cu);
    return lo | hi;
}
// Four codes times a scale.
__device__ __forceinline__ f4 from_codes8(uint32_t codes, float scale) {
    return f4{(float)(int8_t)codes * scale, (float)(int8_t)(codes >> 8) * scale, (float)(int8_t)(codes >> 16) * scale,
              (float)(int8_t)(codes >> 24) * scale};
}

// ---- host side of the entries ------------------------------------------------------

inline size_t row_element(int type) { return type == MP_TYPE_I8 ? 1 : element_bytes(type); }

// nullptr, or what is wrong with a matrix.
inline const char* w4_wrong_size(int rows, int depth) {
    if (rows < 1 || rows > kW4MostMatrixRows) return "4-bit matrix: rows must be 1 to 2^24";
    if (depth < kW4Group || depth > kW4MostDepth || depth % kW4Group)
        return "4-bit matrix: depth must be a multiple of 32, 32 to 2^20";
    return nullptr;
}
inline const char* w4_wrong_matrix(const mp_w4_matrix* m) {
    if (!m || !m->codes || !m->scales) return "4-bit matrix: codes or scales are missing";
    if (reinterpret_cast<uintptr_t>(m->codes) % 16 || reinterpret_cast<uintptr_t>(m->scales) % 16)
        return "4-bit matrix: codes and scales must be 16-byte aligned";
    return w4_wrong_size(m->rows, m->depth);
}

// nullptr, or what is wrong with rows of `width` elements; `eight`: 8-bit rows
// are taken, too.
inline const char* rows_wrong(const mp_rows* r, int64_t width, bool eight) {
    if (!r) return "rows: a row matrix is missing";
    if (r->type != MP_TYPE_F32 && r->type != MP_TYPE_BF16 && r->type != MP_TYPE_F16 &&
        (r->type != MP_TYPE_I8 || !eight))
        return "rows: element type unknown or not taken here";
    if (!r->data || reinterpret_cast<uintptr_t>(r->data) % row_element(r->type))
        return "rows: a row matrix is missing or misaligned";
    if (r->stride < width || r->stride > (int64_t)1 << 40) return "rows: a row stride is smaller than the row";
    if (r->type != MP_TYPE_I8) return nullptr;
    if (width % kW4Group) return "rows: 8-bit rows are whole groups of 32 elements";
    if (reinterpret_cast<uintptr_t>(r->data) % 16 || r->stride % 16)
        return "rows: 8-bit rows and their stride must be 16-byte aligned";
    if (!r->scales || reinterpret_cast<uintptr_t>(r->scales) % 4 || r->scale_stride % 4 ||
        r->scale_stride < width / kW4Group || r->scale_stride > (int64_t)1 << 40)
        return "rows: scales of 8-bit rows must be there, 4-byte aligned with their stride, a byte for 32 elements";
    return nullptr;
}

// Whether rows can be read and written by 16 bytes.
inline bool rows_wide(const mp_rows& r) {
    const int64_t bytes = r.stride * (int64_t)row_element(r.type);
    return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && bytes % 16 == 0;
}

// Rows on the device.
struct RowsView {
    void* data;
    uint8_t* scales;
    int64_t stride, scale_stride;
    int type;
};
inline RowsView rows_view(const mp_rows& r) {
    return RowsView{r.data, r.scales, r.stride, r.scale_stride, r.type};
}
// Whether a call that reads `a` and writes `b` row by row may have both at one
// address: there they are the same rows.
inline bool rows_clash(const mp_rows& a, const mp_rows& b) {
    return a.data == b.data && (a.type != b.type || a.stride != b.stride ||
                                (a.type == MP_TYPE_I8 && (a.scales != b.scales || a.scale_stride != b.scale_stride)));
}

}  // namespace mphip
