// Elements of rows in a caller's type (MP_TYPE_*).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../../include/mp_hip.h"

namespace mphip {

__device__ __forceinline__ float from_bf16(uint32_t low_half) { return __uint_as_float(low_half << 16); }
__device__ __forceinline__ float from_f16(uint32_t low_half) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)low_half);
}
// Rounded to nearest, ties to even; NaN stays NaN.
__device__ __forceinline__ uint16_t to_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ uint16_t to_f16(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }

__device__ __forceinline__ float load_one(const void* p, int type, int64_t i) {
    if (type == MP_TYPE_F32) return static_cast<const float*>(p)[i];
    const uint32_t b = static_cast<const uint16_t*>(p)[i];
    return type == MP_TYPE_BF16 ? from_bf16(b) : from_f16(b);
}
__device__ __forceinline__ void store_one(void* p, int type, int64_t i, float x) {
    if (type == MP_TYPE_F32) static_cast<float*>(p)[i] = x;
    else static_cast<uint16_t*>(p)[i] = type == MP_TYPE_BF16 ? to_bf16(x) : to_f16(x);
}

// N (a multiple of 4) consecutive elements from i on; `wide`: they start at a
// multiple of 16 bytes (FP32) or 8 (16-bit types).
template <int N>
__device__ __forceinline__ void load_row(const void* p, int type, bool wide, int64_t i, float (&x)[N]) {
    if (!wide) {
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = load_one(p, type, i + k);
    } else if (type == MP_TYPE_F32) {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + k);
            x[k] = v.x, x[k + 1] = v.y, x[k + 2] = v.z, x[k + 3] = v.w;
        }
    } else {
        uint2 v[N / 4];
#pragma unroll
        for (int k = 0; k < N; k += 4)
            v[k / 4] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i + k);
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const uint32_t two = k % 4 ? v[k / 4].y : v[k / 4].x;
            x[k] = type == MP_TYPE_BF16 ? from_bf16(two) : from_f16(two & 0xFFFF);
            x[k + 1] = type == MP_TYPE_BF16 ? __uint_as_float(two & 0xFFFF0000u) : from_f16(two >> 16);
        }
    }
}
__device__ __forceinline__ void store_four(void* p, int type, bool wide, int64_t i, float a, float b, float c,
                                           float d) {
    if (!wide) {
        store_one(p, type, i, a);
        store_one(p, type, i + 1, b);
        store_one(p, type, i + 2, c);
        store_one(p, type, i + 3, d);
    } else if (type == MP_TYPE_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(a, b, c, d);
    } else {
        const bool bf = type == MP_TYPE_BF16;
        const uint32_t lo = (bf ? to_bf16(a) : to_f16(a)) | (uint32_t)(bf ? to_bf16(b) : to_f16(b)) << 16;
        const uint32_t hi = (bf ? to_bf16(c) : to_f16(c)) | (uint32_t)(bf ? to_bf16(d) : to_f16(d)) << 16;
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = make_uint2(lo, hi);
    }
}

// V consecutive elements from i on, 16 bytes of them; `wide`: they start at a
// multiple of 16 bytes.
template <int TYPE, int V>
__device__ __forceinline__ void store_row(void* p, bool wide, int64_t i, const float (&x)[V]) {
    static_assert(V == (TYPE == MP_TYPE_F32 ? 4 : 8));
    if (!wide) {
#pragma unroll
        for (int k = 0; k < V; ++k) store_one(p, TYPE, i + k, x[k]);
    } else if constexpr (TYPE == MP_TYPE_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w[k] = TYPE == MP_TYPE_BF16 ? to_bf16(x[2 * k]) | (uint32_t)to_bf16(x[2 * k + 1]) << 16
                                        : to_f16(x[2 * k]) | (uint32_t)to_f16(x[2 * k + 1]) << 16;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

inline size_t element_bytes(int type) { return type == MP_TYPE_F32 ? 4 : 2; }

}  // namespace mphip
