// What the decoder-layer operators share: element types, vector loads at the alignment the library guarantees, and the
// geometry of a paged cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace tb200 {

template <int TYPE>
struct ElemOf;
template <>
struct ElemOf<TB200_TYPE_F32> { using type = float; };
template <>
struct ElemOf<TB200_TYPE_F16> { using type = __half; };
template <>
struct ElemOf<TB200_TYPE_BF16> { using type = __nv_bfloat16; };

__host__ __device__ __forceinline__ int type_bytes(int type) { return type == TB200_TYPE_F32 ? 4 : 2; }
static inline bool valid_type(int type) { return type == TB200_TYPE_F32 || type == TB200_TYPE_F16 || type == TB200_TYPE_BF16; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// to the nearest value, ties to even
__device__ __forceinline__ void from_f32(float &d, float v) { d = v; }
__device__ __forceinline__ void from_f32(__half &d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(__nv_bfloat16 &d, float v) { d = __float2bfloat16_rn(v); }

__device__ __forceinline__ float2 unpack2(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Eight consecutive elements as floats.  ALIGN: 16 or 8 bytes that the address is a multiple of (payloads behind a
// 24-byte header are 8 modulo 16).
template <int ALIGN, class T>
__device__ __forceinline__ void load8(const T *p, float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (ALIGN == 16) {
            const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = *reinterpret_cast<const float2 *>(p + 2 * i);
                f[2 * i] = a.x, f[2 * i + 1] = a.y;
            }
        }
    } else {
        uint32_t w[4];
        if constexpr (ALIGN == 16) {
            const uint4 a = *reinterpret_cast<const uint4 *>(p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
            const uint2 a = *reinterpret_cast<const uint2 *>(p), b = *reinterpret_cast<const uint2 *>(p + 4);
            w[0] = a.x, w[1] = a.y, w[2] = b.x, w[3] = b.y;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpack2(w[i], T());
            f[2 * i] = a.x, f[2 * i + 1] = a.y;
        }
    }
}

template <int ALIGN, class T>
__device__ __forceinline__ void store8(T *p, const float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (ALIGN == 16) {
            *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4 *>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<float2 *>(p + 2 * i) = make_float2(f[2 * i], f[2 * i + 1]);
        }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack2(f[2 * i], f[2 * i + 1], T());
        if constexpr (ALIGN == 16) {
            *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
            *reinterpret_cast<uint2 *>(p + 4) = make_uint2(w[2], w[3]);
        }
    }
}

// The largest of two values; a NaN wins (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

}  // namespace tb200
