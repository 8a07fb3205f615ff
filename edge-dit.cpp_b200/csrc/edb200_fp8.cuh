// e4m3 helpers shared by the block-128 quantisers: conversion, the scale rule, typed loads and stores.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <string.h>

namespace edb {

constexpr float kF8Max = 448.0f;              // largest e4m3 number
constexpr float kF8Floor = 0x1p-100f;         // least magnitude a block's scale is made from: 448 / a stays finite

// Two and four f32 to e4m3, ties to even; NaN stays NaN (0x7f).  Callers scale to at most 448 first.
__device__ __forceinline__ uint32_t f8_pack2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
    return f8_pack2(a, b) | (f8_pack2(c, d) << 16);
}

// The block maximum.  f8_peak takes |v| as it comes: NaN passes by (fmaxf returns its other operand) and stays NaN in e4m3,
// so only an infinity needs care (e4m3 has none, and a saturated one would read as a number).  It shows in the maximum;
// the block's infinities then become NaN and the maximum is taken again.
__device__ __forceinline__ float f8_peak(float a, float v) { return fmaxf(a, fabsf(v)); }
__device__ __forceinline__ bool f8_has_infinity(float peak) { return peak > 3.402823466e38f; }
__device__ __forceinline__ float f8_no_infinity(float v) { return fabsf(v) <= 3.402823466e38f ? v : __int_as_float(0x7fffffff); }
// The scale rule: block maximum -> scale and its inverse, each one f32 division.
__device__ __forceinline__ void f8_scale(float amax, float& scale, float& inv) {
    const float a = fmaxf(amax, kF8Floor);
    scale = __fdiv_rn(a, kF8Max);
    inv = __fdiv_rn(kF8Max, a);
}

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive values at a 16-byte aligned address.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
// Four consecutive values as they lie in memory (8 or 16 bytes in registers), read once and past the first-level cache:
// what streams through must not push out the vectors that every row reads again.
template <typename T>
struct Four {
    uint2 u;
    __device__ __forceinline__ void load(const T* p) {
        asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "l"(p));
    }
    // element-wise, for rows that are not aligned or end inside; values from column `left` on are zero
    __device__ __forceinline__ void load_some(const T* p, int left) {
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < left ? p[e] : narrow<T>(0.0f);
        memcpy(&u, v, 8);
    }
    __device__ __forceinline__ void get(float2& a, float2& b) const {
        T v[4];
        memcpy(v, &u, 8);
        a = make_float2(widen<T>(v[0]), widen<T>(v[1]));
        b = make_float2(widen<T>(v[2]), widen<T>(v[3]));
    }
};
template <>
struct Four<float> {
    float4 f;
    __device__ __forceinline__ void load(const float* p) {
        asm volatile("ld.global.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "l"(p));
    }
    __device__ __forceinline__ void load_some(const float* p, int left) {
        f.x = left > 0 ? p[0] : 0.0f;
        f.y = left > 1 ? p[1] : 0.0f;
        f.z = left > 2 ? p[2] : 0.0f;
        f.w = left > 3 ? p[3] : 0.0f;
    }
    __device__ __forceinline__ void get(float2& a, float2& b) const {
        a = make_float2(f.x, f.y);
        b = make_float2(f.z, f.w);
    }
};

// Four values to memory, written once (streaming).
__device__ __forceinline__ void put4(float* p, float2 a, float2 b) { __stcs(reinterpret_cast<float4*>(p), make_float4(a.x, a.y, b.x, b.y)); }
__device__ __forceinline__ void put4(__half* p, float2 a, float2 b) {
    const __half2 x = __float22half2_rn(a), y = __float22half2_rn(b);
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y)));
}
__device__ __forceinline__ void put4(__nv_bfloat16* p, float2 a, float2 b) {
    const __nv_bfloat162 x = __float22bfloat162_rn(a), y = __float22bfloat162_rn(b);
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y)));
}

}  // namespace edb
