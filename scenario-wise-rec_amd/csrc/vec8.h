// 8 consecutive elements of a row of bf16 or fp32 values, loaded and stored 8, 4 or 1 at a time (whatever the row's alignment allows).
#pragma once
#include "common.h"
#include "split3.h"

template <typename T> struct Raw8;
template <> struct Raw8<uint16_t> { uint4 v; };
template <> struct Raw8<float> { float4 a, b; };

// n: elements of the row from `p` on (<= 0: none, zeros come back); vw: 8 / 4 / 1 elements per load (swr_vec8)
__device__ __forceinline__ Raw8<uint16_t> load8(const uint16_t* p, int n, int vw) {
    Raw8<uint16_t> r;
    r.v = make_uint4(0, 0, 0, 0);
    if (n <= 0) return r;
    if (vw == 8) {
        r.v = *reinterpret_cast<const uint4*>(p);
    } else if (vw == 4) {
        const uint2 lo = *reinterpret_cast<const uint2*>(p);
        r.v.x = lo.x; r.v.y = lo.y;
        if (n > 4) { const uint2 hi = *reinterpret_cast<const uint2*>(p + 4); r.v.z = hi.x; r.v.w = hi.y; }
    } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) w[j >> 1] |= static_cast<uint32_t>(p[j]) << (16 * (j & 1));
        r.v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
}
__device__ __forceinline__ Raw8<float> load8(const float* p, int n, int vw) {
    Raw8<float> r;
    r.a = make_float4(0.f, 0.f, 0.f, 0.f);
    r.b = r.a;
    if (n <= 0) return r;
    if (vw >= 4) {
        r.a = *reinterpret_cast<const float4*>(p);
        if (n > 4) r.b = *reinterpret_cast<const float4*>(p + 4);
    } else {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = j < n ? p[j] : 0.f;
        r.a = make_float4(w[0], w[1], w[2], w[3]);
        r.b = make_float4(w[4], w[5], w[6], w[7]);
    }
    return r;
}
__device__ __forceinline__ Raw8<uint16_t> zero8(Raw8<uint16_t> r) { r.v = make_uint4(0, 0, 0, 0); return r; }
__device__ __forceinline__ Raw8<float> zero8(Raw8<float> r) { r.a = r.b = make_float4(0.f, 0.f, 0.f, 0.f); return r; }
__device__ __forceinline__ void floats8(const Raw8<uint16_t>& r, float* f) {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = __uint_as_float(w[j] << 16);
        f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
}
__device__ __forceinline__ void floats8(const Raw8<float>& r, float* f) {
    f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w; f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
}
__device__ __forceinline__ void store8(uint16_t* p, int n, int vw, const float* x) {
    if (n <= 0) return;
    bf16x8 b;
#pragma unroll
    for (int j = 0; j < 8; j += 2) CVT_PAIR(x[j], x[j + 1], b, j);
    const uint4 v = __builtin_bit_cast(uint4, b);
    if (vw == 8) {
        *reinterpret_cast<uint4*>(p) = v;
    } else if (vw == 4) {
        *reinterpret_cast<uint2*>(p) = make_uint2(v.x, v.y);
        if (n > 4) *reinterpret_cast<uint2*>(p + 4) = make_uint2(v.z, v.w);
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) p[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
    }
}
__device__ __forceinline__ void store8(float* p, int n, int vw, const float* x) {
    if (n <= 0) return;
    if (vw >= 4) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        if (n > 4) *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) p[j] = x[j];
    }
}

// elements per load of rows of `width` elements (strides in elements): 8 needs 16-byte, 4 its own size alignment
static inline int swr_vec8(const void* p, int64_t stride0, int64_t stride1, int width, int elem) {
    const uintptr_t u = reinterpret_cast<uintptr_t>(p);
    if (width % 8 == 0 && u % 16 == 0 && stride0 * elem % 16 == 0 && stride1 * elem % 16 == 0) return 8;
    if (width % 4 == 0 && u % (4 * elem) == 0 && stride0 % 4 == 0 && stride1 % 4 == 0) return 4;
    return 1;
}
