// Elements of 32 or 16 bits read as 32-bit floats and written with one rounding to nearest; e^t, 2^t and 1 / d for arguments that stay away
// from the ends of the range: one instruction each beside a product, with numbers below the normal ones taken for 0 (the general forms spend
// three to four more on those). All are off by two units in the last place at most, e^t by 1.2 |t| more for the product's rounding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace vm {

__device__ __forceinline__ float to_float(float v) {
    return v;
}
__device__ __forceinline__ float to_float(__half v) {
    return __half2float(v);
}
__device__ __forceinline__ float to_float(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
__device__ __forceinline__ float exp_of(float t) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t * 1.44269504f));
    return e;
}
__device__ __forceinline__ float one_over(float d) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return r;
}

// 2^t
__device__ __forceinline__ float exp2_of(float t) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    return e;
}

// Two floats in one instruction each.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{.reg .b64 x, y, z, w; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 w, x, y, z; mov.b64 {%0, %1}, w;}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

// Two neighbouring elements: as floats, the larger of each (a number beside NaN), and not below `low` (NaN stays NaN).
template <typename T>
struct Pair;
template <>
struct Pair<float> {
    using type = float2;
    __device__ static __forceinline__ float2 floats(float2 v) {
        return v;
    }
    __device__ static __forceinline__ float2 larger(float2 a, float2 b) {
        return make_float2(fmaxf(a.x, b.x), fmaxf(a.y, b.y));
    }
    __device__ static __forceinline__ float2 bounded(float2 v, float2 low) {
        float2 r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r.x) : "f"(v.x), "f"(low.x));
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r.y) : "f"(v.y), "f"(low.y));
        return r;
    }
    __device__ static __forceinline__ float2 both(float v) {
        return make_float2(v, v);
    }
};
template <>
struct Pair<__half> {
    using type = __half2;
    __device__ static __forceinline__ float2 floats(__half2 v) {
        return __half22float2(v);
    }
    __device__ static __forceinline__ __half2 larger(__half2 a, __half2 b) {
        return __hmax2(a, b);
    }
    __device__ static __forceinline__ __half2 bounded(__half2 v, __half2 low) {
        return __hmax2_nan(v, low);
    }
    __device__ static __forceinline__ __half2 both(float v) {
        return __float2half2_rn(v);
    }
};
template <>
struct Pair<__nv_bfloat16> {
    using type = __nv_bfloat162;
    __device__ static __forceinline__ float2 floats(__nv_bfloat162 v) {
        return __bfloat1622float2(v);
    }
    __device__ static __forceinline__ __nv_bfloat162 larger(__nv_bfloat162 a, __nv_bfloat162 b) {
        return __hmax2(a, b);
    }
    __device__ static __forceinline__ __nv_bfloat162 bounded(__nv_bfloat162 v, __nv_bfloat162 low) {
        return __hmax2_nan(v, low);
    }
    __device__ static __forceinline__ __nv_bfloat162 both(float v) {
        return __float2bfloat162_rn(v);
    }
};

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

}  // namespace vm
