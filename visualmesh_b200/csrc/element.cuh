// Elements of 32 or 16 bits read as 32-bit floats and written with one rounding to nearest; e^t and 1 / d for arguments that stay away
// from the ends of the range: one instruction each beside a product, with numbers below the normal ones taken for 0 (the general forms spend
// three to four more on those). Both are off by two units in the last place at most, e^t by 1.2 |t| more for the product's rounding.
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
