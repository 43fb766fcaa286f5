// f8blk.cuh - e4m3 with one f32 scale per block of 128: the quantizer's rule, shared by every kernel that writes such operands.
//
//   weights      q e4m3 [out][in], scale f32 [ceil(out / 128)][ceil(in / 128)]: one per 128 x 128 tile
//   activations  q e4m3 [token][in], scale f32 [token][ceil(in / 128)]: one per token and 128 elements
//
// Rule for the values of a block: a = max |v|, s = max(a / 448, 2^-126), code = RN_e4m3(v * (1 / s)), all in f32 with the IEEE
// quotient; 448 is the largest e4m3 value, and the conversion saturates, so v * (1 / s) an ulp above 448 is 448.  The floor keeps 1 / s
// finite and makes a block of zeros codes of zero.  A NaN leaves the maximum alone and keeps its own code (NaN); an infinity
// makes the scale infinite and its own code NaN.  Either way the whole token is NaN behind a product, as it would be in f32.
#pragma once
#include <cuda_fp8.h>

#include "pdk_common.cuh"

namespace f8blk {

constexpr uint32_t kBlock = 128;

__host__ __device__ __forceinline__ uint32_t blocks_of(uint32_t n) { return n / kBlock + (n % kBlock != 0u); }

__device__ __forceinline__ float scale_of(float amax) { return fmaxf(amax / 448.0f, 1.17549435e-38f); }

// two codes, the first in the low byte
__device__ __forceinline__ uint32_t codes2(float a, float b, float r) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a * r, b * r), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float r) {
    return codes2(a, b, r) | codes2(c, d, r) << 16;
}
__device__ __forceinline__ uint8_t code1(float v, float r) {
    return (uint8_t)__nv_cvt_float_to_fp8(v * r, __NV_SATFINITE, __NV_E4M3);
}
// two values of two codes
__device__ __forceinline__ float2 values2(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace f8blk
