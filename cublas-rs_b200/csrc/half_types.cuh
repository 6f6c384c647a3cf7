// half_types.cuh -- the two 16-bit element types (binary16 and bfloat16) of
// the grouped and 4-bit-weight kernels, as bit patterns in uint16_t.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace b2b {

template <bool BF16>
struct Half16;

template <>
struct Half16<false> {
    static constexpr float kMax = 65504.0f;
    static constexpr float kNormal = 6.103515625e-05f;  // 2^-14
    __device__ __forceinline__ static float get(uint16_t v) { return __half2float(__ushort_as_half(v)); }
    __device__ __forceinline__ static uint16_t put(float v) { return __half_as_ushort(__float2half_rn(v)); }
    // Two values to one word, the first in the low half.
    __device__ __forceinline__ static uint32_t put2(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    __device__ __forceinline__ static float2 get2(uint32_t v) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&v));
    }
};

template <>
struct Half16<true> {
    static constexpr float kMax = 3.38953138925153547590e38f;
    static constexpr float kNormal = 1.17549435082228750797e-38f;  // 2^-126
    __device__ __forceinline__ static float get(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
    __device__ __forceinline__ static uint16_t put(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
    __device__ __forceinline__ static uint32_t put2(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    __device__ __forceinline__ static float2 get2(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
};

}  // namespace b2b
