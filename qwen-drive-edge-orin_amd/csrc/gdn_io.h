// 16-bit element I/O shared by the state-space kernels: IO = 0 bf16, 1 fp16,
// 2 fp32 (parameters only); pairs are packed with element 0 in the low half.
#pragma once

#include "gdn_common.h"

namespace gdn {

template <int IO>
__device__ __forceinline__ float io_lo(uint32_t u) {
    if constexpr (IO == 0) return __uint_as_float(u << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(u & 0xffffu));
}

template <int IO>
__device__ __forceinline__ float io_hi(uint32_t u) {
    if constexpr (IO == 0) return __uint_as_float(u & 0xffff0000u);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
}

// two fp32 values rounded to nearest-even 16-bit values and packed (a low)
template <int IO>
__device__ __forceinline__ uint32_t io_pack(float a, float b) {
    if constexpr (IO == 0) {
        uint32_t u;
        asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(u) : "v"(a), "v"(b));
        return u;
    } else {
        const uint16_t x = __builtin_bit_cast(uint16_t, (_Float16)a);
        const uint16_t y = __builtin_bit_cast(uint16_t, (_Float16)b);
        return (uint32_t)x | ((uint32_t)y << 16);
    }
}

template <int IO>
__device__ __forceinline__ float io_elem(const void* p, size_t i) {
    if constexpr (IO == 2) return static_cast<const float*>(p)[i];
    return io_lo<IO>(static_cast<const uint16_t*>(p)[i]);
}

// z / (1 + e^-z) from the hardware base-2 exponential and reciprocal (each
// within about an fp32 ulp; below -87 the result is -0, exactly |y| < 1e-36)
__device__ __forceinline__ float silu_fast(float z) {
    return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

}  // namespace gdn
