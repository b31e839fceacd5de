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

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// two fp32 values rounded to nearest-even 16-bit values and packed (a low): one
// v_cvt_pk_bf16_f32 / v_cvt_pk_f16_f32.  Not as inline asm: its result may be
// an MFMA operand and its inputs MFMA results, and the wait states between
// those and a vector instruction are placed by the compiler, which does not
// look into asm.
template <int IO>
__device__ __forceinline__ uint32_t io_pack(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (IO == 0) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2v));
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
