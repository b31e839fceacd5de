// What the state-space kernels share: the argument struct's device view, the
// step size and decay of a token, and the host checks.
#pragma once

#include "gdn_common.h"
#include "gdn_hip.h"
#include "gdn_io.h"

#include <math.h>

namespace gdn {

// d = clamp(softplus(raw + bias), lo, hi), softplus(x) = log1p(e^x), to a few
// fp32 ulps for any size of e^x: e^x from the base-2 exponential of x log2(e)
// in two parts, log1p(e) = log(u) e / (u - 1) with u = fl(1 + e), in which the
// rounding of u cancels (Goldberg, "What every computer scientist should know
// about floating-point arithmetic", theorem 4).  Above 20, log1p(e^x) is x;
// below -104, -infinity among it, e^x is 0 in fp32.  NaN stays NaN (the
// comparisons are written so that it does).
__device__ __forceinline__ float ssm_delta(float raw, float bias, float lo, float hi) {
    const float x = raw + bias;
    const float y = x > 20.f ? 20.f : x < -104.f ? -104.f : x;
    constexpr float kL = 1.44269502f, kLlo = 1.92596303e-08f;   // log2(e) and what it rounds off
    const float t = y * kL, r = fmaf(y, kLlo, fmaf(y, kL, -t));
    const float e0 = __builtin_amdgcn_exp2f(t);
    const float e = fmaf(e0, r * 0.693147182f, e0);
    const float u = 1.f + e, v = u - 1.f;
    const float q = __builtin_amdgcn_logf(u) * 0.693147182f * (e / v);
    const float d = x > 20.f ? x : v == 0.f ? e : q;
    return d < lo ? lo : d > hi ? hi : d;
}

inline bool ssm_aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int64_t kSsmMaxToken = 1 << 24;   // token strides: a chunk's offsets fit 32 bits

// Row strides that every 16-byte lane access of x, B, C and z needs
inline bool ssm_rows_ok(const void* p, int64_t batch, int64_t token) {
    return p && ssm_aligned(p, 16) && batch >= 0 && token >= 0 && token < kSsmMaxToken &&
           batch % 8 == 0 && token % 8 == 0;
}

// The sizes of gdn_ssm_inputs
inline bool ssm_sizes_ok(const gdn_ssm_inputs* a) {
    if (!a || a->batch < 1 || a->tokens < 0 || a->heads < 1 || a->groups < 1 ||
        a->heads % a->groups != 0)
        return false;
    if (a->head_dim < 16 || a->head_dim > 256 || a->head_dim % 16 != 0) return false;
    if (a->state_dim != 16 && a->state_dim != 32 && a->state_dim != 64 && a->state_dim != 128 &&
        a->state_dim != 256)
        return false;
    if ((int64_t)a->heads * a->head_dim >= kSsmMaxToken) return false;
    return true;
}

// Sizes, types and pointers
inline bool ssm_inputs_ok(const gdn_ssm_inputs* a) {
    if (!ssm_sizes_ok(a)) return false;
    if (a->io_dtype != GDN_DTYPE_BF16 && a->io_dtype != GDN_DTYPE_FP16) return false;
    if (a->dt_dtype != a->io_dtype && a->dt_dtype != GDN_DTYPE_FP32) return false;
    if (!(a->dt_min >= 0.f) || !(a->dt_max >= a->dt_min)) return false;
    if (a->tokens == 0) return true;
    if (!ssm_rows_ok(a->x, a->x_batch, a->x_token) || !ssm_rows_ok(a->b, a->b_batch, a->b_token) ||
        !ssm_rows_ok(a->c, a->c_batch, a->c_token) || !a->dt || !a->A_log || a->dt_batch < 0 ||
        a->dt_token < 0 || a->dt_token >= kSsmMaxToken)
        return false;
    return !a->z || ssm_rows_ok(a->z, a->z_batch, a->z_token);
}

// The recurrence over whole sequences, one wave per 32 columns of a head
// (ssm_step.hip): s0 null is zeros, s0 may be sf
hipError_t ssm_recurrent(const gdn_ssm_inputs& in, void* y, const float* s0, float* sf,
                         const int32_t* cu, int seqs, hipStream_t stream);

}  // namespace gdn
