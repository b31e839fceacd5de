// Gated norm over groups of a row of channels, for gfx950:
//   u = x silu(z) (gate first) or x
//   y = u rsqrt(mean_group(u^2) + eps) w  [silu(z)]
// in fp32 with one rounding at the end.  The norm behind a state-space scan,
// whose groups are 512 to 8192 channels wide (the gated RMSNorm of the
// gated-delta layers covers 128-wide rows, gates after the norm and rounds
// where transformers does).
//
// A group of S channels belongs to LPG lanes, each with 16-byte pieces at
// stride 8 LPG, so that a piece index is one coalesced run; up to 64 lanes it
// is a lane-group sum, with 256 lanes the four waves add up in LDS.  x and z
// stay in registers between the sum and the output: HBM sees each once.
// HBM-bound: 19,861 rows of 4096 in one group 85 us (5.7 TB/s, more than a large
// copy's 4.7); 48 rows 2.6 us, a launch.
#include "gdn_common.h"
#include "gdn_hip.h"
#include "gdn_io.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;

template <int IO, int W, int LPG, int NP, bool kGateFirst>
__global__ __launch_bounds__(kThreads) void gated_groupnorm_kernel(
    const uint16_t* __restrict__ x, int64_t x_row, const uint16_t* __restrict__ z, int64_t z_row,
    const void* __restrict__ w, uint16_t* __restrict__ y, int64_t tasks, int groups, int S,
    float eps) {
    __shared__ float red[kThreads / 64];
    const int64_t task = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / LPG;
    const int sub = threadIdx.x % LPG;
    const bool active = task < tasks;   // (only whole lane groups are inactive)
    const int64_t tk = active ? task : tasks - 1;
    const int64_t row = tk / groups;
    const int c0 = (int)(tk - row * groups) * S;
    const uint16_t* xp = x + row * x_row + c0;
    const uint16_t* zp = z + row * z_row + c0;
    u32x4 xr[NP], zr[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int e = (sub + j * LPG) * 8;
        const bool in = e < S;
        xr[j] = in ? *reinterpret_cast<const u32x4*>(xp + e) : u32x4{0, 0, 0, 0};
        zr[j] = in ? *reinterpret_cast<const u32x4*>(zp + e) : u32x4{0, 0, 0, 0};
    }
    float u[NP][8], gate[NP][8];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            u[j][2 * p] = io_lo<IO>(xr[j][p]);
            u[j][2 * p + 1] = io_hi<IO>(xr[j][p]);
            gate[j][2 * p] = silu_fast(io_lo<IO>(zr[j][p]));
            gate[j][2 * p + 1] = silu_fast(io_hi<IO>(zr[j][p]));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (kGateFirst) u[j][e] *= gate[j][e];
            ss = fmaf(u[j][e], u[j][e], ss);
        }
    }
    if constexpr (LPG <= 64) {
        ss = lane_group_sum<LPG>(ss);
    } else {
        ss = lane_group_sum<64>(ss);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
        __syncthreads();
        ss = red[0] + red[1] + red[2] + red[3];
    }
    const float r = 1.0f / sqrtf(ss / (float)S + eps);
    if (!active) return;
    uint16_t* yp = y + tk * S;   // packed rows: row * C + c0
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int e = (sub + j * LPG) * 8;
        if (e >= S) continue;
        float wf[8];
        if constexpr (W == 2) {
            const f32x4* wp = reinterpret_cast<const f32x4*>(static_cast<const float*>(w) + c0 + e);
            const f32x4 a = wp[0], b = wp[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                wf[i] = a[i];
                wf[4 + i] = b[i];
            }
        } else {
            const u32x4 a = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(w) + c0 + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                wf[2 * i] = io_lo<IO>(a[i]);
                wf[2 * i + 1] = io_hi<IO>(a[i]);
            }
        }
        u32x4 o;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            float v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 2 * p + h;
                v[h] = u[j][i] * r * wf[i];
                if (!kGateFirst) v[h] *= gate[j][i];
            }
            o[p] = io_pack<IO>(v[0], v[1]);
        }
        *reinterpret_cast<u32x4*>(yp + e) = o;
    }
}

struct NormArgs {
    const uint16_t *x, *z;
    const void* w;
    uint16_t* y;
    int64_t x_row, z_row, tasks;
    int groups, S;
    float eps;
};

template <int IO, int W, int LPG, int NP>
hipError_t launch(const NormArgs& a, bool gate_first, hipStream_t stream) {
    const int64_t per = kThreads / LPG, blocks = (a.tasks + per - 1) / per;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    auto kern = gate_first ? gated_groupnorm_kernel<IO, W, LPG, NP, true>
                           : gated_groupnorm_kernel<IO, W, LPG, NP, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kThreads), 0, stream, a.x, a.x_row, a.z,
                       a.z_row, a.w, a.y, a.tasks, a.groups, a.S, a.eps);
    return hipGetLastError();
}

// The fewest lanes that hold a group in at most two pieces each, in whole
// waves from 512 channels on
template <int IO, int W>
hipError_t launch_any(const NormArgs& a, bool gate_first, hipStream_t stream) {
    if (a.S <= 128) return launch<IO, W, 16, 1>(a, gate_first, stream);
    if (a.S <= 512) return launch<IO, W, 64, 1>(a, gate_first, stream);
    if (a.S <= 1024) return launch<IO, W, 64, 2>(a, gate_first, stream);
    if (a.S <= 2048) return launch<IO, W, 256, 1>(a, gate_first, stream);
    if (a.S <= 4096) return launch<IO, W, 256, 2>(a, gate_first, stream);
    if (a.S <= 8192) return launch<IO, W, 256, 4>(a, gate_first, stream);
    return launch<IO, W, 256, 8>(a, gate_first, stream);
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" hipError_t gdn_gated_groupnorm_forward(const void* x, int64_t x_row, const void* z,
                                                  int64_t z_row, const void* w, void* y,
                                                  int64_t rows, int C, int groups, float eps,
                                                  int gate_first, int io_dtype, int w_dtype,
                                                  hipStream_t stream) {
    if (rows < 0 || C < 8 || groups < 1 || C % groups != 0) return hipErrorInvalidValue;
    const int S = C / groups;
    if (S % 8 != 0 || S > 16384 || !(eps >= 0.f)) return hipErrorInvalidValue;
    if (io_dtype != GDN_DTYPE_BF16 && io_dtype != GDN_DTYPE_FP16) return hipErrorInvalidValue;
    if (w_dtype != io_dtype && w_dtype != GDN_DTYPE_FP32) return hipErrorInvalidValue;
    if (gate_first != 0 && gate_first != 1) return hipErrorInvalidValue;
    if (rows > (int64_t)1 << 40) return hipErrorInvalidValue;
    if (rows == 0) return hipSuccess;
    if (!x || !z || !w || !y || x_row < 0 || z_row < 0 || (x_row | z_row) % 8 != 0 ||
        ((uintptr_t)x | (uintptr_t)z | (uintptr_t)y | (uintptr_t)w) % 16 != 0)
        return hipErrorInvalidValue;
    NormArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(z), w,
               static_cast<uint16_t*>(y), x_row, z_row, rows * groups, groups, S, eps};
    const bool w32 = w_dtype == GDN_DTYPE_FP32, gf = gate_first != 0;
    if (io_dtype == GDN_DTYPE_BF16)
        return w32 ? launch_any<0, 2>(a, gf, stream) : launch_any<0, 0>(a, gf, stream);
    return w32 ? launch_any<1, 2>(a, gf, stream) : launch_any<1, 1>(a, gf, stream);
}
