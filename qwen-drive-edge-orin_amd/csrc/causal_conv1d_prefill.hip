// Causal depthwise conv1d over prompts that continue from a state and hand one
// on, fixed-length or packed, for gfx950.  Channel d, token t of a sequence:
//   y[t][d] = act( sum_{j<K} w[d][j] r[t-K+1+j][d] + bias[d] )
// with r the sequence's tokens, and before its first one the state0 columns
// (newest last; zeros without one).  fp32 from the taps to the activation, one
// rounding at the end (causal_conv1d.hip rounds the sum to the weights' type
// in front of the activation, as the functions that it stands for do).
// state[d][p] = r[n - L + p][d], the last L tokens of state0 and sequence.
//
// Bound by HBM (x once, y once) and, next to it, by SiLU's exponential and
// reciprocal.  A thread owns 8 channels (16 bytes) and a run of kRun consecutive
// tokens of the row, whose loads are all issued before
// anything is waited for; neighbouring runs share K - 1 rows (L2).  The
// sequence of a run's first token comes from a search in cu_seqlens that
// overlaps those loads (their addresses do not depend on it), and where a
// run crosses into the next sequence (or into the first, where cu_seqlens does
// not start at 0) the window is refilled from that sequence's state, so that
// packed rows need neither padding nor a table.
// The new states are formed by threads of their own behind the last run
// (K rows each, in the cache), empty sequences among them.
#include "gdn_common.h"
#include "gdn_hip.h"
#include "gdn_io.h"
#include "gdn_seq.h"

#include <algorithm>

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxState = 8;

struct ConvArgs {
    const uint16_t* x;
    const void *w, *bias;
    const uint16_t* state0;
    uint16_t *y, *state;
    const int32_t* cu;
    int64_t xbs, xts, ybs, yts;
    int B, T, D, L, seqs;
    int vecs;        // D / 8
    int runs;        // runs of a batch row
    uint32_t units;  // (B x runs + seqs) x vecs
};

// Work-groups are dealt round-robin to the 8 XCDs: one contiguous range of
// units per XCD keeps neighbouring runs' shared rows in one L2
__device__ __forceinline__ uint32_t xcd_group(uint32_t id, uint32_t n) {
    const uint32_t q = n / 8, r = n % 8, xcd = id % 8;
    return xcd * q + min(xcd, r) + id / 8;
}

// COUNT consecutive parameters (a multiple of 8) at a 16-byte boundary
template <int WT, int COUNT>
__device__ __forceinline__ void load_params(const void* p, size_t first, float (&out)[COUNT]) {
    if constexpr (WT == 2) {
        const f32x4* v = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + first);
#pragma unroll
        for (int i = 0; i < COUNT / 4; ++i) {
            const f32x4 r = v[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) out[4 * i + j] = r[j];
        }
    } else {
        const u32x4* v = reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + first);
#pragma unroll
        for (int i = 0; i < COUNT / 8; ++i) {
            const u32x4 r = v[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                out[8 * i + 2 * j] = io_lo<WT>(r[j]);
                out[8 * i + 2 * j + 1] = io_hi<WT>(r[j]);
            }
        }
    }
}

__device__ __forceinline__ uint16_t half_of(const u32x4& v, int e) {
    const uint32_t u = e < 2 ? v[0] : e < 4 ? v[1] : e < 6 ? v[2] : v[3];
    return (uint16_t)(e & 1 ? u >> 16 : u);
}

template <int IO, int WT, int K, bool SILU, int kRun>
__global__ __launch_bounds__(kThreads) void causal_conv1d_prefill_kernel(const ConvArgs a) {
    const uint32_t unit = xcd_group(blockIdx.x, gridDim.x) * kThreads + threadIdx.x;
    if (unit >= a.units) return;
    const uint32_t row = unit / (uint32_t)a.vecs;
    const int d0 = 8 * (int)(unit - row * a.vecs);
    const uint32_t token_units = (uint32_t)a.B * a.runs;

    if (row >= token_units) {   // the state that sequence s hands on
        const int s = (int)(row - token_units);
        const int b = a.cu ? 0 : s;
        const int64_t lo = seq_lo(a.cu, 0, a.T, a.cu ? s : 0);
        const int n = seq_count(a.cu, a.T, a.T, s);
        const uint16_t* xb = a.x + b * a.xbs + lo * a.xts + d0;
        const size_t so = ((size_t)s * a.D + d0) * a.L;
        uint16_t col[kMaxState][8];
#pragma unroll
        for (int p = 0; p < kMaxState; ++p) {
            if (p >= a.L) break;
            const int i = n - a.L + p;
            if (i >= 0) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(xb + (size_t)i * a.xts);
#pragma unroll
                for (int e = 0; e < 8; ++e) col[p][e] = half_of(v, e);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) col[p][e] = a.state0 ? a.state0[so + (size_t)e * a.L + a.L + i] : (uint16_t)0;
            }
        }
        if (a.L == 4) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                u32x4 v;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    v[q] = (uint32_t)col[2 * (q & 1)][e + (q >> 1)] |
                           ((uint32_t)col[2 * (q & 1) + 1][e + (q >> 1)] << 16);
                *reinterpret_cast<u32x4*>(a.state + so + e * 4) = v;
            }
        } else {
#pragma unroll
            for (int p = 0; p < kMaxState; ++p) {
                if (p >= a.L) break;
#pragma unroll
                for (int e = 0; e < 8; ++e) a.state[so + (size_t)e * a.L + p] = col[p][e];
            }
        }
        return;
    }

    const int b = (int)(row / (uint32_t)a.runs);
    const int t0 = (int)(row - (uint32_t)b * a.runs) * kRun;
    const int len = min(kRun, a.T - t0);   // >= 1
    const uint16_t* xb = a.x + b * a.xbs + d0;
    uint16_t* yb = a.y + b * a.ybs + d0;
    // rows t0-K+1 .. t0+len-1; slots in front of the row and past the run
    // read a row of it again
    u32x4 raw[kRun + K - 1];
#pragma unroll
    for (int i = 0; i < kRun + K - 1; ++i) {
        const int t = min(max(t0 - (K - 1) + i, 0), t0 + len - 1);
        raw[i] = *reinterpret_cast<const u32x4*>(xb + (size_t)t * a.xts);
    }
    float wf[8 * K], bf[8];   // wf[e K + j]
    load_params<WT>(a.w, (size_t)d0 * K, wf);
    load_params<WT>(a.bias ? a.bias : a.w, a.bias ? d0 : 0, bf);
#pragma unroll
    for (int e = 0; e < 8; ++e) bf[e] = a.bias ? bf[e] : 0.f;
    __builtin_amdgcn_sched_barrier(0);   // every load is issued before the search waits

    int s = b, lo = 0, hi = a.T;
    if (a.cu) {   // the first sequence that ends behind t0
        int l = 0, h = a.seqs;
        while (l < h) {
            const int mid = (l + h) >> 1;
            if (clamp_tok(a.cu[mid + 1], a.T) > t0) h = mid;
            else l = mid + 1;
        }
        s = l;
        if (s >= a.seqs) return;   // behind the last sequence
        lo = seq_lo(a.cu, 0, a.T, s);
        hi = lo + seq_count(a.cu, 0, a.T, s);
    }
    int edge = t0 < lo ? lo : hi;   // the next token at which a sequence begins or ends
    auto state_tap = [&](int e, int back) {   // channel e of sequence s, `back` tokens before its first
        return a.state0 ? io_elem<IO>(a.state0, ((size_t)s * a.D + d0 + e) * a.L + a.L - back) : 0.f;
    };
    float win[K][8];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        const int t = t0 - (K - 1) + j;
        if (t >= lo) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                win[j][2 * p] = io_lo<IO>(raw[j][p]);
                win[j][2 * p + 1] = io_hi<IO>(raw[j][p]);
            }
        } else {
            const int back = min(lo - t, a.L);
#pragma unroll
            for (int e = 0; e < 8; ++e) win[j][e] = state_tap(e, back);
        }
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        if (i >= len) return;
        const int t = t0 + i;
        if (t == edge) {
            while (hi <= t) {   // into the next sequence that has tokens
                if (++s >= a.seqs) return;
                lo = seq_lo(a.cu, 0, a.T, s);
                hi = lo + seq_count(a.cu, 0, a.T, s);
            }
            edge = t < lo ? lo : hi;
            if (t >= lo) {
#pragma unroll
                for (int j = 0; j < K - 1; ++j) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) win[j][e] = state_tap(e, K - 1 - j);
                }
            }
        }
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            win[K - 1][2 * p] = io_lo<IO>(raw[i + K - 1][p]);
            win[K - 1][2 * p + 1] = io_hi<IO>(raw[i + K - 1][p]);
        }
        u32x4 out;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            float v[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int e = 2 * p + q;
                float acc = bf[e];
#pragma unroll
                for (int j = 0; j < K; ++j) acc = fmaf(wf[e * K + j], win[j][e], acc);
                v[q] = SILU ? silu_fast(acc) : acc;
            }
            out[p] = io_pack<IO>(v[0], v[1]);
        }
        // (rows in front of the first sequence are no sequence's)
        if (t >= lo) __builtin_nontemporal_store(out, reinterpret_cast<u32x4*>(yb + (size_t)t * a.yts));
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) win[j][e] = win[j + 1][e];
        }
    }
}

template <int IO, int WT, int K, bool SILU, int kRun>
hipError_t launch_run(ConvArgs& a, hipStream_t stream) {
    a.runs = (a.T + kRun - 1) / kRun;
    const int64_t units = ((int64_t)a.B * a.runs + a.seqs) * a.vecs;
    if (units > 0x7fffffff) return hipErrorInvalidValue;
    a.units = (uint32_t)units;
    const int64_t groups = (units + kThreads - 1) / kThreads;
    hipLaunchKernelGGL((causal_conv1d_prefill_kernel<IO, WT, K, SILU, kRun>), dim3((unsigned)groups),
                       dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

// Runs of 8 tokens re-read the fewest rows, but leave a short prompt too few
// waves: below 3 a SIMD, runs of 3 (1141 tokens x 6144 channels: 8.2 us against
// 9.6; 19,861 packed x 4352: 96.0 against 73.8, which is 4.7 TB/s).
template <int IO, int WT, int K>
hipError_t launch(ConvArgs& a, int silu, hipStream_t stream) {
    const bool wide = (int64_t)a.B * ((a.T + 7) / 8) * a.vecs >= 3 * 1024 * 64;
    if (silu) return wide ? launch_run<IO, WT, K, true, 8>(a, stream) : launch_run<IO, WT, K, true, 3>(a, stream);
    return wide ? launch_run<IO, WT, K, false, 8>(a, stream) : launch_run<IO, WT, K, false, 3>(a, stream);
}

template <int IO, int WT>
hipError_t launch_taps(ConvArgs& a, int K, int silu, hipStream_t stream) {
    if (K == 4) return launch<IO, WT, 4>(a, silu, stream);
    if (K == 3) return launch<IO, WT, 3>(a, silu, stream);
    return launch<IO, WT, 2>(a, silu, stream);
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" hipError_t gdn_causal_conv1d_prefill(const void* x, const void* w, const void* bias,
                                                const void* state0, void* y, void* state, int B,
                                                int T, int D, int K, int state_len,
                                                int64_t x_bstride, int64_t x_tstride,
                                                int64_t y_bstride, int64_t y_tstride,
                                                const int32_t* cu_seqlens, int num_seqs,
                                                int io_dtype, int w_dtype, int silu,
                                                hipStream_t stream) {
    if (B < 1 || T < 0 || D < 8 || D % 8 != 0 || K < 2 || K > 4) return hipErrorInvalidValue;
    if (state_len < K - 1 || state_len > kMaxState || (silu != 0 && silu != 1))
        return hipErrorInvalidValue;
    if (io_dtype != GDN_DTYPE_BF16 && io_dtype != GDN_DTYPE_FP16) return hipErrorInvalidValue;
    if (w_dtype != io_dtype && w_dtype != GDN_DTYPE_FP32) return hipErrorInvalidValue;
    if (num_seqs < 1 || (cu_seqlens ? B != 1 : num_seqs != B)) return hipErrorInvalidValue;
    if (!w || !state || state == state0 || (T > 0 && (!x || !y))) return hipErrorInvalidValue;
    if ((x_bstride | x_tstride | y_bstride | y_tstride) % 8 != 0 || x_bstride < 0 ||
        x_tstride < 0 || y_bstride < 0 || y_tstride < 0 ||
        ((uintptr_t)x | (uintptr_t)y | (uintptr_t)state | (uintptr_t)state0 | (uintptr_t)w |
         (uintptr_t)bias) %
                16 !=
            0)
        return hipErrorInvalidValue;
    ConvArgs a{static_cast<const uint16_t*>(x), w, bias, static_cast<const uint16_t*>(state0),
               static_cast<uint16_t*>(y), static_cast<uint16_t*>(state), cu_seqlens, x_bstride,
               x_tstride, y_bstride, y_tstride, B, T, D, state_len, num_seqs, D / 8, 0, 0};
    const bool w32 = w_dtype == GDN_DTYPE_FP32;
    if (io_dtype == GDN_DTYPE_BF16)
        return w32 ? launch_taps<0, 2>(a, K, silu, stream) : launch_taps<0, 0>(a, K, silu, stream);
    return w32 ? launch_taps<1, 2>(a, K, silu, stream) : launch_taps<1, 1>(a, K, silu, stream);
}
