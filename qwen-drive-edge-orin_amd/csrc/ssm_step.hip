// Selective state-space step (decode, T >= 1 tokens a sequence) for gfx950,
// and the same recurrence over whole sequences where the chunked scan has no
// instance.  Per token of a head, state S [N][P] in fp32, B and C of the head's group:
//   d = clamp(softplus(dt + dt_bias), dt_min, dt_max),  a = exp(-exp(A_log) d)
//   S <- a S + (d B) x^T
//   y = (S^T C + D x) silu(z)
//
// Columns of S evolve independently, so a wave takes 32 columns of one head on
// its own: lane l owns columns 4 (l % 8) .. + 3 of the N / 8 rows from
// (l / 8) N / 8 on.  Every load of the state moves eight whole 128-byte lines,
// a lane's B and C values are consecutive, the sum over rows is three lane
// exchanges, and nothing meets in LDS: no barrier stands between the state's
// arrival and its way back.  The state crosses HBM once each way; tokens after
// the first reuse the registers.  (16 columns a wave, twice the waves with
// half the loads each: 5.5 us against 5.3 for one user of 64 heads, 51.8
// against 39.4 for 48.)
#include "gdn_seq.h"
#include "gdn_ssm.h"

namespace gdn {
namespace {


constexpr int kStepCols = 32;   // columns of a wave

struct StepArgs {
    gdn_ssm_inputs in;
    uint16_t* y;
    const float* state_in;    // null: zeros; may be state_out
    float* state_out;
    const int32_t* slots;     // the state of batch row b, or null: b
    const int32_t* cu;        // packed sequences (in.batch is 1), or null
    int num_slots, seqs;
    int col_tiles;    // waves a head
    int64_t tasks;    // sequences x heads x col_tiles
};

// RN consecutive 16-bit values as they lie in memory
template <int RN>
struct Raw {
    uint32_t w[RN / 2];
    __device__ __forceinline__ void load(const uint16_t* p) {
        if constexpr (RN >= 8) {
#pragma unroll
            for (int i = 0; i < RN / 8; ++i) {
                const u32x4 v = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < RN / 2; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        }
    }
};

template <int IO, int N>
__global__ __launch_bounds__(256) void ssm_step_kernel(const StepArgs a) {
    constexpr int RN = N / 8;   // rows of a lane
    const int lane = threadIdx.x & 63;
    const int64_t task = (int64_t)blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    if (task >= a.tasks) return;
    const gdn_ssm_inputs& in = a.in;
    const int H = in.heads, P = in.head_dim;
    const unsigned bh = (unsigned)(task / a.col_tiles);
    const int tile = (int)(task - (int64_t)bh * a.col_tiles);
    const int b = bh / (unsigned)H, h = bh - b * H;
    const int g = h / (H / in.groups);
    const int p0 = tile * kStepCols + 4 * (lane & 7);
    const bool cols = p0 < P;           // P is a multiple of 16: a lane's four columns are in or out
    const int pc = cols ? p0 : 0;
    const int n0 = (lane >> 3) * RN;

    // the sequence's rows: batch row `row`, tokens t0 .. t0 + T - 1
    const int row = a.cu ? 0 : b, T = seq_count(a.cu, in.tokens, in.tokens, b);
    const int64_t t0 = a.cu ? seq_lo(a.cu, in.tokens, in.tokens, b) : 0;
    uint16_t* yp = a.y + (((size_t)row * in.tokens + t0) * H + h) * P + pc;
    int64_t slot = b;
    if (a.slots) {
        slot = a.slots[b];
        if (slot < 0 || slot >= a.num_slots) {   // a row of the batch without a request
            if (cols && lane < 8)
                for (int t = 0; t < T; ++t) *reinterpret_cast<uint2*>(yp + (size_t)t * H * P) = make_uint2(0, 0);
            return;
        }
    }
    const uint16_t* xp = static_cast<const uint16_t*>(in.x) + row * in.x_batch + t0 * in.x_token + (size_t)h * P + pc;
    const uint16_t* bp = static_cast<const uint16_t*>(in.b) + row * in.b_batch + t0 * in.b_token + (size_t)g * N + n0;
    const uint16_t* cp = static_cast<const uint16_t*>(in.c) + row * in.c_batch + t0 * in.c_token + (size_t)g * N + n0;
    const uint16_t* zp = in.z ? static_cast<const uint16_t*>(in.z) + row * in.z_batch + t0 * in.z_token + (size_t)h * P + pc : nullptr;
    const size_t dp = (size_t)(row * in.dt_batch + t0 * in.dt_token + h);
    const bool dt32 = in.dt_dtype == GDN_DTYPE_FP32;
    auto load_dt = [&](int t) {
        const size_t i = dp + (size_t)t * in.dt_token;
        return dt32 ? io_elem<2>(in.dt, i) : io_elem<IO>(in.dt, i);
    };

    // token 0's inputs first, then the state: the short chain from dt to the
    // decay runs while the state is on its way
    Raw<RN> br, cr;
    float dtr = 0.f;
    uint2 xr = make_uint2(0, 0), zr = make_uint2(0, 0);
    if (T > 0) {   // (an empty sequence only hands its state on)
        dtr = load_dt(0);
        xr = *reinterpret_cast<const uint2*>(xp);
        if (zp) zr = *reinterpret_cast<const uint2*>(zp);
        br.load(bp);
        cr.load(cp);
    }
    const float A = -expf(in.A_log[h]);
    const float bias = in.dt_bias ? in.dt_bias[h] : 0.f;
    const float D = in.D ? in.D[h] : 0.f;
    const size_t so = (((size_t)slot * H + h) * N + n0) * P + pc;
    f32x4 s[RN];
#pragma unroll
    for (int r = 0; r < RN; ++r) s[r] = zero4();
    if (a.state_in) {
#pragma unroll
        for (int r = 0; r < RN; ++r)
            s[r] = *reinterpret_cast<const f32x4_a4*>(a.state_in + so + (size_t)r * P);
    }

    for (int t = 0; t < T; ++t) {
        const float d = ssm_delta(dtr, bias, in.dt_min, in.dt_max);
        const float decay = expf(A * d);
        f32x4 x, z;
        x[0] = io_lo<IO>(xr.x); x[1] = io_hi<IO>(xr.x);
        x[2] = io_lo<IO>(xr.y); x[3] = io_hi<IO>(xr.y);
        z[0] = io_lo<IO>(zr.x); z[1] = io_hi<IO>(zr.x);
        z[2] = io_lo<IO>(zr.y); z[3] = io_hi<IO>(zr.y);
        const Raw<RN> bt = br, ct = cr;
        if (t + 1 < T) {   // the next token's inputs, behind this one's arithmetic
            dtr = load_dt(t + 1);
            xr = *reinterpret_cast<const uint2*>(xp + (size_t)(t + 1) * in.x_token);
            if (zp) zr = *reinterpret_cast<const uint2*>(zp + (size_t)(t + 1) * in.z_token);
            br.load(bp + (size_t)(t + 1) * in.b_token);
            cr.load(cp + (size_t)(t + 1) * in.c_token);
        }
        const f32x4 u = x * d;
        f32x4 acc = zero4();
#pragma unroll
        for (int r = 0; r < RN; ++r) {
            const float bv = r & 1 ? io_hi<IO>(bt.w[r / 2]) : io_lo<IO>(bt.w[r / 2]);
            const float cv = r & 1 ? io_hi<IO>(ct.w[r / 2]) : io_lo<IO>(ct.w[r / 2]);
            s[r] = s[r] * decay + u * bv;
            acc += s[r] * cv;
        }
#pragma unroll
        for (int off = 8; off < 64; off <<= 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], off, 64);
        }
        if (cols && lane < 8) {
            f32x4 o = acc + x * D;
            if (zp) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] *= silu_fast(z[i]);
            }
            *reinterpret_cast<uint2*>(yp + (size_t)t * H * P) =
                make_uint2(io_pack<IO>(o[0], o[1]), io_pack<IO>(o[2], o[3]));
        }
    }
    if (cols) {
#pragma unroll
        for (int r = 0; r < RN; ++r)
            __builtin_nontemporal_store(
                s[r], reinterpret_cast<f32x4_a4*>(a.state_out + so + (size_t)r * P));
    }
}

template <int IO>
hipError_t launch(StepArgs& a, hipStream_t stream) {
    a.col_tiles = (a.in.head_dim + kStepCols - 1) / kStepCols;
    a.tasks = (int64_t)a.seqs * a.in.heads * a.col_tiles;
    // one wave a group while the waves cannot fill the chip twice over: they
    // then spread over all compute units
    const int waves = a.tasks <= 2048 ? 1 : 4;
    const int64_t groups = (a.tasks + waves - 1) / waves;
    if (groups > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)groups), block(64 * waves);
    switch (a.in.state_dim) {
        case 16: hipLaunchKernelGGL((ssm_step_kernel<IO, 16>), grid, block, 0, stream, a); break;
        case 32: hipLaunchKernelGGL((ssm_step_kernel<IO, 32>), grid, block, 0, stream, a); break;
        case 64: hipLaunchKernelGGL((ssm_step_kernel<IO, 64>), grid, block, 0, stream, a); break;
        case 128: hipLaunchKernelGGL((ssm_step_kernel<IO, 128>), grid, block, 0, stream, a); break;
        default: hipLaunchKernelGGL((ssm_step_kernel<IO, 256>), grid, block, 0, stream, a); break;
    }
    return hipGetLastError();
}

hipError_t launch_step(StepArgs& a, hipStream_t stream) {
    if ((int64_t)a.seqs * a.in.heads > 0x7fffffff) return hipErrorInvalidValue;
    return a.in.io_dtype == GDN_DTYPE_BF16 ? launch<0>(a, stream) : launch<1>(a, stream);
}

}  // namespace

hipError_t ssm_recurrent(const gdn_ssm_inputs& in, void* y, const float* s0, float* sf,
                         const int32_t* cu, int seqs, hipStream_t stream) {
    StepArgs a{};
    a.in = in;
    a.y = static_cast<uint16_t*>(y);
    a.state_in = s0;
    a.state_out = sf;
    a.cu = cu;
    a.seqs = seqs;
    return launch_step(a, stream);
}

}  // namespace gdn

using namespace gdn;

extern "C" hipError_t gdn_ssm_step(const gdn_ssm_inputs* in, void* y, float* state,
                                   const int32_t* slots, int num_slots, hipStream_t stream) {
    if (!ssm_inputs_ok(in) || !state || (slots && num_slots < 1)) return hipErrorInvalidValue;
    if (in->tokens == 0) return hipSuccess;
    if (!y || !ssm_aligned(y, 8) || !ssm_aligned(state, 4)) return hipErrorInvalidValue;
    StepArgs a{};
    a.in = *in;
    a.y = static_cast<uint16_t*>(y);
    a.state_in = a.state_out = state;
    a.slots = slots;
    a.num_slots = num_slots;
    a.seqs = in->batch;
    return launch_step(a, stream);
}
