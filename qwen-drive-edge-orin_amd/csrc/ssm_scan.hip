// Selective state-space scan over prompts for gfx950.
//
// Per head, with d_t = clamp(softplus(dt_t + dt_bias)), l_t = -exp(A_log) d_t
// and the head's group's B and C, a chunk of 64 tokens with state S [N][P] in
// front of it gives, with c = cumsum(l) in the chunk and c_Q its last value,
//   y_t = e^{c_t} S^T C_t + sum_{s <= t} (C_t . B_s) e^{c_t - c_s} d_s x_s + D x_t
//   S  <- e^{c_Q} S + sum_s B_s (e^{c_Q - c_s} d_s x_s)^T
// all of it matrix products (C B^T, S^T C^T, X^T M^T, B^T X) on MFMA, where
// the recurrence would pass over S once a token.
//
// Runs of `block` tokens (segments) are worked on side by side: a first pass
// forms each segment's state from zero (from s0 for a sequence's first one;
// the last segment needs none), a join turns those into the states in front
// of the segments, and the main pass starts each segment from its own.  A
// call whose sequences have one segment each runs the main pass alone.
//
// A wave owns 16 PT columns of one head: its slice of S stays in fp32
// accumulators through the segment, and the columns need nothing from one
// another.  Four waves of one group share B, C and the products C B^T in LDS.
// The MFMA operand and result layouts (gdn_common.h) chain without shuffles:
// S's tiles are the A operand of S^T C^T, C B^T comes out transposed as the B
// operand of X^T M^T, and rows are numbered so that two result tiles hold 8
// consecutive channels (perm below), 16 bytes of y.
//
// Rounding.  bf16: x, B and C are exact operands; S and M = (C B^T) o decay
// enter y's products as pairs of bf16 (2^-17 of each term, y itself has 2^-8),
// and d x, which enters the state, as three (2^-25).  Sums, states, decays:
// fp32.  Logarithms are summed in fp32 forwards for c and backwards for the
// state's weights, so that the weights of the newest tokens, the largest, are
// sums of few terms; a token's base-2 logarithm is held at -150, where its
// decay is 0 in fp32, to keep differences of c exact for the tokens behind it.
#include "gdn_seq.h"
#include "gdn_ssm.h"

#include <algorithm>

namespace gdn {
namespace {

constexpr int kMaxBlock = 1 << 20;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;

struct Seg {
    int seq, t0, n, idx;
    bool last;
};

struct ScanArgs {
    gdn_ssm_inputs in;
    uint16_t* y;
    const float* s0;
    float* sf;
    const int4* table;   // packed: blocks; null: `segs` segments of `block` tokens per batch row
    int rows;            // segments (bound)
    int segs, seqs, block;
    int slices;          // column slices of a head: ceil(P / PW)
    int tasks;           // slices of a group: heads / groups x slices
    int quads;           // ceil(tasks / 4): work-groups per group and segment
    f32x4* states;       // [row][group][task] fragments of a slice's state
    float* decays;       // [row][group][task]
};

// Segment r, clamped so that whatever a table holds its tokens lie in the row
__device__ __forceinline__ bool segment(const ScanArgs& a, int r, Seg& s) {
    if (!a.table) {
        s.seq = r / a.segs;
        s.idx = r - s.seq * a.segs;
        s.t0 = s.idx * a.block;
        s.n = min(a.block, a.in.tokens - s.t0);
        s.last = s.idx + 1 == a.segs;
        return true;
    }
    const int4 b = a.table[r];
    if (b.x < 0 || b.x >= a.seqs) return false;
    s.seq = b.x;
    s.t0 = min(max(b.y, 0), a.in.tokens);
    s.n = min(min(max(b.z, 0), a.block), a.in.tokens - s.t0);
    s.idx = b.w > 0 && r > 0 ? b.w : 0;
    s.last = r + 1 >= a.rows || a.table[r + 1].x != b.x;
    return true;
}

// Pieces (8 elements) of row r of a 16-bit tile with PR pieces a row, spread
// over the banks both for 16 rows' one piece (16-byte reads) and for 4 rows x
// 4 pieces (transposing reads)
template <int PR>
__device__ __forceinline__ int swz(int r) {
    if constexpr (PR >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (PR == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return 0;
}

template <int PR>
__device__ __forceinline__ const uint16_t* piece_at(const uint16_t* base, int r, int p) {
    return base + (size_t)(r * PR + (p ^ swz<PR>(r))) * 8;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// LDS transposing read (ds_read_b64_tr_b16): within 16 lanes, source lane s
// names elements X[s][0..3] and lane i receives X[4 j + i / 4][i % 4], j = 0..3
__device__ __forceinline__ s16x4 read_tr(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

// Transposed operand of a 64-row tile: lane (g, m) gets column
// perm(t, m) = 32 (t / 2) + 8 (m / 4) + 4 (t % 2) + m % 4 of the 8 rows 32 kb + kmap(g, j)
template <int PR>
__device__ __forceinline__ s16x8 tr_operand(const uint16_t* base, int t, int kb, int lane) {
    const int g = lane >> 4, m = lane & 15;
    const int p = 4 * (t >> 1) + (m & 3), r = 32 * kb + 4 * g + (m >> 2);
    const s16x4 a = read_tr(piece_at<PR>(base, r, p) + 4 * (t & 1));
    const s16x4 b = read_tr(piece_at<PR>(base, r + 16, p) + 4 * (t & 1));
    return s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

template <int PR>
__device__ __forceinline__ s16x8 row_operand(const uint16_t* base, int r, int p) {
    return *reinterpret_cast<const s16x8*>(piece_at<PR>(base, r, p));
}

__device__ __forceinline__ f32x4 mma(s16x8 a, s16x8 b, f32x4 c) {
    return mfma16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
}

// 8 floats as a sum of bf16 operands: x = t[0] + t[1] (+ t[2])
template <int TERMS>
__device__ __forceinline__ void split(const float (&x)[8], s16x8 (&t)[TERMS]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
        u32x4 w;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            w[p] = io_pack<0>(r[2 * p], r[2 * p + 1]);
            if (k + 1 < TERMS) {
                r[2 * p] -= io_lo<0>(w[p]);
                r[2 * p + 1] -= io_hi<0>(w[p]);
            }
        }
        t[k] = __builtin_bit_cast(s16x8, w);
    }
}

// rows [0, n) of a 64-row tile with PR pieces a row, straight into LDS by
// `waves` waves; rows past n repeat the last one (finite wherever the row is)
template <int PR>
__device__ __forceinline__ void stage(const uint16_t* src, int64_t stride, int n, int last_piece,
                                      uint16_t* lds, int wave, int waves, int lane) {
    for (int i = wave; i < PR; i += waves) {   // 64 slots of 16 bytes each
        const int q = 64 * i + lane, r = q / PR, p = (q % PR) ^ swz<PR>(r);
        const uint16_t* from = src + (int64_t)min(r, n - 1) * stride + 8 * min(p, last_piece);
        __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void*)(lds + 512 * i),
                                         16, 0, 0);
    }
}

template <int N, int PT, bool kLocal>
struct Smem {
    uint16_t b[64 * N];
    uint16_t c[kLocal ? 8 : 64 * N];
    uint16_t x[kWaves][64 * 16 * PT];
    f32x4 cb[kLocal ? 1 : 10][64];   // (C B^T)^T tiles of the lower triangle, as fragments
    float c2[kWaves][64], d[kWaves][64], w[kWaves][64];
};

__device__ __forceinline__ int tri(int tt, int st) { return tt * (tt + 1) / 2 + st; }

// kLocal: the first pass (states only)
template <int IO, int N, int PT, bool kLocal>
__global__ __launch_bounds__(kThreads) void ssm_scan_kernel(const ScanArgs a) {
    constexpr int NT = N / 16, NKB = N / 32, PR = N / 8, XR = 2 * PT, PW = 16 * PT;
    __shared__ Smem<N, PT, kLocal> sm;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g = lane >> 4, m = lane & 15;
    const gdn_ssm_inputs& in = a.in;

    // work-groups are dealt round-robin to the XCDs: those of one segment and
    // group, which share B and C, get ids of one XCD
    const int total = gridDim.x, per = total / 8, extra = total % 8, xcd = blockIdx.x % 8;
    const int id = xcd * per + min(xcd, extra) + blockIdx.x / 8;
    const int quad = id % a.quads, rest = id / a.quads;
    const int grp = rest % in.groups, row = rest / in.groups;
    Seg s;
    if (!segment(a, row, s) || (kLocal && s.last)) return;
    const int task = quad * kWaves + wave;
    const bool store = task < a.tasks;   // waves past the group's last slice repeat it
    const int tk = min(task, a.tasks - 1);
    const int h = grp * (in.heads / in.groups) + tk / a.slices;
    const int p0 = (tk % a.slices) * PW;
    const int P = in.head_dim, H = in.heads;

    const int bi = a.table ? 0 : s.seq;
    const uint16_t* xp = static_cast<const uint16_t*>(in.x) + bi * in.x_batch + s.t0 * in.x_token + (int64_t)h * P + p0;
    const uint16_t* bp = static_cast<const uint16_t*>(in.b) + bi * in.b_batch + s.t0 * in.b_token + (int64_t)grp * N;
    const uint16_t* cp = static_cast<const uint16_t*>(in.c) + bi * in.c_batch + s.t0 * in.c_token + (int64_t)grp * N;
    const uint16_t* zp = in.z ? static_cast<const uint16_t*>(in.z) + bi * in.z_batch + s.t0 * in.z_token + (int64_t)h * P + p0 : nullptr;
    const size_t dp = (size_t)(bi * in.dt_batch + s.t0 * in.dt_token + h);
    uint16_t* yp = a.y + (((size_t)bi * in.tokens + s.t0) * H + h) * P + p0;
    const int last_piece = (P - p0) / 8 - 1;   // of the head, from p0 on

    // state tiles [nt][pt]: lane (g, m), element i is
    // n = 32 (nt / 2) + 8 g + 4 (nt % 2) + i, p = p0 + perm(pt, m)
    f32x4 S[NT][PT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int pt = 0; pt < PT; ++pt) S[nt][pt] = zero4();
    const size_t hs = ((size_t)s.seq * H + h) * N * P;
    const size_t rec = ((size_t)row * in.groups + grp) * a.tasks + tk;   // state record
    auto n_of = [&](int nt, int i) { return 32 * (nt >> 1) + 8 * g + 4 * (nt & 1) + i; };
    auto p_of = [&](int pt) { return p0 + 32 * (pt >> 1) + 8 * (m >> 2) + 4 * (pt & 1) + (m & 3); };
    if (s.idx == 0) {
        if (a.s0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int pt = 0; pt < PT; ++pt)
                    if (p_of(pt) < P) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) S[nt][pt][i] = a.s0[hs + (size_t)n_of(nt, i) * P + p_of(pt)];
                    }
        }
    } else if (!kLocal) {
        const f32x4* from = a.states + (rec - (size_t)in.groups * a.tasks) * (NT * PT * 64) + lane;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PT; ++pt) S[nt][pt] = from[(nt * PT + pt) * 64];
    }

    const float A2 = -expf(in.A_log[h]) * kLog2e;
    const float bias = in.dt_bias ? in.dt_bias[h] : 0.f;
    const float D = in.D ? in.D[h] : 0.f;
    float log_total = 0.f;   // the segment's base-2 log decay
    float* const c2s = sm.c2[wave];
    float* const dss = sm.d[wave];
    float* const wss = sm.w[wave];
    const uint16_t* const xs = sm.x[wave];

    for (int t0 = 0; t0 < s.n; t0 += kChunk) {
        const int n = min(s.n - t0, kChunk);
        __syncthreads();   // the previous chunk's tiles are read
        stage<PR>(bp + t0 * in.b_token, in.b_token, n, PR, sm.b, wave, kWaves, lane);
        if (!kLocal) stage<PR>(cp + t0 * in.c_token, in.c_token, n, PR, sm.c, wave, kWaves, lane);
        stage<XR>(xp + t0 * in.x_token, in.x_token, n, last_piece, sm.x[wave], 0, 1, lane);

        // token `lane`: step, log decay, its sums from the chunk's start and end
        const size_t di = dp + (size_t)(t0 + min(lane, n - 1)) * in.dt_token;
        const float raw = in.dt_dtype == GDN_DTYPE_FP32 ? io_elem<2>(in.dt, di) : io_elem<IO>(in.dt, di);
        const float dv = lane < n ? ssm_delta(raw, bias, in.dt_min, in.dt_max) : 0.f;
        const float l2 = fmaxf(A2 * dv, -150.f);
        float up = l2, down = l2;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const float u = __shfl_up(up, off, 64), v = __shfl_down(down, off, 64);
            if (lane >= off) up += u;
            if (lane + off < 64) down += v;
        }
        const float after = __shfl_down(down, 1, 64);
        c2s[lane] = up;
        dss[lane] = dv;
        wss[lane] = dv * __builtin_amdgcn_exp2f(lane < 63 ? after : 0.f);
        const float total2 = __shfl(up, 63, 64);
        log_total += total2;
        __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the tiles are in LDS
        __syncthreads();

        if constexpr (!kLocal) {
            // (C B^T)^T: rows s of tile st, columns t of tile tt
            for (int k = wave; k < 10; k += kWaves) {
                const int tt = k < 1 ? 0 : k < 3 ? 1 : k < 6 ? 2 : 3, st = k - tt * (tt + 1) / 2;
                f32x4 acc = zero4();
#pragma unroll
                for (int kb = 0; kb < NKB; ++kb)
                    acc = mma(row_operand<PR>(sm.b, 16 * st + m, 4 * kb + g),
                              row_operand<PR>(sm.c, 16 * tt + m, 4 * kb + g), acc);
                sm.cb[k][lane] = acc;
            }
            // S^T C^T: rows p, columns t
            f32x4 Y[PT][4];
#pragma unroll
            for (int pt = 0; pt < PT; ++pt)
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) Y[pt][tt] = zero4();
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb) {
                s16x8 cop[4];
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) cop[tt] = row_operand<PR>(sm.c, 16 * tt + m, 4 * kb + g);
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[i] = S[2 * kb][pt][i];
                        v[4 + i] = S[2 * kb + 1][pt][i];
                    }
                    s16x8 sop[2];
                    split<2>(v, sop);
#pragma unroll
                    for (int tt = 0; tt < 4; ++tt) {
                        Y[pt][tt] = mma(sop[0], cop[tt], Y[pt][tt]);
                        Y[pt][tt] = mma(sop[1], cop[tt], Y[pt][tt]);
                    }
                }
            }
            float ct[4];
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                ct[tt] = c2s[16 * tt + m];
                const float e = __builtin_amdgcn_exp2f(ct[tt]);
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) Y[pt][tt] *= e;
            }
            __syncthreads();   // C B^T is complete

            // + X^T M^T, M[t][s] = (C B^T) e^{c_t - c_s} d_s for s <= t
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                s16x8 xop[PT];
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) xop[pt] = tr_operand<XR>(xs, pt, kb, lane);
                f32x4 cs[2], ds[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    cs[q] = *reinterpret_cast<const f32x4*>(c2s + 32 * kb + 16 * q + 4 * g);
                    ds[q] = *reinterpret_cast<const f32x4*>(dss + 32 * kb + 16 * q + 4 * g);
                }
#pragma unroll
                for (int tt = 2 * kb; tt < 4; ++tt) {
                    float v[8];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int st = 2 * kb + q;
                        if (st > tt) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[4 * q + i] = 0.f;
                            continue;
                        }
                        const f32x4 cb = sm.cb[tri(tt, st)][lane];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float e = cb[i] * __builtin_amdgcn_exp2f(ct[tt] - cs[q][i]) * ds[q][i];
                            v[4 * q + i] = st < tt || 4 * g + i <= m ? e : 0.f;
                        }
                    }
                    s16x8 mop[2];
                    split<2>(v, mop);
#pragma unroll
                    for (int pt = 0; pt < PT; ++pt) {
                        Y[pt][tt] = mma(xop[pt], mop[0], Y[pt][tt]);
                        Y[pt][tt] = mma(xop[pt], mop[1], Y[pt][tt]);
                    }
                }
            }
            // + D x, the gate, out: 8 channels of one token a lane
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                const int t = 16 * tt + m;
#pragma unroll
                for (int q = 0; q < PT / 2; ++q) {
                    const int p = 32 * q + 8 * g;   // from p0
                    if (!store || t >= n || p0 + p >= P) continue;
                    const u32x4 xr = __builtin_bit_cast(u32x4, row_operand<XR>(xs, t, 4 * q + g));
                    u32x4 zr = {0, 0, 0, 0};
                    if (zp) zr = *reinterpret_cast<const u32x4*>(zp + (int64_t)(t0 + t) * in.z_token + p);
                    u32x4 o;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const f32x4& yv = Y[2 * q + (k >> 1)][tt];
                        float u = yv[2 * (k & 1)] + D * io_lo<IO>(xr[k]);
                        float v = yv[2 * (k & 1) + 1] + D * io_hi<IO>(xr[k]);
                        if (zp) {
                            u *= silu_fast(io_lo<IO>(zr[k]));
                            v *= silu_fast(io_hi<IO>(zr[k]));
                        }
                        o[k] = io_pack<IO>(u, v);
                    }
                    *reinterpret_cast<u32x4*>(yp + (size_t)(t0 + t) * H * P + p) = o;
                }
            }
        }

        // S <- e^{c_Q} S + B^T (w x)
        const float dec = __builtin_amdgcn_exp2f(total2);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PT; ++pt) S[nt][pt] *= dec;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            s16x8 wx[PT][3];
            const f32x4 w0 = *reinterpret_cast<const f32x4*>(wss + 32 * kb + 4 * g);
            const f32x4 w1 = *reinterpret_cast<const f32x4*>(wss + 32 * kb + 16 + 4 * g);
#pragma unroll
            for (int pt = 0; pt < PT; ++pt) {
                const u32x4 xr = __builtin_bit_cast(u32x4, tr_operand<XR>(xs, pt, kb, lane));
                float v[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x4& w = k < 2 ? w0 : w1;
                    v[2 * k] = io_lo<IO>(xr[k]) * w[2 * (k & 1)];
                    v[2 * k + 1] = io_hi<IO>(xr[k]) * w[2 * (k & 1) + 1];
                }
                split<3>(v, wx[pt]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const s16x8 bop = tr_operand<PR>(sm.b, nt, kb, lane);
#pragma unroll
                for (int k = 2; k >= 0; --k)   // the smallest parts first
#pragma unroll
                    for (int pt = 0; pt < PT; ++pt) S[nt][pt] = mma(bop, wx[pt][k], S[nt][pt]);
            }
        }
    }

    if (!store) return;
    if (kLocal) {
        f32x4* to = a.states + rec * (NT * PT * 64) + lane;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PT; ++pt) to[(nt * PT + pt) * 64] = S[nt][pt];
        if (lane == 0) a.decays[rec] = __builtin_amdgcn_exp2f(log_total);
    } else if (s.last) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PT; ++pt)
                if (p_of(pt) < P) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) a.sf[hs + (size_t)n_of(nt, i) * P + p_of(pt)] = S[nt][pt][i];
                }
    }
}

// The states behind segments 1, 2, .. of a sequence from its segments' own:
// R_j = decay_j R_{j-1} + L_j in place, elementwise (fragment order)
__global__ __launch_bounds__(kThreads) void ssm_join_kernel(const ScanArgs a, int elems, int parts) {
    const int id = blockIdx.x;
    const int part = id % parts, task = id / parts % (a.in.groups * a.tasks), row0 = id / parts / (a.in.groups * a.tasks);
    int row = a.table ? row0 : row0 * a.segs;
    Seg s;
    if (!segment(a, row, s) || s.idx != 0 || s.last) return;
    const int e = part * kThreads + threadIdx.x;
    if (e >= elems) return;
    const size_t all = (size_t)a.in.groups * a.tasks;
    f32x4 R = a.states[((size_t)row * all + task) * elems + e];
    const int seq = s.seq;
    while (++row < a.rows && segment(a, row, s) && s.seq == seq && !s.last) {
        f32x4* at = a.states + ((size_t)row * all + task) * elems + e;
        R = R * a.decays[(size_t)row * all + task] + *at;
        *at = R;
    }
}

// blocks from cu_seqlens (clamped values), for callers without a table: one
// group forms the sequences' first rows, the rows are found by search
constexpr int kTableSeqs = 4096;

__device__ __forceinline__ int seq_rows(const int32_t* cu, int total, int s, int block) {
    const int n = seq_count(cu, 0, total, s);
    return max(1, n / block + (n % block != 0));
}

// First row of each sequence, start[0 .. seqs], saturating at `rows`
template <int NT>
__device__ void table_starts(const int32_t* cu, int seqs, int total, int block, int rows, int* start,
                             int* red) {
    int base = 0;
    if (threadIdx.x == 0) start[0] = 0;
    for (int s0 = 0; s0 < seqs; s0 += NT) {
        const int s = s0 + threadIdx.x;
        int v = s < seqs ? min(seq_rows(cu, total, s, block), rows) : 0;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int u = __shfl_up(v, off, 64);
            if (lane >= off) v = min(v + u, rows);
        }
        __syncthreads();
        if (lane == 63) red[wave] = v;
        __syncthreads();
        int sum = base;
        for (int w = 0; w < NT / 64; ++w) {
            if (w == wave) v = min(v + sum, rows);
            sum = min(sum + red[w], rows);
        }
        if (s < seqs) start[s + 1] = v;
        base = sum;
    }
    __syncthreads();
}

__device__ __forceinline__ void table_rows(const int32_t* cu, const int* start, int seqs, int total,
                                           int block, int rows, int4* table) {
    for (int r = blockIdx.x * kThreads + threadIdx.x; r < rows; r += gridDim.x * kThreads) {
        int lo = 0, hi = seqs;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (start[mid + 1] > r) hi = mid;
            else lo = mid + 1;
        }
        int4 v = make_int4(-1, 0, 0, 0);
        if (lo < seqs) {
            const int idx = r - start[lo], t0 = seq_lo(cu, 0, total, lo) + idx * block;
            v = make_int4(lo, t0, min(seq_count(cu, 0, total, lo) - idx * block, block), idx);
        }
        table[r] = v;
    }
}

__global__ __launch_bounds__(kThreads) void ssm_table_kernel(const int32_t* __restrict__ cu, int seqs,
                                                             int total, int block, int rows,
                                                             int4* __restrict__ table) {
    __shared__ int start[kTableSeqs + 1], red[kWaves];
    table_starts<kThreads>(cu, seqs, total, block, rows, start, red);
    table_rows(cu, start, seqs, total, block, rows, table);
}

__global__ __launch_bounds__(1024) void ssm_starts_kernel(const int32_t* __restrict__ cu, int seqs,
                                                          int total, int block, int rows,
                                                          int* __restrict__ start) {
    __shared__ int red[16];
    table_starts<1024>(cu, seqs, total, block, rows, start, red);
}

__global__ __launch_bounds__(kThreads) void ssm_rows_kernel(const int32_t* __restrict__ cu,
                                                            const int* __restrict__ start, int seqs,
                                                            int total, int block, int rows,
                                                            int4* __restrict__ table) {
    table_rows(cu, start, seqs, total, block, rows, table);
}

bool scan_sizes_ok(const gdn_ssm_inputs* in, int seqs, int block, bool packed) {
    return ssm_sizes_ok(in) && seqs >= 1 && seqs <= (1 << 24) && in->tokens <= (1 << 30) &&
           block >= kChunk && block <= kMaxBlock && block % kChunk == 0 &&
           (packed ? in->batch == 1 : seqs == in->batch);
}

// Whether the chunked scan has an instance; the rest takes the recurrence
bool chunked(const gdn_ssm_inputs* in) {
    return in->io_dtype == GDN_DTYPE_BF16 && in->state_dim >= 64;
}

int cols_of(const gdn_ssm_inputs* in) { return in->state_dim == 256 ? 32 : 64; }

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct Layout {
    int segs;        // segments of a batch row (0: packed)
    int64_t rows;
    int slices, tasks, quads;
    size_t table, starts, states, decays, total;   // byte offsets

    Layout(const gdn_ssm_inputs* in, int seqs, int block, bool packed) {
        segs = packed ? 0 : std::max(1, (in->tokens + block - 1) / block);
        rows = packed ? (int64_t)in->tokens / block + seqs : (int64_t)segs * seqs;
        const int pw = cols_of(in);
        slices = (in->head_dim + pw - 1) / pw;
        tasks = in->heads / in->groups * slices;
        quads = (tasks + kWaves - 1) / kWaves;
        size_t off = 0;
        table = off;
        if (packed) off += align256((size_t)rows * 16);
        starts = off;
        if (packed) off += align256(((size_t)seqs + 1) * 4);
        // no states where every sequence is one segment
        const size_t recs = packed || segs > 1 ? (size_t)rows * in->groups * tasks : 0;
        states = off;
        off += align256(recs * in->state_dim * pw * 4);
        decays = off;
        off += align256(recs * 4);
        total = std::max<size_t>(off, 256);
    }
};

template <int IO, int N, int PT>
hipError_t launch_scan(const ScanArgs& a, hipStream_t stream) {
    const int64_t groups = (int64_t)a.rows * a.in.groups * a.quads;
    if (groups > 0x7fffffff) return hipErrorInvalidValue;
    if (a.table || a.segs > 1) {
        hipLaunchKernelGGL((ssm_scan_kernel<IO, N, PT, true>), dim3((unsigned)groups),
                           dim3(kThreads), 0, stream, a);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        if (a.table || a.segs > 2) {
            const int elems = N * PT * 4, parts = (elems + kThreads - 1) / kThreads;
            const int64_t join = (int64_t)(a.table ? a.rows : a.seqs) * a.in.groups * a.tasks * parts;
            if (join > 0x7fffffff) return hipErrorInvalidValue;
            hipLaunchKernelGGL(ssm_join_kernel, dim3((unsigned)join), dim3(kThreads), 0, stream, a,
                               elems, parts);
            if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
    }
    hipLaunchKernelGGL((ssm_scan_kernel<IO, N, PT, false>), dim3((unsigned)groups), dim3(kThreads), 0,
                       stream, a);
    return hipGetLastError();
}

template <int IO>
hipError_t launch_any(const ScanArgs& a, hipStream_t stream) {
    switch (a.in.state_dim) {
        case 64: return launch_scan<IO, 64, 4>(a, stream);
        case 128: return launch_scan<IO, 128, 4>(a, stream);
        default: return launch_scan<IO, 256, 2>(a, stream);
    }
}

hipError_t form_table(const int32_t* cu, int seqs, int total, int block, int rows, int4* table,
                      int* starts, hipStream_t stream) {
    const unsigned grid = (unsigned)std::min((rows + kThreads - 1) / kThreads, 1024);
    if (seqs <= kTableSeqs) {
        hipLaunchKernelGGL(ssm_table_kernel, dim3(grid), dim3(kThreads), 0, stream, cu, seqs, total,
                           block, rows, table);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(ssm_starts_kernel, dim3(1), dim3(1024), 0, stream, cu, seqs, total, block,
                       rows, starts);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    hipLaunchKernelGGL(ssm_rows_kernel, dim3(grid), dim3(kThreads), 0, stream, cu, starts, seqs,
                       total, block, rows, table);
    return hipGetLastError();
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_ssm_scan_block(const gdn_ssm_inputs* in, int num_seqs) {
    if (!ssm_sizes_ok(in) || num_seqs < 1 || in->tokens > (1 << 30)) return 0;
    // about two waves per SIMD of a 256-CU chip
    const int pw = cols_of(in);
    const int64_t slices = (int64_t)in->heads * ((in->head_dim + pw - 1) / pw);
    const int64_t tokens = (int64_t)in->batch * in->tokens;
    const int64_t want = std::max<int64_t>(1, 2048 / slices);
    const int64_t block = (tokens + want * kChunk - 1) / (want * kChunk) * kChunk;
    return (int)std::min<int64_t>(std::max<int64_t>(block, kChunk), kMaxBlock);
}

extern "C" size_t gdn_ssm_scan_workspace_size(const gdn_ssm_inputs* in, int num_seqs, int block,
                                              int packed) {
    if (!scan_sizes_ok(in, num_seqs, block, packed != 0)) return 0;
    const Layout l(in, num_seqs, block, packed != 0);
    return l.rows <= 0x7fffffff ? l.total : 0;
}

extern "C" hipError_t gdn_ssm_scan(const gdn_ssm_inputs* in, void* y, const float* s0, float* sf,
                                   const int32_t* cu_seqlens, const int32_t* blocks, int num_seqs,
                                   int block, void* workspace, size_t workspace_bytes,
                                   hipStream_t stream) {
    const bool packed = cu_seqlens != nullptr;
    if (!ssm_inputs_ok(in) || !scan_sizes_ok(in, num_seqs, block, packed) || (blocks && !packed))
        return hipErrorInvalidValue;
    if (!sf || !ssm_aligned(sf, 4) || !ssm_aligned(s0, 4) || (in->tokens > 0 && !y) ||
        !ssm_aligned(y, 16) || !ssm_aligned(workspace, 256) || !ssm_aligned(blocks, 16))
        return hipErrorInvalidValue;
    const size_t need = gdn_ssm_scan_workspace_size(in, num_seqs, block, packed);
    if (need == 0 || !workspace || workspace_bytes < need) return hipErrorInvalidValue;
    if (!chunked(in)) return ssm_recurrent(*in, y, s0, sf, cu_seqlens, num_seqs, stream);
    const Layout l(in, num_seqs, block, packed);
    char* ws = static_cast<char*>(workspace);
    ScanArgs a{};
    a.in = *in;
    a.y = static_cast<uint16_t*>(y);
    a.s0 = s0;
    a.sf = sf;
    a.rows = (int)l.rows;
    a.segs = l.segs;
    a.seqs = num_seqs;
    a.block = block;
    a.slices = l.slices;
    a.tasks = l.tasks;
    a.quads = l.quads;
    a.states = reinterpret_cast<f32x4*>(ws + l.states);
    a.decays = reinterpret_cast<float*>(ws + l.decays);
    if (packed) {
        a.table = reinterpret_cast<const int4*>(blocks);
        if (!blocks) {
            auto table = reinterpret_cast<int4*>(ws + l.table);
            if (const hipError_t e = form_table(cu_seqlens, num_seqs, in->tokens, block, a.rows, table,
                                                reinterpret_cast<int*>(ws + l.starts), stream);
                e != hipSuccess)
                return e;
            a.table = table;
        }
    }
    return launch_any<0>(a, stream);
}
