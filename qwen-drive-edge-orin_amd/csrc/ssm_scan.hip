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
// of the segments, and the main pass starts each segment from its own.  A call
// that no sequence of which can be split runs the main pass alone (a packed one
// where all its tokens fit in a block: the lengths are on the GPU).  Only
// segments with another behind them have a record: 1500 requests, nearly all
// single tokens, x 64 heads take 4 MB of workspace, not 3 GB.
//
// A wave owns 32 columns of one head: its slice of S stays in fp32 accumulators
// through the segment, and the columns need nothing from one another.  Four
// waves of one group share B, C and the products C B^T in LDS, 80 KB a
// work-group (state 128), so that two groups fit a CU and their 2 waves a SIMD
// cover each other's waits; 64 columns a wave would save a fifth of the vector
// work (M is formed once per wave) but hold 128 registers of S more and leave
// one wave a SIMD (measured at an early stage: 693 us against 398 for the
// packed call below).  The next chunk's tiles go into LDS while the present
// one is worked on.
// The MFMA operand and result layouts (gdn_common.h) chain without shuffles:
// S's tiles are the A operand of S^T C^T, C B^T comes out transposed as the B
// operand of X^T M^T, and rows are numbered so that two result tiles hold 8
// consecutive channels (perm below), 16 bytes of y.
//
// Measured (state 128): 8 packed prompts, 19,861 tokens x 64 heads of 64 with
// the gate: a call of 303 us, 2.0 TB/s of what must move; traced, where kernels
// do not run into one another, main pass 225, first pass 65, join 16, table 5.
// 16,384 tokens x 16 heads 78 us, 1141 x 64 38 us.  No unit is at its limit in
// the main pass: the SIMDs issue vector instructions 52 % of the time and the
// MFMA units are busy 27 % (0.6 PFLOP/s).  A wave runs in order and there are
// two a SIMD: of a wave's time 43 % is its own issue, 34 % the other's turn and
// 23 % a wait for memory, LDS or the barrier.  A wave's chunk takes 1,600 vector
// instructions, 216 of them MFMA, the rest the splits of operands into parts,
// M's exponentials (M is formed once per 32 columns, by each wave of a head) and
// the gate.  Measured without gain: waves' priorities raised in the MFMA or the
// vector phases, update and M interleaved by quarters of the chunk (spills),
// 8-wave groups, operand residuals by dot products.
//
// Rounding.  bf16: x, B and C are exact operands.  M = (C B^T) o decay, which
// carries D and the newest tokens, the largest terms of y, and d x, which enters
// the state, go into products as three bf16 (fp32's 24 bits).  S enters y's
// product as two, 2^-18 of each term, where C has 2^-9 already: M as two put
// 1.2e-4 of y (its norm) on the other side of a bf16 border than fp32 does, as
// three 2.2e-5 for 2 to 3 % of a call; S as three left that as it was for 4 to
// 6 % more.  fp16: pairs of fp16 (22 bits) behind powers of two, one for each
// column of S and of w x, so that what is off is relative to a column's own
// largest value, and one for M, off by 2^-40 of the chunk's largest
// |C . B| d (y itself: 2^-11).  Sums, states, decays: fp32.  Logarithms are
// summed in fp32, backwards for the state's weights, so that those of the
// newest tokens, the largest, are sums of few terms, and forwards within 16
// tokens for M, in two parts, so that differences of two sums are as exact as
// the shorter sum; a token's base-2 logarithm is held at -150, where its decay
// is 0 in fp32, to keep those sums small.
//
// Not finite.  A product sums over the zeros of M too, and 0 x infinity would
// reach tokens in front, so x that is not finite is 0 in the products and its
// channel NaN from its token on.  4 MFMAs on zeros and a ballot find it, 0 to
// 2 % of a call.  fp16's scales come from what is finite.
#include "gdn_seq.h"
#include "gdn_ssm.h"

#include <algorithm>
#include <cmath>

namespace gdn {
namespace {

constexpr int kMaxBlock = 1 << 20;
// Segments of a fixed-length sequence that the main pass joins by itself: each
// group reads the records in front of its own, which is less than a launch of
// the join up to here (1141 tokens x 64 heads in 6 segments: 38 us against 41;
// 4 x 2048 tokens x 32 in 8: 85 against 83)
constexpr int kMaxFold = 6;
// Work-groups of a packed call up to which the main pass takes the longest
// segments first (8 rounds of 512: what the last round wastes still counts
// against a group's one more trip to memory; 30 prompts of 50 to 2000 tokens x
// 64 heads 346 us against 371 in the table's order)
constexpr int kMaxOrder = 4096;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kTiles = 2;          // 16-column tiles of a wave
constexpr int kCols = 16 * kTiles;
constexpr float kLog2e = 1.4426950408889634f;

struct Seg {
    int seq, t0, n, idx;
    int rec;      // its record's place (the last of a sequence has none); the one in front is rec - 1
    bool last;
};

struct ScanArgs {
    gdn_ssm_inputs in;
    uint16_t* y;
    const float* s0;
    float* sf;
    const int4* table;   // packed: blocks; null: `segs` segments of `block` tokens per batch row
    int rows;            // segments (bound)
    int recs;            // records: segments that are not the last of their sequence (bound)
    int segs, seqs, block;
    int slices;          // column slices of a head: ceil(P / PW)
    int tasks;           // slices of a group: heads / groups x slices
    bool fold;           // the main pass joins the segments' states itself
    int quads;           // work-groups per group and segment: ceil(tasks / waves)
    int* order;          // the main pass's rows, longest first; null: as they lie
    f32x4* states;       // [record][group][task] fragments of a slice's state
    float* decays;       // [record][group][task]
};

// Segment r, clamped so that whatever a table holds its tokens lie in the row
__device__ __forceinline__ bool segment(const ScanArgs& a, int r, Seg& s) {
    if (!a.table) {
        s.seq = r / a.segs;
        s.idx = r - s.seq * a.segs;
        s.t0 = s.idx * a.block;
        s.n = min(a.block, a.in.tokens - s.t0);
        s.rec = s.seq * (a.segs - 1) + s.idx;
        s.last = s.idx + 1 == a.segs;
        return true;
    }
    // Records of packed segments lie at first token / block: a segment that is
    // not its sequence's last is `block` tokens long, and no two overlap.
    const int4 b = a.table[r];
    if (b.x < 0 || b.x >= a.seqs) return false;
    s.seq = b.x;
    s.t0 = min(max(b.y, 0), a.in.tokens);
    s.n = min(min(max(b.z, 0), a.block), a.in.tokens - s.t0);
    s.rec = min(s.t0 / a.block, a.recs);
    s.idx = s.rec > 0 ? max(b.w, 0) : 0;
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

typedef int i32x4 __attribute__((ext_vector_type(4)));
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

// x that is not finite becomes 0 in a 64-row tile of 32 columns.  Lane's column
// (lane % 32): the first row that had one, or 64.
template <int IO, int PR>
__device__ __forceinline__ int clear_not_finite(uint16_t* tile, int lane) {
    static_assert(PR == 4, "32 columns, half of the rows a lane");
    constexpr int kExp = IO == 0 ? 0x7f80 : 0x7c00;
    int first = 64;
#pragma unroll 1
    for (int i = 31; i >= 0; --i) {
        const int r = (lane & 32) + i;
        uint16_t* at = const_cast<uint16_t*>(piece_at<PR>(tile, r, (lane & 31) / 8)) + lane % 8;
        if ((*at & kExp) == kExp) {
            first = r;
            *at = 0;
        }
    }
    return min(first, __shfl_xor(first, 32, 64));
}

template <int IO>
__device__ __forceinline__ f32x4 mma(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (IO == 0) return mfma16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
    else return mfma16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c);
}

// 8 floats as a sum of 16-bit operands: x = t[0] + t[1] (+ t[2])
template <int IO, int TERMS>
__device__ __forceinline__ void split(const float (&x)[8], s16x8 (&t)[TERMS]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
        u32x4 w;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            w[p] = io_pack<IO>(r[2 * p], r[2 * p + 1]);
            if (k + 1 < TERMS) {
                r[2 * p] -= io_lo<IO>(w[p]);
                r[2 * p + 1] -= io_hi<IO>(w[p]);
            }
        }
        t[k] = __builtin_bit_cast(s16x8, w);
    }
}

// A 64-row tile with PR pieces a row on its way into LDS, 64 slots of 16 bytes
// per load, loads wave, wave + WAVES, ..; rows past n repeat the last one
// (finite wherever the row is)
//
// The load is asm because the compiler, which cannot tell the tiles apart,
// would wait for it before the next access to any of them, and these are
// prefetches: who reads a tile waits for vmcnt(0) and a barrier first.  It has
// no output register, and to the compiler's own waits it is one more
// operation in flight, which can only make them longer.
template <int PR, int WAVES>
struct Stager {
    static constexpr int kRows = 64 * WAVES / PR;   // rows between a wave's loads
    const char* base;      // the next chunk's first row
    uint32_t row;          // bytes from row to row (below 2^25)
    uint32_t at;           // byte offset of this lane's piece of its first row
    int last_piece;
    uint32_t lds;          // byte address of load 0's slots

    __device__ __forceinline__ int piece(int r, int lane) const { return min((lane % PR) ^ swz<PR>(r), last_piece); }

    __device__ __forceinline__ void init(const uint16_t* src, int64_t stride, int last_piece_,
                                         const uint16_t* tile, int wave, int lane) {
        base = reinterpret_cast<const char*>(src);
        row = 2 * (uint32_t)stride;
        last_piece = last_piece_;
        const int r0 = (64 * wave + lane) / PR;
        at = row * r0 + 16 * piece(r0, lane);
        lds = __builtin_amdgcn_readfirstlane(
            (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint16_t*)(tile + 512 * wave));
    }
    __device__ __forceinline__ static void send(const char* from, uint32_t off, uint32_t to) {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                     :: "v"(off), "s"(from), "s"(to) : "memory", "m0");
    }
    // the next chunk's n rows, `offset` bytes into the tile
    __device__ __forceinline__ void load(int n, uint32_t offset, int wave, int lane) {
        constexpr bool kOneSwizzle = kRows % 16 == 0 || PR <= 4;   // for all rows of a lane
        if (kOneSwizzle && n == kChunk) {
            const char* from = base;
#pragma unroll
            for (int j = 0; j < PR / WAVES; ++j) {
                send(from, at, lds + offset + 1024 * WAVES * j);
                from += kRows * row;
            }
        } else {
            const int r0 = (64 * wave + lane) / PR;
#pragma unroll
            for (int j = 0; j < PR / WAVES; ++j) {
                const int r = r0 + kRows * j;
                send(base, row * min(r, n - 1) + 16 * piece(r, lane), lds + offset + 1024 * WAVES * j);
            }
        }
        base += kChunk * (uint64_t)row;
    }
};

// Inclusive sums within a row of 16 lanes: over the lanes up to this one
__device__ __forceinline__ float row_prefix(float x) {
#define GDN_DPP(ctrl)                                                                             \
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(                                   \
                                       0, __builtin_bit_cast(int, x), ctrl, 0xf, 0xf, false))
    GDN_DPP(0x111);   // row_shr:1
    GDN_DPP(0x112);
    GDN_DPP(0x114);
    GDN_DPP(0x118);
    return x;
}

// and over this one and the lanes behind it
__device__ __forceinline__ float row_suffix(float x) {
    GDN_DPP(0x101);   // row_shl:1
    GDN_DPP(0x102);
    GDN_DPP(0x104);
    GDN_DPP(0x108);
#undef GDN_DPP
    return x;
}

// x of the next lane of the row, 0 for its last
__device__ __forceinline__ float row_next(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x101, 0xf, 0xf, false));
}

// The largest of non-negative x over the wave
__device__ __forceinline__ float wave_max(float x) {
#define GDN_DPP(ctrl, rows)                                                                       \
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(                           \
                                               __builtin_bit_cast(int, x),                        \
                                               __builtin_bit_cast(int, x), ctrl, rows, 0xf, false)))
    GDN_DPP(0x111, 0xf);
    GDN_DPP(0x112, 0xf);
    GDN_DPP(0x114, 0xf);
    GDN_DPP(0x118, 0xf);
    GDN_DPP(0x142, 0xa);
    GDN_DPP(0x143, 0xc);
#undef GDN_DPP
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// x, or NaN for an infinity: the maxima that scales come from do not see NaN
__device__ __forceinline__ float finite_or_nan(float x) { return fmaf(x, 0.f, x); }

// Two non-negative floats' upper halves in one word, x low (what fit_fp16 looks at)
__device__ __forceinline__ uint32_t pack_tops(float x, float y) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302);
}

// Their maxima over the four lanes of a column (m, m + 16, m + 32 and m + 48)
__device__ __forceinline__ uint32_t column_max(uint32_t v) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int off = 16; off < 64; off <<= 1)
        v = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(
                                             __builtin_bit_cast(u16x2, v),
                                             __builtin_bit_cast(u16x2, (uint32_t)__shfl_xor((int)v, off, 64))));
    return v;
}

__device__ __forceinline__ float top_of(uint32_t v, int i) {
    return __builtin_bit_cast(float, i == 0 ? v << 16 : v & 0xffff0000u);
}

// k that brings x >= 0 into [2^14, 2^15), fp16's top binade but one; within
// +-100, so that 2^k and a few sums of such k stay inside fp32's exponents
__device__ __forceinline__ int fit_fp16(float x) {
    const int e = (int)(__builtin_bit_cast(uint32_t, x) >> 23) - 127;
    return min(max(14 - e, -100), 100);
}

__device__ __forceinline__ float pow2(int k) {   // -126 <= k <= 127
    return __builtin_bit_cast(float, (uint32_t)(k + 127) << 23);
}

template <int N, int PT, int WAVES, bool kLocal>
struct Smem {
    uint16_t b[2][64 * N];           // this chunk's and the next one's
    uint16_t c[kLocal ? 8 : 64 * N];
    uint16_t x[WAVES][64 * 16 * PT];
    f32x4 cb[kLocal ? 1 : 10][64];   // (C B^T)^T tiles of the lower triangle, as fragments
    // per token of the chunk, for each wave's head: the weight in S; the sum of
    // the log decays of its 16 up to it, r in steps of 2^-8 and q the rest; the
    // step d; d times the decay up to the end of its 16
    static constexpr int kTok = kLocal ? 4 : 64;
    struct {
        float w[64], r[kTok], q[kTok], d[kTok], f[kTok];
        int k[kLocal ? 4 : 16 * PT];   // fp16: the power of two on each column of S^T C^T
        uint16_t first[kLocal ? 8 : 16 * PT];   // each column's first token whose x is not finite
    } tok[WAVES];
    alignas(16) float cb_top[WAVES];   // fp16: the largest of C B^T's column tile of each wave
};

__device__ __forceinline__ constexpr int tri(int tt, int st) { return tt * (tt + 1) / 2 + st; }

// Row r's place in the main pass, by a whole group: the longest segments first,
// so that what ends last is short.  Places are unique whatever the table holds.
__device__ __forceinline__ void order_row(const ScanArgs& a, int r) {
    __shared__ int count[kWaves];
    const int n = a.table[r].z;
    int before = 0;
    for (int j = threadIdx.x; j < a.rows; j += kThreads) {
        const int m = a.table[j].z;
        before += m > n || (m == n && j < r);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) before += __shfl_xor(before, off, 64);
    if ((threadIdx.x & 63) == 0) count[threadIdx.x >> 6] = before;
    __syncthreads();
    if (threadIdx.x == 0) a.order[count[0] + count[1] + count[2] + count[3]] = r;
}

// kLocal: the first pass (states only)
template <int IO, int N, int PT, int WAVES, bool kLocal>
__global__ __launch_bounds__(64 * WAVES, N > 128 ? 1 : 2) void ssm_scan_kernel(const ScanArgs a) {
    constexpr int NT = N / 16, NKB = N / 32, PR = N / 8, XR = 2 * PT, PW = 16 * PT;
    constexpr int kParts = IO == 0 ? 3 : 2;   // of w x and M: 24 or 22 bits
    __shared__ Smem<N, PT, WAVES, kLocal> sm;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, m = lane & 15;
    const gdn_ssm_inputs& in = a.in;

    // Work-groups are dealt round-robin to the 8 XCDs.  The quads of a segment
    // and group, which share B and C, are consecutive on one XCD; the segments
    // are dealt over all of them, so that short ones even out.
    const int xcd = blockIdx.x % 8, nth = blockIdx.x / 8;
    const int quad = nth % a.quads, unit = nth / a.quads * 8 + xcd;
    const int grp = unit % in.groups;
    int row = unit / in.groups;
    if (a.order && row < a.rows) {
        if (!kLocal) row = a.order[row];
        else if (grp == 0 && quad == 0) order_row(a, row);
    }
    Seg s;
    if (row >= a.rows || !segment(a, row, s) || (kLocal && (s.last || s.rec >= a.recs))) return;
    const int task = quad * WAVES + wave;
    const bool store = task < a.tasks;   // waves past the group's last slice repeat it
    const int tk = min(task, a.tasks - 1);
    const int h = grp * (in.heads / in.groups) + tk / a.slices;
    const int p0 = (tk % a.slices) * PW;
    const int P = in.head_dim, H = in.heads;
    auto& tok = sm.tok[wave];

    const int bi = a.table ? 0 : s.seq;
    const uint16_t* xp = static_cast<const uint16_t*>(in.x) + bi * in.x_batch + s.t0 * in.x_token + (int64_t)h * P + p0;
    const uint16_t* bp = static_cast<const uint16_t*>(in.b) + bi * in.b_batch + s.t0 * in.b_token + (int64_t)grp * N;
    const uint16_t* cp = static_cast<const uint16_t*>(in.c) + bi * in.c_batch + s.t0 * in.c_token + (int64_t)grp * N;
    const int last_piece = (P - p0) / 8 - 1;   // of the head, from p0 on
    // the chunk's first row of z, y and dt, and byte offsets of this lane's
    // values from there (row strides are below 2^24)
    const uint16_t* zp = in.z ? static_cast<const uint16_t*>(in.z) + bi * in.z_batch + s.t0 * in.z_token + (int64_t)h * P + p0 : nullptr;
    const bool gate = in.z != nullptr;
    const uint32_t zrow = 2 * (uint32_t)in.z_token, z0 = 16 * min(g, last_piece), zm = m * zrow + z0;
    const uint32_t yrow = 2 * (uint32_t)(H * P), ym = m * yrow + 16 * g;
    char* yp = reinterpret_cast<char*>(a.y + ((int64_t)bi * in.tokens + s.t0) * H * P + (int64_t)h * P + p0);
    const uint32_t dt_size = in.dt_dtype == GDN_DTYPE_FP32 ? 4 : 2, dt_row = (uint32_t)in.dt_token * dt_size;
    const char* dtp = static_cast<const char*>(in.dt) + (bi * in.dt_batch + s.t0 * in.dt_token + h) * dt_size;
    auto load_dt = [&](int n) {   // of the next chunk's token `lane`, or of its last
        const char* at = dtp + (uint32_t)min(lane, n - 1) * dt_row;
        dtp += kChunk * (uint64_t)dt_row;
        return dt_size == 4 ? *reinterpret_cast<const float*>(at) : io_elem<IO>(at, 0);
    };
    Stager<PR, WAVES> bst, cst;
    Stager<XR, 1> xst;
    bst.init(bp, in.b_token, PR, sm.b[0], wave, lane);
    if (!kLocal) cst.init(cp, in.c_token, PR, sm.c, wave, lane);
    xst.init(xp, in.x_token, last_piece, sm.x[wave], 0, lane);
    float raw_dt = 0.f;
    if (s.n > 0) {
        const int n = min(s.n, kChunk);
        raw_dt = load_dt(n);
        bst.load(n, 0, wave, lane);
        if (!kLocal) cst.load(n, 0, wave, lane);
        xst.load(n, 0, 0, lane);
    }

    // state tiles [nt][pt]: lane (g, m), element i is
    // n = 32 (nt / 2) + 8 g + 4 (nt % 2) + i, p = p0 + perm(pt, m)
    f32x4 S[NT][PT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int pt = 0; pt < PT; ++pt) S[nt][pt] = zero4();
    const size_t hs = ((size_t)s.seq * H + h) * N * P;
    const int64_t rec = ((int64_t)s.rec * in.groups + grp) * a.tasks + tk;   // state record
    // element (nt, pt, i) of a lane in a state [N][P]: so + n_off(nt, i) P + p_off(pt)
    const size_t so = hs + (size_t)(8 * g) * P + p0 + 8 * (m >> 2) + (m & 3);
    auto n_off = [](int nt, int i) { return 32 * (nt >> 1) + 4 * (nt & 1) + i; };
    auto p_off = [](int pt) { return 32 * (pt >> 1) + 4 * (pt & 1); };
    const int p_lane = p0 + 8 * (m >> 2) + (m & 3);
    if (s.idx == 0) {
        if (a.s0) {
            const float* from = a.s0 + so;
#pragma unroll
            for (int pt = 0; pt < PT; ++pt)
                if (p_lane + p_off(pt) < P) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) S[nt][pt][i] = from[n_off(nt, i) * P + p_off(pt)];
                }
        }
    } else if (!kLocal) {
        // the record of the segment in front, joined already, or (few segments)
        // the segments' own, joined here
        const int64_t all = (int64_t)in.groups * a.tasks;
        const int count = a.fold ? min(s.idx, kMaxFold - 1) : 1;
        for (int k = count; k > 0; --k) {
            const f32x4* from = a.states + (rec - k * all) * (NT * PT * 64) + lane;
            const float decay = k < count ? a.decays[rec - k * all] : 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) {
                    const f32x4 L = from[(nt * PT + pt) * 64];
                    S[nt][pt] = k < count ? S[nt][pt] * decay + L : L;
                }
        }
    }

    const float A2 = -expf(in.A_log[h]) * kLog2e;
    const float bias = in.dt_bias ? in.dt_bias[h] : 0.f;
    const float D = in.D ? in.D[h] : 0.f;
    float log_total = 0.f;   // the segment's base-2 log decay

    // fp16: what enters an MFMA is scaled by a power of two first, so that
    // neither large nor small values leave the five exponent bits.  The state
    // and w x have one for each column, so that a small channel next to a large
    // one keeps its bits: the accumulators S hold 2^kappa times the state.
    int kappa[PT];
    float d_max = 0.f;
    static_assert(PT == 2, "a word holds the maxima of a lane's columns, lane 16 pt + m keeps column m of tile pt");
    auto column_tops = [&] {   // of S
        float top[PT] = {0.f, 0.f};
#pragma unroll
        for (int pt = 0; pt < PT; ++pt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) top[pt] = fmaxf(top[pt], fabsf(S[nt][pt][i]));
        return column_max(pack_tops(top[0], top[1]));
    };
    auto scale_columns = [&](int sign) {
#pragma unroll
        for (int pt = 0; pt < PT; ++pt) {
            const float f = pow2(sign * kappa[pt]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) S[nt][pt] *= f;
        }
    };
    if constexpr (IO == 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PT; ++pt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    S[nt][pt][i] = finite_or_nan(S[nt][pt][i]);
        const uint32_t tops = column_tops();
#pragma unroll
        for (int pt = 0; pt < PT; ++pt) kappa[pt] = fit_fp16(top_of(tops, pt));
        scale_columns(1);
    }

    // Token `lane` of a chunk of n: step, log decay, its sums.  They are kept
    // by 16 tokens, with the sums of whole 16s apart, which are only ever added.
    // Within 16 tokens M takes differences of two sums, and there a reset in
    // front of both tokens must cost nothing: the sum up to a token is r + q, r
    // the sum of the logarithms rounded to 2^-8 (at most 16 x 150 x 2^8 such
    // steps: exact in fp32, and so are differences) and q that of what is left
    // (below 2^-5, off by 2^-25).
    float sums[4];
    auto token_vectors = [&](float raw, int n) {
        const float d = lane < n ? ssm_delta(raw, bias, in.dt_min, in.dt_max) : 0.f;
        const float l2 = lane < n ? fmaxf(A2 * d, -150.f) : 0.f;
        const float from = row_suffix(l2);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            sums[k] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, from), 16 * k));
        const float after = row_next(from);
        const float behind = g == 0 ? sums[1] + (sums[2] + sums[3]) : g == 1 ? sums[2] + sums[3] : g == 2 ? sums[3] : 0.f;
        const float w = d * __builtin_amdgcn_exp2f(after + behind);
        tok.w[lane] = w;
        if (IO == 1) d_max = wave_max(fmaxf(finite_or_nan(d), 0.f));
        if (!kLocal) {
            constexpr float kStep = 1.5f * 32768;   // fp32 is in steps of 2^-8 here
            const float coarse = (l2 + kStep) - kStep;
            tok.r[lane] = row_prefix(coarse);
            tok.q[lane] = row_prefix(l2 - coarse);
            tok.d[lane] = d;
            tok.f[lane] = d * __builtin_amdgcn_exp2f(after);
        }
    };

    f32x4 Dd;   // D on the diagonal of a tile
#pragma unroll
    for (int i = 0; i < 4; ++i) Dd[i] = 4 * g + i == m ? D : 0.f;
    const bool cols[2] = {store && g <= last_piece, store && 4 + g <= last_piece};

    int cur = 0;
    for (int t0 = 0; t0 < s.n; t0 += kChunk, cur ^= 1) {
        const int n = min(s.n - t0, kChunk);
        const uint16_t* const bs = sm.b[cur];
        const uint16_t* const cs_ = sm.c;
        const uint16_t* const xs = sm.x[wave];

        __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's part of the tiles is in LDS
        __syncthreads();                      // and the others'; the last chunk's tiles are read
        const float raw = raw_dt;
        const int next = min(s.n - t0 - kChunk, kChunk);   // tokens of the next chunk
        if (next > 0) {
            raw_dt = load_dt(next);
            bst.load(next, (cur ^ 1) * (uint32_t)sizeof(sm.b[0]), wave, lane);
        }
        u32x4 zr[PT / 2][4];
        f32x4 Y[PT][4];
        if constexpr (!kLocal) {
            if (gate) {
                const char* z = reinterpret_cast<const char*>(zp);
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) {
                    // (rows past the chunk: its first row again)
                    const uint32_t off = 16 * tt + m < n ? zm + 16 * tt * zrow : z0;
#pragma unroll
                    for (int q = 0; q < PT / 2; ++q)
                        zr[q][tt] = *reinterpret_cast<const u32x4*>(z + (4 * q + g <= last_piece ? off + 64 * q : off));
                }
                zp += kChunk * (int64_t)in.z_token;
            }
        }
        // From here to the barrier there is no branch: the token vectors' chain
        // of lane exchanges and C B^T's of LDS reads run beside S^T C^T
        token_vectors(raw, n);
        uint32_t s_tops = 0;   // fp16: the largest of each column of S
        if constexpr (IO == 1) s_tops = column_tops();
        if constexpr (!kLocal) {
            // (C B^T)^T: rows s, columns t of tile `wave` (of the tiles above the
            // diagonal, which nobody reads, too); S^T C^T: rows p, columns t
            static_assert(WAVES == 4, "a column tile of C B^T per wave");
            float s_scale[PT];
            if constexpr (IO == 1) {
                int k_s[PT];
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) {
                    k_s[pt] = fit_fp16(top_of(s_tops, pt));
                    s_scale[pt] = pow2(k_s[pt]);
                }
                if (g < PT) tok.k[lane] = g == 0 ? k_s[0] + kappa[0] : k_s[1] + kappa[1];
            }
            f32x4 acc[4];
#pragma unroll
            for (int st = 0; st < 4; ++st) acc[st] = zero4();
#pragma unroll
            for (int pt = 0; pt < PT; ++pt)
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) Y[pt][tt] = zero4();
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb) {
                s16x8 cop[4];
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) cop[tt] = row_operand<PR>(cs_, 16 * tt + m, 4 * kb + g);
                const s16x8 own = row_operand<PR>(cs_, 16 * wave + m, 4 * kb + g);
#pragma unroll
                for (int st = 0; st < 4; ++st)
                    acc[st] = mma<IO>(row_operand<PR>(bs, 16 * st + m, 4 * kb + g), own, acc[st]);
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[i] = S[2 * kb][pt][i];
                        v[4 + i] = S[2 * kb + 1][pt][i];
                        if (IO == 1) {
                            v[i] *= s_scale[pt];
                            v[4 + i] *= s_scale[pt];
                        }
                    }
                    s16x8 sop[2];
                    split<IO, 2>(v, sop);
#pragma unroll
                    for (int k = 1; k >= 0; --k)
#pragma unroll
                        for (int tt = 0; tt < 4; ++tt) Y[pt][tt] = mma<IO>(sop[k], cop[tt], Y[pt][tt]);
                }
            }
#pragma unroll
            for (int st = 0; st < 4; ++st)
                if (st <= wave) sm.cb[tri(wave, st)][lane] = acc[st];
            if constexpr (IO == 1) {   // (with what lies above the diagonal: a bound)
                float top = 0.f;
#pragma unroll
                for (int st = 0; st < 4; ++st)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(finite_or_nan(acc[st][i])));
                top = wave_max(top);
                if (lane == 0) sm.cb_top[wave] = top;
            }
        }
        s16x8 xop[PT][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int pt = 0; pt < PT; ++pt) xop[pt][kb] = tr_operand<XR>(xs, pt, kb, lane);
        bool poisoned = false;   // main pass: x has values that are not finite
        if constexpr (!kLocal) {
            f32x4 none = zero4();
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) none = mma<IO>(xop[pt][kb], s16x8{}, none);
            poisoned = __any((none[0] + none[1]) + (none[2] + none[3]) != 0.f);
            if (__builtin_expect(poisoned, 0)) {
                const int first = clear_not_finite<IO, XR>(sm.x[wave], lane);
                if (lane < 16 * PT) tok.first[lane] = (uint16_t)first;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int pt = 0; pt < PT; ++pt) xop[pt][kb] = tr_operand<XR>(xs, pt, kb, lane);
            }
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): x is read
        __syncthreads();   // the vectors and C B^T are complete, C is read
        if (next > 0) {
            // (z is here before they go out: waits count operations in order)
            if (!kLocal && gate) {
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                    for (int q = 0; q < PT / 2; ++q) asm volatile("" ::"v"(zr[q][tt]));
            }
            if (!kLocal) cst.load(next, 0, wave, lane);
            xst.load(next, 0, 0, lane);
        }

        if constexpr (!kLocal) {
            // fp16: M, at most max |C B^T| max d + |D|, times 2^k_m, and Y with it
            int k_m = 0;
            f32x4 Dm = Dd;
            if constexpr (IO == 1) {
                const f32x4 t = *reinterpret_cast<const f32x4*>(sm.cb_top);
                const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
                k_m = fit_fp16(2.f * fmaxf(top * d_max, fabsf(D)));
                k_m = __builtin_amdgcn_readfirstlane(k_m);
                Dm *= pow2(k_m);
            }
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                const float before = tt == 0 ? 0.f : tt == 1 ? sums[0] : tt == 2 ? sums[0] + sums[1] : sums[0] + (sums[1] + sums[2]);
                const float c = tok.r[16 * tt + m] + (tok.q[16 * tt + m] + before);
                const float e = __builtin_amdgcn_exp2f(c);
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) {
                    Y[pt][tt] *= e;
                    if constexpr (IO == 1) {   // from its columns' scales to M's
                        const i32x4 k = *reinterpret_cast<const i32x4*>(tok.k + 16 * pt + 4 * g);
#pragma unroll
                        for (int i = 0; i < 4; ++i) Y[pt][tt][i] = __builtin_ldexpf(Y[pt][tt][i], k_m - k[i]);
                    }
                }
            }
            // + X^T M^T, M[t][s] = (C B^T) e^{c_t - c_s} d_s for s <= t, + D for s = t.
            // Below the diagonal tiles the exponential is a product of one per
            // column and one per row, both at most 1.
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                const float rt = tok.r[16 * tt + m] + (IO == 1 ? (float)k_m : 0.f), qt = tok.q[16 * tt + m];
#pragma unroll
                for (int kb = 0; kb <= tt / 2; ++kb) {
                    float v[8];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int st = 2 * kb + q;
                        if (st > tt) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[4 * q + i] = 0.f;
                        } else if (st == tt) {
                            const f32x4 cb = sm.cb[tri(tt, st)][lane];
                            const f32x4 rs = *reinterpret_cast<const f32x4*>(tok.r + 16 * st + 4 * g);
                            const f32x4 qs = *reinterpret_cast<const f32x4*>(tok.q + 16 * st + 4 * g);
                            const f32x4 ds = *reinterpret_cast<const f32x4*>(tok.d + 16 * st + 4 * g);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float e = cb[i] * __builtin_amdgcn_exp2f((rt - rs[i]) + (qt - qs[i])) * ds[i];
                                v[4 * q + i] = (4 * g + i <= m ? e : 0.f) + Dm[i];
                            }
                        } else {
                            const f32x4 cb = sm.cb[tri(tt, st)][lane];
                            const f32x4 fs = *reinterpret_cast<const f32x4*>(tok.f + 16 * st + 4 * g);
                            const float between = tt - st == 1 ? 0.f : tt - st == 2 ? sums[st + 1] : sums[1] + sums[2];
                            const float ht = __builtin_amdgcn_exp2f(rt + (qt + between));
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[4 * q + i] = cb[i] * (fs[i] * ht);
                        }
                    }
                    s16x8 mop[kParts];
                    split<IO, kParts>(v, mop);
#pragma unroll
                    for (int k = kParts - 1; k >= 0; --k)
#pragma unroll
                        for (int pt = 0; pt < PT; ++pt) Y[pt][tt] = mma<IO>(xop[pt][kb], mop[k], Y[pt][tt]);
                }
            }
            // the gate, out: 8 channels of one token a lane
            if constexpr (IO == 1) {
                const float down = pow2(-k_m);
#pragma unroll
                for (int pt = 0; pt < PT; ++pt)
#pragma unroll
                    for (int tt = 0; tt < 4; ++tt) Y[pt][tt] *= down;
            }
            if (__builtin_expect(poisoned, 0)) {   // (by integer masks: as many conditions would spill scalar registers)
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int behind = tok.first[8 * g + 4 * pt + i] - m - 1;
#pragma unroll
                        for (int tt = 0; tt < 4; ++tt)
                            Y[pt][tt][i] = __uint_as_float(__float_as_uint(Y[pt][tt][i]) |
                                                           (uint32_t)((behind - 16 * tt) >> 31));
                    }
                    // and through w x the state
                    const int own = tok.first[8 * (m >> 2) + 4 * pt + (m & 3)];
                    xop[pt][0][0] = (short)(xop[pt][0][0] | (((own - kChunk) >> 31) & 0x7fff));
                }
            }
            if (gate) {
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                    for (int q = 0; q < PT / 2; ++q)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            f32x4& yv = Y[2 * q + (k >> 1)][tt];
                            yv[2 * (k & 1)] *= silu_fast(io_lo<IO>(zr[q][tt][k]));
                            yv[2 * (k & 1) + 1] *= silu_fast(io_hi<IO>(zr[q][tt][k]));
                        }
            }
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
#pragma unroll
                for (int q = 0; q < PT / 2; ++q) {
                    const f32x4 &u = Y[2 * q][tt], &v = Y[2 * q + 1][tt];
                    const u32x4 o = {io_pack<IO>(u[0], u[1]), io_pack<IO>(u[2], u[3]),
                                     io_pack<IO>(v[0], v[1]), io_pack<IO>(v[2], v[3])};
                    if (cols[q] && 16 * tt + m < n) *reinterpret_cast<u32x4*>(yp + (ym + 16 * tt * yrow + 64 * q)) = o;
                }
            }
            yp += kChunk * (uint64_t)yrow;
        }

        // S <- e^{c_Q} S + B^T (w x)
        const float total2 = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        const float decay = __builtin_amdgcn_exp2f(total2);
        log_total += total2;
        float dec[PT], w_scale[PT];
        uint32_t wx_tops = 0;   // fp16: the largest of each column of w x
        if constexpr (IO == 1) {
            float top[PT] = {0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const f32x4 w = *reinterpret_cast<const f32x4*>(tok.w + 32 * kb + 16 * q + 4 * g);
#pragma unroll
                    for (int pt = 0; pt < PT; ++pt)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t xr = __builtin_bit_cast(u32x4, xop[pt][kb])[2 * q + k];
                            top[pt] = fmaxf(fmaxf(top[pt], fabsf(io_lo<IO>(xr) * w[2 * k])),
                                            fabsf(io_hi<IO>(xr) * w[2 * k + 1]));
                        }
                }
            wx_tops = column_max(pack_tops(top[0], top[1]));
        }
#pragma unroll
        for (int pt = 0; pt < PT; ++pt) {
            dec[pt] = decay;
            if constexpr (IO == 1) {
                // the new kappa: the larger of the decayed state and w x fits
                const float left = decay * top_of(s_tops, pt);
                const int next_kappa = fit_fp16(fmaxf(left * pow2(-kappa[pt]), top_of(wx_tops, pt)));
                // (a state that is 0 takes any scale)
                dec[pt] = left == 0.f ? 0.f : __builtin_ldexpf(decay, next_kappa - kappa[pt]);
                kappa[pt] = next_kappa;
                w_scale[pt] = pow2(next_kappa);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PT; ++pt) S[nt][pt] *= dec[pt];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            s16x8 wx[PT][kParts];
            const f32x4 w0 = *reinterpret_cast<const f32x4*>(tok.w + 32 * kb + 4 * g);
            const f32x4 w1 = *reinterpret_cast<const f32x4*>(tok.w + 32 * kb + 16 + 4 * g);
#pragma unroll
            for (int pt = 0; pt < PT; ++pt) {
                const u32x4 xr = __builtin_bit_cast(u32x4, xop[pt][kb]);
                float v[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x4& w = k < 2 ? w0 : w1;
                    v[2 * k] = io_lo<IO>(xr[k]) * w[2 * (k & 1)];
                    v[2 * k + 1] = io_hi<IO>(xr[k]) * w[2 * (k & 1) + 1];
                    if (IO == 1) {
                        v[2 * k] *= w_scale[pt];
                        v[2 * k + 1] *= w_scale[pt];
                    }
                }
                split<IO, kParts>(v, wx[pt]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const s16x8 bop = tr_operand<PR>(bs, nt, kb, lane);
#pragma unroll
                for (int k = kParts - 1; k >= 0; --k)   // the smallest parts first
#pragma unroll
                    for (int pt = 0; pt < PT; ++pt) S[nt][pt] = mma<IO>(bop, wx[pt][k], S[nt][pt]);
            }
        }
    }

    if constexpr (IO == 1) scale_columns(-1);
    if (!store) return;
    if (kLocal) {
        f32x4* to = a.states + rec * (NT * PT * 64) + lane;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PT; ++pt) to[(nt * PT + pt) * 64] = S[nt][pt];
        if (lane == 0) a.decays[rec] = __builtin_amdgcn_exp2f(log_total);
    } else if (s.last) {
        float* to = a.sf + so;
#pragma unroll
        for (int pt = 0; pt < PT; ++pt)
            if (p_lane + p_off(pt) < P) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) to[n_off(nt, i) * P + p_off(pt)] = S[nt][pt][i];
            }
    }
}

// The states behind segments 1, 2, .. of a sequence from its segments' own:
// R_j = decay_j R_{j-1} + L_j in place, elementwise (fragment order), kAhead
// segments' loads ahead of the products, so that the chain waits for memory
// once per kAhead segments.  V is f32x4, or float where that leaves too few
// threads to carry the traffic (launch_scan).
template <typename V>
__global__ __launch_bounds__(kThreads) void ssm_join_kernel(const ScanArgs a, int elems, int parts) {
    const int64_t all = (int64_t)a.in.groups * a.tasks;   // records of a segment
    const int part = blockIdx.x % parts, rest = blockIdx.x / parts;
    const int rec = rest % (int)all, nth = rest / (int)all;
    int first = nth * (a.segs - 1), count = a.segs;   // a sequence's first record, and its segments
    if (a.table) {
        // packed: sequence nth, or where those outnumber the records the one that
        // begins at record nth: its row is the last in front of the next record's
        const bool by_seq = a.seqs < a.recs;
        int lo = 0, hi = a.rows;   // (rows behind the last block are -1)
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            const int4 b = a.table[mid];
            if (b.x < 0 || (by_seq ? b.x >= nth : b.y >= (nth + 1) * a.block)) hi = mid;
            else lo = mid + 1;
        }
        const int row = by_seq ? lo : lo - 1;
        if (row < 0 || row + 2 >= a.rows) return;
        const int4 b = a.table[row];
        const int seq = b.x;
        if ((by_seq && seq != nth) || b.w != 0 || a.table[row + 2].x != seq) return;
        for (int base = row;; base += 64) {
            const int r = base + (threadIdx.x & 63);
            const unsigned long long other = __ballot(r >= a.rows || a.table[min(r, a.rows - 1)].x != seq);
            if (other != 0) {
                count = base - row + __builtin_ctzll(other);
                break;
            }
        }
        first = min(max(b.y, 0) / a.block, a.recs);
        count = min(count, a.recs - first + 1);   // (as it is, for a table of this batch)
    }
    const int e = part * kThreads + threadIdx.x;
    if (count < 3 || e >= elems) return;
    V* const at = reinterpret_cast<V*>(a.states) + (first * all + rec) * elems + e;
    const float* const decay = a.decays + first * all + rec;
    const int64_t step = all * elems;
    constexpr int kAhead = 8;
    V R = at[0];
    for (int j0 = 1; j0 < count - 1; j0 += kAhead) {
        V L[kAhead];
        float d[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const bool on = j0 + k < count - 1;
            L[k] = on ? at[(j0 + k) * step] : V{};
            d[k] = on ? decay[(j0 + k) * all] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (j0 + k < count - 1) {
                R = R * d[k] + L[k];
                at[(j0 + k) * step] = R;
            }
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

// Whether the chunked scan has an instance (an MFMA sums over 32 state rows);
// a state of 16 rows takes the recurrence
bool chunked(const gdn_ssm_inputs* in) { return in->state_dim >= 32; }

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct Layout {
    int segs;        // segments of a batch row (0: packed)
    int64_t rows, recs;
    int slices, tasks, quads;
    bool ordered;
    size_t table, starts, order, states, decays, total;   // byte offsets

    Layout(const gdn_ssm_inputs* in, int seqs, int block, bool packed) {
        segs = packed ? 0 : std::max(1, (in->tokens + block - 1) / block);
        rows = packed ? (int64_t)in->tokens / block + seqs : (int64_t)segs * seqs;
        slices = (in->head_dim + kCols - 1) / kCols;
        tasks = in->heads / in->groups * slices;
        quads = (tasks + kWaves - 1) / kWaves;
        // a record for each segment but the last of a sequence: packed, whole
        // blocks with a token behind them (the recurrence needs none, and no table)
        recs = !chunked(in) ? 0 : packed ? std::max(in->tokens - 1, 0) / block : (int64_t)(segs - 1) * seqs;
        size_t off = 0;
        table = off;
        if (packed && chunked(in)) off += align256((size_t)rows * 16);
        starts = off;
        if (packed && chunked(in)) off += align256(((size_t)seqs + 1) * 4);
        order = off;
        ordered = packed && recs > 0 && rows * in->groups * quads <= kMaxOrder;
        if (ordered) off += align256((size_t)rows * 4);
        const size_t states_of = (size_t)recs * in->groups * tasks;
        states = off;
        off += align256(states_of * in->state_dim * kCols * 4);
        decays = off;
        off += align256(states_of * 4);
        total = std::max<size_t>(off, 256);
    }
};

template <int IO, int N, int PT, int WAVES>
hipError_t launch_scan(const ScanArgs& a, hipStream_t stream) {
    const int64_t groups = ((int64_t)a.rows * a.in.groups + 7) / 8 * 8 * a.quads;
    if (groups > 0x7fffffff) return hipErrorInvalidValue;
    if (a.recs > 0) {
        hipLaunchKernelGGL((ssm_scan_kernel<IO, N, PT, WAVES, true>), dim3((unsigned)groups),
                           dim3(64 * WAVES), 0, stream, a);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        if (a.table ? a.recs > 1 : a.segs > kMaxFold) {
            // 16 bytes a thread from 2^17 such threads on (8 sequences of 2..7
            // segments x 128 records: 13 us against 35 with 4 bytes; one of 64
            // segments x 32 records: 30 us against 15)
            const int64_t all = (int64_t)a.in.groups * a.tasks;
            const int64_t records = (a.table ? std::min(a.seqs, a.recs) : a.seqs) * all;
            const bool wide = records * N * PT * 4 >= 1 << 17;
            const int elems = N * PT * (wide ? 4 : 16), parts = (elems + kThreads - 1) / kThreads;
            if (records * parts > 0x7fffffff) return hipErrorInvalidValue;
            const dim3 grid((unsigned)(records * parts));
            if (wide) hipLaunchKernelGGL(ssm_join_kernel<f32x4>, grid, dim3(kThreads), 0, stream, a, elems, parts);
            else hipLaunchKernelGGL(ssm_join_kernel<float>, grid, dim3(kThreads), 0, stream, a, elems, parts);
            if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
    }
    hipLaunchKernelGGL((ssm_scan_kernel<IO, N, PT, WAVES, false>), dim3((unsigned)groups), dim3(64 * WAVES), 0,
                       stream, a);
    return hipGetLastError();
}

template <int IO>
hipError_t launch_any(const ScanArgs& a, hipStream_t stream) {
    switch (a.in.state_dim) {
        case 32: return launch_scan<IO, 32, kTiles, kWaves>(a, stream);
        case 64: return launch_scan<IO, 64, kTiles, kWaves>(a, stream);
        case 128: return launch_scan<IO, 128, kTiles, kWaves>(a, stream);
        default: return launch_scan<IO, 256, kTiles, kWaves>(a, stream);
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

// Microseconds of `groups` work-groups of `chunks` chunks each on 256 CUs that
// hold `deep` of them at a time: a chunk takes t[k - 1] with k on a CU, and a
// group `start` on top.
static double passes_us(double groups, double chunks, int deep, const double* t, double start) {
    const double full = std::floor(groups / (256.0 * deep));
    const double rest = groups - full * 256 * deep;
    double us = full * (chunks * t[deep - 1] + start);
    if (rest > 0) us += chunks * t[std::min(deep, (int)std::ceil(rest / 256)) - 1] + start;
    return us;
}

// The run of chunks with the least estimated time.  Longer runs leave CUs idle
// or the last round of work-groups thin, shorter ones move more states (16 KB
// to 64 KB a record and pass).  The constants are measured at state_dim 128
// (main pass: 5.7 and 8.8 us a chunk with one and two groups on a CU; first pass
// 2.9, 3.3 and 3.6 with one to three; about 5 us to start a group from its
// state), the rule's choices 1 % slower on average than the best of 1 .. 256
// chunks over 23 calls (130 to 65,536 tokens, 8 to 128 heads, 1 to 101
// sequences), at most 15 % (130 tokens x 64 heads, 3 chunks 20.6 us against 17.8).
//
// A packed batch whose sequences fill the chip 1.2 times without a split is
// split only where one would hold the others up: at 1.5 times the chunks that
// a place then works off (30 prompts of 50 to 2000 tokens x 64 heads: 47 chunks
// 336 us against 449 at the estimate's 8).  The lengths are on the GPU, so what a
// packed call takes is a guess: over 37 batches (2 to 300 prompts, uniform
// lengths, and one long among short ones) the choices are 5 % slower on average
// than the best, at most 33 %.
extern "C" int gdn_ssm_scan_block(const gdn_ssm_inputs* in, int num_seqs) {
    if (!ssm_sizes_ok(in) || num_seqs < 1 || in->tokens > (1 << 30)) return 0;
    const int tasks = in->heads / in->groups * ((in->head_dim + kCols - 1) / kCols);
    const double units = (double)in->groups * ((tasks + kWaves - 1) / kWaves);
    const bool packed = in->batch == 1 && num_seqs > 1;
    // chunks of a sequence (of the average one, half a chunk of it partial)
    const double tokens = packed ? (double)in->tokens / num_seqs : in->tokens;
    const double per_seq = std::max(1.0, packed ? tokens / kChunk + 0.5 : std::ceil(tokens / kChunk));
    // a group's chunks: packed sequences differ, the longest of a few is about
    // 1.7 times the average
    const double longest = packed ? 1.7 * per_seq : per_seq;
    const int deep = in->state_dim == 256 ? 1 : 2, local_deep = in->state_dim == 256 ? 1 : 3;
    const double places = 256.0 * deep;
    if (packed && num_seqs * units >= 1.2 * places) {
        const double each = ((double)in->tokens / kChunk + 0.5 * num_seqs) * units / places;
        return (int)std::min(std::ceil(1.5 * each), (double)(kMaxBlock / kChunk)) * kChunk;
    }
    const double main_t[2] = {5.7, 8.8}, local_t[3] = {2.9, 3.3, 3.6};
    const double record_us = (double)in->groups * tasks * in->state_dim * kCols * 4 / 5e6;
    const double scale = in->state_dim / 128.0;
    int best = 1;
    double least = 0;
    for (int c = 1; c <= kMaxBlock / kChunk; c += c < 16 ? 1 : c / 8) {
        const double segs = packed ? std::max(1.0, per_seq / c + 0.5) : std::ceil(per_seq / c);
        double us = passes_us(num_seqs * segs * units, std::min<double>(c, longest), deep, main_t, 4) * scale;
        if (segs > 1)
            us += 3 + passes_us(num_seqs * (segs - 1) * units, std::min<double>(c, longest), local_deep, local_t,
                                4) * scale;
        // records: written by the first pass, and read by the main pass (all
        // in front of a segment, where it joins them) or the join
        const bool fold = !packed && segs <= kMaxFold;
        us += num_seqs * (segs - 1) * record_us * (fold ? 1 + segs / 2 : 2);
        if (segs > 2 && !fold) us += 4 + 2 * num_seqs * (segs - 2) * record_us;
        if (c == 1 || us < least) {
            least = us;
            best = c;
        }
        if (c >= (packed ? 4 : 1) * per_seq) break;
    }
    return best * kChunk;
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
    if (!in->A_log || !sf || sf == s0 || !ssm_aligned(sf, 4) || !ssm_aligned(s0, 4) || (in->tokens > 0 && !y) ||
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
    a.recs = (int)l.recs;
    a.segs = l.segs;
    a.seqs = num_seqs;
    a.block = block;
    a.slices = l.slices;
    a.tasks = l.tasks;
    a.quads = l.quads;
    a.fold = !packed && l.segs <= kMaxFold;
    a.states = reinterpret_cast<f32x4*>(ws + l.states);
    a.decays = reinterpret_cast<float*>(ws + l.decays);
    if (packed) {
        if (l.ordered) a.order = reinterpret_cast<int*>(ws + l.order);
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
    return in->io_dtype == GDN_DTYPE_BF16 ? launch_any<0>(a, stream) : launch_any<1>(a, stream);
}
