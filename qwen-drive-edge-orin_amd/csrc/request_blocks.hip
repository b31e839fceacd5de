// Tables of a packed batch, built on the GPU from request lengths (gfx950).
//
//   cu[n]      = min(sum_{m < n} max(len_m, 0), total)          n = 0 .. N
//   rows(n)    = max(1, ceil((cu[n+1] - cu[n]) / block))         blocks of request n
//   start[n]   = sum_{m < n} rows(m)
//   blocks[r]  = (n, first token, tokens, index within n) for start[n] <= r < start[n+1],
//                (-1, 0, 0, 0) past the last one
//   slot[t]    = slots[n] (or n), pos[t] = t - cu[n] for cu[n] <= t < cu[n+1],
//                -1 and 0 behind the last request
// An empty request owns one empty block, so that a kernel that walks the
// table still visits it (its state passes through).  Rows never exceed
// total / block + N, the bound that a caller allocates without reading the
// lengths.
//
// Bytes are few (8 per token); what counts is launches and the chain from the
// lengths to the last store.  Up to kOneLaunch requests every work-group
// forms both prefix sums of the whole batch for itself in LDS and then fills
// its own part of the tables; past that a single group writes them and a
// second launch searches them in the cache.  4.5 us for 8 requests, 8.4 for
// 1500 with 274,000 tokens (12 with a scan per 256 requests in place of a
// thread's run of requests and one scan), 20 for 6000 with 1,093,000: sums 9,
// tables 11.
#include "gdn_common.h"
#include "gdn_hip.h"

#include <algorithm>

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kOneLaunch = 4096;            // requests whose sums fit in a group's LDS (32 KB)
constexpr int kTokens = 4;                  // consecutive tokens a thread fills (one 16-byte store each)
constexpr int kScanThreads = 1024;          // the single group of the two-launch form

__device__ __forceinline__ int sat(int a, int b, int top) {   // 0 <= a, b <= top <= 2^30
    return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)top);   // (2^30 + 2^30 passes an int)
}

__device__ __forceinline__ int rows_of(int n, int block) { return max(1, (n + block - 1) / block); }

// Inclusive saturating prefix sum of one value per thread over the group;
// `all` gets the group's sum.  red: one int per wave.
template <int NT>
__device__ __forceinline__ int group_scan(int v, int top, int* red, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int u = __shfl_up(v, off, 64);
        if (lane >= off) v = sat(v, u, top);
    }
    __syncthreads();
    if (lane == 63) red[wave] = v;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w == wave) before = sum;
        sum = sat(sum, red[w], top);
    }
    all = sum;
    return sat(v, before, top);
}

// cu[0..N] and start[0..N] by one group: a thread adds up `each` consecutive
// requests, so that the batch takes two scans over the group however long it is
template <int NT>
__device__ void form_sums(const int32_t* lens, int N, int total, int block, int* cu, int* start,
                          int* red) {
    const int each = (N + NT - 1) / NT;
    const int n0 = min((int)threadIdx.x * each, N), n1 = min(n0 + each, N);
    auto len = [&](int n) { return min(max(lens[n], 0), total); };
    int sum = 0, all;
    for (int n = n0; n < n1; ++n) sum = sat(sum, len(n), total);
    const int incl = group_scan<NT>(sum, total, red, all);
    // what lies in front of this thread's requests: its neighbour's sum
    int before = __shfl_up(incl, 1, 64);
    if ((threadIdx.x & 63) == 0) {
        before = 0;
        for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) before = sat(before, red[w], total);
    }
    int rows = 0, at = before;
    for (int n = n0; n < n1; ++n) {
        const int next = sat(at, len(n), total);
        rows += rows_of(next - at, block);
        cu[n + 1] = at = next;
    }
    int row = group_scan<NT>(rows, 0x40000000, red, all) - rows;
    at = before;
    for (int n = n0; n < n1; ++n) {
        const int next = sat(at, len(n), total);
        start[n + 1] = row += rows_of(next - at, block);
        at = next;
    }
    if (threadIdx.x == 0) cu[0] = start[0] = 0;
    __syncthreads();
}

// The n in [0, N) with a[n] <= v < a[n + 1]; N where v >= a[N] (a[0] = 0)
__device__ __forceinline__ int owner(const int* a, int N, int v) {
    int lo = 0, hi = N;   // the first n with a[n + 1] > v
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a[mid + 1] > v) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__device__ __forceinline__ void fill(const int* cu, const int* start, const int32_t* slots, int N,
                                     int total, int block, int rows, int4* blocks, int* slot,
                                     int* pos) {
    const int id = blockIdx.x * kThreads + threadIdx.x, all = gridDim.x * kThreads;
    for (int r = id; r < rows; r += all) {
        const int n = owner(start, N, r);
        int4 row = make_int4(-1, 0, 0, 0);
        if (n < N) {
            const int idx = r - start[n], t0 = cu[n] + idx * block;
            row = make_int4(n, t0, min(cu[n + 1] - t0, block), idx);
        }
        blocks[r] = row;
    }
    for (int t0 = id * kTokens; t0 < total; t0 += all * kTokens) {
        int n = owner(cu, N, t0);
        int s[kTokens], p[kTokens];
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            while (n < N && cu[n + 1] <= t0 + i) ++n;   // past empty requests too
            s[i] = n < N ? (slots ? slots[n] : n) : -1;
            p[i] = n < N ? t0 + i - cu[n] : 0;
        }
        if (t0 + kTokens <= total) {
            *reinterpret_cast<int4*>(slot + t0) = make_int4(s[0], s[1], s[2], s[3]);
            *reinterpret_cast<int4*>(pos + t0) = make_int4(p[0], p[1], p[2], p[3]);
        } else {
            for (int i = 0; t0 + i < total; ++i) {
                slot[t0 + i] = s[i];
                pos[t0 + i] = p[i];
            }
        }
    }
}

__global__ __launch_bounds__(kThreads) void request_blocks_kernel(
    const int32_t* __restrict__ lens, const int32_t* __restrict__ slots, int N, int total, int block,
    int rows, int* __restrict__ cu, int4* __restrict__ blocks, int* __restrict__ slot,
    int* __restrict__ pos) {
    __shared__ int red[kWaves], scu[kOneLaunch + 1], sstart[kOneLaunch + 1];
    form_sums<kThreads>(lens, N, total, block, scu, sstart, red);
    if (blockIdx.x == 0)
        for (int n = threadIdx.x; n <= N; n += kThreads) cu[n] = scu[n];
    fill(scu, sstart, slots, N, total, block, rows, blocks, slot, pos);
}

__global__ __launch_bounds__(kScanThreads) void request_sums_kernel(
    const int32_t* __restrict__ lens, int N, int total, int block, int* __restrict__ cu,
    int* __restrict__ start) {
    __shared__ int red[kScanThreads / 64];
    form_sums<kScanThreads>(lens, N, total, block, cu, start, red);
}

__global__ __launch_bounds__(kThreads) void request_fill_kernel(
    const int* __restrict__ cu, const int* __restrict__ start, const int32_t* __restrict__ slots,
    int N, int total, int block, int rows, int4* __restrict__ blocks, int* __restrict__ slot,
    int* __restrict__ pos) {
    fill(cu, start, slots, N, total, block, rows, blocks, slot, pos);
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_request_block_rows(int total_tokens, int num_requests, int block) {
    if (total_tokens < 0 || total_tokens > (1 << 30) || num_requests < 1 ||
        num_requests > (1 << 24) || block < 64 || block % 64 != 0)
        return 0;
    return total_tokens / block + num_requests;
}

extern "C" hipError_t gdn_request_blocks(const int32_t* lengths, const int32_t* slots,
                                         int num_requests, int total_tokens, int block,
                                         int32_t* cu_seqlens, int32_t* row_start, int32_t* blocks,
                                         int32_t* token_slots, int32_t* token_pos,
                                         hipStream_t stream) {
    const int rows = gdn_request_block_rows(total_tokens, num_requests, block);
    if (rows == 0 || !lengths || !cu_seqlens || !row_start || !blocks) return hipErrorInvalidValue;
    if (total_tokens > 0 && (!token_slots || !token_pos)) return hipErrorInvalidValue;
    if (((uintptr_t)blocks | (uintptr_t)token_slots | (uintptr_t)token_pos) % 16 != 0)
        return hipErrorInvalidValue;
    const int64_t per = (int64_t)kThreads * kTokens;
    const unsigned grid = (unsigned)std::min<int64_t>(
        std::max<int64_t>((total_tokens + per - 1) / per, (rows + kThreads - 1) / kThreads), 1024);
    auto tab = reinterpret_cast<int4*>(blocks);
    if (num_requests <= kOneLaunch) {
        hipLaunchKernelGGL(request_blocks_kernel, dim3(grid), dim3(kThreads), 0, stream, lengths,
                           slots, num_requests, total_tokens, block, rows, cu_seqlens, tab,
                           token_slots, token_pos);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(request_sums_kernel, dim3(1), dim3(kScanThreads), 0, stream, lengths,
                       num_requests, total_tokens, block, cu_seqlens, row_start);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    hipLaunchKernelGGL(request_fill_kernel, dim3(grid), dim3(kThreads), 0, stream, cu_seqlens,
                       row_start, slots, num_requests, total_tokens, block, rows, tab, token_slots,
                       token_pos);
    return hipGetLastError();
}
