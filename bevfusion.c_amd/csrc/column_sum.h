// Sums of partial results over their parts, in a fixed order.
#pragma once

#include "gemm_core.h"

namespace bfhip {

// out[i] = sum over p of partial[p][i], i < n; from `split` on the results go to
// out2[i - split].  A workgroup has 16 neighbouring columns and 32 shares of the
// parts, eight loads in flight each, added up in order at the end.  Bound by the
// latency of its loads (512 parts of 1536 columns: 4 us, 11 with 16 shares and
// one load in flight).
constexpr int kSumThreads = 512;

static __global__ __launch_bounds__(kSumThreads) void column_sum_kernel(const float *partial, long long parts, float *out,
                                                                        float *out2, long long split, long long n) {
    constexpr int kShares = kSumThreads / 16;
    __shared__ float sum[kShares][17];
    const long long c = (long long)blockIdx.x * 16 + threadIdx.x % 16;
    const int w = threadIdx.x / 16;
    float s = 0.f;
    if (c < n) {
#pragma unroll 8
        for (long long p = w; p < parts; p += kShares) s += partial[p * n + c];
    }
    sum[w][threadIdx.x % 16] = s;
    __syncthreads();
    if (w || c >= n) return;
#pragma unroll
    for (int i = 1; i < kShares; ++i) s += sum[i][threadIdx.x];
    if (c < split) out[c] = s;
    else out2[c - split] = s;
}

// Whether a launch holds n columns' workgroups.
inline bool column_sum_fits(long long n) { return launch_fits((n + 15) / 16, kSumThreads); }

inline void column_sum(const float *partial, long long parts, float *out, float *out2, long long split, long long n, hipStream_t s) {
    hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)((n + 15) / 16)), dim3(kSumThreads), 0, s, partial, parts, out, out2,
                       split, n);
}

}  // namespace bfhip
