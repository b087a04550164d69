// Learned position bias by buckets: a table spread over a map, and the table's
// gradient (include/bfhip_transformer.h).
#include "bfhip_transformer.h"
#include "gemm_core.h"

using namespace bfhip;

namespace {

constexpr int kThreads = 256;

__global__ __launch_bounds__(kThreads) void bias_forward_kernel(const float *table, const int *map,
                                                                float *bias, int buckets, int heads,
                                                                long long n) {
    const long long p = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (p >= n) return;
    const int b = map[p];
    for (int h = 0; h < heads; ++h)
        bias[h * n + p] = (unsigned)b < (unsigned)buckets ? table[(size_t)b * heads + h] : 0.f;
}

// One workgroup per (bucket, head): the sum over the map in a fixed order.
__global__ __launch_bounds__(kThreads) void bias_backward_kernel(const float *dbias, const int *map,
                                                                 float *dtable, int heads,
                                                                 long long n) {
    __shared__ float part[kThreads / kWave];
    const int b = blockIdx.x / heads, h = blockIdx.x % heads;
    float sum = 0.f;
    for (long long p = threadIdx.x; p < n; p += kThreads)
        if (map[p] == b) sum += dbias[h * n + p];
    sum = group_sum<kWave>(sum);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) dtable[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

bool bad_bias(int buckets, int heads, long long positions) {
    return buckets <= 0 || heads <= 0 || positions < 0 || (long long)buckets * heads > 1 << 28 ||
           positions > (1ll << 40) / heads;
}

}  // namespace

extern "C" int bfhip_position_bias_forward(const float *table, const int *map, float *bias,
                                           int buckets, int heads, long long positions,
                                           void *stream, char *error, size_t cap) {
    if (bad_bias(buckets, heads, positions) || (positions && (!table || !map || !bias)))
        return fail(error, cap, "invalid position bias contract");
    if (positions == 0) return 1;
    const long long grid = (positions + kThreads - 1) / kThreads;
    if (!launch_fits(grid, kThreads)) return fail(error, cap, "position bias has too many positions");
    hipLaunchKernelGGL(bias_forward_kernel, dim3((unsigned)grid), dim3(kThreads), 0,
                       (hipStream_t)stream, table, map, bias, buckets, heads, positions);
    return launch_ok(error, cap, "position bias launch");
}

extern "C" size_t bfhip_position_bias_backward_workspace(int buckets, int heads, long long positions) {
    (void)buckets, (void)heads, (void)positions;
    return 0;
}

extern "C" int bfhip_position_bias_backward(const float *dbias, const int *map, float *dtable,
                                            int buckets, int heads, long long positions,
                                            void *workspace, size_t workspace_bytes, void *stream,
                                            char *error, size_t cap) {
    (void)workspace, (void)workspace_bytes;
    if (bad_bias(buckets, heads, positions) || !dtable || (positions && (!dbias || !map)))
        return fail(error, cap, "invalid position bias contract");
    if (!launch_fits((long long)buckets * heads, kThreads))
        return fail(error, cap, "position bias has too many buckets");
    hipLaunchKernelGGL(bias_backward_kernel, dim3(buckets * heads), dim3(kThreads), 0,
                       (hipStream_t)stream, dbias, map, dtable, heads, positions);
    return launch_ok(error, cap, "position bias launch");
}
