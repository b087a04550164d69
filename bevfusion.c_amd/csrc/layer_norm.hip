// Stateless layer norm, forward and backward (include/bfhip_transformer.h).
#include "bfhip_transformer.h"
#include "element.h"
#include "gemm_core.h"

using namespace bfhip;

namespace {

constexpr int kRowWaves = 4;  // rows of a workgroup, one wave each

// One wave per row: the mean, then the centred squares (not E[x^2] - E[x]^2,
// which loses a spread that is small beside the mean), then the result.
template <class E>
__global__ __launch_bounds__(kRowWaves *kWave) void norm_forward_kernel(
    const typename E::Word *x, long long xs, const float *gamma, const float *beta,
    typename E::Word *y, long long ys, float *mean, float *rstd, long long rows, int n, float eps) {
    const int lane = threadIdx.x % kWave;
    const long long r = (long long)blockIdx.x * kRowWaves + threadIdx.x / kWave;
    if (r >= rows) return;
    x += r * xs;
    y += r * ys;
    float sum = 0.f, dev = 0.f;
    for (int c = lane; c < n; c += kWave) sum += E::get(x[c]);
    const float m = group_sum<kWave>(sum) / (float)n;
    for (int c = lane; c < n; c += kWave) {
        const float d = E::get(x[c]) - m;
        dev = fmaf(d, d, dev);
    }
    const float s = 1.f / sqrtf(group_sum<kWave>(dev) / (float)n + eps);
    for (int c = lane; c < n; c += kWave) {
        float v = (E::get(x[c]) - m) * s;
        if (gamma) v *= gamma[c];
        if (beta) v += beta[c];
        y[c] = E::put(v);
    }
    if (mean && lane == 0) {
        mean[r] = m;
        rstd[r] = s;
    }
}

template <class E>
__global__ __launch_bounds__(kRowWaves *kWave) void norm_backward_kernel(
    const typename E::Word *dy, long long dys, const typename E::Word *x, long long xs,
    const float *gamma, const float *mean, const float *rstd, typename E::Word *dx, long long dxs,
    long long rows, int n) {
    const int lane = threadIdx.x % kWave;
    const long long r = (long long)blockIdx.x * kRowWaves + threadIdx.x / kWave;
    if (r >= rows) return;
    dy += r * dys;
    x += r * xs;
    dx += r * dxs;
    const float m = mean[r], s = rstd[r];
    float sg = 0.f, sgh = 0.f;
    for (int c = lane; c < n; c += kWave) {
        const float g = E::get(dy[c]) * (gamma ? gamma[c] : 1.f);
        sg += g;
        sgh = fmaf(g, (E::get(x[c]) - m) * s, sgh);
    }
    sg = group_sum<kWave>(sg) / (float)n;
    sgh = group_sum<kWave>(sgh) / (float)n;
    for (int c = lane; c < n; c += kWave) {
        const float g = E::get(dy[c]) * (gamma ? gamma[c] : 1.f), h = (E::get(x[c]) - m) * s;
        dx[c] = E::put(s * (g - sg - h * sgh));
    }
}

// Sums over rows of dy * h and dy: workgroup (column block, part) sums every
// parts-th group of 4 rows; partial [parts][2][n].
template <class E>
__global__ __launch_bounds__(256) void norm_weight_kernel(
    const typename E::Word *dy, long long dys, const typename E::Word *x, long long xs,
    const float *mean, const float *rstd, float *partial, long long rows, int n) {
    __shared__ float sum[2][4][64];
    const int c = blockIdx.x * 64 + threadIdx.x % 64, w = threadIdx.x / 64;
    float a = 0.f, b = 0.f;
    if (c < n)
        for (long long r = 4ll * blockIdx.y + w; r < rows; r += 4ll * gridDim.y) {
            const float g = E::get(dy[r * dys + c]);
            a = fmaf(g, (E::get(x[r * xs + c]) - mean[r]) * rstd[r], a);
            b += g;
        }
    sum[0][w][threadIdx.x % 64] = a;
    sum[1][w][threadIdx.x % 64] = b;
    __syncthreads();
    if (w > 1 || c >= n) return;
    const float(*q)[64] = sum[w];
    const int t = threadIdx.x % 64;
    partial[(size_t)(2 * blockIdx.y + w) * n + c] = (q[0][t] + q[1][t]) + (q[2][t] + q[3][t]);
}

__global__ __launch_bounds__(256) void norm_weight_sum_kernel(const float *partial, int parts,
                                                              float *dgamma, float *dbeta, int n) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    float a = 0.f, b = 0.f;
    for (int p = 0; p < parts; ++p) {
        a += partial[(size_t)(2 * p) * n + c];
        b += partial[(size_t)(2 * p + 1) * n + c];
    }
    dgamma[c] = a;
    dbeta[c] = b;
}

constexpr int kMaxFeatures = 65536;

int norm_parts(long long rows) { return (int)(rows <= 0 ? 0 : rows >= 256 ? 64 : (rows + 3) / 4); }

bool bad_norm(int type, long long rows, int n) {
    return type < BFHIP_F32 || type > BFHIP_BF16 || rows < 0 || n <= 0 || n > kMaxFeatures;
}

}  // namespace

extern "C" int bfhip_layer_norm_forward(int type, const void *x, long long x_stride,
                                        const float *gamma, const float *beta, void *y,
                                        long long y_stride, float *mean, float *rstd,
                                        long long rows, int features, float eps, void *stream,
                                        char *error, size_t cap) {
    if (bad_norm(type, rows, features) || !(eps >= 0.f) || !mean != !rstd)
        return fail(error, cap, "invalid layer norm contract");
    if (rows == 0) return 1;
    if (!x || !y || (rows > 1 && (x_stride < 0 || y_stride < features)))
        return fail(error, cap, "invalid layer norm contract");
    const long long grid = (rows + kRowWaves - 1) / kRowWaves;
    if (!launch_fits(grid, kRowWaves * kWave)) return fail(error, cap, "layer norm has too many rows");
    with_element(type, [&](auto e) {
        using E = decltype(e);
        using W = typename E::Word;
        hipLaunchKernelGGL(norm_forward_kernel<E>, dim3((unsigned)grid), dim3(kRowWaves * kWave), 0,
                           (hipStream_t)stream, (const W *)x, x_stride, gamma, beta, (W *)y,
                           y_stride, mean, rstd, rows, features, eps);
    });
    return launch_ok(error, cap, "layer norm launch");
}

extern "C" size_t bfhip_layer_norm_backward_workspace(long long rows, int features) {
    if (bad_norm(BFHIP_F32, rows, features)) return 0;
    return (size_t)norm_parts(rows) * 2 * features * sizeof(float);
}

extern "C" int bfhip_layer_norm_backward(int type, const void *dy, long long dy_stride,
                                         const void *x, long long x_stride, const float *gamma,
                                         const float *mean, const float *rstd, void *dx,
                                         long long dx_stride, float *dgamma, float *dbeta,
                                         long long rows, int features, void *workspace,
                                         size_t workspace_bytes, void *stream, char *error,
                                         size_t cap) {
    if (bad_norm(type, rows, features) || !dgamma != !dbeta)
        return fail(error, cap, "invalid layer norm contract");
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx ||
                     (rows > 1 && (dy_stride < 0 || x_stride < 0 || dx_stride < features))))
        return fail(error, cap, "invalid layer norm contract");
    const long long grid = (rows + kRowWaves - 1) / kRowWaves;
    if (!launch_fits(grid, kRowWaves * kWave)) return fail(error, cap, "layer norm has too many rows");
    const int parts = norm_parts(rows);
    if (dgamma && parts && (!workspace || ((uintptr_t)workspace & 15) ||
                            workspace_bytes < bfhip_layer_norm_backward_workspace(rows, features)))
        return fail(error, cap, "layer norm workspace too small or not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    with_element(type, [&](auto e) {
        using E = decltype(e);
        using W = typename E::Word;
        // The weights' sums first: dx may overwrite dy or x.
        if (dgamma && parts)
            hipLaunchKernelGGL(norm_weight_kernel<E>, dim3((features + 63) / 64, parts), dim3(256),
                               0, s, (const W *)dy, dy_stride, (const W *)x, x_stride, mean, rstd,
                               (float *)workspace, rows, features);
        if (grid)
            hipLaunchKernelGGL(norm_backward_kernel<E>, dim3((unsigned)grid), dim3(kRowWaves * kWave),
                               0, s, (const W *)dy, dy_stride, (const W *)x, x_stride, gamma, mean,
                               rstd, (W *)dx, dx_stride, rows, features);
    });
    if (dgamma)
        hipLaunchKernelGGL(norm_weight_sum_kernel, dim3((features + 255) / 256), dim3(256), 0, s,
                           (const float *)workspace, parts, dgamma, dbeta, features);
    return launch_ok(error, cap, "layer norm launch");
}
