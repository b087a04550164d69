// Stateless layer norm, forward and backward (include/bfhip_transformer.h).
#include "bfhip_transformer.h"
#include "column_sum.h"
#include "element.h"
#include "gemm_core.h"

#include <type_traits>

using namespace bfhip;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxFeatures = 65536;

// What bounds these kernels is memory: a row is read once, held in registers
// (as words, converted where they are used) by a group of LANES threads, CHUNKS
// 16-byte chunks each, and written once.  Chunks of a group's lanes are
// neighbours in memory; a group walks rows with the norm's weights and, in the
// backward pass, its columns' gradient sums in registers, and loads the next row
// before it works on one.
template <class E, int LANES, int CHUNKS>
struct NormRow {
    static constexpr int kWords = 16 / E::kSize, kGroups = kThreads / LANES;
    using Chunk = Words<E, kWords>;
    using Floats = Words<ElemF32, kWords>;
    // Threads of one group; LANES > 64: the workgroup's waves together.
    __device__ static int lane() { return threadIdx.x % LANES; }
    __device__ static int group() { return threadIdx.x / LANES; }
    __device__ static int column(int k) { return (k * LANES + lane()) * kWords; }

    // Elements past the row's end read as zero.
    template <class W>
    __device__ __forceinline__ static void load(const typename W::Word *row, int n, W (&v)[CHUNKS]) {
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int c = column(k);
            if (c + kWords <= n) {
                v[k] = W::load(row + c);
            } else {
#pragma unroll
                for (int e = 0; e < kWords; ++e) v[k].w[e] = c + e < n ? row[c + e] : (typename W::Word)0.f;
            }
        }
    }
    __device__ __forceinline__ static void store(typename E::Word *row, int n, const Chunk (&v)[CHUNKS]) {
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int c = column(k);
            if (c + kWords <= n) {
                v[k].store(row + c);
            } else {
#pragma unroll
                for (int e = 0; e < kWords; ++e)
                    if (c + e < n) row[c + e] = v[k].w[e];
            }
        }
    }
    // The group's sums of two values, in a fixed order.
    __device__ __forceinline__ static float2 sum(float a, float b) {
        constexpr int wave = LANES < kWave ? LANES : kWave;
        a = group_sum<wave>(a);
        b = group_sum<wave>(b);
        if constexpr (LANES > kWave) {
            __shared__ float2 part[LANES / kWave];
            const int w = threadIdx.x / kWave;
            __syncthreads();  // the sums before have been read
            if (threadIdx.x % kWave == 0) part[w] = make_float2(a, b);
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int i = 0; i < LANES / kWave; ++i) {
                a += part[i].x;
                b += part[i].y;
            }
        }
        return make_float2(a, b);
    }
};

struct NormArgs {
    const void *x, *dy;
    void *y;  // y or dx
    long long xs, dys, ys, rows;
    const float *gamma, *beta;
    float *mean, *rstd;
    float *partial;  // [workgroups][2][n], unless there is one workgroup
    float *dgamma, *dbeta;
    int n;
    float eps;
};

// 65536 x 768 bf16: 37 us, 5.4 TB/s; 200 x 128 fp32: 3 us, latency.
// The mean, then the centred squares (not E[x^2] - E[x]^2, which loses a
// spread that is small beside the mean), then the result.
template <class E, int LANES, int CHUNKS>
__global__ __launch_bounds__(kThreads) void norm_forward_kernel(NormArgs a) {
    using R = NormRow<E, LANES, CHUNKS>;
    using W = typename E::Word;
    typename R::Floats gamma[CHUNKS], beta[CHUNKS];
    if (a.gamma) R::load(a.gamma, a.n, gamma);
    if (a.beta) R::load(a.beta, a.n, beta);
    const float n = (float)a.n;
    const long long step = (long long)gridDim.x * R::kGroups;
    long long r = (long long)blockIdx.x * R::kGroups + R::group();
    typename R::Chunk next[CHUNKS];
    if (r < a.rows) R::load((const W *)a.x + r * a.xs, a.n, next);
    for (; r < a.rows; r += step) {
        typename R::Chunk x[CHUNKS];
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) x[k] = next[k];
        if (r + step < a.rows) R::load((const W *)a.x + (r + step) * a.xs, a.n, next);
        float s = 0.f, d = 0.f;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int e = 0; e < R::kWords; ++e) s += x[k].get(e);
        const float m = R::sum(s, 0.f).x / n;  // (a row of equal values has exactly their mean)
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int e = 0; e < R::kWords; ++e) {
                const float v = R::column(k) + e < a.n ? x[k].get(e) - m : 0.f;
                d = fmaf(v, v, d);
            }
        const float rs = 1.f / sqrtf(R::sum(d, 0.f).x / n + a.eps);
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int e = 0; e < R::kWords; ++e) {
                float v = (x[k].get(e) - m) * rs;
                if (a.gamma) v *= gamma[k].w[e];
                if (a.beta) v += beta[k].w[e];
                x[k].put(e, v);
            }
        R::store((W *)a.y + r * a.ys, a.n, x);
        if (a.mean && R::lane() == 0) {
            a.mean[r] = m;
            a.rstd[r] = rs;
        }
    }
}

// 65536 x 768 bf16: 58 us, 5.2 TB/s (and 4 us for the sums of 512 parts).
// dx row by row, and the workgroup's share of dgamma and dbeta: each thread
// keeps its columns' sums over its group's rows, then the groups' are added in
// order through LDS.
template <class E, int LANES, int CHUNKS>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(NormArgs a) {
    using R = NormRow<E, LANES, CHUNKS>;
    using W = typename E::Word;
    __shared__ float sums[2][LANES * CHUNKS * R::kWords];
    typename R::Floats gamma[CHUNKS], dg[CHUNKS], db[CHUNKS];
    if (a.gamma) R::load(a.gamma, a.n, gamma);
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int e = 0; e < R::kWords; ++e) {
            if (!a.gamma) gamma[k].w[e] = 1.f;
            dg[k].w[e] = db[k].w[e] = 0.f;
        }
    const float per = 1.f / (float)a.n;
    const long long step = (long long)gridDim.x * R::kGroups;
    long long r = (long long)blockIdx.x * R::kGroups + R::group();
    typename R::Chunk next_x[CHUNKS], next_dy[CHUNKS];
    float next_m = 0.f, next_rs = 0.f;
    const auto fetch = [&](long long row) {
        R::load((const W *)a.x + row * a.xs, a.n, next_x);
        R::load((const W *)a.dy + row * a.dys, a.n, next_dy);
        next_m = a.mean[row];
        next_rs = a.rstd[row];
    };
    if (r < a.rows) fetch(r);
    for (; r < a.rows; r += step) {
        typename R::Chunk x[CHUNKS], dy[CHUNKS];
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            x[k] = next_x[k];
            dy[k] = next_dy[k];
        }
        const float m = next_m, rs = next_rs;
        if (r + step < a.rows) fetch(r + step);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int e = 0; e < R::kWords; ++e) {
                // Past the row's end dy is zero; h could be infinite there.
                const float d = dy[k].get(e), g = d * gamma[k].w[e];
                const float h = R::column(k) + e < a.n ? (x[k].get(e) - m) * rs : 0.f;
                dg[k].w[e] = fmaf(d, h, dg[k].w[e]);
                db[k].w[e] += d;
                s1 += g;
                s2 = fmaf(g, h, s2);
            }
        const float2 s = R::sum(s1, s2);
        s1 = s.x * per;
        s2 = s.y * per;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int e = 0; e < R::kWords; ++e)
                x[k].put(e, rs * (dy[k].get(e) * gamma[k].w[e] - s1 - (x[k].get(e) - m) * rs * s2));
        R::store((W *)a.y + r * a.ys, a.n, x);
    }
    if (!a.dgamma) return;
    for (int q = 0; q < R::kGroups; ++q) {
        if (R::group() == q)
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int e = 0; e < R::kWords; ++e) {
                    const int c = R::column(k) + e;
                    sums[0][c] = q ? sums[0][c] + dg[k].w[e] : dg[k].w[e];
                    sums[1][c] = q ? sums[1][c] + db[k].w[e] : db[k].w[e];
                }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * a.n; c += kThreads) {
        const float s = c < a.n ? sums[0][c] : sums[1][c - a.n];
        if (gridDim.x > 1) a.partial[(size_t)blockIdx.x * 2 * a.n + c] = s;
        else (c < a.n ? a.dgamma : a.dbeta - a.n)[c] = s;
    }
}

// Rows too long for a workgroup's registers: the row is read again for each
// step.  dx may overwrite x or dy, so the weights' sums have a kernel of their
// own, which runs first.
template <class E>
__global__ __launch_bounds__(kThreads) void norm_forward_long_kernel(NormArgs a) {
    using W = typename E::Word;
    using R = NormRow<E, kThreads, 1>;
    const long long r = blockIdx.x;
    const W *x = (const W *)a.x + r * a.xs;
    W *y = (W *)a.y + r * a.ys;
    float s = 0.f, d = 0.f;
    for (int c = threadIdx.x; c < a.n; c += kThreads) s += E::get(x[c]);
    const float m = R::sum(s, 0.f).x / (float)a.n;
    for (int c = threadIdx.x; c < a.n; c += kThreads) {
        const float v = E::get(x[c]) - m;
        d = fmaf(v, v, d);
    }
    const float rs = 1.f / sqrtf(R::sum(d, 0.f).x / (float)a.n + a.eps);
    for (int c = threadIdx.x; c < a.n; c += kThreads) {
        float v = (E::get(x[c]) - m) * rs;
        if (a.gamma) v *= a.gamma[c];
        if (a.beta) v += a.beta[c];
        y[c] = E::put(v);
    }
    if (a.mean && threadIdx.x == 0) {
        a.mean[r] = m;
        a.rstd[r] = rs;
    }
}

template <class E>
__global__ __launch_bounds__(kThreads) void norm_backward_long_kernel(NormArgs a) {
    using W = typename E::Word;
    using R = NormRow<E, kThreads, 1>;
    const long long r = blockIdx.x;
    const W *x = (const W *)a.x + r * a.xs, *dy = (const W *)a.dy + r * a.dys;
    W *dx = (W *)a.y + r * a.ys;
    const float m = a.mean[r], rs = a.rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.n; c += kThreads) {
        const float g = E::get(dy[c]) * (a.gamma ? a.gamma[c] : 1.f);
        s1 += g;
        s2 = fmaf(g, (E::get(x[c]) - m) * rs, s2);
    }
    const float2 s = R::sum(s1, s2);
    s1 = s.x / (float)a.n;
    s2 = s.y / (float)a.n;
    for (int c = threadIdx.x; c < a.n; c += kThreads) {
        const float g = E::get(dy[c]) * (a.gamma ? a.gamma[c] : 1.f), h = (E::get(x[c]) - m) * rs;
        dx[c] = E::put(rs * (g - s1 - h * s2));
    }
}

// Sums over every parts-th group of 4 rows; workgroup (column block, part).
template <class E>
__global__ __launch_bounds__(kThreads) void norm_weight_long_kernel(NormArgs a) {
    using W = typename E::Word;
    __shared__ float sum[2][4][64];
    const int t = threadIdx.x % 64, c = blockIdx.x * 64 + t, w = threadIdx.x / 64;
    float dg = 0.f, db = 0.f;
    if (c < a.n)
        for (long long r = 4ll * blockIdx.y + w; r < a.rows; r += 4ll * gridDim.y) {
            const float g = E::get(((const W *)a.dy)[r * a.dys + c]);
            dg = fmaf(g, (E::get(((const W *)a.x)[r * a.xs + c]) - a.mean[r]) * a.rstd[r], dg);
            db += g;
        }
    sum[0][w][t] = dg;
    sum[1][w][t] = db;
    __syncthreads();
    if (w > 1 || c >= a.n) return;
    const float(*q)[64] = sum[w];
    a.partial[(size_t)(2 * blockIdx.y + w) * a.n + c] = (q[0][t] + q[1][t]) + (q[2][t] + q[3][t]);
}

// Lanes of a row's group: the fewest of 16, 32, 64 and 256 that hold the row in
// at most four chunks each (0: none does).  Fewer lanes leave fewer of them
// without a chunk, need fewer steps to add up, and keep more of a row in flight
// per wave.  The backward pass of 16-bit types takes at most two chunks where
// four would leave less than four waves per SIMD: 9999 x 257 fp16 12.3 us with
// two, 14.9 with three; 65536 x 768 bf16 94 us with two, 58 with three.
int norm_lanes(long long rows, int n, int size, bool backward) {
    const int words = 16 / size, chunks = (n + words - 1) / words;
    for (int lanes : {16, 32, 64})
        if (chunks <= 4 * lanes && (!backward || size == 4 || chunks <= 2 * lanes || rows * lanes >= 4096ll * kWave))
            return lanes;
    return chunks <= 4 * 256 ? 256 : 0;
}

template <class E, class F>
void with_row(int lanes, int n, F f) {
    const int words = 16 / E::kSize;
    const auto with_chunks = [&](auto l) {
        constexpr int L = decltype(l)::value;
        const int chunks = (n + L * words - 1) / (L * words);
        if (chunks <= 1) f(l, std::integral_constant<int, 1>{});
        else if (chunks == 2) f(l, std::integral_constant<int, 2>{});
        else if (chunks == 3) f(l, std::integral_constant<int, 3>{});
        else f(l, std::integral_constant<int, 4>{});
    };
    if (lanes == 16) with_chunks(std::integral_constant<int, 16>{});
    else if (lanes == 32) with_chunks(std::integral_constant<int, 32>{});
    else if (lanes == 64) with_chunks(std::integral_constant<int, 64>{});
    else with_chunks(std::integral_constant<int, 256>{});
}

// Workgroups for rows of `groups` groups each: eight per CU, which walk the rest.
long long norm_grid(long long rows, int groups) {
    const long long grid = (rows + groups - 1) / groups;
    return grid < 2048 ? grid : 2048;
}

// Partial sums of the weights' gradients: one per workgroup of the backward
// pass, at most two workgroups per CU (more of them wait less for memory, but
// their sums have to be written and read again).
long long norm_parts(long long rows, int n, int size) {
    const int lanes = norm_lanes(rows, n, size, true);
    const long long parts = lanes ? (rows + kThreads / lanes - 1) / (kThreads / lanes) : (rows + 3) / 4, most = lanes ? 512 : 64;
    return parts < most ? parts : most;
}

bool bad_norm(int type, long long rows, int n) {
    return type < BFHIP_F32 || type > BFHIP_BF16 || rows < 0 || n <= 0 || n > kMaxFeatures;
}

}  // namespace

extern "C" int bfhip_layer_norm_forward(int type, const void *x, long long x_stride, const float *gamma, const float *beta,
                                        void *y, long long y_stride, float *mean, float *rstd, long long rows,
                                        int features, float eps, void *stream, char *error, size_t cap) {
    if (bad_norm(type, rows, features) || !(eps >= 0.f) || !mean != !rstd)
        return fail(error, cap, "invalid layer norm contract");
    if (rows == 0) return 1;
    if (!x || !y || (rows > 1 && (x_stride < 0 || y_stride < features)))
        return fail(error, cap, "invalid layer norm contract");
    NormArgs a{};
    a.x = x; a.xs = x_stride;
    a.y = y; a.ys = y_stride;
    a.gamma = gamma; a.beta = beta;
    a.mean = mean; a.rstd = rstd;
    a.rows = rows; a.n = features; a.eps = eps;
    hipStream_t s = (hipStream_t)stream;
    int ok = 1;
    with_element(type, [&](auto e) {
        using E = decltype(e);
        const int row_lanes = norm_lanes(rows, features, E::kSize, false);
        if (!row_lanes) {
            ok = launch_fits(rows, kThreads);
            if (ok) hipLaunchKernelGGL(norm_forward_long_kernel<E>, dim3((unsigned)rows), dim3(kThreads), 0, s, a);
            return;
        }
        with_row<E>(row_lanes, features, [&](auto lanes, auto chunks) {
            constexpr int L = decltype(lanes)::value, K = decltype(chunks)::value;
            hipLaunchKernelGGL((norm_forward_kernel<E, L, K>), dim3((unsigned)norm_grid(rows, kThreads / L)), dim3(kThreads),
                               0, s, a);
        });
    });
    if (!ok) return fail(error, cap, "layer norm has too many rows");
    return launch_ok(error, cap, "layer norm launch");
}

extern "C" size_t bfhip_layer_norm_backward_workspace(long long rows, int features) {
    if (bad_norm(BFHIP_F32, rows, features)) return 0;
    // The type that needs more.
    const long long a = norm_parts(rows, features, 4), b = norm_parts(rows, features, 2);
    return (size_t)(a > b ? a : b) * 2 * features * sizeof(float);
}

extern "C" int bfhip_layer_norm_backward(int type, const void *dy, long long dy_stride, const void *x, long long x_stride,
                                         const float *gamma, const float *mean, const float *rstd, void *dx,
                                         long long dx_stride, float *dgamma, float *dbeta, long long rows, int features,
                                         void *workspace, size_t workspace_bytes, void *stream, char *error, size_t cap) {
    if (bad_norm(type, rows, features) || !dgamma != !dbeta)
        return fail(error, cap, "invalid layer norm contract");
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx ||
                     (rows > 1 && (dy_stride < 0 || x_stride < 0 || dx_stride < features))))
        return fail(error, cap, "invalid layer norm contract");
    if (dgamma && rows && (!workspace || ((uintptr_t)workspace & 15) ||
                           workspace_bytes < bfhip_layer_norm_backward_workspace(rows, features)))
        return fail(error, cap, "layer norm workspace too small or not 16-byte aligned");
    NormArgs a{};
    a.x = x; a.xs = x_stride;
    a.dy = dy; a.dys = dy_stride;
    a.y = dx; a.ys = dx_stride;
    a.gamma = gamma;
    a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd);
    a.partial = (float *)workspace;
    a.dgamma = dgamma; a.dbeta = dbeta;
    a.rows = rows; a.n = features;
    hipStream_t s = (hipStream_t)stream;
    long long parts = 0;
    int ok = 1;
    if (rows) with_element(type, [&](auto e) {
        using E = decltype(e);
        parts = norm_parts(rows, features, E::kSize);
        const int row_lanes = norm_lanes(rows, features, E::kSize, true);
        if (!row_lanes) {
            ok = launch_fits(rows, kThreads);
            if (!ok) return;
            if (dgamma)
                hipLaunchKernelGGL(norm_weight_long_kernel<E>, dim3((features + 63) / 64, (unsigned)parts), dim3(kThreads), 0,
                                   s, a);
            hipLaunchKernelGGL(norm_backward_long_kernel<E>, dim3((unsigned)rows), dim3(kThreads), 0, s, a);
            return;
        }
        with_row<E>(row_lanes, features, [&](auto lanes, auto chunks) {
            constexpr int L = decltype(lanes)::value, K = decltype(chunks)::value;
            hipLaunchKernelGGL((norm_backward_kernel<E, L, K>), dim3((unsigned)parts), dim3(kThreads), 0, s, a);
        });
    });
    if (!ok) return fail(error, cap, "layer norm has too many rows");
    const bool one = parts == 1 && norm_lanes(rows, features, type == BFHIP_F32 ? 4 : 2, true);
    if (dgamma && !one) column_sum((const float *)workspace, parts, dgamma, dbeta, features, 2ll * features, s);
    return launch_ok(error, cap, "layer norm launch");
}
