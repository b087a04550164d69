// Learned position bias by buckets: a table spread over a map, and the table's
// gradient (include/bfhip_transformer.h).
#include "bfhip_transformer.h"
#include "column_sum.h"
#include "gemm_core.h"

using namespace bfhip;

namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kAhead = 4;  // quads of positions per thread

// Bound by writing heads x positions: a thread writes four neighbouring
// positions of a head as one float4.  The map is read once; a position's table
// row is read head by head from the caches (a table row is heads neighbours, so
// a line serves many heads).  16 heads x 1024 x 1024: 14 us, 4.8 TB/s written.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void bias_forward_kernel(const float *table, const int *map, float *bias,
                                                                int buckets, int heads, int per, long long n) {
    constexpr int N = VEC ? 4 : 1;
    const long long p = ((long long)blockIdx.x * kThreads + threadIdx.x) * N;
    if (p >= n) return;
    const int h0 = blockIdx.y * per, h1 = min(heads, h0 + per);
    long long row[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int b = map[p + e];
        row[e] = (unsigned)b < (unsigned)buckets ? (long long)b * heads : -1;
    }
#pragma unroll 4
    for (int h = h0; h < h1; ++h) {
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = row[e] >= 0 ? table[row[e] + h] : 0.f;
        if constexpr (VEC) *reinterpret_cast<float4 *>(bias + h * n + p) = make_float4(v[0], v[1], v[2], v[3]);
        else bias[h * n + p] = v[0];
    }
}

// Sums by bucket without atomics between lanes: a wave takes HEADS heads by
// 64 / HEADS quads of neighbouring positions at a time, and every lane adds
// into sums of its own (bucket by lane, in LDS), so each address is one lane's
// and the order of every sum is fixed (and a read and a write do: an LDS float
// atomic takes some 200 cycles per wave: 16 heads x 1024 x 1024 89 us with them).  LDS holds `range` buckets per wave; a
// table with more is walked in ranges, a workgroup each.  The lanes of a head
// and the waves are added up in order at the end: partial [parts][range x
// ranges][HEADS x head tiles], or the result where there is one part.
template <int HEADS, bool VEC>
__global__ __launch_bounds__(kThreads) void bias_backward_kernel(const float *dbias, const int *map, float *out,
                                                                 int buckets, int heads, int range, int waves,
                                                                 long long n) {
    constexpr int QUADS = kWave / HEADS;
    extern __shared__ float smem[];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int tiles = (heads + HEADS - 1) / HEADS, tile = blockIdx.y % tiles, b0 = blockIdx.y / tiles * range;
    const int count = min(range, buckets - b0);
    // Neighbouring lanes take neighbouring quads of one head.
    const int head = tile * HEADS + lane / QUADS, quad = lane % QUADS;
    float *const sums = smem + (size_t)wave * range * kWave + lane;
    for (int b = 0; b < count; ++b) sums[b * kWave] = 0.f;
    const float *const row = dbias + (size_t)min(head, heads - 1) * n;
    const long long step = (long long)gridDim.x * waves * QUADS * 4;
    for (long long p0 = ((long long)blockIdx.x * waves + wave) * QUADS * 4 + quad * 4; p0 < n; p0 += step * kAhead) {
        // Positions past the end are loaded from within it and add 0 to the
        // first bucket, as do those of other buckets: no lane branches.
        float v[kAhead][4];
        int at[kAhead][4];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const long long p = p0 + a * step;
            if constexpr (VEC) {
                const long long q = min(p, n - 4);
                const float4 f = *reinterpret_cast<const float4 *>(row + q);
                const int4 m = *reinterpret_cast<const int4 *>(map + q);
                v[a][0] = f.x, v[a][1] = f.y, v[a][2] = f.z, v[a][3] = f.w;
                at[a][0] = m.x, at[a][1] = m.y, at[a][2] = m.z, at[a][3] = m.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[a][e] = row[min(p + e, n - 1)];
                    at[a][e] = map[min(p + e, n - 1)];
                }
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned b = (unsigned)(at[a][e] - b0);
                const bool in = b < (unsigned)count && p0 + a * step + e < n;
                sums[(in ? b : 0) * kWave] += in ? v[a][e] : 0.f;
            }
    }
    __syncthreads();
    // Four threads per result, a quarter of its lanes each (from a place that
    // differs by bucket, so that a wave's reads lie on different banks).
    for (int i = threadIdx.x / 4; i < count * HEADS; i += blockDim.x / 4) {
        const int b = i / HEADS, h = i % HEADS, quarter = threadIdx.x % 4;
        float s = 0.f;
        for (int w = 0; w < waves; ++w)
#pragma unroll
            for (int q = 0; q < QUADS / 4; ++q)
                s += smem[((size_t)w * range + b) * kWave + h * QUADS + (4 * q + quarter + b) % QUADS];
        s = group_sum<4>(s);
        if (quarter == 0 && tile * HEADS + h < heads)
            out[((size_t)blockIdx.x * buckets + b0 + b) * heads + tile * HEADS + h] = s;
    }
}

// How a gradient is dealt: buckets per range and waves by the LDS they need;
// heads per wave, 16 or the fewest of 1 and 4 that hold them, so that the map is
// read once for them; and parts of a round of loads or more.  Where a workgroup
// per head gets through all positions in four rounds, one launch is all: heads
// one by one, and no parts.
struct BiasPlan {
    int lanes, range, waves, ranges, tiles, parts;
};

BiasPlan bias_plan(int buckets, int heads, long long positions) {
    constexpr int kLds = 128 << 10, kRow = kWave * sizeof(float);
    BiasPlan p{};
    p.lanes = heads == 1 ? 1 : heads <= 4 ? 4 : 16;
    p.range = buckets < kLds / kRow ? buckets : kLds / kRow;
    p.waves = kLds / (p.range * kRow);
    p.waves = p.waves < kWaves ? p.waves : kWaves;
    p.ranges = (buckets + p.range - 1) / p.range;
    const bool small = positions <= 4ll * p.waves * kWave * 4 * kAhead;
    if (small) p.lanes = 1;
    p.tiles = (heads + p.lanes - 1) / p.lanes;
    const long long round = (long long)p.waves * (kWave / p.lanes) * 4 * kAhead;
    const long long most = (positions + round - 1) / round;
    // Four workgroups per CU.
    long long parts = 1024 / ((long long)p.ranges * p.tiles);
    parts = parts < 1 ? 1 : parts;
    p.parts = (int)(small || most < 1 ? 1 : most < parts ? most : parts);
    return p;
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
    const bool vec = positions % 4 == 0 && !(((uintptr_t)bias | (uintptr_t)map) & 15);
    const long long threads = vec ? positions / 4 : positions, grid = (threads + kThreads - 1) / kThreads;
    if (!launch_fits(grid, kThreads)) return fail(error, cap, "position bias has too many positions");
    // Heads are split over workgroups while the grid leaves CUs without one.
    int parts = grid >= 1024 ? 1 : (int)(1024 / grid);
    parts = parts < heads ? parts : heads;
    parts = parts < 65535 ? parts : 65535;
    const int per = (heads + parts - 1) / parts;
    const dim3 blocks((unsigned)grid, (heads + per - 1) / per);
    if (vec)
        hipLaunchKernelGGL(bias_forward_kernel<true>, blocks, dim3(kThreads), 0, (hipStream_t)stream, table, map, bias,
                           buckets, heads, per, positions);
    else
        hipLaunchKernelGGL(bias_forward_kernel<false>, blocks, dim3(kThreads), 0, (hipStream_t)stream, table, map, bias,
                           buckets, heads, per, positions);
    return launch_ok(error, cap, "position bias launch");
}

extern "C" size_t bfhip_position_bias_backward_workspace(int buckets, int heads, long long positions) {
    if (bad_bias(buckets, heads, positions)) return 0;
    const BiasPlan p = bias_plan(buckets, heads, positions);
    return p.parts > 1 ? (size_t)p.parts * buckets * heads * sizeof(float) : 0;
}

extern "C" int bfhip_position_bias_backward(const float *dbias, const int *map, float *dtable, int buckets, int heads,
                                            long long positions, void *workspace, size_t workspace_bytes, void *stream,
                                            char *error, size_t cap) {
    if (bad_bias(buckets, heads, positions) || !dtable || (positions && (!dbias || !map)))
        return fail(error, cap, "invalid position bias contract");
    const BiasPlan p = bias_plan(buckets, heads, positions);
    const long long blocks = (long long)p.ranges * p.tiles;
    if (blocks > 65535) return fail(error, cap, "position bias has too many buckets and heads");
    const size_t need = bfhip_position_bias_backward_workspace(buckets, heads, positions);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
        return fail(error, cap, "position bias workspace too small or not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const bool vec = positions % 4 == 0 && !(((uintptr_t)dbias | (uintptr_t)map) & 15);
    float *const out = p.parts > 1 ? (float *)workspace : dtable;
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(p.parts, (unsigned)blocks), dim3(p.waves * kWave),
                           (size_t)p.waves * p.range * kWave * sizeof(float), s, dbias, map, out, buckets, heads, p.range,
                           p.waves, positions);
    };
    if (p.lanes == 1) launch(vec ? bias_backward_kernel<1, true> : bias_backward_kernel<1, false>);
    else if (p.lanes == 4) launch(vec ? bias_backward_kernel<4, true> : bias_backward_kernel<4, false>);
    else launch(vec ? bias_backward_kernel<16, true> : bias_backward_kernel<16, false>);
    const long long n = (long long)buckets * heads;
    if (p.parts > 1) column_sum(out, p.parts, dtable, dtable, n, n, s);
    return launch_ok(error, cap, "position bias launch");
}
