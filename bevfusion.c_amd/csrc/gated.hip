// The gated linear of a feed-forward block, forward and backward
// (include/bfhip_transformer.h): small tiles, the gradients of the two products, and
// the entry points.
#include <algorithm>
#include <cmath>

#include "gated.h"

using namespace bfhip;

namespace {

// Small and low tiles, where there are too few large ones.  `kStages` steps' tiles lie in
// LDS; while one is multiplied the others are on their way.  Small ones have two: two
// workgroups then share a CU and cover each other's waits, ways in and ways out.  (With
// four a workgroup is alone there: forward, 999 rows of 776 -> 2056 fp16, 264 tiles: 17
// us, 25 with four; both gradients of 512 rows of 2048 -> 5632 bf16: 74 and 102.)  With
// four they are `deep` ones, for tiles that are no more than the CUs and stream weights from
// memory (128 rows of 4096 -> 11008 bf16: 48 us, 60 with two).  Low ones have three, and share
// a CU by twos (64 rows of 4096 -> 11008 bf16: 41 us, 57 with two stages).
constexpr int kSmallStages = 2, kDeepStages = 4, kLowStages = 3;

template <class E, Form F, class S, int kStages>
constexpr int kProductLds = gated_lds<E, F, S>(kStages * S::kStage);

template <class E, Form F, class S, int kStages>
__device__ __forceinline__ void gated_product(const GatedArgs &a, int block, char *smem) {
    constexpr int kCopies = S::MTile::kIssue + S::NTile::kIssue;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const auto stage = [&](int t) { return smem + (uint32_t)t % kStages * S::kStage; };
    GatedWork<E, F, S> w;
    w.init(a, block, wave, lane);
    f32x4 acc[S::kMB][S::kNB];
#pragma unroll
    for (int j = 0; j < S::kMB; ++j)
#pragma unroll
        for (int i = 0; i < S::kNB; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) w.fetch(w.begin + s, stage(w.begin + s));
    for (int t = w.begin; t < w.end; ++t) {
        wait_vmcnt<(kStages - 2) * kCopies>();
        lds_barrier();  // this tile is there, and the one before has been read
        w.fetch(t + kStages - 1, stage(t + kStages - 1));
        const char *const ml = stage(t), *const nl = ml + S::MTile::kBytes;
#pragma unroll
        for (int kk = 0; kk < S::BK / 32; ++kk) {
            typename E::Frag nf[S::kNB], mf[S::kMB];
#pragma unroll
            for (int i = 0; i < S::kNB; ++i) nf[i] = S::NTile::frag(nl, w.n_at, i, kk);
#pragma unroll
            for (int j = 0; j < S::kMB; ++j) mf[j] = S::MTile::frag(ml, w.m_at, j, kk);
#pragma unroll
            for (int i = 0; i < S::kNB; ++i)
#pragma unroll
                for (int j = 0; j < S::kMB; ++j) acc[j][i] = E::mfma(nf[i], mf[j], acc[j][i]);
        }
    }
    wait_vmcnt<0>();
    lds_barrier();  // no copy and no read of a tile is left
    w.store(a, acc, smem, wave, lane);
}

template <class E, Form F, class S, int kStages>
__global__ __launch_bounds__(S::kThreads) void gated_product_kernel(GatedArgs a) {
    __shared__ __attribute__((aligned(512))) char smem[kProductLds<E, F, S, kStages>];
    gated_product<E, F, S, kStages>(a, blockIdx.x, smem);
}

template <class E, Form F>
using SmallShape = GatedShape<E, F, 128, 128, 2, 2>;
template <class E, Form F>
using LowShape = GatedShape<E, F, 64, 128, 1, 4>;

// Both gradients in one launch, the inputs' in the first `first` workgroups: neither
// fills the chip by itself.  (The whole backward pass with them in one launch and in two,
// bf16: 1024 rows of 512 -> 2048 31 and 39 us, 64 rows 14 and 18.)
template <class E, class S, int kStages, class W = SmallShape<E, kWeights>>
__global__ __launch_bounds__(S::kThreads) void gated_gradients_kernel(GatedArgs inputs, GatedArgs weights, int first) {
    static_assert(S::kThreads == W::kThreads, "one workgroup's size");
    __shared__ __attribute__((aligned(512))) char smem[std::max(kProductLds<E, kInputs, S, kStages>, kProductLds<E, kWeights, W, kSmallStages>)];
    const int block = blockIdx.x;
    if (block < first) gated_product<E, kInputs, S, kStages>(inputs, block, smem);
    else gated_product<E, kWeights, W, kSmallStages>(weights, block - first, smem);
}
template <class E, class S, class W = SmallShape<E, kWeights>>
__global__ __launch_bounds__(S::kThreads) void gated_gradients_join_kernel(GatedArgs inputs, GatedArgs weights, int first) {
    __shared__ __attribute__((aligned(16))) float smem[std::max(kJoinFloats<E, kInputs, S>, kJoinFloats<E, kWeights, W>)];
    const int block = blockIdx.x;
    if (block < first) gated_join<E, kInputs, S>(inputs, block, smem);
    else gated_join<E, kWeights, W>(weights, block - first, smem);
}

// ------------------------------------------------------------------ few rows
// Up to 16 MB rows: bound by reading both weights once (one row of 4096 -> 11008, bf16:
// 37 us, 4.9 TB/s), so these go from memory to the matrix cores without LDS.  A
// workgroup has 16 HB hidden elements; its waves take turns along the features, 64 at a
// time (a line of a 16-bit row), and their sums are added in order at the end.  The lanes
// of rows that are not there load nothing.
constexpr int kFewWaves = 8, kFewDeep = 64;

template <class E, int MB, int HB>
__global__ __launch_bounds__(kFewWaves *kWave) void gated_few_kernel(GatedArgs a) {
    constexpr int kSum = 2 * HB * MB * kWave;
    __shared__ f32x4 sums[kFewWaves][kSum];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), waves = blockDim.x / kWave;
    const int l16 = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16 * HB;
    using Word = typename E::Word;
    using Frag = typename E::Frag;
    const Word *w[2][HB], *x[MB];
#pragma unroll
    for (int b = 0; b < HB; ++b) {
        const long long r = min(n0 + 16 * b + l16, a.n - 1);  // (rows past the last one give results that are not stored)
        w[0][b] = (const Word *)(a.n_op.gate + r * a.n_op.stride);
        w[1][b] = (const Word *)(a.n_op.up + r * a.n_op.stride);
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) x[b] = (const Word *)(a.m_op.gate + (long long)min(16 * b + l16, a.m - 1) * a.m_op.stride);
    f32x4 acc[2][HB][MB];
#pragma unroll
    for (int b = 0; b < HB; ++b)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[0][b][m] = acc[1][b][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    // The fragments of 64 features.  Lane group g's k of the two products are 16
    // neighbours: any order will do that both operands have.
    struct Step {
        Frag x[2][MB], w[2][2][HB];
    };
    const auto fetch = [&](Step &f, int k, auto load) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = k + 16 * g + 8 * h;
#pragma unroll
            for (int b = 0; b < HB; ++b) {
                f.w[h][0][b] = load(w[0][b], at);
                f.w[h][1][b] = load(w[1][b], at);
            }
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                f.x[h][m] = Frag{};
                if (16 * m + l16 < a.m) f.x[h][m] = load(x[m], at);
            }
        }
    };
    const auto multiply = [&](const Step &f) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int b = 0; b < HB; ++b)
#pragma unroll
                for (int m = 0; m < MB; ++m) {
                    acc[0][b][m] = E::mfma(f.w[h][0][b], f.x[h][m], acc[0][b][m]);
                    acc[1][b][m] = E::mfma(f.w[h][1][b], f.x[h][m], acc[1][b][m]);
                }
    };
    const auto whole = [&](const Word *row, int k) {
        Frag f;
        __builtin_memcpy(&f, row + k, sizeof f);
        return f;
    };
    const auto ragged = [&](const Word *row, int k) {
        Words<E, 8> f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f.w[e] = k + e < a.k ? row[k + e] : (Word)0.f;
        return __builtin_bit_cast(Frag, f.w);
    };
    // kAhead steps' loads are in flight.
    constexpr int kAhead = E::kSize == 4 ? 2 : 4;
    const int stride = waves * kFewDeep, steps = a.k / kFewDeep;  // whole ones, the waves' in turn
    Step ring[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
        if (wave + s * waves < steps) fetch(ring[s], wave * kFewDeep + s * stride, whole);
    for (int s = wave; s < steps; s += kAhead * waves) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int now = s + i * waves, next = now + kAhead * waves;
            if (now < steps) multiply(ring[i]);
            if (next < steps) fetch(ring[i], next * kFewDeep, whole);
        }
    }
    if (steps * kFewDeep < a.k && steps % waves == wave) {
        fetch(ring[0], steps * kFewDeep, ragged);
        multiply(ring[0]);
    }
#pragma unroll
    for (int b = 0; b < HB; ++b)
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int u = 0; u < 2; ++u) sums[wave][((b * MB + m) * 2 + u) * kWave + lane] = acc[u][b][m];
    __syncthreads();
    for (int i = threadIdx.x; i < HB * MB * kWave; i += blockDim.x) {
        const int block = i / kWave, row = 16 * (block % MB) + (i & 15), n = n0 + 16 * (block / MB) + 4 * (i % kWave / 16);
        if (row >= a.m || n >= a.n) continue;
        const int at = block * 2 * kWave + i % kWave;
        f32x4 gate = sums[0][at], up = sums[0][at + kWave];
        for (int v = 1; v < waves; ++v) {
            gate += sums[v][at];
            up += sums[v][at + kWave];
        }
        f32x4 h;
        with_activation(a.activation, [&](auto kind) {
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = activate<E, decltype(kind)::value>(gate[e]) * up[e];
        });
        const auto put = [&](auto type, int o, const f32x4 &v) {
            using T = decltype(type);
            typename T::Word *p = (typename T::Word *)(a.out[o] + row * a.out_stride[o]) + n;
            Words<T, 4> w4;
#pragma unroll
            for (int e = 0; e < 4; ++e) w4.put(e, v[e]);
            if (n + 4 <= a.n) {
                w4.store(p);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < a.n) p[e] = w4.w[e];
            }
        };
        put(E{}, 0, h);
        if (a.out[1]) {
            put(ElemF32{}, 1, gate);
            put(ElemF32{}, 2, up);
        }
    }
}

// -------------------------------------------------------------------- alignment
constexpr int kChunkThreads = 256;

// The threads of `blocks` workgroups walk the chunks of eight elements in the rows' order
// (`per` a row): f(chunk, row, first element).
template <class G>
__device__ __forceinline__ void each_chunk(int block, int blocks, long long rows, int per, G f) {
    const long long step = (long long)blocks * kChunkThreads, first = (long long)block * kChunkThreads + threadIdx.x;
    const long long step_r = step / per;
    const int step_c = (int)(step % per);
    long long r = first / per;
    int c = (int)(first % per);
    for (long long i = first; r < rows; i += step) {
        f(i, r, 8 * c);
        r += step_r;
        c += step_c;
        if (c >= per) {
            c -= per;
            ++r;
        }
    }
}

// Rows of any alignment into rows of whole chunks, their ends filled with zeros (bound by
// memory: 999 and twice 2055 rows of 771, fp16: 5 us).
struct PadArgs {
    const char *from[3];
    char *to[3];
    long long stride[3];  // bytes
    long long rows[3];
    int length;
    int blocks;  // workgroups of each of the three
};

// The copies of workgroup `block`; false if it is none of theirs.
template <class E>
__device__ __forceinline__ bool gated_pad(const PadArgs &a, int block) {
    using Word = typename E::Word;
    if (block >= 3 * a.blocks) return false;
    const int i = block / a.blocks, per = (a.length + 7) / 8;
    if (!a.from[i]) return true;
    each_chunk(block % a.blocks, a.blocks, a.rows[i], per, [&](long long chunk, long long r, int c) {
        const Word *row = (const Word *)(a.from[i] + r * a.stride[i]) + c;
        Words<E, 8> v;
        if (c + 8 <= a.length) {
            v = Words<E, 8>::load(row);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v.w[e] = c + e < a.length ? row[e] : (Word)0.f;
        }
        v.store((Word *)a.to[i] + chunk * 8);
    });
    return true;
}

template <class E>
__global__ __launch_bounds__(kChunkThreads) void gated_pad_kernel(PadArgs a) {
    gated_pad<E>(a, blockIdx.x);
}

// ------------------------------------------------- gradients of the two products
struct SlopeArgs {
    const char *dh, *gate, *up;
    long long dh_stride, gate_stride, up_stride;  // bytes
    char *dg, *du;
    long long low;     // bytes from dg and du to what their rounding leaves, 0: nowhere
    long long stride;  // elements between the rows of dg and du
    long long rows;
    int hidden;
    float *most;  // fp16: the workgroups' largest |dg| and |du|
    int *shift;
};

constexpr int kMostGroups = 1024;

// dg and du of eight neighbouring elements; those past the row's end are zero.
template <class E, int kActivation>
__device__ __forceinline__ void slope8(const SlopeArgs &a, long long r, int c, float (&dg)[8], float (&du)[8]) {
    using Word = typename E::Word;
    const Word *dh = (const Word *)(a.dh + r * a.dh_stride) + c;
    const float *gate = (const float *)(a.gate + r * a.gate_stride) + c, *up = (const float *)(a.up + r * a.up_stride) + c;
    Words<E, 8> d;
    Words<ElemF32, 8> g, u;
    if (c + 8 <= a.hidden) {
        d = Words<E, 8>::load(dh);
        g = Words<ElemF32, 8>::load(gate);
        u = Words<ElemF32, 8>::load(up);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = c + e < a.hidden;
            d.w[e] = in ? dh[e] : (Word)0.f;
            g.w[e] = in ? gate[e] : 0.f;
            u.w[e] = in ? up[e] : 0.f;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float2 s = slope<E, kActivation>(g.get(e));
        dg[e] = d.get(e) * u.get(e) * s.y;
        du[e] = d.get(e) * s.x;
    }
}

// Largest finite |dg| and |du| of a workgroup's share.  (The first workgroups copy x and
// the weights, as the next kernel's do for other types.)
template <int kActivation>
__global__ __launch_bounds__(kChunkThreads) void gated_most_kernel(SlopeArgs a, PadArgs pad) {
    if (gated_pad<ElemF16>(pad, blockIdx.x)) return;
    const int block = blockIdx.x - 3 * pad.blocks, blocks = gridDim.x - 3 * pad.blocks;
    __shared__ float part[kChunkThreads / kWave];
    float most = 0.f;
    each_chunk(block, blocks, a.rows, (a.hidden + 7) / 8, [&](long long, long long r, int c) {
        float dg[8], du[8];
        slope8<ElemF16, kActivation>(a, r, c, dg, du);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            most = fmaxf(most, __builtin_isinf(dg[e]) ? 0.f : fabsf(dg[e]));
            most = fmaxf(most, __builtin_isinf(du[e]) ? 0.f : fabsf(du[e]));
        }
    });
    most = group_max<kWave>(most);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kChunkThreads / kWave; ++w) most = fmaxf(most, part[w]);
        a.most[block] = most;
    }
}

// The type's word next to v on zero's side.
template <class E>
__device__ __forceinline__ typename E::Word toward_zero(float v) {
    if constexpr (std::is_same_v<E, ElemF16>) return __builtin_bit_cast(_Float16, __builtin_amdgcn_cvt_pkrtz(v, 0.f)[0]);
    else return __builtin_bit_cast(typename E::Word, (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16));
}

// What that left of v, rounded to nearest: off by 2^-16 of v (bf16) or 2^-22 (fp16), and in
// fp16 by 2^-24.  It has v's sign and is nothing only where `taken` is, so that the two
// agree on what an infinite weight makes of them.
template <class E>
__device__ __forceinline__ typename E::Word left_of(float v, typename E::Word taken) {
    constexpr float least = std::is_same_v<E, ElemF16> ? 0x1p-24f : 0x1p-126f;
    const float most = E::get(taken), left = E::get(E::put(fabsf(most) < INFINITY ? v - most : 0.f));
    return E::put(left == 0.f && most != 0.f ? copysignf(least, v) : left);
}

// dg and du, rounded to the type; fp16's times a power of two that takes the
// largest of them to 2^14 or just above.  With `low` in two parts of one sign (then fp16's
// largest comes to 2^15, so that 2^-24 is as little of it).
// Bound by memory (8192 rows of 5632, bf16: 135 us, 4.8 TB/s).
template <class E, int kActivation>
__global__ __launch_bounds__(kChunkThreads) void gated_slope_kernel(SlopeArgs a, int groups, PadArgs pad) {
    if (gated_pad<E>(pad, blockIdx.x)) return;
    const int block = blockIdx.x - 3 * pad.blocks, blocks = gridDim.x - 3 * pad.blocks;
    int shift = 0;
    if constexpr (std::is_same_v<E, ElemF16>) {
        __shared__ float part[kChunkThreads / kWave];
        float most = 0.f;
        for (int i = threadIdx.x; i < groups; i += kChunkThreads) most = fmaxf(most, a.most[i]);
        most = group_max<kWave>(most);
        if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = most;
        __syncthreads();
        most = part[0];
        for (int w = 1; w < kChunkThreads / kWave; ++w) most = fmaxf(most, part[w]);
        if (most > 0.f) shift = (a.low ? 15 : 14) - ilogbf(most);
        if (block == 0 && threadIdx.x == 0) *a.shift = shift;
    }
    each_chunk(block, blocks, a.rows, (int)(a.stride / 8), [&](long long i, long long r, int c) {
        float dg[8], du[8];
        slope8<E, kActivation>(a, r, c, dg, du);
        Words<E, 8> x, y;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dg[e] = shift ? ldexpf(dg[e], shift) : dg[e];
            du[e] = shift ? ldexpf(du[e], shift) : du[e];
            x.put(e, dg[e]);
            y.put(e, du[e]);
        }
        if constexpr (E::kSize == 2) {
            if (a.low) {
                Words<E, 8> left_x, left_y;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x.w[e] = toward_zero<E>(dg[e]);
                    y.w[e] = toward_zero<E>(du[e]);
                    left_x.w[e] = left_of<E>(dg[e], x.w[e]);
                    left_y.w[e] = left_of<E>(du[e], y.w[e]);
                }
                left_x.store((typename E::Word *)(a.dg + a.low) + i * 8);
                left_y.store((typename E::Word *)(a.du + a.low) + i * 8);
            }
        }
        x.store((typename E::Word *)a.dg + i * 8);
        y.store((typename E::Word *)a.du + i * 8);
    });
}

// ------------------------------------------------------------------ the host
constexpr long long kPartBytes = 128ll << 20;  // of one product's sums

bool bad_gated(const bfhip_gated_desc *d) {
    // (tiles past the last row are counted in an int, and a tile's rows in 32-bit offsets)
    const long long most_rows = 0x7fff0000, most = 1 << 20, elements = 1ll << 40;
    return !d || d->type < BFHIP_F32 || d->type > BFHIP_BF16 || d->activation < BFHIP_SILU || d->activation > BFHIP_RELU ||
           d->rows < 0 || d->rows > most_rows || d->features < 1 || d->features > most || d->hidden < 1 || d->hidden > most ||
           d->rows * d->features > elements || d->rows * d->hidden > elements || d->features * d->hidden > elements;
}

// Rows of `length`.
bool bad_matrix(const bfhip_matrix *x, long long rows, long long length) {
    return !x || (rows && !x->data) || (rows > 1 && (x->stride < length || x->stride > 1ll << 40));
}

// Whether a matrix can be copied to LDS in chunks of 16 bytes.
bool chunked(const bfhip_matrix *x, long long rows, long long length, int size) {
    const long long words = 16 / size;
    return ((uintptr_t)x->data & 15) == 0 && length % words == 0 && (rows <= 1 || (x->stride % words == 0 && x->stride < 1 << 21));
}

enum GatedTiles { kSmall, kDeep, kLow, kLarge };

struct GatedPlan {
    GatedTiles kind;
    int tiles_m, tiles_n, whole, parts, per;
    size_t bytes;  // of the parts' sums
    double time;   // an estimate, in us
};

// Times in us that fit what products of 100 random sizes took to a tenth or so.
struct GatedTimes {
    int resident;  // workgroups that a CU holds at once
    double step;   // of the contraction, where a CU always has one to multiply
    double alone;  // a step where it waits for its tiles
    double ends;   // the way into a tile and out of it
};

// Tiles in rounds of as many workgroups as the chip holds; those of the last round may
// be split along the contraction, whichever number of parts is estimated to take least.
// `least`: the time that the operands' way from memory takes at least, in us.
template <class S>
GatedPlan plan_tiles(GatedTiles kind, Form f, long long m, long long n, long long k, int passes, double least, const GatedTimes &c) {
    constexpr int kCus = 256;
    GatedPlan best{};
    best.kind = kind;
    best.tiles_m = (int)((m + S::BM - 1) / S::BM * (f == kWeights ? 2 : 1));
    best.tiles_n = (int)((n + S::kCols - 1) / S::kCols);
    const long long steps = (k + S::BK - 1) / S::BK * passes * (f == kInputs ? 2 : 1), tiles = (long long)best.tiles_m * best.tiles_n;
    const long long tile_bytes = (long long)S::BM * S::BN * sizeof(float), rest = tiles % (kCus * c.resident);
    const auto time = [&](long long groups, long long each) {
        const long long turns = (groups + kCus - 1) / kCus, rounds = (turns + c.resident - 1) / c.resident;
        return groups ? std::max(turns * (each * c.step + c.ends), rounds * each * c.alone + c.ends) : 0;
    };
    best.whole = (int)std::min(tiles, 0x7fffffffll);
    best.parts = 1;
    best.time = std::max(time(tiles, steps), least);
    for (const int p : {2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        const long long per = (steps + p - 1) / p, parts = per ? (steps + per - 1) / per : 0, bytes = parts * rest * tile_bytes;
        if (!rest || steps < 2 * p || bytes > kPartBytes) break;
        // (the launch that joins the parts: 4 us with the host's time for it, 0.17 a part, 4.2 TB/s)
        const double t = std::max(time(tiles - rest, steps) + time(rest * parts, per), least) + 4 + 0.17 * parts + bytes / 4.2e6;
        if (t >= best.time) continue;
        best.time = t;
        best.whole = (int)(tiles - rest);
        best.parts = (int)parts;
        best.per = (int)per;
        best.bytes = (size_t)bytes;
    }
    return best;
}

// Whether a launch holds a product's workgroups, and with another product's beside them.
bool gated_fits(const GatedPlan &p) {
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    return tiles <= 0x7fffffff && launch_fits(p.whole + (tiles - p.whole) * p.parts, 512);
}

// Large, small, deep or low tiles (deep and large ones of 16-bit types, deep and low ones
// where rows of m are contiguous along k), whichever are estimated to take the least
// time.  passes: 2 where what the rounding of the slopes left is taken too (not by large
// tiles), 1 otherwise.
template <class E, Form F>
GatedPlan gated_plan(long long m, long long n, long long k, int passes = 1, bool large = true) {
    constexpr bool kHalf = E::kSize == 2;
    const double least = (double)k * ((F == kForward ? 1 : 2) * m + (F == kWeights ? 1 : 2) * n) * E::kSize / 4.8e6;
    GatedPlan best{};
    const auto take = [&](auto shape, GatedTiles kind, const GatedTimes &c) {
        const GatedPlan p = plan_tiles<decltype(shape)>(kind, F, m, n, k, passes, least, c);
        // (a launch that holds its tiles before one that does not)
        if (!best.parts || gated_fits(p) > gated_fits(best) || (gated_fits(p) == gated_fits(best) && p.time < best.time)) best = p;
    };
    take(SmallShape<E, F>{}, kSmall, kHalf ? GatedTimes{2, 0.56, 0.74, 1.4} : GatedTimes{2, 1.9, 2.17, 1.95});
    if constexpr (F != kWeights) take(LowShape<E, F>{}, kLow, kHalf ? GatedTimes{2, 0.41, 0.45, 1.0} : GatedTimes{2, 1.06, 1.22, 1.45});
    if constexpr (kHalf && F != kWeights) take(SmallShape<E, F>{}, kDeep, GatedTimes{1, 0.64, 0.64, 3.0});
    if constexpr (kHalf) {
        if (large && passes == 1) take(LargeShape<E, F>{}, kLarge, GatedTimes{1, 1.18, 1.18, 6.8});
    }
    return best;
}

// A product's workgroups, and of those the tiles that are split.
struct GatedGrid {
    long long groups, split;
};

GatedGrid gated_deal(GatedArgs &a, const GatedPlan &p) {
    a.tiles_m = p.tiles_m;
    a.tiles_n = p.tiles_n;
    a.whole = p.whole;
    a.parts = p.parts;
    a.per = p.per;
    const long long split = (long long)p.tiles_m * p.tiles_n - p.whole;
    return {p.whole + split * p.parts, split};
}

template <int kStages>
using Stages = std::integral_constant<int, kStages>;

template <class E, Form F>
void gated_launch(GatedArgs a, const GatedPlan &p, hipStream_t s) {
    const GatedGrid g = gated_deal(a, p);
    const auto run = [&](auto shape, auto stages) {
        using S = decltype(shape);
        hipLaunchKernelGGL((gated_product_kernel<E, F, S, decltype(stages)::value>), dim3((unsigned)g.groups), dim3(S::kThreads), 0, s, a);
        if (g.split) hipLaunchKernelGGL((gated_join_kernel<E, F, S>), dim3((unsigned)(g.split * S::kMB)), dim3(S::kThreads), 0, s, a);
    };
    if constexpr (E::kSize == 2) {
        if (p.kind == kLarge) {
            launch_gated_large<E, F>(a, g.groups, s);
            return;
        }
        if constexpr (F != kWeights) {
            if (p.kind == kDeep) {
                run(SmallShape<E, F>{}, Stages<kDeepStages>{});
                return;
            }
        }
    }
    if constexpr (F != kWeights) {
        if (p.kind == kLow) {
            run(LowShape<E, F>{}, Stages<kLowStages>{});
            return;
        }
    }
    run(SmallShape<E, F>{}, Stages<kSmallStages>{});
}

// Both gradients, none of them by large tiles (deep ones share CUs here: they are small).
template <class E>
void gated_gradients(GatedArgs inputs, const GatedPlan &pi, GatedArgs weights, const GatedPlan &pw, hipStream_t s) {
    const GatedGrid gi = gated_deal(inputs, pi), gw = gated_deal(weights, pw);
    const auto run = [&](auto shape, auto stages) {
        using S = decltype(shape);
        hipLaunchKernelGGL((gated_gradients_kernel<E, S, decltype(stages)::value>), dim3((unsigned)(gi.groups + gw.groups)), dim3(S::kThreads), 0, s, inputs, weights, (int)gi.groups);
        const long long ji = gi.split * S::kMB, jw = gw.split * SmallShape<E, kWeights>::kMB;
        if (ji + jw) hipLaunchKernelGGL((gated_gradients_join_kernel<E, S>), dim3((unsigned)(ji + jw)), dim3(S::kThreads), 0, s, inputs, weights, (int)ji);
    };
    if (pi.kind == kLow) run(LowShape<E, kInputs>{}, Stages<kLowStages>{});
    else run(SmallShape<E, kInputs>{}, Stages<kSmallStages>{});
}

// Whether a forward pass goes by the kernel for few rows: up to 16, or up to 32 where the
// weights are small.  us, few or tiles (rows that lie on 16 bytes: others would be copied for the
// tiles):
//              1 row       8           16          17          32
//   bf16 1024 -> 4096   5.8, 10.0   6.1,  9.8   6.3,  9.7   8.9,  9.7   9.3,  9.8
//        2048 -> 5632  13.2, 14.9  13.5, 14.4  14.5, 14.4  15.1, 14.6  15.2, 14.5
//        4096 -> 11008 35.3, 37.5  41.0, 36.0  46.1, 40.7
//   fp32 512 -> 2048    5.5, 16.6   5.8, 15.8   6.0, 16.0  10.5, 16.8  11.1, 16.0
//        2048 -> 5632  28.0, 41.1  30.0, 40.3  32.0, 40.5
//        4096 -> 11008 82.9, 116   82.9, 115   91.9, 115
// So 4 to 16 rows of large 16-bit weights would be 5 to 13 % faster by tiles: each of the few
// kernel's workgroups reads all of x for 16 hidden elements.
bool few_rows(const bfhip_gated_desc *d) {
    return d->rows <= 16 || (d->rows <= 32 && d->features * d->hidden <= (d->type == BFHIP_F32 ? 4 : 12) << 20);
}

// Few rows.  Eight waves a workgroup where workgroups of four would leave CUs idle.
template <class E>
void gated_few_launch(const GatedArgs &a, hipStream_t s) {
    const auto run = [&](auto rows, auto cols) {
        constexpr int MB = decltype(rows)::value, HB = decltype(cols)::value;
        const long long grid = ((long long)a.n + 16 * HB - 1) / (16 * HB);
        const int waves = grid < 512 ? kFewWaves : 4;
        hipLaunchKernelGGL((gated_few_kernel<E, MB, HB>), dim3((unsigned)grid), dim3(waves * kWave), 0, s, a);
    };
    if (a.m <= 16) run(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
}

// dg and du: rows of whole 16-byte chunks.
long long slope_stride(const bfhip_gated_desc *d) { return (d->hidden + 7) / 8 * 8; }

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Where x and the weights lie for the products: as they are, or in the workspace in
// rows of whole chunks.
struct Aligned {
    bfhip_matrix x, gate, up;
    size_t bytes;
    PadArgs pad;

    Aligned(const bfhip_gated_desc *d, const bfhip_matrix *x_, const bfhip_matrix *gate_, const bfhip_matrix *up_, char *work)
        : x(*x_), gate(*gate_), up(*up_), bytes(0), pad{} {
        const int size = d->type == BFHIP_F32 ? 4 : 2;
        const long long length = (d->features + 7) / 8 * 8;
        pad.length = (int)d->features;
        int i = 0;
        const auto move = [&](bfhip_matrix &m, long long rows) {
            pad.from[i] = (const char *)m.data;
            pad.to[i] = work + bytes;
            pad.stride[i] = rows > 1 ? m.stride * size : 0;
            pad.rows[i++] = rows;
            m = bfhip_matrix{work + bytes, length};
            bytes += up256((size_t)rows * length * size);
        };
        if (!chunked(x_, d->rows, d->features, size)) move(x, d->rows);
        if (!chunked(gate_, d->hidden, d->features, size) || !chunked(up_, d->hidden, d->features, size)) {
            move(gate, d->hidden);  // (both: they have one stride)
            move(up, d->hidden);
        }
        const long long most = std::max({pad.rows[0], pad.rows[1], pad.rows[2]}) * ((pad.length + 7) / 8);
        pad.blocks = (int)std::min<long long>(4096, (most + kChunkThreads - 1) / kChunkThreads);
    }
};

// Up to this many slopes (rows * hidden) enter the products in two parts, the type's word
// next to them on zero's side and what that left.  Of many slopes the roundings average out to
// about the error that the results' own rounding has (together 0.0023 of the gradients' norm in
// bf16, 0.0017 in two parts); of few one or two large ones can make it more.  So few products
// are bound by their launches and the weights: the backward pass of 16 rows of 1024 -> 1024 bf16
// 14.3 us, 11.7 without; one row of 4096 -> 11008 104 and 90.  Many would pay for it: a training
// step of 999 rows of 771 -> 2055 fp16 93 us instead of 75, of 8192 rows of 2048 -> 5632 bf16
// 1980 instead of 1060.
constexpr long long kFewSlopes = 1 << 14;

struct BackwardPlan {
    GatedPlan inputs, weights;
    bool together;  // in one launch, where both are wanted
    size_t slope, slopes;  // bytes of dg, and of all that is kept of dg and du
    size_t parts;          // of the two products' parts
    long long low;         // from dg and du to what their rounding left, or 0
    size_t all() const { return slopes + parts + up256((kMostGroups + 64) * sizeof(float)); }
};

BackwardPlan backward_plan(const bfhip_gated_desc *d) {
    BackwardPlan b{};
    with_element(d->type, [&](auto e) {
        using E = decltype(e);
        const int passes = E::kSize == 2 && d->rows * d->hidden <= kFewSlopes ? 2 : 1;
        const auto plan = [&](bool large) {
            b.inputs = gated_plan<E, kInputs>(d->rows, d->features, d->hidden, passes, large);
            b.weights = gated_plan<E, kWeights>(d->hidden, d->features, d->rows, passes, large);
            return b.inputs.time + b.weights.time;
        };
        // (one launch takes about 6 us less than two: see gated_gradients_kernel)
        const double one = plan(false) - 6;
        const bool held = gated_fits(b.inputs) && gated_fits(b.weights);
        b.together = true;
        if (plan(true) < one || !held) b.together = b.inputs.kind != kLarge && b.weights.kind != kLarge;
        else plan(false);
        b.slope = up256((size_t)d->rows * slope_stride(d) * E::kSize);
        b.slopes = 2 * passes * b.slope;
        b.low = passes > 1 ? 2 * b.slope : 0;
        b.parts = up256(b.inputs.bytes) + up256(b.weights.bytes);
    });
    return b;
}

size_t forward_parts(const bfhip_gated_desc *d) {
    size_t n = 0;
    with_element(d->type, [&](auto e) { n = gated_plan<decltype(e), kForward>(d->rows, d->hidden, d->features).bytes; });
    return up256(n);
}

bool bad_inputs(const bfhip_gated_desc *d, const bfhip_matrix *x, const bfhip_matrix *w_gate, const bfhip_matrix *w_up) {
    return bad_matrix(x, d->rows, d->features) || bad_matrix(w_gate, d->hidden, d->features) ||
           bad_matrix(w_up, d->hidden, d->features) || (d->hidden > 1 && w_gate->stride != w_up->stride);
}

// A single row, whose stride is of no account, takes that of a matrix without gaps, so that
// a tile's further rows lie past its end as the last rows of other matrices do.
GatedOperand operand(const bfhip_matrix *gate, const bfhip_matrix *up, long long rows, long long length, int size) {
    const long long stride = rows > 1 ? gate->stride : (length + 7) / 8 * 8;
    return GatedOperand{(const char *)gate->data, (const char *)up->data, stride * size};
}

}  // namespace

extern "C" size_t bfhip_gated_linear_workspace(const bfhip_gated_desc *d, const bfhip_matrix *x, const bfhip_matrix *w_gate,
                                               const bfhip_matrix *w_up) {
    if (bad_gated(d) || bad_inputs(d, x, w_gate, w_up) || few_rows(d)) return 0;
    return Aligned(d, x, w_gate, w_up, nullptr).bytes + forward_parts(d);
}

extern "C" int bfhip_gated_linear(const bfhip_gated_desc *d, const bfhip_matrix *x, const bfhip_matrix *w_gate,
                                  const bfhip_matrix *w_up, const bfhip_matrix *h, const bfhip_matrix *gate,
                                  const bfhip_matrix *up, void *workspace, size_t workspace_bytes, void *stream, char *error,
                                  size_t cap) {
    if (bad_gated(d) || !gate != !up) return fail(error, cap, "invalid gated linear contract");
    if (bad_inputs(d, x, w_gate, w_up) || bad_matrix(h, d->rows, d->hidden) ||
        (gate && (bad_matrix(gate, d->rows, d->hidden) || bad_matrix(up, d->rows, d->hidden))))
        return fail(error, cap, "invalid gated linear matrices: strides of at least a row, one stride for both weights");
    if (!d->rows) return 1;
    const bool few = few_rows(d);
    GatedPlan p{};
    if (!few) with_element(d->type, [&](auto e) { p = gated_plan<decltype(e), kForward>(d->rows, d->hidden, d->features); });
    if (!few && !gated_fits(p)) return fail(error, cap, "gated linear has too many rows");
    const Aligned in(d, x, w_gate, w_up, (char *)workspace);
    const size_t need = few ? 0 : in.bytes + up256(p.bytes);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
        return fail(error, cap, "gated linear workspace too small or not 16-byte aligned");
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    GatedArgs a{};
    a.m_op = few ? operand(x, x, d->rows, d->features, size) : operand(&in.x, &in.x, d->rows, d->features, size);
    a.n_op = few ? operand(w_gate, w_up, d->hidden, d->features, size) : operand(&in.gate, &in.up, d->hidden, d->features, size);
    a.m = (int)d->rows;
    a.n = (int)d->hidden;
    a.k = (int)d->features;
    const bfhip_matrix *out[3] = {h, gate, up};
    for (int i = 0; i < (gate ? 3 : 1); ++i) {
        a.out[i] = (char *)out[i]->data;
        a.out_stride[i] = d->rows > 1 ? out[i]->stride * (i ? (int)sizeof(float) : size) : 0;
    }
    a.activation = d->activation;
    a.partial = (float *)((char *)workspace + in.bytes);
    hipStream_t s = (hipStream_t)stream;
    with_element(d->type, [&](auto e) {
        using E = decltype(e);
        if (few) {
            gated_few_launch<E>(a, s);
            return;
        }
        if (in.pad.blocks) hipLaunchKernelGGL(gated_pad_kernel<E>, dim3((unsigned)(3 * in.pad.blocks)), dim3(kChunkThreads), 0, s, in.pad);
        gated_launch<E, kForward>(a, p, s);
    });
    return launch_ok(error, cap, "gated linear launch");
}

extern "C" size_t bfhip_gated_linear_backward_workspace(const bfhip_gated_desc *d, const bfhip_matrix *x,
                                                        const bfhip_matrix *w_gate, const bfhip_matrix *w_up) {
    if (bad_gated(d) || bad_inputs(d, x, w_gate, w_up)) return 0;
    return Aligned(d, x, w_gate, w_up, nullptr).bytes + backward_plan(d).all();
}

extern "C" int bfhip_gated_linear_backward(const bfhip_gated_desc *d, const bfhip_matrix *dh, const bfhip_matrix *x,
                                           const bfhip_matrix *w_gate, const bfhip_matrix *w_up, const bfhip_matrix *gate,
                                           const bfhip_matrix *up, const bfhip_matrix *dx, const bfhip_matrix *dw_gate,
                                           const bfhip_matrix *dw_up, void *workspace, size_t workspace_bytes, void *stream,
                                           char *error, size_t cap) {
    if (bad_gated(d) || !dw_gate != !dw_up || (!dx && !dw_gate)) return fail(error, cap, "invalid gated linear contract");
    if (bad_inputs(d, x, w_gate, w_up) || bad_matrix(dh, d->rows, d->hidden) || bad_matrix(gate, d->rows, d->hidden) ||
        bad_matrix(up, d->rows, d->hidden) || (dx && bad_matrix(dx, d->rows, d->features)) ||
        (dw_gate && (bad_matrix(dw_gate, d->hidden, d->features) || bad_matrix(dw_up, d->hidden, d->features))))
        return fail(error, cap, "invalid gated linear matrices: strides of at least a row, one stride for both weights");
    if (!d->rows && !dw_gate) return 1;
    const BackwardPlan p = backward_plan(d);
    if ((dx && !gated_fits(p.inputs)) || (dw_gate && !gated_fits(p.weights))) return fail(error, cap, "gated linear has too many rows");
    char *work = (char *)workspace;
    const Aligned in(d, x, w_gate, w_up, work + p.all());
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < in.bytes + p.all())
        return fail(error, cap, "gated linear workspace too small or not 16-byte aligned");
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    const long long stride = slope_stride(d);
    SlopeArgs e{};
    const auto step = [&](const bfhip_matrix *t, long long rows, int bytes) { return rows > 1 ? t->stride * bytes : 0; };
    e.dh = (const char *)dh->data; e.dh_stride = step(dh, d->rows, size);
    e.gate = (const char *)gate->data; e.gate_stride = step(gate, d->rows, sizeof(float));
    e.up = (const char *)up->data; e.up_stride = step(up, d->rows, sizeof(float));
    e.dg = work;
    e.du = work + p.slope;
    e.low = p.low;
    e.stride = stride;
    e.rows = d->rows;
    e.hidden = (int)d->hidden;
    e.most = (float *)(work + p.slopes + p.parts);
    e.shift = (int *)(e.most + kMostGroups);
    const long long groups = std::min<long long>(kMostGroups, (d->rows * (stride / 8) + kChunkThreads - 1) / kChunkThreads);
    const long long grid = std::min<long long>(8192, (d->rows * (stride / 8) + kChunkThreads - 1) / kChunkThreads);
    const bfhip_matrix slopes_g{e.dg, stride}, slopes_u{e.du, stride};
    hipStream_t s = (hipStream_t)stream;
    with_element(d->type, [&](auto el) {
        using E = decltype(el);
        if (d->rows) {
            const int pads = 3 * in.pad.blocks;
            with_activation(d->activation, [&](auto kind) {
                constexpr int A = decltype(kind)::value;
                PadArgs pad = in.pad;
                if (d->type == BFHIP_F16) {
                    hipLaunchKernelGGL(gated_most_kernel<A>, dim3((unsigned)(groups + pads)), dim3(kChunkThreads), 0, s, e, pad);
                    pad.blocks = 0;
                }
                hipLaunchKernelGGL((gated_slope_kernel<E, A>), dim3((unsigned)(grid + 3 * pad.blocks)), dim3(kChunkThreads), 0, s, e, (int)groups, pad);
            });
        }
        GatedArgs a{};
        a.shift = d->type == BFHIP_F16 && d->rows ? e.shift : nullptr;
        a.m_op = operand(&slopes_g, &slopes_u, d->rows, stride, size);
        a.low = p.low;
        GatedArgs b = a;
        a.partial = (float *)(work + p.slopes);
        b.partial = (float *)(work + p.slopes + up256(p.inputs.bytes));
        if (dx) {
            a.n_op = operand(&in.gate, &in.up, d->hidden, d->features, size);
            a.m = (int)d->rows;
            a.n = (int)d->features;
            a.k = (int)d->hidden;
            a.out[0] = (char *)dx->data;
            a.out_stride[0] = step(dx, d->rows, size);
        }
        if (dw_gate) {
            b.n_op = operand(&in.x, &in.x, d->rows, d->features, size);
            b.m = (int)d->hidden;
            b.n = (int)d->features;
            b.k = (int)d->rows;
            b.out[0] = (char *)dw_gate->data;
            b.out[1] = (char *)dw_up->data;
            b.out_stride[0] = step(dw_gate, d->hidden, size);
            b.out_stride[1] = step(dw_up, d->hidden, size);
        }
        if (dx && dw_gate && d->rows && p.together) {
            gated_gradients<E>(a, p.inputs, b, p.weights, s);
        } else {
            if (dx && d->rows) gated_launch<E, kInputs>(a, p.inputs, s);
            if (dw_gate) gated_launch<E, kWeights>(b, p.weights, s);
        }
    });
    return launch_ok(error, cap, "gated linear launch");
}

extern "C" int bfhip_gated_linear_plan(const bfhip_gated_desc *d, int product, int plan[6], char *error, size_t cap) {
    if (bad_gated(d) || product < 0 || product > 2 || !plan) return fail(error, cap, "invalid gated plan contract");
    const auto put = [&](const GatedPlan &p) {
        plan[0] = p.kind;
        plan[1] = p.whole;
        plan[2] = (int)((long long)p.tiles_m * p.tiles_n - p.whole);
        plan[3] = p.parts;
    };
    std::fill(plan, plan + 6, 0);
    if (product) {
        const BackwardPlan b = backward_plan(d);
        put(product == 1 ? b.inputs : b.weights);
        plan[4] = b.together;
        plan[5] = b.low != 0;
    } else if (few_rows(d)) {
        plan[0] = kLarge + 1;
    } else {
        with_element(d->type, [&](auto e) { put(gated_plan<decltype(e), kForward>(d->rows, d->hidden, d->features)); });
    }
    return 1;
}
