// The gated linear of a feed-forward block, forward and backward
// (include/bfhip_transformer.h).
//
// Three products share one tiled kernel, which multiplies a tile of m x n
// results over a contraction axis k:
//   forward        h = act(x Wg^T) * (x Wu^T)   m rows,   n hidden,   k features
//   inputs' grad.  dx = dg Wg + du Wu           m rows,   n features, k hidden, twice
//   weights' grad. dWg = dg^T x, dWu = du^T x   m hidden, n features, k rows
// An operand whose k is contiguous in memory (x and W forward, dg and du in dx)
// lies in LDS as rows of BK elements; one whose k is the row (W in dx, both in
// dW) as BK rows, and is read transposed.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention.h"

using namespace bfhip;

namespace {

enum Form { kForward, kInputs, kWeights };

struct GatedOperand {
    const char *gate, *up;  // one matrix each, or the same
    long long stride;       // bytes
};

struct GatedArgs {
    GatedOperand m_op, n_op;
    int m, n, k;     // of the result, and of the contraction (of one of its two halves)
    char *out[3];    // forward: h, gate, up; inputs: dx; weights: dWg, dWu
    long long out_stride[3];  // bytes
    const int *shift;         // fp16 gradients were multiplied by 2^shift
    int activation;
    int tiles_m, tiles_n;
    int parts, per;  // of the contraction's steps
    float *partial;  // parts > 1: accumulators, [part][tile][wave][block][lane][4]
};

// ---------------------------------------------------------------- activations
template <class E>
__device__ __forceinline__ float exp_of(float v) {
    if constexpr (E::kSize == 4) return expf(v);
    else return __expf(v);
}
template <class E>
__device__ __forceinline__ float over(float a, float b) {
    if constexpr (E::kSize == 4) return a / b;
    else return a * __builtin_amdgcn_rcpf(b);
}

// act(g); erfc keeps gelu's relative precision where it is small.
template <class E>
__device__ __forceinline__ float activate(int kind, float g) {
    if (kind == BFHIP_SILU) return over<E>(g, 1.f + exp_of<E>(-g));
    if (kind == BFHIP_GELU) return 0.5f * g * erfcf(-0.70710678118654752f * g);
    return g > 0.f ? g : g == g ? 0.f : g;
}

// act(g) and its derivative.
template <class E>
__device__ __forceinline__ float2 slope(int kind, float g) {
    if (kind == BFHIP_SILU) {
        const float s = over<E>(1.f, 1.f + exp_of<E>(-g)), rest = over<E>(1.f, 1.f + exp_of<E>(g));
        return make_float2(g * s, s * fmaf(g, rest, 1.f));
    }
    if (kind == BFHIP_GELU) {
        const float cdf = 0.5f * erfcf(-0.70710678118654752f * g);
        return make_float2(g * cdf, fmaf(g * 0.39894228040143268f, exp_of<E>(-0.5f * g * g), cdf));
    }
    return make_float2(g > 0.f ? g : g == g ? 0.f : g, g > 0.f ? 1.f : 0.f);
}

// ------------------------------------------------------------------- tiles
// One operand's tile of OUTER (m or n) x BK (k) elements in LDS.  DMA: rows start
// on 16 bytes and hold whole chunks of 16 bytes.
template <class E, int OUTER, int BK, int THREADS, bool COL, bool DMA>
struct GatedTile {
    using T = std::conditional_t<COL, AttnTile<E, OUTER>, AttnTile<E, BK>>;
    static constexpr int kRows = COL ? BK : OUTER, kWords = 16 / E::kSize;
    static constexpr int kBytes = kRows * T::kRow, kIssue = kRows * T::kChunks / THREADS;
    static_assert(kRows * T::kChunks % THREADS == 0, "whole chunks per thread");
    typedef uint32_t Chunk __attribute__((ext_vector_type(4)));

    // PAIR > 0: outer rows are PAIR / 2 of the gate's, PAIR / 2 of the up's in turn.
    template <int PAIR>
    __device__ __forceinline__ static int source(int r) { return PAIR ? r / PAIR * (PAIR / 2) + r % (PAIR / 2) : r; }

    // Rows that the threads' j-th chunks span; chunk j of a thread is chunk 0 moved
    // by j times as many (a multiple of the swizzle's period).
    static constexpr int kSpan = THREADS / T::kChunks;
    static_assert(kSpan % 16 == 0 && THREADS % T::kChunks == 0, "chunks repeat with the swizzle");
    uint32_t off;  // DMA: bytes of chunk 0 from the tile's first row
    int row, first;  // its row in the matrix, and its first element along the row
    Chunk held[DMA ? 1 : kIssue];
    const char *base_a, *base_b;
    long long stride;
    int wave, left, thread;

    // Row of the matrix at which the span j begins.
    template <int PAIR>
    __device__ __forceinline__ static constexpr int span_row(int j) { return source<PAIR>(j * kSpan); }

    // The tile from `outer0` on, of `count` outer elements in all.
    template <int PAIR>
    __device__ __forceinline__ void init(const GatedOperand &op, bool up, int outer0, int count) {
        static_assert(!PAIR || PAIR % (2 * kSpan) == 0 || kSpan % PAIR == 0, "a span is of one matrix or of whole pairs");
        thread = threadIdx.x;
        wave = __builtin_amdgcn_readfirstlane(thread / kWave);
        stride = op.stride;
        left = count - outer0;
        const long long at = COL ? (long long)outer0 * E::kSize : outer0 * op.stride;
        base_a = (PAIR || !up ? op.gate : op.up) + at;
        base_b = op.up + at;
        const int r = thread / T::kChunks, c = (thread % T::kChunks) ^ T::swizzle(r);
        row = source<PAIR>(r);
        first = c * kWords;
        off = (uint32_t)row * (uint32_t)stride + 16u * c;
    }
    // Whether the wave's j-th chunks are the second matrix's.
    template <int PAIR>
    __device__ __forceinline__ bool second(int j) const {
        if constexpr (PAIR == 0) return false;
        else return (j * kSpan + wave * kWave / T::kChunks) % PAIR >= PAIR / 2;
    }
    // Fetches the tile from k0 on, of k elements in all, out of the matrix at `a` (with
    // PAIR, the up's rows out of that at `b`).
    template <int PAIR>
    __device__ __forceinline__ void fetch(const char *a, const char *b, int k0, int k, char *lds) {
        const long long at = COL ? k0 * stride : (long long)k0 * E::kSize;
        const int rows = COL ? k - k0 : left, length = COL ? left : k - k0;  // what there is of the tile
        if constexpr (DMA) {
            const __amdgpu_buffer_rsrc_t ra = buffer_rsrc(a + at, kDmaOutOfRange - 1), rb = buffer_rsrc(b + at, kDmaOutOfRange - 1);
#pragma unroll
            for (int j = 0; j < kIssue; ++j) {
                const bool in = row + span_row<PAIR>(j) < rows && first < length;
                dma16(second<PAIR>(j) ? rb : ra, reinterpret_cast<bf16 *>(lds + (j * THREADS + wave * kWave) * 16),
                      in ? off + (uint32_t)span_row<PAIR>(j) * (uint32_t)stride : kDmaOutOfRange);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kIssue; ++j) {
                const int r = row + span_row<PAIR>(j), n = r < rows ? length - first : 0;
                const char *p = (second<PAIR>(j) ? b : a) + at + r * stride + first * E::kSize;
                Chunk v = {0, 0, 0, 0};
                if (n >= kWords) {
                    __builtin_memcpy(&v, p, 16);
                } else if (n > 0) {
                    typedef typename E::Word Row __attribute__((ext_vector_type(kWords)));
                    Row w = __builtin_bit_cast(Row, v);
#pragma unroll
                    for (int e = 0; e < kWords; ++e)
                        if (e < n) w[e] = ((const typename E::Word *)p)[e];
                    v = __builtin_bit_cast(Chunk, w);
                }
                held[j] = v;
            }
        }
    }
    __device__ __forceinline__ void put(char *lds) const {
        if constexpr (!DMA)
#pragma unroll
            for (int j = 0; j < kIssue; ++j) *reinterpret_cast<Chunk *>(lds + (j * THREADS + thread) * 16) = held[j];
    }
    // Where in the tile the lane reads the fragments of the outer elements from o0
    // on (a multiple of 64).
    __device__ __forceinline__ static uint32_t lane_at(int o0, int lane) {
        const int c16 = lane & 15, g = lane >> 4;
        if constexpr (!COL) {
            return (o0 + c16) * T::kRow + 16 * ((E::kSize == 2 ? g : 2 * g) ^ T::swizzle(c16));
        } else if constexpr (E::kSize == 2) {
            // (see col_frag: here the lane's k are neighbours)
            const int r = 8 * g + (c16 >> 2);
            return r * T::kRow + 16 * ((o0 / 8 + ((c16 & 3) >> 1)) ^ T::swizzle(r)) + 8 * (c16 & 1);
        } else {
            return 8 * g * T::kRow + 16 * ((o0 / 4 + (c16 >> 2)) ^ (8 * (g & 1))) + 4 * (c16 & 3);
        }
    }
    // Fragment i of 16 outer elements, k 32 kk ..+31: lane l holds outer element l & 15,
    // k 8 (l >> 4) ..+7.  Tiles start on 512 bytes and the swizzle is an exclusive or
    // of address bits, so that every fragment is one exclusive or away from the first.
    __device__ __forceinline__ static typename E::Frag frag(const char *lds, uint32_t at, int i, int kk) {
        const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)(lds) + at;
        if constexpr (!COL) {
            const uint32_t p = (base ^ 64u * kk) + i * 16 * T::kRow;
            if constexpr (E::kSize == 2) {
                return *(__attribute__((address_space(3))) const bf16x8 *)p;
            } else {
                static_assert(E::kSize == 2 || BK == 32, "one step of 32");
                const f32x4 a = *(__attribute__((address_space(3))) const f32x4 *)p;
                const f32x4 b = *(__attribute__((address_space(3))) const f32x4 *)(p ^ 16u);
                return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        } else if constexpr (E::kSize == 2) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4 *Ptr;
            // Four rows on, the swizzle differs in chunk bit 3.
            const uint32_t p = (base ^ 32u * i) + 32 * kk * T::kRow, q = (base ^ 32u * i ^ 128u) + (32 * kk + 4) * T::kRow;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)p), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)q);
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            f32x8 v;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = *(__attribute__((address_space(3))) const float *)((base ^ (64u * i ^ 16u * e)) + (32 * kk + e) * T::kRow);
            return v;
        }
    }
};

// BM x BN results by WM x WN waves.
template <class E, Form F, int BM_, int BN_, int WM_, int WN_, bool DMA_>
struct GatedShape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = 128 / E::kSize;
    static constexpr bool DMA = DMA_;
    static constexpr int kThreads = WM * WN * kWave, kM = BM / WM, kN = BN / WN, kMB = kM / 16, kNB = kN / 16;
    using MTile = GatedTile<E, BM, BK, kThreads, F == kWeights, DMA>;
    using NTile = GatedTile<E, BN, BK, kThreads, F != kForward, DMA>;
    static constexpr int kPair = F == kForward ? kN : 0;  // gate and up columns of a wave
    static constexpr int kCols = F == kForward ? BN / 2 : BN;
    static constexpr int kStage = MTile::kBytes + NTile::kBytes;
};

struct TileAt {
    int tm, tn;
};

// Tiles are dealt to the XCDs in runs, each of which walks groups of eight rows
// of tiles column by column, so that what runs together on an XCD's L2 shares
// its operands' panels.
__device__ __forceinline__ TileAt tile_at(int id, int tiles_m, int tiles_n) {
    constexpr int kGroup = 8;
    id = xcd_swizzle(id, tiles_m * tiles_n);
    const int group = id / (kGroup * tiles_n), first = group * kGroup, rows = min(kGroup, tiles_m - first);
    const int in = id - group * kGroup * tiles_n;
    return TileAt{first + in % rows, in / rows};
}

// Four neighbouring results of a row, of which `n` exist.
template <class E>
__device__ __forceinline__ void put4(char *row, int at, int n, const float *v) {
    typename E::Word *p = (typename E::Word *)row + at;
    if (n >= 4) {
        Words<E, 4> w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.put(e, v[e]);
        w.store(p);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) p[e] = E::put(v[e]);
    }
}

// A lane holds row m (of its block of 16) and four neighbouring columns.
template <class E, Form F, class S>
__device__ __forceinline__ void gated_store(const GatedArgs &a, const f32x4 (&acc)[S::kNB][S::kMB], TileAt at, int wave, int lane) {
    const int wm = wave / S::WN, wn = wave % S::WN, l16 = lane & 15, g = lane >> 4;
    const int tiles = F == kWeights ? a.tiles_m / 2 : a.tiles_m;
    const bool up = F == kWeights && at.tm >= tiles;
    const int m0 = (up ? at.tm - tiles : at.tm) * S::BM + wm * S::kM, n0 = at.tn * S::kCols + wn * (S::kPair ? S::kN / 2 : S::kN);
    const int shift = F != kForward && a.shift ? -*a.shift : 0;
#pragma unroll
    for (int j = 0; j < S::kMB; ++j) {
        const int m = m0 + 16 * j + l16;
        if (m >= a.m) continue;
        if constexpr (F == kForward) {
#pragma unroll
            for (int i = 0; i < S::kNB / 2; ++i) {
                const int n = n0 + 16 * i + 4 * g;
                if (n >= a.n) continue;
                const f32x4 gate = acc[i][j], up4 = acc[i + S::kNB / 2][j];
                float h[4], p[4], q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = gate[e];
                    q[e] = up4[e];
                    h[e] = activate<E>(a.activation, gate[e]) * up4[e];
                }
                put4<E>(a.out[0] + m * a.out_stride[0], n, a.n - n, h);
                if (a.out[1]) {
                    put4<E>(a.out[1] + m * a.out_stride[1], n, a.n - n, p);
                    put4<E>(a.out[2] + m * a.out_stride[2], n, a.n - n, q);
                }
            }
        } else {
            char *const row = (up ? a.out[1] : a.out[0]) + m * (up ? a.out_stride[1] : a.out_stride[0]);
#pragma unroll
            for (int i = 0; i < S::kNB; ++i) {
                const int n = n0 + 16 * i + 4 * g;
                if (n >= a.n) continue;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = std::is_same_v<E, ElemF16> ? ldexpf(acc[i][j][e], shift) : acc[i][j][e];
                put4<E>(row, n, a.n - n, v);
            }
        }
    }
}

template <class E, Form F, class S>
__global__ __launch_bounds__(S::kThreads) void gated_product_kernel(GatedArgs a) {
    __shared__ __attribute__((aligned(512))) char smem[2 * S::kStage];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave / S::WN, wn = wave % S::WN;
    const int tiles = a.tiles_m * a.tiles_n, part = blockIdx.x / tiles;
    const TileAt at = tile_at(blockIdx.x % tiles, a.tiles_m, a.tiles_n);
    const int half = F == kWeights ? a.tiles_m / 2 : a.tiles_m;
    const bool up = F == kWeights && at.tm >= half;
    typename S::MTile mt;
    typename S::NTile nt;
    mt.template init<0>(a.m_op, up, (up ? at.tm - half : at.tm) * S::BM, a.m);
    nt.template init<S::kPair>(a.n_op, up, at.tn * S::kCols, a.n);
    // The contraction's steps: for the inputs' gradient the gate's, then the up's.
    const int each = (a.k + S::BK - 1) / S::BK, steps = F == kInputs ? 2 * each : each;
    const int begin = part * a.per, end = min(steps, begin + a.per);
    const auto fetch = [&](int t) {
        const bool second = F == kInputs && t >= each;
        const int k0 = (second ? t - each : t) * S::BK;
        char *const to = smem + (t & 1) * S::kStage;
        mt.template fetch<0>(second ? mt.base_b : mt.base_a, mt.base_b, k0, a.k, to);
        nt.template fetch<S::kPair>(second ? nt.base_b : nt.base_a, nt.base_b, k0, a.k, to + S::MTile::kBytes);
    };
    f32x4 acc[S::kNB][S::kMB];
#pragma unroll
    for (int i = 0; i < S::kNB; ++i)
#pragma unroll
        for (int j = 0; j < S::kMB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto put = [&](int t) {
        char *const to = smem + (t & 1) * S::kStage;
        mt.put(to);
        nt.put(to + S::MTile::kBytes);
    };
    const uint32_t m_at = S::MTile::lane_at(wm * S::kM, lane), n_at = S::NTile::lane_at(wn * S::kN, lane);
    if (begin < end) {
        fetch(begin);
        put(begin);
    }
    for (int t = begin; t < end; ++t) {
        if constexpr (S::DMA) wait_vmcnt<0>();
        lds_barrier();  // this tile is there, and the one before has been read
        if (t + 1 < end) fetch(t + 1);
        const char *const ml = smem + (t & 1) * S::kStage, *const nl = ml + S::MTile::kBytes;
#pragma unroll
        for (int kk = 0; kk < S::BK / 32; ++kk) {
            typename E::Frag nf[S::kNB], mf[S::kMB];
#pragma unroll
            for (int i = 0; i < S::kNB; ++i) nf[i] = S::NTile::frag(nl, n_at, i, kk);
#pragma unroll
            for (int j = 0; j < S::kMB; ++j) mf[j] = S::MTile::frag(ml, m_at, j, kk);
#pragma unroll
            for (int i = 0; i < S::kNB; ++i)
#pragma unroll
                for (int j = 0; j < S::kMB; ++j) acc[i][j] = E::mfma(nf[i], mf[j], acc[i][j]);
        }
        if (t + 1 < end) put(t + 1);
    }
    if (a.parts > 1) {
        f32x4 *to = reinterpret_cast<f32x4 *>(a.partial) +
                    (((size_t)part * tiles + blockIdx.x % tiles) * S::WM * S::WN + wave) * S::kNB * S::kMB * kWave + lane;
#pragma unroll
        for (int i = 0; i < S::kNB; ++i)
#pragma unroll
            for (int j = 0; j < S::kMB; ++j) to[(i * S::kMB + j) * kWave] = acc[i][j];
        return;
    }
    gated_store<E, F, S>(a, acc, at, wave, lane);
}

// Adds up the parts' accumulators in order and stores the results.
template <class E, Form F, class S>
__global__ __launch_bounds__(S::kThreads) void gated_join_kernel(GatedArgs a) {
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int tiles = a.tiles_m * a.tiles_n;
    const TileAt at = tile_at(blockIdx.x, a.tiles_m, a.tiles_n);
    const f32x4 *from = reinterpret_cast<const f32x4 *>(a.partial) + ((size_t)blockIdx.x * S::WM * S::WN + wave) * S::kNB * S::kMB * kWave + lane;
    const size_t step = (size_t)tiles * S::WM * S::WN * S::kNB * S::kMB * kWave;
    f32x4 acc[S::kNB][S::kMB];
#pragma unroll
    for (int i = 0; i < S::kNB; ++i)
#pragma unroll
        for (int j = 0; j < S::kMB; ++j) acc[i][j] = from[(i * S::kMB + j) * kWave];
    for (int p = 1; p < a.parts; ++p) {
        from += step;
#pragma unroll
        for (int i = 0; i < S::kNB; ++i)
#pragma unroll
            for (int j = 0; j < S::kMB; ++j) acc[i][j] += from[(i * S::kMB + j) * kWave];
    }
    gated_store<E, F, S>(a, acc, at, wave, lane);
}

// ------------------------------------------------- gradients of the two products
struct SlopeArgs {
    const char *dh, *gate, *up;
    long long dh_stride, gate_stride, up_stride;  // bytes
    char *dg, *du;
    long long stride;  // elements between the rows of dg and du
    long long rows;
    int hidden, activation;
    float *most;  // fp16: the workgroups' largest |dg| and |du|
    int *shift;
};

constexpr int kSlopeThreads = 256, kMostGroups = 1024;

// dg and du of eight neighbouring elements; those past the row's end are zero.
template <class E>
__device__ __forceinline__ void slope8(const SlopeArgs &a, long long r, int c, float (&dg)[8], float (&du)[8]) {
    using Word = typename E::Word;
    const Word *dh = (const Word *)(a.dh + r * a.dh_stride) + c, *gate = (const Word *)(a.gate + r * a.gate_stride) + c;
    const Word *up = (const Word *)(a.up + r * a.up_stride) + c;
    Words<E, 8> d, g, u;
    if (c + 8 <= a.hidden) {
        d = Words<E, 8>::load(dh);
        g = Words<E, 8>::load(gate);
        u = Words<E, 8>::load(up);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = c + e < a.hidden;
            d.w[e] = in ? dh[e] : (Word)0.f;
            g.w[e] = in ? gate[e] : (Word)0.f;
            u.w[e] = in ? up[e] : (Word)0.f;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float2 s = slope<E>(a.activation, g.get(e));
        dg[e] = d.get(e) * u.get(e) * s.y;
        du[e] = d.get(e) * s.x;
    }
}

// Largest finite |dg| and |du| of a workgroup's share.
__global__ __launch_bounds__(kSlopeThreads) void gated_most_kernel(SlopeArgs a) {
    __shared__ float part[kSlopeThreads / kWave];
    const int per = (a.hidden + 7) / 8;
    const long long n = a.rows * per;
    float most = 0.f;
    for (long long i = (long long)blockIdx.x * kSlopeThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kSlopeThreads) {
        float dg[8], du[8];
        slope8<ElemF16>(a, i / per, (int)(i % per) * 8, dg, du);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            most = fmaxf(most, __builtin_isinf(dg[e]) ? 0.f : fabsf(dg[e]));
            most = fmaxf(most, __builtin_isinf(du[e]) ? 0.f : fabsf(du[e]));
        }
    }
    most = group_max<kWave>(most);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kSlopeThreads / kWave; ++w) most = fmaxf(most, part[w]);
        a.most[blockIdx.x] = most;
    }
}

// dg and du, rounded to the type; fp16's times a power of two that takes the
// largest of them to 2^14 or just above.
template <class E>
__global__ __launch_bounds__(kSlopeThreads) void gated_slope_kernel(SlopeArgs a, int groups) {
    int shift = 0;
    if constexpr (std::is_same_v<E, ElemF16>) {
        __shared__ float part[kSlopeThreads / kWave];
        float most = 0.f;
        for (int i = threadIdx.x; i < groups; i += kSlopeThreads) most = fmaxf(most, a.most[i]);
        most = group_max<kWave>(most);
        if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = most;
        __syncthreads();
        most = part[0];
        for (int w = 1; w < kSlopeThreads / kWave; ++w) most = fmaxf(most, part[w]);
        if (most > 0.f) shift = 14 - ilogbf(most);
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.shift = shift;
    }
    const int per = (int)(a.stride / 8);
    const long long n = a.rows * per;
    for (long long i = (long long)blockIdx.x * kSlopeThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kSlopeThreads) {
        const long long r = i / per;
        const int c = (int)(i - r * per) * 8;
        float dg[8], du[8];
        slope8<E>(a, r, c, dg, du);
        Words<E, 8> x, y;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x.put(e, shift ? ldexpf(dg[e], shift) : dg[e]);
            y.put(e, shift ? ldexpf(du[e], shift) : du[e]);
        }
        x.store((typename E::Word *)a.dg + i * 8);
        y.store((typename E::Word *)a.du + i * 8);
    }
}

// ------------------------------------------------------------------ the host
constexpr long long kPartBytes = 256ll << 20;

bool bad_gated(const bfhip_gated_desc *d) {
    const long long most = 0x7fffffff, elements = 1ll << 40;
    return !d || d->type < BFHIP_F32 || d->type > BFHIP_BF16 || d->activation < BFHIP_SILU || d->activation > BFHIP_RELU ||
           d->rows < 0 || d->rows > most || d->features < 1 || d->features > most || d->hidden < 1 || d->hidden > most ||
           d->rows * d->features > elements || d->rows * d->hidden > elements || d->features * d->hidden > elements;
}

// Rows of `length`.
bool bad_matrix(const bfhip_matrix *x, long long rows, long long length) {
    return !x || (rows && !x->data) || (rows > 1 && (x->stride < length || x->stride > 1ll << 40));
}

struct GatedPlan {
    bool big;
    int tiles_m, tiles_n, parts, per;
    size_t bytes;  // of the parts' sums
};

// Whether a matrix can be copied to LDS in chunks of 16 bytes.
bool chunks(const bfhip_matrix *x, long long rows, long long length, int size) {
    const long long words = 16 / size;
    return ((uintptr_t)x->data & 15) == 0 && length % words == 0 && (rows <= 1 || x->stride % words == 0) &&
           (rows <= 1 || x->stride < 1 << 21);
}

// Tiles, and where they are fewer than CUs the contraction's parts, of eight steps
// or more, as many as fill the CUs twice.
template <class S>
void plan_tiles(GatedPlan &p, Form f, long long m, long long n, long long k) {
    p.tiles_m = (int)((m + S::BM - 1) / S::BM * (f == kWeights ? 2 : 1));
    p.tiles_n = (int)((n + S::kCols - 1) / S::kCols);
    const long long steps = (k + S::BK - 1) / S::BK * (f == kInputs ? 2 : 1), tiles = (long long)p.tiles_m * p.tiles_n;
    const long long tile_bytes = (long long)S::BM * S::BN * sizeof(float);
    long long parts = p.big ? 1 : std::min({512 / std::max(1ll, tiles), steps / 8, kPartBytes / std::max(1ll, tiles * tile_bytes)});
    if (parts < 2) parts = 1;
    p.per = (int)((steps + parts - 1) / std::max(1ll, parts));
    if (p.per < 1) p.per = 1;
    p.parts = (int)std::max(1ll, (steps + p.per - 1) / p.per);
    p.bytes = p.parts > 1 ? (size_t)p.parts * tiles * tile_bytes : 0;
}

// The shapes: large tiles where there are enough of them to fill the chip, and
// only for matrices that are copied in whole chunks.
template <class E, Form F, bool DMA>
using SmallShape = GatedShape<E, F, 128, 128, 2, E::kSize == 4 ? 4 : 2, DMA>;
template <class E, Form F>
using BigShape = GatedShape<E, F, 256, 256, 2, 4, true>;

template <class E, Form F>
GatedPlan gated_plan(long long m, long long n, long long k, bool dma) {
    GatedPlan p{};
    const long long cols = F == kForward ? 128 : 256;
    p.big = dma && E::kSize == 2 && (m + 255) / 256 * ((n + cols - 1) / cols) * (F == kWeights ? 2 : 1) >= 192;
    if (p.big) plan_tiles<BigShape<ElemBf16, F>>(p, F, m, n, k);
    else plan_tiles<SmallShape<E, F, true>>(p, F, m, n, k);
    return p;
}

template <class E, Form F>
int gated_launch(GatedArgs a, const GatedPlan &p, bool dma, hipStream_t s) {
    a.tiles_m = p.tiles_m;
    a.tiles_n = p.tiles_n;
    a.parts = p.parts;
    a.per = p.per;
    const long long tiles = (long long)p.tiles_m * p.tiles_n, grid = tiles * p.parts;
    if (grid > 0x7fffffff || !launch_fits(grid, 512)) return 0;
    const auto run = [&](auto shape) {
        using S = decltype(shape);
        hipLaunchKernelGGL((gated_product_kernel<E, F, S>), dim3((unsigned)grid), dim3(S::kThreads), 0, s, a);
    };
    if constexpr (E::kSize == 2) {
        if (p.big) {
            run(BigShape<E, F>{});
            return 1;
        }
    }
    using Join = SmallShape<E, F, true>;
    if (dma) run(Join{});
    else run(SmallShape<E, F, false>{});
    if (p.parts > 1) hipLaunchKernelGGL((gated_join_kernel<E, F, Join>), dim3((unsigned)tiles), dim3(Join::kThreads), 0, s, a);
    return 1;
}

// dg and du: rows of whole 16-byte chunks.
long long slope_stride(const bfhip_gated_desc *d) { return (d->hidden + 7) / 8 * 8; }

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Bytes of a product's parts, whichever way its matrices are copied.
template <class E, Form F>
size_t part_bytes(long long m, long long n, long long k) {
    return std::max(gated_plan<E, F>(m, n, k, true).bytes, gated_plan<E, F>(m, n, k, false).bytes);
}

struct BackwardBytes {
    size_t slopes, parts;  // of each of dg and du, and of the larger of the products' parts
    size_t all() const { return 2 * slopes + parts + (kMostGroups + 64) * sizeof(float); }
};

BackwardBytes backward_bytes(const bfhip_gated_desc *d) {
    BackwardBytes b{};
    with_element(d->type, [&](auto e) {
        using E = decltype(e);
        b.slopes = up256((size_t)d->rows * slope_stride(d) * E::kSize);
        b.parts = up256(std::max(part_bytes<E, kInputs>(d->rows, d->features, d->hidden),
                                 part_bytes<E, kWeights>(d->hidden, d->features, d->rows)));
    });
    return b;
}

GatedOperand operand(const bfhip_matrix *gate, const bfhip_matrix *up, long long rows, int size) {
    return GatedOperand{(const char *)gate->data, (const char *)up->data, rows > 1 ? gate->stride * size : 0};
}

}  // namespace

extern "C" size_t bfhip_gated_linear_workspace(const bfhip_gated_desc *d) {
    if (bad_gated(d) || !d->rows) return 0;
    size_t n = 0;
    with_element(d->type, [&](auto e) { n = part_bytes<decltype(e), kForward>(d->rows, d->hidden, d->features); });
    return n;
}

extern "C" int bfhip_gated_linear(const bfhip_gated_desc *d, const bfhip_matrix *x, const bfhip_matrix *w_gate,
                                  const bfhip_matrix *w_up, const bfhip_matrix *h, const bfhip_matrix *gate,
                                  const bfhip_matrix *up, void *workspace, size_t workspace_bytes, void *stream, char *error,
                                  size_t cap) {
    if (bad_gated(d) || !gate != !up) return fail(error, cap, "invalid gated linear contract");
    if (bad_matrix(x, d->rows, d->features) || bad_matrix(w_gate, d->hidden, d->features) ||
        bad_matrix(w_up, d->hidden, d->features) || bad_matrix(h, d->rows, d->hidden) ||
        (gate && (bad_matrix(gate, d->rows, d->hidden) || bad_matrix(up, d->rows, d->hidden))))
        return fail(error, cap, "invalid gated linear matrices: strides of at least a row");
    if (d->hidden > 1 && w_gate->stride != w_up->stride) return fail(error, cap, "invalid gated linear matrices: the weights need one stride");
    if (!d->rows) return 1;
    const size_t need = bfhip_gated_linear_workspace(d);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
        return fail(error, cap, "gated linear workspace too small or not 16-byte aligned");
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    GatedArgs a{};
    a.m_op = operand(x, x, d->rows, size);
    a.n_op = operand(w_gate, w_up, d->hidden, size);
    a.m = (int)d->rows;
    a.n = (int)d->hidden;
    a.k = (int)d->features;
    const bfhip_matrix *out[3] = {h, gate, up};
    for (int i = 0; i < (gate ? 3 : 1); ++i) {
        a.out[i] = (char *)out[i]->data;
        a.out_stride[i] = d->rows > 1 ? out[i]->stride * size : 0;
    }
    a.activation = d->activation;
    a.partial = (float *)workspace;
    const bool dma = chunks(x, d->rows, d->features, size) && chunks(w_gate, d->hidden, d->features, size) &&
                     chunks(w_up, d->hidden, d->features, size);
    int ok = 1;
    with_element(d->type, [&](auto e) {
        using E = decltype(e);
        ok = gated_launch<E, kForward>(a, gated_plan<E, kForward>(d->rows, d->hidden, d->features, dma), dma, (hipStream_t)stream);
    });
    if (!ok) return fail(error, cap, "gated linear has too many rows");
    return launch_ok(error, cap, "gated linear launch");
}

extern "C" size_t bfhip_gated_linear_backward_workspace(const bfhip_gated_desc *d) {
    if (bad_gated(d)) return 0;
    return backward_bytes(d).all();
}

extern "C" int bfhip_gated_linear_backward(const bfhip_gated_desc *d, const bfhip_matrix *dh, const bfhip_matrix *x,
                                           const bfhip_matrix *w_gate, const bfhip_matrix *w_up, const bfhip_matrix *gate,
                                           const bfhip_matrix *up, const bfhip_matrix *dx, const bfhip_matrix *dw_gate,
                                           const bfhip_matrix *dw_up, void *workspace, size_t workspace_bytes, void *stream,
                                           char *error, size_t cap) {
    if (bad_gated(d) || !dw_gate != !dw_up || (!dx && !dw_gate)) return fail(error, cap, "invalid gated linear contract");
    if (bad_matrix(dh, d->rows, d->hidden) || bad_matrix(gate, d->rows, d->hidden) || bad_matrix(up, d->rows, d->hidden) ||
        bad_matrix(x, d->rows, d->features) || bad_matrix(w_gate, d->hidden, d->features) || bad_matrix(w_up, d->hidden, d->features) ||
        (dx && bad_matrix(dx, d->rows, d->features)) ||
        (dw_gate && (bad_matrix(dw_gate, d->hidden, d->features) || bad_matrix(dw_up, d->hidden, d->features))))
        return fail(error, cap, "invalid gated linear matrices: strides of at least a row");
    if (d->hidden > 1 && w_gate->stride != w_up->stride) return fail(error, cap, "invalid gated linear matrices: the weights need one stride");
    if (!d->rows && !dw_gate) return 1;
    const BackwardBytes p = backward_bytes(d);
    const size_t need = p.all();
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
        return fail(error, cap, "gated linear workspace too small or not 16-byte aligned");
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    char *work = (char *)workspace;
    const long long stride = slope_stride(d);
    SlopeArgs e{};
    const auto step = [&](const bfhip_matrix *t, long long rows) { return rows > 1 ? t->stride * size : 0; };
    e.dh = (const char *)dh->data; e.dh_stride = step(dh, d->rows);
    e.gate = (const char *)gate->data; e.gate_stride = step(gate, d->rows);
    e.up = (const char *)up->data; e.up_stride = step(up, d->rows);
    e.dg = work;
    e.du = work + p.slopes;
    e.stride = stride;
    e.rows = d->rows;
    e.hidden = (int)d->hidden;
    e.activation = d->activation;
    e.most = (float *)(work + 2 * p.slopes + p.parts);
    e.shift = (int *)(e.most + kMostGroups);
    const long long groups = std::min<long long>(kMostGroups, (d->rows * (stride / 8) + kSlopeThreads - 1) / kSlopeThreads);
    const long long grid = std::min<long long>(8192, (d->rows * (stride / 8) + kSlopeThreads - 1) / kSlopeThreads);
    const bfhip_matrix slopes_g{e.dg, stride}, slopes_u{e.du, stride};
    hipStream_t s = (hipStream_t)stream;
    int ok = 1;
    with_element(d->type, [&](auto el) {
        using E = decltype(el);
        if (d->rows) {
            if (d->type == BFHIP_F16) hipLaunchKernelGGL(gated_most_kernel, dim3((unsigned)groups), dim3(kSlopeThreads), 0, s, e);
            hipLaunchKernelGGL(gated_slope_kernel<E>, dim3((unsigned)grid), dim3(kSlopeThreads), 0, s, e, (int)groups);
        }
        GatedArgs a{};
        a.activation = d->activation;
        a.shift = d->type == BFHIP_F16 && d->rows ? e.shift : nullptr;
        a.partial = (float *)(work + 2 * p.slopes);
        if (dx && d->rows) {
            a.m_op = operand(&slopes_g, &slopes_u, 2, size);
            a.n_op = operand(w_gate, w_up, d->hidden, size);
            a.m = (int)d->rows;
            a.n = (int)d->features;
            a.k = (int)d->hidden;
            a.out[0] = (char *)dx->data;
            a.out_stride[0] = step(dx, d->rows);
            const bool dma = stride < 1 << 21 && chunks(w_gate, d->hidden, d->features, size) && chunks(w_up, d->hidden, d->features, size);
            ok = gated_launch<E, kInputs>(a, gated_plan<E, kInputs>(a.m, a.n, a.k, dma), dma, s) && ok;
        }
        if (dw_gate) {
            a.m_op = operand(&slopes_g, &slopes_u, 2, size);
            a.n_op = operand(x, x, d->rows, size);
            a.m = (int)d->hidden;
            a.n = (int)d->features;
            a.k = (int)d->rows;
            a.out[0] = (char *)dw_gate->data;
            a.out[1] = (char *)dw_up->data;
            a.out_stride[0] = step(dw_gate, d->hidden);
            a.out_stride[1] = step(dw_up, d->hidden);
            const bool dma = stride < 1 << 21 && chunks(x, d->rows, d->features, size);
            ok = gated_launch<E, kWeights>(a, gated_plan<E, kWeights>(a.m, a.n, a.k, dma), dma, s) && ok;
        }
    });
    if (!ok) return fail(error, cap, "gated linear has too many rows");
    return launch_ok(error, cap, "gated linear launch");
}
