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
#pragma once

#include <type_traits>

#include "attention.h"

namespace bfhip {

enum Form { kForward, kInputs, kWeights };

struct GatedOperand {
    const char *gate, *up;  // one matrix each, or the same
    long long stride;       // bytes
};

struct GatedArgs {
    GatedOperand m_op, n_op;
    int m, n, k;     // of the result, and of the contraction (of one of its two halves)
    char *out[3];    // forward: h, and gate and up in fp32; inputs: dx; weights: dWg, dWu
    long long out_stride[3];  // bytes
    const int *shift;         // fp16 gradients were multiplied by 2^shift
    long long low;            // bytes from dg and du to what their rounding left; 0: that is not taken
    int activation;
    int tiles_m, tiles_n;
    // Tiles from `whole` on are split into `parts` of `per` of the contraction's
    // steps each, whose accumulators are added up by a second launch.
    int whole, parts, per;
    float *partial;  // [split tile][part][wave][block][lane][4]
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

// erfc, which keeps gelu's relative precision where it is small.  For 16-bit types with
// t = 1 / (1 + |v| / 2), the substitution that approximations of erfc use since Hastings (1955), as
// t 2^(p(t) - v^2 log2 e), p a polynomial fitted here to log2(e^(v^2) erfc(v) / t) at Chebyshev's
// nodes: off by 3e-6 of it for |v| < 4, beyond by 1e-5 (v^2's rounding); half a step of fp16 is
// 2.4e-4.  17 instructions, erfcf takes 50 (the epilogue of a tile of 256 x 256: 8 us more).
template <class E>
__device__ __forceinline__ float erfc_of(float v) {
    if constexpr (E::kSize == 4) {
        return erfcf(v);
    } else {
        const float z = fabsf(v), t = __builtin_amdgcn_rcpf(fmaf(0.5f, z, 1.f));
        float p = -0.07674804329872131f;
        p = fmaf(p, t, 0.0673188790678978f);
        p = fmaf(p, t, 0.46563780307769775f);
        p = fmaf(p, t, -0.8372750878334045f);
        p = fmaf(p, t, 0.16038353741168976f);
        p = fmaf(p, t, 0.05617106333374977f);
        p = fmaf(p, t, 0.5478323698043823f);
        p = fmaf(p, t, 1.4424240589141846f);
        p = fmaf(p, t, -1.8257462978363037f);
        const float y = t * __builtin_amdgcn_exp2f(fmaf(z * z, -1.4426950408889634f, p));
        return v < 0.f ? 2.f - y : y;
    }
}

// act(g).
template <class E, int kind>
__device__ __forceinline__ float activate(float g) {
    if (kind == BFHIP_SILU) return over<E>(g, 1.f + exp_of<E>(-g));
    if (kind == BFHIP_GELU) return 0.5f * g * erfc_of<E>(-0.70710678118654752f * g);
    return g > 0.f ? g : g == g ? 0.f : g;
}

// act(g) and its derivative.
template <class E, int kind>
__device__ __forceinline__ float2 slope(float g) {
    if (kind == BFHIP_SILU) {
        const float s = over<E>(1.f, 1.f + exp_of<E>(-g)), rest = over<E>(1.f, 1.f + exp_of<E>(g));
        return make_float2(g * s, s * fmaf(g, rest, 1.f));
    }
    if (kind == BFHIP_GELU) {
        const float cdf = 0.5f * erfc_of<E>(-0.70710678118654752f * g);
        return make_float2(g * cdf, fmaf(g * 0.39894228040143268f, exp_of<E>(-0.5f * g * g), cdf));
    }
    return make_float2(g > 0.f ? g : g == g ? 0.f : g, g > 0.f ? 1.f : 0.f);
}

// Calls f with the activation as a constant (one branch for all that it does).
template <class G>
__host__ __device__ __forceinline__ void with_activation(int kind, G f) {
    if (kind == BFHIP_SILU) f(std::integral_constant<int, BFHIP_SILU>{});
    else if (kind == BFHIP_GELU) f(std::integral_constant<int, BFHIP_GELU>{});
    else f(std::integral_constant<int, BFHIP_RELU>{});
}

// ------------------------------------------------------------------- tiles
// A buffer resource as four words, and a copy of 16 bytes per lane through it:
// LDS[lds + 16 * lane] = buffer[voffset].  In assembly because the compiler would
// wait for every copy that it knows in flight before each transposing LDS read;
// the kernels wait for their copies themselves.  (M0, which holds the LDS
// address, is read one instruction after it is written at the earliest.)
typedef uint32_t Resource __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Resource resource(const char *base) {
    const uint64_t p = (uint64_t)(uintptr_t)base;
    return Resource{(uint32_t)__builtin_amdgcn_readfirstlane((int)p), (uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32) & 0xffff),
                    kDmaOutOfRange - 1, 0x00020000u};
}
__device__ __forceinline__ uint32_t lds_address(const char *lds) {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uintptr_t)(__attribute__((address_space(3))) const char *)(lds));
}
__device__ __forceinline__ void copy16(Resource r, const char *lds, uint32_t voffset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(lds_address(lds)), "v"(voffset), "s"(r)
                 : "memory", "m0");
}

// One operand's tile of OUTER (m or n) x BK (k) elements in LDS, copied in chunks of 16
// bytes: rows start on 16 bytes and hold whole chunks.
template <class E, int OUTER, int BK, int THREADS, bool COL>
struct GatedTile {
    using T = std::conditional_t<COL, AttnTile<E, OUTER>, AttnTile<E, BK>>;
    static constexpr int kOuter = OUTER, kRows = COL ? BK : OUTER, kWords = 16 / E::kSize;
    static constexpr int kBytes = kRows * T::kRow, kIssue = kRows * T::kChunks / THREADS;
    static_assert(kRows * T::kChunks % THREADS == 0, "whole chunks per thread");

    // PAIR > 0: outer rows are PAIR / 2 of the gate's, PAIR / 2 of the up's in turn.
    template <int PAIR>
    __device__ __forceinline__ static int source(int r) { return PAIR ? r / PAIR * (PAIR / 2) + r % (PAIR / 2) : r; }

    // Rows that the threads' j-th chunks span; chunk j of a thread is chunk 0 moved
    // by j times as many, a multiple of the swizzle's period
    // (or of half of it: then every other chunk is at the other half's place).
    static constexpr int kSpan = THREADS / T::kChunks, kPlaces = kSpan % 16 ? 2 : 1;
    static_assert(kSpan % 8 == 0 && THREADS % T::kChunks == 0, "chunks repeat with the swizzle");
    uint32_t off[kPlaces];    // bytes of chunk 0 from the tile's first row
    int row, first[kPlaces];  // its row in the matrix, and its first element along the row
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
        const int r = thread / T::kChunks;
        row = source<PAIR>(r);
#pragma unroll
        for (int p = 0; p < kPlaces; ++p) {
            const int c = (thread % T::kChunks) ^ T::swizzle(r + p * kSpan);
            first[p] = c * kWords;
            off[p] = (uint32_t)row * (uint32_t)stride + 16u * c;
        }
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
    __device__ __forceinline__ void fetch(const char *a, const char *b, int k0, int k, const char *lds) const {
        const long long at = COL ? k0 * stride : (long long)k0 * E::kSize;
        const int rows = COL ? k - k0 : left, length = COL ? left : k - k0;  // what there is of the tile
        const Resource ra = resource(a + at), rb = resource(b + at);
#pragma unroll
        for (int j = 0; j < kIssue; ++j) {
            const bool in = row + span_row<PAIR>(j) < rows && first[j % kPlaces] < length;
            copy16(second<PAIR>(j) ? rb : ra, lds + (j * THREADS + wave * kWave) * 16,
                   in ? off[j % kPlaces] + (uint32_t)span_row<PAIR>(j) * (uint32_t)stride : kDmaOutOfRange);
        }
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

// BM x BN results by WM x WN waves, BK of the contraction at a time.
template <class E, Form F, int BM_, int BN_, int WM_, int WN_>
struct GatedShape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = 128 / E::kSize;
    static constexpr int kThreads = WM * WN * kWave, kM = BM / WM, kN = BN / WN, kMB = kM / 16, kNB = kN / 16;
    using MTile = GatedTile<E, BM, BK, kThreads, F == kWeights>;
    using NTile = GatedTile<E, BN, BK, kThreads, F != kForward>;
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
__device__ __forceinline__ TileAt tile_at(int id, int whole, int tiles_m, int tiles_n) {
    constexpr int kGroup = 8;
    if (id < whole) id = xcd_swizzle(id, whole);
    const int group = id / (kGroup * tiles_n), first = group * kGroup, rows = min(kGroup, tiles_m - first);
    const int in = id - group * kGroup * tiles_n;
    return TileAt{first + in % rows, in / rows};
}

// Results leave by way of LDS, so that a row's neighbours are stored together: a wave
// lays down block columns of its accumulators, 16 rows each, in rows of kN + 4 floats
// of its own, and then goes through them eight results at a time.
template <class E, Form F, class S>
struct GatedStore {
    static constexpr int kRow = S::kN + 4, kCols = S::kPair ? S::kN / 2 : S::kN, kRounds = S::kMB > 1 ? 2 : 1;
    static constexpr int kColumns = S::kMB / kRounds;                  // block columns of a round
    static constexpr int kFloats = 16 * kColumns * kRow;               // of a wave
    int m0, n0, shift;
    char *out;
    long long stride;

    __device__ __forceinline__ GatedStore(const GatedArgs &a, TileAt at, int wave) {
        const int wm = wave / S::WN, wn = wave % S::WN, tiles = F == kWeights ? a.tiles_m / 2 : a.tiles_m;
        const bool up = F == kWeights && at.tm >= tiles;
        m0 = (up ? at.tm - tiles : at.tm) * S::BM + wm * S::kM;
        n0 = at.tn * S::kCols + wn * kCols;
        shift = F != kForward && a.shift ? -*a.shift : 0;
        out = up ? a.out[1] : a.out[0];
        stride = up ? a.out_stride[1] : a.out_stride[0];
    }
    __device__ __forceinline__ static void lay(float *mine, const f32x4 (&acc)[S::kNB], int column, int lane) {
#pragma unroll
        for (int i = 0; i < S::kNB; ++i)
            *reinterpret_cast<f32x4 *>(mine + (16 * column + (lane & 15)) * kRow + 16 * i + 4 * (lane >> 4)) = acc[i];
    }
    template <class T>
    __device__ __forceinline__ static void put(char *row, int n, int count, const float (&v)[8]) {
        typename T::Word *p = (typename T::Word *)row + n;
        Words<T, 8> w;
#pragma unroll
        for (int e = 0; e < 8; ++e) w.put(e, v[e]);
        if (count >= 8) {
            w.store(p);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < count) p[e] = w.w[e];
        }
    }
    template <int kActivation>
    __device__ __forceinline__ void forward(const GatedArgs &a, int m, int n, const float (&g)[8], const float (&u)[8]) const {
        float h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = activate<E, kActivation>(g[e]) * u[e];
        put<E>(a.out[0] + m * a.out_stride[0], n, a.n - n, h);
        if (a.out[1]) {
            put<ElemF32>(a.out[1] + m * a.out_stride[1], n, a.n - n, g);
            put<ElemF32>(a.out[2] + m * a.out_stride[2], n, a.n - n, u);
        }
    }
    // Stores the rows from block column `first` on that lie in `mine`.
    __device__ __forceinline__ void rows(const GatedArgs &a, const float *mine, int first, int columns, int lane) const {
        for (int i = lane; i < 16 * columns * (kCols / 8); i += kWave) {
            const int r = i / (kCols / 8), c = i % (kCols / 8) * 8, m = m0 + 16 * first + r, n = n0 + c;
            if (m >= a.m || n >= a.n) continue;
            float v[8], u[8];
            __builtin_memcpy(v, __builtin_assume_aligned(mine + r * kRow + c, 16), sizeof v);
            if constexpr (F == kForward) {
                __builtin_memcpy(u, __builtin_assume_aligned(mine + r * kRow + kCols + c, 16), sizeof u);
                with_activation(a.activation, [&](auto kind) { forward<decltype(kind)::value>(a, m, n, v, u); });
            } else {
                if constexpr (std::is_same_v<E, ElemF16>)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], shift);
                put<E>(out + m * stride, n, a.n - n, v);
            }
        }
    }
};

// What a workgroup multiplies: its tile, and the contraction's steps from `begin`.
template <class E, Form F, class S>
struct GatedWork {
    TileAt at;
    int split, each, begin, end;  // split: part among all split tiles' parts, -1 for a whole tile
    typename S::MTile mt;
    typename S::NTile nt;
    uint32_t m_at, n_at;  // where the lane reads its fragments
    int k;
    long long low;

    __device__ __forceinline__ void init(const GatedArgs &a, int block, int wave, int lane) {
        split = block - a.whole;
        const int tile = split < 0 ? block : a.whole + split / a.parts;
        at = tile_at(tile, a.whole, a.tiles_m, a.tiles_n);
        const int half = F == kWeights ? a.tiles_m / 2 : a.tiles_m;
        const bool up = F == kWeights && at.tm >= half;
        mt.template init<0>(a.m_op, up, (up ? at.tm - half : at.tm) * S::BM, a.m);
        nt.template init<S::kPair>(a.n_op, up, at.tn * S::kCols, a.n);
        m_at = S::MTile::lane_at(wave / S::WN * S::kM, lane);
        n_at = S::NTile::lane_at(wave % S::WN * S::kN, lane);
        // For the inputs' gradient the gate's steps, then the up's.  With `low` each step is
        // followed by that of what the rounding left, on the same tile of n.
        k = a.k;
        low = F == kForward ? 0 : a.low;
        each = (k + S::BK - 1) / S::BK;
        const int steps = (F == kInputs ? 2 : 1) * (low ? 2 : 1) * each;
        begin = split < 0 ? 0 : split % a.parts * a.per;
        end = split < 0 ? steps : min(steps, begin + a.per);
    }
    // Past the last step the tiles are empty: zeros, without a read.
    __device__ __forceinline__ void fetch(int t, const char *to) const {
        const int i = low ? t / 2 : t;
        const bool second = F == kInputs && i >= each;
        const int k0 = t < end ? (second ? i - each : i) * S::BK : k;
        mt.template fetch<0>((second ? mt.base_b : mt.base_a) + (t & 1 ? low : 0), mt.base_b, k0, k, to);
        nt.template fetch<S::kPair>(second ? nt.base_b : nt.base_a, nt.base_b, k0, k, to + S::MTile::kBytes);
    }
    // Hands the accumulators to the results, by way of `smem`, or to the parts' sums.
    // No copy into LDS may be in flight and no wave may still read its tiles.
    __device__ __forceinline__ void store(const GatedArgs &a, const f32x4 (&acc)[S::kMB][S::kNB], char *smem, int wave, int lane) const {
        if (split >= 0) {
            f32x4 *to = reinterpret_cast<f32x4 *>(a.partial) + ((size_t)split * S::WM * S::WN + wave) * S::kNB * S::kMB * kWave + lane;
#pragma unroll
            for (int j = 0; j < S::kMB; ++j)
#pragma unroll
                for (int i = 0; i < S::kNB; ++i) to[(j * S::kNB + i) * kWave] = acc[j][i];
            return;
        }
        using Out = GatedStore<E, F, S>;
        const Out out(a, at, wave);
        float *const mine = reinterpret_cast<float *>(smem) + wave * Out::kFloats;
#pragma unroll
        for (int round = 0; round < Out::kRounds; ++round) {
#pragma unroll
            for (int j = 0; j < Out::kColumns; ++j) Out::lay(mine, acc[round * Out::kColumns + j], j, lane);
            out.rows(a, mine, round * Out::kColumns, Out::kColumns, lane);
        }
    }
};

// LDS of a product's kernel: its tiles, or the results on their way out.
template <class E, Form F, class S>
constexpr int gated_lds(int tiles) {
    constexpr int results = GatedStore<E, F, S>::kFloats * S::WM * S::WN * (int)sizeof(float);
    return results > tiles ? results : tiles;
}

// Adds up the parts' accumulators of a split tile in order and stores the results,
// a block column per workgroup.
template <class E, Form F, class S>
constexpr int kJoinFloats = S::WM * S::WN * 16 * GatedStore<E, F, S>::kRow;

template <class E, Form F, class S>
__device__ __forceinline__ void gated_join(const GatedArgs &a, int block, float *smem) {
    using Out = GatedStore<E, F, S>;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int tile = block / S::kMB, j = block % S::kMB;
    constexpr size_t kBlocks = (size_t)S::kNB * S::kMB * kWave, kStep = kBlocks * S::WM * S::WN;
    const f32x4 *from = reinterpret_cast<const f32x4 *>(a.partial) + (size_t)tile * a.parts * kStep + wave * kBlocks + j * S::kNB * kWave + lane;
    f32x4 acc[S::kNB];
#pragma unroll
    for (int i = 0; i < S::kNB; ++i) acc[i] = from[i * kWave];
#pragma unroll 2
    for (int p = 1; p < a.parts; ++p) {
#pragma unroll
        for (int i = 0; i < S::kNB; ++i) acc[i] += from[p * kStep + i * kWave];
    }
    const Out out(a, tile_at(a.whole + tile, a.whole, a.tiles_m, a.tiles_n), wave);
    float *const mine = smem + wave * 16 * Out::kRow;
    Out::lay(mine, acc, 0, lane);
    out.rows(a, mine, j, 1, lane);
}

template <class E, Form F, class S>
__global__ __launch_bounds__(S::kThreads) void gated_join_kernel(GatedArgs a) {
    __shared__ __attribute__((aligned(16))) float smem[kJoinFloats<E, F, S>];
    gated_join<E, F, S>(a, blockIdx.x, smem);
}

// A product by large tiles (gated_large.hip).
template <class E, Form F>
using LargeShape = GatedShape<E, F, 256, 256, 2, 2>;
template <class E, Form F>
__attribute__((visibility("hidden"))) void launch_gated_large(const GatedArgs &a, long long grid, hipStream_t s);

}  // namespace bfhip

