// Shared parts of the packed-sequence attention kernels: where a workgroup's
// rows are, operand tiles in LDS, and their matrix-core fragments.
#pragma once

#include <cfloat>

#include "bfhip_transformer.h"
#include "element.h"
#include "gemm_core.h"

namespace bfhip {

constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// One tensor of the call: bytes between tokens and heads.
struct AttnRows {
    char *data;
    long long token, head;
    // Address of `head` of `token`.
    __device__ __forceinline__ char *at(long long t, int h) const { return data + t * token + h * head; }
};

struct AttnArgs {
    AttnRows q, k, v, out;
    const int *q_starts, *k_starts;
    const float *bias;  // [heads, 2 reach + 1] or null
    float *lse;         // [heads, q_tokens] or null
    long long q_tokens, k_tokens;
    int sequences, heads, kv_heads, dim, causal, reach;
    float scale, scale2;  // scale2 = scale * log2(e): softmax runs in base 2
    int slots;            // of the grid
    int flip;             // the queries' signs change (forward)
    int ordered;          // tiles in the order of their work
    int parts;            // most parts that a sequence's keys are split into
    int chunk;            // keys (few queries), tiles (forward) or steps (backward) of a part, at least
    int few_rows;         // > 0: sequences of no more queries x group are attention_few_kernel's, the others attention_forward_kernel's
    float *part_out;      // parts > 1: sums of each part, [parts][q_tokens][heads][padded dim]
    float2 *part_stat;    // and their (m, l), [parts][q_tokens][heads]
};

// Work on packed sequences is dealt in slots of `rows` rows without knowing the
// lengths on the host: sequence b owns the slots
//   floor(start_b / rows) + b  ..  floor(start_{b+1} / rows) + b,
// which are at least ceil(length / rows) (at most one more), so slot_count()
// slots always suffice and a slot finds its sequence by searching the starts.
inline long long slot_count(long long tokens, int sequences, int rows) { return tokens / rows + sequences; }

struct Slot {
    int sequence;       // -1: none
    int index;          // of the sequence's slots
    int first;          // row within the sequence (find_rows)
    int start, length;  // the sequence's rows
};

__device__ __forceinline__ long long clamp_start(const int *starts, int b, long long tokens) {
    const long long s = starts[b];
    return s < 0 ? 0 : s > tokens ? tokens : s;
}

// The rows of sequence b: ascending starts within the tensor whatever the array holds.
__device__ __forceinline__ void sequence_rows(const int *starts, int b, long long tokens, int &start, int &length) {
    const long long s = clamp_start(starts, b, tokens), e = clamp_start(starts, b + 1, tokens);
    start = __builtin_amdgcn_readfirstlane((int)s);
    length = __builtin_amdgcn_readfirstlane((int)(e > s ? e - s : 0));
}

// One wave searches 64 candidates at a time (one load for up to 64 sequences,
// two for up to 4096).
__device__ __forceinline__ Slot find_slot(const int *starts, int sequences, long long tokens, int slot, int rows) {
    const int lane = threadIdx.x % kWave;
    int lo = 0, span = sequences;
    while (span > 1) {
        const int step = (span + kWave - 1) / kWave;
        const int at = lo + lane * step;
        const bool below = lane * step < span && clamp_start(starts, at, tokens) / rows + at <= slot;
        const int n = __popcll(__ballot(below));  // a prefix of the lanes
        const int skip = n > 0 ? (n - 1) * step : 0;
        lo += skip;
        span = min(step, span - skip);
    }
    Slot s;
    s.sequence = __builtin_amdgcn_readfirstlane(lo);
    sequence_rows(starts, s.sequence, tokens, s.start, s.length);
    s.index = slot - (s.start / rows + s.sequence);
    if (s.index < 0) s.sequence = -1;  // before the first sequence
    return s;
}

// The sequence of a row, -1 for rows outside every sequence.
__device__ __forceinline__ int find_token(const int *starts, int sequences, long long tokens, int token) {
    const int lane = threadIdx.x % kWave;
    int lo = 0, span = sequences;
    while (span > 1) {
        const int step = (span + kWave - 1) / kWave;
        const int n = __popcll(__ballot(lane * step < span && clamp_start(starts, lo + lane * step, tokens) <= token));
        const int skip = n > 0 ? (n - 1) * step : 0;
        lo += skip;
        span = min(step, span - skip);
    }
    int start, length;
    lo = __builtin_amdgcn_readfirstlane(lo);
    sequence_rows(starts, lo, tokens, start, length);
    return token >= start && token - start < length ? lo : -1;
}

// Slots that have rows of their sequence.
template <int ROWS>
__device__ __forceinline__ Slot find_rows(const int *starts, int sequences, long long tokens, int slot) {
    Slot s = find_slot(starts, sequences, tokens, slot, ROWS);
    if (s.index * (long long)ROWS >= s.length) s.sequence = -1;
    s.first = s.index * ROWS;
    return s;
}

// Slots of the sequences of `least` rows or more alone (least <= ROWS), where
// most have fewer: one for every row whose number is a multiple of `least`.  Such
// a sequence has at least one of them and as many as it has tiles; rows are few
// where places of a batch are empty, so that these cost no workgroups.
template <int ROWS>
__device__ __forceinline__ Slot long_rows(const int *starts, int sequences, long long tokens, int slot, int least) {
    Slot s{-1, 0, 0, 0, 0};
    const int b = find_token(starts, sequences, tokens, slot * least);
    if (b < 0) return s;
    sequence_rows(starts, b, tokens, s.start, s.length);
    s.index = slot - (s.start + least - 1) / least;
    s.first = s.index * ROWS;
    if (s.length >= least && s.index * (long long)ROWS < s.length) s.sequence = b;
    return s;
}

// The rows of rank `rank` when tiles of ROWS rows are put in the order of their
// work, most first, so that no long tile is left for the end.  In causal
// sequences a tile's work grows with its place in its sequence, from the front
// (queries: the keys before them) or the back (keys: the queries after them):
// rank 0 is the last (first) tile of the longest sequence, and the tiles of one
// level come one after the other.  The search has a lane per sequence.
// Where `ordered` says no (by_work below), tiles come in the rows' own order.
template <int ROWS, bool FRONT>
__device__ __forceinline__ Slot ranked_rows(const int *starts, int sequences, long long tokens, int rank, int slots, int ordered) {
    if (!ordered) return find_rows<ROWS>(starts, sequences, tokens, FRONT ? rank : slots - 1 - rank);
    const int lane = threadIdx.x % kWave;
    int start = 0, length = 0;
    if (lane < sequences) {
        const long long b = clamp_start(starts, lane, tokens), e = clamp_start(starts, lane + 1, tokens);
        start = (int)b;
        length = (int)(e > b ? e - b : 0);
    }
    const int tiles = (length + ROWS - 1) / ROWS;
    int most = tiles;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) most = max(most, __shfl_xor(most, o));
    // Tiles of a level above `level`.
    const auto above = [&](int level) {
        int n = 0;
        for (int b = 0; b < sequences; ++b) n += max(0, __builtin_amdgcn_readlane(tiles, b) - 1 - level);
        return n;
    };
    Slot s{-1, 0, 0, 0, 0};
    if (rank >= __builtin_amdgcn_readfirstlane(above(-1))) return s;
    // The lowest level with at most `rank` tiles above it.
    int level = 0, span = __builtin_amdgcn_readfirstlane(most);
    while (span > 1) {
        const int step = (span + kWave - 1) / kWave;
        const int last = level + min((lane + 1) * step, span) - 1;
        const int skip = __builtin_ctzll(__ballot(above(last) <= rank)) * step;
        level += skip;
        span = min(step, span - skip);
    }
    level = __builtin_amdgcn_readfirstlane(level);
    const int nth = rank - __builtin_amdgcn_readfirstlane(above(level));
    const unsigned long long has = __ballot(tiles > level);
    const bool mine = tiles > level && __popcll(has & ((1ull << lane) - 1)) == nth;
    s.sequence = (int)__builtin_ctzll(__ballot(mine));
    s.start = __builtin_amdgcn_readlane(start, s.sequence);
    s.length = __builtin_amdgcn_readlane(length, s.sequence);
    s.index = FRONT ? __builtin_amdgcn_readlane(tiles, s.sequence) - 1 - level : level;
    s.first = s.index * ROWS;
    return s;
}

// Workgroup `id` of slots x heads: its rank and head.  Workgroups are dealt
// round-robin over the eight XCDs, each with an L2 of its own, so the deal keeps
// a key head's workgroups on as few XCDs as it can: with kv_heads a multiple or
// a divisor of eight, id % 8 names the key head (and which share of its work).
struct Deal {
    int rank, head;
};

__device__ __forceinline__ Deal deal(int id, int heads, int kv_heads) {
    const int group = heads / kv_heads;
    int kv = id % kv_heads, rest = id / kv_heads;
    if (kv_heads % 8 == 0) {
        const int per = kv_heads / 8, l = id / 8;
        kv = id % 8 + 8 * (l % per);
        rest = l / per;
    }
    Deal d;
    d.rank = rest / group;
    d.head = kv * group + rest % group;
    return d;
}

// Key tiles per part when `tiles` of them are split evenly into parts of about
// `least` or more, at most `parts` of them.
__device__ __forceinline__ int part_tiles(int tiles, int parts, int least) {
    const int n = min(parts, max(1, tiles / least));
    return max(1, (tiles + n - 1) / n);
}

// ------------------------------------------------------------- operand tiles
// A tile of ROWS rows x DIM elements in LDS, in 16-byte chunks: chunk c of row
// r sits at chunk c ^ swizzle(r) of its row.  16-byte reads are served for the
// rows 0-3 and 12-15 of one lane group together with the rows 4-11 of the next,
// which reads chunk c ^ 1; a transposing read of 16-bit words takes two
// neighbouring chunks of eight neighbouring rows.  With x the row's number among
// those that share their banks, t its highest bit and s the one below, the
// swizzle (s ^ t, the bits below s, t) puts either set on all banks (x itself
// and x turned by one bit each leave one of them two-way conflicts).
template <class E, int DIM>
struct AttnTile {
    static constexpr int kRow = DIM * E::kSize;  // bytes
    static constexpr int kChunks = kRow / 16;
    __device__ __forceinline__ static int swizzle(int r) {
        constexpr int per = kRow >= 256 ? 1 : 256 / kRow;  // rows in one pass over the banks
        constexpr int n = kChunks < 16 ? kChunks : 16;
        const int x = r / per & (n - 1);
        const int t = x / (n / 2);
        return E::kSize == 2 ? ((x ^ t * (n / 4)) << 1 & (n - 1)) | t : x;
    }
};

// One 4-byte LDS-DMA per lane: LDS[lds + 4 * lane] = buffer[voffset].
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rsrc, char *lds, uint32_t voffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void *)(lds), 4, voffset, 0, 0, 0);
}

// Copies ROWS rows to LDS with THREADS threads by LDS-DMA.  Rows past `left`
// and elements past dim read as zero.
template <class E, int DIM, int ROWS, int THREADS>
struct AttnTileCopy {
    using T = AttnTile<E, DIM>;
    static constexpr int kIssue = ROWS * T::kChunks / THREADS;
    static_assert(ROWS * T::kChunks % THREADS == 0, "whole chunks per thread");
    uint32_t off[kIssue];
    uint32_t stride, row;  // bytes between rows, bytes of a row
    int wave;
    __device__ __forceinline__ void init(long long token_bytes, int dim, int thread) {
        stride = (uint32_t)token_bytes;
        row = (uint32_t)dim * E::kSize;
        wave = __builtin_amdgcn_readfirstlane(thread / kWave);
#pragma unroll
        for (int j = 0; j < kIssue; ++j) {
            const int id = j * THREADS + thread, r = id / T::kChunks;
            const uint32_t c = 16u * ((uint32_t)(id % T::kChunks) ^ (uint32_t)T::swizzle(r));
            off[j] = c < row ? (uint32_t)r * stride + c : kDmaOutOfRange;
        }
    }
    __device__ __forceinline__ void issue(const char *base, int left, char *lds) const {
        const int n = left < ROWS ? left : ROWS;
        const __amdgpu_buffer_rsrc_t rsrc = buffer_rsrc(base, n > 0 ? (uint32_t)(n - 1) * stride + row : 0u);
#pragma unroll
        for (int j = 0; j < kIssue; ++j)
            dma16(rsrc, reinterpret_cast<bf16 *>(lds + (j * THREADS + wave * kWave) * 16), off[j]);
    }
};

// Fragment of 16 rows from `r0` (a multiple of 16), elements 32 kk ..+31 of
// each: lane l holds row l & 15, elements 8 (l >> 4) ..+7.
template <class E, int DIM>
__device__ __forceinline__ typename E::Frag row_frag(const char *lds, int r0, int kk, int lane) {
    using T = AttnTile<E, DIM>;
    const int r = lane & 15, g = lane >> 4, f = T::swizzle(r);
    const char *p = lds + (r0 + r) * T::kRow;
    if constexpr (E::kSize == 2) {
        return *reinterpret_cast<const bf16x8 *>(p + 16 * ((4 * kk + g) ^ f));
    } else {
        const f32x4 a = *reinterpret_cast<const f32x4 *>(p + 16 * ((8 * kk + 2 * g) ^ f));
        const f32x4 b = *reinterpret_cast<const f32x4 *>(p + 16 * ((8 * kk + 2 * g + 1) ^ f));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// Fragment of the transposed tile: rows are elements 16 db ..+15, the k axis
// the 32 tile rows from `r0`.  Lane l holds element 16 db + (l & 15); its slot
// e (of 8) is tile row r0 + 16 (e >> 2) + 4 (l >> 4) + (e & 3): the order in
// which two 16-row product blocks leave their rows in a lane's accumulators,
// so a product can be the other operand without leaving its registers.
template <class E, int DIM>
__device__ __forceinline__ typename E::Frag col_frag(const char *lds, int r0, int db, int lane) {
    using T = AttnTile<E, DIM>;
    const int c16 = lane & 15, g = lane >> 4;
    if constexpr (E::kSize == 2) {
        // ds_read_b64_tr_b16: of 16 lanes, lane i gets column i of the 4 x 16
        // words whose row e the lanes 4 e .. 4 e + 3 address, 8 bytes each.
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 *Ptr;
        const int r = 4 * g + (c16 >> 2);
        const char *p = lds + (r0 + r) * T::kRow + 16 * ((2 * db + ((c16 & 3) >> 1)) ^ T::swizzle(r)) + 8 * (c16 & 1);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(p));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(p + 16 * T::kRow));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
        f32x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int r = 4 * g + (e & 3);
            v[e] = *reinterpret_cast<const float *>(lds + (r0 + 16 * (e >> 2) + r) * T::kRow +
                                                    16 * ((4 * db + (c16 >> 2)) ^ T::swizzle(r)) + 4 * (c16 & 3));
        }
        return v;
    }
}

// All fragments of the transposed 32-row tile at `lds`, as col_frag gives them,
// read and waited for in one piece.  The compiler waits for every LDS-DMA copy
// in flight before a transposing read of its own; this form leaves them in
// flight, for loops that keep copies running behind the products.
template <class E, int DIM>
__device__ __forceinline__ void col_frags_in_flight(const char *lds, int lane, typename E::Frag (&f)[DIM / 16]) {
    if constexpr (E::kSize == 4) {
#pragma unroll
        for (int db = 0; db < DIM / 16; ++db) f[db] = col_frag<E, DIM>(lds, 0, db, lane);
    } else {
        using T = AttnTile<E, DIM>;
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        const int c16 = lane & 15, r = 4 * (lane >> 4) + (c16 >> 2);
        const uint32_t row = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)(lds) + r * T::kRow + 8 * (c16 & 1);
#pragma unroll
        for (int db = 0; db < DIM / 16; db += 2) {
            const uint32_t c = (c16 & 3) >> 1, p = row + 16 * ((2 * db + c) ^ T::swizzle(r)), q = row + 16 * ((2 * db + 2 + c) ^ T::swizzle(r));
            s16x4 a, b, x, y;
            asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
                         "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(a), "=&v"(b), "=&v"(x), "=&v"(y)
                         : "v"(p), "v"(q), "n"(16 * T::kRow)
                         : "memory");
            f[db] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
            f[db + 1] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
}

// A bias in base 2.  A finite one stays finite: the lowest fp32 value masks a key
// beside others, but leaves a softmax where every key has it.  Up to kLargeBias
// that takes nothing but the product.
constexpr float kLargeBias = 2e38f;
__device__ __forceinline__ float base2_bias(float bias) {
    const float b = bias * kLog2E;
    return __builtin_isinf(b) && !__builtin_isinf(bias) ? __builtin_copysignf(FLT_MAX, bias) : b;
}

// A head's bias row in LDS, in base 2, with its ends repeated kPad times so
// that a block of 16 x 16 scores that meets distances within the reach is read
// without clamping.
struct BiasRow {
    static constexpr int kPad = 32;
    const float *zero;  // the bias of distance 0
    int reach;
    __host__ __device__ __forceinline__ static int floats(int reach) { return 2 * (reach + kPad) + 1; }
    // Copies `bias` [2 reach + 1] to `lds` (the caller waits).
    __device__ __forceinline__ static BiasRow fill(float *lds, const float *bias, int reach, int thread, int threads) {
        for (int i = thread; i < floats(reach); i += threads) lds[i] = base2_bias(bias[min(max(i - kPad, 0), 2 * reach)]);
        return BiasRow{lds + reach + kPad, reach};
    }
    // Of the four distances from `at` on, in a block of 16 x 16 scores with the
    // distances far0 - 15 .. far0 + 15.  Beyond the reach all have one bias.
    __device__ __forceinline__ f32x4 block(int far0, int at) const {
        f32x4 v;
        if (far0 + 15 <= -reach || far0 - 15 >= reach) {
            const float one = zero[far0 < 0 ? -reach : reach];
            v = f32x4{one, one, one, one};
        } else {
            __builtin_memcpy(&v, zero + at, sizeof v);
        }
        return v;
    }
};

// Eight elements at p, which is on 16 bytes (fp32's are two loads).
template <class E>
__device__ __forceinline__ typename E::Frag load_frag(const char *p) {
    typename E::Frag f;
    __builtin_memcpy(&f, __builtin_assume_aligned(p, 16), sizeof f);
    return f;
}

// Fragment of 16 rows in global memory (row 0 at `base`): elements 32 kk ..+31.
// Rows past `rows` and elements past dim are zero.
template <class E>
__device__ __forceinline__ typename E::Frag global_frag(const char *base, long long token_bytes, int rows, int dim,
                                                        int kk, int lane) {
    const int r = lane & 15, d = 32 * kk + 8 * (lane >> 4);
    typename E::Frag f = {};
    if (r < rows && d < dim) f = load_frag<E>(base + r * token_bytes + d * E::kSize);
    return f;
}

// The fragment, its signs changed if `flip`.
template <class E>
__device__ __forceinline__ typename E::Frag signed_frag(typename E::Frag f, int flip) {
    if (!flip) return f;
    if constexpr (E::kSize == 4) {
        return -f;
    } else {
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(bf16x8, __builtin_bit_cast(s16x8, f) ^ (short)0x8000);
    }
}

// Eight fp32 values as operand words, rounded to nearest even.
template <class E>
__device__ __forceinline__ typename E::Frag to_frag(const f32x4 &a, const f32x4 &b) {
    const f32x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    if constexpr (E::kSize == 4) {
        return v;
    } else {
        typedef typename E::Word Words8 __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(bf16x8, __builtin_convertvector(v, Words8));
    }
}

// What the rounding of to_frag left, as operand words; nothing of a value that the
// type holds as an infinity.
template <class E>
__device__ __forceinline__ typename E::Frag rest_frag(const f32x4 &a, const f32x4 &b) {
    typedef typename E::Word Words4 __attribute__((ext_vector_type(4)));
    const auto rest = [](const f32x4 &v) {
        const f32x4 w = __builtin_convertvector(__builtin_convertvector(v, Words4), f32x4);
        f32x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = __builtin_isinf(w[e]) ? 0.f : v[e] - w[e];
        return r;
    };
    return to_frag<E>(rest(a), rest(b));
}

// Sum of the products of two fragments' eight values.
template <class E>
__device__ __forceinline__ float frag_dot(const typename E::Frag &a, const typename E::Frag &b) {
    typedef typename E::Word Words8 __attribute__((ext_vector_type(8)));
    const f32x8 x = __builtin_convertvector(__builtin_bit_cast(Words8, a), f32x8);
    const f32x8 y = __builtin_convertvector(__builtin_bit_cast(Words8, b), f32x8);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
    return s;
}

// Stores an accumulated transposed product of DB x 16 elements by 16 rows: lane
// l holds row l & 15 (at `row`, if `live`), elements 16 db + 4 (l >> 4) ..+3.
template <class E, int DB>
__device__ __forceinline__ void store_rows(const f32x4 (&o)[DB], float scale, char *row, bool live, int dim, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
        const int d = 16 * db + 4 * g;
        if (!live || d >= dim) continue;
        Words<E, 4> w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.put(e, o[db][e] * scale);
        __builtin_memcpy(__builtin_assume_aligned(row + d * E::kSize, 4 * E::kSize), &w, sizeof w);
    }
}

// 2^v where v may be -inf (0).
__device__ __forceinline__ float exp2_raw(float v) { return __builtin_amdgcn_exp2f(v); }

// ------------------------------------------------------------------ the host
inline bool bad_rows(const bfhip_rows *r, long long tokens, int dim, int size) {
    if (!r || (!r->data && tokens)) return true;
    const long long step = 16 / size;
    return ((uintptr_t)r->data & 15) || r->head_stride % step || r->head_stride < 0 ||
           (tokens > 1 && (r->token_stride % step || r->token_stride < dim || r->token_stride >= 4 << 20));
}

// Rows that a call writes: also no row on another, whichever of tokens and
// heads is the outer one.
inline bool bad_result(const bfhip_rows *r, long long tokens, int heads, int dim, int size) {
    if (bad_rows(r, tokens, dim, size)) return true;
    const long long t = tokens > 1 ? r->token_stride : 0, h = heads > 1 ? r->head_stride : 0;
    return tokens && ((heads > 1 && h < dim) || (tokens > 1 && heads > 1 && t < (heads - 1) * h + dim && h < (tokens - 1) * t + dim));
}

inline AttnRows attn_rows(const bfhip_rows *r, long long tokens, int dim, int size) {
    const long long t = tokens > 1 ? r->token_stride : dim;
    return AttnRows{(char *)r->data, t * size, r->head_stride * size};
}

constexpr long long kMostTokens = 0x7ffff000;  // a tile past the last row is still an int

inline bool bad_attention(const bfhip_attention_desc *d) {
    return !d || d->type < BFHIP_F32 || d->type > BFHIP_BF16 || d->sequences < 0 || d->heads <= 0 || d->kv_heads <= 0 ||
           d->heads % d->kv_heads || d->head_dim <= 0 || d->head_dim > 128 || d->head_dim % 8 || d->heads > 65535 ||
           (d->causal != 0 && d->causal != 1) || d->q_tokens < 0 || d->k_tokens < 0 || d->q_tokens > kMostTokens ||
           d->k_tokens > kMostTokens || !(d->scale == d->scale) || __builtin_isinf(d->scale) ||
           (d->sequences && (!d->q_starts || !d->k_starts)) || (d->bias && (d->reach < 0 || d->reach > 2047));
}

inline AttnArgs attn_args(const bfhip_attention_desc *d, const bfhip_rows *q, const bfhip_rows *k, const bfhip_rows *v,
                          const bfhip_rows *out, float *lse) {
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    AttnArgs a{};
    a.q = attn_rows(q, d->q_tokens, d->head_dim, size);
    a.k = attn_rows(k, d->k_tokens, d->head_dim, size);
    a.v = attn_rows(v, d->k_tokens, d->head_dim, size);
    a.out = attn_rows(out, d->q_tokens, d->head_dim, size);
    a.q_starts = d->q_starts;
    a.k_starts = d->k_starts;
    a.bias = d->bias;
    a.lse = lse;
    a.q_tokens = d->q_tokens;
    a.k_tokens = d->k_tokens;
    a.sequences = d->sequences;
    a.heads = d->heads;
    a.kv_heads = d->kv_heads;
    a.dim = d->head_dim;
    a.causal = d->causal;
    a.reach = d->bias ? d->reach : 0;
    a.slots = 0;
    a.scale = d->scale;
    a.scale2 = d->scale * kLog2E;
    return a;
}

// Whether tiles are dealt in the order of their work: up to four rounds of two
// workgroups per CU, where the last round's tail counts (forward of 4096 + 2049
// + .. causal tokens, 16 heads of 128, 1104 workgroups: 124 us, 149 in the rows'
// order); in more rounds the rows' order reads keys while the XCD's L2 still
// has them (8192 + 4097 + .. tokens, 32 heads, 4352 workgroups: 761 us, 741).
inline int by_work(const bfhip_attention_desc *d, long long workgroups) {
    return d->causal && d->sequences <= kWave && workgroups <= 2048;
}

// Calls f with the padded head size.
template <class F>
inline void with_dim(int dim, F f) {
    if (dim <= 32) f(std::integral_constant<int, 32>{});
    else if (dim <= 64) f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, 128>{});
}

}  // namespace bfhip
