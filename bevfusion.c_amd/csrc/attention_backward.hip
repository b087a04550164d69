// Attention over packed sequences, backward (include/bfhip_transformer.h).
//
// With p = 2^(s - lse) recomputed from the forward's lse (base 2 inside):
//   delta_i = dout_i . out_i,  ds_ij = p_ij (dout_i . v_j - delta_i),
//   dv_j = sum_i p_ij dout_i,  dk_j = scale sum_i ds_ij q_i,
//   dq_i = scale sum_j ds_ij k_j,  dbias[e] = sum of ds over pairs at e.
// Two passes: dq and dbias, a workgroup per tile of queries and head that walks
// the keys, and writes the rows' delta and lse for the second; dk and dv, a
// workgroup per tile of keys and key head that walks the queries of the group's
// heads.  Walking twice costs two products of seven more than adding dq up with atomics would,
// and gives the same bits every time.
//
// Precision of the 16-bit types.  p and ds are rounded to the type for the matrix
// cores, and delta is computed from the forward's rounded out.  Over many keys
// these errors average out; a query that sees few keys has large p and a large
// out, and there they show (64 causal tokens: dq and dk off by 1.7 times what
// their own rounding is).  So where no query of a tile sees more than kFineKeys
// keys, the rounding's rest is multiplied too, and delta is summed from p and
// dout . v in fp32, in a walk of its own over the keys.  A bias's gradient sums
// very many ds, whose sum over a row is zero but for delta's error: with dbias,
// delta is always summed so.
//
// lse is one fp32, so p is off by a factor of about 1 +- |lse| 2^-22: beside a
// large bias log l is lost in it, and with it the sum of the row's p.  Where a
// bias takes |lse| past far_lse, the queries' walk finds the row's maximum m and
// sum l again, in a walk over the keys of its own, and p = 2^((s - m) - log2 l).
#include <algorithm>
#include <type_traits>

#include "attention.h"
#include "column_sum.h"

using namespace bfhip;

namespace {

constexpr int kTile = 64;       // rows per LDS tile
constexpr int kFineKeys = 256;  // see above

// 1024 takes p off by less than the 16-bit types' rounding does.
constexpr float far_lse(int size) { return size == 4 ? 64.f : 1024.f; }

// fp16 holds 2^-24 to 65504; p of many keys and score gradients lie outside.  p is
// at most 1 and enters the matrix cores times kSpread.  ds enters times a power of
// two, the growth, one per wave.  In the queries' walk it takes the largest
// |dout . v| of the wave's 32 rows to 2^13 or more (kGrowth at most) where delta is
// summed: |ds| is at most twice that.  Elsewhere the largest ds is watched, and
// what has been summed shrinks when one passes kMost.  The keys' walk gets a bound
// of ds, over all queries that it meets, from the queries' (`most`).  So what is
// lost lies 2^-36 below the largest |dout . v|; powers of two change no other
// bits.
constexpr float kSpread = 0x1p12f, kLogSpread = 12.f, kGrowth = 0x1p40f, kMost = 0x1p15f;

template <class E>
constexpr bool kScaled = std::is_same_v<E, ElemF16>;

// The wave's largest of each lane's rows' (infinite rows stay so, whatever they
// grow by).
template <int B>
__device__ __forceinline__ float wave_most(const float (&rows)[B]) {
    float most = 0.f;
#pragma unroll
    for (int r = 0; r < B; ++r) most = fmaxf(most, rows[r] < INFINITY ? rows[r] : 0.f);
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) most = fmaxf(most, __shfl_xor(most, o));
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, most)));
}

// The power of two that takes `most` to 2^13 .. 2^14.
__device__ __forceinline__ float growth_of(float most) {
    return most > 0.f ? fminf(ldexpf(1.f, 14 - __builtin_amdgcn_frexp_expf(most)), kGrowth) : kGrowth;
}

// What everything shrinks by where one of ds, grown, passes kMost; 1 otherwise.
template <int B>
__device__ __forceinline__ float shrink(const f32x4 (&ds)[2][B]) {
    float rows[B];
    bool over = false;
#pragma unroll
    for (int r = 0; r < B; ++r) {
        rows[r] = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) rows[r] = fmaxf(rows[r], fabsf(ds[b][r][e]));
        over |= rows[r] > kMost;
    }
    if (!__any(over)) return 1.f;
    const float most = wave_most(rows);
    return most > kMost ? growth_of(most) : 1.f;
}

template <int B>
__device__ __forceinline__ void scale_rows(f32x4 (&ds)[2][B], float by) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < B; ++r) ds[b][r] *= by;
}

__device__ __forceinline__ bf16x8 scaled_frag(const bf16x8 &f, float by) {
    typedef _Float16 Words8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(bf16x8, __builtin_bit_cast(Words8, f) * (_Float16)by);
}

// Keys per tile: two tiles of keys and values, and five rows of the longest
// bias, have to fit the LDS.
constexpr int tile_keys(int size, int dim) { return size == 4 && dim > 64 ? 32 : 64; }

// Blocks of 16 rows per wave: two, so that a fragment read from LDS serves two
// products; one for fp32, whose products take eight times as long as the reads.
constexpr int row_blocks(int size) { return size == 4 ? 1 : 2; }

struct GradArgs {
    AttnArgs f;
    AttnRows dout, dq, dk, dv;
    float *nlse, *delta;  // [heads, q_tokens]; nlse: -lse in base 2, -inf for a query without keys (every p is then 0)
    int sum_delta;        // delta is summed over the keys everywhere: with dbias, and in fp16 with a bias
    float *most;          // fp16: of ds in each query slot's four waves, [heads][slots][4]
    int q_slots;
    float *rest;          // with a bias: -log2 l where nlse is -m (see above), 0 elsewhere
    float *part;          // dbias: [query slots, heads, 2 reach + 1] or null
    float *part_kv;       // f.parts > 1: [parts][k_tokens][kv_heads][dk, dv][padded dim]
    float *part_q;        // q_parts > 1: dq, [parts][q_tokens][heads][padded dim]
    int q_parts, q_chunk; // most parts that a sequence's keys are split into, and their tiles, at least
    int joins;            // workgroups that join dk and dv, before those of dq
};

// The queries that a tile of keys meets, as steps of 64 queries of one head.
struct Steps {
    int begin, tiles;  // first query (a multiple of 64), tiles of each head
};
__device__ __forceinline__ Steps query_steps(int causal, int first_key, int offset, int q_len) {
    Steps s;
    s.begin = causal ? max(0, first_key - offset) / kTile * kTile : 0;
    s.tiles = s.begin < q_len ? (q_len - s.begin + kTile - 1) / kTile : 0;
    return s;
}

template <class E, int DIM, int KB, bool BIAS>
struct KeyTile {
    static constexpr int kRows = 64 * KB, kThreads = 4 * kWave;
    static constexpr int kTerms = BIAS ? 3 : 2;                // nlse, delta and rest of a query
    static constexpr int kQ = kTile * AttnTile<E, DIM>::kRow;  // bytes of a tile of q or dout
    static constexpr int kStage = 2 * kQ + kTerms * kTile * (int)sizeof(float);
};

// KB blocks of 16 keys per wave, four waves.  Scores come out with a key per
// lane, so P and dS are the second operands of dv^T = dout^T P and dk^T = q^T dS
// without leaving their registers.  8192 causal tokens, 16 heads of 128 on 4, bf16: 267
// us, 0.70 PFLOP/s: q and dout are read from LDS twice, as rows and transposed,
// for KB x 16 keys, and with the registers for two waves per SIMD the reads'
// latency shows (matrix cores 32 % busy, LDS 36 %).  Measured when this one took
// 300 us: two blocks of keys, which halve the reads but leave one wave per SIMD,
// 380; three waves on tiles of 32 queries 324; parts that are dealt last
// instead of one after the other 300 (the longest work then ends the grid).
template <class E, int DIM, int KB, bool BIAS>
__global__ __launch_bounds__(256, 1) void attention_keys_kernel(GradArgs a) {
    using K = KeyTile<E, DIM, KB, BIAS>;
    constexpr int kRows = K::kRows, kKB = DIM / 32, kDB = DIM / 16, kThreads = K::kThreads;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const AttnArgs &f = a.f;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, g = lane >> 4, group = f.heads / f.kv_heads;
    // A tile's parts one after the other: the longest work is then dealt first.
    const Deal deal_ = deal(blockIdx.x, f.kv_heads * f.parts, f.kv_heads);
    const int kv = deal_.head / f.parts, part = deal_.head % f.parts;
    const Slot s = ranked_rows<kRows, true>(f.k_starts, f.sequences, f.k_tokens, deal_.rank, f.slots, f.ordered);
    if (s.sequence < 0) return;
    int q_start, q_len;
    sequence_rows(f.q_starts, s.sequence, f.q_tokens, q_start, q_len);
    const int offset = s.length - q_len;
    const int key0 = s.first + wave * 16 * KB;
    const Steps steps = query_steps(f.causal, s.first, offset, q_len);
    const int all = steps.tiles * group, per = part_tiles(all, f.parts, f.chunk);
    if (part && part >= (all + per - 1) / per) return;  // (the first part is always there)
    const int first = part * per, end = min(all, first + per);

    AttnTileCopy<E, DIM, kTile, kThreads> qc, gc;
    qc.init(f.q.token, f.dim, threadIdx.x);
    gc.init(a.dout.token, f.dim, threadIdx.x);
    const auto issue = [&](int step) {
        const int head = kv * group + step / steps.tiles, i0 = steps.begin + step % steps.tiles * kTile, left = q_len - i0;
        char *const to = smem + (step & 1) * K::kStage;
        qc.issue(f.q.at((long long)q_start + i0, head), left, to);
        gc.issue(a.dout.at((long long)q_start + i0, head), left, to + K::kQ);
        // Past the last query q, dout and the terms are zero: ds is 0, and p is 1
        // (or what a bias makes it, which may be infinite: masked below).
        if (wave < K::kTerms) {
            const float *const term = (wave == 0 ? a.nlse : wave == 1 ? a.delta : a.rest) + (size_t)head * f.q_tokens + q_start + i0;
            dma4(buffer_rsrc(term, 4u * min(left, kTile)), to + 2 * K::kQ + wave * kTile * sizeof(float), 4u * lane);
        }
    };
    typename E::Frag kf[KB][kKB], vf[KB][kKB];
    f32x4 dk[KB][kDB], dv[KB][kDB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int r0 = key0 + 16 * kb;
#pragma unroll
        for (int kk = 0; kk < kKB; ++kk) {
            kf[kb][kk] = global_frag<E>(f.k.at((long long)s.start + r0, kv), f.k.token, s.length - r0, f.dim, kk, lane);
            vf[kb][kk] = global_frag<E>(f.v.at((long long)s.start + r0, kv), f.v.token, s.length - r0, f.dim, kk, lane);
        }
#pragma unroll
        for (int db = 0; db < kDB; ++db) dk[kb][db] = dv[kb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float growth = 1.f;  // of ds
    if constexpr (kScaled<E>) {
        constexpr int kQueries = 64 * row_blocks(E::kSize);  // of a slot
        const int slot = q_start / kQueries + s.sequence, from = 4 * (slot + steps.begin / kQueries);
        const int to = 4 * (slot + (q_len + kQueries - 1) / kQueries);
        float most[1] = {0.f};
        for (int hg = first < end ? first / steps.tiles : group; hg < group && hg * steps.tiles < end; ++hg)
            for (int i = from + lane; i < to; i += kWave)
                most[0] = fmaxf(most[0], a.most[(size_t)(kv * group + hg) * a.q_slots * 4 + i]);
        growth = growth_of(wave_most(most)) / kSpread;  // (ds has p's)
    }
    BiasRow bias{};
    int bias_head = -1;
    if (first < end) issue(first);
    for (int step = first; step < end; ++step) {
        wait_vmcnt<0>();
        lds_barrier();  // this tile is there, and the one before has been read
        if (step + 1 < end) issue(step + 1);
        const char *const qt = smem + (step & 1) * K::kStage, *const gt = qt + K::kQ;
        const float *const terms = reinterpret_cast<const float *>(gt + K::kQ);
        const int hg = step / steps.tiles, i0 = steps.begin + step % steps.tiles * kTile;
        if constexpr (BIAS) {
            if (hg != bias_head) {
                bias_head = hg;
                bias = BiasRow::fill(reinterpret_cast<float *>(smem + 2 * K::kStage),
                                     f.bias + (size_t)(kv * group + hg) * (2 * f.reach + 1), f.reach, threadIdx.x, kThreads);
                lds_barrier();
            }
        }
        // No key of the wave's is there, or is seen.
        if (key0 >= s.length || (f.causal && i0 + kTile - 1 + offset < key0)) continue;
        // A query that does not see every key of the wave's.
        const bool edge = f.causal && i0 + offset < key0 + 16 * KB - 1;
        const bool fine = E::kSize == 2 && (f.causal ? min(s.length, i0 + kTile + offset) : s.length) <= kFineKeys;
        // Whether a query of the tile's may have a rest.
        const bool far = BIAS && __any(fabsf(terms[lane]) > far_lse(E::kSize) / 2.f && __builtin_isfinite(terms[lane]));
        // Scores of the whole tile first: the compiler waits for the copies in
        // flight before the transposed reads, which by then have had the time.
        typename E::Frag pf[2][KB], sf[2][KB];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            f32x4 p[2][KB], ds[2][KB];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int r0 = 32 * c + 16 * b;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) p[b][kb] = ds[b][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < kKB; ++kk) {
                    const typename E::Frag qf = row_frag<E, DIM>(qt, r0, kk, lane);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) p[b][kb] = E::mfma(qf, kf[kb][kk], p[b][kb]);
                }
#pragma unroll
                for (int kk = 0; kk < kKB; ++kk) {
                    const typename E::Frag gf = row_frag<E, DIM>(gt, r0, kk, lane);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) ds[b][kb] = E::mfma(gf, vf[kb][kk], ds[b][kb]);
                }
                f32x4 nlse = *reinterpret_cast<const f32x4 *>(terms + r0 + 4 * g);
                if constexpr (kScaled<E>)  // (part of the exponent; its rounding is nlse's own)
                    if (!far) nlse += kLogSpread;
                const f32x4 delta = *reinterpret_cast<const f32x4 *>(terms + kTile + r0 + 4 * g);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    // Key minus query of the block's first ones.
                    const int far0 = key0 + 16 * kb - (i0 + r0 + offset);
                    f32x4 x;
                    if constexpr (BIAS) {  // (rounded as the forward's scores are)
                        const f32x4 b4 = bias.block(far0, far0 + l16 - 4 * g - 3);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = fmaf(p[b][kb][e], f.scale2, b4[3 - e]) + nlse[e];
                        if (far) x += *reinterpret_cast<const f32x4 *>(terms + 2 * kTile + r0 + 4 * g) + (kScaled<E> ? kLogSpread : 0.f);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = fmaf(p[b][kb][e], f.scale2, nlse[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[b][kb][e] = exp2_raw(x[e]);
                        ds[b][kb][e] = p[b][kb][e] * (ds[b][kb][e] - delta[e]);
                    }
                }
            }
            if (edge) {
                const int far = key0 + l16 - (i0 + 32 * c + 4 * g + offset);
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (far > 16 * (b - kb) + e) p[b][kb][e] = ds[b][kb][e] = 0.f;
            }
            if (BIAS && i0 + kTile > q_len) {
                const int left = q_len - (i0 + 32 * c + 4 * g);
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (16 * b + e >= left) p[b][kb][e] = ds[b][kb][e] = 0.f;
            }
            if constexpr (kScaled<E>) scale_rows(ds, growth);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                pf[c][kb] = to_frag<E>(p[0][kb], p[1][kb]);
                sf[c][kb] = to_frag<E>(ds[0][kb], ds[1][kb]);
            }
            if constexpr (E::kSize == 2) {
                if (fine) {
#pragma unroll
                    for (int db = 0; db < kDB; ++db) {
                        const typename E::Frag gf = col_frag<E, DIM>(gt, 32 * c, db, lane);
                        const typename E::Frag qf = col_frag<E, DIM>(qt, 32 * c, db, lane);
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb) {
                            dv[kb][db] = E::mfma(gf, rest_frag<E>(p[0][kb], p[1][kb]), dv[kb][db]);
                            dk[kb][db] = E::mfma(qf, rest_frag<E>(ds[0][kb], ds[1][kb]), dk[kb][db]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int db = 0; db < kDB; ++db) {
                const typename E::Frag gf = col_frag<E, DIM>(gt, 32 * c, db, lane);
                const typename E::Frag qf = col_frag<E, DIM>(qt, 32 * c, db, lane);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    dv[kb][db] = E::mfma(gf, pf[c][kb], dv[kb][db]);
                    dk[kb][db] = E::mfma(qf, sf[c][kb], dk[kb][db]);
                }
            }
        }
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int r = key0 + 16 * kb + l16;
        const bool live = r < s.length;
        const float dk_by = kScaled<E> ? 1.f / (kSpread * growth) : 1.f, dv_by = kScaled<E> ? 1.f / kSpread : 1.f;
        if (per < all) {
            if (!live) continue;
            float *const row = a.part_kv + (((size_t)part * f.k_tokens + s.start + r) * f.kv_heads + kv) * 2 * DIM + 4 * g;
#pragma unroll
            for (int db = 0; db < kDB; ++db) {
                *reinterpret_cast<f32x4 *>(row + 16 * db) = dk[kb][db] * dk_by;
                *reinterpret_cast<f32x4 *>(row + DIM + 16 * db) = dv[kb][db] * dv_by;
            }
        } else {
            store_rows<E, kDB>(dk[kb], f.scale * dk_by, a.dk.at((long long)s.start + r, kv), live, f.dim, lane);
            store_rows<E, kDB>(dv[kb], dv_by, a.dv.at((long long)s.start + r, kv), live, f.dim, lane);
        }
    }
}

// dq of one token from the parts' sums, in order: four elements per thread.
template <class E, int DIM>
__device__ __forceinline__ void join_queries(const GradArgs &a, int block) {
    constexpr int kPer = 256 * 4 / DIM, kRows = 64 * row_blocks(E::kSize), kKeys = tile_keys(E::kSize, DIM);
    const AttnArgs &f = a.f;
    const int per_token = (f.heads + kPer - 1) / kPer, token = block / per_token;
    const int head = block % per_token * kPer + threadIdx.x / (DIM / 4), d = threadIdx.x % (DIM / 4) * 4;
    const int sequence = find_token(f.q_starts, f.sequences, f.q_tokens, token);
    if (sequence < 0 || head >= f.heads) return;
    int q_start, q_len, k_start, k_len;
    sequence_rows(f.q_starts, sequence, f.q_tokens, q_start, q_len);
    sequence_rows(f.k_starts, sequence, f.k_tokens, k_start, k_len);
    const int tile = (token - q_start) / kRows * kRows;
    const int last = f.causal ? min(k_len, min(tile + kRows, q_len) + k_len - q_len) : k_len;
    const int tiles = last > 0 ? (last + kKeys - 1) / kKeys : 0, per = part_tiles(tiles, a.q_parts, a.q_chunk);
    if (per >= tiles) return;  // written by the queries' walk
    const int used = (tiles + per - 1) / per;
    const size_t step = (size_t)f.q_tokens * f.heads * DIM;
    const float *const at = a.part_q + ((size_t)token * f.heads + head) * DIM + d;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < used; ++p) v += *reinterpret_cast<const f32x4 *>(at + p * step);
    if (d >= f.dim) return;
    Words<E, 4> w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w.put(e, v[e] * f.scale);
    w.store(reinterpret_cast<typename E::Word *>(a.dq.at(token, head)) + d);
}

// dk and dv from the parts' sums, in order: four elements per thread, 2 DIM / 4
// threads per key and key head; and, by the workgroups behind, dq.
template <class E, int DIM, int ROWS>
__global__ __launch_bounds__(256) void attention_gradient_join_kernel(GradArgs a) {
    constexpr int kPer = 256 * 4 / (2 * DIM);  // key heads of a workgroup, all of one token
    const AttnArgs &f = a.f;
    if ((int)blockIdx.x >= a.joins) return join_queries<E, DIM>(a, blockIdx.x - a.joins);
    const int per_token = (f.kv_heads + kPer - 1) / kPer, token = blockIdx.x / per_token;
    const int kv = blockIdx.x % per_token * kPer + threadIdx.x / (DIM / 2), d = threadIdx.x % (DIM / 2) * 4;
    const int sequence = find_token(f.k_starts, f.sequences, f.k_tokens, token);
    if (sequence < 0 || kv >= f.kv_heads) return;
    int q_start, q_len, k_start, k_len;
    sequence_rows(f.q_starts, sequence, f.q_tokens, q_start, q_len);
    sequence_rows(f.k_starts, sequence, f.k_tokens, k_start, k_len);
    const Steps steps = query_steps(f.causal, (token - k_start) / ROWS * ROWS, k_len - q_len, q_len);
    const int all = steps.tiles * (f.heads / f.kv_heads), per = part_tiles(all, f.parts, f.chunk);
    if (per >= all) return;  // written by the kernel before
    const int used = (all + per - 1) / per;
    const size_t step = (size_t)f.k_tokens * f.kv_heads * 2 * DIM;
    const float *const at = a.part_kv + ((size_t)token * f.kv_heads + kv) * 2 * DIM + d;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < used; ++p) v += *reinterpret_cast<const f32x4 *>(at + p * step);
    const bool is_k = d < DIM;
    const int e0 = is_k ? d : d - DIM;
    if (e0 >= f.dim) return;
    Words<E, 4> w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w.put(e, v[e] * (is_k ? f.scale : 1.f));
    w.store(reinterpret_cast<typename E::Word *>((is_k ? a.dk : a.dv).at(token, kv)) + e0);
}

// The value of the lane N places on (SHL) or back (SHR) in the row of 16, 0
// past its ends.
template <bool SHL, int N>
__device__ __forceinline__ float row_shift(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), (SHL ? 0x100 : 0x110) + N, 0xf, 0xf, true));
}

// Sums of a 16 x 16 block of dS^T along its diagonals into `sum` (this wave's
// own array).  Lane (query i, group g) holds the keys 4 g + e, distance far0 +
// 4 g + e - i.  Within a group, shifts along the row of lanes add the four e up
// where the diagonal meets e = 0 (`main`) and, for the three diagonals that
// begin left of it, in the last lanes (`rest`).  The groups' lanes (i + 4 n, g +
// n) lie on one diagonal: two shuffles add them in the lane that starts it.
// Either write is then to addresses of one lane each.  A sum's next addition may
// be another lane's, which the compiler, who sees one lane's addresses differ,
// must not move before this one: LDS serves a wave in its order, so that keeping
// the instructions' order fixes the sums'.  Distances at or beyond the reach are
// left to the caller's low and high sums.
__device__ __forceinline__ void diagonal_sums(const f32x4 &ds, int far0, int reach, float *sum, float &low, float &high,
                                              int lane) {
    const int i = lane & 15, g = lane >> 4;
    if (far0 + 15 <= -reach) {
        low += (ds[0] + ds[1]) + (ds[2] + ds[3]);
        return;
    }
    if (far0 - 15 >= reach) {
        high += (ds[0] + ds[1]) + (ds[2] + ds[3]);
        return;
    }
    float main = (ds[0] + row_shift<true, 1>(ds[1])) + (row_shift<true, 2>(ds[2]) + row_shift<true, 3>(ds[3]));
    const float rest = row_shift<false, 15>(ds[1]) + row_shift<false, 14>(ds[2]) + row_shift<false, 13>(ds[3]);
    float next = __shfl(main, (lane + 20) & 63);
    if (g < 3 && i < 12) main += next;
    next = __shfl(main, (lane + 40) & 63);
    if (g < 2 && i < 8) main += next;
    const auto add = [&](int far, float v) {
        asm volatile("" ::: "memory");
        if (far <= -reach) low += v;
        else if (far >= reach) high += v;
        else sum[far + reach] += v;
    };
    if (g == 0 || i < 4) add(far0 + 4 * g - i, main);
    if (i >= 13) add(far0 + 4 * g + 16 - i, rest);
    asm volatile("" ::: "memory");
}

// IB blocks of 16 queries per wave, four waves.  Scores come out with a query
// per lane, so dS is the second operand of dq^T = k^T dS^T without leaving its
// registers.  Bound by the matrix cores and the exponentials: the same tokens
// 156 us, 0.89 PFLOP/s, the rows' delta included (a launch of its own for it took
// 17 us more).
template <class E, int DIM, int IB, bool BIAS>
__global__ __launch_bounds__(256, 1) void attention_queries_kernel(GradArgs a) {
    constexpr int kRows = 64 * IB, kKB = DIM / 32, kDB = DIM / 16, kKeys = tile_keys(E::kSize, DIM);
    using T = AttnTile<E, DIM>;
    constexpr int kStage = 2 * kKeys * T::kRow;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float *const bias_row = reinterpret_cast<float *>(smem + 2 * kStage);
    const AttnArgs &f = a.f;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, g = lane >> 4;
    constexpr bool kParts = E::kSize == 4 && !BIAS;  // (backward_plan)
    const int items = f.slots * f.heads, nth = kParts ? blockIdx.x / items : 0;  // part of the keys
    const Deal deal_ = deal(kParts ? blockIdx.x % items : blockIdx.x, f.heads, f.kv_heads);
    const int head = deal_.head, kv = head / (f.heads / f.kv_heads), width = 2 * f.reach + 1;
    const Slot s = ranked_rows<kRows, false>(f.q_starts, f.sequences, f.q_tokens, deal_.rank, f.slots, f.ordered);
    float *const part = BIAS && a.part ? a.part + ((size_t)deal_.rank * f.heads + head) * width : nullptr;
    if (s.sequence < 0) {
        if (part)
            for (int i = threadIdx.x; i < width; i += 256) part[i] = 0.f;
        return;
    }
    int k_start, k_len;
    sequence_rows(f.k_starts, s.sequence, f.k_tokens, k_start, k_len);
    const int offset = k_len - s.length, row0 = s.first + wave * 16 * IB;
    const int last = f.causal ? min(k_len, min(s.first + kRows, s.length) + offset) : k_len;
    const int full = f.causal ? min(k_len, row0 + offset + 1) : k_len;
    // Keys that the wave has work on.
    const int own = row0 >= s.length ? 0 : f.causal ? min(k_len, min(row0 + 16 * IB, s.length) + offset) : k_len;
    const int tiles = last > 0 ? (last + kKeys - 1) / kKeys : 0;
    const int per = kParts ? part_tiles(tiles, a.q_parts, a.q_chunk) : tiles;
    const int begin = nth * per, end = min(tiles, begin + per);
    if (kParts && nth && begin >= tiles) return;

    AttnTileCopy<E, DIM, kKeys, 256> kc, vc;
    kc.init(f.k.token, f.dim, threadIdx.x);
    vc.init(f.v.token, f.dim, threadIdx.x);
    const auto issue = [&](int t, int buffer) {
        const int j0 = t * kKeys;
        char *const to = smem + buffer * kStage;
        kc.issue(f.k.at((long long)k_start + j0, kv), k_len - j0, to);
        vc.issue(f.v.at((long long)k_start + j0, kv), k_len - j0, to + kKeys * T::kRow);
    };
    float *const sums = bias_row + BiasRow::floats(f.reach) + width * wave;
    BiasRow bias{};
    if constexpr (BIAS) {
        bias = BiasRow::fill(bias_row, f.bias + (size_t)head * width, f.reach, threadIdx.x, 256);
        if (part)
            for (int i = lane; i < width; i += kWave) sums[i] = 0.f;
    }

    // Whether a row of the workgroup's is far; every wave looks at all rows.
    bool far_tile = false;
    if constexpr (BIAS) {
        for (int r = s.first + lane; r < min(s.first + kRows, s.length); r += kWave) {
            const float lse = f.lse[(size_t)head * f.q_tokens + s.start + r];
            far_tile |= __builtin_isfinite(lse) && fabsf(lse) > far_lse(E::kSize);
        }
        far_tile = __any(far_tile);
    }
    // This wave's rows' rest, where one is far.
    float *const rests = bias_row + BiasRow::floats(f.reach) + (part ? 4 * width : 0) + 16 * IB * wave;
    const bool fine = E::kSize == 2 && last <= kFineKeys, sum_delta = fine || a.sum_delta;
    typename E::Frag qf[IB][kKB], gf[IB][kKB];
    f32x4 dq[IB][kDB];
    float nlse[IB], delta[IB];
    bool far_row[IB];
    int limit[IB];
#pragma unroll
    for (int ib = 0; ib < IB; ++ib) {
        const int r0 = row0 + 16 * ib, r = r0 + l16;
#pragma unroll
        for (int kk = 0; kk < kKB; ++kk) {
            qf[ib][kk] = global_frag<E>(f.q.at((long long)s.start + r0, head), f.q.token, s.length - r0, f.dim, kk, lane);
            gf[ib][kk] = global_frag<E>(a.dout.at((long long)s.start + r0, head), a.dout.token, s.length - r0, f.dim, kk, lane);
        }
        delta[ib] = 0.f;
        if (!sum_delta) {
#pragma unroll
            for (int kk = 0; kk < kKB; ++kk)
                delta[ib] += frag_dot<E>(gf[ib][kk], global_frag<E>(f.out.at((long long)s.start + r0, head), f.out.token, s.length - r0, f.dim, kk, lane));
            delta[ib] += __shfl_xor(delta[ib], 16);
            delta[ib] += __shfl_xor(delta[ib], 32);
        }
        const size_t at = (size_t)head * f.q_tokens + s.start + r;
        const float lse = r < s.length ? f.lse[at] : -INFINITY;
        nlse[ib] = lse == -INFINITY ? -INFINITY : -lse * kLog2E;
        far_row[ib] = BIAS && __builtin_isfinite(lse) && fabsf(lse) > far_lse(E::kSize);
        if (nth == 0 && g == 0 && r < s.length) {
            a.nlse[at] = nlse[ib];
            if constexpr (BIAS) a.rest[at] = 0.f;
            if (!sum_delta) a.delta[at] = delta[ib];
        }
        limit[ib] = f.causal ? min(k_len, r + offset + 1) : k_len;
#pragma unroll
        for (int db = 0; db < kDB; ++db) dq[ib][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // q . k of 16 keys from tile row r0.
    const auto scores = [&](const char *kt, int r0, f32x4 (&p)[IB]) {
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) p[ib] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < kKB; ++kk) {
            const typename E::Frag kf = row_frag<E, DIM>(kt, r0, kk, lane);
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) p[ib] = E::mfma(kf, qf[ib][kk], p[ib]);
        }
    };
    // p and dp = dout . v of 16 keys from tile row r0.
    const auto products = [&](const char *kt, const char *vt, int j0, int r0, f32x4 (&p)[IB], f32x4 (&dp)[IB]) {
        scores(kt, r0, p);
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) dp[ib] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < kKB; ++kk) {
            const typename E::Frag vf = row_frag<E, DIM>(vt, r0, kk, lane);
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) dp[ib] = E::mfma(vf, gf[ib][kk], dp[ib]);
        }
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) {
            const int far0 = j0 + r0 - (row0 + 16 * ib + offset);
            if constexpr (BIAS) {  // (rounded as the forward's scores are)
                const f32x4 b4 = bias.block(far0, far0 + 4 * g - l16);
#pragma unroll
                for (int e = 0; e < 4; ++e) p[ib][e] = fmaf(p[ib][e], f.scale2, b4[e]) + nlse[ib];
                if (far_tile) p[ib] += rests[16 * ib + l16];
#pragma unroll
                for (int e = 0; e < 4; ++e) p[ib][e] = exp2_raw(p[ib][e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) p[ib][e] = exp2_raw(fmaf(p[ib][e], f.scale2, nlse[ib]));
            }
        }
        if (j0 + r0 + 16 > full) {
            const int j = j0 + r0 + 4 * g;
#pragma unroll
            for (int ib = 0; ib < IB; ++ib)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (j + e >= limit[ib]) p[ib][e] = dp[ib][e] = 0.f;
        }
    };
    int buffer = 0;
    if constexpr (BIAS) {
        if (far_tile) {
            float m[IB], l[IB];  // of the keys that the lane meets
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) m[ib] = -INFINITY, l[ib] = 0.f;
            if (tiles > 0) issue(0, buffer);
            for (int t = 0; t < tiles; ++t, buffer ^= 1) {
                wait_vmcnt<0>();
                lds_barrier();  // this tile is there, and the one before has been read
                if (t + 1 < tiles) issue(t + 1, buffer ^ 1);
                const int j0 = t * kKeys;
                if (j0 >= own) continue;
#pragma unroll 1
                for (int r0 = 0; r0 < kKeys; r0 += 16) {
                    f32x4 x[IB];
                    scores(smem + buffer * kStage, r0, x);
#pragma unroll
                    for (int ib = 0; ib < IB; ++ib) {
                        const int far0 = j0 + r0 - (row0 + 16 * ib + offset), j = j0 + r0 + 4 * g;
                        const f32x4 b4 = bias.block(far0, far0 + 4 * g - l16);
                        float top = m[ib];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            x[ib][e] = j + e < limit[ib] ? fmaf(x[ib][e], f.scale2, b4[e]) : -INFINITY;
                            top = fmaxf(top, x[ib][e]);
                        }
                        const float at = top == -INFINITY ? 0.f : top;
                        l[ib] *= exp2_raw(m[ib] - at);
                        m[ib] = top;
#pragma unroll
                        for (int e = 0; e < 4; ++e) l[ib] += exp2_raw(x[ib][e] - at);
                    }
                }
            }
            lds_barrier();  // the last tile has been read
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) {
                rests[16 * ib + l16] = 0.f;
                if (!far_row[ib]) continue;  // (a row's four lanes say the same)
                float top = fmaxf(m[ib], __shfl_xor(m[ib], 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                l[ib] *= exp2_raw(m[ib] - top);
                l[ib] += __shfl_xor(l[ib], 16);
                l[ib] += __shfl_xor(l[ib], 32);
                nlse[ib] = -top;
                const float rest = -__builtin_amdgcn_logf(l[ib]);
                rests[16 * ib + l16] = rest;
                if (g == 0) {
                    const size_t at = (size_t)head * f.q_tokens + s.start + row0 + 16 * ib + l16;
                    a.nlse[at] = nlse[ib];
                    a.rest[at] = rest;
                }
            }
        }
    }
    float growth = kGrowth;  // of ds
    if constexpr (BIAS || E::kSize == 2) {
        if (sum_delta) {  // (there is one part then)
            float most[IB];  // of |dout . v|
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) most[ib] = 0.f;
            if (tiles > 0) issue(0, buffer);
            for (int t = 0; t < tiles; ++t, buffer ^= 1) {
                wait_vmcnt<0>();
                lds_barrier();
                issue(t + 1 < tiles ? t + 1 : 0, buffer ^ 1);  // (the first tile again for the walk below)
                const char *const kt = smem + buffer * kStage, *const vt = kt + kKeys * T::kRow;
                if (t * kKeys >= own) continue;
#pragma unroll
                for (int r0 = 0; r0 < kKeys; r0 += 16) {
                    f32x4 p[IB], dp[IB];
                    products(kt, vt, t * kKeys, r0, p, dp);
#pragma unroll
                    for (int ib = 0; ib < IB; ++ib)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (kScaled<E>) most[ib] = fmaxf(most[ib], fabsf(dp[ib][e]));
                            delta[ib] = fmaf(p[ib][e], dp[ib][e], delta[ib]);
                        }
                }
            }
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) {
                delta[ib] += __shfl_xor(delta[ib], 16);
                delta[ib] += __shfl_xor(delta[ib], 32);
                const int r = row0 + 16 * ib + l16;
                if (g == 0 && r < s.length) a.delta[(size_t)head * f.q_tokens + s.start + r] = delta[ib];
            }
            if constexpr (kScaled<E>) growth = growth_of(wave_most(most));
        }
    }
    if (begin < end && !sum_delta) issue(begin, buffer);
    if constexpr (kScaled<E>) {
        // From here on p, ds and the sums of ds carry the growth, which is part of
        // the exponent (its rounding is nlse's own).
        const float by = __builtin_amdgcn_logf(growth);
#pragma unroll
        for (int ib = 0; ib < IB; ++ib)
            if (far_tile) rests[16 * ib + l16] += by;
            else nlse[ib] += by;
    }
    float low = 0.f, high = 0.f;
    for (int t = begin; t < end; ++t, buffer ^= 1) {
        wait_vmcnt<0>();
        lds_barrier();  // this tile is there, and the one before has been read
        if (t + 1 < end) issue(t + 1, buffer ^ 1);
        const char *const kt = smem + buffer * kStage, *const vt = kt + kKeys * T::kRow;
        const int j0 = t * kKeys;
        if (j0 >= own) continue;
        typename E::Frag sf[kKeys / 32][IB];  // (the whole tile first, as above)
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) {
            f32x4 ds[2][IB];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int r0 = 32 * c + 16 * b;
                f32x4 p[IB];
                products(kt, vt, j0, r0, p, ds[b]);
#pragma unroll
                for (int ib = 0; ib < IB; ++ib) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) ds[b][ib][e] = p[ib][e] * (ds[b][ib][e] - delta[ib]);
                }
            }
            if constexpr (BIAS)
                if (part) {
                    // Blocks on one diagonal first.
                    const int far0 = j0 + 32 * c - (row0 + offset);
                    if constexpr (IB == 1) {
                        diagonal_sums(ds[0][0], far0, f.reach, sums, low, high, lane);
                    } else {
                        diagonal_sums(ds[0][0] + ds[1][1], far0, f.reach, sums, low, high, lane);
                        diagonal_sums(ds[0][1], far0 - 16, f.reach, sums, low, high, lane);
                    }
                    diagonal_sums(ds[1][0], far0 + 16, f.reach, sums, low, high, lane);
                }
            if constexpr (kScaled<E>) {
                if constexpr (!BIAS)
                    if (!sum_delta) {
                        const float by = shrink(ds);
                        if (by != 1.f) {
                            growth *= by;
                            scale_rows(ds, by);
#pragma unroll
                            for (int ib = 0; ib < IB; ++ib) {
                                nlse[ib] += __builtin_amdgcn_logf(by);
                                if (c) sf[0][ib] = scaled_frag(sf[0][ib], by);
#pragma unroll
                                for (int db = 0; db < kDB; ++db) dq[ib][db] *= by;
                            }
                        }
                    }
            }
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) sf[c][ib] = to_frag<E>(ds[0][ib], ds[1][ib]);
            if constexpr (E::kSize == 2) {
                if (fine) {
#pragma unroll
                    for (int db = 0; db < kDB; ++db) {
                        const typename E::Frag kf = col_frag<E, DIM>(kt, 32 * c, db, lane);
#pragma unroll
                        for (int ib = 0; ib < IB; ++ib) dq[ib][db] = E::mfma(kf, rest_frag<E>(ds[0][ib], ds[1][ib]), dq[ib][db]);
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) {
#pragma unroll
            for (int db = 0; db < kDB; ++db) {
                const typename E::Frag kf = col_frag<E, DIM>(kt, 32 * c, db, lane);
#pragma unroll
                for (int ib = 0; ib < IB; ++ib) dq[ib][db] = E::mfma(kf, sf[c][ib], dq[ib][db]);
            }
        }
    }
#pragma unroll
    for (int ib = 0; ib < IB; ++ib) {
        const int r = row0 + 16 * ib + l16;
        if (kParts && per < tiles) {
            if (r >= s.length) continue;
            float *const row = a.part_q + (((size_t)nth * f.q_tokens + s.start + r) * f.heads + head) * DIM + 4 * g;
#pragma unroll
            for (int db = 0; db < kDB; ++db) *reinterpret_cast<f32x4 *>(row + 16 * db) = dq[ib][db];
            continue;
        }
        store_rows<E, kDB>(dq[ib], kScaled<E> ? f.scale / growth : f.scale, a.dq.at((long long)s.start + r, head), r < s.length, f.dim, lane);
    }
    if constexpr (kScaled<E>)  // ds of this wave's is below 2^15 / growth
        if (lane == 0) a.most[((size_t)head * a.q_slots + s.start / kRows + s.sequence + s.index) * 4 + wave] = kMost / growth;
    if constexpr (BIAS) {
        if (!part) return;
        low = group_sum<kWave>(low);
        high = group_sum<kWave>(high);
        if (lane == 0) {
            sums[0] += low;
            sums[2 * f.reach] += high;
        }
        if constexpr (kScaled<E>) {
            asm volatile("" ::: "memory");  // (other lanes' additions)
            for (int i = lane; i < width; i += kWave) sums[i] *= 1.f / growth;
        }
        lds_barrier();
        for (int i = threadIdx.x; i < width; i += 256) {
            const float *q = bias_row + BiasRow::floats(f.reach) + i;
            part[i] = (q[0] + q[width]) + (q[2 * width] + q[3 * width]);
        }
    }
}

constexpr int key_blocks(int size, int dim) { return size == 4 || dim > 64 ? 1 : 2; }

// How a call is dealt: slots of queries and of keys, and parts of the queries
// that a tile of keys meets, so that uneven tiles even out over the CUs.  Parts
// of the keys that a tile of queries meets only in fp32, whose products take eight
// times as long, and where there is less than a workgroup per CU (not with a
// bias, whose gradient takes a walk over all keys first).
struct BackwardPlan {
    int dim, q_rows, k_rows, parts, chunk, q_parts, q_chunk;
    long long q_slots, k_slots;
    size_t terms, most, part, part_kv, part_q;  // bytes
};

BackwardPlan backward_plan(const bfhip_attention_desc *d) {
    BackwardPlan p{};
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    p.dim = d->head_dim <= 32 ? 32 : d->head_dim <= 64 ? 64 : 128;
    p.q_rows = 64 * row_blocks(size);
    p.k_rows = 64 * key_blocks(size, p.dim);
    p.q_slots = slot_count(d->q_tokens, d->sequences, p.q_rows);
    p.k_slots = slot_count(d->k_tokens, d->sequences, p.k_rows);
    // Parts of 16 tiles of queries or more, as many as the average sequence has;
    // of 4 or more where there is less than a workgroup per CU, 2 in fp32, whose
    // products take longer.
    const long long units = p.k_slots * d->kv_heads, group = d->heads / d->kv_heads;
    p.chunk = units >= 256 ? 16 : size == 4 ? 2 : 4;
    const long long rows = units < 256 ? d->q_tokens : d->sequences ? d->q_tokens / d->sequences : 0;
    const long long parts = units ? 2048 / units : 1, steps = rows * group / (kTile * p.chunk);
    p.parts = (int)std::max(1ll, std::min({32ll, parts, steps}));
    const long long q_units = std::max(1ll, (d->q_tokens + p.q_rows - 1) / p.q_rows) * d->heads;
    p.q_chunk = 2 * 64 / tile_keys(size, p.dim);
    p.q_parts = size == 4 && !d->bias && q_units < 256
                    ? (int)std::max(1ll, std::min({32ll, 1024 / q_units, d->k_tokens / 128})) : 1;
    const auto round = [](size_t n) { return (n + 255) / 256 * 256; };
    p.terms = round((size_t)d->heads * d->q_tokens * sizeof(float)) * (d->bias ? 3 : 2);
    p.most = d->type == BFHIP_F16 ? round((size_t)d->heads * p.q_slots * 4 * sizeof(float)) : 0;
    p.part = d->bias ? round((size_t)p.q_slots * d->heads * (2 * d->reach + 1) * sizeof(float)) : 0;
    p.part_kv = p.parts > 1 ? (size_t)p.parts * d->k_tokens * d->kv_heads * 2 * p.dim * sizeof(float) : 0;
    p.part_q = p.q_parts > 1 ? (size_t)p.q_parts * d->q_tokens * d->heads * p.dim * sizeof(float) : 0;
    return p;
}

}  // namespace

extern "C" size_t bfhip_attention_backward_workspace(const bfhip_attention_desc *d) {
    if (bad_attention(d)) return 0;
    const BackwardPlan p = backward_plan(d);
    return p.terms + p.most + p.part + p.part_kv + p.part_q;
}

extern "C" int bfhip_attention_backward(const bfhip_attention_desc *d, const bfhip_rows *q, const bfhip_rows *k,
                                        const bfhip_rows *v, const bfhip_rows *out, const float *lse,
                                        const bfhip_rows *dout, const bfhip_rows *dq, const bfhip_rows *dk,
                                        const bfhip_rows *dv, float *dbias, void *workspace, size_t workspace_bytes,
                                        void *stream, char *error, size_t cap) {
    if (bad_attention(d) || (dbias && !d->bias) || (!lse && d->q_tokens)) return fail(error, cap, "invalid attention contract");
    const int size = d->type == BFHIP_F32 ? 4 : 2, n = d->head_dim;
    if (bad_rows(q, d->q_tokens, n, size) || bad_rows(k, d->k_tokens, n, size) || bad_rows(v, d->k_tokens, n, size) ||
        bad_rows(out, d->q_tokens, n, size) || bad_rows(dout, d->q_tokens, n, size) || bad_result(dq, d->q_tokens, d->heads, n, size) ||
        bad_result(dk, d->k_tokens, d->kv_heads, n, size) || bad_result(dv, d->k_tokens, d->kv_heads, n, size))
        return fail(error, cap, "invalid attention rows: pointers and strides in steps of 16 bytes, token strides of at least head_dim, no results on one another");
    const BackwardPlan p = backward_plan(d);
    const size_t need = p.terms + p.most + p.part + p.part_kv + p.part_q;
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
        return fail(error, cap, "attention workspace too small or not 16-byte aligned");
    const long long q_grid = p.q_slots * d->heads * p.q_parts;
    const long long k_grid = p.k_slots * d->kv_heads * p.parts;
    const long long k_joins = p.parts > 1 ? ((long long)d->kv_heads * 2 * p.dim + 1023) / 1024 * d->k_tokens : 0;
    const long long joins = k_joins + (p.q_parts > 1 ? ((long long)d->heads * p.dim + 1023) / 1024 * d->q_tokens : 0);
    if (!launch_fits(q_grid, 256) || !launch_fits(k_grid, 256) || !launch_fits(joins, 256))
        return fail(error, cap, "attention has too many rows");
    const long long width = 2 * (d->bias ? d->reach : 0) + 1, count = width * d->heads;
    if (dbias && !column_sum_fits(count)) return fail(error, cap, "attention has too many biases");
    GradArgs a{};
    a.f = attn_args(d, q, k, v, out, const_cast<float *>(lse));
    a.f.parts = p.parts;
    a.f.chunk = p.chunk;
    a.dout = attn_rows(dout, d->q_tokens, n, size);
    a.dq = attn_rows(dq, d->q_tokens, n, size);
    a.dk = attn_rows(dk, d->k_tokens, n, size);
    a.dv = attn_rows(dv, d->k_tokens, n, size);
    char *const work = (char *)workspace;
    a.nlse = (float *)work;
    const size_t term = p.terms / (d->bias ? 3 : 2);
    a.delta = (float *)(work + term);
    a.rest = d->bias ? (float *)(work + 2 * term) : nullptr;
    a.most = (float *)(work + p.terms);
    a.q_slots = (int)p.q_slots;
    a.sum_delta = dbias || (d->bias && d->type == BFHIP_F16);
    a.part = dbias ? (float *)(work + p.terms + p.most) : nullptr;
    a.part_kv = (float *)(work + p.terms + p.most + p.part);
    a.part_q = (float *)(work + p.terms + p.most + p.part + p.part_kv);
    a.q_parts = p.q_parts;
    a.q_chunk = p.q_chunk;
    a.joins = (int)k_joins;
    hipStream_t s = (hipStream_t)stream;
    if (d->sequences)
        with_element(d->type, [&](auto e) {
            with_dim(n, [&](auto dim) {
                using E = decltype(e);
                constexpr int DIM = decltype(dim)::value, QB = row_blocks(E::kSize), KB = key_blocks(E::kSize, DIM);
                using T = AttnTile<E, DIM>;
                const auto run = [&](auto with_bias) {
                    constexpr bool B = decltype(with_bias)::value;
                    using K = KeyTile<E, DIM, KB, B>;
                    const size_t row = B ? BiasRow::floats(d->reach) * sizeof(float) : 0;
                    GradArgs b = a;
                    if (d->q_tokens) {
                        b.f.slots = (int)p.q_slots;
                        b.f.ordered = by_work(d, q_grid);
                        hipLaunchKernelGGL((attention_queries_kernel<E, DIM, QB, B>), dim3((unsigned)q_grid), dim3(256),
                                           4 * tile_keys(E::kSize, DIM) * T::kRow + row + (a.part ? 4 * width * sizeof(float) : 0) +
                                               (B ? p.q_rows * sizeof(float) : 0), s, b);
                    }
                    if (d->k_tokens) {
                        b.f.slots = (int)p.k_slots;
                        b.f.ordered = by_work(d, k_grid);
                        hipLaunchKernelGGL((attention_keys_kernel<E, DIM, KB, B>), dim3((unsigned)k_grid),
                                           dim3(K::kThreads), 2 * K::kStage + row, s, b);
                    }
                };
                if (d->bias) run(std::true_type{});
                else run(std::false_type{});
                if (joins)
                    hipLaunchKernelGGL((attention_gradient_join_kernel<E, DIM, 64 * KB>), dim3((unsigned)joins), dim3(256), 0, s, a);
            });
        });
    if (dbias) column_sum(a.part, d->q_tokens && d->sequences ? p.q_slots : 0, dbias, dbias, count, count, s);
    return launch_ok(error, cap, "attention launch");
}
