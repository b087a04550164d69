// Attention over packed sequences, forward (include/bfhip_transformer.h).
//
// One pass over the keys with a running maximum m and sum l per query, in base
// 2 (scores carry log2 e): for each tile of 64 keys
//   S^T = K Q^T, m' = max(m, S), P = 2^(S - m'), l = l 2^(m - m') + sum P,
//   O^T = O^T 2^(m - m') + V^T P^T,
// then O / l and lse = (m + log2 l) ln 2.  Scores come out transposed, so a
// lane holds scores of one query only: the row statistics are one value per
// lane, and P is the second product's operand without leaving its registers.
#include <algorithm>
#include <type_traits>

#include "attention.h"

using namespace bfhip;

namespace {

constexpr int kKeys = 64;      // keys per tile

// Running maximum, sum and result of IB blocks of 16 queries, one wave's.
template <int IB, int DB>
struct Running {
    float m[IB], l[IB];  // of the lane's query; l of the keys that the lane holds
    f32x4 o[IB][DB];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) {
            m[ib] = -INFINITY;
            l[ib] = 0.f;
#pragma unroll
            for (int db = 0; db < DB; ++db) o[ib][db] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // Takes the scores of JB blocks of 16 keys (base 2: score = raw * scale, scale >
    // 0) and leaves 2^(score - m) in their place.  m only has to be near
    // the maximum: it moves, and what has been summed is scaled, when a score
    // passes it by more than 8 (probabilities then stay below 2^8, which fp16
    // holds and fp32 sums); most tiles need no scaling.
    template <int JB>
    __device__ __forceinline__ void take(f32x4 (&sc)[JB][IB], float scale) {
        float top[IB];
        bool moves = false;
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) {
            float t = -INFINITY;
#pragma unroll
            for (int jb = 0; jb < JB; ++jb) {
                t = fmaxf(fmaxf(t, sc[jb][ib][0]), sc[jb][ib][1]);
                t = fmaxf(fmaxf(t, sc[jb][ib][2]), sc[jb][ib][3]);
            }
            t = fmaxf(t, __shfl_xor(t, 16));
            t = fmaxf(t, __shfl_xor(t, 32));
            top[ib] = t * scale;
            moves |= top[ib] > m[ib] + 8.f;
        }
        if (__any(moves)) {
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) {
                // (each query by its own scores: its bits do not depend on others)
                const float to = top[ib] > m[ib] + 8.f ? top[ib] : m[ib];
                const float fade = exp2_raw(m[ib] - (to == -INFINITY ? 0.f : to));
                m[ib] = to;
                l[ib] *= fade;
#pragma unroll
                for (int db = 0; db < DB; ++db) o[ib][db] *= fade;
            }
        }
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) {
            // No key seen yet: any finite value keeps 2^(-inf - it) at 0.
            const float at = m[ib] == -INFINITY ? 0.f : -m[ib];
#pragma unroll
            for (int jb = 0; jb < JB; ++jb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[jb][ib][e] = exp2_raw(fmaf(sc[jb][ib][e], scale, at));
                    l[ib] += sc[jb][ib][e];
                }
        }
    }
    // l over all lanes of a query.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) {
            l[ib] += __shfl_xor(l[ib], 16);
            l[ib] += __shfl_xor(l[ib], 32);
        }
    }
};

// 1 / l, 0 for a query without keys; NaN stays.
__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : l == 0.f ? 0.f : l; }

__device__ __forceinline__ float natural_lse(float m, float l) {
    return l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// IB blocks of 16 queries per wave, four waves.  Bound by the matrix cores and
// the exponentials, which take about as long (two waves per SIMD run one under
// the other): 16384 causal tokens in eight sequences, 32 heads of 128 on 8 key
// heads, bf16: 720 us, 1.02 PFLOP/s, where a large library product reaches
// 1.15 (matrix cores 46 % busy, vector instructions 51 %); 200 queries, 8 heads
// of 16 on 32400 keys, fp16: 24 us, where half of each product is padding.
// Keys and values of a tile come by LDS-DMA into one of two buffers while the
// tile before is multiplied.
template <class E, int DIM, int IB, bool BIAS>
__global__ __launch_bounds__(256, 1) void attention_forward_kernel(AttnArgs a) {
    constexpr int kRows = 64 * IB, kKB = DIM / 32, kDB = DIM / 16;
    using T = AttnTile<E, DIM>;
    constexpr int kStage = 2 * kKeys * T::kRow;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, g = lane >> 4;
    // Part after part: workgroups that run together then read the same keys.
    const int items = a.slots * a.heads, part = blockIdx.x / items;
    const Deal deal_ = deal(blockIdx.x % items, a.heads, a.kv_heads);
    const int head = deal_.head, kv = head / (a.heads / a.kv_heads);
    const Slot s = a.few_rows
                       ? long_rows<kRows>(a.q_starts, a.sequences, a.q_tokens, deal_.rank, a.few_rows / (a.heads / a.kv_heads) + 1)
                       : ranked_rows<kRows, false>(a.q_starts, a.sequences, a.q_tokens, deal_.rank, a.slots, a.ordered);
    if (s.sequence < 0) return;
    int k_start, k_len;
    sequence_rows(a.k_starts, s.sequence, a.k_tokens, k_start, k_len);
    const int offset = k_len - s.length;  // query i stands at position i + offset
    const int row0 = s.first + wave * 16 * IB;  // this wave's first query
    // Keys seen by the workgroup's last query, and by the wave's first.
    const int last = a.causal ? min(k_len, min(s.first + kRows, s.length) + offset) : k_len;
    const int full = a.causal ? min(k_len, row0 + offset + 1) : k_len;
    // Keys that the wave has work on.
    const int own = row0 >= s.length ? 0 : a.causal ? min(k_len, min(row0 + 16 * IB, s.length) + offset) : k_len;
    const int tiles = last > 0 ? (last + kKeys - 1) / kKeys : 0;
    const int per = part_tiles(tiles, a.parts, a.chunk), begin = part * per, end = min(tiles, begin + per);
    if (part && begin >= tiles) return;

    AttnTileCopy<E, DIM, kKeys, 256> kc, vc;
    kc.init(a.k.token, a.dim, threadIdx.x);
    vc.init(a.v.token, a.dim, threadIdx.x);
    const auto issue = [&](int t) {
        const int j0 = t * kKeys;
        char *const to = smem + (t & 1) * kStage;
        kc.issue(a.k.at((long long)k_start + j0, kv), k_len - j0, to);
        vc.issue(a.v.at((long long)k_start + j0, kv), k_len - j0, to + kKeys * T::kRow);
    };
    BiasRow bias{};
    if constexpr (BIAS)
        bias = BiasRow::fill(reinterpret_cast<float *>(smem + 2 * kStage), a.bias + (size_t)head * (2 * a.reach + 1),
                             a.reach, threadIdx.x, 256);
    typename E::Frag qf[IB][kKB];
    int limit[IB];  // keys that the lane's query sees
#pragma unroll
    for (int ib = 0; ib < IB; ++ib) {
        const int r0 = row0 + 16 * ib;
        const char *q = a.q.at((long long)s.start + r0, head);
#pragma unroll
        for (int kk = 0; kk < kKB; ++kk)
            qf[ib][kk] = signed_frag<E>(global_frag<E>(q, a.q.token, s.length - r0, a.dim, kk, lane), a.flip);
        limit[ib] = a.causal ? min(k_len, r0 + l16 + offset + 1) : k_len;
    }
    if (begin < end) issue(begin);
    Running<IB, kDB> run;
    run.clear();
    for (int t = begin; t < end; ++t) {
        wait_vmcnt<0>();
        lds_barrier();  // this tile is there, and the one before has been read
        if (t + 1 < end) issue(t + 1);
        const char *const kt = smem + (t & 1) * kStage, *const vt = kt + kKeys * T::kRow;
        const int j0 = t * kKeys;
        if (j0 >= own) continue;
        f32x4 sc[4][IB];
#pragma unroll
        for (int jb = 0; jb < 4; ++jb) {
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) sc[jb][ib] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < kKB; ++kk) {
                const typename E::Frag kf = row_frag<E, DIM>(kt, 16 * jb, kk, lane);
#pragma unroll
                for (int ib = 0; ib < IB; ++ib) sc[jb][ib] = E::mfma(kf, qf[ib][kk], sc[jb][ib]);
            }
        }
        if constexpr (BIAS) {
            // Beyond the reach on either side all distances have one bias;
            // nearer ones are looked up.
#pragma unroll
            for (int ib = 0; ib < IB; ++ib)
#pragma unroll
                for (int jb = 0; jb < 4; ++jb) {
                    const int far = j0 + 16 * jb - (row0 + 16 * ib + offset);  // of the block's first key and query
                    const f32x4 b = bias.block(far, far + 4 * g - l16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[jb][ib][e] = fmaf(sc[jb][ib][e], a.scale2, b[e]);
                }
        }
        if (j0 + kKeys > full) {
            const int j = j0 + 4 * g;
#pragma unroll
            for (int ib = 0; ib < IB; ++ib)
#pragma unroll
                for (int jb = 0; jb < 4; ++jb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sc[jb][ib][e] = j + 16 * jb + e < limit[ib] ? sc[jb][ib][e] : -INFINITY;
        }
        run.template take<4>(sc, BIAS ? 1.f : a.scale2);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            typename E::Frag pf[IB];
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) pf[ib] = to_frag<E>(sc[2 * c][ib], sc[2 * c + 1][ib]);
#pragma unroll
            for (int db = 0; db < kDB; ++db) {
                const typename E::Frag vf = col_frag<E, DIM>(vt, 32 * c, db, lane);
#pragma unroll
                for (int ib = 0; ib < IB; ++ib) run.o[ib][db] = E::mfma(vf, pf[ib], run.o[ib][db]);
            }
        }
    }
    run.finish();
    if (a.parts > 1) {
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) {
            const int r = row0 + 16 * ib + l16;
            const size_t row = ((size_t)part * a.q_tokens + s.start + r) * a.heads + head;
            if (r >= s.length) continue;
#pragma unroll
            for (int db = 0; db < kDB; ++db)
                *reinterpret_cast<f32x4 *>(a.part_out + row * DIM + 16 * db + 4 * g) = run.o[ib][db];
            if (g == 0) a.part_stat[row] = make_float2(run.m[ib], run.l[ib]);
        }
        return;
    }
#pragma unroll
    for (int ib = 0; ib < IB; ++ib) {
        const int r = row0 + 16 * ib + l16;
        const bool live = r < s.length;
        store_rows<E, kDB>(run.o[ib], inverse(run.l[ib]), a.out.at((long long)s.start + r, head), live, a.dim, lane);
        if (a.lse && live && g == 0)
            a.lse[(size_t)head * a.q_tokens + s.start + r] = natural_lse(run.m[ib], run.l[ib]);
    }
}

// Few queries per sequence on many keys (single tokens): bound by reading the
// keys and values once, so the work is dealt by keys: a workgroup has a part of
// a sequence's keys, for one key head, and the queries of the head's whole group
// share a tile of 16 rows (row = token * group + head in group; more rows are
// walked tile by tile, reading the keys again).  Each wave walks key tiles of
// its own, 32 keys at a time through its own two LDS buffers, so two tiles are
// in flight per wave and no wave waits for another; the waves' sums are joined
// at the end.
template <class E, int DIM>
struct FewQueries {
    static constexpr int kKeys = 32;
    static constexpr int kStage = 2 * kKeys * AttnTile<E, DIM>::kRow;  // K and V of a tile
    static constexpr int kWaves = kStage <= 8192 ? 4 : 2;              // two workgroups per CU (one for long fp32 rows)
    static constexpr int kThreads = kWaves * kWave;
};

template <class E, int DIM, bool BIAS>
__global__ __launch_bounds__(256, 1) void attention_few_kernel(AttnArgs a) {
    using F = FewQueries<E, DIM>;
    using T = AttnTile<E, DIM>;
    constexpr int kKB = DIM / 32, kDB = DIM / 16, kKeyRows = F::kKeys, kWaves = F::kWaves;
    // One LDS object: with two the compiler waits for every copy in flight
    // before any LDS read.
    __shared__ __attribute__((aligned(16))) char smem[kWaves * (2 * F::kStage + 16 * sizeof(float2))];
    float2(*const stat)[16] = reinterpret_cast<float2(*)[16]>(smem + kWaves * 2 * F::kStage);
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, g = lane >> 4, group = a.heads / a.kv_heads;
    const int kv = blockIdx.x % a.kv_heads;
    const Slot s = find_slot(a.k_starts, a.sequences, a.k_tokens, blockIdx.x / a.kv_heads, a.chunk);
    if (s.sequence < 0) return;
    const int k_start = s.start, k_len = s.length, all = (k_len + kKeyRows - 1) / kKeyRows;
    const int part = s.index, per = part_tiles(all, a.parts, a.chunk / kKeyRows);
    if (part && part >= (all + per - 1) / per) return;  // (the first part is always there)
    const int begin = part * per;
    const bool split = per < all;
    int q_start, q_len;
    sequence_rows(a.q_starts, s.sequence, a.q_tokens, q_start, q_len);
    const int offset = k_len - q_len, rows = q_len * group;
    if (a.few_rows && rows > a.few_rows) return;

    AttnTileCopy<E, DIM, kKeyRows, kWave> kc, vc;
    kc.init(a.k.token, a.dim, lane);
    vc.init(a.v.token, a.dim, lane);
    char *const mine = smem + wave * 2 * F::kStage;
    const auto issue = [&](int t, int buffer) {
        const int j0 = t * kKeyRows;
        char *const to = mine + buffer * F::kStage;
        kc.issue(a.k.at((long long)k_start + j0, kv), k_len - j0, to);
        vc.issue(a.v.at((long long)k_start + j0, kv), k_len - j0, to + kKeyRows * T::kRow);
    };
    for (int first = 0; first < rows; first += 16) {
        const int row = first + l16, token = row / group, head = kv * group + row % group;
        const bool live = row < rows;
        typename E::Frag qf[kKB];
        {
            const char *q = a.q.at((long long)q_start + token, head);
#pragma unroll
            for (int kk = 0; kk < kKB; ++kk) {
                const int d = 32 * kk + 8 * g;
                qf[kk] = typename E::Frag{};
                if (live && d < a.dim) qf[kk] = signed_frag<E>(load_frag<E>(q + d * E::kSize), a.flip);
            }
        }
        const int limit = a.causal ? min(k_len, token + offset + 1) : k_len;
        const int last = a.causal ? min(k_len, (min(first + 16, rows) - 1) / group + 1 + offset) : k_len;
        const int full = a.causal ? min(k_len, first / group + offset + 1) : k_len;
        const int tiles = last > 0 ? (last + kKeyRows - 1) / kKeyRows : 0, end = min(tiles, begin + per);
        if (first) __syncthreads();  // the tile before has been written out
        Running<1, kDB> run;
        run.clear();
        int t = begin + wave;
        if (t < end) issue(t, 0);
        for (int buffer = 0; t < end; t += kWaves, buffer ^= 1) {
            if (t + kWaves < end) {
                issue(t + kWaves, buffer ^ 1);
                wait_vmcnt<2 * AttnTileCopy<E, DIM, kKeyRows, kWave>::kIssue>();  // this tile's, not the next one's
            } else {
                wait_vmcnt<0>();
            }
            asm volatile("" ::: "memory");
            const char *const kt = mine + buffer * F::kStage, *const vt = kt + kKeyRows * T::kRow;
            const int j0 = t * kKeyRows;
            f32x4 sc[2][1];
#pragma unroll
            for (int jb = 0; jb < 2; ++jb) {
                sc[jb][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < kKB; ++kk) sc[jb][0] = E::mfma(row_frag<E, DIM>(kt, 16 * jb, kk, lane), qf[kk], sc[jb][0]);
            }
            if constexpr (BIAS) {
                float b[2][4], most = 0.f;
#pragma unroll
                for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int far = min(max(j0 + 16 * jb + 4 * g + e - (token + offset), -a.reach), a.reach) + a.reach;
                        b[jb][e] = live ? a.bias[(size_t)head * (2 * a.reach + 1) + far] : 0.f;
                        most = fmaxf(most, fabsf(b[jb][e]));
                    }
                const bool large = __any(most > kLargeBias);
#pragma unroll
                for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)  // (rounded as in the other kernels)
                        sc[jb][0][e] = fmaf(sc[jb][0][e], a.scale2, large ? base2_bias(b[jb][e]) : b[jb][e] * kLog2E);
            }
            if (j0 + kKeyRows > full) {
                const int j = j0 + 4 * g;
#pragma unroll
                for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[jb][0][e] = j + 16 * jb + e < limit ? sc[jb][0][e] : -INFINITY;
            }
            run.template take<2>(sc, BIAS ? 1.f : a.scale2);
            const typename E::Frag pf = to_frag<E>(sc[0][0], sc[1][0]);
            typename E::Frag vf[kDB];
            col_frags_in_flight<E, DIM>(vt, lane, vf);
#pragma unroll
            for (int db = 0; db < kDB; ++db) run.o[0][db] = E::mfma(vf[db], pf, run.o[0][db]);
            // The next round's copy goes into the buffer just read.
            __builtin_amdgcn_s_waitcnt(0xC07F);
            asm volatile("" ::: "memory");
        }
        // The waves' sums at their common maximum, added in order.
        run.finish();
        if (g == 0) stat[wave][l16] = make_float2(run.m[0], run.l[0]);
        __syncthreads();
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stat[w][l16].x);
        const float at = top == -INFINITY ? 0.f : top;
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) total += stat[w][l16].y * exp2_raw(stat[w][l16].x - at);
        const float fade = exp2_raw(run.m[0] - at);
        float *const sums = reinterpret_cast<float *>(smem);  // [wave][16][DIM + 4]
#pragma unroll
        for (int db = 0; db < kDB; ++db)
            *reinterpret_cast<f32x4 *>(sums + (wave * 16 + l16) * (DIM + 4) + 16 * db + 4 * g) = run.o[0][db] * fade;
        __syncthreads();
        // Four elements of a row at a time: wave w has the blocks w, w + waves, ...
        const float inv = inverse(total);
        const size_t out_row = ((size_t)part * a.q_tokens + q_start + token) * a.heads + head;
#pragma unroll
        for (int b = 0; b < kDB; b += kWaves) {
            const int d = 16 * (b + wave) + 4 * g;
            if (b + wave >= kDB) break;
            f32x4 v = *reinterpret_cast<const f32x4 *>(sums + l16 * (DIM + 4) + d);
#pragma unroll
            for (int w = 1; w < kWaves; ++w) v += *reinterpret_cast<const f32x4 *>(sums + (w * 16 + l16) * (DIM + 4) + d);
            if (!live) continue;
            if (split) {
                *reinterpret_cast<f32x4 *>(a.part_out + out_row * DIM + d) = v;
            } else if (d < a.dim) {
                Words<E, 4> w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w.put(e, v[e] * inv);
                w.store(reinterpret_cast<typename E::Word *>(a.out.at((long long)q_start + token, head)) + d);
            }
        }
        if (wave == 0 && g == 0 && live) {
            if (split) a.part_stat[out_row] = make_float2(top, total);
            else if (a.lse) a.lse[(size_t)head * a.q_tokens + q_start + token] = natural_lse(top, total);
        }
    }
}

// Joins the parts' sums of each query and head: DIM / 4 threads, four elements
// each, times four shares of the parts, which are added up in order at the end.
// The parts are those that the kernel before dealt: of the keys that a tile of
// ROWS queries sees, or of all the sequence's keys (ROWS == 0).
template <class E, int DIM, int ROWS>
__global__ __launch_bounds__(256) void attention_join_kernel(AttnArgs a) {
    constexpr int kShares = 4, kPer = 256 * 4 / DIM / kShares;
    __shared__ float2 stat_part[kShares][kPer];
    __shared__ __attribute__((aligned(16))) float sums[kShares][kPer][DIM];
    const int q = threadIdx.x / (DIM / 4), share = q % kShares, i = q / kShares, d = threadIdx.x % (DIM / 4) * 4;
    // A workgroup's rows are neighbouring heads of one token.
    const int per_token = (a.heads + kPer - 1) / kPer, token = blockIdx.x / per_token;
    const int head = blockIdx.x % per_token * kPer + i;
    const int sequence = find_token(a.q_starts, a.sequences, a.q_tokens, token);
    if (sequence < 0) return;
    int q_start, q_len, k_start, k_len;
    sequence_rows(a.q_starts, sequence, a.q_tokens, q_start, q_len);
    sequence_rows(a.k_starts, sequence, a.k_tokens, k_start, k_len);
    if (ROWS == 0 && a.few_rows && q_len * (a.heads / a.kv_heads) > a.few_rows) return;
    int keys = k_len, size = 32, least = a.chunk / size;
    if constexpr (ROWS > 0) {
        const int tile = (token - q_start) / ROWS * ROWS;
        if (a.causal) keys = min(k_len, min(tile + ROWS, q_len) + k_len - q_len);
        size = kKeys;
        least = a.chunk;
    }
    const int tiles = keys > 0 ? (keys + size - 1) / size : 0, per = part_tiles(tiles, a.parts, least);
    const int used = max(1, (tiles + per - 1) / per);
    if (ROWS == 0 && used == 1) return;  // written by the kernel before
    const size_t step = (size_t)a.q_tokens * a.heads, row = (size_t)token * a.heads + min(head, a.heads - 1);
    const float2 *const stat = a.part_stat + row;
    const float *const out = a.part_out + row * DIM + d;
    float m = -INFINITY, l = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = share; p < used; p += kShares) {
        const float2 ml = stat[p * step];
        const f32x4 x = *reinterpret_cast<const f32x4 *>(out + p * step * DIM);
        const float to = fmaxf(m, ml.x), at = to == -INFINITY ? 0.f : to;
        const float old = exp2_raw(m - at), now = exp2_raw(ml.x - at);
        m = to;
        l = l * old + ml.y * now;
        v = v * old + x * now;
    }
    *reinterpret_cast<f32x4 *>(&sums[share][i][d]) = v;
    if (d == 0) stat_part[share][i] = make_float2(m, l);
    __syncthreads();
    if (share || head >= a.heads) return;
    float top = -INFINITY;
#pragma unroll
    for (int p = 0; p < kShares; ++p) top = fmaxf(top, stat_part[p][i].x);
    const float at = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < kShares; ++p) {
        const float f = exp2_raw(stat_part[p][i].x - at);
        total += stat_part[p][i].y * f;
        v += *reinterpret_cast<const f32x4 *>(&sums[p][i][d]) * f;
    }
    if (d < a.dim) {
        const float inv = inverse(total);
        Words<E, 4> w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.put(e, v[e] * inv);
        w.store(reinterpret_cast<typename E::Word *>(a.out.at(token, head)) + d);
    }
    if (a.lse && d == 0) a.lse[(size_t)head * a.q_tokens + token] = natural_lse(top, total);
}

// Queries of a workgroup: two blocks of 16 per wave, so that a fragment read from
// LDS serves two products; one for fp32, whose products take eight times as long
// as the reads.
constexpr int query_rows(int size) { return size == 4 ? 64 : 128; }

// How a call is dealt.  `few`: so few queries per sequence that a key head's
// group of them fills at most a tile of 16 rows on average, or one query each.
// Unless there are as many queries as sequences, the average says little of the
// longest (places of a batch may be empty): then (`mixed`) only the sequences of
// no more than few_rows rows are dealt so, and the others, prompts among single
// tokens, by a second launch.
// Heads of 128, bf16, 2000 keys per sequence, by this deal and by the prompts'
// launch alone: 32 heads on 8: 48 x 4 queries 98 and 178 us, 63 single tokens and
// a prompt of 100 164 and 229, 256 places with 25 single tokens and a prompt of
// 200 93 and 122, without the prompt 47 and 119; 32 heads on 32, where no head
// shares its keys, 63 and 100 423 and 363, but with 16000 keys in one sequence and
// 500 in the others 165 and 471.  Lengths are not known here, so the deal
// that bears uneven ones is taken.
// The keys are split into parts where the work would leave CUs idle: `few` takes
// parts of `chunk` keys, a 1536th of all that is read (a tile or more), so that
// about 1536 workgroups read keys whatever the lengths are, and a sequence has at
// most `parts` of them, whose sums take kPartBytes at most (which wide groups
// reach: 512 single tokens, 128 heads on one); otherwise a tile's keys are split
// into as many parts as bring about four workgroups per CU, but no more than the
// average sequence has keys for, four tiles or more in each.  fp32's products take
// eight times as long as other types', so that a walk costs more than a join
// where CUs are idle: parts of two tiles, as many as the longest sequence may have.
constexpr long long kPartBytes = 1ll << 30;

struct ForwardPlan {
    bool few, mixed;
    int rows, parts, chunk, dim, few_rows;
    long long slots, grid;
};

ForwardPlan forward_plan(const bfhip_attention_desc *d) {
    ForwardPlan p{};
    const int size = d->type == BFHIP_F32 ? 4 : 2, group = d->heads / d->kv_heads;
    p.dim = d->head_dim <= 32 ? 32 : d->head_dim <= 64 ? 64 : 128;
    p.parts = 1;
    if (!d->sequences || !d->q_tokens) return p;
    p.few_rows = group > 16 ? group : 16;
    p.few = d->q_tokens * group <= (long long)p.few_rows * d->sequences && d->q_tokens * group < 1 << 30;
    p.mixed = p.few && d->q_tokens != d->sequences;
    p.rows = query_rows(size);
    if (p.few) {
        const long long units = (long long)d->sequences * d->kv_heads, least = size * p.dim <= 128 ? 128 : 64;
        const long long chunk = (d->k_tokens * d->kv_heads / 1536 + least - 1) / least * least;
        p.chunk = (int)(chunk < least ? least : chunk > 1 << 20 ? 1 << 20 : chunk);
        const long long fit = kPartBytes / (d->q_tokens * d->heads * (long long)(p.dim * sizeof(float) + sizeof(float2)));
        p.parts = (int)std::max(1ll, std::min({32ll, d->k_tokens / p.chunk, 16384 / units, fit}));
        p.slots = slot_count(d->k_tokens, d->sequences, p.chunk);
        p.grid = p.slots * d->kv_heads;
        return p;
    }
    p.slots = slot_count(d->q_tokens, d->sequences, p.rows);
    // Slots are at most one per sequence more than there is work for.
    const long long tiles = (d->q_tokens + p.rows - 1) / p.rows;
    const long long units = (tiles > d->sequences ? tiles : d->sequences) * d->heads;
    const bool longest = size == 4 && units < 256;
    p.chunk = longest ? 2 : 4;
    const long long keys = (longest ? d->k_tokens : d->k_tokens / d->sequences) / (p.chunk * kKeys), parts = 1024 / units;
    p.parts = (int)(parts < 1 || keys < 1 ? 1 : parts < keys ? parts : keys);
    p.grid = p.slots * d->heads * p.parts;
    return p;
}

size_t part_rows(const bfhip_attention_desc *d, const ForwardPlan &p) {
    return p.parts > 1 ? (size_t)p.parts * d->q_tokens * d->heads : 0;
}

}  // namespace

extern "C" size_t bfhip_attention_forward_workspace(const bfhip_attention_desc *d) {
    if (bad_attention(d)) return 0;
    const ForwardPlan p = forward_plan(d);
    return part_rows(d, p) * (p.dim * sizeof(float) + sizeof(float2));
}

extern "C" int bfhip_attention_forward(const bfhip_attention_desc *d, const bfhip_rows *q, const bfhip_rows *k,
                                       const bfhip_rows *v, const bfhip_rows *out, float *lse, void *workspace,
                                       size_t workspace_bytes, void *stream, char *error, size_t cap) {
    if (bad_attention(d)) return fail(error, cap, "invalid attention contract");
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    if (bad_rows(q, d->q_tokens, d->head_dim, size) || bad_rows(k, d->k_tokens, d->head_dim, size) ||
        bad_rows(v, d->k_tokens, d->head_dim, size) ||
        bad_result(out, d->q_tokens, d->heads, d->head_dim, size))
        return fail(error, cap, "invalid attention rows: pointers and strides in steps of 16 bytes, token strides of at least head_dim, no results on one another");
    const ForwardPlan p = forward_plan(d);
    const size_t rows = part_rows(d, p), need = rows * (p.dim * sizeof(float) + sizeof(float2));
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
        return fail(error, cap, "attention workspace too small or not 16-byte aligned");
    if (!d->sequences || !d->q_tokens) return 1;
    const long long joins = p.parts > 1 ? ((long long)d->heads * p.dim + 255) / 256 * d->q_tokens : 0;
    const int least = p.few_rows / (d->heads / d->kv_heads) + 1;  // queries of a prompt
    const long long rest_slots = p.mixed ? (d->q_tokens + least - 1) / least : 0, rest = rest_slots * d->heads;
    if (!launch_fits(p.grid, 256) || !launch_fits(rest, 256) || !launch_fits(joins, 256)) return fail(error, cap, "attention has too many rows");
    AttnArgs a = attn_args(d, q, k, v, out, lse);
    a.slots = (int)p.slots;
    a.parts = p.parts;
    a.chunk = p.chunk;
    a.ordered = by_work(d, p.grid);
    a.few_rows = p.mixed ? p.few_rows : 0;
    // Scores are compared before they are scaled, which takes a positive scale:
    // a negative one flips the queries' signs, and zero becomes the smallest
    // number there is, with which no product that fp32 holds makes scores differ.
    a.flip = d->scale < 0.f;
    a.scale2 = d->scale == 0.f ? __FLT_DENORM_MIN__ : __builtin_fabsf(a.scale2);
    a.part_out = (float *)workspace;
    a.part_stat = (float2 *)(a.part_out + rows * p.dim);
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)p.grid);
    with_element(d->type, [&](auto e) {
        with_dim(d->head_dim, [&](auto n) {
            using E = decltype(e);
            constexpr int DIM = decltype(n)::value, ROWS = query_rows(E::kSize), IB = ROWS / 64;
            using Few = FewQueries<E, DIM>;
            using T = AttnTile<E, DIM>;
            const auto run = [&](auto bias) {
                constexpr bool B = decltype(bias)::value;
                const size_t lds = 4 * kKeys * T::kRow + (B ? BiasRow::floats(d->reach) * sizeof(float) : 0);
                if (p.few) hipLaunchKernelGGL((attention_few_kernel<E, DIM, B>), grid, dim3(Few::kThreads), 0, s, a);
                else hipLaunchKernelGGL((attention_forward_kernel<E, DIM, IB, B>), grid, dim3(256), lds, s, a);
                if (p.mixed) {
                    AttnArgs b = a;
                    b.slots = (int)rest_slots;
                    b.parts = 1;
                    hipLaunchKernelGGL((attention_forward_kernel<E, DIM, IB, B>), dim3((unsigned)rest), dim3(256), lds, s, b);
                }
            };
            if (d->bias) run(std::true_type{});
            else run(std::false_type{});
            if (p.parts == 1) return;
            const dim3 blocks((unsigned)joins);
            if (p.few) hipLaunchKernelGGL((attention_join_kernel<E, DIM, 0>), blocks, dim3(256), 0, s, a);
            else hipLaunchKernelGGL((attention_join_kernel<E, DIM, ROWS>), blocks, dim3(256), 0, s, a);
        });
    });
    return launch_ok(error, cap, "attention launch");
}
