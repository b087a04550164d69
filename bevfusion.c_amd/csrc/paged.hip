// A paged cache of keys and values, and attention of new tokens over it
// (include/bfhip_transformer.h).
#include <algorithm>
#include <type_traits>

#include "attention.h"
#include "attention_running.h"

using namespace bfhip;

namespace {

constexpr int kKeys = 32;   // keys per tile
constexpr int kRows = 16;   // rows (token, head in group) per tile
constexpr int kFine = 16;   // units of time per key tile

struct PagedPool {
    char *data;
    long long page, token, head;  // bytes
    __device__ __forceinline__ char *at(long long id, int row, int h) const { return data + id * page + row * token + h * head; }
};

struct PagedArgs {
    AttnRows q, out;
    PagedPool k, v;
    const int *starts, *lengths, *table;
    const float *bias;
    float *lse;
    long long tokens, pages, table_stride;
    int sequences, heads, kv_heads, dim, page_size, table_pages, reach;
    float scale2;
    int flip;
    int shares;        // workgroups of a key head
    int least;         // key tiles' time of a share, at least
    int piece;         // key tiles that a row tile's beginning and end take the time of
    float *part_out;   // [2 shares][kv_heads][kRows][padded dim]
    float2 *part_stat; // [2 shares][kv_heads][kRows]
    long long *info;   // [sequences + 1]: first unit of each sequence that has some; units of a share
};

// Keys of sequence b.
__device__ __forceinline__ int cache_length(const PagedArgs &a, int b) {
    return min(max(a.lengths[b], 0), a.table_pages * a.page_size);
}

// Page of position j of sequence b, -1 where the table names none.
__device__ __forceinline__ int page_of(const PagedArgs &a, int b, int j) {
    const int id = a.table[b * a.table_stride + j / a.page_size];
    return id >= 0 && id < a.pages ? id : -1;
}

// ------------------------------------------------------------------- append
// A wave per token and turn: bound by memory (each row is read and written once:
// 12319 tokens, 8 heads of 128, fp16 21 us, 4.7 TB/s) and, for few tokens, by the latency of
// finding a token's place (48 tokens 4.4 us).
template <class E>
__global__ __launch_bounds__(256) void cache_append_kernel(PagedArgs a, AttnRows k, AttnRows v) {
    constexpr int kWords = 16 / E::kSize;
    using W = Words<E, kWords>;
    using Word = typename E::Word;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int chunks = a.dim / kWords, n = a.kv_heads * chunks;
    for (long long token = (long long)blockIdx.x * 4 + wave; token < a.tokens; token += (long long)gridDim.x * 4) {
        const int b = find_token(a.starts, a.sequences, a.tokens, (int)token);
        if (b < 0) continue;
        int start, length;
        sequence_rows(a.starts, b, a.tokens, start, length);
        const int j = cache_length(a, b) - length + ((int)token - start);
        if (j < 0) continue;
        const int id = page_of(a, b, j), row = j % a.page_size;
        if (id < 0) continue;
        for (int i = lane; i < 2 * n; i += kWave) {
            const bool second = i >= n;
            const int c = second ? i - n : i, head = c / chunks, at = (c - head * chunks) * kWords;
            const W w = W::load((const Word *)(second ? v : k).at(token, head) + at);
            w.store((Word *)(second ? a.v : a.k).at(id, row, head) + at);
        }
    }
}

// ---------------------------------------------------------------- attention
// How the work is dealt.  Lengths are on the device alone, so every workgroup
// works the deal out for itself.  Sequence b has row tiles (16 rows, token * group +
// head in group) and key tiles; a row tile takes kFine units of time for each of its key
// tiles and `piece` tiles' for its queries' way in and its results' way out.  Units, row tile after row
// tile, sequence after sequence, are dealt in equal shares, one per workgroup
// that the chip holds at once, whatever the lengths are.  So a share has whole row
// tiles and at most one that an earlier share began and one that it leaves to a
// later one: two places for sums that are to be joined.  (A sequence without new
// tokens has no units.)
struct SequenceWork {
    int start, queries, keys, row_tiles, tiles, piece;
    __device__ __forceinline__ int cost() const { return (tiles + piece) * kFine; }  // below 2^31: tiles of 32 keys
    __device__ __forceinline__ long long units() const { return (long long)row_tiles * cost(); }
    // Key tiles up to unit x of a row tile.
    __device__ __forceinline__ int tile(int x) const { return (int)((long long)x * tiles / cost()); }
};

// (All loads come before the first use, so that they wait together.)
__device__ __forceinline__ SequenceWork sequence_work(const PagedArgs &a, int b) {
    if (b >= a.sequences) return SequenceWork{0, 0, 0, 0, 0, a.piece};
    const int first = a.starts[b], next = a.starts[b + 1], length = a.lengths[b];
    const long long s = min(max((long long)first, 0ll), a.tokens), e = min(max((long long)next, 0ll), a.tokens);
    const int queries = (int)(e > s ? e - s : 0), keys = queries ? min(max(length, 0), a.table_pages * a.page_size) : 0;
    return SequenceWork{(int)s, queries, keys, (int)(((long long)queries * (a.heads / a.kv_heads) + kRows - 1) / kRows),
                        (keys + kKeys - 1) / kKeys, a.piece};
}

// The sequences from the one that a share begins in, 64 at a time, a lane each.
struct Sequences {
    int first, at;           // the lanes' first sequence, and the lane in turn
    SequenceWork lane_work;  // of the lane's sequence
    long long lane_upto;     // units up to its end

    // Units of the sequences before the lanes' in `before`.
    __device__ __forceinline__ void load(const PagedArgs &a, int b, long long before) {
        const int lane = threadIdx.x % kWave;
        first = b;
        lane_work = sequence_work(a, b + lane);
        lane_upto = lane_work.units();
#pragma unroll
        for (int o = 1; o < kWave; o *= 2) {
            const long long x = __shfl_up(lane_upto, o);
            if (lane >= o) lane_upto += x;
        }
        lane_upto += before;
    }
    __device__ __forceinline__ static long long read(long long v, int lane) {
        return (long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)v, lane) |
                           (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32);
    }
    __device__ __forceinline__ SequenceWork work() const {
        return SequenceWork{__builtin_amdgcn_readlane(lane_work.start, at), __builtin_amdgcn_readlane(lane_work.queries, at),
                            __builtin_amdgcn_readlane(lane_work.keys, at), __builtin_amdgcn_readlane(lane_work.row_tiles, at),
                            __builtin_amdgcn_readlane(lane_work.tiles, at), lane_work.piece};
    }
    __device__ __forceinline__ long long upto() const { return read(lane_upto, at); }
    // Turns to the sequence that holds `unit`, from the lanes' on; false if none does.
    __device__ __forceinline__ bool seek(const PagedArgs &a, long long unit) {
        for (;;) {
            const unsigned long long in = __ballot(unit < lane_upto);
            if (in) {
                at = (int)__builtin_ctzll(in);
                return true;
            }
            if (first + kWave >= a.sequences) return false;
            load(a, first + kWave, read(lane_upto, kWave - 1));
        }
    }
};

// Units of a share; `at` holds the first sequences.
__device__ __forceinline__ long long share_units(const PagedArgs &a, const Sequences &at) {
    if (a.shares == 1) return 0x7fffffffffffffffll;
    long long total = Sequences::read(at.lane_upto, kWave - 1);
    if (a.sequences > kWave) {
        long long rest = 0;
        for (int b = kWave + threadIdx.x % kWave; b < a.sequences; b += kWave) rest += sequence_work(a, b).units();
#pragma unroll
        for (int o = 1; o < kWave; o *= 2) rest += __shfl_xor(rest, o);
        total += Sequences::read(rest, 0);
    }
    const long long share = (total + a.shares - 1) / a.shares;
    return share > a.least * kFine ? share : a.least * kFine;
}

// What a lane reads in place of a row that is not there.
__device__ __attribute__((aligned(16))) const uint32_t no_row[4] = {0, 0, 0, 0};

// One 16-byte LDS-DMA per lane, each from an address of its own: LDS[lds + 16 *
// lane] = *p.
__device__ __forceinline__ void dma16_from(const char *p, char *lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)p,
                                     (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

template <class E, int DIM>
struct PagedTile {
    using T = AttnTile<E, DIM>;
    static constexpr int kStage = 2 * kKeys * T::kRow;     // K and V of a tile
    static constexpr int kWaves = kStage <= 8192 ? 4 : 2;  // two workgroups per CU (one for long fp32 rows)
    static constexpr int kThreads = kWaves * kWave;
    static constexpr int kIssue = kKeys * T::kChunks / kWave;  // copies of one of the two
};

// Bound by reading the keys and values once (131071 keys, 32 heads on 8 of 128, bf16: 107
// us, 5.0 TB/s, and 5 us for the join).  A workgroup has a share of the units
// of one key head, whose whole group of query heads shares each tile.  Each wave
// walks tiles of its own, 32 keys at a time, through its own two LDS buffers, two
// tiles in flight, without a barrier; the waves' sums are joined at a row tile's
// end.  Rows of a tile may lie in different pages, so every lane copies from an
// address of its own: lane r knows the page of row r, loaded a tile ahead.
template <class E, int DIM, bool BIAS>
struct PagedWalk {
    using P = PagedTile<E, DIM>;
    using T = typename P::T;
    static constexpr int kKB = DIM / 32, kDB = DIM / 16, kWaves = P::kWaves;
    const PagedArgs &a;
    char *smem;
    int kv, share, lane, wave;

    // Row tile `row_tile` of sequence b, its units x0 .. x1.
    __device__ __forceinline__ void piece(int b, const SequenceWork &s, int row_tile, int x0, int x1) {
        float2(*const stat)[kRows] = reinterpret_cast<float2(*)[kRows]>(smem + kWaves * 2 * P::kStage);
        const int l16 = lane & 15, g = lane >> 4, group = a.heads / a.kv_heads;
        const bool whole = x0 == 0 && x1 == s.cost();
        const int t0 = s.tile(x0), t1 = s.tile(x1);
        const int q_start = s.start, k_len = s.keys, rows = s.queries * group;
        const int offset = k_len - s.queries, first = row_tile * kRows;

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
        const int limit = min(k_len, token + offset + 1);  // keys that the lane's row sees
        const int last = min(k_len, (min(first + kRows, rows) - 1) / group + 1 + offset);
        const int full = min(k_len, first / group + offset + 1);
        const int end = min(last > 0 ? (last + kKeys - 1) / kKeys : 0, t1);

        char *const mine = smem + wave * 2 * P::kStage;
        const int *const table = a.table + b * a.table_stride;
        // The page of row lane % 32 of tile t.
        const auto page = [&](int t) {
            const int j = t * kKeys + lane % kKeys;
            return t < end && j < last ? table[j / a.page_size] : -1;
        };
        const auto issue = [&](int t, int ids, int buffer) {
            const int in = (t * kKeys + lane % kKeys) % a.page_size;
            char *const to = mine + buffer * P::kStage;
#pragma unroll
            for (int i = 0; i < P::kIssue; ++i) {
                const int id = i * kWave + lane, r = id / T::kChunks;
                const int c = 16 * ((id % T::kChunks) ^ T::swizzle(r));
                const int pg = __shfl(ids, r), at = __shfl(in, r);
                const bool there = pg >= 0 && pg < a.pages && c < a.dim * E::kSize;
                dma16_from(there ? a.k.at(pg, at, kv) + c : (const char *)no_row, to + i * kWave * 16);
                dma16_from(there ? a.v.at(pg, at, kv) + c : (const char *)no_row, to + kKeys * T::kRow + i * kWave * 16);
            }
        };
        Running<1, kDB> run;
        // Probabilities meet the values rounded to the type and with what their rounding
        // left, or it would add as much again to the results' error as their own rounding
        // has: bf16, random values, 0.0023 of the results' norm, 0.0017 with it.  (One
        // sequence of 131071 keys 113 us, 109 without; 48 mixed ones 110 and 107; 3 tokens
        // for each of 100 50.6 and 50.1.)  An infinite value would meet parts of both signs:
        // sums that are not finite are found again without what was left.
        f32x4 finite[kDB];
        for (bool left_too = E::kSize == 2;; left_too = false) {
            int t = t0 + wave;
            run.clear();
            int ids = page(t);
            uint32_t there = 0;  // keys of the tile that have a page
            if (t < end) {
                there = (uint32_t)__ballot(ids >= 0 && ids < a.pages);
                issue(t, ids, 0);
            }
            ids = page(t + kWaves);
            for (int buffer = 0; t < end; t += kWaves, buffer ^= 1) {
                uint32_t next_there = 0;
                if (t + kWaves < end) {
                    const int now = ids;
                    ids = page(t + 2 * kWaves);
                    next_there = (uint32_t)__ballot(now >= 0 && now < a.pages);
                    issue(t + kWaves, now, buffer ^ 1);
                    wait_vmcnt<(2 * P::kIssue > 63 ? 63 : 2 * P::kIssue)>();  // this tile's, not the next one's
                } else {
                    wait_vmcnt<0>();
                }
                asm volatile("" ::: "memory");
                const char *const kt = mine + buffer * P::kStage, *const vt = kt + kKeys * T::kRow;
                const int j0 = t * kKeys;
                f32x4 sc[2][1];
#pragma unroll
                for (int jb = 0; jb < 2; ++jb) {
                    sc[jb][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kk = 0; kk < kKB; ++kk) sc[jb][0] = E::mfma(row_frag<E, DIM>(kt, 16 * jb, kk, lane), qf[kk], sc[jb][0]);
                }
                if constexpr (BIAS) {
#pragma unroll
                    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int far = min(max(j0 + 16 * jb + 4 * g + e - (token + offset), -a.reach), a.reach) + a.reach;
                            const float bias = live ? a.bias[(size_t)head * (2 * a.reach + 1) + far] : 0.f;
                            sc[jb][0][e] = fmaf(sc[jb][0][e], a.scale2, base2_bias(bias));
                        }
                }
                if (j0 + kKeys > full || there != ~0u) {
#pragma unroll
                    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = 16 * jb + 4 * g + e;
                            sc[jb][0][e] = j0 + j < limit && (there >> j & 1) ? sc[jb][0][e] : -INFINITY;
                        }
                }
                there = next_there;
                run.template take<2>(sc, BIAS ? 1.f : a.scale2);
                const typename E::Frag pf = to_frag<E>(sc[0][0], sc[1][0]);
                typename E::Frag vf[kDB];
                col_frags_in_flight<E, DIM>(vt, lane, vf);
#pragma unroll
                for (int db = 0; db < kDB; ++db) run.o[0][db] = E::mfma(vf[db], pf, run.o[0][db]);
                if (left_too) {  // (probabilities are at most 2^8 or NaN)
                    typedef typename E::Word Words8 __attribute__((ext_vector_type(8)));
                    const f32x8 taken = __builtin_convertvector(__builtin_bit_cast(Words8, pf), f32x8);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[0][0][e] -= taken[e];
                        sc[1][0][e] -= taken[e + 4];
                    }
                    const typename E::Frag left = to_frag<E>(sc[0][0], sc[1][0]);
#pragma unroll
                    for (int db = 0; db < kDB; ++db) run.o[0][db] = E::mfma(vf[db], left, run.o[0][db]);
                }
                // The next round's copy goes into the buffer just read.
                __builtin_amdgcn_s_waitcnt(0xC07F);
                asm volatile("" ::: "memory");
            }
            if (E::kSize == 4) break;
            if (!left_too) {
#pragma unroll
                for (int db = 0; db < kDB; ++db)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        run.o[0][db][e] = fabsf(finite[db][e]) < INFINITY ? finite[db][e] : run.o[0][db][e];
                break;
            }
            float none = 0.f;
#pragma unroll
            for (int db = 0; db < kDB; ++db) {
                finite[db] = run.o[0][db];
#pragma unroll
                for (int e = 0; e < 4; ++e) none = fmaf(finite[db][e], 0.f, none);
            }
            if (!__any(none != 0.f)) break;
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
        const float inv = inverse(total);
        const size_t part_row = ((size_t)(2 * share + (x0 == 0)) * a.kv_heads + kv) * kRows + l16;
#pragma unroll
        for (int d0 = 0; d0 < kDB; d0 += kWaves) {
            const int d = 16 * (d0 + wave) + 4 * g;
            if (d0 + wave >= kDB) break;
            f32x4 v = *reinterpret_cast<const f32x4 *>(sums + l16 * (DIM + 4) + d);
#pragma unroll
            for (int w = 1; w < kWaves; ++w) v += *reinterpret_cast<const f32x4 *>(sums + (w * 16 + l16) * (DIM + 4) + d);
            if (!live) continue;
            if (!whole) {
                *reinterpret_cast<f32x4 *>(a.part_out + part_row * DIM + d) = v;
            } else if (d < a.dim) {
                Words<E, 4> w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w.put(e, v[e] * inv);
                w.store(reinterpret_cast<typename E::Word *>(a.out.at((long long)q_start + token, head)) + d);
            }
        }
        if (wave == 0 && g == 0 && live) {
            if (!whole) a.part_stat[part_row] = make_float2(top, total);
            else if (a.lse) a.lse[(size_t)head * a.tokens + q_start + token] = natural_lse(top, total);
        }
    }
};

template <class E, int DIM, bool BIAS>
__global__ __launch_bounds__(256, 1) void paged_attention_kernel(PagedArgs a) {
    using Walk = PagedWalk<E, DIM, BIAS>;
    // One LDS object: with two the compiler waits for every copy in flight
    // before any LDS read.
    __shared__ __attribute__((aligned(16))) char smem[Walk::kWaves * (2 * Walk::P::kStage + kRows * sizeof(float2))];
    Walk walk{a, smem, (int)blockIdx.x % a.kv_heads, (int)blockIdx.x / a.kv_heads, (int)threadIdx.x % kWave,
              __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)};
    Sequences at;
    at.load(a, 0, 0);
    const long long units = share_units(a, at);
    long long u = walk.share * units;
    const long long end = a.shares == 1 ? units : u + units;
    const bool writes = a.info && walk.kv == 0 && threadIdx.x == 0;
    if (writes && walk.share == 0) a.info[a.sequences] = units;
    while (u < end && at.seek(a, u)) {
        const SequenceWork s = at.work();
        const long long begin = at.upto() - s.units(), in = u - begin;
        const int row_tile = (int)(in / s.cost()), x0 = (int)(in - (long long)row_tile * s.cost());
        const int x1 = (int)min((long long)s.cost(), x0 + (end - u));
        if (writes && in == 0) a.info[at.first + at.at] = begin;
        walk.piece(at.first + at.at, s, row_tile, x0, x1);
        u += x1 - x0;
        __syncthreads();  // the sums have been read
    }
}

// Joins the parts' sums of each query and head: DIM / 4 threads, four elements
// each, times eight (or fewer) of the parts, which are added up in order at the end.
// The launch's tokens begin at first_token.
template <class E, int DIM>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, int first_token) {
    constexpr int kShares = 8, kPer = 256 * 4 / DIM / kShares;
    __shared__ float2 stat_part[kShares][kPer];
    __shared__ __attribute__((aligned(16))) float sums[kShares][kPer][DIM];
    const int q = threadIdx.x / (DIM / 4), share = q % kShares, i = q / kShares, d = threadIdx.x % (DIM / 4) * 4;
    // A workgroup's rows are neighbouring heads of one token.
    const int per_token = (a.heads + kPer - 1) / kPer, token = first_token + blockIdx.x / per_token;
    const int head = blockIdx.x % per_token * kPer + i, group = a.heads / a.kv_heads;
    const int sequence = find_token(a.starts, a.sequences, a.tokens, token);
    if (sequence < 0) return;
    const long long units = a.info[a.sequences], first = a.info[sequence];
    const SequenceWork s = sequence_work(a, sequence);
    const int kv = min(head, a.heads - 1) / group, row = (token - s.start) * group + min(head, a.heads - 1) % group;
    // Shares that have units of the row's tile: the first in their second place, the
    // others in their first.  (Where starts descend, a row's sequence need not be one
    // that was dealt: any place within the workspace will do then.)
    const long long begin = first + (long long)(row / kRows) * s.cost();
    const long long from = begin / units, to = (begin + s.cost() - 1) / units;
    // (One share has written the result.  Heads of a workgroup may end here apart, for
    // they can lie in different row tiles: a head has whole waves, and the barrier
    // waits for those that have not ended.)
    static_assert(kShares * (DIM / 4) % kWave == 0, "whole waves per head");
    if (from == to || from < 0 || to >= a.shares) return;
    const int parts = (int)(to - from) + 1;
    const size_t step = (size_t)a.kv_heads * kRows, place = (size_t)kv * kRows + row % kRows;
    float m = -INFINITY, l = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = share; p < parts; p += kShares) {
        const size_t at_row = (2 * (size_t)(from + p) + (p == 0)) * step + place;
        const float2 ml = a.part_stat[at_row];
        const f32x4 x = *reinterpret_cast<const f32x4 *>(a.part_out + at_row * DIM + d);
        const float top = fmaxf(m, ml.x), at = top == -INFINITY ? 0.f : top;
        const float old = exp2_raw(m - at), now = exp2_raw(ml.x - at);
        m = top;
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
    if (a.lse && d == 0) a.lse[(size_t)head * a.tokens + token] = natural_lse(top, total);
}

// ------------------------------------------------------------------ the host
bool bad_paged(const bfhip_paged_desc *d) {
    return !d || d->type < BFHIP_F32 || d->type > BFHIP_BF16 || d->sequences < 0 || d->kv_heads <= 0 || d->kv_heads > 65535 ||
           d->head_dim <= 0 || d->head_dim > 128 || d->head_dim % 8 || d->page_size <= 0 || d->table_pages < 0 ||
           (long long)d->page_size * d->table_pages > kMostTokens || d->tokens < 0 || d->tokens > kMostTokens || d->pages < 0 ||
           d->pages > kMostTokens || d->table_stride < 0 || (d->sequences > 1 && d->table_stride < d->table_pages) ||
           (d->sequences && (!d->starts || !d->lengths || (!d->table && d->table_pages)));
}

bool bad_paged_queries(const bfhip_paged_desc *d) {
    return d->heads <= 0 || d->heads > 65535 || d->heads % d->kv_heads || !(d->scale == d->scale) ||
           __builtin_isinf(d->scale) || (d->bias && (d->reach < 0 || d->reach > 2047));
}

bool bad_pages(const bfhip_pages *p, const bfhip_paged_desc *d) {
    if (!p || (!p->data && d->pages)) return true;
    const long long step = 16 / (d->type == BFHIP_F32 ? 4 : 2);
    const auto bad = [&](long long n, long long stride) { return n > 1 && (stride < 0 || stride % step); };
    return ((uintptr_t)p->data & 15) || bad(d->pages, p->page_stride) || bad(d->page_size, p->token_stride) ||
           bad(d->kv_heads, p->head_stride);
}

// Whether two heads' rows of a pool share memory: strides from the smallest up
// have to step over what those before them span.
bool pages_overlap(const bfhip_pages *p, const bfhip_paged_desc *d) {
    std::pair<long long, long long> s[3] = {{p->page_stride, d->pages}, {p->token_stride, d->page_size}, {p->head_stride, d->kv_heads}};
    std::sort(s, s + 3);
    long long span = d->head_dim;
    for (const auto &[stride, n] : s) {
        if (n <= 1) continue;
        if (stride < span) return true;
        span += stride * (n - 1);
    }
    return false;
}

PagedPool pool(const bfhip_pages *p, int size) {
    return PagedPool{(char *)p->data, p->page_stride * size, p->token_stride * size, p->head_stride * size};
}

PagedArgs paged_args(const bfhip_paged_desc *d, const bfhip_pages *k, const bfhip_pages *v) {
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    PagedArgs a{};
    a.k = pool(k, size);
    a.v = pool(v, size);
    a.starts = d->starts;
    a.lengths = d->lengths;
    a.table = d->table;
    a.bias = d->bias;
    a.tokens = d->tokens;
    a.pages = d->pages;
    a.table_stride = d->table_stride;
    a.sequences = d->sequences;
    a.heads = d->heads;
    a.kv_heads = d->kv_heads;
    a.dim = d->head_dim;
    a.page_size = d->page_size;
    a.table_pages = d->table_pages;
    a.reach = d->bias ? d->reach : 0;
    return a;
}

struct PagedPlan {
    int dim, shares, least, piece;
    size_t bytes;
};

// Shares of a key head: as many as make the workgroups that the chip holds at once,
// two per CU (one for long fp32 rows; there is room for four of 16-bit heads of up to 32,
// which get two all the same).  Heads of 128, 32 on 8, bf16, with probabilities rounded once:
// one sequence of 131071 keys 108 us, 48 of 1 to 16384 107 (with three times as many, cut at
// whole tiles, 131 and 129).
PagedPlan paged_plan(const bfhip_paged_desc *d) {
    PagedPlan p{};
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    p.dim = d->head_dim <= 32 ? 32 : d->head_dim <= 64 ? 64 : 128;
    if (!d->sequences || !d->tokens) return p;
    p.least = size * p.dim <= 128 ? 4 : 2;
    // A row tile's beginning and end take about as long as 64 KiB of keys and values
    // (3 tokens for each of 100 sequences of 3 to 1500 keys, 12 heads of 64: 45 us, 82
    // where they are not counted and a share of short sequences has many of them).
    p.piece = (64 << 10) / (2 * kKeys * size * p.dim);
    p.shares = std::max(1, (size * p.dim > 256 ? 256 : 512) / d->kv_heads);
    const size_t rows = (size_t)2 * p.shares * d->kv_heads * kRows;
    if (p.shares > 1) p.bytes = rows * (p.dim * sizeof(float) + sizeof(float2)) + ((size_t)d->sequences + 1) * sizeof(long long);
    return p;
}

}  // namespace

extern "C" int bfhip_cache_append(const bfhip_paged_desc *d, const bfhip_rows *k, const bfhip_rows *v, const bfhip_pages *k_pages,
                                  const bfhip_pages *v_pages, void *stream, char *error, size_t cap) {
    if (bad_paged(d)) return fail(error, cap, "invalid paged cache contract");
    if (bad_pages(k_pages, d) || bad_pages(v_pages, d))
        return fail(error, cap, "invalid cache pages: pointers and strides in steps of 16 bytes");
    if (pages_overlap(k_pages, d) || pages_overlap(v_pages, d)) return fail(error, cap, "cache pages on one another");
    const auto bad = [&](const bfhip_rows *r) {
        return !r || (!r->data && d->tokens) || (d->tokens > 1 && r->token_stride < 0) || (d->kv_heads > 1 && r->head_stride < 0);
    };
    if (bad(k) || bad(v)) return fail(error, cap, "invalid cache rows");
    if (!d->sequences || !d->tokens || !d->table_pages || !d->pages) return 1;
    PagedArgs a = paged_args(d, k_pages, v_pages);
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    const auto rows = [&](const bfhip_rows *r) {
        return AttnRows{(char *)r->data, d->tokens > 1 ? r->token_stride * size : 0, d->kv_heads > 1 ? r->head_stride * size : 0};
    };
    const long long grid = std::min((d->tokens + 3) / 4, 65536ll);
    with_element(d->type, [&](auto e) {
        hipLaunchKernelGGL(cache_append_kernel<decltype(e)>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a, rows(k), rows(v));
    });
    return launch_ok(error, cap, "cache append launch");
}

extern "C" size_t bfhip_paged_attention_workspace(const bfhip_paged_desc *d) {
    if (bad_paged(d) || bad_paged_queries(d)) return 0;
    return paged_plan(d).bytes;
}

extern "C" int bfhip_paged_attention(const bfhip_paged_desc *d, const bfhip_rows *q, const bfhip_pages *k_pages,
                                     const bfhip_pages *v_pages, const bfhip_rows *out, float *lse, void *workspace,
                                     size_t workspace_bytes, void *stream, char *error, size_t cap) {
    if (bad_paged(d) || bad_paged_queries(d)) return fail(error, cap, "invalid paged attention contract");
    if (bad_pages(k_pages, d) || bad_pages(v_pages, d))
        return fail(error, cap, "invalid cache pages: pointers and strides in steps of 16 bytes");
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    if (bad_rows(q, d->tokens, d->head_dim, size) || bad_result(out, d->tokens, d->heads, d->head_dim, size))
        return fail(error, cap, "invalid attention rows: pointers and strides in steps of 16 bytes, token strides of at least head_dim, no results on one another");
    if (d->tokens * (d->heads / d->kv_heads) > 1 << 30) return fail(error, cap, "paged attention has too many rows");
    const PagedPlan p = paged_plan(d);
    const size_t need = p.bytes;
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
        return fail(error, cap, "paged attention workspace too small or not 16-byte aligned");
    if (!d->sequences || !d->tokens) return 1;
    const long long grid = (long long)p.shares * d->kv_heads, per_token = (d->heads * p.dim + 127) / 128;
    const long long at_once = (1ll << 23) / per_token;  // tokens that a launch joins: it holds 2^24 - 1 workgroups
    PagedArgs a = paged_args(d, k_pages, v_pages);
    a.q = attn_rows(q, d->tokens, d->head_dim, size);
    a.out = attn_rows(out, d->tokens, d->head_dim, size);
    a.lse = lse;
    // Scores are compared before they are scaled: see bfhip_attention_forward.
    a.flip = d->scale < 0.f;
    a.scale2 = d->scale == 0.f ? __FLT_DENORM_MIN__ : __builtin_fabsf(d->scale * kLog2E);
    a.shares = p.shares;
    a.least = p.least;
    a.piece = p.piece;
    if (need) {
        const size_t rows = (size_t)2 * p.shares * d->kv_heads * kRows;
        a.part_out = (float *)workspace;
        a.part_stat = (float2 *)(a.part_out + rows * p.dim);
        a.info = (long long *)(a.part_stat + rows);
    }
    hipStream_t s = (hipStream_t)stream;
    with_element(d->type, [&](auto e) {
        with_dim(d->head_dim, [&](auto n) {
            using E = decltype(e);
            constexpr int DIM = decltype(n)::value;
            constexpr int kThreads = PagedTile<E, DIM>::kThreads;
            if (d->bias) hipLaunchKernelGGL((paged_attention_kernel<E, DIM, true>), dim3((unsigned)grid), dim3(kThreads), 0, s, a);
            else hipLaunchKernelGGL((paged_attention_kernel<E, DIM, false>), dim3((unsigned)grid), dim3(kThreads), 0, s, a);
            for (long long t = 0; need && t < d->tokens; t += at_once)
                hipLaunchKernelGGL((paged_join_kernel<E, DIM>), dim3((unsigned)(per_token * std::min(at_once, d->tokens - t))), dim3(256), 0, s, a, (int)t);
        });
    });
    return launch_ok(error, cap, "paged attention launch");
}
