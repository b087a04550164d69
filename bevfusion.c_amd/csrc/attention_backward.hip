// Attention over packed sequences, backward (include/bfhip_transformer.h).
//
// With p = 2^(s - lse) recomputed from the forward's lse (base 2 inside):
//   delta_i = dout_i . out_i,  ds_ij = p_ij (dout_i . v_j - delta_i),
//   dv_j = sum_i p_ij dout_i,  dk_j = scale sum_i ds_ij q_i,
//   dq_i = scale sum_j ds_ij k_j,  dbias[e] = sum of ds over pairs at e.
// Three launches: the row terms (delta and lse); dk and dv, a workgroup per
// tile of keys and key head that walks the queries of the group's heads; dq
// and dbias, a workgroup per tile of queries and head that walks the keys.
// Walking twice costs two products of seven more than adding dq up with
// atomics would, and gives the same bits every time.
#include <type_traits>

#include "attention.h"

using namespace bfhip;

namespace {

constexpr int kTile = 64;  // rows per LDS tile

struct GradArgs {
    AttnArgs f;
    AttnRows dout, dq, dk, dv;
    float *lse2, *delta;  // [heads, q_tokens]
    float *part;          // [query slots, heads, 2 reach + 1] or null
};

// lse in base 2, +inf for a query without keys (every p of it is then 0), and
// delta; 16 lanes per (token, head).
template <class E>
__global__ __launch_bounds__(256) void attention_terms_kernel(GradArgs a) {
    const long long id = (long long)blockIdx.x * 16 + threadIdx.x / 16;
    if (id >= a.f.q_tokens * a.f.heads) return;
    const long long t = id / a.f.heads;
    const int h = (int)(id % a.f.heads), d = 8 * (threadIdx.x % 16);
    float sum = 0.f;
    if (d < a.f.dim) {
        using W = Words<E, 8>;
        const W o = *reinterpret_cast<const W *>(__builtin_assume_aligned(a.f.out.at(t, h) + d * E::kSize, 16));
        const W g = *reinterpret_cast<const W *>(__builtin_assume_aligned(a.dout.at(t, h) + d * E::kSize, 16));
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(o.get(e), g.get(e), sum);
    }
    sum = group_sum<16>(sum);
    if (threadIdx.x % 16) return;
    const size_t at = (size_t)h * a.f.q_tokens + t;
    const float lse = a.f.lse[at];
    a.lse2[at] = lse == -INFINITY ? INFINITY : lse * kLog2E;
    a.delta[at] = sum;
}

// KB blocks of 16 keys per wave, four waves.  Scores come out with a key per
// lane, so P and dS are the second operands of dv^T = dout^T P and dk^T = q^T
// dS without leaving their registers.
template <class E, int DIM, int KB, bool BIAS>
__global__ __launch_bounds__(256, 1) void attention_keys_kernel(GradArgs a) {
    constexpr int kRows = 64 * KB, kKB = DIM / 32, kDB = DIM / 16;
    using T = AttnTile<E, DIM>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char *const qt = smem, *const gt = smem + kTile * T::kRow;
    float *const terms = reinterpret_cast<float *>(gt + kTile * T::kRow);  // lse2 [64], delta [64]
    float *const bias = terms + 2 * kTile;
    const AttnArgs &f = a.f;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, g = lane >> 4, group = f.heads / f.kv_heads;
    const int kv = blockIdx.x % f.kv_heads, slot_id = blockIdx.x / f.kv_heads;
    const Slot s = find_rows<kRows>(f.k_starts, f.sequences, f.k_tokens, slot_id);
    if (s.sequence < 0) return;
    int q_start, q_len;
    sequence_rows(f.q_starts, s.sequence, f.q_tokens, q_start, q_len);
    const int offset = s.length - q_len;
    const int key0 = s.first + wave * 16 * KB;

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
    AttnTileCopy<E, DIM, kTile, 256> qc, gc;
    qc.init(f.q.token, f.dim, threadIdx.x);
    gc.init(a.dout.token, f.dim, threadIdx.x);
    // The first query that sees the tile's first key.
    const int begin = f.causal ? max(0, s.first - offset) / kTile * kTile : 0;

    for (int hg = 0; hg < group; ++hg) {
        const int head = kv * group + hg;
        if constexpr (BIAS) {
            lds_barrier();
            const float *b = f.bias + (size_t)head * (2 * f.reach + 1);
            for (int i = threadIdx.x; i <= 2 * f.reach; i += 256) bias[i] = b[i] * kLog2E;
        }
        for (int i0 = begin; i0 < q_len; i0 += kTile) {
            lds_barrier();  // the tile before has been read
            qc.issue(f.q.at((long long)q_start + i0, head), q_len - i0, qt);
            gc.issue(a.dout.at((long long)q_start + i0, head), q_len - i0, gt);
            if (threadIdx.x < 2 * kTile) {
                const int i = threadIdx.x % kTile;
                const bool lse = threadIdx.x < kTile;
                const size_t at = (size_t)head * f.q_tokens + q_start + i0 + i;
                terms[threadIdx.x] = i0 + i < q_len ? (lse ? a.lse2 : a.delta)[at] : lse ? INFINITY : 0.f;
            }
            wait_vmcnt<0>();
            lds_barrier();
            // A query that does not see every key of the tile.
            const bool edge = f.causal && i0 + offset < key0 + 16 * KB - 1;
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
                    const f32x4 lse = *reinterpret_cast<const f32x4 *>(terms + r0 + 4 * g);
                    const f32x4 delta = *reinterpret_cast<const f32x4 *>(terms + kTile + r0 + 4 * g);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            // Position of the query before the key.
                            const int far = key0 + 16 * kb + l16 - (i0 + r0 + 4 * g + e + offset);
                            float x = p[b][kb][e] * f.scale2;
                            if constexpr (BIAS) x += bias[min(max(far, -f.reach), f.reach) + f.reach];
                            x = exp2_raw(x - lse[e]);
                            float y = x * (ds[b][kb][e] - delta[e]);
                            if (edge && far > 0) x = y = 0.f;
                            p[b][kb][e] = x;
                            ds[b][kb][e] = y;
                        }
                }
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const typename E::Frag pf = to_frag<E>(p[0][kb], p[1][kb]);
                    const typename E::Frag sf = to_frag<E>(ds[0][kb], ds[1][kb]);
#pragma unroll
                    for (int db = 0; db < kDB; ++db) {
                        dv[kb][db] = E::mfma(col_frag<E, DIM>(gt, 32 * c, db, lane), pf, dv[kb][db]);
                        dk[kb][db] = E::mfma(col_frag<E, DIM>(qt, 32 * c, db, lane), sf, dk[kb][db]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int r = key0 + 16 * kb + l16;
        const bool live = r < s.length;
        store_rows<E, kDB>(dk[kb], f.scale, a.dk.at((long long)s.start + r, kv), live, f.dim, lane);
        store_rows<E, kDB>(dv[kb], 1.f, a.dv.at((long long)s.start + r, kv), live, f.dim, lane);
    }
}

// Sums of a 16 x 16 block of dS^T along its diagonals into `sum` (this wave's
// own array): the lane (query i, group g) holds keys 4 g + e, so for one e the
// lanes (i + 4 n, g + n) lie on one diagonal; two shuffles add them up in the
// lane that starts the diagonal, and no two such lanes share an address.
// Distances at or beyond the reach are left to the caller's low and high sums.
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
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float v = ds[e], w = __shfl(v, (lane + 20) & 63);
        if (g < 3 && i < 12) v += w;
        w = __shfl(v, (lane + 40) & 63);
        if (g < 2 && i < 8) v += w;
        if (g == 0 || i < 4) {
            const int far = far0 + 4 * g + e - i;
            if (far <= -reach) low += v;
            else if (far >= reach) high += v;
            else __hip_atomic_fetch_add(sum + far + reach, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    }
}

// IB blocks of 16 queries per wave, four waves.
template <class E, int DIM, int IB, bool BIAS>
__global__ __launch_bounds__(256, 1) void attention_queries_kernel(GradArgs a) {
    constexpr int kRows = 64 * IB, kKB = DIM / 32, kDB = DIM / 16;
    using T = AttnTile<E, DIM>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char *const kt = smem, *const vt = smem + kTile * T::kRow;
    float *const bias = reinterpret_cast<float *>(vt + kTile * T::kRow);
    const AttnArgs &f = a.f;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % f.heads, slot_id = blockIdx.x / f.heads, kv = head / (f.heads / f.kv_heads);
    const int width = 2 * f.reach + 1;
    const Slot s = find_rows<kRows>(f.q_starts, f.sequences, f.q_tokens, slot_id);
    float *const part = BIAS && a.part ? a.part + (size_t)blockIdx.x * width : nullptr;
    if (s.sequence < 0) {
        if (part)
            for (int i = threadIdx.x; i < width; i += 256) part[i] = 0.f;
        return;
    }
    int k_start, k_len;
    sequence_rows(f.k_starts, s.sequence, f.k_tokens, k_start, k_len);
    const int offset = k_len - s.length, row0 = s.first + wave * 16 * IB;
    float *const sums = bias + width * (1 + wave);
    if constexpr (BIAS) {
        const float *b = f.bias + (size_t)head * width;
        for (int i = threadIdx.x; i < width; i += 256) bias[i] = b[i] * kLog2E;
        if (part)
            for (int i = lane; i < width; i += kWave) sums[i] = 0.f;
    }
    float low = 0.f, high = 0.f;

    typename E::Frag qf[IB][kKB], gf[IB][kKB];
    f32x4 dq[IB][kDB];
    float lse[IB], delta[IB];
    int limit[IB];
#pragma unroll
    for (int ib = 0; ib < IB; ++ib) {
        const int r0 = row0 + 16 * ib, r = r0 + l16;
#pragma unroll
        for (int kk = 0; kk < kKB; ++kk) {
            qf[ib][kk] = global_frag<E>(f.q.at((long long)s.start + r0, head), f.q.token, s.length - r0, f.dim, kk, lane);
            gf[ib][kk] = global_frag<E>(a.dout.at((long long)s.start + r0, head), a.dout.token, s.length - r0, f.dim, kk, lane);
        }
        const size_t at = (size_t)head * f.q_tokens + s.start + r;
        lse[ib] = r < s.length ? a.lse2[at] : INFINITY;
        delta[ib] = r < s.length ? a.delta[at] : 0.f;
        limit[ib] = f.causal ? min(k_len, r + offset + 1) : k_len;
#pragma unroll
        for (int db = 0; db < kDB; ++db) dq[ib][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int last = f.causal ? min(k_len, min(s.first + kRows, s.length) + offset) : k_len;
    const int full = f.causal ? min(k_len, row0 + offset + 1) : k_len;

    AttnTileCopy<E, DIM, kTile, 256> kc, vc;
    kc.init(f.k.token, f.dim, threadIdx.x);
    vc.init(f.v.token, f.dim, threadIdx.x);
    for (int j0 = 0; j0 < last; j0 += kTile) {
        lds_barrier();  // the tile before has been read
        kc.issue(f.k.at((long long)k_start + j0, kv), k_len - j0, kt);
        vc.issue(f.v.at((long long)k_start + j0, kv), k_len - j0, vt);
        wait_vmcnt<0>();
        lds_barrier();
        const bool edge = j0 + kTile > full;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            f32x4 p[2][IB], ds[2][IB];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int r0 = 32 * c + 16 * b;
#pragma unroll
                for (int ib = 0; ib < IB; ++ib) p[b][ib] = ds[b][ib] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < kKB; ++kk) {
                    const typename E::Frag kf = row_frag<E, DIM>(kt, r0, kk, lane);
#pragma unroll
                    for (int ib = 0; ib < IB; ++ib) p[b][ib] = E::mfma(kf, qf[ib][kk], p[b][ib]);
                }
#pragma unroll
                for (int kk = 0; kk < kKB; ++kk) {
                    const typename E::Frag vf = row_frag<E, DIM>(vt, r0, kk, lane);
#pragma unroll
                    for (int ib = 0; ib < IB; ++ib) ds[b][ib] = E::mfma(vf, gf[ib][kk], ds[b][ib]);
                }
#pragma unroll
                for (int ib = 0; ib < IB; ++ib) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = j0 + r0 + 4 * g + e;
                        float x = p[b][ib][e] * f.scale2;
                        if constexpr (BIAS) {
                            const int far = j - (row0 + 16 * ib + l16 + offset);
                            x += bias[min(max(far, -f.reach), f.reach) + f.reach];
                        }
                        float y = exp2_raw(x - lse[ib]) * (ds[b][ib][e] - delta[ib]);
                        if (edge && j >= limit[ib]) y = 0.f;
                        ds[b][ib][e] = y;
                    }
                    if constexpr (BIAS)
                        if (part) diagonal_sums(ds[b][ib], j0 + r0 - (row0 + 16 * ib + offset), f.reach, sums, low, high, lane);
                }
            }
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) {
                const typename E::Frag sf = to_frag<E>(ds[0][ib], ds[1][ib]);
#pragma unroll
                for (int db = 0; db < kDB; ++db)
                    dq[ib][db] = E::mfma(col_frag<E, DIM>(kt, 32 * c, db, lane), sf, dq[ib][db]);
            }
        }
    }
#pragma unroll
    for (int ib = 0; ib < IB; ++ib) {
        const int r = row0 + 16 * ib + l16;
        store_rows<E, kDB>(dq[ib], f.scale, a.dq.at((long long)s.start + r, head), r < s.length, f.dim, lane);
    }
    if constexpr (BIAS) {
        if (!part) return;
        low = group_sum<kWave>(low);
        high = group_sum<kWave>(high);
        if (lane == 0) {
            sums[0] += low;
            sums[2 * f.reach] += high;
        }
        lds_barrier();
        for (int i = threadIdx.x; i < width; i += 256) {
            const float *q = bias + width + i;
            part[i] = (q[0] + q[width]) + (q[2 * width] + q[3 * width]);
        }
    }
}

// dbias[h, i] = sum over the slots of part[slot, h, i].
__global__ __launch_bounds__(256) void attention_bias_sum_kernel(const float *part, float *dbias, long long n, int slots) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float sum = 0.f;
    for (int s = 0; s < slots; ++s) sum += part[s * n + i];
    dbias[i] = sum;
}

template <class E, int DIM>
constexpr int row_blocks() { return E::kSize == 4 && DIM == 128 ? 1 : 2; }

int query_rows(const bfhip_attention_desc *d) { return d->type == BFHIP_F32 && d->head_dim > 64 ? 64 : 128; }

size_t terms_bytes(const bfhip_attention_desc *d) {
    return ((size_t)d->heads * d->q_tokens * 2 * sizeof(float) + 255) / 256 * 256;
}

}  // namespace

extern "C" size_t bfhip_attention_backward_workspace(const bfhip_attention_desc *d) {
    if (bad_attention(d)) return 0;
    size_t n = terms_bytes(d);
    if (d->bias) n += (size_t)slot_count(d->q_tokens, d->sequences, query_rows(d)) * d->heads * (2 * d->reach + 1) * sizeof(float);
    return n;
}

extern "C" int bfhip_attention_backward(const bfhip_attention_desc *d, const bfhip_rows *q, const bfhip_rows *k,
                                        const bfhip_rows *v, const bfhip_rows *out, const float *lse,
                                        const bfhip_rows *dout, const bfhip_rows *dq, const bfhip_rows *dk,
                                        const bfhip_rows *dv, float *dbias, void *workspace, size_t workspace_bytes,
                                        void *stream, char *error, size_t cap) {
    if (bad_attention(d) || (dbias && !d->bias) || (!lse && d->q_tokens)) return fail(error, cap, "invalid attention contract");
    const int size = d->type == BFHIP_F32 ? 4 : 2, n = d->head_dim;
    if (bad_rows(q, d->q_tokens, n, size) || bad_rows(k, d->k_tokens, n, size) || bad_rows(v, d->k_tokens, n, size) ||
        bad_rows(out, d->q_tokens, n, size) || bad_rows(dout, d->q_tokens, n, size) || bad_rows(dq, d->q_tokens, n, size) ||
        bad_rows(dk, d->k_tokens, n, size) || bad_rows(dv, d->k_tokens, n, size))
        return fail(error, cap, "invalid attention rows: pointers and strides in steps of 16 bytes, token strides of at least head_dim");
    const size_t need = bfhip_attention_backward_workspace(d);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
        return fail(error, cap, "attention workspace too small or not 16-byte aligned");
    GradArgs a{};
    a.f = attn_args(d, q, k, v, out, const_cast<float *>(lse));
    a.dout = attn_rows(dout, d->q_tokens, n, size);
    a.dq = attn_rows(dq, d->q_tokens, n, size);
    a.dk = attn_rows(dk, d->k_tokens, n, size);
    a.dv = attn_rows(dv, d->k_tokens, n, size);
    a.lse2 = (float *)workspace;
    a.delta = a.lse2 + (size_t)d->heads * d->q_tokens;
    a.part = dbias ? (float *)((char *)workspace + terms_bytes(d)) : nullptr;
    hipStream_t s = (hipStream_t)stream;
    const long long terms = (d->q_tokens * d->heads + 15) / 16, width = 2 * a.f.reach + 1;
    int ok = launch_fits(terms, 256);
    long long q_slots = 0;
    with_element(d->type, [&](auto e) {
        with_dim(n, [&](auto dim) {
            using E = decltype(e);
            constexpr int DIM = decltype(dim)::value, RB = row_blocks<E, DIM>();
            q_slots = slot_count(d->q_tokens, d->sequences, 64 * RB);
            const long long q_grid = q_slots * d->heads;
            const long long k_grid = slot_count(d->k_tokens, d->sequences, 64 * RB) * d->kv_heads;
            ok = ok && launch_fits(q_grid, 256) && launch_fits(k_grid, 256);
            if (!ok) return;
            const size_t tiles = 2 * kTile * AttnTile<E, DIM>::kRow, terms_lds = 2 * kTile * sizeof(float);
            if (terms) hipLaunchKernelGGL(attention_terms_kernel<E>, dim3((unsigned)terms), dim3(256), 0, s, a);
            const auto run = [&](auto with_bias) {
                constexpr bool B = decltype(with_bias)::value;
                const size_t row = B ? width * sizeof(float) : 0;
                if (d->k_tokens && d->sequences)
                    hipLaunchKernelGGL((attention_keys_kernel<E, DIM, RB, B>), dim3((unsigned)k_grid), dim3(256),
                                       tiles + terms_lds + row, s, a);
                if (d->q_tokens && d->sequences)
                    hipLaunchKernelGGL((attention_queries_kernel<E, DIM, RB, B>), dim3((unsigned)q_grid), dim3(256),
                                       tiles + (a.part ? 5 : 1) * row, s, a);
            };
            if (d->bias) run(std::true_type{});
            else run(std::false_type{});
        });
    });
    if (!ok) return fail(error, cap, "attention has too many rows");
    if (dbias) {
        const long long count = width * d->heads;
        hipLaunchKernelGGL(attention_bias_sum_kernel, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, s, a.part,
                           dbias, count, d->q_tokens && d->sequences ? (int)q_slots : 0);
    }
    return launch_ok(error, cap, "attention launch");
}
