// Attention over packed sequences, forward (include/bfhip_transformer.h).
//
// One pass over the keys with a running maximum m and sum l per query, in base
// 2 (scores carry log2 e): for each tile of 64 keys
//   S^T = K Q^T, m' = max(m, S), P = 2^(S - m'), l = l 2^(m - m') + sum P,
//   O^T = O^T 2^(m - m') + V^T P^T,
// then O / l and lse = (m + log2 l) ln 2.  Scores come out transposed, so a
// lane holds scores of one query only: the row statistics are one value per
// lane, and P is the second product's operand without leaving its registers.
#include <type_traits>

#include "attention.h"

using namespace bfhip;

namespace {

constexpr int kKeys = 64;  // keys per tile

// IB blocks of 16 queries per wave, four waves.
template <class E, int DIM, int IB, bool BIAS>
__global__ __launch_bounds__(256, 1) void attention_forward_kernel(AttnArgs a) {
    constexpr int kRows = 64 * IB, kKB = DIM / 32, kDB = DIM / 16;
    using T = AttnTile<E, DIM>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char *const kt = smem, *const vt = smem + kKeys * T::kRow;
    float *const bias = reinterpret_cast<float *>(vt + kKeys * T::kRow);
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % a.heads, slot_id = blockIdx.x / a.heads, kv = head / (a.heads / a.kv_heads);
    const Slot s = find_slot<kRows>(a.q_starts, a.sequences, a.q_tokens, slot_id);
    if (s.sequence < 0) return;
    int k_start, k_len;
    sequence_rows(a.k_starts, s.sequence, a.k_tokens, k_start, k_len);
    const int offset = k_len - s.length;  // query i stands at position i + offset

    if constexpr (BIAS) {
        const float *b = a.bias + (size_t)head * (2 * a.reach + 1);
        for (int i = threadIdx.x; i <= 2 * a.reach; i += 256) bias[i] = b[i] * kLog2E;
    }
    const int row0 = s.first + wave * 16 * IB;  // this wave's first query
    typename E::Frag qf[IB][kKB];
    int limit[IB];  // keys that the lane's query sees
#pragma unroll
    for (int ib = 0; ib < IB; ++ib) {
        const int r0 = row0 + 16 * ib;
        const char *q = a.q.at((long long)s.start + r0, head);
#pragma unroll
        for (int kk = 0; kk < kKB; ++kk)
            qf[ib][kk] = global_frag<E>(q, a.q.token, s.length - r0, a.dim, kk, lane);
        limit[ib] = a.causal ? min(k_len, r0 + l16 + offset + 1) : k_len;
    }
    // Keys seen by the workgroup's last query, and by the wave's first.
    const int last = a.causal ? min(k_len, min(s.first + kRows, s.length) + offset) : k_len;
    const int full = a.causal ? min(k_len, row0 + offset + 1) : k_len;
    const int tiles = last > 0 ? (last + kKeys - 1) / kKeys : 0;

    AttnTileCopy<E, DIM, kKeys, 256> kc, vc;
    kc.init(a.k.token, a.dim, threadIdx.x);
    vc.init(a.v.token, a.dim, threadIdx.x);

    float m[IB], l[IB];
    f32x4 o[IB][kDB];
#pragma unroll
    for (int ib = 0; ib < IB; ++ib) {
        m[ib] = -INFINITY;
        l[ib] = 0.f;
#pragma unroll
        for (int db = 0; db < kDB; ++db) o[ib][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int t = 0; t < tiles; ++t) {
        const int j0 = t * kKeys;
        lds_barrier();  // the tile before has been read
        kc.issue(a.k.at((long long)k_start + j0, kv), k_len - j0, kt);
        vc.issue(a.v.at((long long)k_start + j0, kv), k_len - j0, vt);
        wait_vmcnt<0>();
        lds_barrier();
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
        const bool edge = j0 + kKeys > full;
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) {
            float top = m[ib];
#pragma unroll
            for (int jb = 0; jb < 4; ++jb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = j0 + 16 * jb + 4 * g + e;
                    float x = sc[jb][ib][e] * a.scale2;
                    if constexpr (BIAS) {
                        const int far = j - (row0 + 16 * ib + l16 + offset);
                        x += bias[min(max(far, -a.reach), a.reach) + a.reach];
                    }
                    if (edge) x = j < limit[ib] ? x : -INFINITY;
                    sc[jb][ib][e] = x;
                    top = fmaxf(top, x);
                }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // No key seen yet: any finite value keeps 2^(-inf - it) at 0.
            const float at = top == -INFINITY ? 0.f : top;
            const float fade = exp2_raw(m[ib] - at);
            m[ib] = top;
            float sum = 0.f;
#pragma unroll
            for (int jb = 0; jb < 4; ++jb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[jb][ib][e] = exp2_raw(sc[jb][ib][e] - at);
                    sum += sc[jb][ib][e];
                }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            l[ib] = l[ib] * fade + sum;
#pragma unroll
            for (int db = 0; db < kDB; ++db) o[ib][db] *= fade;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            typename E::Frag pf[IB];
#pragma unroll
            for (int ib = 0; ib < IB; ++ib) pf[ib] = to_frag<E>(sc[2 * c][ib], sc[2 * c + 1][ib]);
#pragma unroll
            for (int db = 0; db < kDB; ++db) {
                const typename E::Frag vf = col_frag<E, DIM>(vt, 32 * c, db, lane);
#pragma unroll
                for (int ib = 0; ib < IB; ++ib) o[ib][db] = E::mfma(vf, pf[ib], o[ib][db]);
            }
        }
    }
#pragma unroll
    for (int ib = 0; ib < IB; ++ib) {
        const int r = row0 + 16 * ib + l16;
        const bool live = r < s.length;
        const float inv = l[ib] > 0.f ? 1.f / l[ib] : l[ib] == 0.f ? 0.f : l[ib];  // NaN stays
        store_rows<E, kDB>(o[ib], inv, a.out.at((long long)s.start + r, head), live, a.dim, lane);
        if (a.lse && live && g == 0)
            a.lse[(size_t)head * a.q_tokens + s.start + r] =
                l[ib] == 0.f ? -INFINITY : (m[ib] + __builtin_amdgcn_logf(l[ib])) * kLn2;
    }
}

template <class E, int DIM>
constexpr int query_blocks() { return E::kSize == 4 && DIM == 128 ? 1 : 2; }

}  // namespace

extern "C" size_t bfhip_attention_forward_workspace(const bfhip_attention_desc *d) {
    (void)d;
    return 0;
}

extern "C" int bfhip_attention_forward(const bfhip_attention_desc *d, const bfhip_rows *q, const bfhip_rows *k,
                                       const bfhip_rows *v, const bfhip_rows *out, float *lse, void *workspace,
                                       size_t workspace_bytes, void *stream, char *error, size_t cap) {
    (void)workspace, (void)workspace_bytes;
    if (bad_attention(d)) return fail(error, cap, "invalid attention contract");
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    if (bad_rows(q, d->q_tokens, d->head_dim, size) || bad_rows(k, d->k_tokens, d->head_dim, size) ||
        bad_rows(v, d->k_tokens, d->head_dim, size) || bad_rows(out, d->q_tokens, d->head_dim, size))
        return fail(error, cap, "invalid attention rows: pointers and strides in steps of 16 bytes, token strides of at least head_dim");
    if (!d->sequences || !d->q_tokens) return 1;
    const AttnArgs a = attn_args(d, q, k, v, out, lse);
    int ok = 1;
    with_element(d->type, [&](auto e) {
        with_dim(d->head_dim, [&](auto n) {
            using E = decltype(e);
            constexpr int DIM = decltype(n)::value, IB = query_blocks<E, DIM>();
            const long long grid = slot_count(d->q_tokens, d->sequences, 64 * IB) * d->heads;
            if (!launch_fits(grid, 256)) {
                ok = fail(error, cap, "attention has too many rows");
                return;
            }
            const size_t lds = 2 * kKeys * AttnTile<E, DIM>::kRow;
            if (d->bias)
                hipLaunchKernelGGL((attention_forward_kernel<E, DIM, IB, true>), dim3((unsigned)grid), dim3(256),
                                   lds + (2 * d->reach + 1) * sizeof(float), (hipStream_t)stream, a);
            else
                hipLaunchKernelGGL((attention_forward_kernel<E, DIM, IB, false>), dim3((unsigned)grid), dim3(256), lds,
                                   (hipStream_t)stream, a);
        });
    });
    return ok ? launch_ok(error, cap, "attention launch") : 0;
}
