// The running softmax of the attention kernels that walk a query's keys once.
#pragma once

#include "attention.h"

namespace bfhip {

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

}  // namespace bfhip
