// Element types of the stateless transformer operators: loads and stores of
// fp32, fp16 and bf16 as fp32, and matrix-core products of each.
#pragma once

#include "hip_common.h"

namespace bfhip {

typedef float f32x8 __attribute__((ext_vector_type(8)));

struct ElemF32 {
    using Word = float;
    using Frag = f32x8;  // 8 consecutive k of one row
    static constexpr int kSize = 4;
    __device__ static float get(float v) { return v; }
    __device__ static float put(float v) { return v; }
    // acc[16x16] += A[16x32] B[32x16], the operands laid out as for the 16-bit
    // products (lane l: row or column l & 15, slots 8 (l >> 4) ..+7): step t
    // multiplies slot t of each lane group, which the fp32 instruction's lane
    // group holds as its one k.
    __device__ static f32x4 mfma(f32x8 a, f32x8 b, f32x4 acc) {
#pragma unroll
        for (int t = 0; t < 8; ++t) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], acc, 0, 0, 0);
        return acc;
    }
};

struct ElemF16 {
    using Word = _Float16;
    using Frag = bf16x8;
    static constexpr int kSize = 2;
    __device__ static float get(_Float16 v) { return (float)v; }
    // Rounded once from the fp32 value (see to_half).
    __device__ static _Float16 put(float v) { return __builtin_bit_cast(_Float16, to_half(v)); }
    __device__ static f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 acc) { return mfma16_f16(a, b, acc); }
};

struct ElemBf16 {
    using Word = bf16;
    using Frag = bf16x8;
    static constexpr int kSize = 2;
    __device__ static float get(bf16 v) { return (float)v; }
    __device__ static bf16 put(float v) { return (bf16)v; }
    __device__ static f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 acc) { return mfma16(a, b, acc); }
};

// N words at p as floats and back, in one access where N words are a power of
// two of bytes; p needs no alignment beyond the word's (gfx950 serves
// unaligned vector accesses).  A vector, so that 16-bit words stay packed in
// registers.
template <class E, int N>
struct Words {
    using Word = typename E::Word;
    typedef Word Vec __attribute__((ext_vector_type(N)));
    Vec w;
    __device__ __forceinline__ static Words load(const Word *p) {
        Words v;
        __builtin_memcpy(&v.w, p, sizeof v.w);
        return v;
    }
    __device__ __forceinline__ void store(Word *p) const { __builtin_memcpy(p, &w, sizeof w); }
    __device__ __forceinline__ float get(int i) const { return E::get(w[i]); }
    __device__ __forceinline__ void put(int i, float v) { w[i] = E::put(v); }
};

// Calls f with the element type that `type` (BFHIP_F32 ..) names.
template <class F>
inline void with_element(int type, F f) {
    switch (type) {
        case 0: f(ElemF32{}); break;
        case 1: f(ElemF16{}); break;
        default: f(ElemBf16{}); break;
    }
}

}  // namespace bfhip
