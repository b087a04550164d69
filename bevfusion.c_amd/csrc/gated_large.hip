// The gated linear's products by large tiles (gated.h).  Compiled with accumulators
// in the accumulation registers: a wave's are 256 of them.
#include "gated.h"

namespace bfhip {

namespace {

// A wave's copies of one operand's tiles, step by step, with as few instructions as
// it takes: a wave that is alone on its SIMD issues one in four cycles, and a product
// takes sixteen.  What lies outside the matrix reads as zero by the range check of
// the buffer resources: rows beyond the last one by the resource's size, elements
// beyond a row's end by the lane's offset.
template <class E, class Tile, int PAIR, bool COL, int BK>
struct GatedStream {
    Resource a, b;                  // of the step's tile (b: the up's rows)
    uint32_t off[Tile::kPlaces];    // the lane's offsets
    uint32_t span[Tile::kIssue];    // bytes from copy 0 to copy J
    const Tile &tile;
    int k;

    __device__ __forceinline__ GatedStream(const Tile &t, int k_) : tile(t), k(k_) {
#pragma unroll
        for (int j = 0; j < Tile::kIssue; ++j)
            span[j] = (uint32_t)__builtin_amdgcn_readfirstlane((int)(Tile::template span_row<PAIR>(j) * (int)t.stride));
#pragma unroll
        for (int p = 0; p < Tile::kPlaces; ++p) off[p] = COL && t.first[p] >= t.left ? kDmaOutOfRange : t.off[p];
    }
    // Turns to the tile from k0 on of the matrix at base_a (and base_b).
    __device__ __forceinline__ void seek(const char *base_a, const char *base_b, int k0, bool there) {
        const int rest = there ? k - k0 : 0;
        const long long at = there ? (COL ? k0 * tile.stride : (long long)k0 * E::kSize) : 0;
        int size = 0;
        if (rest > 0) {
            // To the end of the last row that there is, in whole chunks.
            const int length = ((COL ? tile.left : rest) + Tile::kWords - 1) / Tile::kWords * 16;
            size = (min(COL ? rest : tile.left, COL ? BK : Tile::kOuter) - 1) * (int)tile.stride + length;
        }
        a = resource(base_a + at);
        a[2] = (uint32_t)__builtin_amdgcn_readfirstlane(size);
        if (PAIR) {
            b = resource(base_b + at);
            b[2] = a[2];
        }
        if (!COL) off[0] = tile.first[0] < rest ? tile.off[0] : kDmaOutOfRange;
    }
    template <int J>
    __device__ __forceinline__ static constexpr bool up() { return PAIR > 0 && J * Tile::kSpan % (PAIR ? PAIR : 1) >= PAIR / 2; }
};

// One workgroup of four waves per CU, one per SIMD, each with 128 x 128 results, so
// that an LDS read of 16 rows serves eight products (with eight waves of 128 x 64 the
// LDS was the bound).  A wave covers its own waits: each step of 64 is multiplied
// in two halves, and while a half's fragments are multiplied the next half's are read
// and one tile is copied, spread over the products.  The tiles of m and n take turns
// in a ring of five buffers: in a step's first half m's of two steps on, in its
// second half n's, into the buffer that m's of this step has left.  One barrier a
// step, between the halves: behind it every wave has read the step's fragments and
// every wave's copies of the next step's tiles have come in.  Bound by the matrix cores'
// clock under load and by the issue (forward, 8192 rows of 4096 -> 11008, bf16: 1035 to 1080
// us, 1.4 PFLOP/s, cores busy 68 % of the cycles at 1.95 GHz).
constexpr int kRing = 5;

template <class E, Form F, class S>
struct LargeLoop {
    using Frag = typename E::Frag;
    static constexpr int kN = S::kNB, kM = S::kMB, kTile = S::MTile::kBytes, kCopy = S::kThreads * 16;
    static_assert(S::WM * S::WN == 4 && S::BK == 64 && kN == 8 && kM == 8 && S::MTile::kIssue == 8 && S::NTile::kIssue == 8 &&
                      kTile == S::NTile::kBytes,
                  "a copy and two reads per block of products");
    GatedWork<E, F, S> w;
    f32x4 acc[kM][kN];
    Frag n0[kN], m0[kM], n1[kN], m1[kM];  // of a step's two halves
    char *smem;
    int at;  // the buffer of the step's m

    // The buffer i places on in the ring.
    __device__ __forceinline__ char *ring(int i) const { return smem + (at + i < kRing ? at + i : at + i - kRing) * kTile; }
    // Products in assembly, which ties a product's accumulators to its results: with
    // all 256 accumulation registers taken the compiler moves them about otherwise
    // (three moves per product).
    __device__ __forceinline__ static void product(f32x4 &c, const Frag &n, const Frag &m) {
        if constexpr (std::is_same_v<E, ElemF16>) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(n), "v"(m));
        else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(n), "v"(m));
    }
    // A product and a copy to LDS address `to` + SHIFT (M0 is written one instruction
    // before it is read at least).
    template <int SHIFT>
    __device__ __forceinline__ static void product_and_copy(f32x4 &c, const Frag &n, const Frag &m, Resource r, uint32_t to, uint32_t voff, uint32_t soff) {
        if constexpr (std::is_same_v<E, ElemF16>)
            asm volatile("s_add_u32 m0, %3, %7\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0\n\tbuffer_load_dwordx4 %4, %5, %6 offen lds"
                         : "+a"(c) : "v"(n), "v"(m), "s"(to), "v"(voff), "s"(r), "s"(soff), "n"(SHIFT) : "memory", "m0", "scc");
        else
            asm volatile("s_add_u32 m0, %3, %7\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0\n\tbuffer_load_dwordx4 %4, %5, %6 offen lds"
                         : "+a"(c) : "v"(n), "v"(m), "s"(to), "v"(voff), "s"(r), "s"(soff), "n"(SHIFT) : "memory", "m0", "scc");
    }
    // Block row I of n against all of m, and copy I of a stream's tile.
    template <int I, class Stream>
    __device__ __forceinline__ void block(const Frag (&n)[kN], const Frag (&m)[kM], const Stream &s, uint32_t to) {
        product(acc[0][I], n[I], m[0]);
        product_and_copy<I * kCopy>(acc[1][I], n[I], m[1], Stream::template up<I>() ? s.b : s.a, to,
                                    s.off[I % (int)(sizeof s.off / sizeof s.off[0])], s.span[I]);
#pragma unroll
        for (int j = 2; j < kM; ++j) product(acc[j][I], n[I], m[j]);
        __builtin_amdgcn_sched_barrier(0);
    }
    // Fragment K of half KK of a step, m's first, with which the half's products begin.
    template <int K, int KK>
    __device__ __forceinline__ void read(Frag (&n)[kN], Frag (&m)[kM], const char *mt, const char *nt) const {
        if constexpr (K < kM) m[K] = S::MTile::frag(mt, w.m_at, K, KK);
        else n[K - kM] = S::NTile::frag(nt, w.n_at, K - kM, KK);
    }
    // Lets the last products end before their results are read, and the accumulators
    // be written before the first: the compiler does not know the products' latencies.
    __device__ __forceinline__ void settle() {
        const auto fix = [&] {
#pragma unroll
            for (int j = 0; j < kM; ++j)
#pragma unroll
                for (int i = 0; i < kN; ++i) asm volatile("" : "+a"(acc[j][i]));
        };
        fix();
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
        fix();
    }
    template <int I, class Stream>
    __device__ __forceinline__ void first(const Stream &s, uint32_t to, const char *mt, const char *nt) {
        read<2 * I, 1>(n1, m1, mt, nt);
        read<2 * I + 1, 1>(n1, m1, mt, nt);
        block<I>(n0, m0, s, to);
    }
    template <int I, class Stream>
    __device__ __forceinline__ void second(const Stream &s, uint32_t to, const char *mt, const char *nt) {
        read<2 * I, 0>(n0, m0, mt, nt);
        read<2 * I + 1, 0>(n0, m0, mt, nt);
        block<I>(n1, m1, s, to);
    }
    __device__ __forceinline__ void run(const GatedArgs &a, int wave, int lane) {
        w.init(a, blockIdx.x, wave, lane);
        GatedStream<E, typename S::MTile, 0, F == kWeights, S::BK> ms(w.mt, w.k);
        GatedStream<E, typename S::NTile, S::kPair, F != kForward, S::BK> ns(w.nt, w.k);
        // Past the last step the tiles are empty: zeros, without a read.
        const auto seek = [&](auto &s, const auto &tile, int t) {
            const bool up = F == kInputs && t >= w.each;
            s.seek(up ? tile.base_b : tile.base_a, tile.base_b, (up ? t - w.each : t) * S::BK, t < w.end);
        };
        const uint32_t mine = wave * kWave * 16;
        at = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int t = w.begin + s;
            seek(ms, w.mt, t);
            copies(ms, lds_address(ring(2 * s)) + mine);
            seek(ns, w.nt, t);
            copies(ns, lds_address(ring(2 * s + 1)) + mine);
        }
#pragma unroll
        for (int j = 0; j < kM; ++j)
#pragma unroll
            for (int i = 0; i < kN; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        wait_vmcnt<16>();
        lds_barrier();
#pragma unroll
        for (int i = 0; i < kM; ++i) m0[i] = S::MTile::frag(ring(0), w.m_at, i, 0);
#pragma unroll
        for (int i = 0; i < kN; ++i) n0[i] = S::NTile::frag(ring(1), w.n_at, i, 0);
        settle();
        for (int t = w.begin; t < w.end; ++t) {
            {
                seek(ms, w.mt, t + 2);
                const uint32_t to = lds_address(ring(4)) + mine;
                const char *const mt = ring(0), *const nt = ring(1);
                first<0>(ms, to, mt, nt); first<1>(ms, to, mt, nt); first<2>(ms, to, mt, nt); first<3>(ms, to, mt, nt);
                first<4>(ms, to, mt, nt); first<5>(ms, to, mt, nt); first<6>(ms, to, mt, nt); first<7>(ms, to, mt, nt);
            }
            wait_vmcnt<8>();  // all but the copies just issued
            lds_barrier();
            {
                seek(ns, w.nt, t + 2);
                const uint32_t to = lds_address(ring(0)) + mine;
                const char *const mt = ring(2), *const nt = ring(3);
                second<0>(ns, to, mt, nt); second<1>(ns, to, mt, nt); second<2>(ns, to, mt, nt); second<3>(ns, to, mt, nt);
                second<4>(ns, to, mt, nt); second<5>(ns, to, mt, nt); second<6>(ns, to, mt, nt); second<7>(ns, to, mt, nt);
            }
            at = at + 2 < kRing ? at + 2 : at + 2 - kRing;
        }
        settle();
        wait_vmcnt<0>();
        lds_barrier();  // no copy and no read of a tile is left
        w.store(a, acc, smem, wave, lane);
    }
    template <class Stream, int I = 0>
    __device__ __forceinline__ void copies(const Stream &s, uint32_t to) {
        asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :: "s"(to), "v"(s.off[I % (int)(sizeof s.off / sizeof s.off[0])]), "s"(Stream::template up<I>() ? s.b : s.a), "s"(s.span[I]),
                        "n"(I * kCopy)
                     : "memory", "m0", "scc");
        if constexpr (I < 7) copies<Stream, I + 1>(s, to);
    }
};

template <class E, Form F, class S>
__global__ __launch_bounds__(S::kThreads) void gated_large_kernel(GatedArgs a) {
    __shared__ __attribute__((aligned(512))) char smem[gated_lds<E, F, S>(kRing * S::MTile::kBytes)];
    LargeLoop<E, F, S> loop;
    loop.smem = smem;
    loop.run(a, __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), threadIdx.x % kWave);
}

}  // namespace

template <class E, Form F>
void launch_gated_large(const GatedArgs &a, long long grid, hipStream_t s) {
    using S = LargeShape<E, F>;
    hipLaunchKernelGGL((gated_large_kernel<E, F, S>), dim3((unsigned)grid), dim3(S::kThreads), 0, s, a);
    const long long split = (long long)a.tiles_m * a.tiles_n - a.whole;
    if (split) hipLaunchKernelGGL((gated_join_kernel<E, F, S>), dim3((unsigned)(split * S::kMB)), dim3(S::kThreads), 0, s, a);
}

template void launch_gated_large<ElemF16, kForward>(const GatedArgs &, long long, hipStream_t);
template void launch_gated_large<ElemF16, kInputs>(const GatedArgs &, long long, hipStream_t);
template void launch_gated_large<ElemF16, kWeights>(const GatedArgs &, long long, hipStream_t);
template void launch_gated_large<ElemBf16, kForward>(const GatedArgs &, long long, hipStream_t);
template void launch_gated_large<ElemBf16, kInputs>(const GatedArgs &, long long, hipStream_t);
template void launch_gated_large<ElemBf16, kWeights>(const GatedArgs &, long long, hipStream_t);

}  // namespace bfhip
