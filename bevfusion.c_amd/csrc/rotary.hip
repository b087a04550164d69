// Rotary positions, forward and backward (include/bfhip_transformer.h).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "bfhip_transformer.h"
#include "element.h"
#include "gemm_core.h"

using namespace bfhip;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 4096;
constexpr int kAngles = kMaxDim / 2;  // cosines and sines in LDS: at least one token's

struct RotaryRows {
    const char *x;
    char *y;
    long long x_token, x_head, y_token, y_head;  // bytes
    int heads;
};

// n / d of n < 2^31 by a product: d's reciprocal, rounded up, in 32 bits.
struct Divisor {
    uint32_t factor;
    int shift;
    static Divisor of(uint32_t d) {
        int l = 0;
        while (l < 31 && (1u << l) < d) ++l;
        return Divisor{(uint32_t)(((1ull << 31 << l) / d) + 1), 31 + l};
    }
    __device__ __forceinline__ int divide(int n) const { return (int)((uint64_t)(uint32_t)n * factor >> shift); }
};

struct RotaryArgs {
    RotaryRows rows[2];
    const int *positions;
    const double *frequencies;
    long long tokens;
    int dim, half, group;  // group: tokens of a workgroup's turn
    int copy;              // elements past the turned part are copied
    int per_head;          // chunks of a head
    Divisor by_token, by_head, by_half;  // chunks of a token and of a head, pairs
    float amplitude, sign;
};

// What bounds it is memory: every element is read and written once (16384 tokens, 40
// heads of 128, bf16: 62 us, 5.4 TB/s; 48 tokens: 3.9 us, latency).  The angles
// of a token are the same for all its heads, so a workgroup first lays down the
// cosines and sines of its tokens in LDS, then its threads walk the tokens'
// heads, WORDS elements of both halves (or of neighbouring pairs) at a time.
// Angles are counted in turns in 64 bits and reduced to half a turn either way
// before they become fp32, so that a far position loses nothing.
template <class E, int WORDS, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
    using W = Words<E, WORDS>;
    using Word = typename E::Word;
    __shared__ float2 turn[kAngles];
    const int half = a.half, part = 2 * half;
    const int turned = INTERLEAVED ? part / WORDS : half / WORDS;  // chunks of a head that turn
    const int per_head = a.per_head, per_token = (a.rows[0].heads + a.rows[1].heads) * per_head;
    constexpr int kAhead = 2;  // chunks that a thread loads before it stores one
    for (long long first = (long long)blockIdx.x * a.group; first < a.tokens; first += (long long)gridDim.x * a.group) {
        const int count = (int)min((long long)a.group, a.tokens - first);
        __syncthreads();  // the angles before have been read
        for (int i = threadIdx.x; i < count * half; i += kThreads) {
            const int t = a.by_half.divide(i), p = i - t * half;
            const double turns = (double)a.positions[first + t] * a.frequencies[p] * 0.15915494309189533577;
            float s, c;
            sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
            turn[i] = make_float2(a.amplitude * c, a.amplitude * a.sign * s);
        }
        __syncthreads();
        const int chunks = count * per_token;
        for (int i0 = threadIdx.x; i0 < chunks; i0 += kAhead * kThreads) {
            W v[kAhead], w[kAhead];
            Word *to[kAhead];
            int by[kAhead];    // its first angle, -1: copied
            int left[kAhead];  // elements of the chunk
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + u * kThreads;
                left[u] = 0;
                if (i >= chunks) continue;
                const int t = a.by_token.divide(i), in_token = i - t * per_token;
                int head = a.by_head.divide(in_token);
                const int chunk = in_token - head * per_head;
                const bool second = head >= a.rows[0].heads;
                if (second) head -= a.rows[0].heads;
                const RotaryRows &r = a.rows[second];
                const int c = chunk < turned ? chunk * WORDS : part + (chunk - turned) * WORDS;
                const Word *x = (const Word *)(r.x + (first + t) * r.x_token + head * r.x_head) + c;
                to[u] = (Word *)(r.y + (first + t) * r.y_token + head * r.y_head) + c;
                left[u] = min(WORDS, a.dim - c);
                by[u] = chunk < turned ? t * half + (INTERLEAVED ? c / 2 : c) : -1;
                if (left[u] == WORDS) {
                    v[u] = W::load(x);
                } else {
#pragma unroll
                    for (int e = 0; e < WORDS; ++e) v[u].w[e] = e < left[u] ? x[e] : (Word)0.f;
                }
                if (!INTERLEAVED && by[u] >= 0) w[u] = W::load(x + half);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (!left[u]) continue;
                if (by[u] < 0) {
                    if (left[u] == WORDS) {
                        v[u].store(to[u]);
                    } else {
#pragma unroll
                        for (int e = 0; e < WORDS; ++e)
                            if (e < left[u]) to[u][e] = v[u].w[e];
                    }
                } else if constexpr (INTERLEAVED) {
#pragma unroll
                    for (int e = 0; e < WORDS / 2; ++e) {
                        const float2 cs = turn[by[u] + e];
                        const float p = v[u].get(2 * e), q = v[u].get(2 * e + 1);
                        v[u].put(2 * e, p * cs.x - q * cs.y);
                        v[u].put(2 * e + 1, p * cs.y + q * cs.x);
                    }
                    v[u].store(to[u]);
                } else {
#pragma unroll
                    for (int e = 0; e < WORDS; ++e) {
                        const float2 cs = turn[by[u] + e];
                        const float p = v[u].get(e), q = w[u].get(e);
                        v[u].put(e, p * cs.x - q * cs.y);
                        w[u].put(e, p * cs.y + q * cs.x);
                    }
                    v[u].store(to[u]);
                    w[u].store(to[u] + half);
                }
            }
        }
    }
}

bool bad_head_rows(const bfhip_rows *x, const bfhip_rows *y, long long tokens, int heads, int dim) {
    if (!x || !y || !x->data || !y->data) return true;
    if (tokens > 1 && (x->token_stride < 0 || y->token_stride < 0)) return true;
    if (heads > 1 && (x->head_stride < 0 || y->head_stride < 0)) return true;
    const long long t = tokens > 1 ? y->token_stride : 0, h = heads > 1 ? y->head_stride : 0;
    // No head of the result on another, whichever of tokens and heads is the outer one.
    if ((heads > 1 && h < dim) || (tokens > 1 && t < dim)) return true;
    if (tokens > 1 && heads > 1 && t < (heads - 1) * h + dim && h < (tokens - 1) * t + dim) return true;
    return x->data == y->data && ((tokens > 1 && x->token_stride != t) || (heads > 1 && x->head_stride != h));
}

RotaryRows rotary_rows(const bfhip_rows *x, const bfhip_rows *y, long long tokens, int heads, int size) {
    const auto step = [&](long long n, long long stride) { return n > 1 ? stride * size : 0; };
    return RotaryRows{(const char *)x->data, (char *)y->data, step(tokens, x->token_stride), step(heads, x->head_stride),
                      step(tokens, y->token_stride), step(heads, y->head_stride), heads};
}

}  // namespace

extern "C" int bfhip_rotary_frequencies(int part, double base, double factor, double length, double low, double high,
                                        double *frequencies, char *error, size_t cap) {
    if (part <= 0 || part % 2 || part > kMaxDim || !(base > 0) || !(factor > 0) || !(length >= 0) || !(low < high) ||
        std::isinf(base) || std::isinf(factor) || std::isinf(length) || std::isinf(low) || std::isinf(high) || !frequencies)
        return fail(error, cap, "invalid rotary frequencies contract");
    for (int i = 0; i < part / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / part);
        const double turns = length * f / (2 * 3.14159265358979323846);
        double keep = length > 0 ? (turns - low) / (high - low) : 0.0;
        keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
        frequencies[i] = f * (keep + (1 - keep) / factor);
    }
    return 1;
}

extern "C" int bfhip_rotary(const bfhip_rotary_desc *d, const bfhip_rows *x, const bfhip_rows *y, const bfhip_rows *x2,
                            const bfhip_rows *y2, void *stream, char *error, size_t cap) {
    if (!d || d->type < BFHIP_F32 || d->type > BFHIP_BF16 || d->head_dim <= 0 || d->head_dim > kMaxDim || d->part <= 0 ||
        d->part % 2 || d->part > d->head_dim || (d->interleaved != 0 && d->interleaved != 1) ||
        (d->inverse != 0 && d->inverse != 1) || d->heads <= 0 || d->heads > 65535 || d->heads2 < 0 || d->heads2 > 65535 ||
        !std::isfinite(d->amplitude) || d->tokens < 0 || d->tokens > 0x7ffff000)
        return fail(error, cap, "invalid rotary contract");
    if (!d->tokens) return 1;
    if (!d->positions || !d->frequencies || bad_head_rows(x, y, d->tokens, d->heads, d->head_dim) ||
        (d->heads2 && bad_head_rows(x2, y2, d->tokens, d->heads2, d->head_dim)))
        return fail(error, cap, "invalid rotary rows: no head of a result on another, in place with one stride");
    const int size = d->type == BFHIP_F32 ? 4 : 2;
    RotaryArgs a{};
    a.rows[0] = rotary_rows(x, y, d->tokens, d->heads, size);
    if (d->heads2) a.rows[1] = rotary_rows(x2, y2, d->tokens, d->heads2, size);
    a.positions = d->positions;
    a.frequencies = d->frequencies;
    a.tokens = d->tokens;
    a.dim = d->head_dim;
    a.half = d->part / 2;
    a.copy = d->part < d->head_dim && (x->data != y->data || (d->heads2 && x2->data != y2->data));
    a.amplitude = d->amplitude;
    a.sign = d->inverse ? -1.f : 1.f;
    hipStream_t s = (hipStream_t)stream;
    // Chunks of 16 bytes where the turned part divides into them, of 8, or the
    // fewest elements there can be.
    with_element(d->type, [&](auto e) {
        using E = decltype(e);
        const auto launch = [&](auto inter, auto words) {
            constexpr int WORDS = decltype(words)::value;
            constexpr bool I = decltype(inter)::value;
            const int rest = a.copy ? (a.dim - d->part + WORDS - 1) / WORDS : 0;
            a.per_head = (I ? d->part : a.half) / WORDS + rest;
            a.by_head = Divisor::of(a.per_head);
            a.by_token = Divisor::of(a.per_head * (d->heads + d->heads2));
            a.by_half = Divisor::of(a.half);
            // Tokens of a turn: two chunks per thread, unless that leaves CUs idle, and
            // as LDS holds.  (16384 tokens, 40 heads of 128, bf16: one a turn 62 us, two
            // 65, eight 71: then all workgroups work on their angles at one time.)
            const long long per_token = (long long)a.per_head * (d->heads + d->heads2);
            a.group = (int)std::max(1ll, std::min({2 * kThreads / per_token, d->tokens / 1024, (long long)kAngles / a.half}));
            const long long turns = (d->tokens + a.group - 1) / a.group;
            const dim3 grid((unsigned)std::min(turns, 65536ll));
            hipLaunchKernelGGL((rotary_kernel<E, WORDS, I>), grid, dim3(kThreads), 0, s, a);
        };
        const auto choose = [&](auto inter, int n) {
            constexpr int kMost = 16 / E::kSize, kLeast = decltype(inter)::value ? 2 : 1;
            if (n % kMost == 0) launch(inter, std::integral_constant<int, kMost>{});
            else if (n % (kMost / 2) == 0) launch(inter, std::integral_constant<int, kMost / 2>{});
            else launch(inter, std::integral_constant<int, kLeast>{});
        };
        if (d->interleaved) choose(std::true_type{}, d->part);
        else choose(std::false_type{}, a.half);
    });
    return launch_ok(error, cap, "rotary launch");
}
