// Rotary positions, forward and backward (include/bfhip_transformer.h).
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

struct RotaryArgs {
    RotaryRows rows[2];
    const int *positions;
    const double *frequencies;
    long long tokens;
    int dim, half, group;  // group: tokens of a workgroup's turn
    int copy;              // elements past the turned part are copied
    float amplitude, sign;
};

// What bounds it is memory: every element is read and written once.  The angles
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
    const int rest = a.copy ? (a.dim - part + WORDS - 1) / WORDS : 0, per_head = turned + rest;
    const int heads = a.rows[0].heads + a.rows[1].heads, per_token = heads * per_head;
    for (long long first = (long long)blockIdx.x * a.group; first < a.tokens; first += (long long)gridDim.x * a.group) {
        const int count = (int)min((long long)a.group, a.tokens - first);
        __syncthreads();  // the angles before have been read
        for (int i = threadIdx.x; i < count * half; i += kThreads) {
            const int t = i / half, p = i - t * half;
            const double turns = (double)a.positions[first + t] * a.frequencies[p] * 0.15915494309189533577;
            float s, c;
            sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
            turn[i] = make_float2(a.amplitude * c, a.amplitude * a.sign * s);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < count * per_token; i += kThreads) {
            const int t = i / per_token, in_token = i - t * per_token;
            int head = in_token / per_head;
            const int chunk = in_token - head * per_head;
            const bool second = head >= a.rows[0].heads;
            if (second) head -= a.rows[0].heads;
            const RotaryRows &r = a.rows[second];
            const Word *x = (const Word *)(r.x + (first + t) * r.x_token + head * r.x_head);
            Word *y = (Word *)(r.y + (first + t) * r.y_token + head * r.y_head);
            if (chunk >= turned) {
                const int c = part + (chunk - turned) * WORDS;
                if (c + WORDS <= a.dim) {
                    W::load(x + c).store(y + c);
                } else {
                    for (int e = c; e < a.dim; ++e) y[e] = x[e];
                }
                continue;
            }
            const int c = chunk * WORDS;
            if constexpr (INTERLEAVED) {
                W v = W::load(x + c);
#pragma unroll
                for (int e = 0; e < WORDS / 2; ++e) {
                    const float2 cs = turn[t * half + c / 2 + e];
                    const float p = v.get(2 * e), q = v.get(2 * e + 1);
                    v.put(2 * e, p * cs.x - q * cs.y);
                    v.put(2 * e + 1, p * cs.y + q * cs.x);
                }
                v.store(y + c);
            } else {
                W v = W::load(x + c), w = W::load(x + half + c);
#pragma unroll
                for (int e = 0; e < WORDS; ++e) {
                    const float2 cs = turn[t * half + c + e];
                    const float p = v.get(e), q = w.get(e);
                    v.put(e, p * cs.x - q * cs.y);
                    w.put(e, p * cs.y + q * cs.x);
                }
                v.store(y + c);
                w.store(y + half + c);
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
    // Tokens of a turn: as many as leave eight workgroups per CU, as LDS holds.
    const long long most = kAngles / a.half, share = d->tokens / 2048;
    a.group = (int)(share < 1 ? 1 : share < most ? share : most);
    if (a.group > 16) a.group = 16;
    if ((long long)a.group * (d->heads + d->heads2) * d->head_dim > 1 << 30) a.group = 1;  // (counted in an int)
    const long long turns = (d->tokens + a.group - 1) / a.group;
    const dim3 grid((unsigned)(turns < 65536 ? turns : 65536));
    hipStream_t s = (hipStream_t)stream;
    // Chunks of 16 bytes where the turned part divides into them, of 8, or the
    // fewest elements there can be.
    with_element(d->type, [&](auto e) {
        using E = decltype(e);
        const auto launch = [&](auto inter, auto words) {
            constexpr int WORDS = decltype(words)::value;
            hipLaunchKernelGGL((rotary_kernel<E, WORDS, decltype(inter)::value>), grid, dim3(kThreads), 0, s, a);
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
