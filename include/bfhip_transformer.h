/*
 * Stateless transformer operators on AMD gfx950, served by libbfhip.so: layer
 * norm, learned position bias by buckets, rotary positions, attention over
 * packed sequences and the gated linear of a feed-forward block, each with its
 * backward pass; and for serving a paged cache of keys and values with the
 * attention of new tokens over it.  They stand beside the stateless linear and
 * convolution of bf_cuda_ops.h and have no counterpart in the reference, whose
 * transformer blocks exist inside its fixed contexts only.
 *
 * Conventions, as in bf_cuda_ops.h:
 *   - tensor pointers are device pointers; `stream` is a hipStream_t of the
 *     current device (NULL = the default stream);
 *   - returns 1 on success, 0 on failure with a message written to
 *     error[0..error_cap) (error may be NULL or error_cap 0);
 *   - the contract is validated before anything is launched; launch errors
 *     are reported from hipGetLastError.
 * Nothing is allocated, cleared by memset, synchronised or kept between calls,
 * so every call may be captured into a HIP graph, and calls on different
 * streams do not disturb each other as long as each has a workspace of its
 * own.  A workspace is scratch: it need not be cleared, holds nothing between
 * calls, and must be 16-byte aligned and at least as large as the matching
 * *_workspace function says (0: NULL will do).  Results do not depend on
 * timing: no floating-point atomics whose order is left open, so equal calls
 * give equal bits.
 *
 * Types: activations and their gradients are BFHIP_F32, BFHIP_F16 or
 * BFHIP_BF16, all of one call the same.  Norm weights, statistics, biases and
 * their gradients are fp32.  Sums, softmax and statistics run in fp32; 16-bit
 * results are rounded once.
 */
#ifndef BFHIP_TRANSFORMER_H
#define BFHIP_TRANSFORMER_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { BFHIP_F32 = 0, BFHIP_F16 = 1, BFHIP_BF16 = 2 };

/* ---------------------------------------------------------------- layer norm
 * Rows of `features` elements, row r at element r * <name>_stride; elements of
 * a row are contiguous and need no alignment beyond their own type's.
 * features <= 65536.
 *
 *   y = (x - mean) * rstd * gamma + beta,  rstd = 1 / sqrt(var + eps), var the
 *   mean squared deviation.  gamma, beta: [features] or NULL (1 and 0).  mean,
 *   rstd: [rows], both or neither NULL.  y may be x (in place, one stride).
 *
 * Backward, with g = dy * gamma and h = (x - mean) * rstd:
 *   dx     = rstd * (g - mean_c(g) - h * mean_c(g * h))
 *   dgamma = sum over rows of dy * h,   dbeta = sum over rows of dy
 *   dgamma, dbeta: [features], both or neither NULL.  dx may be dy or x (one
 *   stride).
 *   rows == 0 writes zeros to dgamma and dbeta. */
int bfhip_layer_norm_forward(int type, const void *x, long long x_stride, const float *gamma,
                             const float *beta, void *y, long long y_stride, float *mean,
                             float *rstd, long long rows, int features, float eps,
                             void *stream, char *error, size_t error_cap);

size_t bfhip_layer_norm_backward_workspace(long long rows, int features);

int bfhip_layer_norm_backward(int type, const void *dy, long long dy_stride, const void *x,
                              long long x_stride, const float *gamma, const float *mean,
                              const float *rstd, void *dx, long long dx_stride, float *dgamma,
                              float *dbeta, long long rows, int features,
                              void *workspace, size_t workspace_bytes,
                              void *stream, char *error, size_t error_cap);

/* ------------------------------------------------------------- position bias
 * A learned table [buckets, heads] spread over positions by a map from
 * position to bucket, and the table's gradient:
 *   bias[h, p]   = table[map[p], h]                          p in [0, positions)
 *   dtable[b, h] = sum over p with map[p] == b of dbias[h, p]
 * A position is whatever the caller's map runs over: the 49 x 49 pairs of a
 * window (Swin's relative_position_index; `bias` is then what
 * bfhip_debug_window_attention takes), all pairs of a sequence, or the signed
 * distances that bfhip_attention_forward's bias runs over.  A map entry
 * outside [0, buckets) belongs to no bucket: its bias is 0 and its gradient
 * goes nowhere.  bias and dbias are [heads, positions], contiguous. */
int bfhip_position_bias_forward(const float *table, const int *map, float *bias, int buckets,
                                int heads, long long positions,
                                void *stream, char *error, size_t error_cap);

size_t bfhip_position_bias_backward_workspace(int buckets, int heads, long long positions);

int bfhip_position_bias_backward(const float *dbias, const int *map, float *dtable, int buckets,
                                 int heads, long long positions,
                                 void *workspace, size_t workspace_bytes,
                                 void *stream, char *error, size_t error_cap);

/* ----------------------------------------------------------------- attention
 * Packed sequences: sequence b has the query rows q_starts[b] .. q_starts[b+1]
 * and the key rows k_starts[b] .. k_starts[b+1] (device arrays of sequences + 1
 * ascending int32; lengths may be zero and may differ between queries and
 * keys).  Starts are clamped to [0, tokens]; rows outside every sequence are
 * not written, and what they hold is ignored.  (Where starts descend all the
 * same, what the rows get is open, but nothing outside the rows is touched.)
 * Query head h reads key head h / (heads / kv_heads).
 *
 * With Lq queries and Lk keys, query i stands at position i + Lk - Lq, so the
 * last query stands at the last key.  Key j is seen if not causal, or if
 * j <= i + Lk - Lq.
 *   s = scale * q.k + bias[h, clamp(j - position, -reach, reach) + reach]
 *   out = softmax over the seen keys of s, times v;   lse = log sum exp s
 * A query that sees no key, or only keys of score -inf, gets out = 0,
 * lse = -inf and no gradient.  Keys that a query does not see do not reach its
 * scores, whatever they hold; a value row reaches every query of its
 * sequence whose tile of the product it shares, so a NaN or infinity in a
 * value can also reach queries of its sequence that do not see it (0 * NaN).  In
 * the backward pass that holds for the keys (dq) and for q and dout (dk, dv)
 * too.
 *
 * Scores and the softmax are fp32; for 16-bit types the probabilities, and in
 * the backward pass the gradients of the scores, are rounded to the type where
 * they enter the matrix cores (where a query sees few keys, their rounding's rest
 * enters too).  fp16: the forward pass loses probabilities 2^-25 below a row's
 * largest; the backward pass multiplies by powers of two on the way, so that
 * gradients of scores may be of any size: it loses what lies 2^-36 below the
 * largest |dout . v| of 32 neighbouring queries (dq) or of all queries that meet a
 * key (dk).  Results beyond the type's range become infinite.  fp32 is multiplied
 * in fp32.
 *
 * A score and its bias are added in fp32: a large bias (1e9, the lowest fp32
 * value) swallows the score, so that a query all of whose keys have it takes
 * their mean.  Finite biases beyond 2.3e38 of either sign count as that.  The
 * backward pass finds the sum of a query's probabilities again where a bias has
 * taken its lse far from zero; without a bias it takes them from lse alone, off
 * by a factor of about 1 +- |lse| 2^-22.
 *
 * Workspaces: the forward's holds the sums of keys that are split (few queries
 * on many keys, at most 1 GiB; mostly none), the backward's two fp32 per query
 * and head (three with a bias), sums of queries that are split (at most 128 MiB;
 * of keys in fp32, 32 MiB), and for every head, every 64 (fp32) or 128 queries
 * and every sequence 2 * reach + 1 fp32 with a bias and four in fp16.
 *
 * head_dim: a multiple of 8, at most 128.  Rows: pointer, token and head
 * stride in elements; the elements of one head are contiguous, pointers and
 * strides are multiples of 16 bytes, token strides at least head_dim and below
 * 4 Mi elements (of no account where there is at most one token); no row of a
 * result on another.  At most 0x7ffff000 query and key rows.
 * bias: [heads, 2 * reach + 1] or NULL (reach is then ignored); reach in
 * [0, 2047].  out must not overlap the other tensors. */
typedef struct {
    void *data;
    long long token_stride;
    long long head_stride;
} bfhip_rows;

typedef struct {
    int type;
    int sequences;
    int heads;
    int kv_heads;
    int head_dim;
    int causal;
    int reach;
    float scale;
    long long q_tokens; /* rows of q, out and their gradients */
    long long k_tokens; /* rows of k, v and their gradients */
    const int *q_starts;
    const int *k_starts;
    const float *bias;
} bfhip_attention_desc;

/* Bytes of workspace; 0 for an invalid descriptor too. */
size_t bfhip_attention_forward_workspace(const bfhip_attention_desc *desc);
size_t bfhip_attention_backward_workspace(const bfhip_attention_desc *desc);

/* lse: [heads, q_tokens] fp32 or NULL. */
int bfhip_attention_forward(const bfhip_attention_desc *desc, const bfhip_rows *q,
                            const bfhip_rows *k, const bfhip_rows *v, const bfhip_rows *out,
                            float *lse, void *workspace, size_t workspace_bytes,
                            void *stream, char *error, size_t error_cap);

/* Gradients of q, k, v and of the bias (dbias: [heads, 2 * reach + 1], or NULL)
 * from dout; out and lse are the forward's.  dq, dk and dv must not overlap any
 * other tensor of the call. */
int bfhip_attention_backward(const bfhip_attention_desc *desc, const bfhip_rows *q,
                             const bfhip_rows *k, const bfhip_rows *v, const bfhip_rows *out,
                             const float *lse, const bfhip_rows *dout, const bfhip_rows *dq,
                             const bfhip_rows *dk, const bfhip_rows *dv, float *dbias,
                             void *workspace, size_t workspace_bytes,
                             void *stream, char *error, size_t error_cap);

/* ---------------------------------------------------------- rotary positions
 * Pairs of a head's elements turned by angles that grow with the token's
 * position, t_i = position * frequencies[i], i < part / 2, part <= head_dim even:
 *   (a, b) -> amplitude * (a cos t - b sin t, a sin t + b cos t)
 * Pair i is the elements (i, i + part / 2), or (2 i, 2 i + 1) if interleaved;
 * elements from part on are copied.  The gradient is the transposed map: with
 * `inverse` the angles change their sign (and the amplitude stays).
 *
 * x and y: rows of `heads` heads of head_dim elements, strides in elements, of
 * any alignment; the elements of one head are contiguous, and no head of y lies
 * on another.  y may be x (in place, the same strides), else they do not
 * overlap.  A second pair of rows (x2, y2, heads2; heads2 == 0: none) of the same
 * tokens, type and head_dim shares the angles: queries and keys take one call.
 * positions: int32 [tokens], of either sign.  frequencies: fp64 [part / 2], in
 * radians per position.  Angles are reduced in 64 bits, off by at most 2^-51 of
 * the angle; cosine, sine and products are fp32, results are rounded once.
 * tokens at most 0x7ffff000, heads and heads2 at most 65535, head_dim at most
 * 4096. */
typedef struct {
    int type;
    int head_dim;
    int part;
    int interleaved;
    int inverse;
    int heads;
    int heads2;
    float amplitude;
    long long tokens;
    const int *positions;
    const double *frequencies;
} bfhip_rotary_desc;

int bfhip_rotary(const bfhip_rotary_desc *desc, const bfhip_rows *x, const bfhip_rows *y,
                 const bfhip_rows *x2, const bfhip_rows *y2,
                 void *stream, char *error, size_t error_cap);

/* frequencies[i] = base^(-2 i / part) on the host, scaled for contexts `factor`
 * times as long as the trained one.  length == 0: all of them divided by factor
 * (positions are interpolated).  Otherwise by parts: a pair that turns r =
 * length * frequency / 2 pi times over the trained length is kept where
 * r >= high, divided by factor where r <= low, and mixed linearly in between.
 * base > 0, factor > 0, length >= 0, low < high. */
int bfhip_rotary_frequencies(int part, double base, double factor, double length, double low,
                             double high, double *frequencies, char *error, size_t error_cap);

/* --------------------------------------------------------------- paged cache
 * Keys and values of many sequences in pages of page_size tokens.  Position j
 * of sequence b is row j % page_size of page table[b * table_stride +
 * j / page_size]; a table has table_pages entries per sequence.  Pages may
 * stand in any order and be shared by sequences.  lengths[b] counts the keys of
 * sequence b with its new tokens among them: its new tokens, the rows
 * starts[b] .. starts[b + 1] of q, k and v (starts as in
 * bfhip_attention_forward; there may be none), stand at its last positions.
 * Lengths are clamped to [0, table_pages * page_size], which is below 2^31.
 * starts, lengths and table are int32 on the device.  A table entry outside
 * [0, pages) is never followed: its positions are written nowhere and seen by no
 * query.  Entries past a sequence's length are not read.
 *
 * Pages: [pages, page_size, kv_heads, head_dim] by strides in elements, of any
 * size; the elements of one head are contiguous, pointers and strides multiples
 * of 16 bytes and not negative.  head_dim: a multiple of 8, at most 128. */
typedef struct {
    void *data;
    long long page_stride;
    long long token_stride;
    long long head_stride;
} bfhip_pages;

typedef struct {
    int type;
    int sequences;
    int heads;    /* of the queries; of no account to bfhip_cache_append */
    int kv_heads;
    int head_dim;
    int page_size;
    int table_pages;
    int reach;    /* as in bfhip_attention_desc */
    float scale;
    long long tokens; /* rows of q, k, v and out */
    long long pages;
    long long table_stride;
    const int *starts;
    const int *lengths;
    const int *table;
    const float *bias;
} bfhip_paged_desc;

/* Copies the new tokens' keys and values (rows of any alignment) into their
 * pages.  A token that stands before position 0 (more new tokens than
 * lengths[b]) or outside every sequence is written nowhere.  Two tokens of one
 * call must not have the same place. */
int bfhip_cache_append(const bfhip_paged_desc *desc, const bfhip_rows *k, const bfhip_rows *v,
                       const bfhip_pages *k_pages, const bfhip_pages *v_pages,
                       void *stream, char *error, size_t error_cap);

/* Attention of the new tokens over the cache, causal: token i of n stands at
 * position lengths[b] - n + i and sees the keys up to its own.  Scores, bias,
 * softmax, out and lse ([heads, tokens] or NULL) are those of
 * bfhip_attention_forward, and so is what is said there of rows without keys and
 * of rows outside every sequence; but probabilities meet the values with what their
 * rounding left, as if they had twice the type's precision.  Made for few tokens per sequence: a key head's
 * keys are read once for each 16 rows (token, head of its group), so that long
 * prompts take several times as long as by bfhip_attention_forward; the work is
 * split over the keys as the lengths on the device say.  Keys past a query's
 * position and what pages hold past a length reach no result, but a NaN or
 * infinity in the value of a token reaches the queries of the same sequence in
 * the same call that stand before it.
 * The workspace holds sums of keys that are shared out (at most 16 MiB) and eight
 * bytes per sequence.  tokens * heads / kv_heads at most 2^30. */
size_t bfhip_paged_attention_workspace(const bfhip_paged_desc *desc);

int bfhip_paged_attention(const bfhip_paged_desc *desc, const bfhip_rows *q,
                          const bfhip_pages *k_pages, const bfhip_pages *v_pages,
                          const bfhip_rows *out, float *lse, void *workspace,
                          size_t workspace_bytes, void *stream, char *error, size_t error_cap);

/* -------------------------------------------------------------- gated linear
 * h = act(x Wg^T) * (x Wu^T), both products, the activation and their product
 * in one kernel: x [rows, features], Wg and Wu [hidden, features], h [rows,
 * hidden].  act: silu, v / (1 + e^-v); gelu, v (1 + erf(v / sqrt 2)) / 2; relu,
 * max(v, 0).  gate and up (both or neither NULL): the two products in fp32,
 * which the backward pass takes (in 16 bits they would double the error of its
 * gradients).
 *
 * Backward, with g = gate, u = up and dh the gradient of h:
 *   dg = dh * u * act'(g),  du = dh * act(g)
 *   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
 * dx, or dWg and dWu together, may be NULL where they are not wanted.  dg and du
 * are rounded to the type where they enter the matrix cores (up to 16384 of each enter
 * with what the rounding left, as if they had twice the precision); fp16's are
 * multiplied by a power of two on the way (their largest comes near 2^14 or 2^15), so
 * that they may be of any size.  A result beyond the type's range is infinite.
 * relu'(0) = 0.
 *
 * Matrices: row r at element r * <name>.stride (at least the row's length, of no
 * account where there is at most one row), the elements of a row contiguous.
 * Any alignment will do; x and weights whose pointers, strides and rows are
 * multiples of 16 bytes (and strides below 2 Mi elements) need no copy.  Wg and Wu
 * have one stride.  Results overlap nothing.  rows at most 0x7fff0000, features and
 * hidden 1 .. 2^20, no matrix of more than 2^40 elements; calls of which a product has
 * 2^23 tiles or more are refused (of 128 rows by 64 hidden elements forward, of 128 by 128
 * elements of dx or of both dWg and dWu backward; in 16 bits of twice as many both ways).  The workspace holds dg and
 * du (and what their rounding left), copies of x and the weights where they need them
 * (backward, and forward with more than 32 rows, or 16 where hidden * features is above
 * 12 Mi, in fp32 4 Mi), and, where results are few beside the sums'
 * lengths, parts of sums (at most 256 MiB). */
enum { BFHIP_SILU = 0, BFHIP_GELU = 1, BFHIP_RELU = 2 };

typedef struct {
    void *data;
    long long stride;
} bfhip_matrix;

typedef struct {
    int type;
    int activation;
    long long rows;
    long long features;
    long long hidden;
} bfhip_gated_desc;

size_t bfhip_gated_linear_workspace(const bfhip_gated_desc *desc, const bfhip_matrix *x,
                                    const bfhip_matrix *w_gate, const bfhip_matrix *w_up);
size_t bfhip_gated_linear_backward_workspace(const bfhip_gated_desc *desc, const bfhip_matrix *x,
                                             const bfhip_matrix *w_gate, const bfhip_matrix *w_up);

int bfhip_gated_linear(const bfhip_gated_desc *desc, const bfhip_matrix *x,
                       const bfhip_matrix *w_gate, const bfhip_matrix *w_up,
                       const bfhip_matrix *h, const bfhip_matrix *gate, const bfhip_matrix *up,
                       void *workspace, size_t workspace_bytes,
                       void *stream, char *error, size_t error_cap);

int bfhip_gated_linear_backward(const bfhip_gated_desc *desc, const bfhip_matrix *dh,
                                const bfhip_matrix *x, const bfhip_matrix *w_gate,
                                const bfhip_matrix *w_up, const bfhip_matrix *gate,
                                const bfhip_matrix *up, const bfhip_matrix *dx,
                                const bfhip_matrix *dw_gate, const bfhip_matrix *dw_up,
                                void *workspace, size_t workspace_bytes,
                                void *stream, char *error, size_t error_cap);

/* Which kernel a product goes by; on the host, nothing is launched.  For tests,
 * which see by it that their sizes reach every kernel.  product: 0 the forward
 * pass, 1 dx, 2 dWg and dWu.  plan[0] the kind: 0 small tiles, 1 deep, 2 low, 3
 * large, 4 the forward kernel for few rows (whose other entries are zero); plan[1]
 * tiles that one workgroup computes, plan[2] tiles that are split along the
 * contraction, plan[3] into how many parts, plan[4] whether both gradients go in
 * one launch where both are wanted, plan[5] whether dg and du enter in two parts. */
int bfhip_gated_linear_plan(const bfhip_gated_desc *desc, int product, int plan[6], char *error,
                            size_t error_cap);

#ifdef __cplusplus
}
#endif

#endif
