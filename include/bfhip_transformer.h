/*
 * Stateless transformer operators on AMD gfx950, served by libbfhip.so: layer
 * norm, learned position bias by buckets, and attention over packed sequences,
 * each with its backward pass.  They stand beside the stateless linear and
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

#ifdef __cplusplus
}
#endif

#endif
