/* nxg_rows.h -- floating-point operators over the packed rows of a batch, with their gradients.
 *
 * Next to the encoder's own fp32 operators (nxg_linear.h), whose every rounding is the
 * reference's, these are what a layer needs between its projections when it is trained, or run
 * with 16-bit rows or a causal mask:
 *
 *   nxg_rope_rows        rotary positions                     (beside nxg_qk_prep)
 *   nxg_layer_norm_rows  layer norm, forward and backward     (beside nxg_layer_norm)
 *   nxg_attention_rows   attention, forward and backward      (beside nxg_attention)
 *   nxg_qk_norm_rope_rows  RMS norms of queries and keys for each head, then their rotation, forward and backward: of layers that have
 *                          them (the encoder's own heads have nxg_qk_prep's tanh there, which has no gradient here)
 *   nxg_dropout_rows     dropout whose mask is drawn again where it is needed
 *   nxg_adapter_rows     low-rank adapters of many requests, forward and backward (beside nxg_linear_i8, which has no gradient)
 *
 * They have no counterpart in the reference (NexteraBERT.cpp), which only infers. Conventions
 * are nxg_linear.h's: device pointers on the current device, `stream` a hipStream_t, NXG_OK or an
 * NXG_E* code with nxg_last_error(), calls return without waiting. Nothing is allocated and nothing
 * kept between calls, so calls on different streams may overlap as long as they share no output
 * and no workspace. Every call can be captured into a HIP graph. An output shares no memory with
 * another array of its call, except where it may be that array itself.
 *
 * Types are nxg_type's numbers: NXG_TYPE_F32, NXG_TYPE_F16, NXG_TYPE_BF16. Sums, statistics and
 * products are fp32 or wider whatever the rows' type, but where a function says what it carries in
 * fewer bits; a result is rounded to its type once.
 *
 * Rows of several heads are given as a pointer and two strides in values (not bytes): value
 * (t, h, d) is at data + t * token_stride + h * head_stride + d. So the heads may lie inside a fused
 * projection's rows, or head after head. A stride of 0 repeats a row (inputs only).
 *
 * Packed documents: cu is device int32, n_seqs + 1 offsets, from 0 and not decreasing (an empty
 * document is allowed). Rows that no document covers have no part in a result of
 * nxg_attention_rows, nxg_adapter_rows and their gradients, and are not written. Other offsets give
 * unspecified rows but no access out of bounds.
 */
#ifndef NXG_ROWS_H
#define NXG_ROWS_H

#include "nxg_linear.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct nxg_rows {
    void *  data;
    int64_t token_stride;      /* in values */
    int64_t head_stride;
} nxg_rows;

/* ---------------------------------------------------------------------------
 * Rotary positions
 * ------------------------------------------------------------------------- */

/* How frequencies are scaled for positions past the trained length. */
#define NXG_ROPE_NONE     0   /* f_i = base^(-2i / n_rot) */
#define NXG_ROPE_LINEAR   1   /* f_i / factor */
#define NXG_ROPE_NTK      2   /* base * factor^(n_rot / (n_rot - 2)): what nxg_encoder does past rope.ntk_train_length */
#define NXG_ROPE_BY_PARTS 3   /* each f_i between f_i / factor (a pair of at most 1 turn over train_len positions) and f_i
                               * (32 turns or more), in between by its turns; results times 0.1 ln(factor) + 1 */

/* On the host: the n_rot / 2 frequencies in radians per position, and the factor on the result.
 *   n_rot  even, > 0 (> 2 for NTK);  base > 0;  factor >= 1 (ignored with NONE);  train_len > 0 with BY_PARTS
 *   freq   host double [n_rot / 2];  mscale  host float */
NXG_API int32_t nxg_rope_frequencies(int32_t n_rot, double base, int32_t scaling, double factor, int32_t train_len,
                                     double * freq, float * mscale);

/* How the n_rot first values of a head pair up. */
#define NXG_ROPE_HALF        0   /* (i, i + n_rot / 2) */
#define NXG_ROPE_INTERLEAVED 1   /* (2i, 2i + 1) */

/* Turns each pair (a, b) of the first n_rot values of every head by t = position * freq[i]:
 * (a cos t - b sin t, a sin t + b cos t) * mscale; values behind n_rot are copied. With `inverse`
 * it turns by -t: the gradient of the same call (with mscale as in the forward call), and the
 * sense in which the encoder's nxg_qk_prep turns. Angles are position * frequency in 64 bits, less
 * whole turns, so that far positions keep theirs.
 *   x, out     device rows of `type`, [T][n_head][head_dim]; out may be x (same strides). Sizes that would take
 *              2^24 workgroups of about 12 KiB of rows are refused
 *   freq       device double [n_rot / 2];  n_rot even, 0 < n_rot <= head_dim <= 1024
 *   positions  device int32 [T] (any value), or null: the row's place in its document by cu
 *   cu         device int32 [n_seqs + 1] (positions null); rows outside the documents count from the
 *              start of the nearest document before them */
NXG_API int32_t nxg_rope_rows(int32_t type, const nxg_rows * x, int32_t T, int32_t n_head, int32_t head_dim,
                              const double * freq, int32_t n_rot, int32_t layout, float mscale, int32_t inverse,
                              const int32_t * positions, const int32_t * cu, int32_t n_seqs, const nxg_rows * out,
                              void * stream);

/* ---------------------------------------------------------------------------
 * Layer norm
 * ------------------------------------------------------------------------- */

/* y = (x - mean) * rstd * w + b per row, rstd = 1 / sqrt(mean((x - mean)^2) + eps).
 *   x, y         device rows of `type`, T x C, x_stride and y_stride values apart (y may be x, with its stride);
 *                C at most 2^23, T below 2^24 (2^26 with C up to 1,024)
 *   w, b         device [C] of w_type (`type` or F32), or null: 1 and 0
 *   mean, rstd   device float [T], or null: what nxg_layer_norm_rows_backward takes */
NXG_API int32_t nxg_layer_norm_rows(int32_t type, const void * x, int64_t x_stride, const void * w, const void * b,
                                    int32_t w_type, float eps, int32_t T, int32_t C, void * y, int64_t y_stride,
                                    float * mean, float * rstd, void * stream);

/* The gradients, with h = (x - mean) * rstd and g = dy * w:
 *   dx = rstd * (g - mean(g) - h * mean(g * h)),  dw = sum over rows of dy * h,  db = sum of dy
 * The sums over rows are taken in a fixed order: the same call gives the same bits.
 *   dy, x        device rows of `type`;  mean, rstd  as nxg_layer_norm_rows left them
 *   w            device [C] of w_type, or null: 1
 *   dx           device rows of `type`, or null;  may be dy or x, with its stride
 *   dw, db       device [C] of w_type, or null;  T = 0 gives zeros
 *   workspace    device memory, 16-byte aligned, nxg_layer_norm_rows_workspace_bytes(T, C) bytes (none with dw and db null) */
NXG_API int64_t nxg_layer_norm_rows_workspace_bytes(int32_t T, int32_t C);
NXG_API int32_t nxg_layer_norm_rows_backward(int32_t type, const void * dy, int64_t dy_stride, const void * x,
                                             int64_t x_stride, const float * mean, const float * rstd, const void * w,
                                             int32_t w_type, int32_t T, int32_t C, void * dx, int64_t dx_stride, void * dw,
                                             void * db, void * workspace, int64_t workspace_bytes, void * stream);

/* ---------------------------------------------------------------------------
 * Attention
 * ------------------------------------------------------------------------- */

/* Query i of a document of n queries and m keys stands at key position i + m - n (the last query at the
 * last key) and sees the keys j with i + m - n - left <= j <= i + m - n + right; -1 is no limit.
 * So (-1, -1) is full attention, (-1, 0) causal, (h, h) the encoder's sliding window |i - j| <= h. Query head
 * h reads KV head h / (n_head / n_kv_head). */
typedef struct nxg_attention_rows_params {
    int32_t type;              /* of every row: NXG_TYPE_F16 or NXG_TYPE_BF16 */
    int32_t n_head, n_kv_head, head_dim;   /* n_head: 1 to 65,536 times n_kv_head; head_dim: a multiple of 8, at most 128 */
    int32_t T_q, T_k;          /* rows of q and out, and of k and v: up to 2^30, T_q * n_head and T_k * n_kv_head below 2^31,
                                * and n_kv_head * 128-row tiles of both below 2^24 (a document more: a tile more) */
    int32_t n_seqs;
    const int32_t * cu_q;      /* device int32 [n_seqs + 1] */
    const int32_t * cu_k;
    int32_t left, right;
    float   scale;             /* of q k, positive */
} nxg_attention_rows_params;

/* out = softmax(scale q k^T) v over the keys that a query sees, lse = log of the sum of exp(scale q k)
 * over them. A query that sees no key gets zeros and -infinity. Keys and queries outside each
 * other's window have no part in a result, whatever they hold.
 *   q, out     T_q rows of n_head heads;  k, v  T_k rows of n_kv_head heads (data 16-byte aligned, strides
 *              multiples of 8). out may not overlap an input
 *   lse        device float [T_q][n_head]
 *   workspace  device memory, 16-byte aligned, or null: nxg_attention_rows_workspace_bytes gives the size on the current device (0 for
 *              all but launches of few queries over many keys, which share a document's keys out over
 *              workgroups; with less they share less) */
NXG_API int64_t nxg_attention_rows_workspace_bytes(const nxg_attention_rows_params * params);
NXG_API int32_t nxg_attention_rows(const nxg_attention_rows_params * params, const nxg_rows * q, const nxg_rows * k,
                                   const nxg_rows * v, const nxg_rows * out, float * lse, void * workspace,
                                   int64_t workspace_bytes, void * stream);

/* The gradients of nxg_attention_rows, summed over the query heads that share a KV head, in a fixed
 * order: the same call gives the same bits.
 *   dout       T_q rows of n_head heads;  q, k, v, out, lse  as the forward call had and left them
 *   dq, dk, dv rows as q, k and v (written for every row of a document; keys that no query sees get zeros).
 *              They may not overlap an input or each other
 *   workspace  device memory, 16-byte aligned, nxg_attention_rows_backward_workspace_bytes (on the current device) bytes */
NXG_API int64_t nxg_attention_rows_backward_workspace_bytes(const nxg_attention_rows_params * params);
NXG_API int32_t nxg_attention_rows_backward(const nxg_attention_rows_params * params, const nxg_rows * dout,
                                            const nxg_rows * q, const nxg_rows * k, const nxg_rows * v,
                                            const nxg_rows * out, const float * lse, const nxg_rows * dq,
                                            const nxg_rows * dk, const nxg_rows * dv, void * workspace,
                                            int64_t workspace_bytes, void * stream);

/* ---------------------------------------------------------------------------
 * Norms of queries and keys, and their rotation
 * ------------------------------------------------------------------------- */

/* What both directions take. Per head of a token: y = turn(x * rstd * w), rstd = 1 / sqrt(mean(x^2) + eps) over the
 * head's values, turn as nxg_rope_rows with the same freq, n_rot, layout, mscale, positions and cu. */
typedef struct nxg_qk_norm_rope_params {
    int32_t type;              /* of every row */
    int32_t T, n_head, n_kv_head, head_dim;    /* queries have n_head heads, keys n_kv_head; head_dim up to 1024 */
    const void * wq, * wk;     /* device [head_dim] of w_type */
    int32_t w_type;            /* `type` or F32 */
    float   eps;
    const double * freq;       /* as nxg_rope_rows */
    int32_t n_rot, layout;
    float   mscale;
    const int32_t * positions, * cu;
    int32_t n_seqs;
} nxg_qk_norm_rope_params;

/* Both in one launch. q_out and k_out may be q and k (same strides); k and k_out null: queries alone (n_kv_head 0). Sizes that
 * would take 2^24 workgroups of about 12 KiB of rows are refused. */
NXG_API int32_t nxg_qk_norm_rope_rows(const nxg_qk_norm_rope_params * params, const nxg_rows * q, const nxg_rows * k,
                                      const nxg_rows * q_out, const nxg_rows * k_out, void * stream);

/* The gradients, with u = the turn back of dy (times mscale), h = x * rstd, g = u * w:
 *   dx = rstd * (g - h * mean(g * h)),  dw = sum over tokens and heads of u * h
 * The sums are taken in a fixed order: the same call gives the same bits.
 *   dq_out, dk_out  gradients of q_out and k_out;  q, k  the forward call's inputs
 *   dq, dk          may be dq_out or q, dk_out or k, with their strides
 *   dwq, dwk        device [head_dim] of w_type;  T = 0 gives zeros
 *   workspace       device memory, 16-byte aligned, nxg_qk_norm_rope_rows_workspace_bytes(params) bytes */
NXG_API int64_t nxg_qk_norm_rope_rows_workspace_bytes(const nxg_qk_norm_rope_params * params);
NXG_API int32_t nxg_qk_norm_rope_rows_backward(const nxg_qk_norm_rope_params * params, const nxg_rows * dq_out,
                                               const nxg_rows * dk_out, const nxg_rows * q, const nxg_rows * k,
                                               const nxg_rows * dq, const nxg_rows * dk, void * dwq, void * dwk,
                                               void * workspace, int64_t workspace_bytes, void * stream);

/* ---------------------------------------------------------------------------
 * Dropout
 * ------------------------------------------------------------------------- */

/* out = residual + (kept ? x / (1 - p) : 0), p rounded to a multiple of 2^-16. Whether value (t, c) is kept is drawn again by
 * every call from (seed, offset, t, c) alone, whatever the strides and types: the same call on the gradient of out, without the
 * residual, gives the gradient of x. The generator is Philox 4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): key = seed's low and
 * high 32 bits, counter = (c / 8, t, offset's low and high 32 bits); value c takes the 16 bits 16 (c % 2) of result word
 * (c % 8) / 2 and is dropped where they are below p 2^16.
 *   x, residual, out  device rows of `type`, T x C (C up to 2^30), their strides in values; residual may be null; out may be x or residual,
 *                     with its stride
 *   p        0 up to 65535 / 65536
 *   offset   another for every mask of a seed;  step  device int64 [1] that is added to it, or null: read when the call
 *            runs, so that replays of a captured graph draw new masks */
NXG_API int32_t nxg_dropout_rows(int32_t type, const void * x, int64_t x_stride, const void * residual, int64_t residual_stride,
                                 int32_t T, int32_t C, double p, uint64_t seed, uint64_t offset, const int64_t * step,
                                 void * out, int64_t out_stride, void * stream);

/* ---------------------------------------------------------------------------
 * Low-rank adapters
 * ------------------------------------------------------------------------- */

/* Document d has adapter i = ids[d], or none (an id that is not in 0 .. n_adapters - 1). All adapters have one rank and one
 * scale: a smaller rank is filled up with zeros in a and b, another scale multiplied into b (db is then that product's gradient). */
typedef struct nxg_adapter_rows_params {
    int32_t type;              /* of the rows */
    int32_t w_type;            /* of a and b: `type`; F32 rows take F32, F16 or BF16 */
    int32_t T, n_in, n_out;    /* T below 2^24; n_in, n_out up to 2^20 */
    int32_t rank;              /* 1 to 128 */
    int32_t n_adapters;        /* n_adapters * rank * n_in and * n_out below 2^31, * (n_in + n_out) below 2^30 */
    int32_t n_seqs;            /* below 2^22 */
    const int32_t * cu;        /* device int32 [n_seqs + 1] */
    const int32_t * ids;       /* device int32 [n_seqs] */
    const void * a;            /* device [n_adapters][rank][n_in] */
    const void * b;            /* device [n_adapters][n_out][rank] */
    float   scale;             /* of every adapter's share, finite */
} nxg_adapter_rows_params;

/* s = x a_i^T,  y = base + scale * s b_i^T  per row of a document; rows of a document without an adapter get base, and 0 as s.
 * s is fp32. Beside F16 and BF16 rows it enters the product with b as the sum of two bf16 values, off by at most 2^-16 of it, and F16
 * weights as such a sum too, without the product of both second parts (2^-16 of a term more); beside F32 rows every product is
 * fp32. A row of x or base that holds an infinity or a NaN, or whose s does, may give NaN where it would give an infinity; it has no
 * part in other rows.
 *   x      device rows of n_in values, base, y  of n_out (their strides in values); base may be null: 0. y may be base, with its stride
 *   s      device float [T][rank]: what nxg_adapter_rows_backward takes */
NXG_API int32_t nxg_adapter_rows(const nxg_adapter_rows_params * params, const void * x, int64_t x_stride, const void * base,
                                 int64_t base_stride, void * y, int64_t y_stride, float * s, void * stream);

/* The gradients, with g = scale * dy b_i:
 *   dx = base + g a_i,  da_i = sum of g^T x,  db_i = scale * sum of dy^T s  over the rows of the documents with adapter i
 * The sums are taken in a fixed order: the same call gives the same bits. g and s are carried as s in the forward call. A row of dy or x
 * that holds an infinity or a NaN, or whose g or s does, may give NaN for infinities in its row of dx and anywhere in da_i and db_i of
 * its adapter; it has no part in other rows' dx and other adapters' gradients.
 *   dy       device rows of n_out values;  x, s  as the forward call had and left them
 *   base     rows of n_in values (the shared projection's part of dx), or null: 0;  dx  rows, or null; may be base, with its stride
 *   da, db   device, as a and b, or null; zeros for an adapter that no row has. n_adapters * (n_in / 64 + n_out / 64), each rounded up,
 *            below 2^22 - 1
 *   workspace  device memory, 16-byte aligned, nxg_adapter_rows_backward_workspace_bytes (on the current device) bytes */
NXG_API int64_t nxg_adapter_rows_backward_workspace_bytes(const nxg_adapter_rows_params * params);
NXG_API int32_t nxg_adapter_rows_backward(const nxg_adapter_rows_params * params, const void * dy, int64_t dy_stride, const void * x,
                                          int64_t x_stride, const float * s, const void * base, int64_t base_stride, void * dx,
                                          int64_t dx_stride, void * da, void * db, void * workspace, int64_t workspace_bytes,
                                          void * stream);

#ifdef __cplusplus
}
#endif

#endif /* NXG_ROWS_H */
