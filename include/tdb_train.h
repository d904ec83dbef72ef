/*
 * tdb_train.h -- C ABI of the operators that training a DeBERTa-v2/v3 encoder needs beside tdb_attn.h's forward ones: dropout,
 * LayerNorm (with dropout and residual in front of it), attention, the loss over a vocabulary, each with its gradient, and the norm of all gradients with clipping.
 *
 * Conventions are those of tdb_attn.h: plain pointers and sizes, element strides, buffers (workspaces too) of the caller, TDB_OK or a
 * negative TDB_ERR_* code, nothing allocated, freed or synchronised, launches on the stream passed in.
 *
 * Random numbers.  `seed` is a device pointer to one 64-bit number.  A counter of four 32-bit words gives eight 16-bit numbers, the halves (low
 * first) of the words that Philox-4x32 with seven rounds makes of it under the seed as its key (low word first).  A value is dropped where its
 * number is below `threshold` (0 .. 65536, the probability in units of 2^-16; 0: nothing is dropped and `seed` is not read); the
 * others are multiplied by 65536 / (65536 - threshold).  No mask is stored: whoever needs it again computes it again.
 * A dropped value is 0 whatever it was, infinities and NaN included.
 */
#ifndef TDB_TRAIN_H
#define TDB_TRAIN_H

#include <stdint.h>

#include "tdb_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * y = dropout(x), n values back to back; also its backward pass (x: the gradient of y).  Value i has number i mod 8 of counter
 * (i / 8, low word and high word, 0, 0).  x and y may be the same memory.
 */
int tdb_dropout(const void* x, void* y, int64_t n, int32_t dtype, int32_t threshold, const int64_t* seed, void* stream);

/*
 * LayerNorm over rows of `hidden` (1 .. 32768) values, z = dropout(x) + residual, y = (z - mean) / sqrt(var + eps) * weight + bias, var without
 * Bessel's correction.  residual NULL: z = dropout(x).  The random numbers of row r, column c are those of value r * hidden + c in
 * tdb_dropout.  weight and bias (both or neither NULL) have weight_dtype: that of x, or TDB_F32.  Strides are those of rows.
 * Backward: dx, dresidual (NULL: not wanted, or no residual) from x, residual, dy; dweight and dbias (NULL: not wanted; both or neither) of weight_dtype.
 * The statistics are computed again from x and residual.  workspace: tdb_norm_workspace() floats, where dweight is wanted.
 */
typedef struct tdb_norm_args {
    int32_t dtype, weight_dtype, hidden, threshold;
    int64_t rows;
    float   eps;
    int32_t reserved;
    const void *x, *residual, *weight, *bias, *dy;
    void *y, *dx, *dresidual, *dweight, *dbias;
    float* workspace;
    const int64_t* seed;
    int64_t x_stride, residual_stride, dy_stride, y_stride, dx_stride, dresidual_stride;
} tdb_norm_args;

int tdb_norm_fwd(const tdb_norm_args* args, void* stream);
int tdb_norm_bwd(const tdb_norm_args* args, void* stream);
/* floats of workspace for a backward call of these sizes (host only; at most 2^31) */
int64_t tdb_norm_workspace(int64_t rows, int32_t hidden);

/*
 * Attention as in tdb_attn.h (fixed layout [batch, heads, max_seqlen, head_dim] with optional lengths, or packed where cu_seqlens is there:
 * [total_tokens, heads, head_dim], stride_b unused), position terms as tables, with dropout on the probabilities; head_dim a multiple of 8 up to 64.
 * The probability of key j for query i of head h in sequence b has number 4 (j / 16 mod 2) + j mod 4 of counter (4 (j / 32) + j / 4 mod 4, i, b * heads + h, 1).
 * Forward writes o and lse, float32 [heads, rows], rows = batch * max_seqlen or total_tokens: the logarithm (base 2) of the sum of each row's exponentials, for the backward
 * call, which also reads o.  In 16 bits o_rest, [heads, rows, head_dim] back to back, takes what rounding took from o and goes to the backward call with it; NULL in both calls:
 * the gradients are made from o as it is rounded, and are the less exact the longer the rows.
 * Backward writes dq, dk, dv and the gradients of the tables, [heads, 2 span, head_dim] with rows back to back.  Rows beyond a sequence's length, and packed rows of no
 * sequence, are zeros in every result; what the inputs hold there does not matter.  workspace: tdb_attn_train_workspace() bytes for the same arguments, 16-byte aligned.  Besides a few bytes for each row and table
 * it holds, for as many heads at a time as fit (at least one), the scores' gradients in 2 GiB: element size * sum of (length * max_seqlen), lengths rounded up to 64 and max_seqlen
 * at most total_tokens where packed; and where there are tables, in 2 GiB as well, 1 KiB for each 64 x 64 of these scores and sums by relative position: at most the largest of half
 * the scores' gradients in 16 bits, 96 MiB, and 128 KiB for each of these heads and 64 tokens of max_seqlen.
 * delta_lut must not fall as the relative position rises, from 1 - max_seqlen to max_seqlen - 1 (max_seqlen: at most total_tokens where packed): the gradients' sums are made by runs
 * of positions that share a row.  tdb_delta_table's rows fall where max_position - 1 <= position_buckets / 2, beyond position_buckets / 2 + 1 tokens.
 * delta_lut, lut_half and span belong to the tables: without pos_key and pos_query they are not looked at.
 * The gradient of rows whose sequence has one token is zero in q, k and the tables.  Results must not overlap each other or an input.
 */
typedef struct tdb_train_attn_args {
    int32_t dtype, batch, heads, head_dim, max_seqlen, total_tokens, threshold, span, lut_half;
    float   sm_scale;               /* positive */
    const void *q, *k, *v;
    void*   o;
    const void* dout;
    void *dq, *dk, *dv;
    int64_t q_stride_b, q_stride_h, q_stride_l;
    int64_t k_stride_b, k_stride_h, k_stride_l;
    int64_t v_stride_b, v_stride_h, v_stride_l;
    int64_t o_stride_b, o_stride_h, o_stride_l;
    int64_t dout_stride_b, dout_stride_h, dout_stride_l;
    int64_t dq_stride_b, dq_stride_h, dq_stride_l;
    int64_t dk_stride_b, dk_stride_h, dk_stride_l;
    int64_t dv_stride_b, dv_stride_h, dv_stride_l;
    const int32_t *seqlens_k, *cu_seqlens, *delta_lut;
    const void *pos_key, *pos_query;
    int64_t pos_key_stride_h, pos_key_stride_r, pos_query_stride_h, pos_query_stride_r;
    void *dpos_key, *dpos_query;
    int64_t dpos_key_stride_h, dpos_query_stride_h;
    float*  lse;
    void*   workspace;
    int64_t workspace_bytes;
    const int64_t* seed;
    void*   o_rest;
} tdb_train_attn_args;

int tdb_attn_train_fwd(const tdb_train_attn_args* args, void* stream);
int tdb_attn_train_bwd(const tdb_train_attn_args* args, void* stream);
int64_t tdb_attn_train_workspace(const tdb_train_attn_args* args);

/*
 * Softmax cross entropy over a vocabulary, from hidden states x [rows, hidden] and an output layer weight [vocab, hidden], bias [vocab] or NULL (bias_dtype: that of x, or
 * TDB_F32): of each row whose label (64 bits) is not ignore_index the logarithm of the sum of the exponentials of its logits less the label's logit, in natural units.  The logits are
 * never in memory.  reduction 0: loss [rows], 0 where a row does not count; 1: their sum; 2: their mean over the rows that count (none: NaN).  loss is float32.
 * A label that is neither ignore_index nor in [0, vocab) makes its row's loss NaN, and every gradient that the row goes into.  Rows that do not count are not read.
 * weight: rows 4-byte aligned (so of an even stride in 16 bits) and at most 4 MiB apart.  dweight: rows at most 4 MiB apart.  x: rows of any stride, aligned to their values.
 * Forward fills `state` (tdb_loss_state() bytes), which the backward call reads; x is not read again.  Both take a workspace of tdb_loss_workspace() bytes, 16-byte aligned like
 * the state.  The backward one holds the gradient of the logits in the type of x, up to 2 GiB at a time or 256 columns of it, partial sums of dx of 1 KiB hidden for each CU or 4
 * bytes for each value of x, those of dweight of at most 256 MiB where a small vocabulary meets many rows, and without a reduction one more x.
 * Backward: dx, dweight, dbias (of bias_dtype); NULL: not wanted.  dloss: of the sum or mean one float32, without reduction one for each row, dloss_stride apart.
 * Rows of dx that do not count are zeros.  Everything is added up in a fixed order.
 */
typedef struct tdb_loss_args {
    int32_t dtype, bias_dtype, hidden, reduction;
    int64_t rows, vocab, ignore_index;
    const void *x, *weight, *bias;
    const int64_t* labels;
    float*  loss;
    void*   state;
    int64_t state_bytes;
    void*   workspace;
    int64_t workspace_bytes;
    const float* dloss;
    void *dx, *dweight, *dbias;
    int64_t x_stride, weight_stride, dloss_stride, dx_stride, dweight_stride;
} tdb_loss_args;

int tdb_loss_fwd(const tdb_loss_args* args, void* stream);
int tdb_loss_bwd(const tdb_loss_args* args, void* stream);
/* bytes for these sizes, types and reduction (host only) */
int64_t tdb_loss_state(const tdb_loss_args* args);
int64_t tdb_loss_workspace(const tdb_loss_args* args, int32_t backward);

/*
 * The norm of many tensors together, and clipping.  from, to, numel, from_dtype, to_dtype: host arrays with an entry for each tensor, read before the call returns; a tensor's values lie
 * back to back and are aligned to their own size.  norm: 2 (square root of the sum of squares), 1 (sum of magnitudes) or 0 (largest magnitude).  Sums are held in 64 bits and
 * added up in a fixed order; a NaN makes every norm NaN.
 * tdb_grads_norm writes the norm to `total` (float32, device) and leaves it in the workspace, tdb_grads_workspace() bytes for these sizes, 8-byte aligned.
 * tdb_grads_clip, behind it with the same sizes and workspace: to = from * min(1, max_norm / (norm + 1e-6)), in float32, rounded to to_dtype.  A result may be its own input (same
 * address and type), which is not written where that factor is 1; any other overlap of a result with an input or a result is refused.
 */
typedef struct tdb_grads_args {
    int32_t tensors, norm;
    double  max_norm;
    const void* const* from;
    void* const* to;
    const int64_t* numel;
    const int32_t *from_dtype, *to_dtype;
    float*  total;
    void*   workspace;
    int64_t workspace_bytes;
} tdb_grads_args;

int tdb_grads_norm(const tdb_grads_args* args, void* stream);
int tdb_grads_clip(const tdb_grads_args* args, void* stream);
int64_t tdb_grads_workspace(const tdb_grads_args* args);

#ifdef __cplusplus
}
#endif
#endif /* TDB_TRAIN_H */
