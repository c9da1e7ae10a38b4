/*
 * cchip operators: layer operators of language models on device-resident
 * data, next to the graphs of cchip_backend.h. The array DSL cannot express
 * them: its scans carry scalars, its tensors have no 16-bit types, and a
 * fused norm, gate, dropout and residual is several of its kernels. Like
 * cchip_program_run_resident_noalloc every call only issues work on `stream`
 * (NULL: the default stream), allocates nothing and may be captured into a
 * HIP graph; synchronise the stream before reading results on the host.
 *
 * Status codes and cchip_last_error() are those of cchip_runtime.h: a shape,
 * type, stride or missing buffer that an operator does not take is
 * CCHIP_INVALID_ARGUMENT before any device work.
 */
#ifndef CCHIP_OPERATORS_H
#define CCHIP_OPERATORS_H

#include <stddef.h>
#include <stdint.h>

#include "cchip_runtime.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the operators (the codes of cchip_backend.h go on). */
#define CCHIP_F32 0
#define CCHIP_BF16 5
#define CCHIP_F16 6

/* ---- Gated delta rule ---------------------------------------------------- */

/*
 * A linear recurrence whose state S is a key_dim x value_dim matrix, one for
 * each sequence and value head:
 *
 *   u_t = beta_t (v_t - exp(g_t) S_{t-1}^T k_t)
 *   S_t = exp(g_t) S_{t-1} + k_t u_t^T
 *   o_t = scale S_t^T q_t
 *
 * q and k have key_heads heads, v and o value_heads, a multiple of it: value
 * head h goes with key head h / (value_heads / key_heads). g and beta have
 * value_heads values a token and, like all tensors below, the type `dtype`;
 * states are f32, [sequence][value head][key_dim][value_dim], contiguous.
 * With `sequences` 0 the rows of the batch are the sequences; otherwise batch
 * is 1 and sequence i is the tokens offsets[i] .. offsets[i + 1] - 1 (i32 on
 * the device, `sequences` + 1 values from 0 to tokens, not decreasing;
 * values out of that range are clamped to it). A sequence may be empty: its
 * last state is its first.
 *
 * `states` non-zero: sequences begin from `state` (NULL: zeros) and their
 * last states or the gradients of their first ones are wanted; the products
 * that make a state then keep 24 bits of f32 operands. With `states` zero,
 * those arguments are NULL and a bf16 operator keeps 16 bits of them. Sums
 * and the states that go from chunk to chunk are f32 either way.
 *
 * A NaN or infinity in a token reaches the outputs of its own sequence and
 * value heads from the 64-token chunk it stands in onwards, in the backward
 * pass those up to that chunk's end.
 */
typedef struct {
  int dtype;
  int64_t batch, tokens, sequences;
  int key_heads, value_heads, key_dim, value_dim; /* key_dim <= 128 */
  int states;
  float scale;
} cchip_gated_delta;

/* What a call writes overlaps nothing that it reads, but for state_out, nor
   itself. A tensor [batch][token][head][dim]: the distances, in elements, of
   neighbours along the first three, of tokens 0 to 2^23; the elements of a
   head are adjacent. g and beta have no last dimension. */
typedef struct {
  void *data;
  int64_t batch, token, head;
} cchip_heads;

typedef struct {
  cchip_heads q, k, v, g, beta;
  cchip_heads o;                       /* forward: written */
  cchip_heads d_o;                     /* backward: read */
  cchip_heads dq, dk, dv, dg, dbeta;   /* backward: written */
  const int32_t *offsets;
  const float *state;                  /* forward: read */
  float *state_out;                    /* forward: written; may be `state` */
  const float *dstate_out;             /* backward: gradient of state_out, NULL: zero */
  float *dstate;                       /* backward: gradient of state, NULL: not wanted */
  void *saved;                         /* forward: written (NULL: no backward pass follows); backward: read */
} cchip_gated_delta_io;

/* Bytes of workspace that a forward and a backward call need (a workspace
   holds nothing between calls; calls that overlap need one each), and of
   `saved`. All are aligned to 16 bytes. A forward call that saves needs no
   workspace, nor does one of at most 16 tokens a sequence, not packed, that
   does not: it runs the recurrence itself. */
int cchip_gated_delta_sizes(const cchip_gated_delta *op, size_t *forward, size_t *backward, size_t *saved);
int cchip_gated_delta_forward(const cchip_gated_delta *op, const cchip_gated_delta_io *io, void *workspace,
                              size_t workspace_bytes, void *stream);
int cchip_gated_delta_backward(const cchip_gated_delta *op, const cchip_gated_delta_io *io, void *workspace,
                               size_t workspace_bytes, void *stream);

/* ---- Attention ----------------------------------------------------------- */

/*
 * Causal attention with grouped heads: query t of head h sees, of key head
 * h / (heads / kv_heads), the keys up to its own token, counted from the end
 * of both,
 *
 *   j <= t + (keys of the sequence) - (tokens of the sequence)
 *   p_j = softmax_j(scale q_t . k_j),   o_t = sum_j p_j v_j
 *
 * heads is a multiple of kv_heads; sums, maxima and scores are f32. Weights
 * of 16-bit types are rounded to them on their way to the values, and the sum
 * that divides is of the rounded ones. A query
 * that sees no key, or whose every score is -infinity, has zeros for o. Three
 * kinds of batches:
 *
 *   `sequences` and `keys` 0: the rows of the batch are the sequences, with a
 *   key for each token.
 *   `sequences` > 0: batch is 1 and sequence i is the tokens offsets[i] ..
 *   offsets[i + 1] - 1, as for the gated delta rule; tokens of no sequence
 *   are left as they were in all that is written.
 *   `keys` > 0: k and v are caches of `keys` tokens a row of the batch, of
 *   which row i holds lengths[i] (i32 on the device, clamped to 0 .. keys),
 *   and q the last `tokens` of them; what a cache has behind its length is
 *   not looked at. Forward only.
 *
 * A NaN or infinity in k or v reaches the queries that see it and no others:
 * one in v as it is in f32, and in 16 bits as one or the other. Weighted
 * values are summed in f32 before the division by the weights' sum, which
 * values beyond 2^96 may overflow.
 * In the backward pass one in q, k, v or the gradient of o may reach the
 * gradients of other tokens of its sequence that stand within 128 of it, and
 * 16-bit elements there are taken in steps of 2^-38 of the largest among 64
 * neighbouring rows (tokens, for q and the gradient of o times the heads of a
 * group): whole down to 2^-28 of it.
 */
typedef struct {
  int dtype;
  int64_t batch, tokens, sequences, keys;
  int heads, kv_heads, head_dim; /* head_dim <= 128 */
  float scale;
} cchip_attention;

/* Tensors as in cchip_gated_delta_io; k, v, dk and dv have kv_heads heads and,
   with a cache, `keys` tokens. */
typedef struct {
  cchip_heads q, k, v;
  cchip_heads o;            /* forward: written; backward: read */
  cchip_heads d_o;          /* backward: read */
  cchip_heads dq, dk, dv;   /* backward: written */
  const int32_t *offsets, *lengths;
  void *saved;              /* forward: written (NULL: no backward pass follows); backward: read */
} cchip_attention_io;

int cchip_attention_sizes(const cchip_attention *op, size_t *forward, size_t *backward, size_t *saved);
int cchip_attention_forward(const cchip_attention *op, const cchip_attention_io *io, void *workspace, size_t workspace_bytes,
                            void *stream);
int cchip_attention_backward(const cchip_attention *op, const cchip_attention_io *io, void *workspace, size_t workspace_bytes,
                             void *stream);

/* ---- Dropout ------------------------------------------------------------- */

/*
 * Column c of row r is kept iff half c % 8 (16 bits, low halves first) of
 * Philox-4x32-10 at counter (c / 8, r, offset, offset >> 32) and key (seed,
 * seed >> 32) is at least round(65536 p). A kept value is scaled by
 * 65536 / (65536 - round(65536 p)); one that is not is zero whatever it was.
 * The mask is never stored: the backward pass draws it again. It does not
 * depend on strides. `step`, if not NULL, is a device word added to offset
 * when the kernel runs, so that a captured graph draws anew on each replay.
 */
typedef struct {
  int dtype;
  int64_t rows, cols; /* rows < 2^32, cols < 2^35, at most 2^42 elements */
  double p;           /* 0 <= p <= 1 */
  float scale;
} cchip_dropout;

/* A matrix: rows `row` elements apart, the elements of a row adjacent. */
typedef struct {
  void *data;
  int64_t row;
} cchip_rows;

typedef struct {
  uint64_t seed, offset;
  const uint64_t *step;
  cchip_rows x, residual, out;
} cchip_dropout_io;

/* out = residual + scale drop(x); residual.data NULL: no residual. The
   gradient of x is the same call on the gradient of out, without residual.
   out may be x or residual, row for row. */
int cchip_dropout_run(const cchip_dropout *op, const cchip_dropout_io *io, void *stream);

/* ---- Norm block ---------------------------------------------------------- */

/*
 * What stands between a block and the next one, on each row of `width`:
 *
 *   a = norm(y) post_weight + post_bias      (post: the norm, or none)
 *   b = a act(gate)                          (gate: none, sigmoid or silu)
 *   h = residual + scale channel_scale drop(b)
 *   n = norm(h) pre_weight + pre_bias        (pre: the next block's norm, or none)
 *
 * norm(x) is x / sqrt(mean(x^2) + eps), of x minus its mean for a layer
 * norm. Every parameter vector may be NULL (1 or 0 in its place), of type
 * dtype or f32. Rows of every tensor are apart by a stride of its own.
 */
#define CCHIP_NORM_NONE 0
#define CCHIP_NORM_RMS 1
#define CCHIP_NORM_LAYER 2
#define CCHIP_GATE_NONE 0
#define CCHIP_GATE_SIGMOID 1
#define CCHIP_GATE_SILU 2

typedef struct {
  int dtype, weight_dtype;
  int64_t rows, width; /* rows < 2^32, width <= 32768 */
  int post, pre, gate;
  float scale, eps;
  double p; /* of dropout */
} cchip_norm_block;

typedef struct {
  void *post_weight, *post_bias, *channel_scale, *pre_weight, *pre_bias;
} cchip_norm_params;

typedef struct {
  uint64_t seed, offset; /* of dropout, as in cchip_dropout_io */
  const uint64_t *step;
  cchip_norm_params params;
  cchip_norm_params grads;            /* backward: written; NULL: not wanted */
  cchip_rows y, gate;                 /* read by both */
  cchip_rows residual;                /* forward: read */
  cchip_rows h, n;                    /* forward: written; backward: h is read */
  cchip_rows dh, dn;                  /* backward: read */
  cchip_rows dy, dgate, dresidual;    /* backward: written; dgate, dresidual NULL: not wanted */
} cchip_norm_block_io;

/* h and n may each be `residual`, y or the gate, row for row, but not both the
   same. n is NULL iff pre is none. */
int cchip_norm_block_forward(const cchip_norm_block *op, const cchip_norm_block_io *io, void *stream);
/* From y, gate, the forward pass's h (needed iff pre is not none), and the
   gradients dh and dn of its results: the gradients of y, gate, residual and
   the parameters, those summed over rows in f32 in an order that does not
   change from run to run. What it writes overlaps nothing that it reads. */
int cchip_norm_block_workspace(const cchip_norm_block *op, size_t *bytes);
int cchip_norm_block_backward(const cchip_norm_block *op, const cchip_norm_block_io *io, void *workspace,
                              size_t workspace_bytes, void *stream);

/* ---- Norm and rotation of heads ------------------------------------------ */

/*
 * What stands between the projections of q and k and attention, on each head:
 *
 *   n = x / sqrt(mean(x^2) + eps) weight          (norm rms; none: n = x)
 *   (y_i, y_j) = (n_i cos a - n_j sin a, n_j cos a + n_i sin a),  a = position frequency_p
 *
 * for the rotary / 2 pairs p of the first `rotary` elements (even), (i, j) =
 * (p, p + rotary / 2) or, interleaved, (2 p, 2 p + 1); the others are n. The
 * angle is made in 64 bits. Weights are vectors of head_dim, of dtype or f32,
 * one of q and one of k (NULL: ones).
 *
 * With `keys` a call also writes to caches of `keys` tokens a row of the
 * batch: a token's y of k to k_cache and its v to v_cache, at its position;
 * one whose position is not in 0 .. keys - 1 is not written. Positions of a
 * row differ there.
 */
typedef struct {
  int dtype, weight_dtype;
  int64_t batch, tokens, keys; /* batch * tokens < 2^31 */
  int heads, kv_heads, head_dim, rotary; /* head_dim <= 512 */
  int interleaved, norm;       /* CCHIP_NORM_NONE or CCHIP_NORM_RMS */
  float eps;
} cchip_head_norm;

typedef struct {
  cchip_heads q, k;            /* read by both */
  cchip_heads v;               /* forward with keys: read */
  cchip_heads q_out, k_out;    /* forward: written, may be q and k; with keys k_out may be NULL */
  cchip_heads k_cache, v_cache; /* forward with keys: written at the tokens' positions */
  cchip_heads dq_out, dk_out;  /* backward: read */
  cchip_heads dq, dk;          /* backward: written, may be dq_out and dk_out */
  const int32_t *positions;    /* [batch][tokens]; NULL: 0, 1, 2, ... in each row */
  const float *frequencies;    /* radians a position, rotary / 2 */
  const void *q_weight, *k_weight;
  void *dq_weight, *dk_weight; /* backward: written; NULL: not wanted */
} cchip_head_norm_io;

int cchip_head_norm_forward(const cchip_head_norm *op, const cchip_head_norm_io *io, void *stream);
/* Gradients of the weights are summed over tokens and heads in f32, in an
   order that does not change from run to run. */
int cchip_head_norm_workspace(const cchip_head_norm *op, size_t *bytes);
int cchip_head_norm_backward(const cchip_head_norm *op, const cchip_head_norm_io *io, void *workspace, size_t workspace_bytes,
                             void *stream);

/* ---- Embedding ----------------------------------------------------------- */

/*
 *   out[t] = scale weight[ids[t]]
 *   dweight[w] = scale sum over t with ids[t] = w of dout[t]
 *
 * ids are i32; one that is not in 0 .. vocab - 1, such as a padding token's,
 * has a row of zeros and no gradient. The table is of dtype or f32. Sums are
 * f32, in an order that does not change from run to run (pieces of a word's
 * tokens, then the pieces). The backward pass writes all of dweight,
 * or, with `accumulate`, adds to the rows of the words that there are.
 */
typedef struct {
  int dtype, weight_dtype;
  int64_t tokens, vocab, width; /* tokens <= 2^30, vocab < 2^31, width <= 2^20 */
  float scale;
} cchip_embedding;

typedef struct {
  const int32_t *ids;
  cchip_rows weight, out;    /* forward: read, written */
  cchip_rows dout, dweight;  /* backward: read, written */
  int64_t accumulate;
} cchip_embedding_io;

int cchip_embedding_forward(const cchip_embedding *op, const cchip_embedding_io *io, void *stream);
int cchip_embedding_workspace(const cchip_embedding *op, size_t *bytes);
int cchip_embedding_backward(const cchip_embedding *op, const cchip_embedding_io *io, void *workspace, size_t workspace_bytes,
                             void *stream);

#ifdef __cplusplus
}
#endif

#endif
