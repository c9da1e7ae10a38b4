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

#ifdef __cplusplus
}
#endif

#endif
