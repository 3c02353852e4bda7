/*
 * snnlib_seq.h -- C ABI of the token-layer operators in libsnnlif_gfx950.so: embedding, group norm with
 * an activation (channels last) and the gated delta rule, as hand-written HIP kernels for MI355X (gfx950).
 *
 * They extend the layer operators of snnlib_lif.h to networks over token sequences on the same time axis;
 * the reference has no counterpart.  Storage types and return codes are those of snnlib_lif.h
 * (snnlif_strerror names them), and so are the conventions: DEVICE pointers on the current HIP device, inputs only read, outputs
 * fully overwritten, nothing allocated or kept between calls, `stream` a hipStream_t passed as void*, no
 * synchronisation, safe under HIP graph capture (only kernels are enqueued).  A `workspace` is device memory
 * of at least the stated size, aligned to 16 bytes and private to the call until the stream has run it.
 * Results do not depend on the order in which workgroups run.
 */
#ifndef SNNLIB_SEQ_H
#define SNNLIB_SEQ_H

#include <stddef.h>
#include <stdint.h>

#include "snnlib_lif.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SNNSEQ_ABI_VERSION 1

/* ABI version of the loaded library (== SNNSEQ_ABI_VERSION it was built with). */
int snnseq_abi_version(void);

/* Types of `tokens`. */
#define SNNSEQ_TOKEN_I32 0
#define SNNSEQ_TOKEN_I64 1

/* Most tokens in a call, most rows in a table, and most columns of a row. */
#define SNNSEQ_MAX_TOKENS   8388608
#define SNNSEQ_MAX_CHANNELS 1048576

/*
 * Embedding lookup: out[n, :] = scale * weight[tokens[n], :].
 * tokens [N]; weight V rows of C values, `row_stride` values apart; out dense [N, C] of `dtype` (F32, F64, BF16).
 * A token outside [0, V) stands for no token: its row of `out` is zero.
 */
int snnseq_embed_fp(const void* tokens, const void* weight, void* out, int dtype, int token_dtype, int64_t N,
                    int64_t V, int64_t C, int64_t row_stride, double scale, void* stream);

/* Bytes of device workspace snnseq_embed_bp needs: the sorted order (8 bytes per token, 4 per table row) and two
 * partial sums of a row per 64 tokens.  0 for invalid arguments. */
size_t snnseq_embed_bp_workspace_bytes(int dtype, int64_t N, int64_t V, int64_t C);

/*
 * Gradient of the table: grad_weight[v, :] = scale * sum of grad[n, :] over n with tokens[n] == v.
 * grad dense [N, C]; grad_weight dense [V, C], rows without a token are zero.  Sums are held in 32 bits (64 for
 * F64) and taken in an order fixed by the tokens alone: results are reproducible.
 */
int snnseq_embed_bp(const void* tokens, const void* grad, void* grad_weight, int dtype, int token_dtype, int64_t N,
                    int64_t V, int64_t C, double scale, void* workspace, size_t workspace_bytes, void* stream);

/* Activations of the group norm. */
#define SNNSEQ_ACT_NONE 0
#define SNNSEQ_ACT_RELU 1
#define SNNSEQ_ACT_SILU 2 /* z / (1 + exp(-z)) */
#define SNNSEQ_ACT_GELU 3 /* z * (1 + erf(z / sqrt(2))) / 2 */

/*
 * Group norm with an activation, channels last.  x, y dense [S, P, C]: S samples (time steps times batch
 * entries), P positions, C channels in G groups of C/G consecutive channels; weight, bias [C].  Per sample and
 * group, over its P * C/G values:
 *   mean = E[x],  rstd = 1 / sqrt(E[(x - mean)^2] + eps),  y = act((x - mean) * rstd * weight[c] + bias[c])
 * mean, rstd [S, G] of the arithmetic type (float for F32 and BF16, double for F64), for the backward.
 * C must be a multiple of G.  P == 0 or C == 0 with S*G > 0 groups is SNNLIF_ERR_ARG (a group without values
 * has no statistics).  `workspace`: snnseq_gn_act_workspace_bytes() bytes.
 */
int snnseq_gn_act_fp(const void* x, const void* weight, const void* bias, void* y, void* mean, void* rstd, int dtype,
                     int64_t S, int64_t P, int64_t C, int64_t G, double eps, int act, void* workspace,
                     size_t workspace_bytes, void* stream);

/*
 * Its backward, from the forward's inputs and statistics:  z = (x - mean) * rstd * weight + bias,  gz = grad_y * act'(z),
 *   grad_bias[c] = sum gz,  grad_weight[c] = sum gz * xhat  over samples and positions,
 *   grad_x = rstd * (gz*weight - E[gz*weight] - xhat * E[gz*weight*xhat])  with the means over the group.
 * act'(0) of the relu is 0.  Sums are held in 32 bits or more, in a fixed order.
 */
int snnseq_gn_act_bp(const void* x, const void* weight, const void* bias, const void* mean, const void* rstd,
                     const void* grad_y, void* grad_x, void* grad_weight, void* grad_bias, int dtype, int64_t S,
                     int64_t P, int64_t C, int64_t G, int act, void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of device workspace of the two calls above (backward = 0 / 1); 0 also where none is needed. */
size_t snnseq_gn_act_workspace_bytes(int dtype, int64_t S, int64_t P, int64_t C, int64_t G, int backward);

#ifdef __cplusplus
}
#endif

#endif /* SNNLIB_SEQ_H */
