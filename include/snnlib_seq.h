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

/* Most tokens in a call (or positions of a sample, or samples times groups), most rows in a table, most columns of a row. */
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
 * partial sums of a row per 16 tokens, 32 where there are more than 8192.  0 for invalid arguments. */
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
 * C must be a multiple of G; S * G and P may be no more than SNNSEQ_MAX_TOKENS.  P == 0 or C == 0 with S*G > 0 groups
 * is SNNLIF_ERR_ARG (a group without values has no statistics).  `workspace`: snnseq_gn_act_workspace_bytes() bytes.
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

/* Most values of a key and of a value, and most heads times batch entries, of a gated delta call.  Over more than one
 * step, heads times batch entries times 2 * ceil(Dv / 32) may be no more than SNNSEQ_MAX_TOKENS. */
#define SNNSEQ_MAX_KEY   128
#define SNNSEQ_MAX_VALUE 65536
#define SNNSEQ_MAX_HEADS 65535

/*
 * Operands of the gated delta rule, F32 or BF16 (F64: SNNLIF_ERR_UNSUPPORTED).  With S [Dk, Dv] per batch entry and
 * value head, zero or `state` before the first step,
 *   S_t = exp(g_t) S_{t-1} + beta_t k_t (v_t - exp(g_t) S_{t-1}^T k_t)^T,   o_t = scale * S_t^T q_t
 * q, k [T, B, Hk, Dk] and v [T, B, Hv, Dv] with the given strides (in elements: step, batch entry, head; the Dk or Dv
 * values of a row are dense); g, beta dense [T, B, Hv] fp32; states dense [B, Hv, Dk, Dv] fp32.  Hv is a multiple
 * of Hk; value head h uses key head h / (Hv / Hk).  g <= 0 is the decay's logarithm (-inf forgets everything);
 * keys are expected at length one or below, as the recurrence multiplies by up to |k|^2 - 1 otherwise.
 * `lengths` ([B] int32, may be NULL): the time steps of batch entry b at or behind lengths[b] do not exist.  They leave the
 * state alone, their outputs and gradients are zero, and what the operands hold there is not looked at.  A value within a
 * sequence that is not finite reaches all later outputs, and may reach earlier ones of its chunk of 64 steps (and the
 * gradients of its chunk); a single step does not have the latter.
 */
typedef struct snnseq_delta {
    int64_t T, B, Hk, Hv, Dk, Dv;
    int64_t q_strides[3], k_strides[3], v_strides[3];
    double scale;
    const void *q, *k, *v;
    const float *g, *beta;
    const float* state;       /* may be NULL */
    const int32_t* lengths;   /* may be NULL */
    int dtype;
} snnseq_delta;

/* Bytes of device memory (`saved`) the forward works in.  for_backward != 0: and leaves behind for the backward, per
 * chunk of 64 steps and value head the fp32 state before it, the rows added to it and 64 x 64 matrices, per key head the
 * keys.  for_backward == 0: scratch, smaller.  0 for invalid arguments. */
size_t snnseq_gated_delta_saved_bytes(const snnseq_delta* call, int for_backward);

/* o dense [T, B, Hv, Dv]; state_out [B, Hv, Dk, Dv] (may be NULL): the state after the last step.  o and state_out do not
 * depend on for_backward by a bit. */
int snnseq_gated_delta_fp(const snnseq_delta* call, void* o, float* state_out, void* saved, size_t saved_bytes,
                          int for_backward, void* stream);

size_t snnseq_gated_delta_bp_workspace_bytes(const snnseq_delta* call);

/*
 * Backward, from the forward's operands and what it saved.  grad_o [T, B, Hv, Dv] with strides; grad_state_out (may be
 * NULL: zero) the gradient of the last state.  Gradients are dense and shaped as their operands (grad_q, grad_k over
 * Hk heads, summed over the value heads that share them); grad_state (may be NULL) that of the initial state.
 */
int snnseq_gated_delta_bp(const snnseq_delta* call, const void* saved, size_t saved_bytes, const void* grad_o,
                          const int64_t* grad_o_strides, const float* grad_state_out, void* grad_q, void* grad_k,
                          void* grad_v, float* grad_g, float* grad_beta, float* grad_state, void* workspace,
                          size_t workspace_bytes, void* stream);

/* One time step (T == 1, `state` given, no lengths): o [B, Hv, Dv], and the state after it in state_out, which may be
 * `state` itself (but must not overlap it otherwise).  One launch, no workspace. */
int snnseq_gated_delta_step(const snnseq_delta* call, void* o, float* state_out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SNNLIB_SEQ_H */
