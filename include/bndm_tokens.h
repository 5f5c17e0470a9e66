/*
 * bndm_tokens.h -- C ABI of libbndm_tokens.so: operators over image and video tokens on the MI355X (gfx950), next to the
 * layers that bndm_hip.h evaluates inside its handles: products with bias, activation and residual (the network's linear
 * layers), rotary positions on several axes, and differential attention.  bndm_amd/tokens.py is their Python form.
 *
 * Conventions are those of bndm_hip.h: plain pointers and sizes, caller-owned device memory (workspaces too), 0 on success, a
 * positive hipError_t or a negative BNDM_E_* code otherwise with bndm_tokens_last_error() naming the reason, launches
 * asynchronous on the given stream (which belongs to the current device), no synchronisation, no state kept between calls.
 * Strides count elements.
 */
#ifndef BNDM_TOKENS_H
#define BNDM_TOKENS_H

#include <stddef.h>
#include <stdint.h>

#include "bndm_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define BNDM_TOKENS_ABI_VERSION 1

int         bndm_tokens_abi_version(void);
const char *bndm_tokens_last_error(void);

/* ------------------------------------------------------------------------------------------
 * Linear layer  y = act(x W^T + b) + r
 *   x [M, K] rows ldx apart, W [N, K] contiguous, b [N] or NULL, r [M, N] rows ldr apart or NULL, y [M, N] contiguous,
 *   all of `dtype` (BNDM_DTYPE_F16 / _BF16), summed in 32 bits and rounded once.
 *   z: NULL, or [M, N] contiguous for x W^T + b before the activation, which the backward pass reads.
 * ------------------------------------------------------------------------------------------ */
#define BNDM_ACT_NONE 0
#define BNDM_ACT_SILU 1
#define BNDM_ACT_GELU 2  /* z Phi(z) */

/* bytes of scratch of the call below (0 where it needs none); scratch starts at 16 bytes */
size_t bndm_tokens_linear_workspace_bytes(int64_t M, int64_t N, int64_t K);

int bndm_tokens_linear(const void *x, int64_t ldx, const void *w, const void *bias, const void *residual, int64_t ldr,
                       void *y, void *z, int64_t M, int64_t N, int64_t K, int act, int dtype, void *workspace,
                       size_t workspace_bytes, void *stream);

size_t bndm_tokens_linear_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int act, int want_dbias);

/* Gradients of the layer from dy [M, N] (rows lddy apart): dz = dy act'(z), dx = dz W, dw = dz^T x, dbias = column sums of dz.
 * z: the forward pass's (NULL for BNDM_ACT_NONE).  dx [M, K], dw [N, K], dbias [N] contiguous; any of them may be NULL. */
int bndm_tokens_linear_backward(const void *dy, int64_t lddy, const void *z, const void *x, int64_t ldx, const void *w,
                                void *dx, void *dw, void *dbias, int64_t M, int64_t N, int64_t K, int act, int dtype,
                                void *workspace, size_t workspace_bytes, void *stream);

/* ------------------------------------------------------------------------------------------
 * Rotary positions on several axes
 *   q [B, N, q_heads, D] and k [B, N, k_heads, D] (or k == NULL, k_heads == 0) with strides {batch, token, head}, elements of a
 *   head contiguous; outputs contiguous.  The D / 2 pairs of a head -- elements (j, j + D/2), or (2j, 2j + 1) if interleaved --
 *   are dealt out to the axes in `sections` (pairs of each axis, adding up to D / 2); pair i of an axis with s pairs turns by
 *   position[axis] * base^(-i / s).  inverse != 0 turns back, which is the backward pass.
 *   positions [B or 1, N, axes] with strides {batch (0: shared), token, axis}; position_type 0 int32, 1 int64, 2 float32.
 *   dtype BNDM_DTYPE_F16 / _BF16 / _F32.  Angles are formed in 64 bits.
 * ------------------------------------------------------------------------------------------ */
#define BNDM_TOKENS_MAX_AXES 4

int bndm_tokens_rotary(const void *q, const int64_t q_strides[3], void *q_out, int q_heads,
                       const void *k, const int64_t k_strides[3], void *k_out, int k_heads,
                       const void *positions, const int64_t position_strides[3], int position_type,
                       int64_t B, int64_t N, int D, const int *sections, int axes, double base, int interleaved, int inverse,
                       int dtype, void *stream);

/* ------------------------------------------------------------------------------------------
 * Differential attention  o = (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v
 *   q [B, Nq, 2 H, D]: heads 2h and 2h + 1 are the first and second map of head h; k [B, Nk, 2 Hk, D] likewise; v [B, Nk, Hk, Dv];
 *   head h reads key head h / (H / Hk).  lam [H] of `dtype` or float.  o [B, Nq, H, Dv] contiguous.  D a multiple of 8 up to 128, Dv a
 *   multiple of 8 up to 256.  Strides {batch, token, head} are multiples of 8, pointers of 16 bytes.
 *   kv_lengths int32 [B] or NULL: keys and values past a sequence's length are not read.
 *   causal != 0: query i of sequence b sees keys j <= start_b + i, start_b = q_start[b] or, where q_start is NULL, Nk - Nq; keys past the
 *   last query's are not read (those that only later queries than some see must be finite).
 *   A query that sees no key gives zeros, and zero gradients.
 * ------------------------------------------------------------------------------------------ */
typedef struct bndm_attention_shape {
    int64_t B, Nq, Nk;
    int     H, Hk, D, Dv;
    int64_t q_strides[3], k_strides[3], v_strides[3];
    int     causal;
    int     dtype;
    int     lam_f32;  /* lam and dlam are float, not `dtype` */
    float   scale;    /* > 0 */
} bndm_attention_shape;

/* bytes of scratch of the forward pass (0 where it needs none) */
size_t bndm_tokens_attention_workspace_bytes(const bndm_attention_shape *s);

/* o2 [B, Nq, H, Dv] (the second map's output) and lse float [B, 2 H, Nq] are what the backward pass reads; both NULL otherwise */
int bndm_tokens_attention(const bndm_attention_shape *s, const void *q, const void *k, const void *v, const void *lam,
                          const int32_t *q_start, const int32_t *kv_lengths, void *o, void *o2, float *lse,
                          void *workspace, size_t workspace_bytes, void *stream);

size_t bndm_tokens_attention_backward_workspace_bytes(const bndm_attention_shape *s);

/* dout: strides {batch, token, head} in dout_strides; dq, dk, dv contiguous in the shapes of q, k, v; dlam [H] */
int bndm_tokens_attention_backward(const bndm_attention_shape *s, const void *q, const void *k, const void *v, const void *lam,
                                   const int32_t *q_start, const int32_t *kv_lengths, const void *o, const void *o2,
                                   const float *lse, const void *dout, const int64_t dout_strides[3], void *dq, void *dk,
                                   void *dv, void *dlam, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* BNDM_TOKENS_H */
