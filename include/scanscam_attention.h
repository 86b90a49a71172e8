/*
 * scanscam_attention.h -- C ABI of the operators of a linear attention layer in
 * libscanscam_hip.so: attention with a decay for each head, over whole sequences
 * and for single tokens, and the norm of its heads with an activation and a gate.
 * They have no counterpart in the reference, whose one operator is the scan of
 * scanscam_hip.h.
 *
 * Conventions, types, sequences and slots are those of scanscam_ops.h. In a
 * scanscam_tokens `group` is the stride from head to head here.
 */
#ifndef SCANSCAM_ATTENTION_H
#define SCANSCAM_ATTENTION_H

#include "scanscam_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Linear attention with a decay for each head over whole sequences. For every head, with S a matrix of K x V values,
 *     S[t] = exp(decay[t]) * S[t-1] + k[t] v[t]^T
 *     y[t] = scale * S[t]^T q[t]
 * with S[-1] = state_in (0 where NULL) and state_out = S after the last token. `groups` heads of q and k are shared by
 * heads / groups neighbouring heads of v each; q, k are [batch, T, groups, K], v, y [batch, T, heads, V], K and V 1 ... 256.
 * decay: logs of the decays, [batch, T, heads] of type `decay_dtype`, unit-stride along the heads (`group` is not looked at), or
 * [heads] where `decay_fixed` is set (strides 0), or NULL (no decay). -infinity forgets everything. Logs above 0 let states
 * grow, as far as fp32 holds them and the exponential of what the logs of any 64 neighbouring tokens sum up to.
 *
 * `saved`: for a backward call, the states that its parts of time start from (scanscam_attend_saved_bytes, which may be 0). The
 * workspace (scanscam_attend_workspace_bytes) is for calls that share the time of a sequence out over
 * workgroups, and for the sums of the backward call. Both need alignment to 16 bytes. Strides from token to token must stay below SCANSCAM_MOST_TOKEN_STRIDE (decay's may be any), and
 * heads * K, heads * V are SCANSCAM_MOST_CHANNELS at most.
 */
#define SCANSCAM_MOST_HEAD 256
typedef struct scanscam_attend {
    int64_t batch, T, sequences, heads, groups, K, V;
    const void *offsets; /* or NULL */
    int32_t offsets64, dtype, decay_dtype, decay_fixed;
    float scale;
    int32_t parts;                 /* of time that a sequence of T tokens is shared out in; 0: chosen */
    scanscam_tokens q, k, v, y;
    scanscam_tokens decay;         /* or NULL */
    const float *state_in;         /* [sequences, heads, K, V], or NULL */
    float *state_out;              /* or NULL */
    void *saved;                   /* forward: written, or NULL; backward: read (NULL where it has no bytes) */
    /* Backward call only. */
    scanscam_tokens gy, gq, gk, gv;
    float *gdecay;                 /* [batch, T, heads], or [heads] where decay_fixed is set; or NULL */
    const float *gstate_out;       /* gradient of state_out, or NULL */
    float *gstate_in;              /* or NULL */
    void *workspace;
    size_t workspace_bytes;
} scanscam_attend;

int scanscam_attend_fwd(const scanscam_attend *args, void *stream);
int scanscam_attend_bwd(const scanscam_attend *args, void *stream);
/* Only the sizes, dtype, parts, decay_fixed and whether offsets are given are looked at. */
size_t scanscam_attend_saved_bytes(const scanscam_attend *args);
size_t scanscam_attend_workspace_bytes(const scanscam_attend *args, int direction);

/*
 * One token of each of `rows` sequences: the formulas above with S[t-1] read from and S[t] written to `state`
 * ([slots, heads, K, V], dense), slots as in the selective scan's step. q, k are [rows, groups, K], v, y [rows, heads, V],
 * decay [rows, heads] (token stride 0: [heads]) or NULL. The `batch` strides are not looked at.
 */
typedef struct scanscam_attend_step {
    int64_t rows, heads, groups, K, V, slots;
    const void *slot; /* or NULL */
    int32_t slot64, dtype, decay_dtype;
    float scale;
    scanscam_tokens q, k, v, y, decay;
    float *state;
} scanscam_attend_step;

int scanscam_attend_step_fwd(const scanscam_attend_step *args, void *stream);

/*
 * Norm of every group of a row's channels, with an activation and a gate:
 *     u = (x - mean) * rstd * weight + bias,  mean and variance over the group's channels,  rstd = 1 / sqrt(variance + eps)
 *     y = act(u) * silu(z)
 * Channels are shared out to the groups in order, channels / groups each, SCANSCAM_MOST_GROUP at most. weight, bias (0 without) and z are each
 * optional. The backward call reads x, z and the parameters again, and the statistics are computed anew from them.
 */
#define SCANSCAM_MOST_GROUP 8192
typedef struct scanscam_group_norm {
    int64_t rows, channels, groups;
    int64_t x_stride, z_stride;      /* from row to row; y and the gradients are dense */
    const void *x, *z;               /* z: or NULL */
    scanscam_param weight, bias;     /* [channels], or NULL */
    void *y;
    float eps;
    int32_t dtype, activation, unused;
    /* Backward call only. */
    const void *gy;
    void *gx, *gz;                   /* gz: exactly where z is given */
    float *gweight, *gbias;          /* each exactly where its parameter is given */
    void *workspace;                 /* scanscam_group_norm_workspace_bytes, aligned to 16 bytes */
    size_t workspace_bytes;
} scanscam_group_norm;

int scanscam_group_norm_fwd(const scanscam_group_norm *args, void *stream);
int scanscam_group_norm_bwd(const scanscam_group_norm *args, void *stream);
size_t scanscam_group_norm_workspace_bytes(const scanscam_group_norm *args); /* only the sizes, dtype and which parameters are given are looked at */

#ifdef __cplusplus
}
#endif

#endif /* SCANSCAM_ATTENTION_H */
