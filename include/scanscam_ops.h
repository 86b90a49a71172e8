/*
 * scanscam_ops.h -- C ABI of the operators of a state space layer in
 * libscanscam_hip.so: the selective scan, the short causal convolution before
 * it, and the root-mean-square norm with the residual's addition. They have no
 * counterpart in the reference, whose one operator is the scan of scanscam_hip.h.
 *
 * Conventions are those of scanscam_hip.h: device pointers, the caller
 * allocates every output and the workspace, calls are asynchronous on `stream`,
 * the return value is 0 or a SCANSCAM_E* code, and nothing is launched when an
 * error is returned. Each call takes one struct of arguments, read during the
 * call only. Pointers marked "or NULL" leave their part of the operator out.
 *
 * Types. `dtype` (SCANSCAM_F32, SCANSCAM_BF16 or SCANSCAM_F16) is that of the
 * activations and of everything not named otherwise; arithmetic is fp32.
 * Parameters have types of their own (a code beside each). Strides are in
 * elements, must be >= 0, and are of the levels above the unit-stride dimension.
 *
 * Sequences. Activations are [batch, T, channels]. With `offsets`
 * ([sequences + 1], 32-bit, or 64-bit where offsets64 is set) batch must be 1 and
 * sequence s is tokens offsets[s] ... offsets[s+1] - 1, which may be none;
 * offsets are read on the device only, must not decrease and should run from 0 to
 * T. Without, sequences must equal batch and each has T tokens. Offsets that break
 * the rule give results without meaning, but no access outside of the tensors.
 */
#ifndef SCANSCAM_OPS_H
#define SCANSCAM_OPS_H

#include "scanscam_hip.h"

/* A call takes up to so many channels (the norm 32768), and fewer than so many tokens of all batch elements, sequences or rows. */
#define SCANSCAM_MOST_CHANNELS (1 << 20)
#define SCANSCAM_MOST_TOKENS ((INT64_C(1) << 31) - (INT64_C(1) << 20))

#ifdef __cplusplus
extern "C" {
#endif

/* 8-bit outputs of the norm: integers, and the floating-point type of 4 exponent and 3 mantissa bits without infinities. */
enum { SCANSCAM_I8 = 16, SCANSCAM_F8 = 17 };
enum { SCANSCAM_ACT_NONE = 0, SCANSCAM_ACT_SILU = 1 };

/* A tensor of activations, [batch, T, channels] or, for B and C, [batch, T, groups, N]. */
typedef struct scanscam_tokens {
    void *p;
    int64_t batch; /* stride from batch element to batch element */
    int64_t token; /* stride from token to token */
    int64_t group; /* B and C: stride from group to group */
} scanscam_tokens;

/* A parameter: dense, of type `dtype`. */
typedef struct scanscam_param {
    const void *p;
    int32_t dtype;
    int32_t unused;
} scanscam_param;

/*
 * Selective scan over whole sequences. With d = dt + dt_bias (softplus of it where `softplus` is set),
 * for every channel c of group g and every n < N
 *     h[t][c][n] = exp(d[t][c] * A[c][n]) * h[t-1][c][n] + d[t][c] * x[t][c] * B[t][g][n]
 *     y[t][c] = (sum_n C[t][g][n] * h[t][c][n] + D[c] * x[t][c]) * silu(z[t][c])
 * with h[-1] = state_in (0 where NULL) and state_out = h after the last token. Channels are shared out to the
 * groups in order, channels / groups each. N is 1 ... 256.
 *
 * `saved`: for a backward call, the states that its tiles of time start from
 * (scanscam_selective_saved_bytes). The workspace (scanscam_selective_workspace_bytes)
 * is for calls that share the time of a sequence out over workgroups, and for
 * the sums of the backward call. Both need alignment to 16 bytes. Strides from token to token must stay below
 * SCANSCAM_MOST_TOKEN_STRIDE.
 */
#define SCANSCAM_MOST_TOKEN_STRIDE (1 << 22)
typedef struct scanscam_selective {
    int64_t batch, T, sequences, channels, groups, N;
    const void *offsets; /* or NULL */
    int32_t offsets64, dtype, softplus, parts; /* parts: of time that a sequence's channels are shared out in; 0: chosen */
    scanscam_tokens x, dt, B, C, z, y;         /* z: or NULL */
    scanscam_param A;                          /* [channels, N] */
    scanscam_param D, dt_bias;                 /* [channels], or NULL */
    const float *state_in;                     /* [sequences, channels, N], or NULL */
    float *state_out;                          /* or NULL */
    void *saved;                               /* forward: written, or NULL; backward: read */
    /* Backward call only. */
    scanscam_tokens gy, gx, gdt, gB, gC, gz;   /* gradients; gz exactly where z is given */
    float *gA, *gD, *gdt_bias;                 /* [channels, N], [channels], [channels]; gD, gdt_bias: or NULL */
    const float *gstate_out;                   /* gradient of state_out, or NULL */
    float *gstate_in;                          /* or NULL */
    void *workspace;
    size_t workspace_bytes;
} scanscam_selective;

int scanscam_selective_fwd(const scanscam_selective *args, void *stream);
int scanscam_selective_bwd(const scanscam_selective *args, void *stream);
/* Only the sizes, dtype, parts and whether offsets are given are looked at. */
size_t scanscam_selective_saved_bytes(const scanscam_selective *args);
size_t scanscam_selective_workspace_bytes(const scanscam_selective *args, int direction);

/*
 * One token of each of `rows` sequences: the formulas above with h[t-1] read from and h[t] written to `state`
 * ([slots, channels, N], dense), at row slot[i] for the token of row i (row i where slot is NULL). A slot outside of
 * 0 ... slots - 1 marks a row without a sequence: its y is 0 and no state changes. Two rows must not share a slot.
 * The `batch` strides are not looked at.
 */
typedef struct scanscam_selective_step {
    int64_t rows, channels, groups, N, slots;
    const void *slot;          /* or NULL */
    int32_t slot64, dtype, softplus, unused;
    scanscam_tokens x, dt, B, C, z, y; /* z: or NULL */
    scanscam_param A, D, dt_bias;      /* D, dt_bias: or NULL */
    float *state;
} scanscam_selective_step;

int scanscam_selective_step_fwd(const scanscam_selective_step *args, void *stream);

/*
 * Causal convolution of every channel with taps of its own, 1 to 8 of them:
 *     y[t][c] = act(bias[c] + sum_k weight[c][k] * x[t - (K-1) + k][c])
 * with state_in ([sequences, K - 1, channels], 0 where NULL) as the K - 1 inputs before a sequence; state_out
 * are the K - 1 inputs before its next token.
 */
typedef struct scanscam_conv {
    int64_t batch, T, sequences, channels, K;
    const void *offsets; /* or NULL */
    int32_t offsets64, dtype, activation, unused;
    scanscam_tokens x, y;
    scanscam_param weight;  /* [channels, K] */
    scanscam_param bias;    /* [channels], or NULL */
    const void *state_in;   /* or NULL */
    void *state_out;        /* or NULL */
    /* Backward call only. */
    scanscam_tokens gy, gx;
    float *gweight, *gbias; /* [channels, K], [channels]; gbias: or NULL */
    const void *gstate_out; /* or NULL */
    void *gstate_in;        /* or NULL */
    void *workspace;        /* scanscam_conv_workspace_bytes, backward */
    size_t workspace_bytes;
} scanscam_conv;

int scanscam_conv_fwd(const scanscam_conv *args, void *stream);
int scanscam_conv_bwd(const scanscam_conv *args, void *stream);
size_t scanscam_conv_workspace_bytes(const scanscam_conv *args); /* only the sizes and dtype are looked at */

/* One token of each of `rows` sequences; `state` is [slots, K - 1, channels], slots as in the selective scan's step. */
typedef struct scanscam_conv_step {
    int64_t rows, channels, K, slots;
    const void *slot; /* or NULL */
    int32_t slot64, dtype, activation, unused;
    scanscam_tokens x, y;
    scanscam_param weight, bias; /* bias: or NULL */
    void *state;
} scanscam_conv_step;

int scanscam_conv_step_fwd(const scanscam_conv_step *args, void *stream);

/*
 * Root-mean-square norm of rows:
 *     sum = x + residual, in the residual's type (x where there is none)
 *     y = sum * rstd * weight,  rstd = 1 / sqrt(mean(sum^2) + eps)
 * What is stored in `sum` is what is normalised, so that the backward call, which has only that, gives the gradient of
 * what was computed. With out_dtype SCANSCAM_I8 or SCANSCAM_F8 a row is stored in 8 bits: scale = max |y| / 127 or / 448
 * (1 where the row is zero) and y / scale, rounded to nearest even; a row that holds a NaN or an infinity has the scale NaN (its integers are 0).
 * Rows whose squares add up to more than fp32 holds (values of some 1e19) come out as zeros, as rstd does. Up to 32768 channels.
 */
typedef struct scanscam_norm {
    int64_t rows, channels;
    int64_t x_stride, residual_stride; /* from row to row; outputs and gradients are dense */
    const void *x, *residual;          /* residual: or NULL */
    scanscam_param weight;             /* [channels] */
    void *y, *sum;                     /* sum: exactly where residual is given */
    float *rstd;                       /* [rows], or NULL */
    float *scale;                      /* [rows], 8-bit outputs only */
    float eps;
    int32_t dtype, residual_dtype, out_dtype;
    /* Backward call only: reads sum (x where there is no residual), rstd, and these. */
    const void *gy;                    /* of `dtype` */
    const void *gsum;                  /* of residual_dtype, or NULL */
    void *gx;                          /* of `dtype` */
    void *gresidual;                   /* of residual_dtype, or NULL */
    float *gweight;
    void *workspace;                   /* scanscam_norm_workspace_bytes, backward */
    size_t workspace_bytes;
} scanscam_norm;

int scanscam_norm_fwd(const scanscam_norm *args, void *stream);
int scanscam_norm_bwd(const scanscam_norm *args, void *stream);
size_t scanscam_norm_workspace_bytes(const scanscam_norm *args); /* only the sizes are looked at */

#ifdef __cplusplus
}
#endif

#endif /* SCANSCAM_OPS_H */
