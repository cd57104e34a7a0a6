/*
 * nengo_hip_tokens.h -- arguments of the operators beside and behind blocks over tokens: the layer norm,
 * the gated projection of a feed-forward block, and the losses over a vocabulary (included by
 * nengo_hip.h, which holds the entry points).  No counterpart in the reference.
 *
 * The structs lie in HOST memory and are read during the call; the pointers in them are
 * device pointers.  Strides are in elements.  Optional arrays are NULL.  Types: NHIP_F32, NHIP_BF16, NHIP_F16.
 */
#ifndef NENGO_HIP_TOKENS_H
#define NENGO_HIP_TOKENS_H

/* v = x, or residual + x;  u = (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps);  out = u weight + bias.
 * Gradients (nhip_layer_norm_grad): dout, and dv of v_out -> dx (that of the residual too), dweight, dbias
 * (float32). */
typedef struct nhip_layer_norm_args {
    int type, channels;
    long long rows;
    float eps;
    const void *x, *residual;            /* [rows, channels], row strides below */
    long long x_stride, residual_stride;
    const float *weight, *bias;          /* [channels]; bias may be NULL */
    void *out, *v_out;                   /* contiguous; v_out with a residual only */
    const void *dout, *dv;
    long long dout_stride, dv_stride;
    void *dx;                            /* contiguous */
    float *dweight, *dbias;
    void *workspace;                     /* gradients only */
    long long workspace_bytes;
} nhip_layer_norm_args;

#define NHIP_ACT_SILU 0  /* g / (1 + exp(-g)) */
#define NHIP_ACT_GELU 1  /* g (1 + erf(g / sqrt(2))) / 2 */

/* y[n, f] = act(x[n] . gate[f]) (x[n] . up[f]).
 * Gradients (nhip_gated_projection_grad): dy -> dx, dgate, dup (contiguous, of the type of x). */
typedef struct nhip_gated_args {
    int type, activation, channels, features;
    long long rows;
    const void *x, *gate, *up;           /* [rows, channels], [features, channels] twice */
    long long x_stride, gate_stride, up_stride;
    void *y;                             /* [rows, features], contiguous */
    const void *dy;
    long long dy_stride;
    void *dx, *dgate, *dup;
    void *workspace;
    long long workspace_bytes;
} nhip_gated_args;

/* z[n, v] = (x[n] . weight[v]) / temperature,  lse[n] = log sum_v exp(z[n, v]);  temperature: 2^-126 to 2^126.
 * top == 0:  targets[n] is a word, loss[n] = lse[n] - z[n, targets[n]].
 * top > 0:   targets[n, top] are words and target_logits[n, top] a teacher's logits there: with
 *            q = softmax(target_logits[n] / temperature),
 *            loss[n] = sum_k q[k] (log q[k] - z[n, targets[n, k]] + lse[n]).
 *            Entries whose word is outside the vocabulary, or whose logit is -inf, are left out.
 * Rows whose word is outside the vocabulary, or without entries, count nothing: loss and lse are zero there,
 * whatever x holds.  Gradients (the *_grad entries): dloss, and lse as the forward pass wrote it -> dx,
 * dweight (contiguous, of the type of x). */
typedef struct nhip_loss_args {
    int type, channels, words, top;
    int wide_targets;                    /* targets are 64-bit integers, otherwise 32-bit ones */
    int logits_type;
    long long rows;
    float temperature;
    const void *x, *weight;              /* [rows, channels], [words, channels] */
    long long x_stride, weight_stride;
    const void *targets, *target_logits; /* contiguous */
    float *loss, *lse;                   /* [rows]; lse is only read by the gradients */
    const float *dloss;                  /* [rows] */
    void *dx, *dweight;
    void *workspace;
    long long workspace_bytes;
} nhip_loss_args;

#endif /* NENGO_HIP_TOKENS_H */
