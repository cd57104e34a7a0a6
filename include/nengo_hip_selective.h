/*
 * nengo_hip_selective.h -- arguments of the operators for blocks that filter selectively: the
 * short causal convolution, the selective scan and the gated norm (included by nengo_hip.h,
 * which holds the entry points).  No counterpart in the reference, whose synapses are filters
 * with constant matrices (nengo_ocl/clra_nonlinearities.py:577-803).
 *
 * The structs lie in HOST memory and are read during the call; the pointers in them are
 * device pointers.  Strides are in elements.  Optional arrays are NULL.
 */
#ifndef NENGO_HIP_SELECTIVE_H
#define NENGO_HIP_SELECTIVE_H

/* types of elements */
#define NHIP_F32 0
#define NHIP_BF16 1
#define NHIP_F16 2

/* An array of rows, one per token of a sequence and (where it has them) head or group: the
 * element c of head h of token t of sequence s lies at
 *     p + s * seq + t * token + h * head + c        (sequences side by side: starts == NULL)
 *     p + (starts[s] + t) * token + h * head + c    (sequences back to back)               */
typedef struct nhip_rows {
    const void *p;
    long long seq, token, head;
} nhip_rows;

/* Which tokens there are.  starts == NULL: n_seqs sequences of `length` tokens.  Otherwise
 * sequence s holds the tokens starts[s] ... starts[s + 1] - 1 of `n_tokens` (int32, device;
 * offsets outside 0 ... n_tokens are cut to that range, lengths below zero are zero; results of
 * tokens that no sequence holds are not written, those of sequences that overlap are undefined).
 * n_tokens is at most 0x7fff0000. */
typedef struct nhip_tokens {
    const int *starts;
    long long n_tokens;
    int n_seqs, length;
} nhip_tokens;

/* u[t, d] = bias[d] + sum_k weight[d, k] x[t - width + 1 + k, d];  y = u, or u / (1 + exp(-u))
 * where silu != 0.  Tokens before a sequence's first: initial[s, width - 1, channels], or
 * zeros.  final[s, width - 1, channels]: the last width - 1 inputs of each sequence, those of
 * `initial` among them where it is shorter.
 * Gradients (nhip_causal_conv_grad): dy, dfinal -> dx, dinitial (type of x), dweight
 * [channels, width], dbias (float32). */
typedef struct nhip_conv_args {
    nhip_tokens tokens;
    int type, channels, width, silu;
    nhip_rows x, dy;
    const float *weight, *bias;          /* [channels, width], [channels] or NULL */
    const void *initial;                 /* type of x, contiguous, or NULL */
    void *y, *final;                     /* y: contiguous, as many rows as tokens */
    const void *dfinal;
    void *dx, *dinitial;
    float *dweight, *dbias;
    void *workspace;                     /* gradients only */
    long long workspace_bytes;
} nhip_conv_args;

/* One token each of n requests: state[slot, width - 1, channels] (oldest first; slot stride
 * `state_stride`) is read, moved on by one token and written.  slots == NULL: request r has
 * slot r.  A request whose slot is not in 0 ... n_slots - 1 gets zeros and changes nothing. */
typedef struct nhip_conv_step_args {
    int type, channels, width, silu, n, n_slots;
    const int *slots;
    const void *x;                       /* [n, channels], row stride x_stride */
    long long x_stride, state_stride;
    const float *weight, *bias;
    void *state, *y;                     /* y: [n, channels], contiguous */
} nhip_conv_step_args;

/* The scan: with step[t, h] = f(dt[t, h] + dt_bias[h]), f the identity or softplus,
 *     S[t] = exp(step A[h]) S[t - 1] + step x[t] (x) B[t]      (dim x states, float32)
 *     y[t] = S[t] C[t] + D[h] x[t]
 * for each of n_heads heads; B and C are shared by the n_heads / n_groups heads of a group.
 * S before a sequence's first token: initial[s, n_heads, dim, states], or zeros; final: after
 * its last.  softplus(-inf), like that of the lowest value of a type, is zero: such a token reads the
 * state and leaves it as it is.  Gradients (nhip_selective_scan_grad): dy, dfinal -> dx, ddt, dB, dC (contiguous,
 * types of x, dt, x, x), dA, dD, ddt_bias (float32, [n_heads]), dinitial (float32). */
typedef struct nhip_scan_args {
    nhip_tokens tokens;
    int type, dt_type, softplus;
    int n_heads, dim, n_groups, states;
    nhip_rows x, dt, B, C, dy;
    const float *A, *D, *dt_bias;        /* [n_heads]; D and dt_bias may be NULL */
    const float *initial, *dfinal;
    void *y;
    float *final;
    void *dx, *ddt, *dB, *dC;
    float *dA, *dD, *ddt_bias, *dinitial;
    void *workspace;
    long long workspace_bytes;
} nhip_scan_args;

/* One token each of n requests: state[slot, n_heads, dim, states] (float32; slot stride
 * `state_stride`) is read and written.  slots as above. */
typedef struct nhip_scan_step_args {
    int type, dt_type, softplus;
    int n_heads, dim, n_groups, states, n, n_slots;
    const int *slots;
    nhip_rows x, dt, B, C;               /* token: stride between requests; seq is not used */
    const float *A, *D, *dt_bias;
    float *state;
    long long state_stride;
    void *y;                             /* [n, n_heads, dim], contiguous */
} nhip_scan_step_args;

/* u = x, or x * gate / (1 + exp(-gate)); norm(v) = v / sqrt(mean(v^2) + eps) over each of
 * `groups` equal parts of a row.
 *   after == 0:  v = residual + scale * u (u without a residual), out = norm(v) * weight
 *   after != 0:  out = residual + scale * (norm(u) * weight)
 * `scale` needs `residual`; v_out (after == 0 with a residual only) gets v.
 * Gradients (nhip_block_norm_grad): dout, and dv of v_out -> dx, dgate, dresidual (not where
 * after != 0: there it is dout), dweight, dscale (float32). */
typedef struct nhip_norm_args {
    int type, channels, groups, after;
    long long rows;
    float eps;
    const void *x, *gate, *residual;     /* [rows, channels], row strides below */
    long long x_stride, gate_stride, residual_stride;
    const float *weight, *scale;
    void *out, *v_out;                   /* contiguous */
    const void *dout, *dv;
    long long dout_stride, dv_stride;
    void *dx, *dgate, *dresidual;
    float *dweight, *dscale;
    void *workspace;
    long long workspace_bytes;
} nhip_norm_args;

#endif /* NENGO_HIP_SELECTIVE_H */
