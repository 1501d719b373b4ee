/*
 * C ABI of the hand-written state space kernels for AMD GPUs (libovl_ssm.so): the selective state space recurrence, its
 * gradient and its form for one new token, and the short causal convolution in front of it, its gradient and its form
 * for one new token.  They stand beside the row scans (ovl_scan.h) and the LSTM cell (ovl_lstm.h): recurrences with
 * run-time shapes that need no code generation on the machine that calls them.  The reference has no counterpart.
 *
 * Scan.  For every sequence b, channel c and token t, with n running over the `state` entries of a channel and g the
 * group of the channel (channels / groups neighbouring channels share the vectors B and C of their group):
 *
 *   dt      = log(1 + exp(delta[b,t,c] + delta_bias[c]))      or, without softplus, delta[b,t,c] + delta_bias[c]
 *   h[t,n]  = exp(dt * A[c,n]) * h[t-1,n] + dt * u[b,t,c] * B[b,t,g,n]         h[-1] = entering[b,c] or zero
 *   y       = sum over n of C[b,t,g,n] * h[t,n]  +  D[c] * u[b,t,c]
 *   out     = y * z * sigmoid(z)  with a gate z, else y
 *
 * Convolution, `width` taps per channel, line = the kept tokens followed by the sequence:
 *
 *   pre[t]  = bias[c] + sum over k of weight[c,k] * line[t + k]                 out = pre * sigmoid(pre), or pre
 *
 * With `lengths`, sequence b ends after lengths[b] tokens (clamped to 0 .. length): states and kept tokens are those
 * after its last token, outputs and gradients behind it are zero, and what the inputs hold there is not looked at.
 *
 * Conventions: tensor memory belongs to the caller and must be device accessible; sequences have their channels side by
 * side, batch and token strides (in elements) are free, but for the scan's token strides, which are 0 to 2^25; outputs are
 * dense.  All sums, states and gradients of parameters are float32; only what is stored in the tensors' type is rounded,
 * once.  The functions enqueue kernels on `hip_stream`, return without synchronising, allocate nothing (scratch memory is
 * handed in, its size is asked for first) and give the same bits for the same call.  They return an ovl_status
 * (ovl_launch.h): OVL_EINVAL for arguments they refuse, OVL_EHIP for a HIP error (text from ovl_ssm_last_error).
 *
 * Sizes: lengths up to 2^30, scans up to 2^22 channels, and what one launch takes (fewer than 2^32 work items), which is
 *   scan           batch * groups * ceil(channels / groups / 64) below 2^26; backward pass and step (there without groups)
 *                  below 2^24
 *                  backward pass also 2 * groups * batch * length * state + 1024 * ceil(channels * (entries + 2) / 64) below
 *                  2^32, entries = the state counted as the next of 8, 16, 32, 64
 *   convolution    batch * channels below 2^32, up to 8 times as much where wide accesses are possible; backward pass
 *                  channels * (width + 1) below 2^28, and batch * channels below 2^29 (more where channels are many)
 * Larger calls are refused.
 */
#ifndef OVL_SSM_H_
#define OVL_SSM_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the sequences: the codes of ovl_launch.h, and bfloat16, which the operator IR does not have. */
enum ovl_ssm_dtype { OVL_SSM_FLOAT16 = 1, OVL_SSM_FLOAT32 = 2, OVL_SSM_BFLOAT16 = 32 };

/* Largest distance of two tokens of a sequence, in elements, that the scan takes. */
#define OVL_SSM_MAX_TOKEN_STRIDE (1 << 25)

/* One sequence tensor [batch, length, channels], channels side by side; data NULL: absent. */
typedef struct ovl_ssm_sequence {
    const void* data;
    int64_t     batch_stride;
    int64_t     token_stride;
} ovl_ssm_sequence;

/* The vectors B or C [batch, length, groups, state], state entries side by side. */
typedef struct ovl_ssm_vectors {
    const void* data;
    int64_t     batch_stride;
    int64_t     token_stride;
    int64_t     group_stride;
} ovl_ssm_vectors;

typedef struct ovl_ssm_scan {
    uint32_t batch, length, channels, state, groups;   /* state 1 .. 64; groups divides channels */
    int32_t  dtype;                                    /* of u, delta, z, B, C and the sequences written */
    int32_t  softplus;
    ovl_ssm_sequence u, delta, z;                      /* z may be absent */
    ovl_ssm_vectors  B, C;
    const float*   A;                                  /* [channels, state] */
    const float*   D;                                  /* [channels] or NULL */
    const float*   delta_bias;                         /* [channels] or NULL */
    const float*   entering;                           /* [batch, channels, state] or NULL */
    const int32_t* lengths;                            /* [batch] or NULL */
} ovl_ssm_scan;

/* Bytes of scratch memory ovl_ssm_scan_forward (backward = 0) or ovl_ssm_scan_backward (backward = 1) needs, and of the
 * states a forward pass may keep for the backward pass; 0 for a scan that would be refused. */
uint64_t ovl_ssm_scan_workspace_bytes(const ovl_ssm_scan* scan, int32_t backward);
uint64_t ovl_ssm_scan_saved_bytes(const ovl_ssm_scan* scan);

/* y [batch, length, channels], last [batch, channels, state]; `saved` (or NULL) keeps the states for the backward
 * pass.  With y NULL only `saved` is written. */
int ovl_ssm_scan_forward(const ovl_ssm_scan* scan, void* y, float* last, float* saved, void* workspace,
                         uint64_t workspace_bytes, void* hip_stream);

/* Gradients: upstream d_y (a sequence; required) and d_last (or NULL); all others are written, dense: d_u, d_delta, d_z
 * like the sequences (d_z only with a gate), d_B and d_C [batch, length, groups, state], and in float32 d_A, d_D,
 * d_delta_bias, d_entering (the last three may be NULL). */
typedef struct ovl_ssm_scan_gradients {
    ovl_ssm_sequence d_y;
    const float* d_last;
    void  *d_u, *d_delta, *d_z, *d_B, *d_C;
    float *d_A, *d_D, *d_delta_bias, *d_entering;
} ovl_ssm_scan_gradients;

int ovl_ssm_scan_backward(const ovl_ssm_scan* scan, const float* saved, const ovl_ssm_scan_gradients* gradients,
                          void* workspace, uint64_t workspace_bytes, void* hip_stream);

/* One token per sequence: length 1, lengths NULL, `entering` is not used; `h` [batch, channels, state] (dense but for its
 * batch stride, in elements) is read and overwritten. */
int ovl_ssm_scan_step(const ovl_ssm_scan* scan, float* h, int64_t h_batch_stride, void* y, void* hip_stream);

typedef struct ovl_ssm_conv {
    uint32_t batch, length, channels, width;           /* width 1 .. 4 */
    int32_t  dtype;                                    /* of x, kept and the sequences written */
    int32_t  silu;
    ovl_ssm_sequence x;
    const void* weight;                                /* [channels, width] */
    const void* bias;                                  /* [channels] or NULL */
    ovl_ssm_sequence kept;                             /* [batch, width - 1, channels]: the tokens before; may be absent */
    const int32_t* lengths;                            /* [batch] or NULL */
    int32_t  own_weights;                              /* weight and bias are of type dtype; 0: float32 */
} ovl_ssm_conv;

/* y [batch, length, channels]; last [batch, width - 1, channels]: the tokens a later call needs in `kept`. */
int ovl_ssm_conv_forward(const ovl_ssm_conv* conv, void* y, void* last, void* hip_stream);

/* Gradients for upstream d_y (required) and d_last (may be absent): d_x like x, d_kept like last (or NULL), and in
 * float32 d_weight and d_bias (or NULL). */
uint64_t ovl_ssm_conv_workspace_bytes(const ovl_ssm_conv* conv);
int ovl_ssm_conv_backward(const ovl_ssm_conv* conv, const ovl_ssm_sequence* d_y, const ovl_ssm_sequence* d_last,
                          void* d_x, void* d_kept, float* d_weight, float* d_bias, void* workspace,
                          uint64_t workspace_bytes, void* hip_stream);

/* One token per sequence (length 1, lengths NULL): `kept` is read and overwritten with the tokens the next call needs. */
int ovl_ssm_conv_step(const ovl_ssm_conv* conv, void* y, void* hip_stream);

/* Text of the last error on the calling thread ("" if none). */
const char* ovl_ssm_last_error(void);

#ifdef __cplusplus
}
#endif

#endif  /* OVL_SSM_H_ */
