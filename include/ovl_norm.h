/*
 * C ABI of the hand-written root-mean-square norm kernels for AMD GPUs (libovl_norm.so): the norm of the rows of a
 * matrix, with the residual's addition in front of it and with an output in 8 bits with scales, and its gradient.  The
 * reference has no counterpart.
 *
 *   s[r,c] = x[r,c] + residual[r,c]   rounded to the residual's type, which is how it is stored; x[r,c] without a residual
 *   y[r,c] = s[r,c] * rstd[r] * weight[c]               rstd[r] = 1 / sqrt(mean over c of s[r,c]^2 + eps)
 *   q[r,c] = e4m3(y[r,c] / scale)                       scale = max |y| / 448 over the row, or over each 128 columns of it
 *                                                       (at least 2^-126, and 1 where all of them are zero; NaN does not
 *                                                       count), both of y in float32 before it is rounded to dtype
 *
 * The norm is that of the sum as stored, so that the layer that reads the sum later, and the backward pass, see the very
 * values that were normalised.  Sums and statistics are float32; y, q and s are rounded once.
 *
 * Conventions: tensor memory belongs to the caller and must be device accessible; the columns of a row lie side by side,
 * the row strides of the inputs (in elements) are free, outputs are dense.  The functions enqueue kernels on `hip_stream`,
 * return without synchronising, allocate nothing and give the same bits for the same call.  They return an ovl_status
 * (ovl_launch.h): OVL_EINVAL for arguments they refuse, OVL_EHIP for a HIP error (text from ovl_norm_last_error).
 */
#ifndef OVL_NORM_H_
#define OVL_NORM_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types: the codes of ovl_launch.h, and bfloat16, which the operator IR does not have. */
enum ovl_norm_dtype { OVL_NORM_FLOAT16 = 1, OVL_NORM_FLOAT32 = 2, OVL_NORM_BFLOAT16 = 32 };

typedef struct ovl_norm {
    uint32_t rows, columns;             /* columns 1 .. 32768 */
    int32_t  dtype;                     /* of x, y and their gradients */
    int32_t  residual_dtype;            /* of residual, s and their gradients: dtype or OVL_NORM_FLOAT32 */
    int32_t  weight_dtype;              /* dtype or OVL_NORM_FLOAT32 */
    float    eps;
    const void* x;        int64_t x_stride;
    const void* residual; int64_t residual_stride;      /* residual may be NULL */
    const void* weight;                                 /* [columns] */
} ovl_norm;

/* y [rows, columns]; summed [rows, columns] (with a residual). */
int ovl_norm_forward(const ovl_norm* norm, void* y, void* summed, void* hip_stream);

/* q [rows, columns] bytes; scales [rows, groups], groups = 1 (group_columns 0) or ceil(columns / 128) (group_columns
 * 128); summed [rows, columns] (with a residual). */
int ovl_norm_forward_quantized(const ovl_norm* norm, uint32_t group_columns, void* q, float* scales, void* summed,
                               void* hip_stream);

/* Gradients.  norm->x is what was normalised (x, or the stored sum), of type residual_dtype; norm->residual is not used.
 * d_y is of type dtype, d_summed of type residual_dtype or NULL.  Written are d_x (dtype; or NULL) and d_residual
 * (residual_dtype; or NULL), which hold the same values, and d_weight (weight_dtype). */
uint64_t ovl_norm_workspace_bytes(const ovl_norm* norm);
int ovl_norm_backward(const ovl_norm* norm, const void* d_y, int64_t d_y_stride, const void* d_summed,
                      int64_t d_summed_stride, void* d_x, void* d_residual, void* d_weight, void* workspace,
                      uint64_t workspace_bytes, void* hip_stream);

/* Text of the last error on the calling thread ("" if none). */
const char* ovl_norm_last_error(void);

#ifdef __cplusplus
}
#endif

#endif  /* OVL_NORM_H_ */
