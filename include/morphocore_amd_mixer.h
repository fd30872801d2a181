/*
 * morphocore_amd — C ABI of the channel-mixing kernels (gfx950): 8-bit blocks, root-mean-square norm, gated
 * activation, and a linear layer's weight gradient from its packed input. No reference counterpart.
 *
 * Conventions are those of morphocore_amd.h (status codes, mca_last_error, streams, caller-owned
 * workspaces). Tensors are rows x cols device arrays whose rows' values are consecutive; `*_stride` is the
 * number of elements between rows (0 and overlapping rows are allowed for what is read), and arrays
 * without one are dense. Rows may start at any multiple of the element's size.
 *
 * dtype (of the activations) and weight_dtype: 0 float32, 1 float16, 2 bfloat16. weight_dtype is the
 * activations' or float32. Sums are float32 or wider.
 *
 * A packed array is `codes`, rows x cols bytes (e4m3), and `scales`, rows x ceil(cols / 32) bytes: block b of
 * a row is its values [32 b, 32 b + 32), and a value is e4m3(code) * 2^(scale - 127). The scale's exponent is
 * the smallest in [-117, 119] with max |v| <= 448 * 2^e over the block's finite values (beyond: saturation);
 * NaN and infinities become NaN.
 */
#ifndef MORPHOCORE_AMD_MIXER_H
#define MORPHOCORE_AMD_MIXER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MCA_FLOAT32 0
#define MCA_FLOAT16 1
#define MCA_BFLOAT16 2

/* x to 8-bit blocks, and back (to nearest even; float16 saturates at its largest value). */
int mca_pack8(int dtype, const void* x, int64_t x_stride, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, void* stream);
int mca_unpack8(int dtype, const uint8_t* codes, const uint8_t* scales, void* out, int64_t rows, int64_t cols, void* stream);

/* h = x + residual (x without one), y = h / sqrt(mean(h^2) + eps) * weight. residual, y, h, the packed y
 * (codes and scales together) and rstd [rows] (1 / sqrt(...), for the backward) may be NULL. The packed y is
 * y as rounded to dtype. */
int mca_rms_norm_forward(int dtype, int weight_dtype, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                         const void* weight, float eps, void* y, void* h, uint8_t* codes, uint8_t* scales, float* rstd, int64_t rows,
                         int64_t cols, void* stream);

/* grad_x (also the residual's gradient) and grad_weight from grad_y, grad_h (the gradient of h as an output),
 * h and rstd. grad_y, grad_h, grad_x and grad_weight may be NULL; without grad_y, grad_x is grad_h (or zeros) whatever h
 * holds, and grad_weight zeros. */
size_t mca_rms_norm_backward_workspace_size(int64_t rows, int64_t cols);
int mca_rms_norm_backward(int dtype, int weight_dtype, const void* grad_y, int64_t grad_y_stride, const void* grad_h, int64_t grad_h_stride,
                          const void* h, int64_t h_stride, const void* weight, const float* rstd, void* grad_x, void* grad_weight,
                          int64_t rows, int64_t cols, void* workspace, size_t workspace_bytes, void* stream);

/* y = gate * sigmoid(gate) * up. Each packed output (codes with scales) may be NULL: gate's and up's, for the
 * backward, and y's (as rounded to dtype). */
int mca_gated_silu_forward(int dtype, const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, void* y, uint8_t* gate_codes,
                           uint8_t* gate_scales, uint8_t* up_codes, uint8_t* up_scales, uint8_t* y_codes, uint8_t* y_scales, int64_t rows,
                           int64_t cols, void* stream);

/* grad_gate and grad_up (rows grad_stride apart) from grad_y and either gate and up or, where both are NULL,
 * their packed form. */
int mca_gated_silu_backward(int dtype, const void* grad_y, int64_t grad_y_stride, const void* gate, int64_t gate_stride, const void* up,
                            int64_t up_stride, const uint8_t* gate_codes, const uint8_t* gate_scales, const uint8_t* up_codes,
                            const uint8_t* up_scales, void* grad_gate, void* grad_up, int64_t grad_stride, int64_t rows, int64_t cols,
                            void* stream);

/* grad_weight [out, cols] = sum over the rows m of grad_y [rows, out]^T times the packed values [rows, cols];
 * weight_dtype is grad_weight's. */
size_t mca_grad_weight8_workspace_size(int dtype, int64_t rows, int64_t out, int64_t cols);
int mca_grad_weight8(int dtype, int weight_dtype, const void* grad_y, int64_t grad_y_stride, const uint8_t* codes, const uint8_t* scales,
                     void* grad_weight, int64_t rows, int64_t out, int64_t cols, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif
