// Host-side launchers of the channel-mixing kernels (norm.hip, gated.hip, weight8.hip), called by their C
// ABI (mixer_api.cpp). Arguments are assumed validated by the caller; every launch is asynchronous on
// `stream`. Tensors are rows x cols, a row's values consecutive, rows `*_stride` elements apart (packed
// ones dense: codes rows x cols bytes, scales rows x ceil(cols / 32) bytes).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mca
{

template <typename T>
hipError_t pack8(const T* x, int64_t x_stride, uint8_t* codes, uint8_t* scales, int64_t rows, int cols, hipStream_t stream);
template <typename T>
hipError_t unpack8(const uint8_t* codes, const uint8_t* scales, T* out, int64_t rows, int cols, hipStream_t stream);

// out = x's rows, or zeros where x is null.
template <typename T>
hipError_t copy_rows(const T* x, int64_t x_stride, T* out, int64_t rows, int cols, hipStream_t stream);

// h = x (+ residual), y = h * rstd * w; residual, y, h, codes with scales, and rstd may be null.
template <typename T, typename WT>
hipError_t rms_norm_forward(const T* x, int64_t x_stride, const T* residual, int64_t r_stride, const WT* w, float eps, T* y, T* h,
                            uint8_t* codes, uint8_t* scales, float* rstd, int64_t rows, int cols, hipStream_t stream);
size_t rms_norm_backward_workspace(int64_t rows, int cols);
// grad_y, grad_h, grad_x or grad_w may be null. The workspace is for grad_w.
template <typename T, typename WT>
hipError_t rms_norm_backward(const T* grad_y, int64_t gy_stride, const T* grad_h, int64_t gh_stride, const T* h, int64_t h_stride, const WT* w,
                             const float* rstd, T* grad_x, WT* grad_w, int64_t rows, int cols, void* workspace, hipStream_t stream);

// y = g * sigmoid(g) * u; gate and up in 8 bits, and y in 8 bits, where their buffers are given.
struct PackedOut
{
    uint8_t *codes, *scales;
};
template <typename T>
hipError_t gated_silu_forward(const T* gate, int64_t g_stride, const T* up, int64_t u_stride, T* y, PackedOut gate8, PackedOut up8,
                              PackedOut y8, int64_t rows, int cols, hipStream_t stream);
// From gate and up as they were, or from their 8-bit form (gate null). grad_gate and grad_up: rows
// grad_stride apart.
template <typename T>
hipError_t gated_silu_backward(const T* grad_y, int64_t gy_stride, const T* gate, int64_t g_stride, const T* up, int64_t u_stride,
                               PackedOut gate8, PackedOut up8, T* grad_gate, T* grad_up, int64_t grad_stride, int64_t rows, int cols,
                               hipStream_t stream);

// grad_weight [out, cols] = sum over the rows of grad_y [rows, out] (outer) the packed values [rows, cols].
template <typename T>
size_t grad_weight8_workspace(int64_t rows, int out, int cols);
template <typename T, typename OT>
hipError_t grad_weight8(const T* grad_y, int64_t gy_stride, const uint8_t* codes, const uint8_t* scales, OT* grad_weight, int64_t rows,
                        int out, int cols, void* workspace, hipStream_t stream);

// out[j] = the sum of part[s * n + j] over the slots s, in a fixed order (in float64), rounded once.
template <typename OT>
hipError_t sum_slots_async(const float* part, int nslots, int64_t n, OT* out, hipStream_t stream);

}  // namespace mca
