// C ABI of the channel-mixing kernels: argument validation, then the asynchronous launchers of norm.hip,
// gated.hip and weight8.hip. Declarations: include/morphocore_amd_mixer.h.
#include "../../include/morphocore_amd_mixer.h"

#include "../../include/morphocore_amd.h"
#include "launch.hpp"
#include "mixer.hpp"

namespace
{

// Column offsets and the padding to whole blocks are 32-bit in the kernels.
constexpr int64_t MAX_COLS = 0x7fffff00;

int check_types(int dtype, int weight_dtype)
{
    if (dtype < MCA_FLOAT32 || dtype > MCA_BFLOAT16) return mca::api_fail("Unknown dtype: expected 0 (float32), 1 (float16) or 2 (bfloat16)");
    if (weight_dtype != dtype && weight_dtype != MCA_FLOAT32) return mca::api_fail("weight_dtype must be the activations' dtype or float32");
    return MCA_OK;
}

int check_rows(int64_t rows, int64_t cols)
{
    if (rows < 0 || cols < 0 || cols > MAX_COLS) return mca::api_fail("rows and cols must be non negative, cols below 2^31 - 256");
    // Every kernel addresses rows * cols elements (and 4 bytes each) with 64-bit offsets.
    if (rows > 0 && cols > INT64_MAX / 64 / rows) return mca::api_fail("rows * cols is too large");
    return MCA_OK;
}

int check_stride(std::initializer_list<int64_t> strides)
{
    for (const int64_t s : strides)
        if (s < 0) return mca::api_fail("row strides must be non negative");
    return MCA_OK;
}

int check_workspace(const void* workspace, size_t given, size_t need)
{
    if (need > 0 && (!workspace || given < need)) return mca::api_fail("Workspace too small: call the workspace_size function");
    return MCA_OK;
}

// f(activation type, weight type) as null pointers.
template <typename F>
int by_type(int dtype, int weight_dtype, F&& f)
{
    hipError_t err;
    if (dtype == MCA_FLOAT32)
        err = f((float*)nullptr, (float*)nullptr);
    else if (dtype == MCA_FLOAT16)
        err = weight_dtype == MCA_FLOAT32 ? f((_Float16*)nullptr, (float*)nullptr) : f((_Float16*)nullptr, (_Float16*)nullptr);
    else
        err = weight_dtype == MCA_FLOAT32 ? f((__bf16*)nullptr, (float*)nullptr) : f((__bf16*)nullptr, (__bf16*)nullptr);
    return mca::api_hip_status(err);
}

}  // namespace

extern "C" {

int mca_pack8(int dtype, const void* x, int64_t x_stride, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, void* stream)
{
    int rc;
    if ((rc = check_types(dtype, dtype)) || (rc = check_rows(rows, cols)) || (rc = check_stride({x_stride}))) return rc;
    if (rows * cols > 0 && (!x || !codes || !scales)) return mca::api_fail("x, codes and scales must not be null");
    return by_type(dtype, dtype, [&](auto* t, auto*) {
        using T = std::remove_pointer_t<decltype(t)>;
        return mca::pack8<T>((const T*)x, x_stride, codes, scales, rows, (int)cols, (hipStream_t)stream);
    });
}

int mca_unpack8(int dtype, const uint8_t* codes, const uint8_t* scales, void* out, int64_t rows, int64_t cols, void* stream)
{
    int rc;
    if ((rc = check_types(dtype, dtype)) || (rc = check_rows(rows, cols))) return rc;
    if (rows * cols > 0 && (!out || !codes || !scales)) return mca::api_fail("codes, scales and out must not be null");
    return by_type(dtype, dtype, [&](auto* t, auto*) {
        using T = std::remove_pointer_t<decltype(t)>;
        return mca::unpack8<T>(codes, scales, (T*)out, rows, (int)cols, (hipStream_t)stream);
    });
}

int mca_rms_norm_forward(int dtype, int weight_dtype, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                         const void* weight, float eps, void* y, void* h, uint8_t* codes, uint8_t* scales, float* rstd, int64_t rows,
                         int64_t cols, void* stream)
{
    int rc;
    if ((rc = check_types(dtype, weight_dtype)) || (rc = check_rows(rows, cols)) || (rc = check_stride({x_stride, residual_stride}))) return rc;
    if (!(eps >= 0.0f)) return mca::api_fail("eps must be non negative");
    if (rows * cols > 0 && (!x || !weight)) return mca::api_fail("x and weight must not be null");
    if ((codes == nullptr) != (scales == nullptr)) return mca::api_fail("codes and scales go together");
    return by_type(dtype, weight_dtype, [&](auto* t, auto* wt) {
        using T = std::remove_pointer_t<decltype(t)>;
        using WT = std::remove_pointer_t<decltype(wt)>;
        return mca::rms_norm_forward<T, WT>((const T*)x, x_stride, (const T*)residual, residual_stride, (const WT*)weight, eps, (T*)y, (T*)h,
                                            codes, scales, rstd, rows, (int)cols, (hipStream_t)stream);
    });
}

size_t mca_rms_norm_backward_workspace_size(int64_t rows, int64_t cols)
{
    if (check_rows(rows, cols) != MCA_OK) return 0;
    return mca::rms_norm_backward_workspace(rows, (int)cols);
}

int mca_rms_norm_backward(int dtype, int weight_dtype, const void* grad_y, int64_t grad_y_stride, const void* grad_h, int64_t grad_h_stride,
                          const void* h, int64_t h_stride, const void* weight, const float* rstd, void* grad_x, void* grad_weight,
                          int64_t rows, int64_t cols, void* workspace, size_t workspace_bytes, void* stream)
{
    int rc;
    if ((rc = check_types(dtype, weight_dtype)) || (rc = check_rows(rows, cols)) ||
        (rc = check_stride({grad_y_stride, grad_h_stride, h_stride})))
        return rc;
    if (rows * cols > 0 && (!h || !weight || !rstd)) return mca::api_fail("h, weight and rstd must not be null");
    if (grad_weight && (rc = check_workspace(workspace, workspace_bytes, mca::rms_norm_backward_workspace(rows, (int)cols)))) return rc;
    return by_type(dtype, weight_dtype, [&](auto* t, auto* wt) {
        using T = std::remove_pointer_t<decltype(t)>;
        using WT = std::remove_pointer_t<decltype(wt)>;
        return mca::rms_norm_backward<T, WT>((const T*)grad_y, grad_y_stride, (const T*)grad_h, grad_h_stride, (const T*)h, h_stride,
                                             (const WT*)weight, rstd, (T*)grad_x, (WT*)grad_weight, rows, (int)cols, workspace,
                                             (hipStream_t)stream);
    });
}

int mca_gated_silu_forward(int dtype, const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, void* y, uint8_t* gate_codes,
                           uint8_t* gate_scales, uint8_t* up_codes, uint8_t* up_scales, uint8_t* y_codes, uint8_t* y_scales, int64_t rows,
                           int64_t cols, void* stream)
{
    int rc;
    if ((rc = check_types(dtype, dtype)) || (rc = check_rows(rows, cols)) || (rc = check_stride({gate_stride, up_stride}))) return rc;
    if (rows * cols > 0 && (!gate || !up || !y)) return mca::api_fail("gate, up and y must not be null");
    if ((gate_codes == nullptr) != (gate_scales == nullptr) || (up_codes == nullptr) != (up_scales == nullptr) ||
        (y_codes == nullptr) != (y_scales == nullptr))
        return mca::api_fail("codes and scales go together");
    return by_type(dtype, dtype, [&](auto* t, auto*) {
        using T = std::remove_pointer_t<decltype(t)>;
        return mca::gated_silu_forward<T>((const T*)gate, gate_stride, (const T*)up, up_stride, (T*)y, {gate_codes, gate_scales},
                                          {up_codes, up_scales}, {y_codes, y_scales}, rows, (int)cols, (hipStream_t)stream);
    });
}

int mca_gated_silu_backward(int dtype, const void* grad_y, int64_t grad_y_stride, const void* gate, int64_t gate_stride, const void* up,
                            int64_t up_stride, const uint8_t* gate_codes, const uint8_t* gate_scales, const uint8_t* up_codes,
                            const uint8_t* up_scales, void* grad_gate, void* grad_up, int64_t grad_stride, int64_t rows, int64_t cols,
                            void* stream)
{
    int rc;
    if ((rc = check_types(dtype, dtype)) || (rc = check_rows(rows, cols)) || (rc = check_stride({grad_y_stride, gate_stride, up_stride})))
        return rc;
    if (grad_stride < cols) return mca::api_fail("grad_stride must be at least cols");
    if (rows * cols > 0)
    {
        if ((gate == nullptr) != (up == nullptr)) return mca::api_fail("gate and up go together");
        if (!grad_y || !grad_gate || !grad_up) return mca::api_fail("grad_y, grad_gate and grad_up must not be null");
        if (!gate && (!gate_codes || !gate_scales || !up_codes || !up_scales)) return mca::api_fail("gate and up, or their packed form, must be given");
    }
    return by_type(dtype, dtype, [&](auto* t, auto*) {
        using T = std::remove_pointer_t<decltype(t)>;
        return mca::gated_silu_backward<T>((const T*)grad_y, grad_y_stride, (const T*)gate, gate_stride, (const T*)up, up_stride,
                                           {(uint8_t*)gate_codes, (uint8_t*)gate_scales}, {(uint8_t*)up_codes, (uint8_t*)up_scales},
                                           (T*)grad_gate, (T*)grad_up, grad_stride, rows, (int)cols, (hipStream_t)stream);
    });
}

size_t mca_grad_weight8_workspace_size(int dtype, int64_t rows, int64_t out, int64_t cols)
{
    if (check_types(dtype, dtype) || check_rows(rows, cols) || check_rows(rows, out) || check_rows(out, cols)) return 0;
    if (dtype == MCA_FLOAT32) return mca::grad_weight8_workspace<float>(rows, (int)out, (int)cols);
    if (dtype == MCA_FLOAT16) return mca::grad_weight8_workspace<_Float16>(rows, (int)out, (int)cols);
    return mca::grad_weight8_workspace<__bf16>(rows, (int)out, (int)cols);
}

int mca_grad_weight8(int dtype, int weight_dtype, const void* grad_y, int64_t grad_y_stride, const uint8_t* codes, const uint8_t* scales,
                     void* grad_weight, int64_t rows, int64_t out, int64_t cols, void* workspace, size_t workspace_bytes, void* stream)
{
    int rc;
    if ((rc = check_types(dtype, weight_dtype)) || (rc = check_rows(rows, cols)) || (rc = check_rows(rows, out)) ||
        (rc = check_rows(out, cols)) || (rc = check_stride({grad_y_stride})))
        return rc;
    if (out * cols > 0 && (!grad_weight || (rows > 0 && (!grad_y || !codes || !scales))))
        return mca::api_fail("grad_y, codes, scales and grad_weight must not be null");
    if ((rc = check_workspace(workspace, workspace_bytes, mca_grad_weight8_workspace_size(dtype, rows, out, cols)))) return rc;
    return by_type(dtype, weight_dtype, [&](auto* t, auto* wt) {
        using T = std::remove_pointer_t<decltype(t)>;
        using WT = std::remove_pointer_t<decltype(wt)>;
        return mca::grad_weight8<T, WT>((const T*)grad_y, grad_y_stride, codes, scales, (WT*)grad_weight, rows, (int)out, (int)cols, workspace,
                                        (hipStream_t)stream);
    });
}

}  // extern "C"
