// Host-side helpers shared by the operators of the PyTorch-ROCm extension that take rows of values
// (mixer_ops.cpp, tokens_ops.cpp): checks of arguments, and tensors as rows.
#pragma once

#include <torch/all.h>
#include <torch/library.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <vector>

#include "../../include/morphocore_amd.h"
#include "../../include/morphocore_amd_mixer.h"

namespace
{

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using OptTensor = std::optional<Tensor>;

void check_rc(int rc) { TORCH_CHECK(rc == MCA_OK, mca_last_error()); }

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int type_code(const char* name, const Tensor& t)
{
    switch (t.scalar_type())
    {
        case c10::kFloat: return MCA_FLOAT32;
        case c10::kHalf: return MCA_FLOAT16;
        case c10::kBFloat16: return MCA_BFLOAT16;
        default: TORCH_CHECK(false, "\"", name, "\" not implemented for '", c10::toString(t.scalar_type()), "'");
    }
    return -1;
}

void check_device(const char* name, const Tensor& x, std::initializer_list<Tensor> others)
{
    TORCH_CHECK(x.is_cuda(), "morphocore_amd: ", name, " runs on AMD GPUs (HIP devices); got an input on ", x.device());
    for (const Tensor& t : others)
        TORCH_CHECK(t.device() == x.device(), "morphocore_amd: ", name, " expects every tensor on ", x.device(), ", got one on ", t.device());
}

void check_type(const Tensor& x, const Tensor& t)
{
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), "expected scalar type ", c10::toString(x.scalar_type()), " but found ",
                c10::toString(t.scalar_type()));
}

void check_first_order(const char* name)
{
    TORCH_CHECK(!torch::GradMode::is_enabled(), name, ": the backward cannot record a graph of its own (create_graph=True)");
}

// Forward-mode derivatives, which the operators do not carry on, are refused, not lost.
void check_no_tangent(const char* name, std::initializer_list<Tensor> tensors)
{
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor& t : tensors)
        TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), name, ": forward-mode derivatives are not supported");
}

// A tensor as rows of its last dimension.
struct Rows
{
    Tensor t;  // keeps the memory
    int64_t rows, cols, stride;

    const void* data() const { return t.const_data_ptr(); }
};

int64_t leading(const Tensor& t)
{
    int64_t n = 1;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) n *= t.size(d);
    return n;
}

// Elements between the rows when one number says it, else -1.
int64_t row_stride(const Tensor& t)
{
    if (t.size(-1) > 1 && t.stride(-1) != 1) return -1;
    int64_t stride = -1, next = 0;
    for (int64_t d = t.dim() - 2; d >= 0; --d)
    {
        if (t.size(d) == 1) continue;
        if (stride < 0)
            stride = t.stride(d);
        else if (t.stride(d) != next)
            return -1;
        next = t.stride(d) * t.size(d);
    }
    return stride < 0 ? t.size(-1) : stride;
}

Rows rows_of(const Tensor& t)
{
    int64_t stride = t.numel() ? row_stride(t) : t.size(-1);
    const Tensor u = stride < 0 ? t.contiguous() : t;
    if (stride < 0) stride = t.size(-1);
    return Rows{u, leading(u), u.size(-1), stride};
}

void check_rank(const char* name, const Tensor& x)
{
    TORCH_CHECK(x.dim() >= 1, name, ": the input must have at least one dimension");
}

bool records(std::initializer_list<Tensor> tensors)
{
    if (!torch::GradMode::is_enabled()) return false;
    for (const Tensor& t : tensors)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

}  // namespace
