// The channel-mixing operators of the PyTorch-ROCm extension: pack8, unpack8, rms_norm, rms_norm8,
// gated_silu, gated_silu8, linear8 and grad_weight8, in the namespace that torch_ops.cpp registers. No
// reference counterpart. Device work is the C ABI of include/morphocore_amd_mixer.h.
//
// An operator whose name ends in 8 keeps 8-bit blocks for its backward, or reads or writes them. Tensors of
// any rank are taken as rows of their last dimension; rows at one distance from each other (a slice of wider
// rows, an expanded row) are read where they are, others are copied. Only HIP devices; everything else is an
// error, never a fallback.
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

constexpr int64_t PACK_BLOCK = 32;

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

struct Packed
{
    Tensor codes, scales;

    uint8_t* c() const { return codes.defined() ? (uint8_t*)codes.data_ptr() : nullptr; }
    uint8_t* s() const { return scales.defined() ? (uint8_t*)scales.data_ptr() : nullptr; }
};

Packed new_packed(at::IntArrayRef shape, const Tensor& like)
{
    std::vector<int64_t> blocks = shape.vec();
    blocks.back() = (blocks.back() + PACK_BLOCK - 1) / PACK_BLOCK;
    return Packed{torch::empty(shape, like.options().dtype(c10::kFloat8_e4m3fn)), torch::empty(blocks, like.options().dtype(c10::kFloat8_e8m0fnu))};
}

// The checks of a packed argument, and its dense form.
Packed packed_arg(const char* name, const Tensor& codes, const Tensor& scales)
{
    TORCH_CHECK(codes.scalar_type() == c10::kFloat8_e4m3fn, name, ": codes must be float8_e4m3fn, got ", c10::toString(codes.scalar_type()));
    TORCH_CHECK(scales.scalar_type() == c10::kFloat8_e8m0fnu, name, ": scales must be float8_e8m0fnu, got ", c10::toString(scales.scalar_type()));
    TORCH_CHECK(codes.dim() >= 1, name, ": codes must have at least one dimension");
    std::vector<int64_t> blocks = codes.sizes().vec();
    blocks.back() = (blocks.back() + PACK_BLOCK - 1) / PACK_BLOCK;
    TORCH_CHECK(scales.sizes() == at::IntArrayRef(blocks), name, ": codes of shape ", codes.sizes(), " need scales of shape ",
                at::IntArrayRef(blocks), ", got ", scales.sizes());
    check_device(name, codes, {scales});
    return Packed{codes.contiguous(), scales.contiguous()};
}

void check_rank(const char* name, const Tensor& x)
{
    TORCH_CHECK(x.dim() >= 1, name, ": the input must have at least one dimension");
}

Packed pack_rows(const Tensor& x)
{
    const c10::DeviceGuard guard(x.device());
    const Rows r = rows_of(x);
    const Packed p = new_packed(x.sizes(), x);
    check_rc(mca_pack8(type_code("pack8", x), r.data(), r.stride, p.c(), p.s(), r.rows, r.cols, stream_of(x)));
    return p;
}

std::tuple<Tensor, Tensor> pack8(const Tensor& input)
{
    check_rank("pack8", input);
    check_device("pack8", input, {});
    const Packed p = pack_rows(input.detach());
    return {p.codes, p.scales};
}

Tensor unpack8(const Tensor& codes, const Tensor& scales, at::ScalarType dtype)
{
    const Packed p = packed_arg("unpack8", codes, scales);
    check_device("unpack8", codes, {});
    const c10::DeviceGuard guard(codes.device());
    Tensor out = torch::empty(codes.sizes(), codes.options().dtype(dtype));
    check_rc(mca_unpack8(type_code("unpack8", out), p.c(), p.s(), out.data_ptr(), leading(codes), codes.size(-1), stream_of(codes)));
    return out;
}

// ------------------------------------------------------------------------------------------------
// Root-mean-square norm.
// ------------------------------------------------------------------------------------------------

struct Normed
{
    Tensor y, h, rstd;
    Packed packed;
};

Normed norm_forward(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, bool full, bool pack, bool keep)
{
    const c10::DeviceGuard guard(x.device());
    const Rows xr = rows_of(x);
    const Rows rr = residual.defined() ? rows_of(residual) : Rows{};
    const Tensor w = weight.contiguous();
    Normed n;
    if (full) n.y = torch::empty(x.sizes(), x.options());
    if (residual.defined()) n.h = torch::empty(x.sizes(), x.options());
    if (keep) n.rstd = torch::empty({xr.rows}, x.options().dtype(c10::kFloat));
    if (pack) n.packed = new_packed(x.sizes(), x);
    check_rc(mca_rms_norm_forward(type_code("rms_norm", x), type_code("rms_norm", w), xr.data(), xr.stride,
                                  residual.defined() ? rr.data() : nullptr, residual.defined() ? rr.stride : 0, w.const_data_ptr(), (float)eps,
                                  full ? n.y.data_ptr() : nullptr, n.h.defined() ? n.h.data_ptr() : nullptr, n.packed.c(), n.packed.s(),
                                  keep ? n.rstd.data_ptr<float>() : nullptr, xr.rows, xr.cols, stream_of(x)));
    return n;
}

class RmsNormFunction : public torch::autograd::Function<RmsNormFunction>
{
public:
    static tensor_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps, bool pack)
    {
        const Normed n = norm_forward(x, weight, residual.value_or(Tensor()), eps, true, pack, true);
        tensor_list out = {n.y};
        if (n.h.defined()) out.push_back(n.h);
        if (pack)
        {
            out.push_back(n.packed.codes);
            out.push_back(n.packed.scales);
            ctx->mark_non_differentiable({n.packed.codes, n.packed.scales});
        }
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({n.h.defined() ? n.h : x, weight, n.rstd});
        ctx->saved_data["residual"] = n.h.defined();
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads)
    {
        const bool residual = ctx->saved_data["residual"].toBool();
        const Tensor gy = grads[0], gh = residual ? grads[1] : Tensor();
        if (!gy.defined() && !gh.defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        check_first_order("rms_norm");
        const auto saved = ctx->get_saved_variables();
        const Tensor& h = saved[0];
        const Tensor w = saved[1].contiguous();
        const Tensor& rstd = saved[2];
        const c10::DeviceGuard guard(h.device());
        const bool need_x = ctx->needs_input_grad(0) || (residual && ctx->needs_input_grad(2)), need_w = ctx->needs_input_grad(1);
        const Rows hr = rows_of(h);
        const Rows gyr = gy.defined() ? rows_of(gy) : Rows{}, ghr = gh.defined() ? rows_of(gh) : Rows{};
        Tensor gx = need_x ? torch::empty(h.sizes(), h.options()) : Tensor(), gw = need_w ? torch::empty(w.sizes(), w.options()) : Tensor();
        const size_t bytes = need_w ? mca_rms_norm_backward_workspace_size(hr.rows, hr.cols) : 0;
        const Tensor ws = torch::empty({(int64_t)bytes}, h.options().dtype(torch::kUInt8));
        check_rc(mca_rms_norm_backward(type_code("rms_norm", h), type_code("rms_norm", w), gy.defined() ? gyr.data() : nullptr,
                                       gy.defined() ? gyr.stride : 0, gh.defined() ? ghr.data() : nullptr, gh.defined() ? ghr.stride : 0, hr.data(),
                                       hr.stride, w.const_data_ptr(), rstd.const_data_ptr<float>(), need_x ? gx.data_ptr() : nullptr,
                                       need_w ? gw.data_ptr() : nullptr, hr.rows, hr.cols, ws.data_ptr(), bytes, stream_of(h)));
        return {ctx->needs_input_grad(0) ? gx : Tensor(), gw, residual && ctx->needs_input_grad(2) ? gx : Tensor(), Tensor(), Tensor()};
    }
};

bool records(std::initializer_list<Tensor> tensors)
{
    if (!torch::GradMode::is_enabled()) return false;
    for (const Tensor& t : tensors)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

void check_norm(const char* name, const Tensor& x, const Tensor& weight, const Tensor& residual, double eps)
{
    check_rank(name, x);
    check_no_tangent(name, {x, weight, residual});
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(-1), name, ": weight must be [", x.size(-1), "], got ", weight.sizes());
    TORCH_CHECK(eps >= 0.0, name, ": eps must be non negative");
    check_device(name, x, {weight});
    type_code(name, x);
    if (weight.scalar_type() != c10::kFloat) check_type(x, weight);
    if (residual.defined())
    {
        TORCH_CHECK(residual.sizes() == x.sizes(), name, ": residual must have the input's shape ", x.sizes(), ", got ", residual.sizes());
        check_device(name, x, {residual});
        check_type(x, residual);
    }
}

// (y, h); h is undefined without a residual.
std::tuple<Tensor, Tensor> rms_norm(const Tensor& input, const Tensor& weight, const OptTensor& residual, double eps)
{
    const Tensor r = residual.value_or(Tensor());
    check_norm("rms_norm", input, weight, r, eps);
    if (!records({input, weight, r}))
    {
        const Normed n = norm_forward(input, weight, r, eps, true, false, false);
        return {n.y, n.h};
    }
    const tensor_list out = RmsNormFunction::apply(input, weight, residual, eps, false);
    return {out[0], r.defined() ? out[1] : Tensor()};
}

// (y, h, codes, scales) with the packed y; y is undefined where full is false.
std::tuple<Tensor, Tensor, Tensor, Tensor> rms_norm8(const Tensor& input, const Tensor& weight, const OptTensor& residual, double eps, bool full)
{
    const Tensor r = residual.value_or(Tensor());
    check_norm("rms_norm8", input, weight, r, eps);
    if (!records({input, weight, r}))
    {
        const Normed n = norm_forward(input, weight, r, eps, full, true, false);
        return {n.y, n.h, n.packed.codes, n.packed.scales};
    }
    TORCH_CHECK(full, "rms_norm8: the 8-bit output alone (full=False) has no gradient; call it under torch.no_grad()");
    const tensor_list out = RmsNormFunction::apply(input, weight, residual, eps, true);
    const size_t at = r.defined() ? 2 : 1;
    return {out[0], r.defined() ? out[1] : Tensor(), out[at], out[at + 1]};
}

// ------------------------------------------------------------------------------------------------
// Gated activation.
// ------------------------------------------------------------------------------------------------

// gate and up as rows: two tensors, or the halves of one.
struct Gated
{
    Rows gate;
    Tensor up_t;
    const void* up;
    int64_t up_stride, cols;
    std::vector<int64_t> shape;  // of y
};

Gated gated_rows(const Tensor& gate, const Tensor& up)
{
    Gated g;
    g.gate = rows_of(gate);
    g.shape = gate.sizes().vec();
    if (up.defined())
    {
        const Rows u = rows_of(up);
        g.cols = g.gate.cols;
        g.up_t = u.t;
        g.up = u.data();
        g.up_stride = u.stride;
    }
    else
    {
        g.cols = g.gate.cols / 2;
        g.shape.back() = g.cols;
        const void* first = g.gate.data();  // null of an empty tensor
        g.up = first ? (const char*)first + g.cols * gate.element_size() : nullptr;
        g.up_stride = g.gate.stride;
    }
    return g;
}

// gate's and up's 8-bit form in one buffer, which the backward alone reads: gate's codes, up's, gate's scales, up's.
struct Kept
{
    Tensor buffer;
    int64_t values, blocks;

    uint8_t* at(int64_t offset) const { return buffer.defined() ? (uint8_t*)buffer.data_ptr() + offset : nullptr; }
    uint8_t* gate_codes() const { return at(0); }
    uint8_t* up_codes() const { return at(values); }
    uint8_t* gate_scales() const { return at(2 * values); }
    uint8_t* up_scales() const { return at(2 * values + blocks); }
};

Kept kept_of(int64_t rows, int64_t cols)
{
    return Kept{Tensor(), rows * cols, rows * ((cols + PACK_BLOCK - 1) / PACK_BLOCK)};
}

struct GatedOut
{
    Tensor y;
    Kept kept;
    Packed packed;
};

GatedOut gated_forward(const Tensor& gate, const Tensor& up, bool keep8, bool pack)
{
    const c10::DeviceGuard guard(gate.device());
    const Gated g = gated_rows(gate, up);
    GatedOut o;
    o.y = torch::empty(g.shape, gate.options());
    o.kept = kept_of(g.gate.rows, g.cols);
    if (keep8) o.kept.buffer = torch::empty({2 * (o.kept.values + o.kept.blocks)}, gate.options().dtype(torch::kUInt8));
    if (pack) o.packed = new_packed(g.shape, gate);
    check_rc(mca_gated_silu_forward(type_code("gated_silu", gate), g.gate.data(), g.gate.stride, g.up, g.up_stride, o.y.data_ptr(),
                                    o.kept.gate_codes(), o.kept.gate_scales(), o.kept.up_codes(), o.kept.up_scales(), o.packed.c(), o.packed.s(),
                                    g.gate.rows, g.cols, stream_of(gate)));
    return o;
}

class GatedSiluFunction : public torch::autograd::Function<GatedSiluFunction>
{
public:
    // eight: keep gate and up in 8 bits, and return the packed y too.
    static tensor_list forward(AutogradContext* ctx, const Tensor& gate, const OptTensor& up, bool eight)
    {
        const Tensor u = up.value_or(Tensor());
        const GatedOut o = gated_forward(gate, u, eight, eight);
        ctx->set_materialize_grads(false);
        ctx->saved_data["eight"] = eight;
        ctx->saved_data["joint"] = !u.defined();
        if (!eight)
        {
            ctx->save_for_backward({gate, u});
            return {o.y};
        }
        ctx->save_for_backward({o.kept.buffer});
        ctx->mark_non_differentiable({o.packed.codes, o.packed.scales});
        return {o.y, o.packed.codes, o.packed.scales};
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads)
    {
        const Tensor gy = grads[0];
        if (!gy.defined()) return {Tensor(), Tensor(), Tensor()};
        check_first_order("gated_silu");
        const bool eight = ctx->saved_data["eight"].toBool(), joint = ctx->saved_data["joint"].toBool();
        const auto saved = ctx->get_saved_variables();
        const c10::DeviceGuard guard(gy.device());
        const Rows g = rows_of(gy);
        std::vector<int64_t> shape = gy.sizes().vec();
        const int64_t cols = shape.back();
        if (joint) shape.back() *= 2;
        Tensor gg = torch::empty(shape, gy.options()), gu = joint ? Tensor() : torch::empty(shape, gy.options());
        char* first = (char*)gg.data_ptr();  // null of an empty tensor
        void* gu_data = !joint ? gu.data_ptr() : first ? (void*)(first + cols * gy.element_size()) : nullptr;
        Gated in{};
        Kept kept = kept_of(g.rows, cols);
        if (eight)
            kept.buffer = saved[0];
        else
            in = gated_rows(saved[0], saved[1]);
        check_rc(mca_gated_silu_backward(type_code("gated_silu", gy), g.data(), g.stride, eight ? nullptr : in.gate.data(),
                                         eight ? 0 : in.gate.stride, eight ? nullptr : in.up, eight ? 0 : in.up_stride, kept.gate_codes(),
                                         kept.gate_scales(), kept.up_codes(), kept.up_scales(), gg.data_ptr(), gu_data, shape.back(), g.rows, cols, stream_of(gy)));
        return {ctx->needs_input_grad(0) ? gg : Tensor(), !joint && ctx->needs_input_grad(1) ? gu : Tensor(), Tensor()};
    }
};

void check_gated(const char* name, const Tensor& gate, const Tensor& up)
{
    check_rank(name, gate);
    check_no_tangent(name, {gate, up});
    check_device(name, gate, {});
    type_code(name, gate);
    if (!up.defined())
    {
        TORCH_CHECK(gate.size(-1) % 2 == 0, name, ": without `up` the last dimension holds gate and up, got ", gate.size(-1), " values");
        return;
    }
    TORCH_CHECK(up.sizes() == gate.sizes(), name, ": up must have gate's shape ", gate.sizes(), ", got ", up.sizes());
    check_device(name, gate, {up});
    check_type(gate, up);
}

Tensor gated_silu(const Tensor& gate, const OptTensor& up)
{
    const Tensor u = up.value_or(Tensor());
    check_gated("gated_silu", gate, u);
    if (!records({gate, u})) return gated_forward(gate, u, false, false).y;
    return GatedSiluFunction::apply(gate, up, false)[0];
}

// (y, codes, scales) with the packed y.
std::tuple<Tensor, Tensor, Tensor> gated_silu8(const Tensor& gate, const OptTensor& up)
{
    const Tensor u = up.value_or(Tensor());
    check_gated("gated_silu8", gate, u);
    if (!records({gate, u}))
    {
        const GatedOut o = gated_forward(gate, u, false, true);
        return {o.y, o.packed.codes, o.packed.scales};
    }
    const tensor_list out = GatedSiluFunction::apply(gate, up, true);
    return {out[0], out[1], out[2]};
}

// ------------------------------------------------------------------------------------------------
// Linear layer with its input kept in 8 bits.
// ------------------------------------------------------------------------------------------------

// grad [.., N] and codes [.., K], their leading dimensions alike.
Tensor weight_gradient(const Tensor& grad, const Packed& p, at::ScalarType dtype)
{
    const c10::DeviceGuard guard(grad.device());
    const Rows g = rows_of(grad);
    const int64_t cols = p.codes.size(-1);
    Tensor gw = torch::empty({g.cols, cols}, grad.options().dtype(dtype));
    const int type = type_code("grad_weight8", grad), weight_type = type_code("grad_weight8", gw);
    const size_t bytes = mca_grad_weight8_workspace_size(type, g.rows, g.cols, cols);
    const Tensor ws = torch::empty({(int64_t)bytes}, grad.options().dtype(torch::kUInt8));
    check_rc(mca_grad_weight8(type, weight_type, g.data(), g.stride, p.c(), p.s(), gw.data_ptr(), g.rows, g.cols, cols, ws.data_ptr(), bytes,
                              stream_of(grad)));
    return gw;
}

Tensor grad_weight8(const Tensor& grad_output, const Tensor& codes, const Tensor& scales, std::optional<at::ScalarType> dtype)
{
    check_rank("grad_weight8", grad_output);
    const Packed p = packed_arg("grad_weight8", codes, scales);
    TORCH_CHECK(codes.dim() == grad_output.dim() && codes.sizes().slice(0, codes.dim() - 1) == grad_output.sizes().slice(0, codes.dim() - 1),
                "grad_weight8: grad_output ", grad_output.sizes(), " and codes ", codes.sizes(), " must have the same leading dimensions");
    check_device("grad_weight8", grad_output, {codes});
    type_code("grad_weight8", grad_output);
    const at::ScalarType out = dtype.value_or(grad_output.scalar_type());
    TORCH_CHECK(out == grad_output.scalar_type() || out == c10::kFloat, "grad_weight8: dtype must be grad_output's or float32, got ",
                c10::toString(out));
    return weight_gradient(grad_output.detach(), p, out);
}

// A tensor as a matrix of its last dimension's rows (a copy where its strides allow no view).
Tensor matrix_of(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({leading(t), t.size(-1)}); }

Tensor with_rows_of(const Tensor& product, const Tensor& t)
{
    if (t.dim() == 2) return product;
    std::vector<int64_t> shape = t.sizes().vec();
    shape.back() = product.size(1);
    return at::_unsafe_view(product, shape);  // no view to autograd: the product is nobody else's
}

// The plain products in the operands' type, under autocast too (a backward called inside its region runs under it as well).
// Always of matrices: of more dimensions with strides that allow no view torch makes a batched product, with the weight's
// transpose for every batch.
Tensor plain_product(const Tensor& x, const Tensor& weight)
{
    const c10::impl::ExcludeDispatchKeyGuard guard(c10::DispatchKey::AutocastCUDA);
    return with_rows_of(at::linear(matrix_of(x), weight), x);
}

Tensor plain_product_grad(const Tensor& grad, const Tensor& weight)
{
    const c10::impl::ExcludeDispatchKeyGuard guard(c10::DispatchKey::AutocastCUDA);
    return with_rows_of(at::mm(matrix_of(grad), weight), grad);
}

class Linear8Function : public torch::autograd::Function<Linear8Function>
{
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& codes, const OptTensor& scales)
    {
        const c10::DeviceGuard guard(x.device());
        Packed p;
        if (weight.requires_grad()) p = codes.has_value() ? Packed{codes->contiguous(), scales->contiguous()} : pack_rows(x);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x.requires_grad() ? weight : Tensor(), p.codes, p.scales});
        ctx->saved_data["type"] = (int64_t)weight.scalar_type();
        return plain_product(x, weight);
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads)
    {
        const Tensor gy = grads[0];
        if (!gy.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        check_first_order("linear8");
        const auto saved = ctx->get_saved_variables();
        const c10::DeviceGuard guard(gy.device());
        Tensor gx, gw;
        if (ctx->needs_input_grad(0)) gx = plain_product_grad(gy, saved[0]);
        if (ctx->needs_input_grad(1)) gw = weight_gradient(gy, Packed{saved[1], saved[2]}, (at::ScalarType)ctx->saved_data["type"].toInt());
        return {gx, gw, Tensor(), Tensor()};
    }
};

Tensor linear8(const Tensor& input, const Tensor& weight, const OptTensor& codes, const OptTensor& scales)
{
    check_rank("linear8", input);
    TORCH_CHECK(weight.dim() == 2 && weight.size(1) == input.size(-1), "linear8: weight must be [out, ", input.size(-1), "], got ", weight.sizes());
    TORCH_CHECK(codes.has_value() == scales.has_value(), "linear8: codes and scales go together");
    check_device("linear8", input, {weight});
    type_code("linear8", input);
    check_type(input, weight);
    if (codes.has_value())
    {
        TORCH_CHECK(codes->sizes() == input.sizes(), "linear8: the packed input must have the input's shape ", input.sizes(), ", got ",
                    codes->sizes());
        packed_arg("linear8", *codes, *scales);
        check_device("linear8", input, {*codes});
    }
    if (!records({input, weight})) return plain_product(input, weight);
    return Linear8Function::apply(input, weight, codes, scales);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(morphocore, m)
{
    m.def("pack8(Tensor input) -> (Tensor, Tensor)");
    m.def("unpack8(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
    m.def("rms_norm(Tensor input, Tensor weight, Tensor? residual=None, float eps=1e-06) -> (Tensor, Tensor)");
    m.def("rms_norm8(Tensor input, Tensor weight, Tensor? residual=None, float eps=1e-06, bool full=True) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("gated_silu(Tensor gate, Tensor? up=None) -> Tensor");
    m.def("gated_silu8(Tensor gate, Tensor? up=None) -> (Tensor, Tensor, Tensor)");
    m.def("linear8(Tensor input, Tensor weight, Tensor? codes=None, Tensor? scales=None) -> Tensor");
    m.def("grad_weight8(Tensor grad_output, Tensor codes, Tensor scales, ScalarType? dtype=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(morphocore, CompositeImplicitAutograd, m)
{
    m.impl("pack8", &pack8);
    m.impl("unpack8", &unpack8);
    m.impl("rms_norm", &rms_norm);
    m.impl("rms_norm8", &rms_norm8);
    m.impl("gated_silu", &gated_silu);
    m.impl("gated_silu8", &gated_silu8);
    m.impl("linear8", &linear8);
    m.impl("grad_weight8", &grad_weight8);
}
