// The token-mixing operators of the PyTorch-ROCm extension: axial_rotary, rms_norm_rotary, linear_attention and
// linear_attention_step, in the namespace that torch_ops.cpp registers. No reference counterpart. Device work is the C ABI
// of include/morphocore_amd_tokens.h.
//
// Tensors are [.., heads, values]; whatever strides their other dimensions have they are read where they are, if a head's values
// are consecutive (and, of rotations, the tokens at one distance), and copied otherwise. Only HIP devices; everything else is
// an error, never a fallback.
#include "ops.hpp"

#include <c10/core/InferenceMode.h>

#include "../../include/morphocore_amd_tokens.h"

namespace
{

mca_heads heads_arg(const Tensor& t, int64_t batch_stride, int64_t token_stride)
{
    return mca_heads{t.const_data_ptr(), batch_stride, token_stride, t.stride(-2), t.size(-2)};
}

// ------------------------------------------------------------------------------------------------
// Rotations.
// ------------------------------------------------------------------------------------------------

// [.., heads, dim] as tokens at one distance.
struct Tokens
{
    Tensor t;  // keeps the memory
    mca_heads heads;
};

Tokens tokens_of(const Tensor& x)
{
    Tensor t = x;
    int64_t stride = 0;
    if (x.numel())
    {
        // The stride of x's rows of heads, as if a head's first value were the whole head.
        const Tensor first = x.select(-1, 0);
        stride = x.size(-1) > 1 && x.stride(-1) != 1 ? -1 : x.dim() == 2 ? 0 : row_stride(first.select(-1, 0).unsqueeze(-1));
        if (stride < 0)
        {
            t = x.contiguous();
            stride = t.size(-2) * t.size(-1);
        }
    }
    return Tokens{t, heads_arg(t, 0, stride)};
}

int64_t token_count(const Tensor& x)
{
    int64_t n = 1;
    for (int64_t d = 0; d + 2 < x.dim(); ++d) n *= x.size(d);
    return n;
}

int position_type(const char* name, const Tensor& positions)
{
    switch (positions.scalar_type())
    {
        case c10::kInt: return MCA_POSITION_INT32;
        case c10::kLong: return MCA_POSITION_INT64;
        case c10::kFloat: return MCA_POSITION_FLOAT32;
        default: TORCH_CHECK(false, name, ": positions must be int32, int64 or float32, got ", c10::toString(positions.scalar_type()));
    }
    return -1;
}

void check_rotation(const char* name, const Tensor& x, const Tensor& positions, const Tensor& frequencies)
{
    TORCH_CHECK(x.dim() >= 2, name, ": the input must be [.., heads, values], got ", x.sizes());
    type_code(name, x);
    position_type(name, positions);
    TORCH_CHECK(frequencies.dim() == 2 && frequencies.scalar_type() == c10::kDouble, name, ": frequencies must be float64 [axes, pairs], got ",
                c10::toString(frequencies.scalar_type()), " ", frequencies.sizes());
    const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 2);
    const int64_t d = positions.dim() - 1;
    TORCH_CHECK(d >= 0 && d <= (int64_t)lead.size() && positions.size(-1) == frequencies.size(0) &&
                    positions.sizes().slice(0, d) == lead.slice(lead.size() - d, d),
                name, ": positions must be [.., ", frequencies.size(0), "] of the tokens ", lead, " or of their last dimensions, got ", positions.sizes());
    TORCH_CHECK(2 * frequencies.size(1) <= x.size(-1), name, ": ", frequencies.size(1), " pairs need at least ", 2 * frequencies.size(1),
                " values a head, got ", x.size(-1));
    TORCH_CHECK(!records({positions, frequencies}), name, ": positions and frequencies have no gradient; detach them");
    check_no_tangent(name, {positions, frequencies});
    check_device(name, x, {positions, frequencies});
}

mca_rotation rotation_arg(const char* name, const Tensor& positions, const Tensor& frequencies, bool interleaved)
{
    return mca_rotation{positions.const_data_ptr(), position_type(name, positions), positions.size(-1) ? positions.numel() / positions.size(-1) : 0,
                        frequencies.size(0), frequencies.size(1), frequencies.const_data_ptr<double>(), interleaved};
}

Tensor rotary_run(const Tensor& x, const Tensor& positions, const Tensor& frequencies, bool interleaved, bool inverse)
{
    const c10::DeviceGuard guard(x.device());
    const Tokens t = tokens_of(x);
    const mca_rotation r = rotation_arg("axial_rotary", positions, frequencies, interleaved);
    Tensor out = torch::empty(x.sizes(), x.options());
    check_rc(mca_axial_rotary(type_code("axial_rotary", x), &t.heads, out.data_ptr(), token_count(x), x.size(-1), &r, inverse, stream_of(x)));
    return out;
}

class AxialRotaryFunction : public torch::autograd::Function<AxialRotaryFunction>
{
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions, const Tensor& frequencies, bool interleaved)
    {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions, frequencies});
        ctx->saved_data["interleaved"] = interleaved;
        return rotary_run(x, positions, frequencies, interleaved, false);
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads)
    {
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        check_first_order("axial_rotary");
        const auto saved = ctx->get_saved_variables();
        return {rotary_run(grads[0], saved[0], saved[1], ctx->saved_data["interleaved"].toBool(), true), Tensor(), Tensor(), Tensor()};
    }
};

Tensor axial_rotary(const Tensor& input, const Tensor& positions, const Tensor& frequencies, bool interleaved)
{
    check_no_tangent("axial_rotary", {input});
    check_rotation("axial_rotary", input, positions, frequencies);
    const Tensor p = positions.contiguous(), f = frequencies.contiguous();
    if (!records({input})) return rotary_run(input, p, f, interleaved, false);
    return AxialRotaryFunction::apply(input, p, f, interleaved);
}

class RmsNormRotaryFunction : public torch::autograd::Function<RmsNormRotaryFunction>
{
public:
    static std::tuple<Tensor, Tensor> run(const Tensor& query, const Tensor& key, const Tensor& query_weight, const Tensor& key_weight,
                                          const Tensor& positions, const Tensor& frequencies, double eps, bool interleaved)
    {
        const c10::DeviceGuard guard(query.device());
        const Tokens q = tokens_of(query), k = tokens_of(key);
        const Tensor qw = query_weight.contiguous(), kw = key_weight.contiguous();
        const mca_rotation r = rotation_arg("rms_norm_rotary", positions, frequencies, interleaved);
        Tensor oq = torch::empty(query.sizes(), query.options()), ok = torch::empty(key.sizes(), key.options());
        check_rc(mca_rms_norm_rotary_forward(type_code("rms_norm_rotary", query), type_code("rms_norm_rotary", qw), &q.heads, &k.heads,
                                             qw.const_data_ptr(), kw.const_data_ptr(), (float)eps, oq.data_ptr(), ok.data_ptr(), token_count(query),
                                             query.size(-1), &r, stream_of(query)));
        return {oq, ok};
    }

    static tensor_list forward(AutogradContext* ctx, const Tensor& query, const Tensor& key, const Tensor& query_weight, const Tensor& key_weight,
                               const Tensor& positions, const Tensor& frequencies, double eps, bool interleaved)
    {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({query, key, query_weight, key_weight, positions, frequencies});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        const auto out = run(query, key, query_weight, key_weight, positions, frequencies, eps, interleaved);
        return {std::get<0>(out), std::get<1>(out)};
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads)
    {
        if (!grads[0].defined() && !grads[1].defined()) return tensor_list(8);
        check_first_order("rms_norm_rotary");
        const auto saved = ctx->get_saved_variables();
        const Tensor &query = saved[0], &key = saved[1];
        const c10::DeviceGuard guard(query.device());
        // A result without a gradient counts as one with zeros.
        const Tensor gq = grads[0].defined() ? grads[0] : torch::zeros(query.sizes(), query.options());
        const Tensor gk = grads[1].defined() ? grads[1] : torch::zeros(key.sizes(), key.options());
        const Tokens q = tokens_of(query), k = tokens_of(key), tq = tokens_of(gq), tk = tokens_of(gk);
        const Tensor qw = saved[2].contiguous(), kw = saved[3].contiguous();
        const mca_rotation r = rotation_arg("rms_norm_rotary", saved[4], saved[5], ctx->saved_data["interleaved"].toBool());
        const int64_t tokens = token_count(query), dim = query.size(-1);
        const bool need_w = ctx->needs_input_grad(2) || ctx->needs_input_grad(3);
        const Tensor xq = ctx->needs_input_grad(0) ? torch::empty(query.sizes(), query.options()) : Tensor();
        const Tensor xk = ctx->needs_input_grad(1) ? torch::empty(key.sizes(), key.options()) : Tensor();
        const Tensor gw = need_w ? torch::empty({2, dim}, qw.options()) : Tensor();
        const size_t bytes = need_w ? mca_rms_norm_rotary_backward_workspace_size(tokens, query.size(-2) + key.size(-2), dim, r.pairs) : 0;
        const Tensor ws = torch::empty({(int64_t)bytes}, query.options().dtype(torch::kUInt8));
        check_rc(mca_rms_norm_rotary_backward(type_code("rms_norm_rotary", query), type_code("rms_norm_rotary", qw), &tq.heads, &tk.heads, &q.heads,
                                              &k.heads, qw.const_data_ptr(), kw.const_data_ptr(), (float)ctx->saved_data["eps"].toDouble(),
                                              xq.defined() ? xq.data_ptr() : nullptr, xk.defined() ? xk.data_ptr() : nullptr,
                                              need_w ? gw.data_ptr() : nullptr, tokens, dim, &r, ws.data_ptr(), bytes, stream_of(query)));
        return {xq, xk, ctx->needs_input_grad(2) ? gw.select(0, 0) : Tensor(), ctx->needs_input_grad(3) ? gw.select(0, 1) : Tensor(), Tensor(), Tensor(),
                Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> rms_norm_rotary(const Tensor& query, const Tensor& key, const Tensor& query_weight, const Tensor& key_weight,
                                           const Tensor& positions, const Tensor& frequencies, double eps, bool interleaved)
{
    const char* name = "rms_norm_rotary";
    check_no_tangent(name, {query, key, query_weight, key_weight});
    TORCH_CHECK(query.dim() >= 2, name, ": the input must be [.., heads, values], got ", query.sizes());
    TORCH_CHECK(key.dim() == query.dim() && key.size(-1) == query.size(-1) &&
                    key.sizes().slice(0, key.dim() - 2) == query.sizes().slice(0, query.dim() - 2),
                name, ": key must be [.., heads, values] with the query's tokens and values ", query.sizes(), ", got ", key.sizes());
    check_type(query, key);
    for (const Tensor& w : {query_weight, key_weight})
    {
        TORCH_CHECK(w.dim() == 1 && w.size(0) == query.size(-1), name, ": weights must be [", query.size(-1), "], got ", w.sizes());
        if (w.scalar_type() != c10::kFloat) check_type(query, w);
    }
    check_type(query_weight, key_weight);
    TORCH_CHECK(eps >= 0.0, name, ": eps must be non negative");
    check_rotation(name, query, positions, frequencies);
    check_device(name, query, {key, query_weight, key_weight});
    const Tensor p = positions.contiguous(), f = frequencies.contiguous();
    if (!records({query, key, query_weight, key_weight})) return RmsNormRotaryFunction::run(query, key, query_weight, key_weight, p, f, eps, interleaved);
    const tensor_list out = RmsNormRotaryFunction::apply(query, key, query_weight, key_weight, p, f, eps, interleaved);
    return {out[0], out[1]};
}

// ------------------------------------------------------------------------------------------------
// Linear attention.
// ------------------------------------------------------------------------------------------------

// [batch, tokens, heads, values], [tokens, heads, values] of packed sequences, or [batch, heads, values] of a step.
struct HeadsOf
{
    Tensor t;  // keeps the memory
    mca_heads heads;
};

HeadsOf heads_of(const Tensor& x)
{
    const Tensor t = x.size(-1) > 1 && x.stride(-1) != 1 ? x.contiguous() : x;
    return HeadsOf{t, heads_arg(t, t.dim() == 4 ? t.stride(0) : 0, t.stride(-3))};
}

// The sequences of a query, and their number.
mca_sequences sequences_of(const Tensor& query, const Tensor& offsets)
{
    if (offsets.defined()) return mca_sequences{offsets.const_data_ptr(), offsets.scalar_type() == c10::kLong, offsets.size(0) - 1, query.size(0)};
    return mca_sequences{nullptr, 0, query.size(0), query.size(1)};
}

Tensor workspace_of(const Tensor& like, size_t bytes) { return torch::empty({(int64_t)bytes}, like.options().dtype(torch::kUInt8)); }

const float* floats(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }

class LinearAttentionFunction : public torch::autograd::Function<LinearAttentionFunction>
{
public:
    // (out, the last state or nothing)
    static std::tuple<Tensor, Tensor> run(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& log_decay, const Tensor& state,
                                          const Tensor& offsets, double scale, bool final_state)
    {
        const c10::DeviceGuard guard(query.device());
        const HeadsOf q = heads_of(query), k = heads_of(key), v = heads_of(value);
        const mca_sequences s = sequences_of(query, offsets);
        const Tensor g = log_decay.contiguous(), first = state.defined() ? state.contiguous() : Tensor();
        const int64_t dim = query.size(-1), value_dim = value.size(-1);
        std::vector<int64_t> shape = query.sizes().vec();
        shape.back() = value_dim;
        Tensor out = torch::empty(shape, query.options());
        Tensor last = final_state ? torch::empty({s.count, query.size(-2), dim, value_dim}, query.options().dtype(c10::kFloat)) : Tensor();
        const int type = type_code("linear_attention", query);
        const size_t bytes = mca_linear_attention_forward_workspace_size(type, &s, query.size(-2), dim, value_dim);
        const Tensor ws = workspace_of(query, bytes);
        check_rc(mca_linear_attention_forward(type, &s, &q.heads, &k.heads, &v.heads, floats(g), floats(first), out.data_ptr(),
                                              final_state ? last.data_ptr<float>() : nullptr, dim, value_dim, (float)scale, ws.data_ptr(), bytes,
                                              stream_of(query)));
        return {out, last};
    }

    static tensor_list forward(AutogradContext* ctx, const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& log_decay,
                               const OptTensor& state, const OptTensor& offsets, double scale, bool final_state)
    {
        const Tensor first = state.value_or(Tensor()), o = offsets.value_or(Tensor());
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({query, key, value, log_decay, first, o});
        ctx->saved_data["scale"] = scale;
        const auto out = run(query, key, value, log_decay, first, o, scale, final_state);
        if (!final_state) return {std::get<0>(out)};
        return {std::get<0>(out), std::get<1>(out)};
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads)
    {
        const Tensor grad_final = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !grad_final.defined()) return tensor_list(8);
        check_first_order("linear_attention");
        const auto saved = ctx->get_saved_variables();
        const Tensor &query = saved[0], &key = saved[1], &value = saved[2], &state = saved[4], &offsets = saved[5];
        const c10::DeviceGuard guard(query.device());
        std::vector<int64_t> shape = query.sizes().vec();
        shape.back() = value.size(-1);
        const HeadsOf go = heads_of(grads[0].defined() ? grads[0] : torch::zeros(shape, query.options()));
        const HeadsOf q = heads_of(query), k = heads_of(key), v = heads_of(value);
        const mca_sequences s = sequences_of(query, offsets);
        const Tensor g = saved[3].contiguous(), first = state.defined() ? state.contiguous() : Tensor();
        const Tensor last = grad_final.defined() ? grad_final.contiguous() : Tensor();
        Tensor result[4];
        const Tensor* of[4] = {&query, &key, &value, &state};
        // needs_input_grad counts the tensors that were given: query, key, value, log_decay, state.
        for (int i = 0; i < 4; ++i)
            if (of[i]->defined() && ctx->needs_input_grad(i < 3 ? i : 4)) result[i] = torch::empty(of[i]->sizes(), of[i]->options());
        auto data = [&](int i) { return result[i].defined() ? result[i].data_ptr() : nullptr; };
        const int64_t dim = query.size(-1), value_dim = value.size(-1);
        const int type = type_code("linear_attention", query);
        const size_t bytes = mca_linear_attention_backward_workspace_size(type, &s, query.size(-2), key.size(-2), dim, value_dim);
        const Tensor ws = workspace_of(query, bytes);
        check_rc(mca_linear_attention_backward(type, &s, &go.heads, floats(last), &q.heads, &k.heads, &v.heads, floats(g), floats(first), data(0),
                                               data(1), data(2), (float*)data(3), dim, value_dim, (float)ctx->saved_data["scale"].toDouble(),
                                               ws.data_ptr(), bytes, stream_of(query)));
        return {result[0], result[1], result[2], Tensor(), result[3], Tensor(), Tensor(), Tensor()};
    }
};

// What linear_attention and its step check alike.
void check_attention(const char* name, const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& log_decay)
{
    type_code(name, query);
    check_type(query, key);
    check_type(query, value);
    check_no_tangent(name, {query, key, value, log_decay});
    const int64_t d = query.dim();
    TORCH_CHECK(key.dim() == d && key.size(-1) == query.size(-1) && key.sizes().slice(0, d - 2) == query.sizes().slice(0, d - 2), name,
                ": key must have the query's tokens and values ", query.sizes(), ", got ", key.sizes());
    TORCH_CHECK(value.dim() == d && value.sizes().slice(0, d - 1) == key.sizes().slice(0, d - 1), name, ": value must have the key's tokens and heads ",
                key.sizes(), ", got ", value.sizes());
    TORCH_CHECK(key.size(-2) > 0 ? query.size(-2) % key.size(-2) == 0 : query.size(-2) == 0, name, ": the query's ", query.size(-2),
                " heads must be a multiple of the key's ", key.size(-2));
    TORCH_CHECK(log_decay.dim() == 1 && log_decay.size(0) == query.size(-2) && log_decay.scalar_type() == c10::kFloat, name,
                ": log_decay must be float32 [", query.size(-2), "], got ", c10::toString(log_decay.scalar_type()), " ", log_decay.sizes());
    TORCH_CHECK(!records({log_decay}), name, ": log_decay has no gradient; detach it");
}

void check_index(const char* name, const char* what, const Tensor& index)
{
    TORCH_CHECK(index.dim() == 1 && (index.scalar_type() == c10::kInt || index.scalar_type() == c10::kLong), name, ": ", what,
                " must be int32 or int64 with one dimension, got ", c10::toString(index.scalar_type()), " ", index.sizes());
}

// (out, last state); the second is undefined unless it is asked for.
std::tuple<Tensor, Tensor> linear_attention(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& log_decay,
                                            const OptTensor& state, const OptTensor& offsets, std::optional<double> scale, bool final_state)
{
    const char* name = "linear_attention";
    const Tensor o = offsets.has_value() ? offsets->contiguous() : Tensor(), first = state.value_or(Tensor());
    TORCH_CHECK(query.dim() == (o.defined() ? 3 : 4), name, o.defined() ? ": with offsets query must be [tokens, heads, values], got " : ": query must be [batch, tokens, heads, values], got ",
                query.sizes());
    check_attention(name, query, key, value, log_decay);
    if (o.defined())
    {
        check_index(name, "offsets", o);
        TORCH_CHECK(o.size(0) >= 1, name, ": offsets must have one entry more than there are sequences");
    }
    if (first.defined())
    {
        const std::vector<int64_t> shape = {o.defined() ? o.size(0) - 1 : query.size(0), query.size(-2), query.size(-1), value.size(-1)};
        check_no_tangent(name, {first});
        TORCH_CHECK(first.sizes() == at::IntArrayRef(shape) && first.scalar_type() == c10::kFloat, name, ": state must be float32 ", at::IntArrayRef(shape),
                    ", got ", c10::toString(first.scalar_type()), " ", first.sizes());
    }
    check_device(name, query, {key, value, log_decay});
    if (o.defined()) check_device(name, query, {o});
    if (first.defined()) check_device(name, query, {first});
    const double s = scale.value_or(1.0 / std::sqrt((double)query.size(-1)));
    if (!records({query, key, value, first})) return LinearAttentionFunction::run(query, key, value, log_decay, first, o, s, final_state);
    const tensor_list out = LinearAttentionFunction::apply(query, key, value, log_decay, state, o.defined() ? OptTensor(o) : OptTensor(), s, final_state);
    return {out[0], final_state ? out[1] : Tensor()};
}

Tensor linear_attention_step(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& log_decay, const Tensor& state,
                             const OptTensor& slots, std::optional<double> scale)
{
    const char* name = "linear_attention_step";
    TORCH_CHECK(query.dim() == 3, name, ": query must be [batch, heads, values], got ", query.sizes());
    check_attention(name, query, key, value, log_decay);
    TORCH_CHECK(!records({query, key, value, state}), name, " has no gradient; call it under torch.no_grad()");
    const int64_t batch = query.size(0), heads = query.size(1), dim = query.size(2), value_dim = value.size(2);
    const Tensor at = slots.has_value() ? slots->contiguous() : Tensor();
    check_no_tangent(name, {state});
    TORCH_CHECK(state.dim() == 4 && state.scalar_type() == c10::kFloat && state.size(1) == heads && state.size(2) == dim && state.size(3) == value_dim,
                name, ": state must be float32 [slots, ", heads, ", ", dim, ", ", value_dim, "], got ", c10::toString(state.scalar_type()), " ",
                state.sizes());
    if (at.defined())
    {
        check_index(name, "slots", at);
        TORCH_CHECK(at.size(0) == batch, name, ": slots must be [", batch, "], got ", at.sizes());
    }
    else
        TORCH_CHECK(state.size(0) == batch, name, ": without slots state must have ", batch, " entries, got ", state.size(0));
    // It is written in place, by workgroups that don't wait for each other: no copy may stand in for it, and no two of its entries may share memory.
    // One of the strides of slots and heads reaches over all that the other one spans.
    const bool dense = (value_dim == 1 || state.stride(3) == 1) && (dim == 1 || state.stride(2) == value_dim);
    const int64_t places = state.size(0), extent = dim * value_dim;
    const int64_t head_stride = heads > 1 ? state.stride(1) : extent, slot_stride = places > 1 ? state.stride(0) : 0;
    TORCH_CHECK(dense && head_stride >= extent && (places <= 1 || slot_stride >= extent) &&
                    (places <= 1 || heads <= 1 || slot_stride >= (heads - 1) * head_stride + extent || head_stride >= (places - 1) * slot_stride + extent),
                name, ": a head's state must be dense and share no memory with another, got strides ", state.strides());
    TORCH_CHECK(!state.is_inference() || c10::InferenceMode::is_enabled(), name, ": state is an inference tensor, which is written to in inference mode alone");
    check_device(name, query, {key, value, log_decay, state});
    if (at.defined()) check_device(name, query, {at});
    const c10::DeviceGuard guard(query.device());
    const HeadsOf q = heads_of(query), k = heads_of(key), v = heads_of(value);
    const Tensor g = log_decay.contiguous();
    Tensor out = torch::empty({batch, heads, value_dim}, query.options());
    check_rc(mca_linear_attention_step(type_code(name, query), &q.heads, &k.heads, &v.heads, floats(g), (float*)state.data_ptr(), slot_stride, head_stride,
                                       at.defined() ? at.const_data_ptr() : nullptr, at.defined() && at.scalar_type() == c10::kLong, state.size(0),
                                       out.data_ptr(), batch, dim, value_dim, (float)scale.value_or(1.0 / std::sqrt((double)dim)), stream_of(query)));
    state.unsafeGetTensorImpl()->bump_version();
    return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(morphocore, m)
{
    m.def("axial_rotary(Tensor input, Tensor positions, Tensor frequencies, bool interleaved=False) -> Tensor");
    m.def("rms_norm_rotary(Tensor query, Tensor key, Tensor query_weight, Tensor key_weight, Tensor positions, Tensor frequencies, float eps=1e-06, bool interleaved=False) -> (Tensor, Tensor)");
    m.def("linear_attention(Tensor query, Tensor key, Tensor value, Tensor log_decay, Tensor? state=None, Tensor? offsets=None, float? scale=None, bool final_state=False) -> (Tensor, Tensor)");
    m.def("linear_attention_step(Tensor query, Tensor key, Tensor value, Tensor log_decay, Tensor(a!) state, Tensor? slots=None, float? scale=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(morphocore, CompositeImplicitAutograd, m)
{
    m.impl("axial_rotary", &axial_rotary);
    m.impl("rms_norm_rotary", &rms_norm_rotary);
    m.impl("linear_attention", &linear_attention);
    m.impl("linear_attention_step", &linear_attention_step);
}
