// C ABI of the token-mixing kernels: argument validation, then the asynchronous launchers of rotary.hip and
// linear_attention.hip. Declarations: include/morphocore_amd_tokens.h.
#include "../../include/morphocore_amd_tokens.h"

#include "../../include/morphocore_amd.h"
#include "launch.hpp"
#include "tokens.hpp"

namespace
{

// What the lanes of one wave hold of a head's row, and the rows and columns of the state that a workgroup holds.
constexpr int64_t MAX_ROTARY_DIM = 512, MAX_STATE_DIM = 256, MAX_AXES = 8;
// Rows of a workgroup's tokens are told apart in float32.
constexpr int64_t MAX_ROTARY_HEADS = 65536;

int check_types(int dtype, int weight_dtype)
{
    if (dtype < MCA_FLOAT32 || dtype > MCA_BFLOAT16) return mca::api_fail("Unknown dtype: expected 0 (float32), 1 (float16) or 2 (bfloat16)");
    if (weight_dtype != dtype && weight_dtype != MCA_FLOAT32) return mca::api_fail("weight_dtype must be the activations' dtype or float32");
    return MCA_OK;
}

// tokens rows of heads of `dim` values, addressed with 64-bit byte offsets.
int check_heads(const mca_heads* x, int64_t tokens, int64_t dim)
{
    if (!x) return mca::api_fail("A tensor's mca_heads must not be null");
    if (tokens < 0 || x->heads < 0 || x->heads > INT32_MAX) return mca::api_fail("tokens and heads must be non negative, heads below 2^31");
    if (x->batch_stride < 0 || x->token_stride < 0 || x->head_stride < 0) return mca::api_fail("strides must be non negative");
    if (tokens > 0 && x->heads > 0)
    {
        if (tokens > INT64_MAX / 64 / dim / x->heads) return mca::api_fail("tokens * heads * dim is too large");
        if (!x->data) return mca::api_fail("A tensor's data must not be null");
    }
    return MCA_OK;
}

int check_rotation(const mca_rotation* r, int64_t tokens, int64_t dim)
{
    if (!r) return mca::api_fail("rotation must not be null");
    if (dim < 1 || dim > MAX_ROTARY_DIM) return mca::api_fail("dim must be from 1 to 512");
    if (r->position_type < MCA_POSITION_INT32 || r->position_type > MCA_POSITION_FLOAT32)
        return mca::api_fail("Unknown position_type: expected 0 (int32), 1 (int64) or 2 (float32)");
    if (r->axes < 1 || r->axes > MAX_AXES) return mca::api_fail("axes must be from 1 to 8");
    if (r->pairs < 0 || 2 * r->pairs > dim) return mca::api_fail("pairs must be from 0 to dim / 2");
    if (r->rows < 0 || (tokens > 0 && r->rows == 0)) return mca::api_fail("positions must have rows");
    if (tokens > 0 && (!r->positions || (r->pairs > 0 && !r->frequencies))) return mca::api_fail("positions and frequencies must not be null");
    return MCA_OK;
}

int check_rotary_heads(const mca_heads* x)
{
    return x->heads > MAX_ROTARY_HEADS ? mca::api_fail("Rotations take at most 65536 heads") : MCA_OK;
}

mca::Rotation rotation_of(const mca_rotation* r)
{
    return mca::Rotation{r->positions, r->position_type, r->rows, (int)r->axes, (int)r->pairs, r->frequencies, r->interleaved != 0};
}

template <typename T>
mca::HeadRows<T> head_rows(const mca_heads* x)
{
    return mca::HeadRows<T>{(const T*)x->data, x->token_stride, x->head_stride, (int)x->heads};
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

template <typename F>
int by_type(int dtype, F&& f)
{
    hipError_t err;
    if (dtype == MCA_FLOAT32)
        err = f((float*)nullptr);
    else if (dtype == MCA_FLOAT16)
        err = f((_Float16*)nullptr);
    else
        err = f((__bf16*)nullptr);
    return mca::api_hip_status(err);
}

int check_sequences(const mca_sequences* s)
{
    if (!s) return mca::api_fail("sequences must not be null");
    if (s->count < 0 || s->tokens < 0) return mca::api_fail("count and tokens must be non negative");
    if (s->count > INT32_MAX / 4) return mca::api_fail("Too many sequences");
    if (!s->offsets && s->count > 0 && s->tokens > INT64_MAX / 1024 / s->count) return mca::api_fail("count * tokens is too large");
    return MCA_OK;
}

int64_t rows_of(const mca_sequences* s) { return s->offsets ? s->tokens : s->count * s->tokens; }

int check_attention(int dtype, int64_t heads, int64_t kv_heads, int64_t dim, int64_t value_dim, int64_t states)
{
    int rc;
    if ((rc = check_types(dtype, dtype))) return rc;
    if (dim < 1 || dim > MAX_STATE_DIM || value_dim < 1 || value_dim > MAX_STATE_DIM) return mca::api_fail("dim and value_dim must be from 1 to 256");
    if (heads < 0 || heads > INT32_MAX || kv_heads < 0 || (heads > 0 && (kv_heads == 0 || heads % kv_heads)))
        return mca::api_fail("The queries' heads must be a multiple of the keys' and values'");
    if (heads > 0 && states > INT64_MAX / 8 / MAX_STATE_DIM / MAX_STATE_DIM / heads) return mca::api_fail("Too many states");
    return MCA_OK;
}

mca::Sequences sequences_of(const mca_sequences* s) { return mca::Sequences{s->offsets, s->wide != 0, s->count, s->tokens}; }

mca::TokenRows token_rows(const mca_heads* x, int64_t heads)
{
    return mca::TokenRows{x->data, x->batch_stride, x->token_stride, x->head_stride, x->heads > 0 ? (int)(heads / x->heads) : 1};
}

// Whether no two of slots x heads states of `extent` values share memory: neither stride is less than a state, and one of them reaches over
// all that the other one spans.
bool apart(int64_t slots, int64_t slot_stride, int64_t heads, int64_t head_stride, int64_t extent)
{
    if ((slots > 1 && slot_stride < extent) || (heads > 1 && head_stride < extent)) return false;
    return slots <= 1 || heads <= 1 || (slot_stride - extent) / head_stride >= heads - 1 || (head_stride - extent) / slot_stride >= slots - 1;
}

// A state as it lies, and transposed.
mca::States states_of(const float* p, int64_t value_dim) { return mca::States{(float*)p, value_dim, 1}; }
mca::States transposed(const float* p, int64_t value_dim) { return mca::States{(float*)p, 1, value_dim}; }

mca::Pass forward_pass(const mca_heads* q, const mca_heads* k, const mca_heads* v, const float* initial, void* out, float* final, int64_t dim,
                       int64_t value_dim, float scale)
{
    mca::Pass p = {};
    p.a = token_rows(q, q->heads), p.b = token_rows(k, q->heads), p.c = token_rows(v, q->heads);
    p.out = out;
    p.first = states_of(initial, value_dim), p.last = states_of(final, value_dim);
    p.dim = (int)dim, p.cols = (int)value_dim;
    p.update = 1.0f, p.read = scale;
    p.together = 1;
    return p;
}

// The backward's passes, and where the float32 gradients of shared heads lie in the workspace.
struct Backward
{
    mca::Pass pass[3];
    int count;
    size_t part_k, part_v, passes;  // bytes of each
};

Backward backward_passes(const mca_heads* go, const float* grad_final, const mca_heads* q, const mca_heads* k, const mca_heads* v, const float* initial,
                         void* grad_q, void* grad_k, void* grad_v, float* grad_initial, int64_t rows, int64_t dim, int64_t value_dim, float scale)
{
    Backward b = {};
    const int64_t heads = go->heads;
    const bool shared = heads > 0 && k->heads < heads;
    const mca::TokenRows rq = token_rows(q, heads), rk = token_rows(k, heads), rv = token_rows(v, heads), rg = token_rows(go, heads);
    if (grad_q)
    {
        mca::Pass p = {};
        p.a = rg, p.b = rv, p.c = rk;
        p.out = grad_q;
        p.first = transposed(initial, value_dim);
        p.dim = (int)value_dim, p.cols = (int)dim;
        p.update = 1.0f, p.read = scale;
        p.together = dim == value_dim ? 3 : 2;
        b.pass[b.count++] = p;
    }
    if (grad_k)
    {
        mca::Pass p = {};
        p.a = rv, p.b = rg, p.c = rq;
        p.out = grad_k;
        p.first = transposed(grad_final, value_dim);
        p.dim = (int)value_dim, p.cols = (int)dim;
        p.update = scale, p.read = 1.0f, p.backwards = true;
        p.together = dim == value_dim ? 3 : 2;
        if (shared) b.part_k = mca::align_up((size_t)(rows * heads * dim) * sizeof(float));
        b.pass[b.count++] = p;
    }
    if (grad_v || grad_initial)
    {
        mca::Pass p = {};
        p.a = rk, p.b = rq, p.c = rg;
        p.out = grad_v;
        p.first = states_of(grad_final, value_dim), p.last = states_of(grad_initial, value_dim);
        p.dim = (int)dim, p.cols = (int)value_dim;
        p.update = scale, p.read = 1.0f, p.backwards = true;
        p.together = dim == value_dim ? 3 : 1;
        if (shared && grad_v) b.part_v = mca::align_up((size_t)(rows * heads * value_dim) * sizeof(float));
        b.pass[b.count++] = p;
    }
    return b;
}

template <typename T>
size_t passes_workspace(const mca_sequences* s, int64_t heads, const mca::Pass* p, int count)
{
    return mca::linear_attention_workspace<T>(sequences_of(s), (int)heads, p, count);
}

size_t passes_workspace(int dtype, const mca_sequences* s, int64_t heads, const mca::Pass* p, int count)
{
    if (dtype == MCA_FLOAT32) return passes_workspace<float>(s, heads, p, count);
    if (dtype == MCA_FLOAT16) return passes_workspace<_Float16>(s, heads, p, count);
    return passes_workspace<__bf16>(s, heads, p, count);
}

}  // namespace

extern "C" {

int mca_axial_rotary(int dtype, const mca_heads* x, void* out, int64_t tokens, int64_t dim, const mca_rotation* rotation, int inverse, void* stream)
{
    int rc;
    if ((rc = check_types(dtype, dtype)) || (rc = check_rotation(rotation, tokens, dim)) || (rc = check_heads(x, tokens, dim)) || (rc = check_rotary_heads(x)))
        return rc;
    if (tokens > 0 && x->heads > 0 && !out) return mca::api_fail("out must not be null");
    return by_type(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return mca::axial_rotary<T>(head_rows<T>(x), (T*)out, tokens, (int)dim, rotation_of(rotation), inverse != 0, (hipStream_t)stream);
    });
}

int mca_rms_norm_rotary_forward(int dtype, int weight_dtype, const mca_heads* q, const mca_heads* k, const void* q_weight, const void* k_weight,
                                float eps, void* out_q, void* out_k, int64_t tokens, int64_t dim, const mca_rotation* rotation, void* stream)
{
    int rc;
    if ((rc = check_types(dtype, weight_dtype)) || (rc = check_rotation(rotation, tokens, dim)) || (rc = check_heads(q, tokens, dim)) ||
        (rc = check_heads(k, tokens, dim)))
        return rc;
    if ((rc = check_rotary_heads(q)) || (rc = check_rotary_heads(k))) return rc;
    if (!(eps >= 0.0f)) return mca::api_fail("eps must be non negative");
    if (tokens > 0 && ((q->heads > 0 && (!q_weight || !out_q)) || (k->heads > 0 && (!k_weight || !out_k))))
        return mca::api_fail("weights and results must not be null");
    return by_type(dtype, weight_dtype, [&](auto* t, auto* wt) {
        using T = std::remove_pointer_t<decltype(t)>;
        using WT = std::remove_pointer_t<decltype(wt)>;
        return mca::rms_norm_rotary_forward<T, WT>(head_rows<T>(q), head_rows<T>(k), (const WT*)q_weight, (const WT*)k_weight, eps, (T*)out_q,
                                                   (T*)out_k, tokens, (int)dim, rotation_of(rotation), (hipStream_t)stream);
    });
}

size_t mca_rms_norm_rotary_backward_workspace_size(int64_t tokens, int64_t heads, int64_t dim, int64_t pairs)
{
    if (tokens < 0 || heads < 0 || heads > 2 * MAX_ROTARY_HEADS || dim < 1 || dim > MAX_ROTARY_DIM || pairs < 0 || 2 * pairs > dim) return 0;
    return mca::rms_norm_rotary_backward_workspace(tokens, (int)heads, (int)dim, (int)pairs);
}

int mca_rms_norm_rotary_backward(int dtype, int weight_dtype, const mca_heads* grad_out_q, const mca_heads* grad_out_k, const mca_heads* q,
                                 const mca_heads* k, const void* q_weight, const void* k_weight, float eps, void* grad_q, void* grad_k,
                                 void* grad_weights, int64_t tokens, int64_t dim, const mca_rotation* rotation, void* workspace,
                                 size_t workspace_bytes, void* stream)
{
    int rc;
    if ((rc = check_types(dtype, weight_dtype)) || (rc = check_rotation(rotation, tokens, dim)) || (rc = check_heads(grad_out_q, tokens, dim)) ||
        (rc = check_heads(grad_out_k, tokens, dim)) || (rc = check_heads(q, tokens, dim)) || (rc = check_heads(k, tokens, dim)))
        return rc;
    if ((rc = check_rotary_heads(q)) || (rc = check_rotary_heads(k))) return rc;
    if (grad_out_q->heads != q->heads || grad_out_k->heads != k->heads) return mca::api_fail("A gradient must have its tensor's heads");
    if (!(eps >= 0.0f)) return mca::api_fail("eps must be non negative");
    if (tokens > 0 && ((q->heads > 0 && !q_weight) || (k->heads > 0 && !k_weight))) return mca::api_fail("weights must not be null");
    if (grad_weights &&
        (rc = check_workspace(workspace, workspace_bytes, mca_rms_norm_rotary_backward_workspace_size(tokens, q->heads + k->heads, dim, rotation->pairs))))
        return rc;
    return by_type(dtype, weight_dtype, [&](auto* t, auto* wt) {
        using T = std::remove_pointer_t<decltype(t)>;
        using WT = std::remove_pointer_t<decltype(wt)>;
        return mca::rms_norm_rotary_backward<T, WT>(head_rows<T>(grad_out_q), head_rows<T>(grad_out_k), head_rows<T>(q), head_rows<T>(k),
                                                    (const WT*)q_weight, (const WT*)k_weight, eps, (T*)grad_q, (T*)grad_k, (WT*)grad_weights,
                                                    tokens, (int)dim, rotation_of(rotation), workspace, (hipStream_t)stream);
    });
}

size_t mca_linear_attention_forward_workspace_size(int dtype, const mca_sequences* sequences, int64_t heads, int64_t dim, int64_t value_dim)
{
    if (check_sequences(sequences) || check_attention(dtype, heads, heads, dim, value_dim, sequences->count)) return 0;
    const mca_heads x = {nullptr, 0, 0, 0, heads};
    float state;  // never read: whether there is one decides the passes' shape
    const mca::Pass p = forward_pass(&x, &x, &x, &state, nullptr, &state, dim, value_dim, 1.0f);
    return passes_workspace(dtype, sequences, heads, &p, 1);
}

int mca_linear_attention_forward(int dtype, const mca_sequences* sequences, const mca_heads* q, const mca_heads* k, const mca_heads* v,
                                 const float* log_decay, const float* initial, void* out, float* final, int64_t dim, int64_t value_dim, float scale,
                                 void* workspace, size_t workspace_bytes, void* stream)
{
    int rc;
    if ((rc = check_sequences(sequences))) return rc;
    const int64_t rows = rows_of(sequences);
    if ((rc = check_heads(q, rows, MAX_STATE_DIM)) || (rc = check_heads(k, rows, MAX_STATE_DIM)) || (rc = check_heads(v, rows, MAX_STATE_DIM)) ||
        (rc = check_attention(dtype, q->heads, k->heads, dim, value_dim, sequences->count)))
        return rc;
    if (k->heads != v->heads) return mca::api_fail("Keys and values must have the same heads");
    if (q->heads > 0 && (!log_decay || (rows > 0 && !out))) return mca::api_fail("log_decay and out must not be null");
    if ((rc = check_workspace(workspace, workspace_bytes, mca_linear_attention_forward_workspace_size(dtype, sequences, q->heads, dim, value_dim))))
        return rc;
    const mca::Pass p = forward_pass(q, k, v, initial, out, final, dim, value_dim, scale);
    return by_type(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return mca::linear_attention<T>(sequences_of(sequences), (int)q->heads, log_decay, &p, 1, workspace, (hipStream_t)stream);
    });
}

size_t mca_linear_attention_backward_workspace_size(int dtype, const mca_sequences* sequences, int64_t heads, int64_t kv_heads, int64_t dim,
                                                    int64_t value_dim)
{
    if (check_sequences(sequences) || check_attention(dtype, heads, kv_heads, dim, value_dim, sequences->count)) return 0;
    const mca_heads x = {nullptr, 0, 0, 0, heads}, y = {nullptr, 0, 0, 0, kv_heads};
    float state;  // never read
    const Backward b = backward_passes(&x, &state, &x, &y, &y, &state, &state, &state, &state, &state, rows_of(sequences), dim, value_dim, 1.0f);
    return b.part_k + b.part_v + passes_workspace(dtype, sequences, heads, b.pass, b.count);
}

int mca_linear_attention_backward(int dtype, const mca_sequences* sequences, const mca_heads* grad_out, const float* grad_final, const mca_heads* q,
                                  const mca_heads* k, const mca_heads* v, const float* log_decay, const float* initial, void* grad_q, void* grad_k,
                                  void* grad_v, float* grad_initial, int64_t dim, int64_t value_dim, float scale, void* workspace,
                                  size_t workspace_bytes, void* stream)
{
    int rc;
    if ((rc = check_sequences(sequences))) return rc;
    const int64_t rows = rows_of(sequences);
    if ((rc = check_heads(grad_out, rows, MAX_STATE_DIM)) || (rc = check_heads(q, rows, MAX_STATE_DIM)) || (rc = check_heads(k, rows, MAX_STATE_DIM)) ||
        (rc = check_heads(v, rows, MAX_STATE_DIM)) || (rc = check_attention(dtype, q->heads, k->heads, dim, value_dim, sequences->count)))
        return rc;
    if (k->heads != v->heads || grad_out->heads != q->heads) return mca::api_fail("Keys and values, and queries and results, must have the same heads");
    if (q->heads > 0 && !log_decay) return mca::api_fail("log_decay must not be null");
    if ((rc = check_workspace(workspace, workspace_bytes,
                              mca_linear_attention_backward_workspace_size(dtype, sequences, q->heads, k->heads, dim, value_dim))))
        return rc;
    Backward b = backward_passes(grad_out, grad_final, q, k, v, initial, grad_q, grad_k, grad_v, grad_initial, rows, dim, value_dim, scale);
    float *part_k = nullptr, *part_v = nullptr;
    char* ws = (char*)workspace;
    if (b.part_k)
    {
        part_k = (float*)ws;
        ws += b.part_k;
    }
    if (b.part_v)
    {
        part_v = (float*)ws;
        ws += b.part_v;
    }
    for (int i = 0; i < b.count; ++i)
    {
        if (part_k && b.pass[i].out == grad_k) b.pass[i].out32 = part_k;
        if (part_v && b.pass[i].out == grad_v) b.pass[i].out32 = part_v;
    }
    const int heads = (int)q->heads, share = heads > 0 ? (int)(heads / k->heads) : 1;
    return by_type(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipError_t err = mca::linear_attention<T>(sequences_of(sequences), heads, log_decay, b.pass, b.count, ws, (hipStream_t)stream);
        if (err == hipSuccess && part_k) err = mca::sum_shared_heads<T>(part_k, (T*)grad_k, rows, heads, share, (int)dim, (hipStream_t)stream);
        if (err == hipSuccess && part_v) err = mca::sum_shared_heads<T>(part_v, (T*)grad_v, rows, heads, share, (int)value_dim, (hipStream_t)stream);
        return err;
    });
}

int mca_linear_attention_step(int dtype, const mca_heads* q, const mca_heads* k, const mca_heads* v, const float* log_decay, float* states,
                              int64_t slot_stride, int64_t head_stride, const void* slot_of, int wide, int64_t slots, void* out, int64_t batch,
                              int64_t dim, int64_t value_dim, float scale, void* stream)
{
    int rc;
    if ((rc = check_heads(q, batch, MAX_STATE_DIM)) || (rc = check_heads(k, batch, MAX_STATE_DIM)) || (rc = check_heads(v, batch, MAX_STATE_DIM)) ||
        (rc = check_attention(dtype, q->heads, k->heads, dim, value_dim, batch)))
        return rc;
    if (k->heads != v->heads) return mca::api_fail("Keys and values must have the same heads");
    if (slots < 0 || slot_stride < 0 || head_stride < dim * value_dim) return mca::api_fail("slots and slot_stride must be non negative, head_stride at least dim * value_dim");
    if (!apart(slots, slot_stride, q->heads, head_stride, dim * value_dim)) return mca::api_fail("States must not share memory");
    if (!slot_of && slots < batch) return mca::api_fail("Without slot_of there must be a slot for every sequence");
    if (batch > 0 && q->heads > 0 && (!log_decay || !out || (slots > 0 && !states))) return mca::api_fail("log_decay, states and out must not be null");
    return by_type(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return mca::linear_attention_step<T>(token_rows(q, q->heads), token_rows(k, q->heads), token_rows(v, q->heads), log_decay, states, slot_stride,
                                             head_stride, slot_of, wide != 0, slots, (T*)out, batch, (int)q->heads, (int)dim, (int)value_dim, scale,
                                             (hipStream_t)stream);
    });
}

}  // extern "C"
