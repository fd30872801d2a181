/*
 * morphocore_amd — C ABI of the token-mixing kernels (gfx950): rotary positions with several axes, the norm of each
 * head's queries and keys with the rotation in the same pass, and linear attention with a decay for each head. No
 * reference counterpart.
 *
 * Conventions are those of morphocore_amd.h (status codes, mca_last_error, streams, caller-owned workspaces) and
 * morphocore_amd_mixer.h (dtype, weight_dtype). Strides count elements; a head's values are consecutive; overlapping
 * rows are allowed for what is read. Results without strides are dense. Sums and states are float32 or wider.
 */
#ifndef MORPHOCORE_AMD_TOKENS_H
#define MORPHOCORE_AMD_TOKENS_H

#include <stddef.h>
#include <stdint.h>

#include "morphocore_amd_mixer.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MCA_POSITION_INT32 0
#define MCA_POSITION_INT64 1
#define MCA_POSITION_FLOAT32 2

/* tokens x heads x dim values. batch_stride is read where there are batches. */
typedef struct
{
    const void* data;
    int64_t batch_stride, token_stride, head_stride, heads;
} mca_heads;

/* The angle of a token's pair j: the sum over the axes a of positions[t % rows, a] * frequencies[a, j], in radians, in float64.
 * positions [rows, axes] of position_type, frequencies [axes, pairs]; axes up to 8. Pair j of a row is its values j and
 * pairs + j, or, interleaved, 2 j and 2 j + 1; (a, b) becomes (a cos - b sin, b cos + a sin), values behind the pairs stay. */
typedef struct
{
    const void* positions;
    int position_type;
    int64_t rows, axes, pairs;
    const double* frequencies;
    int interleaved;
} mca_rotation;

/* out [tokens, x.heads, dim] = x rotated, or by the negative angles (the gradient). dim up to 512, heads up to 65536. */
int mca_axial_rotary(int dtype, const mca_heads* x, void* out, int64_t tokens, int64_t dim, const mca_rotation* rotation, int inverse,
                     void* stream);

/* q and k, each head's row as x / sqrt(mean(x^2) + eps) * weight, rotated. weights [dim]. */
int mca_rms_norm_rotary_forward(int dtype, int weight_dtype, const mca_heads* q, const mca_heads* k, const void* q_weight,
                                const void* k_weight, float eps, void* out_q, void* out_k, int64_t tokens, int64_t dim,
                                const mca_rotation* rotation, void* stream);

/* grad_q, grad_k (dense; either may be NULL) and grad_weights [2, dim] (q_weight's, k_weight's; may be NULL) from the
 * results' gradients and q and k as they were. */
size_t mca_rms_norm_rotary_backward_workspace_size(int64_t tokens, int64_t heads, int64_t dim, int64_t pairs);
int mca_rms_norm_rotary_backward(int dtype, int weight_dtype, const mca_heads* grad_out_q, const mca_heads* grad_out_k, const mca_heads* q,
                                 const mca_heads* k, const void* q_weight, const void* k_weight, float eps, void* grad_q, void* grad_k,
                                 void* grad_weights, int64_t tokens, int64_t dim, const mca_rotation* rotation, void* workspace,
                                 size_t workspace_bytes, void* stream);

/* Sequences of the linear attention: `count` of `tokens` tokens each (offsets NULL), or packed one after another in `tokens` rows:
 * sequence s is the rows from offsets[s] to offsets[s + 1]; offsets [count + 1] must not fall, of 32 or (wide) 64 bits, in device
 * memory. Rows of no sequence get zeros. Offsets outside the rows are taken as the nearest row. */
typedef struct
{
    const void* offsets;
    int wide;
    int64_t count, tokens;
} mca_sequences;

/* S_t = d S_(t-1) + k_t v_t^T, out_t = scale q_t S_t, for each of q's heads with d = exp(log_decay[head]); S_0 = initial [count,
 * heads, dim, value_dim] (NULL: zeros), the last state goes to `final` (may be NULL). k and v have as many heads as each
 * other, of which q's are a multiple: neighbouring heads of q share one. dim and value_dim up to 256. */
size_t mca_linear_attention_forward_workspace_size(int dtype, const mca_sequences* sequences, int64_t heads, int64_t dim, int64_t value_dim);
int mca_linear_attention_forward(int dtype, const mca_sequences* sequences, const mca_heads* q, const mca_heads* k, const mca_heads* v,
                                 const float* log_decay, const float* initial, void* out, float* final, int64_t dim, int64_t value_dim,
                                 float scale, void* workspace, size_t workspace_bytes, void* stream);

/* The gradients of q, k, v (dense, of their own heads) and of the initial state, from grad_out and grad_final (NULL: zeros). Each result
 * may be NULL. */
size_t mca_linear_attention_backward_workspace_size(int dtype, const mca_sequences* sequences, int64_t heads, int64_t kv_heads, int64_t dim,
                                                    int64_t value_dim);
int mca_linear_attention_backward(int dtype, const mca_sequences* sequences, const mca_heads* grad_out, const float* grad_final,
                                  const mca_heads* q, const mca_heads* k, const mca_heads* v, const float* log_decay, const float* initial,
                                  void* grad_q, void* grad_k, void* grad_v, float* grad_initial, int64_t dim, int64_t value_dim, float scale,
                                  void* workspace, size_t workspace_bytes, void* stream);

/* One token for each of `batch` sequences. Sequence b's state, [heads, dim, value_dim] at states + slot * slot_stride (heads head_stride
 * apart, dense within), is updated in place; its slot is slot_of[b], of 32 or (wide) 64 bits, or b without slot_of. States of different
 * slots and heads must not share memory: one of the two strides reaches over all that the other one spans. A slot outside
 * [0, slots) stands for no sequence: its row of out is zero. Rows that name the same slot are taken one after another. The
 * rows' token_stride is read, their batch_stride is not. */
int mca_linear_attention_step(int dtype, const mca_heads* q, const mca_heads* k, const mca_heads* v, const float* log_decay, float* states,
                              int64_t slot_stride, int64_t head_stride, const void* slot_of, int wide, int64_t slots, void* out,
                              int64_t batch, int64_t dim, int64_t value_dim, float scale, void* stream);

#ifdef __cplusplus
}
#endif

#endif
