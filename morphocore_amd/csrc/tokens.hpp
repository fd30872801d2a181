// Host-side launchers of the token-mixing kernels (rotary.hip, linear_attention.hip), called by their C ABI
// (tokens_api.cpp). Arguments are assumed validated by the caller; every launch is asynchronous on `stream`.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mca
{

// tokens x heads x dim values, a head's consecutive.
template <typename T>
struct HeadRows
{
    const T* x;
    int64_t token_stride, head_stride;
    int heads;
};

// Where a token is, and the radians a position of every pair: frequencies [axes, pairs]. Token t has row t % rows
// of positions [rows, axes].
struct Rotation
{
    const void* positions;
    int position_type;  // MCA_POSITION_*
    int64_t rows;
    int axes, pairs;
    const double* frequencies;
    bool interleaved;
};

// out: dense. inverse: by the negative angles (the gradient).
template <typename T>
hipError_t axial_rotary(HeadRows<T> x, T* out, int64_t tokens, int dim, const Rotation& r, bool inverse, hipStream_t stream);

template <typename T, typename WT>
hipError_t rms_norm_rotary_forward(HeadRows<T> q, HeadRows<T> k, const WT* q_weight, const WT* k_weight, float eps, T* out_q, T* out_k,
                                   int64_t tokens, int dim, const Rotation& r, hipStream_t stream);
size_t rms_norm_rotary_backward_workspace(int64_t tokens, int heads, int dim, int pairs);
// grad_weights [2, dim]: the queries', the keys'; it may be null, as either of grad_q and grad_k.
template <typename T, typename WT>
hipError_t rms_norm_rotary_backward(HeadRows<T> gy_q, HeadRows<T> gy_k, HeadRows<T> q, HeadRows<T> k, const WT* q_weight, const WT* k_weight,
                                    float eps, T* grad_q, T* grad_k, WT* grad_weights, int64_t tokens, int dim, const Rotation& r,
                                    void* workspace, hipStream_t stream);

// Rows of heads of a batch, or of packed sequences (batch_stride 0): `heads` of them, each for `share` heads of the call.
struct TokenRows
{
    const void* p;
    int64_t batch_stride, token_stride, head_stride;
    int share;
};

// Where the sequences lie: `count` of `tokens` rows each, or, with offsets (32 or 64 bits), one after another in
// `tokens` rows, sequence s from offsets[s] to offsets[s + 1].
struct Sequences
{
    const void* offsets;
    bool wide;
    int64_t count, tokens;
};

// Every head's state [rows, cols] of every sequence, value (i, j) at i * row_stride + j * col_stride.
struct States
{
    float* p;
    int64_t row_stride, col_stride;
};

// One of linear attention's passes over the sequences, S the head's state, d its decay, a, b and out's c rows:
//   forwards: S = d S + update b_t c_t^T, out_t = read a_t S;  backwards, t falling: S = S + update b_t c_t^T,
//   out_t = read a_t S, S = d S.
// S begins with `first` and ends in `last`. a, b: dim values a row; c, out: cols. out: dense [rows, heads, cols], or in
// float32 where out32 is given; null: only the state is wanted.
struct Pass
{
    TokenRows a, b, c;
    void* out;
    float* out32;
    States first, last;  // null: zeros, not wanted
    int dim, cols;
    float update, read;
    bool backwards;
    int together;  // passes of this shape that the whole call has, whichever are asked for: sequences are split by their number
};

template <typename T>
size_t linear_attention_workspace(const Sequences& seq, int heads, const Pass* passes, int count);
// The passes are independent of each other.
template <typename T>
hipError_t linear_attention(const Sequences& seq, int heads, const float* log_decay, const Pass* passes, int count, void* workspace,
                            hipStream_t stream);

// out [rows, heads / share, cols] = the sum over the `share` heads of part [rows, heads, cols].
template <typename T>
hipError_t sum_shared_heads(const float* part, T* out, int64_t rows, int heads, int share, int cols, hipStream_t stream);

// One token for each of `batch` sequences, whose states [slots, heads, dim, cols] are updated in place.
template <typename T>
hipError_t linear_attention_step(TokenRows q, TokenRows k, TokenRows v, const float* log_decay, float* states, int64_t slot_stride,
                                 int64_t head_stride, const void* slot_of, bool wide, int64_t slots, T* out, int64_t batch, int heads, int dim,
                                 int cols, float scale, hipStream_t stream);

}  // namespace mca
