// Linear attention a token at a time, with a decay for each head:
//   S = d S + k v^T,  out = scale q S,
// and the gradients of shared heads.
#include "linear_attention.hpp"

namespace mca
{

template <typename T>
__global__ __launch_bounds__(BLOCK) void sum_heads_kernel(const float* __restrict__ part, T* __restrict__ out, int64_t n, int share, int cols)
{
    for (int64_t j = (int64_t)blockIdx.x * BLOCK + threadIdx.x; j < n; j += (int64_t)gridDim.x * BLOCK)
    {
        const int64_t row = j / cols;
        const float* __restrict__ p = part + row * share * cols + (j - row * cols);
        float s = 0.0f;
        for (int i = 0; i < share; ++i) s += p[(int64_t)i * cols];
        out[j] = (T)s;
    }
}

template <typename T>
hipError_t sum_shared_heads(const float* part, T* out, int64_t rows, int heads, int share, int cols, hipStream_t stream)
{
    const int64_t n = rows * (heads / share) * cols, blocks = (n + BLOCK - 1) / BLOCK;
    if (n <= 0) return hipSuccess;
    sum_heads_kernel<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), BLOCK, 0, stream>>>(part, out, n, share, cols);
    return hipGetLastError();
}

// One head of one sequence of the batch, `COLS` columns. Rows of the batch that name the same slot are taken by the first of them, in order.
template <typename T>
__global__ __launch_bounds__(BLOCK) void attention_step_kernel(TokenRows q, TokenRows k, TokenRows v, const float* __restrict__ log_decay,
                                                               float* __restrict__ states, int64_t slot_stride, int64_t head_stride,
                                                               const void* __restrict__ slot_of, bool wide, int64_t slots, T* __restrict__ out,
                                                               int64_t batch, int heads, int dim, int cols, float scale, int tiles)
{
    constexpr int ROWS = 64;
    __shared__ float sq[256], sk[256], part[NWAVES][WAVE];
    const int tile = blockIdx.x % tiles, head = blockIdx.x / tiles % heads;
    const int64_t first = blockIdx.x / tiles / heads;
    auto slot_at = [&](int64_t b) -> int64_t {
        if (!slot_of) return b;
        return wide ? ((const int64_t*)slot_of)[b] : (int64_t)((const int32_t*)slot_of)[b];
    };
    const int64_t slot = slot_at(first);
    const int col = tile * WAVE + threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    auto store = [&](int64_t b, float x) {
        if (wave == 0 && col < cols) out[(b * heads + head) * cols + col] = (T)x;
    };
    if (slot < 0 || slot >= slots)
    {
        store(first, 0.0f);
        return;
    }
    if (slot_of)
    {
        bool before = false;
        for (int64_t b = threadIdx.x; b < first; b += BLOCK) before |= slot_at(b) == slot;
        if (__syncthreads_or(before)) return;
    }
    const Decay decay(log_decay_of(log_decay, head), 1);
    float* __restrict__ state = states + slot * slot_stride + head * head_stride;
    float s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
    {
        const int row = NWAVES * i + wave;
        s[i] = row < dim && col < cols ? state[(int64_t)row * cols + col] : 0.0f;
    }
    for (int64_t b = first; b < batch; ++b)
    {
        if (b > first && (!slot_of || slot_at(b) != slot)) continue;
        const T* rq = (const T*)q.p + b * q.token_stride + head / q.share * q.head_stride;
        const T* rk = (const T*)k.p + b * k.token_stride + head / k.share * k.head_stride;
        __syncthreads();
        if ((int)threadIdx.x < dim)
        {
            sq[threadIdx.x] = (float)rq[threadIdx.x];
            sk[threadIdx.x] = (float)rk[threadIdx.x];
        }
        __syncthreads();
        const float c = col < cols ? (float)((const T*)v.p + b * v.token_stride + head / v.share * v.head_stride)[col] : 0.0f;
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
        {
            const int r = NWAVES * i + wave;
            if (r < dim)
            {
                s[i] = fmaf(sk[r], c, decay.of(s[i]));
                x = fmaf(sq[r], s[i], x);
            }
        }
        part[wave][threadIdx.x % WAVE] = x;
        __syncthreads();
        store(b, scale * ((part[0][threadIdx.x % WAVE] + part[1][threadIdx.x % WAVE]) + (part[2][threadIdx.x % WAVE] + part[3][threadIdx.x % WAVE])));
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
    {
        const int row = NWAVES * i + wave;
        if (row < dim && col < cols) state[(int64_t)row * cols + col] = s[i];
    }
}

template <typename T>
hipError_t linear_attention_step(TokenRows q, TokenRows k, TokenRows v, const float* log_decay, float* states, int64_t slot_stride,
                                 int64_t head_stride, const void* slot_of, bool wide, int64_t slots, T* out, int64_t batch, int heads, int dim,
                                 int cols, float scale, hipStream_t stream)
{
    if (batch <= 0 || heads <= 0) return hipSuccess;
    const int tiles = (cols + WAVE - 1) / WAVE;
    attention_step_kernel<T><<<(unsigned)(batch * heads * tiles), BLOCK, 0, stream>>>(q, k, v, log_decay, states, slot_stride, head_stride,
                                                                                     slot_of, wide, slots, out, batch, heads, dim, cols, scale, tiles);
    return hipGetLastError();
}

#define MCA_ATTENTION(T)                                                                                                                       \
    template hipError_t sum_shared_heads<T>(const float*, T*, int64_t, int, int, int, hipStream_t);                                            \
    template hipError_t linear_attention_step<T>(TokenRows, TokenRows, TokenRows, const float*, float*, int64_t, int64_t, const void*, bool,   \
                                                 int64_t, T*, int64_t, int, int, int, float, hipStream_t)
MCA_ATTENTION(float);
MCA_ATTENTION(_Float16);
MCA_ATTENTION(__bf16);

}  // namespace mca
