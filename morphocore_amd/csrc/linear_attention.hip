// Linear attention with a decay for each head, over whole sequences (every pass of it, forwards or backwards in time, see
// Pass) and a token at a time:
//   S_t = d S_(t-1) + k_t v_t^T,  out_t = scale q_t S_t.
#include "block8.hpp"
#include "launch.hpp"
#include "tokens.hpp"

namespace mca
{

// Decays below exp(-16384) are 0 anyway, and times 0 must stay 0.
__device__ __forceinline__ float log_decay_of(const float* __restrict__ log_decay, int head)
{
    const float g = log_decay[head];
    return g < -16384.0f ? -16384.0f : g;
}

// A decay of one token in two float32 terms: one alone is off by up to 2^-25, the same way every token, which a state that keeps
// 1 - 2^-12 of itself adds up to 2^-13.
struct Decay
{
    float hi, lo;

    __device__ __forceinline__ explicit Decay(float log_decay)
    {
        const double d = exp((double)log_decay);
        hi = (float)d, lo = (float)(d - (double)hi);
    }
    __device__ __forceinline__ float of(float s) const { return fmaf(s, hi, s * lo); }
};

// A sequence's rows [start, start + length) and where its batch lies.
struct Rows1
{
    int64_t batch, start, length;
    bool none;  // rows of no sequence
};

__device__ __forceinline__ int64_t offset_at(const Sequences& s, int64_t i)
{
    const int64_t o = s.wide ? ((const int64_t*)s.offsets)[i] : (int64_t)((const int32_t*)s.offsets)[i];
    return o < 0 ? 0 : o > s.tokens ? s.tokens : o;
}

// Of packed sequences 0 is what lies before the first, count + 1 what lies behind the last.
__device__ __forceinline__ Rows1 sequence_rows(const Sequences& s, int64_t i)
{
    if (!s.offsets) return Rows1{i, 0, s.tokens, false};
    const int64_t a = i == 0 ? 0 : offset_at(s, i - 1), b = i == s.count + 1 ? s.tokens : offset_at(s, i);
    return Rows1{i - 1, a, b > a ? b - a : 0, i == 0 || i == s.count + 1};
}

inline int64_t sequence_count(const Sequences& s) { return s.offsets ? s.count + 2 : s.count; }

template <typename T>
__device__ __forceinline__ const T* row_at(const TokenRows& r, const Sequences& s, const Rows1& q, int64_t t, int head)
{
    return (const T*)r.p + (s.offsets ? 0 : q.batch * r.batch_stride) + (q.start + t) * r.token_stride + head / r.share * r.head_stride;
}

// 64 columns of one head of one sequence, token after token: a thread has every 4th row of its column's state.
template <typename T>
__global__ __launch_bounds__(BLOCK) void attention_rows_kernel(Sequences seq, int heads, const float* __restrict__ log_decay, Pass p, int tiles)
{
    constexpr int ROWS = 64;
    __shared__ float a[256], b[256], part[NWAVES][WAVE];
    const int tile = blockIdx.x % tiles, head = blockIdx.x / tiles % heads;
    const Rows1 q = sequence_rows(seq, blockIdx.x / tiles / heads);
    const int col = tile * WAVE + threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const Decay decay(log_decay_of(log_decay, head));
    const int64_t state0 = (q.batch * heads + head) * p.dim * p.cols;
    float s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
    {
        const int row = NWAVES * i + wave;
        s[i] = p.first.p && !q.none && row < p.dim && col < p.cols ? p.first.p[state0 + row * p.first.row_stride + col * p.first.col_stride] : 0.0f;
    }
    for (int64_t n = 0; n < q.length; ++n)
    {
        const int64_t t = p.backwards ? q.length - 1 - n : n;
        const int64_t row = (seq.offsets ? q.start : q.batch * seq.tokens) + t;
        float v = 0.0f;
        if (!q.none)
        {
            const T *ra = row_at<T>(p.a, seq, q, t, head), *rb = row_at<T>(p.b, seq, q, t, head);
            if ((int)threadIdx.x < p.dim)
            {
                a[threadIdx.x] = (float)ra[threadIdx.x];
                b[threadIdx.x] = p.update * (float)rb[threadIdx.x];
            }
            __syncthreads();
            const float c = col < p.cols ? (float)row_at<T>(p.c, seq, q, t, head)[col] : 0.0f;
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
            {
                const int r = NWAVES * i + wave;
                if (r < p.dim)
                {
                    if (!p.backwards) s[i] = decay.of(s[i]);
                    s[i] = fmaf(b[r], c, s[i]);
                    v = fmaf(a[r], s[i], v);
                    if (p.backwards) s[i] = decay.of(s[i]);
                }
            }
            part[wave][threadIdx.x % WAVE] = v;
            __syncthreads();
            v = p.read * ((part[0][threadIdx.x % WAVE] + part[1][threadIdx.x % WAVE]) + (part[2][threadIdx.x % WAVE] + part[3][threadIdx.x % WAVE]));
        }
        if (p.out && wave == 0 && col < p.cols)
        {
            const int64_t at = (row * heads + head) * p.cols + col;
            if (p.out32)
                p.out32[at] = v;
            else
                ((T*)p.out)[at] = (T)v;
        }
    }
    if (!p.last.p || q.none) return;
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
    {
        const int row = NWAVES * i + wave;
        if (row < p.dim && col < p.cols) p.last.p[state0 + row * p.last.row_stride + col * p.last.col_stride] = s[i];
    }
}

template <typename T>
size_t linear_attention_workspace(const Sequences&, int, const Pass*, int)
{
    return 0;
}

template <typename T>
hipError_t linear_attention(const Sequences& seq, int heads, const float* log_decay, const Pass* passes, int count, void*, hipStream_t stream)
{
    const int64_t n = sequence_count(seq) * heads;
    if (n <= 0) return hipSuccess;
    for (int i = 0; i < count; ++i)
    {
        const int tiles = (passes[i].cols + WAVE - 1) / WAVE;
        attention_rows_kernel<T><<<(unsigned)(n * tiles), BLOCK, 0, stream>>>(seq, heads, log_decay, passes[i], tiles);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

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
    const Decay decay(log_decay_of(log_decay, head));
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
    template size_t linear_attention_workspace<T>(const Sequences&, int, const Pass*, int);                                                    \
    template hipError_t linear_attention<T>(const Sequences&, int, const float*, const Pass*, int, void*, hipStream_t);                        \
    template hipError_t sum_shared_heads<T>(const float*, T*, int64_t, int, int, int, hipStream_t);                                            \
    template hipError_t linear_attention_step<T>(TokenRows, TokenRows, TokenRows, const float*, float*, int64_t, int64_t, const void*, bool,   \
                                                 int64_t, T*, int64_t, int, int, int, float, hipStream_t)
MCA_ATTENTION(float);
MCA_ATTENTION(_Float16);
MCA_ATTENTION(__bf16);

}  // namespace mca
