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

// Bound by HBM: the states are read once and written once, float32. A workgroup has 4 LC columns of one head's state in registers, 4
// neighbouring values a thread in every RB-th row, all loads in flight at once; q S is summed over a thread's rows, the lanes and
// the waves, in a fixed order. Rows of the batch that name the same slot are taken by the first of them, in order, the state staying
// where it is. Measured, 32 heads of 128 x 128 in bfloat16: 256 sequences in 231 us (4.65 TB/s of states read and written in place, where a
// copy reaches 5.05; stores past the caches are no faster), one in 5.6 (7.5 with its call).
// With places each workgroup looks through all of them for tokens of its own: 4 us of 256 sequences, but as much as the states of 4096 of 16
// heads of 64 x 64 (423 us without, 800 with).
template <typename T, int LC, int R>
__global__ __launch_bounds__(BLOCK, 4) void attention_step_kernel(TokenRows q, TokenRows k, TokenRows v, const float* __restrict__ log_decay,
                                                               float* __restrict__ states, int64_t slot_stride, int64_t head_stride,
                                                               const void* __restrict__ slot_of, bool wide, int64_t slots, T* __restrict__ out,
                                                               int64_t batch, int heads, int dim, int cols, float scale, int tiles)
{
    constexpr int RB = BLOCK / LC;
    static_assert(LC <= WAVE);
    __shared__ float sq[RB * R], sk[RB * R];
    __shared__ f32x4 part[NWAVES][LC];
    const int lane = threadIdx.x % LC, row0 = threadIdx.x / LC;
    auto slot_at = [&](int64_t b) -> int64_t {
        if (!slot_of) return b;
        return wide ? ((const int64_t*)slot_of)[b] : (int64_t)((const int32_t*)slot_of)[b];
    };
    const int64_t work = batch * heads * tiles;
    for (int64_t item = blockIdx.x; item < work; item += gridDim.x)
    {
        const int tile = (int)(item % tiles), head = (int)(item / tiles % heads);
        const int64_t first = item / tiles / heads, slot = slot_at(first);
        const int col = (tile * LC + lane) * 4, valid = min(max(cols - col, 0), 4);
        if (slot < 0 || slot >= slots)
        {
            if (threadIdx.x < LC)
                for (int j = 0; j < valid; ++j) out[(first * heads + head) * cols + col + j] = (T)0.0f;
            continue;
        }
        float* __restrict__ state = states + slot * slot_stride + head * head_stride + col;
        f32x4 s[R];
#pragma unroll
        for (int i = 0; i < R; ++i)
        {
            const int row = RB * i + row0;
            s[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (row >= dim) continue;
            if (valid == 4)
                __builtin_memcpy(&s[i], state + (int64_t)row * cols, 16);
            else
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    if (j < valid) s[i][j] = state[(int64_t)row * cols + j];
        }
        bool again = false;
        if (slot_of)
        {
            bool before = false, after = false;
            for (int64_t b = threadIdx.x; b < batch; b += BLOCK)
            {
                const bool same = b != first && slot_at(b) == slot;
                before |= same && b < first;
                after |= same && b > first;
            }
            if (__syncthreads_or(before)) continue;
            again = __syncthreads_or(after);
        }
        const Decay decay(log_decay_of(log_decay, head), 1);
        for (int64_t b = first; b < batch; ++b)
        {
            if (b > first && (!again || slot_at(b) != slot))
            {
                if (!again) break;
                continue;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < dim; i += BLOCK)
            {
                sq[i] = (float)((const T*)q.p + b * q.token_stride + head / q.share * q.head_stride)[i];
                sk[i] = (float)((const T*)k.p + b * k.token_stride + head / k.share * k.head_stride)[i];
            }
            const T* __restrict__ pv = (const T*)v.p + b * v.token_stride + head / v.share * v.head_stride + col;
            f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f}, x = c;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < valid) c[j] = (float)pv[j];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < R; ++i)
            {
                const int row = RB * i + row0;
                if (row >= dim) continue;
                const float a = sq[row], w = sk[row];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    s[i][j] = fmaf(w, c[j], decay.of(s[i][j]));
                    x[j] = fmaf(a, s[i][j], x[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int d = LC; d < WAVE; d *= 2) x[j] += __shfl_xor(x[j], d);
            if (threadIdx.x % WAVE < LC) part[threadIdx.x / WAVE][lane] = x;
            __syncthreads();
            if (threadIdx.x < LC)
            {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < valid)
                        out[(b * heads + head) * cols + col + j] =
                            (T)(scale * ((part[0][lane][j] + part[1][lane][j]) + (part[2][lane][j] + part[3][lane][j])));
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
        {
            const int row = RB * i + row0;
            if (row >= dim) continue;
            float* __restrict__ to = state + (int64_t)row * cols;
            if (valid == 4)
                __builtin_memcpy(to, &s[i], 16);
            else
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    if (j < valid) to[j] = s[i][j];
        }
    }
}

template <typename T>
hipError_t linear_attention_step(TokenRows q, TokenRows k, TokenRows v, const float* log_decay, float* states, int64_t slot_stride,
                                 int64_t head_stride, const void* slot_of, bool wide, int64_t slots, T* out, int64_t batch, int heads, int dim,
                                 int cols, float scale, hipStream_t stream)
{
    if (batch <= 0 || heads <= 0) return hipSuccess;
    auto run = [&](auto lc, auto r) {
        constexpr int LC = decltype(lc)::value, R = decltype(r)::value;
        const int tiles = (cols + 4 * LC - 1) / (4 * LC);
        const int64_t work = batch * heads * tiles, most = 1 << 20;
        attention_step_kernel<T, LC, R><<<(unsigned)(work < most ? work : most), BLOCK, 0, stream>>>(
            q, k, v, log_decay, states, slot_stride, head_stride, slot_of, wide, slots, out, batch, heads, dim, cols, scale, tiles);
        return hipGetLastError();
    };
    using std::integral_constant;
    auto by_rows = [&](auto lc) {
        constexpr int LC = decltype(lc)::value, RB = BLOCK / LC, MOST = 256 / RB;
        if constexpr (MOST >= 8)
        {
            if (dim <= RB * (MOST / 8)) return run(lc, integral_constant<int, MOST / 8>());
        }
        if (dim <= RB * (MOST / 4)) return run(lc, integral_constant<int, MOST / 4>());
        if (dim <= RB * (MOST / 2)) return run(lc, integral_constant<int, MOST / 2>());
        return run(lc, integral_constant<int, MOST>());
    };
    // Parts of 256 bytes of the state's rows where there are workgroups enough (256 states of 32 heads of 128 x 128 in 230 us, by whole rows of
    // 512 bytes in 272); of 128 bytes otherwise.
    if (cols > 32 && batch * heads >= 256) return by_rows(integral_constant<int, 16>());
    if (cols > 16) return by_rows(integral_constant<int, 8>());
    return by_rows(integral_constant<int, 4>());
}

#define MCA_ATTENTION(T)                                                                                                                       \
    template hipError_t sum_shared_heads<T>(const float*, T*, int64_t, int, int, int, hipStream_t);                                            \
    template hipError_t linear_attention_step<T>(TokenRows, TokenRows, TokenRows, const float*, float*, int64_t, int64_t, const void*, bool,   \
                                                 int64_t, T*, int64_t, int, int, int, float, hipStream_t)
MCA_ATTENTION(float);
MCA_ATTENTION(_Float16);
MCA_ATTENTION(__bf16);

}  // namespace mca
