// The weight gradient of a linear layer from its packed input:
//   grad_weight[n, k] = sum over the rows m of grad_y[m, n] * value(codes[m, k]).
#include "block8.hpp"
#include "launch.hpp"
#include "mixer.hpp"

namespace mca
{

constexpr int TILE_N = 64, TILE_K = 64, TILE_M = 32;
// Rows a split sums at least: below them the joining of the splits costs more than the products.
constexpr int SPLIT_ROWS = 256;

template <typename T>
__global__ __launch_bounds__(BLOCK) void grad_weight8_kernel(const T* __restrict__ gy, int64_t gys, const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales, float* __restrict__ part, int64_t rows,
                                                             int64_t split_rows, int out, int cols)
{
    __shared__ float a[TILE_M][TILE_N], b[TILE_M][TILE_K];
    const int n0 = blockIdx.x * TILE_N, k0 = blockIdx.y * TILE_K, nb = blocks_of(cols);
    const int tn = threadIdx.x / 16 * 4, tk = threadIdx.x % 16 * 4;
    const int64_t m0 = blockIdx.z * split_rows, m1 = m0 + split_rows < rows ? m0 + split_rows : rows;
    float acc[4][4] = {};
    for (int64_t m = m0; m < m1; m += TILE_M)
    {
        const int r = threadIdx.x / 8, c = threadIdx.x % 8 * UNIT;
        const bool in = m + r < m1;
        float v[UNIT];
        load_unit(gy + (m + r) * gys + n0 + c, in ? out - n0 - c : 0, v);
#pragma unroll
        for (int j = 0; j < UNIT; ++j) a[r][c + j] = v[j];
        const int valid = in ? cols - k0 - c : 0;
        const uint2 code = load_codes(codes + (m + r) * cols + k0 + c, valid);
        unpack_unit(code, valid > 0 ? scale_of(scales[(m + r) * nb + (k0 + c) / MX_BLOCK]) : 1.0f, v);
#pragma unroll
        for (int j = 0; j < UNIT; ++j) b[r][c + j] = v[j];
        __syncthreads();
        for (int i = 0; i < TILE_M; ++i)
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[p][q] += a[i][tn + p] * b[i][tk + q];
        __syncthreads();
    }
    float* __restrict__ o = part + (int64_t)blockIdx.z * out * cols;
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (n0 + tn + p < out && k0 + tk + q < cols) o[(int64_t)(n0 + tn + p) * cols + k0 + tk + q] = acc[p][q];
}

struct WeightPlan
{
    dim3 grid;
    int64_t split_rows;
    int splits;
};

static WeightPlan weight_plan(int64_t rows, int out, int cols)
{
    const int64_t tiles = (int64_t)((out + TILE_N - 1) / TILE_N) * ((cols + TILE_K - 1) / TILE_K);
    int64_t splits = 1024 / tiles, most = (rows + SPLIT_ROWS - 1) / SPLIT_ROWS;
    splits = splits < 1 ? 1 : splits;
    splits = splits < most ? splits : most;
    int64_t per = (rows + splits - 1) / splits;
    per = (per + TILE_M - 1) / TILE_M * TILE_M;
    splits = (rows + per - 1) / per;
    return WeightPlan{dim3((out + TILE_N - 1) / TILE_N, (cols + TILE_K - 1) / TILE_K, (unsigned)splits), per, (int)splits};
}

template <typename T>
size_t grad_weight8_workspace(int64_t rows, int out, int cols)
{
    if (rows <= 0 || out <= 0 || cols <= 0) return 0;
    return align_up((size_t)weight_plan(rows, out, cols).splits * out * cols * sizeof(float));
}

template <typename T, typename OT>
hipError_t grad_weight8(const T* grad_y, int64_t gy_stride, const uint8_t* codes, const uint8_t* scales, OT* grad_weight, int64_t rows,
                        int out, int cols, void* workspace, hipStream_t stream)
{
    if (out <= 0 || cols <= 0) return hipSuccess;
    if (rows <= 0) return sum_slots_async<OT>(nullptr, 0, (int64_t)out * cols, grad_weight, stream);
    const WeightPlan p = weight_plan(rows, out, cols);
    grad_weight8_kernel<T><<<p.grid, BLOCK, 0, stream>>>(grad_y, gy_stride, codes, scales, (float*)workspace, rows, p.split_rows, out, cols);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    return sum_slots_async<OT>((const float*)workspace, p.splits, (int64_t)out * cols, grad_weight, stream);
}

// Q threads a group of 4 columns, each summing every Q-th slot; their sums are added in thread order.
template <typename OT, int Q>
__global__ __launch_bounds__(BLOCK) void sum_slots_kernel(const float* __restrict__ part, int nslots, int64_t n, OT* __restrict__ out)
{
    constexpr int GROUPS = BLOCK / Q;
    __shared__ Acc sums[Q][GROUPS][4];
    const int g = threadIdx.x % GROUPS, q = threadIdx.x / GROUPS;
    const int64_t j = ((int64_t)blockIdx.x * GROUPS + g) * 4;
    Acc s[4] = {};
    if (j < n)
        for (int b = q; b < nslots; b += Q)
        {
            const float* __restrict__ p = part + (int64_t)b * n + j;
            float v[4];
            if (j + 4 <= n)
            {
                __builtin_memcpy(v, p, sizeof(v));
            }
            else
            {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = j + k < n ? p[k] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += (Acc)v[k];
        }
    if constexpr (Q > 1)
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[q][g][k] = s[k];
        __syncthreads();
        if (q != 0) return;
        for (int i = 1; i < Q; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += sums[i][g][k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (j + k < n) out[j + k] = (OT)s[k];
}

template <typename OT>
hipError_t sum_slots_async(const float* part, int nslots, int64_t n, OT* out, hipStream_t stream)
{
    if (n <= 0) return hipSuccess;
    if (nslots <= 16)
        sum_slots_kernel<OT, 1><<<(unsigned)((n + 4 * BLOCK - 1) / (4 * BLOCK)), BLOCK, 0, stream>>>(part, nslots, n, out);
    else
        sum_slots_kernel<OT, 32><<<(unsigned)((n + 31) / 32), BLOCK, 0, stream>>>(part, nslots, n, out);
    return hipGetLastError();
}

template hipError_t sum_slots_async<float>(const float*, int, int64_t, float*, hipStream_t);
template hipError_t sum_slots_async<_Float16>(const float*, int, int64_t, _Float16*, hipStream_t);
template hipError_t sum_slots_async<__bf16>(const float*, int, int64_t, __bf16*, hipStream_t);

#define MCA_WEIGHT(T, OT)                                                                                                             \
    template hipError_t grad_weight8<T, OT>(const T*, int64_t, const uint8_t*, const uint8_t*, OT*, int64_t, int, int, void*, hipStream_t)
template size_t grad_weight8_workspace<float>(int64_t, int, int);
template size_t grad_weight8_workspace<_Float16>(int64_t, int, int);
template size_t grad_weight8_workspace<__bf16>(int64_t, int, int);
MCA_WEIGHT(float, float);
MCA_WEIGHT(_Float16, _Float16);
MCA_WEIGHT(_Float16, float);
MCA_WEIGHT(__bf16, __bf16);
MCA_WEIGHT(__bf16, float);

}  // namespace mca
