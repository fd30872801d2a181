// 8-bit blocks on their own (pack8, unpack8) and the gated activation y = g * sigmoid(g) * u, whose forward
// writes the 8-bit form of g and u for the backward, and of y for the weight gradient of the layer that
// reads it:
//   grad_g = grad_y * u * s * (1 + g * (1 - s)),  grad_u = grad_y * g * s,  s = sigmoid(g).
//
// Bound by HBM: one pass, 8 values a lane (16-byte accesses of 16-bit values). A workgroup's 256 lanes take as
// many whole rows as they hold, a lane a unit (a multiple of 4 lanes a row, so that a block's lanes stay
// together); a row of more than 256 units takes several workgroups (blockIdx.x), so that one row already
// fills many CUs. Lanes a power of two at or above the row's units were 19 to 25% slower for widths between
// (100000 x 300 bfloat16: pack8 25 us, 19 with whole rows) and no faster at others. Copies run at 5.2 TB/s read
// and written; measured, bfloat16: pack8 of 16384 x 8192 82 us (4.9 TB/s), unpack8 67 us (6.0), gated_silu8 of
// 8192 x 8192 forward 111 us (5.4), backward 93 us (5.8); 257 x 1021 float32: 3 us each.
#include "block8.hpp"
#include "launch.hpp"
#include "mixer.hpp"

namespace mca
{

struct RowGrid
{
    dim3 grid;
    int lanes;
    int magic;  // ceil(2^16 / lanes): t / lanes = t * magic >> 16 for t < 256
};

// Rows beyond the grid are taken in the kernels' loop.
static RowGrid row_grid(int64_t rows, int cols)
{
    const int units = blocks_of(cols) * MX_LANES, chunks = (units + BLOCK - 1) / BLOCK;
    const int lanes = ((units + chunks - 1) / chunks + MX_LANES - 1) / MX_LANES * MX_LANES;
    const int64_t per = BLOCK / lanes, y = (rows + per - 1) / per, most = 65535;
    return RowGrid{dim3((unsigned)chunks, (unsigned)(y < most ? y : most)), lanes, (65535 + lanes) / lanes};
}

// The lane's unit of its row, and the loop over the rows.
#define MCA_ROW_LOOP(unit, row)                                                             \
    const int own_row = (int)threadIdx.x * magic >> 16, rows_per = BLOCK * magic >> 16;     \
    const int unit = (int)blockIdx.x * lanes + (int)threadIdx.x - own_row * lanes;          \
    if (unit >= blocks_of(cols) * MX_LANES || own_row >= rows_per) return;                  \
    for (int64_t row = (int64_t)blockIdx.y * rows_per + own_row; row < rows; row += (int64_t)gridDim.y * rows_per)

template <typename T>
__global__ __launch_bounds__(BLOCK) void pack8_kernel(const T* __restrict__ x, int64_t xs, uint8_t* __restrict__ codes,
                                                      uint8_t* __restrict__ scales, int64_t rows, int cols, int lanes, int magic)
{
    const int nb = blocks_of(cols);
    MCA_ROW_LOOP(unit, row)
    {
        const int c = unit * UNIT, valid = cols - c;
        float v[UNIT];
        load_unit(x + row * xs + c, c, valid, v);
        store_packed(codes + row * cols, scales + row * nb, unit, valid, v);
    }
}

// float16 holds less than the packed values: those beyond its largest saturate.
template <typename T>
__device__ __forceinline__ void saturate_unit(float (&v)[UNIT])
{
    if constexpr (std::is_same_v<T, _Float16>)
    {
#pragma unroll
        for (int j = 0; j < UNIT; ++j)
            if (v[j] == v[j]) v[j] = fminf(fmaxf(v[j], -65504.0f), 65504.0f);
    }
}

template <typename T>
__global__ __launch_bounds__(BLOCK) void unpack8_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                        T* __restrict__ out, int64_t rows, int cols, int lanes, int magic, bool streaming)
{
    const int nb = blocks_of(cols);
    MCA_ROW_LOOP(unit, row)
    {
        const int c = unit * UNIT, valid = cols - c;
        if (valid <= 0) continue;
        float v[UNIT];
        unpack_unit(load_codes(codes + row * cols + c, c, valid), scale_of(scales[row * nb + unit / MX_LANES]), v);
        saturate_unit<T>(v);
        // (A lane's 8 float32 values are two stores, which past the caches write half lines: 46 us for 26.)
        store_unit(out + row * cols + c, valid, v, streaming && sizeof(T) == 2);
    }
}

template <typename T>
__global__ __launch_bounds__(BLOCK) void copy_rows_kernel(const T* __restrict__ x, int64_t xs, T* __restrict__ out, int64_t rows, int cols,
                                                          int lanes, int magic)
{
    MCA_ROW_LOOP(unit, row)
    {
        const int c = unit * UNIT, valid = cols - c;
        float v[UNIT] = {};
        if (x) load_unit(x + row * xs + c, c, valid, v);
        store_unit(out + row * cols + c, valid, v);
    }
}

// The library's exponential for float32; the hardware's, whose error grows with the argument to a few
// float32 units in the last place, where the result is rounded to 16 bits (y of 8192 x 8192 bfloat16 is as far from
// float64 with either, 0.00165; with the library's, gated_silu8 of it takes 119 us for 110, of 1999 x 2731 float16 14.4
// for 13.1). g * sigmoid rounds once more in float32 than g / (1 + e) would (y 4.9e-8 from float64 for 4.6e-8), whose
// division takes gated_silu8 of 8192 x 8192 float32 from 176 to 186 us.
template <typename T>
__device__ __forceinline__ float sigmoid_of(float g)
{
    const float e = std::is_same_v<T, float> ? expf(-g) : __expf(-g);
    return 1.0f / (1.0f + e);
}

template <typename T>
__global__ __launch_bounds__(BLOCK) void gated_silu_fwd_kernel(const T* __restrict__ gate, int64_t gs, const T* __restrict__ up, int64_t us,
                                                               T* __restrict__ y, PackedOut g8, PackedOut u8, PackedOut y8, int64_t rows,
                                                               int cols, int lanes, int magic, bool streaming)
{
    const int nb = blocks_of(cols);
    MCA_ROW_LOOP(unit, row)
    {
        const int c = unit * UNIT, valid = cols - c;
        float g[UNIT], u[UNIT], v[UNIT];
        load_unit(gate + row * gs + c, c, valid, g);
        load_unit(up + row * us + c, c, valid, u);
        if (g8.codes) store_packed(g8.codes + row * cols, g8.scales + row * nb, unit, valid, g);
        if (u8.codes) store_packed(u8.codes + row * cols, u8.scales + row * nb, unit, valid, u);
#pragma unroll
        for (int j = 0; j < UNIT; ++j) v[j] = g[j] * sigmoid_of<T>(g[j]) * u[j];
        store_unit(y + row * cols + c, valid, v, streaming);
        if (y8.codes)
        {
            round_unit<T>(v);  // the 8-bit form is y's, as stored
            store_packed(y8.codes + row * cols, y8.scales + row * nb, unit, valid, v);
        }
    }
}

template <typename T, bool PACKED>
__global__ __launch_bounds__(BLOCK) void gated_silu_bwd_kernel(const T* __restrict__ gy, int64_t gys, const T* __restrict__ gate, int64_t gs,
                                                               const T* __restrict__ up, int64_t us, PackedOut g8, PackedOut u8,
                                                               T* __restrict__ gg, T* __restrict__ gu, int64_t grad_s, int64_t rows, int cols,
                                                               int lanes, int magic, bool streaming)
{
    const int nb = blocks_of(cols);
    MCA_ROW_LOOP(unit, row)
    {
        const int c = unit * UNIT, valid = cols - c;
        if (valid <= 0) continue;
        float d[UNIT], g[UNIT], u[UNIT];
        load_unit(gy + row * gys + c, c, valid, d);
        if constexpr (PACKED)
        {
            const int64_t at = row * cols + c, block = row * nb + unit / MX_LANES;
            unpack_unit(load_codes(g8.codes + at, c, valid), scale_of(g8.scales[block]), g);
            unpack_unit(load_codes(u8.codes + at, c, valid), scale_of(u8.scales[block]), u);
        }
        else
        {
            load_unit(gate + row * gs + c, c, valid, g);
            load_unit(up + row * us + c, c, valid, u);
        }
#pragma unroll
        for (int j = 0; j < UNIT; ++j)
        {
            const float s = sigmoid_of<T>(g[j]);
            u[j] = d[j] * u[j] * (s * (1.0f + g[j] * (1.0f - s)));
            g[j] = d[j] * g[j] * s;
        }
        store_unit(gg + row * grad_s + c, valid, u, streaming);
        store_unit(gu + row * grad_s + c, valid, g, streaming);
    }
}

template <typename T>
hipError_t pack8(const T* x, int64_t x_stride, uint8_t* codes, uint8_t* scales, int64_t rows, int cols, hipStream_t stream)
{
    if (rows <= 0 || cols <= 0) return hipSuccess;
    const RowGrid g = row_grid(rows, cols);
    pack8_kernel<T><<<g.grid, BLOCK, 0, stream>>>(x, x_stride, codes, scales, rows, cols, g.lanes, g.magic);
    return hipGetLastError();
}

template <typename T>
hipError_t unpack8(const uint8_t* codes, const uint8_t* scales, T* out, int64_t rows, int cols, hipStream_t stream)
{
    if (rows <= 0 || cols <= 0) return hipSuccess;
    const RowGrid g = row_grid(rows, cols);
    unpack8_kernel<T><<<g.grid, BLOCK, 0, stream>>>(codes, scales, out, rows, cols, g.lanes, g.magic,
                                                      streams((double)rows * cols * (sizeof(T) + 1)));
    return hipGetLastError();
}

template <typename T>
hipError_t copy_rows(const T* x, int64_t x_stride, T* out, int64_t rows, int cols, hipStream_t stream)
{
    if (rows <= 0 || cols <= 0) return hipSuccess;
    const RowGrid g = row_grid(rows, cols);
    copy_rows_kernel<T><<<g.grid, BLOCK, 0, stream>>>(x, x_stride, out, rows, cols, g.lanes, g.magic);
    return hipGetLastError();
}

template <typename T>
hipError_t gated_silu_forward(const T* gate, int64_t g_stride, const T* up, int64_t u_stride, T* y, PackedOut gate8, PackedOut up8,
                              PackedOut y8, int64_t rows, int cols, hipStream_t stream)
{
    if (rows <= 0 || cols <= 0) return hipSuccess;
    const RowGrid g = row_grid(rows, cols);
    gated_silu_fwd_kernel<T><<<g.grid, BLOCK, 0, stream>>>(gate, g_stride, up, u_stride, y, gate8, up8, y8, rows, cols, g.lanes, g.magic,
                                                          streams((double)rows * cols * (3 * sizeof(T) + !!gate8.codes + !!up8.codes + !!y8.codes)));
    return hipGetLastError();
}

template <typename T>
hipError_t gated_silu_backward(const T* grad_y, int64_t gy_stride, const T* gate, int64_t g_stride, const T* up, int64_t u_stride,
                               PackedOut gate8, PackedOut up8, T* grad_gate, T* grad_up, int64_t grad_stride, int64_t rows, int cols,
                               hipStream_t stream)
{
    if (rows <= 0 || cols <= 0) return hipSuccess;
    const RowGrid g = row_grid(rows, cols);
    const bool streaming = streams((double)rows * cols * (gate ? 5 * sizeof(T) : 3 * sizeof(T) + 2));
    if (gate)
        gated_silu_bwd_kernel<T, false><<<g.grid, BLOCK, 0, stream>>>(grad_y, gy_stride, gate, g_stride, up, u_stride, gate8, up8, grad_gate,
                                                                      grad_up, grad_stride, rows, cols, g.lanes, g.magic, streaming);
    else
        gated_silu_bwd_kernel<T, true><<<g.grid, BLOCK, 0, stream>>>(grad_y, gy_stride, gate, g_stride, up, u_stride, gate8, up8, grad_gate,
                                                                     grad_up, grad_stride, rows, cols, g.lanes, g.magic, streaming);
    return hipGetLastError();
}

#define MCA_GATED(T)                                                                                                                    \
    template hipError_t pack8<T>(const T*, int64_t, uint8_t*, uint8_t*, int64_t, int, hipStream_t);                                     \
    template hipError_t unpack8<T>(const uint8_t*, const uint8_t*, T*, int64_t, int, hipStream_t);                                      \
    template hipError_t copy_rows<T>(const T*, int64_t, T*, int64_t, int, hipStream_t);                                                 \
    template hipError_t gated_silu_forward<T>(const T*, int64_t, const T*, int64_t, T*, PackedOut, PackedOut, PackedOut, int64_t, int,  \
                                              hipStream_t);                                                                             \
    template hipError_t gated_silu_backward<T>(const T*, int64_t, const T*, int64_t, const T*, int64_t, PackedOut, PackedOut, T*, T*,   \
                                               int64_t, int64_t, int, hipStream_t)
MCA_GATED(float);
MCA_GATED(_Float16);
MCA_GATED(__bf16);

}  // namespace mca
