// Root-mean-square norm of rows, with the residual's addition and the output's 8-bit form:
//   h = x (+ residual),  rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * w,
// and its gradients, with n = h * rstd and a = grad_y * w:
//   grad_x = grad_residual = rstd * (a - n * mean(a * n)) + grad_h,  grad_w = sum over the rows of grad_y * n.
//
// Bound by HBM: every operand is read once and every result written once. A row lies in the registers of G
// lanes, V units each, between its sum and its scaling; G follows the row's width (a few lanes for rows of
// an image's channels, so that a wave carries several rows; a workgroup for wide ones), so that a lane holds
// one unit where that is possible: registers are what limits the waves, and waves are what keeps loads in
// flight (loading a row ahead instead was slower). Copies of this size run at 5.2 TB/s read and written.
// Measured in training steps, bfloat16 with a residual and the 8-bit form: 8192 x 4096 forward 55 us (5.5 TB/s; 46
// alone, launched back to back), backward 56 us (4.8) and 7 for grad_w's slots (50 alone, with them); float32 without,
// 524288 x 64: 54 us (5.0) and 66 us (6.1, part of it from the cache) and 6. One row of 4096: 3.3 us.
//
// The forward normalises the float32 sum x + residual, not its rounded h (one rounding fewer), sums the squares in
// float64 and rounds y once: of float32 it is the correctly rounded value but for 2^-42, and of 16 bits hardly ever another
// one's neighbour, whose 8-bit code may be another too. (Float32 sums moved a few y in 100000 across a rounding boundary of 16 bits. The
// wider ones cost nothing up to 4096 columns, 1 us of 28 at 2048 x 8192 bfloat16 and 2 of 52 at 2048 x 16384.)
// The backward reads h as stored: x and the residual again would be a quarter more to read and a tensor
// more to keep, for a bfloat16 grad_w that is 0.0017 from the exact one, its own rounding, instead of 0.0025 (float16
// 0.00021 instead of 0.00031). grad_x, where h's rounding enters through n's share alone, is as near as with the exact h.
#include "block8.hpp"
#include "launch.hpp"
#include "mixer.hpp"

namespace mca
{

// Rows up to this many units (16384 values) stay in registers; wider ones are read twice.
constexpr int NORM_MAX_UNITS = 2048;
// Workgroups of a forward launch; the rest of the rows in their loop, which reads the weight once.
constexpr int NORM_BLOCKS = 4096;

constexpr int NUM_CU = 256;

// A workgroup has one row of more than a wave, or the rows of 4 waves.
template <int G>
constexpr int norm_threads()
{
    return G > WAVE ? G : BLOCK;
}

// The workgroup's row of a lane, in a scalar register where a wave has only one.
template <int G>
__device__ __forceinline__ int row_of_lane()
{
    if constexpr (G > WAVE) return 0;
    if constexpr (G == WAVE) return __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    return threadIdx.x / G;
}

// A sum (float or double) as the 32-bit registers that lane exchanges move.
template <typename S>
struct Words
{
    static constexpr int N = sizeof(S) / 4;
    uint32_t w[N];
};

template <int CTRL, typename S>
__device__ __forceinline__ S dpp_add(S s)
{
    Words<S> a = __builtin_bit_cast(Words<S>, s);
#pragma unroll
    for (int i = 0; i < a.N; ++i) a.w[i] = (uint32_t)__builtin_amdgcn_mov_dpp((int)a.w[i], CTRL, 0xf, 0xf, true);
    return s + __builtin_bit_cast(S, a);
}

template <bool HALVES, typename S>
__device__ __forceinline__ S swap_add(S s)
{
    Words<S> a = __builtin_bit_cast(Words<S>, s), b = a;
#pragma unroll
    for (int i = 0; i < a.N; ++i)
    {
        const auto t = HALVES ? __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false) : __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
        a.w[i] = t[0], b.w[i] = t[1];
    }
    return __builtin_bit_cast(S, a) + __builtin_bit_cast(S, b);
}

// The sum over G consecutive lanes (a power of two up to the wave), in every one of them, on the vector unit.
template <int G, typename S>
__device__ __forceinline__ S lane_sum(S s)
{
    if constexpr (G > 1) s = dpp_add<0xb1>(s);   // lane ^ 1
    if constexpr (G > 2) s = dpp_add<0x4e>(s);   // lane ^ 2
    if constexpr (G > 4) s = dpp_add<0x141>(s);  // the other 4 of 8 (mirrored)
    if constexpr (G > 8) s = dpp_add<0x140>(s);  // the other 8 of 16 (mirrored)
    if constexpr (G > 16) s = swap_add<false>(s);
    if constexpr (G > 32) s = swap_add<true>(s);
    return s;
}

// The sum over the G lanes of a row, in every one of them. `part` holds one value per wave, for two rows in
// turn (`turn`), so that one barrier a row suffices.
template <int G, typename S>
__device__ __forceinline__ S row_sum(S s, S* part, int turn)
{
    s = lane_sum<(G < WAVE ? G : WAVE)>(s);
    if constexpr (G > WAVE)
    {
        constexpr int N = G / WAVE;
        S* p = part + turn * N;
        if (threadIdx.x % WAVE == 0) p[threadIdx.x / WAVE] = s;
        __syncthreads();
        s = S(0);
#pragma unroll
        for (int i = 0; i < N; ++i) s += p[i];
    }
    return s;
}

// 1 / sqrt(sum * inv + eps) in two float32 terms: the rounded value, and a Newton step of what it misses. (0 where
// that says nothing: an infinite or zero mean square.)
struct TwoTerms
{
    float hi, lo;
};

__device__ __forceinline__ TwoTerms rstd_of(double sum, double inv, float eps)
{
    const double mean = sum * inv + (double)eps;
    const float a = (float)mean, al = (float)(mean - (double)a), q = 1.0f / sqrtf(a);
    const float t = q * a, tl = fmaf(q, al, fmaf(q, a, -t));
    const float miss = fmaf(-q, tl, fmaf(-q, t, 1.0f));  // 1 - q^2 mean
    return TwoTerms{q, fabsf(miss) < 0x1p-10f ? 0.5f * q * miss : 0.0f};
}

// v q w with one rounding at the end: the products' errors go along. Two roundings would move a value across a
// rounding boundary of 16 or 8 bits several times as often. Where the errors make a NaN (0 or an infinity of the other sign
// times an infinite weight) they are left out; the products alone make one only where v q w is one.
__device__ __forceinline__ float scaled(float v, TwoTerms q, float w)
{
    const float n = v * q.hi;
    const float y = fmaf(n, w, fmaf(v, q.lo, fmaf(v, q.hi, -n)) * w);
    return y == y ? y : n * w;
}

// A lane's values of a row as stored.
template <typename T, int G, int V>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int cols, RawUnit<T> (&raw)[V])
{
#pragma unroll
    for (int k = 0; k < V; ++k)
    {
        const int c = (threadIdx.x % G + G * k) * UNIT;
        load_raw(row + c, c, cols - c, raw[k]);
    }
}

template <typename T, typename WT, int G, int V>
__global__ __launch_bounds__(norm_threads<G>()) void rms_norm_fwd_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ r,
                                                                         int64_t rs, const WT* __restrict__ w, float eps, T* __restrict__ y,
                                                                         T* __restrict__ h, uint8_t* __restrict__ codes,
                                                                         uint8_t* __restrict__ scales, float* __restrict__ rstd, int64_t rows,
                                                                         int cols, bool streaming)
{
    constexpr int ROWS = norm_threads<G>() / G;
    __shared__ double part[2 * (G > WAVE ? G / WAVE : 1)];
    const int lane = threadIdx.x % G, nb = blocks_of(cols);
    const double inv = 1.0 / (double)cols;
    RawUnit<WT> wv[V];
    load_row<WT, G, V>(w, cols, wv);
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + row_of_lane<G>(); row < rows; row += (int64_t)gridDim.x * ROWS, turn ^= 1)
    {
        RawUnit<T> rx[V], rr[V];
        load_row<T, G, V>(x + row * xs, cols, rx);
        if (r) load_row<T, G, V>(r + row * rs, cols, rr);
        float v[V][UNIT];
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int j = 0; j < UNIT; ++j)
            {
                v[k][j] = rx[k][j];
                if (r) v[k][j] += rr[k][j];
                s = fma((double)v[k][j], (double)v[k][j], s);
            }
        const TwoTerms q = rstd_of(row_sum<G>(s, part, turn), inv, eps);
        if (rstd && lane == 0) rstd[row] = q.hi;
#pragma unroll
        for (int k = 0; k < V; ++k)
        {
            const int c = (lane + G * k) * UNIT, valid = cols - c;
            if (h) store_unit(h + row * cols + c, valid, v[k], streaming);
#pragma unroll
            for (int j = 0; j < UNIT; ++j) v[k][j] = scaled(v[k][j], q, wv[k][j]);
            if (y) store_unit(y + row * cols + c, valid, v[k], streaming);
            if (codes)
            {
                round_unit<T>(v[k]);  // the 8-bit form is y's, as stored
                store_packed(codes + row * cols, scales + row * nb, lane + G * k, valid, v[k]);
            }
        }
    }
}

// The same for rows of any width, one workgroup a row, the row read once for its sum and again to scale.
template <typename T, typename WT>
__global__ __launch_bounds__(1024) void rms_norm_fwd_wide_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ r, int64_t rs,
                                                                 const WT* __restrict__ w, float eps, T* __restrict__ y, T* __restrict__ h,
                                                                 uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                 float* __restrict__ rstd, int64_t rows, int cols, bool streaming)
{
    constexpr int G = 1024;
    __shared__ double part[2 * G / WAVE];
    const int nb = blocks_of(cols), padded = nb * MX_LANES;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1)
    {
        const T* __restrict__ xr = x + row * xs;
        const T* __restrict__ rr = r ? r + row * rs : nullptr;
        auto load = [&](int unit, float(&v)[UNIT]) {
            const int c = unit * UNIT;
            load_unit(xr + c, c, cols - c, v);
            if (rr)
            {
                float u[UNIT];
                load_unit(rr + c, c, cols - c, u);
#pragma unroll
                for (int j = 0; j < UNIT; ++j) v[j] += u[j];
            }
        };
        double s = 0.0;
        for (int unit = threadIdx.x; unit < padded; unit += G)
        {
            float v[UNIT];
            load(unit, v);
#pragma unroll
            for (int j = 0; j < UNIT; ++j) s = fma((double)v[j], (double)v[j], s);
        }
        const TwoTerms q = rstd_of(row_sum<G>(s, part, turn), 1.0 / (double)cols, eps);
        if (rstd && threadIdx.x == 0) rstd[row] = q.hi;
        for (int unit = threadIdx.x; unit < padded; unit += G)  // whole blocks: their lanes stay together
        {
            const int c = unit * UNIT, valid = cols - c;
            float v[UNIT], wv[UNIT];
            load(unit, v);
            load_unit(w + c, c, valid, wv);
            if (h) store_unit(h + row * cols + c, valid, v, streaming);
#pragma unroll
            for (int j = 0; j < UNIT; ++j) v[j] = scaled(v[j], q, wv[j]);
            if (y) store_unit(y + row * cols + c, valid, v, streaming);
            if (codes)
            {
                round_unit<T>(v);
                store_packed(codes + row * cols, scales + row * nb, unit, valid, v);
            }
        }
    }
}

// grad_x, and grad_w's sums over the workgroup's rows: lane sums over its rows in registers, then over the
// row groups of the workgroup in lane and wave order, into slot blockIdx.x of `part` (a fixed order, the same
// from run to run).
template <typename T, typename WT, int G, int V>
__global__ __launch_bounds__(norm_threads<G>()) void rms_norm_bwd_kernel(const T* __restrict__ gy, int64_t gys, const T* __restrict__ gh,
                                                                         int64_t ghs, const T* __restrict__ h, int64_t hs,
                                                                         const WT* __restrict__ w, const float* __restrict__ rstd,
                                                                         T* __restrict__ gx, float* __restrict__ gw_part, int64_t rows, int cols,
                                                                         bool streaming)
{
    constexpr int THREADS = norm_threads<G>(), ROWS = THREADS / G;
    __shared__ float part[2 * (G > WAVE ? G / WAVE : 1)];
    const int lane = threadIdx.x % G;
    const float inv = 1.0f / (float)cols;
    RawUnit<WT> wv[V];
    load_row<WT, G, V>(w, cols, wv);
    float gw[V][UNIT] = {};
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + row_of_lane<G>(); row < rows; row += (int64_t)gridDim.x * ROWS, turn ^= 1)
    {
        RawUnit<T> rh[V], ry[V], rg[V];
        load_row<T, G, V>(h + row * hs, cols, rh);
        load_row<T, G, V>(gy + row * gys, cols, ry);
        if (gh && gx) load_row<T, G, V>(gh + row * ghs, cols, rg);
        const float q = rstd[row];
        float n[V][UNIT], a[V][UNIT];
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int j = 0; j < UNIT; ++j)
            {
                const float g = ry[k][j];
                n[k][j] = rh[k][j] * q;
                gw[k][j] += g * n[k][j];
                a[k][j] = g * wv[k][j];
                s += a[k][j] * n[k][j];
                // What of grad_x needs no row sum; the rest is n's share of it.
                a[k][j] *= q;
                if (gh && gx) a[k][j] += rg[k][j];
            }
        if (!gx) continue;
        const float m = row_sum<G>(s, part, turn) * inv * q;
#pragma unroll
        for (int k = 0; k < V; ++k)
        {
            const int c = (lane + G * k) * UNIT;
#pragma unroll
            for (int j = 0; j < UNIT; ++j) a[k][j] -= n[k][j] * m;
            store_unit(gx + row * cols + c, cols - c, a[k], streaming);
        }
    }
    if (!gw_part) return;
    float* __restrict__ out = gw_part + (int64_t)blockIdx.x * cols;
    if constexpr (G > WAVE)
    {
#pragma unroll
        for (int k = 0; k < V; ++k)
        {
            const int c = (lane + G * k) * UNIT;
            store_unit(out + c, cols - c, gw[k]);
        }
    }
    else
    {
        constexpr int L = G < WAVE ? G : WAVE;  // lanes of a wave that hold distinct columns
        __shared__ float sums[NWAVES][V][L][UNIT];
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int j = 0; j < UNIT; ++j)
            {
                float t = gw[k][j];
#pragma unroll
                for (int d = L; d < WAVE; d *= 2) t += __shfl_xor(t, d);
                if (threadIdx.x % WAVE < L) sums[threadIdx.x / WAVE][k][threadIdx.x % L][j] = t;
            }
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += THREADS)
        {
            const int unit = c / UNIT, k = unit / G, l = unit % G, j = c % UNIT;
            out[c] = ((sums[0][k][l][j] + sums[1][k][l][j]) + sums[2][k][l][j]) + sums[3][k][l][j];
        }
    }
}

// grad_x of rows of any width, one workgroup a row, read twice.
template <typename T, typename WT>
__global__ __launch_bounds__(1024) void rms_norm_bwd_wide_kernel(const T* __restrict__ gy, int64_t gys, const T* __restrict__ gh, int64_t ghs,
                                                                 const T* __restrict__ h, int64_t hs, const WT* __restrict__ w,
                                                                 const float* __restrict__ rstd, T* __restrict__ gx, int64_t rows, int cols, bool streaming)
{
    constexpr int G = 1024;
    __shared__ float part[2 * G / WAVE];
    const int units = units_of(cols);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1)
    {
        const float q = rstd[row];
        auto load = [&](int unit, float(&n)[UNIT], float(&a)[UNIT]) {
            const int c = unit * UNIT;
            float wv[UNIT];
            load_unit(h + row * hs + c, c, cols - c, n);
            load_unit(gy + row * gys + c, c, cols - c, a);
            load_unit(w + c, c, cols - c, wv);
#pragma unroll
            for (int j = 0; j < UNIT; ++j)
            {
                n[j] *= q;
                a[j] *= wv[j];
            }
        };
        float s = 0.0f;
        for (int unit = threadIdx.x; unit < units; unit += G)
        {
            float n[UNIT], a[UNIT];
            load(unit, n, a);
#pragma unroll
            for (int j = 0; j < UNIT; ++j) s += a[j] * n[j];
        }
        const float m = row_sum<G>(s, part, turn) * (1.0f / (float)cols);
        for (int unit = threadIdx.x; unit < units; unit += G)
        {
            const int c = unit * UNIT;
            float n[UNIT], a[UNIT];
            load(unit, n, a);
#pragma unroll
            for (int j = 0; j < UNIT; ++j) a[j] = q * (a[j] - n[j] * m);
            if (gh)
            {
                float u[UNIT];
                load_unit(gh + row * ghs + c, c, cols - c, u);
#pragma unroll
                for (int j = 0; j < UNIT; ++j) a[j] += u[j];
            }
            store_unit(gx + row * cols + c, cols - c, a, streaming);
        }
    }
}

// grad_w's sums of wide rows: a lane's unit over every gridDim.y-th row, into slot blockIdx.y.
template <typename T>
__global__ __launch_bounds__(BLOCK) void rms_norm_gw_wide_kernel(const T* __restrict__ gy, int64_t gys, const T* __restrict__ h, int64_t hs,
                                                                 const float* __restrict__ rstd, float* __restrict__ gw_part, int64_t rows,
                                                                 int cols)
{
    const int unit = blockIdx.x * BLOCK + threadIdx.x;
    if (unit >= units_of(cols)) return;
    const int c = unit * UNIT;
    float gw[UNIT] = {};
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y)
    {
        const float q = rstd[row];
        float n[UNIT], a[UNIT];
        load_unit(h + row * hs + c, c, cols - c, n);
        load_unit(gy + row * gys + c, c, cols - c, a);
#pragma unroll
        for (int j = 0; j < UNIT; ++j) gw[j] += a[j] * (n[j] * q);
    }
    store_unit(gw_part + (int64_t)blockIdx.y * cols + c, cols - c, gw);
}

// f(G, V): lanes a row and units a lane for rows of `units`. One unit a lane leaves registers for the most waves and
// is the fastest where it wastes few lanes (16384 x 2000 bfloat16: forward 53 us, 67 with 64 lanes of 4 units;
// 4096 x 8000: 59 and 55 us forward and backward, 74 and 79 with 256 lanes of 4); between the powers of
// two the shape with fewer idle lanes (12000 x 2500: forward 64 us with 256 x 2, 77 with 384 x 1; 3000 x 11000:
// 66 with 512 x 3, 75 with 768 x 2).
template <typename F>
static hipError_t norm_shape(int units, F&& f)
{
    using std::integral_constant;
#define MCA_NORM_SHAPE(MOST, G, V)                                     \
    static_assert((MOST) <= (G) * (V));                                \
    if (units <= (MOST)) return f(integral_constant<int, G>(), integral_constant<int, V>())
    MCA_NORM_SHAPE(4, 4, 1);
    MCA_NORM_SHAPE(8, 8, 1);
    MCA_NORM_SHAPE(16, 16, 1);
    MCA_NORM_SHAPE(32, 32, 1);
    MCA_NORM_SHAPE(64, 64, 1);
    MCA_NORM_SHAPE(128, 64, 2);
    MCA_NORM_SHAPE(192, 192, 1);
    MCA_NORM_SHAPE(256, 256, 1);
    MCA_NORM_SHAPE(384, 256, 2);
    MCA_NORM_SHAPE(512, 512, 1);
    MCA_NORM_SHAPE(768, 768, 1);
    MCA_NORM_SHAPE(1024, 1024, 1);
    MCA_NORM_SHAPE(1536, 512, 3);
    MCA_NORM_SHAPE(NORM_MAX_UNITS, 1024, 2);
#undef MCA_NORM_SHAPE
    return hipErrorInvalidValue;
}

static int norm_grid(int64_t rows, int rows_per_block, int most)
{
    const int64_t n = (rows + rows_per_block - 1) / rows_per_block;
    return (int)(n < most ? n : most);
}

template <typename T, typename WT>
hipError_t rms_norm_forward(const T* x, int64_t x_stride, const T* residual, int64_t r_stride, const WT* w, float eps, T* y, T* h,
                            uint8_t* codes, uint8_t* scales, float* rstd, int64_t rows, int cols, hipStream_t stream)
{
    if (rows <= 0 || cols <= 0) return hipSuccess;
    const int units = units_of(cols);
    // (Of a float32 unit's two stores each is half a line, which past the caches costs a norm without residual, launched
    // alone, up to 6 us: 8192 x 4096 50 us for 43; 524288 x 64 47 for 49. Its training step, whose backward then finds x in the
    // cache, takes 123 us for 137, which is why float32 is not excepted here as it is where nothing is read again, in unpack8.)
    const bool streaming = streams((double)rows * cols * (sizeof(T) * (1.0 + !!residual + !!y + !!h) + !!codes));
    if (units > NORM_MAX_UNITS)
    {
        rms_norm_fwd_wide_kernel<T, WT><<<norm_grid(rows, 1, NORM_BLOCKS), 1024, 0, stream>>>(x, x_stride, residual, r_stride, w, eps, y, h,
                                                                                             codes, scales, rstd, rows, cols, streaming);
        return hipGetLastError();
    }
    return norm_shape(units, [&](auto g, auto v) {
        constexpr int G = decltype(g)::value, V = decltype(v)::value;
        rms_norm_fwd_kernel<T, WT, G, V><<<norm_grid(rows, norm_threads<G>() / G, NORM_BLOCKS * BLOCK / norm_threads<G>()), norm_threads<G>(), 0, stream>>>(
            x, x_stride, residual, r_stride, w, eps, y, h, codes, scales, rstd, rows, cols, streaming);
        return hipGetLastError();
    });
}

// Slots of grad_w's partial sums, one a workgroup of the backward: about as many threads as the 256 CUs hold at once by
// their registers. Fewer leave loads unissued, more leave a last round half empty and make more slots to
// add. bfloat16 with grad_h and with the slots' sum, by the number of workgroups:
//   8192 x 4096 (512 lanes of 1 unit): 62 us with 256, 50 with 512, 54 with 1024;
//   2048 x 8192 (1024 of 1): 39 us with 128, 33 with 256, 39 with 512;  16384 x 2048 (256 of 1): 59 with 512, 51 with 1024, 55 with 1536;
//   65536 x 512 (64 of 1): 57 us with 512, 48 with 1024, 47 with 1536, 56 with 2048;
//   4096 x 11000 (512 of 3): 162 us with 128, 97 with 256, 111 with 512;  2048 x 16384 (1024 of 2): 61 with 128, 53 with 256, 69 with 512.
// A workgroup takes two rows at least where that leaves two workgroups for every CU.
static int norm_slots(int64_t rows, int cols)
{
    const int units = units_of(cols);
    if (units > NORM_MAX_UNITS) return norm_grid(rows, 16, 64);
    int slots = 0;
    (void)norm_shape(units, [&](auto g, auto v) {
        constexpr int G = decltype(g)::value, V = decltype(v)::value;
        constexpr int THREADS = norm_threads<G>();
        const int most = (V >= 3 ? 512 : V == 1 && G == WAVE ? 1536 : 1024) * BLOCK / THREADS, two = norm_grid(rows, 2 * THREADS / G, most);
        slots = two > 2 * NUM_CU ? two : norm_grid(rows, THREADS / G, most < 2 * NUM_CU ? most : 2 * NUM_CU);
        return hipSuccess;
    });
    return slots;
}

size_t rms_norm_backward_workspace(int64_t rows, int cols)
{
    return rows > 0 && cols > 0 ? align_up((size_t)norm_slots(rows, cols) * (size_t)cols * sizeof(float)) : 0;
}

template <typename T, typename WT>
hipError_t rms_norm_backward(const T* grad_y, int64_t gy_stride, const T* grad_h, int64_t gh_stride, const T* h, int64_t h_stride, const WT* w,
                             const float* rstd, T* grad_x, WT* grad_w, int64_t rows, int cols, void* workspace, hipStream_t stream)
{
    if (cols <= 0) return hipSuccess;
    if (rows <= 0 || !grad_y)
    {
        if (grad_w)
        {
            const hipError_t err = sum_slots_async<WT>(nullptr, 0, cols, grad_w, stream);
            if (err != hipSuccess) return err;
        }
        // grad_h alone, whatever h and the weight hold: their products with a zero are NaN where they are not finite.
        return grad_x ? copy_rows<T>(grad_h, gh_stride, grad_x, rows, cols, stream) : hipSuccess;
    }
    if (!grad_x && !grad_w) return hipSuccess;
    const int units = units_of(cols), slots = norm_slots(rows, cols);
    float* part = grad_w ? (float*)workspace : nullptr;
    const bool streaming = streams((double)rows * cols * sizeof(T) * (2.0 + !!grad_h + !!grad_x));
    hipError_t err;
    if (units > NORM_MAX_UNITS)
    {
        if (grad_x)
            rms_norm_bwd_wide_kernel<T, WT><<<norm_grid(rows, 1, NORM_BLOCKS), 1024, 0, stream>>>(grad_y, gy_stride, grad_h, gh_stride, h, h_stride,
                                                                                                 w, rstd, grad_x, rows, cols, streaming);
        if (part)
            rms_norm_gw_wide_kernel<T><<<dim3((units + BLOCK - 1) / BLOCK, slots), BLOCK, 0, stream>>>(grad_y, gy_stride, h, h_stride, rstd, part,
                                                                                                       rows, cols);
        err = hipGetLastError();
    }
    else
    {
        err = norm_shape(units, [&](auto g, auto v) {
            constexpr int G = decltype(g)::value, V = decltype(v)::value;
            rms_norm_bwd_kernel<T, WT, G, V><<<slots, norm_threads<G>(), 0, stream>>>(grad_y, gy_stride, grad_h, gh_stride, h, h_stride, w, rstd,
                                                                                      grad_x, part, rows, cols, streaming);
            return hipGetLastError();
        });
    }
    if (err != hipSuccess || !part) return err;
    return sum_slots_async<WT>(part, slots, cols, grad_w, stream);
}

#define MCA_NORM(T, WT)                                                                                                                     \
    template hipError_t rms_norm_forward<T, WT>(const T*, int64_t, const T*, int64_t, const WT*, float, T*, T*, uint8_t*, uint8_t*, float*, \
                                                int64_t, int, hipStream_t);                                                                 \
    template hipError_t rms_norm_backward<T, WT>(const T*, int64_t, const T*, int64_t, const T*, int64_t, const WT*, const float*, T*, WT*, \
                                                 int64_t, int, void*, hipStream_t)
MCA_NORM(float, float);
MCA_NORM(_Float16, _Float16);
MCA_NORM(_Float16, float);
MCA_NORM(__bf16, __bf16);
MCA_NORM(__bf16, float);

}  // namespace mca
