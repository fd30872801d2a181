// Rotary positions with several axes, alone or with the root-mean-square norm of each head's row before them:
//   n = x / sqrt(mean(x^2) + eps) * w;  angle_j = sum over the axes of position * frequency_j;
//   pair j of a row, (a, b) -> (a cos - b sin, b cos + a sin); values behind the last pair stay.
// Gradients: the rotation by the negative angles gives g, then the norm's, with r = 1 / sqrt(..), m = x r, t = g w:
//   grad_x = r (t - m mean(t m)),  grad_w = sum over tokens and heads of g m.
//
// Bound by HBM: every row is read once and written once. A lane holds 8 pairs (their two halves apart, or side by
// side) or 16 values behind the last pair, so the lanes of a row exchange only the norm's sums. A workgroup takes a few
// tokens of one tensor: it forms their sines and cosines once, in LDS, then all their heads, in the order in which they lie in
// memory (queries and keys each form their own). Few tokens' heads are spread over several workgroups. Measured, bfloat16: 65536 tokens
// of 16 heads of 64 rotated in 54 us (5.0 TB/s, a large copy's rate); 16384 tokens of 32 and 8 heads of 128, normed and rotated in
// 59 us (5.7 TB/s, partly cached), their gradients in 105 (4.8 TB/s) and 7 for the weights' slots; one token of those in 4.1.
//
// Angles are float64 up to a fraction of a turn: in float32 a position of 100000 would be off by 0.004 radians. What is
// left of a turn goes through float32 sine and cosine, the rounding of a result.
#include "block8.hpp"
#include "lanes.hpp"
#include "launch.hpp"
#include "mixer.hpp"
#include "tokens.hpp"

#include "../../include/morphocore_amd_tokens.h"

namespace mca
{

// The lanes of a row: of pairs, 8 a lane, then of the values behind them, 16 a lane.
inline int rotary_lanes(int dim, int pairs) { return (pairs + UNIT - 1) / UNIT + (dim - 2 * pairs + 2 * UNIT - 1) / (2 * UNIT); }

// The two units of a lane.
struct RowPart
{
    int c[2], valid[2], pair, pairs;  // first pair, and how many
};

__device__ __forceinline__ RowPart row_part(int lane, int dim, const Rotation& r)
{
    RowPart p;
    p.pair = lane * UNIT;
    p.pairs = min(max(r.pairs - p.pair, 0), UNIT);
    if (p.pairs > 0)
    {
        p.c[0] = r.interleaved ? 2 * p.pair : p.pair;
        p.c[1] = r.interleaved ? 2 * p.pair + UNIT : r.pairs + p.pair;
        p.valid[0] = r.interleaved ? min(2 * p.pairs, UNIT) : p.pairs;
        p.valid[1] = r.interleaved ? max(2 * p.pairs - UNIT, 0) : p.pairs;
    }
    else
    {
        const int behind = lane - (r.pairs + UNIT - 1) / UNIT;
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            p.c[i] = 2 * r.pairs + (2 * behind + i) * UNIT;
            p.valid[i] = min(max(dim - p.c[i], 0), UNIT);
        }
    }
    return p;
}

// Units as they are stored. A partial one is read as the 8 values that end with it where the row has as many before.
template <typename T>
__device__ __forceinline__ void load_part(const T* __restrict__ row, const RowPart& p, RawUnit<T> (&u)[2])
{
#pragma unroll
    for (int i = 0; i < 2; ++i) load_raw(row + p.c[i], p.c[i] + p.valid[i] >= UNIT, p.valid[i], u[i]);
}

template <typename T>
__device__ __forceinline__ void store_part(T* __restrict__ row, const RowPart& p, const float (&v)[2][UNIT], bool streaming)
{
#pragma unroll
    for (int i = 0; i < 2; ++i) store_unit(row + p.c[i], p.valid[i], v[i], streaming);
}

struct Turn
{
    float cos[UNIT], sin[UNIT];
};

// The sine and cosine of a token's pair.
__device__ __forceinline__ void sine_cosine(const Rotation& r, int64_t token, int pair, bool inverse, float& sine, float& cosine)
{
    const int64_t row = token < r.rows ? token : token % r.rows;
    double angle = 0.0;
    for (int a = 0; a < r.axes; ++a)
    {
        const int64_t at = row * r.axes + a;
        const double position = r.position_type == MCA_POSITION_INT32   ? (double)((const int32_t*)r.positions)[at]
                                : r.position_type == MCA_POSITION_INT64 ? (double)((const int64_t*)r.positions)[at]
                                                                        : (double)((const float*)r.positions)[at];
        angle = fma(position, r.frequencies[(int64_t)a * r.pairs + pair], angle);
    }
    const double turns = angle * 0.15915494309189535;  // 1 / (2 pi)
    sincospif((float)(2.0 * (turns - rint(turns))), &sine, &cosine);
    if (inverse) sine = -sine;
}

// `there`: values behind the pairs are chosen, not turned by 0, which would spread an infinity among them.
__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s, bool there)
{
    const float x = a * c - b * s, y = b * c + a * s;
    a = there ? x : a;
    b = there ? y : b;
}

// Of a unit's pairs those that are there.
template <bool INTERLEAVED>
__device__ __forceinline__ void rotate(float (&v)[2][UNIT], const Turn& t, int pairs)
{
#pragma unroll
    for (int e = 0; e < UNIT; ++e)
    {
        if constexpr (INTERLEAVED)
            turn_pair(v[e / 4][2 * e % UNIT], v[e / 4][2 * e % UNIT + 1], t.cos[e], t.sin[e], e < pairs);
        else
            turn_pair(v[0][e], v[1][e], t.cos[e], t.sin[e], e < pairs);
    }
}

enum RotaryMode
{
    ROTATE,
    NORM_FORWARD,
    NORM_BACKWARD
};

// One tensor of the call: x (or the gradient of the result, with the norm's input in `h`), its scale and its result.
template <typename T, typename WT>
struct RotaryTensor
{
    HeadRows<T> x, h;
    const WT* w;
    T* out;
};

// Sines and cosines that a workgroup holds: of as many tokens as have them, 16 at most.
constexpr int ROTARY_TABLE = 256, ROTARY_TOKENS = 16;

inline int rotary_tokens(int pairs) { return pairs * ROTARY_TOKENS <= ROTARY_TABLE ? ROTARY_TOKENS : ROTARY_TABLE / pairs; }

// Workgroup item b: tokens [b / splits * per, ..), every splits-th share of their rows, of one of the tensors.
template <typename T, typename WT, int G, int MODE, bool INTERLEAVED>
__global__ __launch_bounds__(BLOCK) void rotary_kernel(RotaryTensor<T, WT> q, RotaryTensor<T, WT> k, int64_t tokens, int per, int splits, int dim,
                                                       Rotation r, bool inverse, float eps, float* __restrict__ gw_part, bool streaming)
{
    constexpr int GROUPS = BLOCK / G;
    __shared__ __align__(16) float cosines[ROTARY_TABLE + UNIT], sines[ROTARY_TABLE + UNIT];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const RowPart part = row_part(lane, dim, r);
    const float inv = 1.0f / (float)dim;
    const RotaryTensor<T, WT> t = blockIdx.y ? k : q;
    RawUnit<WT> w[2];
    if (MODE != ROTATE && t.x.heads > 0) load_part(t.w, part, w);
    float gw[2][UNIT] = {};
    const int64_t items = (tokens + per - 1) / per * splits;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x)
    {
        const int64_t token0 = item / splits * per;
        const int split = (int)(item % splits), n = (int)(tokens - token0 < per ? tokens - token0 : per);
        __syncthreads();
        for (int i = threadIdx.x; i < n * r.pairs; i += BLOCK) sine_cosine(r, token0 + i / r.pairs, i % r.pairs, inverse, sines[i], cosines[i]);
        __syncthreads();
        const float per_head = 1.0f / (float)t.x.heads;
        for (int row = split * GROUPS + group; row < n * t.x.heads; row += splits * GROUPS)
        {
            const int at = (int)(((float)row + 0.5f) * per_head), head = row - at * t.x.heads;  // exact below 2^20
            const int64_t token = token0 + at;
            RawUnit<T> raw[2], rawh[2];
            load_part(t.x.x + token * t.x.token_stride + head * t.x.head_stride, part, raw);
            if (MODE == NORM_BACKWARD) load_part(t.h.x + token * t.h.token_stride + head * t.h.head_stride, part, rawh);
            Turn turn;
#pragma unroll
            for (int e = 0; e < UNIT; ++e)
            {
                // (A partial unit's further ones are other pairs', or what lies behind the table, for values that are not there.)
                turn.cos[e] = cosines[min(at * r.pairs + part.pair, ROTARY_TABLE) + e];
                turn.sin[e] = sines[min(at * r.pairs + part.pair, ROTARY_TABLE) + e];
            }
            float v[2][UNIT];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < UNIT; ++j) v[i][j] = raw[i][j];
            if constexpr (MODE == NORM_FORWARD)
            {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) s = fmaf(v[i][j], v[i][j], s);
                const float rstd = 1.0f / sqrtf(fmaf(lane_sum<G>(s), inv, eps));
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) v[i][j] = v[i][j] * rstd * w[i][j];
            }
            rotate<INTERLEAVED>(v, turn, part.pairs);
            if constexpr (MODE == NORM_BACKWARD)
            {
                float s = 0.0f, d = 0.0f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < UNIT; ++j)
                    {
                        s = fmaf(rawh[i][j], rawh[i][j], s);
                        d = fmaf(v[i][j] * w[i][j], rawh[i][j], d);
                    }
                const float rstd = 1.0f / sqrtf(fmaf(lane_sum<G>(s), inv, eps));
                const float mean = lane_sum<G>(d) * rstd * inv;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < UNIT; ++j)
                    {
                        const float m = rawh[i][j] * rstd;
                        gw[i][j] = fmaf(v[i][j], m, gw[i][j]);
                        v[i][j] = rstd * (v[i][j] * w[i][j] - m * mean);
                    }
            }
            if (t.out) store_part(t.out + (token * t.x.heads + head) * dim, part, v, streaming);
        }
    }
    if constexpr (MODE == NORM_BACKWARD)
    {
        if (!gw_part) return;
        // Over the groups of a wave, then over the waves, in a fixed order, into the workgroup's slot.
        __shared__ float sums[NWAVES][G][2 * UNIT];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < UNIT; ++j)
            {
                float s = gw[i][j];
#pragma unroll
                for (int d = G; d < WAVE; d *= 2) s += __shfl_xor(s, d);
                if (threadIdx.x % WAVE < G) sums[threadIdx.x / WAVE][lane][i * UNIT + j] = s;
            }
        __syncthreads();
        float* __restrict__ out = gw_part + ((int64_t)blockIdx.x * 2 + blockIdx.y) * dim;
        for (int i = threadIdx.x; i < G * 2 * UNIT; i += BLOCK)
        {
            const int l = i / (2 * UNIT), at = i % (2 * UNIT);
            const RowPart p = row_part(l, dim, r);
            const int half = at / UNIT, j = at % UNIT;
            if (j < (half ? p.valid[1] : p.valid[0]))
                out[(half ? p.c[1] : p.c[0]) + j] = ((sums[0][l][at] + sums[1][l][at]) + sums[2][l][at]) + sums[3][l][at];
        }
    }
}

template <typename F>
static hipError_t by_lanes(int lanes, F&& f)
{
    using std::integral_constant;
    if (lanes <= 1) return f(integral_constant<int, 1>());
    if (lanes <= 2) return f(integral_constant<int, 2>());
    if (lanes <= 4) return f(integral_constant<int, 4>());
    if (lanes <= 8) return f(integral_constant<int, 8>());
    if (lanes <= 16) return f(integral_constant<int, 16>());
    if (lanes <= 32) return f(integral_constant<int, 32>());
    return f(integral_constant<int, 64>());
}

struct RotaryPlan
{
    int per, splits, blocks;
};

// Few tokens' rows go to several workgroups, down to one row a group of lanes: by whole tokens alone, one token of 40 heads would be
// one workgroup's 10 rounds.
template <int G>
static RotaryPlan rotary_plan(int64_t tokens, int heads, int pairs, int64_t most)
{
    constexpr int64_t ENOUGH = 1024;
    RotaryPlan p;
    p.per = rotary_tokens(pairs);
    while (p.per > 1 && (tokens + p.per - 1) / p.per < ENOUGH) p.per = (p.per + 1) / 2;
    const int64_t blocks = (tokens + p.per - 1) / p.per, rows = ((int64_t)p.per * heads + BLOCK / G - 1) / (BLOCK / G);
    const int64_t want = (ENOUGH + blocks - 1) / blocks;
    p.splits = (int)(want < rows ? want : rows);
    if (p.splits < 1) p.splits = 1;
    p.blocks = (int)(blocks * p.splits < most ? blocks * p.splits : most);
    return p;
}

constexpr int64_t ROTARY_BLOCKS = 1 << 20, ROTARY_SLOTS = 1024;

template <int MODE, typename T, typename WT>
static hipError_t rotary_launch(const RotaryTensor<T, WT>& q, const RotaryTensor<T, WT>& k, int64_t tokens, int dim, const Rotation& r, bool inverse,
                                float eps, float* gw_part, hipStream_t stream)
{
    const int heads = q.x.heads > k.x.heads ? q.x.heads : k.x.heads, tensors = k.out || gw_part ? 2 : 1;
    const double values = (double)tokens * ((double)q.x.heads + k.x.heads) * dim;
    const bool streaming = streams(values * sizeof(T) * (MODE == NORM_BACKWARD ? 3.0 : 2.0));
    return by_lanes(rotary_lanes(dim, r.pairs), [&](auto g) {
        constexpr int G = decltype(g)::value;
        const RotaryPlan p = rotary_plan<G>(tokens, heads, r.pairs, MODE == NORM_BACKWARD ? ROTARY_SLOTS : ROTARY_BLOCKS);
        if (r.interleaved)
            rotary_kernel<T, WT, G, MODE, true><<<dim3(p.blocks, tensors), BLOCK, 0, stream>>>(q, k, tokens, p.per, p.splits, dim, r, inverse, eps, gw_part, streaming);
        else
            rotary_kernel<T, WT, G, MODE, false><<<dim3(p.blocks, tensors), BLOCK, 0, stream>>>(q, k, tokens, p.per, p.splits, dim, r, inverse, eps, gw_part, streaming);
        return hipGetLastError();
    });
}

template <typename T>
hipError_t axial_rotary(HeadRows<T> x, T* out, int64_t tokens, int dim, const Rotation& r, bool inverse, hipStream_t stream)
{
    if (tokens <= 0 || x.heads <= 0) return hipSuccess;
    const RotaryTensor<T, T> q = {x, {}, nullptr, out}, none = {};
    return rotary_launch<ROTATE>(q, none, tokens, dim, r, inverse, 0.0f, nullptr, stream);
}

template <typename T, typename WT>
hipError_t rms_norm_rotary_forward(HeadRows<T> q, HeadRows<T> k, const WT* q_weight, const WT* k_weight, float eps, T* out_q, T* out_k,
                                   int64_t tokens, int dim, const Rotation& r, hipStream_t stream)
{
    if (tokens <= 0 || q.heads + k.heads <= 0) return hipSuccess;
    const RotaryTensor<T, WT> tq = {q, {}, q_weight, out_q}, tk = {k, {}, k_weight, out_k};
    return rotary_launch<NORM_FORWARD>(tq, tk, tokens, dim, r, false, eps, nullptr, stream);
}

static int rotary_slots(int64_t tokens, int heads, int dim, int pairs)
{
    int slots = 0;
    (void)by_lanes(rotary_lanes(dim, pairs), [&](auto g) {
        slots = rotary_plan<decltype(g)::value>(tokens, heads, pairs, ROTARY_SLOTS).blocks;
        return hipSuccess;
    });
    return slots;
}

size_t rms_norm_rotary_backward_workspace(int64_t tokens, int heads, int dim, int pairs)
{
    return tokens > 0 && heads > 0 ? align_up((size_t)rotary_slots(tokens, heads, dim, pairs) * 2 * (size_t)dim * sizeof(float)) : 0;
}

template <typename T, typename WT>
hipError_t rms_norm_rotary_backward(HeadRows<T> gy_q, HeadRows<T> gy_k, HeadRows<T> q, HeadRows<T> k, const WT* q_weight, const WT* k_weight,
                                    float eps, T* grad_q, T* grad_k, WT* grad_weights, int64_t tokens, int dim, const Rotation& r,
                                    void* workspace, hipStream_t stream)
{
    const bool none = tokens <= 0 || q.heads + k.heads <= 0;
    float* part = grad_weights && !none ? (float*)workspace : nullptr;
    if (!none)
    {
        const RotaryTensor<T, WT> tq = {gy_q, q, q_weight, grad_q}, tk = {gy_k, k, k_weight, grad_k};
        const hipError_t err = rotary_launch<NORM_BACKWARD>(tq, tk, tokens, dim, r, true, eps, part, stream);
        if (err != hipSuccess) return err;
    }
    if (!grad_weights) return hipSuccess;
    return sum_slots_async<WT>(part, none ? 0 : rotary_slots(tokens, q.heads > k.heads ? q.heads : k.heads, dim, r.pairs), 2 * (int64_t)dim, grad_weights, stream);
}

#define MCA_ROTARY(T, WT)                                                                                                                    \
    template hipError_t rms_norm_rotary_forward<T, WT>(HeadRows<T>, HeadRows<T>, const WT*, const WT*, float, T*, T*, int64_t, int,          \
                                                       const Rotation&, hipStream_t);                                                        \
    template hipError_t rms_norm_rotary_backward<T, WT>(HeadRows<T>, HeadRows<T>, HeadRows<T>, HeadRows<T>, const WT*, const WT*, float, T*, \
                                                        T*, WT*, int64_t, int, const Rotation&, void*, hipStream_t)
template hipError_t axial_rotary<float>(HeadRows<float>, float*, int64_t, int, const Rotation&, bool, hipStream_t);
template hipError_t axial_rotary<_Float16>(HeadRows<_Float16>, _Float16*, int64_t, int, const Rotation&, bool, hipStream_t);
template hipError_t axial_rotary<__bf16>(HeadRows<__bf16>, __bf16*, int64_t, int, const Rotation&, bool, hipStream_t);
MCA_ROTARY(float, float);
MCA_ROTARY(_Float16, _Float16);
MCA_ROTARY(_Float16, float);
MCA_ROTARY(__bf16, __bf16);
MCA_ROTARY(__bf16, float);

}  // namespace mca
