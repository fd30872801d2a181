// Linear attention over whole sequences, chunk by chunk on the bfloat16 matrix instructions; instantiated for one type of
// the operands by linear_attention_{f32,f16,bf16}.hip. See Pass for what is computed.
//
// With position i of a row in its chunk of C (backwards passes count positions from a sequence's end, so that every pass is
// causal), e = exp(log_decay), S the state before the chunk and s = 1 for backwards passes, 0 forwards:
//   out_i = read (e^(i + 1 - s) a_i S + update sum over j <= i of e^(i - j) (a_i . b_j) c_j),
//   S    <- e^n S + update sum over j of e^(n - 1 + s - j) b_j c_j^T  for a chunk of n rows.
// No quotient of decays is formed, so nothing overflows however fast a head forgets.
//
// A workgroup walks over the chunks of a segment of one head of one sequence, for N of the state's columns: a wave holds all
// rows of its 16 or 32 columns in the accumulators of the state's own product. Long sequences are split into segments
// where there are too few heads to fill the chip: one launch sums every segment's state by itself, a second joins them (both
// read b and c only), then every segment starts from its state.
//
// Products. Operands of 16 bits are one bfloat16 term (bfloat16) or two (float16, exactly), float32 is three; scores and states
// are split into two terms for 16-bit results (2^-16 of each: the result's own rounding is 2^-9) and into three for float32; decayed
// rows of c into three, so that states are float32's.
//
// Layouts. Of a 16 x 16 x 32 product lane l gives the first operand's row l % 16 and the second's column l % 16 with 8 values
// of the summed axis from 8 (l / 16) on, and gets column l % 16, rows 4 (l / 16) to + 3. The transposing LDS read takes a row's 4-value
// groups from wherever a lane points, so the state's 32 rows of two products are numbered such that a lane's two
// results are 8 neighbouring rows: the first operand of a S, with no exchange between lanes. The same numbering of columns makes a
// lane's results of two products 8 neighbouring values of out, stored at once. Rows of the staged tiles are units of 8 values whose order
// changes from row to row, so that row and transposing reads both spread over the banks.
#pragma once

#include "block8.hpp"
#include "launch.hpp"
#include "tokens.hpp"

namespace mca
{

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------------
// Decays and sequences.
// ------------------------------------------------------------------------------------------------

// Decays below exp(-16384) are 0 anyway, and times 0 must stay 0.
__device__ __forceinline__ float log_decay_of(const float* __restrict__ log_decay, int head)
{
    const float g = log_decay[head];
    return g < -16384.0f ? -16384.0f : g;
}

// The decay of n tokens in two float32 terms: one alone is off by up to 2^-25, the same way every time, which a state that is
// decayed and added to for long adds up (one that keeps 1 - 2^-12 of itself a token, to 2^-13).
struct Decay
{
    float hi, lo;

    __device__ __forceinline__ Decay(float log_decay, double n)
    {
        const double d = exp((double)log_decay * n);
        hi = (float)d, lo = d < 1e30 ? (float)(d - (double)hi) : 0.0f;
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

// Where span i of packed rows begins: span 0 is what lies before the first sequence, span count + 1 what lies behind the last.
__device__ __forceinline__ int64_t span_start(const Sequences& s, int64_t i)
{
    return i == 0 ? 0 : i >= s.count + 2 ? s.tokens : offset_at(s, i - 1);
}

// Segments. Sequences of one length have the same number each; span i of packed rows has those from span_start(i) / rows + i on, which
// needs no sum over the spans before it (and leaves some numbers without rows).
struct Segments
{
    int64_t rows, count, each;
};

inline Segments segments_of(const Sequences& s, int64_t rows)
{
    if (s.offsets) return Segments{rows, s.tokens / rows + s.count + 2, 0};
    const int64_t each = s.tokens > 0 ? (s.tokens + rows - 1) / rows : 1;
    return Segments{rows, s.count * each, each};
}

struct Segment
{
    Rows1 q;
    int64_t first, n, number;  // rows [first, first + n) of the sequence, the number-th segment of it
};

// Every lane of a wave calls it.
__device__ __forceinline__ Segment segment_at(const Sequences& s, const Segments& g, int64_t at)
{
    Segment r;
    if (!s.offsets)
    {
        r.q = Rows1{at / g.each, 0, s.tokens, false};
        r.number = at % g.each;
    }
    else
    {
        // The last span whose first number is at most `at`: 64 probes a step.
        int64_t low = 0, high = s.count + 2;
        while (high - low > 1)
        {
            const int64_t step = (high - low + WAVE - 1) / WAVE, i = low + (int64_t)(threadIdx.x % WAVE) * step;
            const bool before = i < high && span_start(s, i) / g.rows + i <= at;
            const int n = __popcll(__ballot(before));
            low += (int64_t)(n > 1 ? n - 1 : 0) * step;
            high = low + step < high ? low + step : high;
        }
        const int64_t a = span_start(s, low), b = span_start(s, low + 1);
        r.q = Rows1{low - 1, a, b > a ? b - a : 0, low == 0 || low == s.count + 1};
        r.number = at - (a / g.rows + low);
    }
    r.first = r.number * g.rows;
    const int64_t left = r.q.length - r.first;
    r.n = r.number < 0 || left < 0 ? 0 : left < g.rows ? left : g.rows;
    return r;
}

// ------------------------------------------------------------------------------------------------
// Tiles.
// ------------------------------------------------------------------------------------------------

template <typename T>
constexpr int terms_of()
{
    return std::is_same_v<T, float> ? 3 : std::is_same_v<T, _Float16> ? 2 : 1;
}

// DK: rows of the state (the values of a and b), W waves of NT * 16 columns each.
template <typename T, int DK_, int W_, int NT_>
struct Walk
{
    static constexpr int DK = DK_, W = W_, NT = NT_, N = 16 * W * NT, THREADS = W * WAVE;
    static constexpr int PL = terms_of<T>(), PS = PL == 3 ? 3 : 2;  // terms of the operands, and of scores and states
    // Rows of a chunk: what two workgroups' tiles leave room for in a CU's 160 KB, or one's.
    static constexpr int C = PL == 3 || (PL == 2 && DK == 256) ? 32 : 64;
    static constexpr int AB = C * DK * 2, V = C * N * 2, P = C * C * 2;  // bytes of a term's tile
    static constexpr int LDS = 2 * PL * AB + PL * V + PS * P;
    static constexpr int BLOCKS = LDS <= 76 * 1024 && W == 4 ? 2 : 1;
};

// Where unit x (8 values) of row r lies in a tile of U units a row: in 64 banks, 16 rows' units x and 4 rows' units x to x + 3 lie apart.
template <int U>
__device__ __forceinline__ int unit_place(int r, int x)
{
    if constexpr (U >= 16) return x ^ (4 * (r & 3) + ((r >> 2) & 3));
    if constexpr (U == 8) return x ^ (4 * ((r >> 1) & 1) + ((r >> 2) & 3));
    if constexpr (U == 4) return x ^ ((r >> 2) & 3);
    return x ^ ((r >> 3) & 1);
}

template <int U>
__device__ __forceinline__ int unit_byte(int r, int x)
{
    return (r * U + unit_place<U>(r, x)) * 16;
}

// A lane's 8 values of the summed axis, which lies along the rows: row `row` + lane % 16, values 32 k + 8 (lane / 16) on.
template <int U>
__device__ __forceinline__ bf16x8 row_fragment(const char* tile, int row, int k)
{
    const int l = threadIdx.x % WAVE;
    return *(const bf16x8*)(tile + unit_byte<U>(row + l % 16, 4 * k + l / 16));
}

// The same where it lies across the rows: rows `row` + 8 (lane / 16) on, of the column that lane % 16 stands for: value lane % 4 of
// the 4 at unit(lane / 4 % 4), half(..). The lane points at the group (lane % 4) of row lane / 4 % 4.
template <int U>
__device__ __forceinline__ bf16x8 column_fragment(const char* tile, int row, int unit, int half)
{
    const int l = threadIdx.x % WAVE, r = row + 8 * (l / 16) + ((l >> 2) & 3);
    typedef __attribute__((address_space(3))) bf16x4* lds4;
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(tile + unit_byte<U>(r, unit) + 8 * half));
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(tile + unit_byte<U>(r + 4, unit) + 8 * half));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Values in bfloat16 terms, each the nearest to what the ones before leave. CUT: the first one by truncation, which takes the largest
// float32 values to no infinity.
template <int TERMS, bool CUT, int N>
__device__ __forceinline__ void split(const float (&v)[N], __bf16 (&term)[TERMS][N])
{
#pragma unroll
    for (int j = 0; j < N; j += 2)
    {
        f32x2 x = {v[j], v[j + 1]};
#pragma unroll
        for (int i = 0; i < TERMS; ++i)
        {
            bf16x2 t;
            if (CUT && i == 0)
                t = __builtin_bit_cast(bf16x2, __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x07060302u));
            else
                t = __builtin_convertvector(x, bf16x2);
            term[i][j] = t[0], term[i][j + 1] = t[1];
            if (i + 1 < TERMS)
            {
                x[0] -= (float)t[0];
                x[1] -= (float)t[1];
            }
        }
    }
}

template <typename V8, int TERMS, int N>
__device__ __forceinline__ V8 term_vector(const __bf16 (&term)[TERMS][N], int i)
{
    V8 v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = term[i][j];
    return v;
}

// Whether one of the 8 values is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(const RawUnit<T>& u)
{
    if constexpr (sizeof(T) == 4)
    {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, u.d[i] & 0x7fffffffu);
        return m >= 0x7f800000u;
    }
    else
    {
        constexpr uint32_t INF = std::is_same_v<T, __bf16> ? 0x7f80u : 0x7c00u;
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, u.d[i] & 0x7fff7fffu));
        return m[0] >= INF || m[1] >= INF;
    }
}

// What of a chunk's b and c is not finite. Such values count as 0 in the products; what depends on them becomes NaN afterwards: a row's
// own and later results, and the state. (0 times an infinity in a product would spoil the rows before it too.)
template <typename L>
struct Spoiled
{
    int any;          // the last chunk's number that has some, plus 1
    int row;          // its first row with such a b
    int col[L::N];    // the first row with such a c, by column
    int dim[L::DK];   // whether b has one in this place
};

template <typename L>
__device__ __forceinline__ void clear_spoiled(Spoiled<L>& s)
{
    for (int i = threadIdx.x; i < L::N; i += L::THREADS) s.col[i] = L::C;
    for (int i = threadIdx.x; i < L::DK; i += L::THREADS) s.dim[i] = 0;
    if (threadIdx.x == 0) s.row = L::C, s.any = 0;
}

// A tile of C rows on its way from memory to LDS.
template <typename T, typename L, int COLS>
struct TileLoad
{
    static constexpr int U = COLS / UNIT, UNITS = L::C * U, COUNT = (UNITS + L::THREADS - 1) / L::THREADS;
    static_assert(UNITS % L::THREADS == 0 || COUNT == 1);
    RawUnit<T> raw[COUNT];

    // Rows [0, n) of `base` + row * stride (which may fall), values [c0, cols).
    __device__ __forceinline__ void load(const T* __restrict__ base, int64_t stride, int n, int c0, int cols)
    {
#pragma unroll
        for (int i = 0; i < COUNT; ++i)
        {
            const int u = threadIdx.x + i * L::THREADS, r = u / U, c = c0 + u % U * UNIT;
            load_raw(base + r * stride + c, c, r < n ? cols - c : 0, raw[i]);  // r >= C of threads without a unit: n is at most C
        }
    }

    template <bool CHECK, typename F>
    __device__ __forceinline__ void store(char* tile, F&& spoil)
    {
        constexpr int BYTES = L::C * COLS * 2;
#pragma unroll
        for (int i = 0; i < COUNT; ++i)
        {
            const int u = threadIdx.x + i * L::THREADS, r = u / U, x = u % U;
            if (UNITS % L::THREADS && u >= UNITS) break;
            if (CHECK && not_finite<T>(raw[i]))
            {
#pragma unroll
                for (int j = 0; j < UNIT; ++j)
                {
                    const float v = raw[i][j];
                    if (fabsf(v) <= 3.4028235e38f) continue;
                    spoil(r, x * UNIT + j);
                    if constexpr (sizeof(T) == 4)
                        raw[i].d[j] = 0;
                    else
                        raw[i].d[j / 2] &= j % 2 ? 0xffffu : 0xffff0000u;
                }
            }
            if constexpr (L::PL == 1)
            {
                *(bf16x8*)(tile + unit_byte<U>(r, x)) = __builtin_bit_cast(bf16x8, raw[i]);
            }
            else
            {
                float v[UNIT];
#pragma unroll
                for (int j = 0; j < UNIT; ++j) v[j] = raw[i][j];
                __bf16 term[L::PL][UNIT];
                split<L::PL, true>(v, term);
#pragma unroll
                for (int p = 0; p < L::PL; ++p) *(bf16x8*)(tile + p * BYTES + unit_byte<U>(r, x)) = term_vector<bf16x8>(term, p);
            }
        }
    }
};

struct Passes
{
    Pass p[3];
    float* states[3];  // of the segments
};

// A lane's place in the state: rows 32 u + 8 (lane / 16) + 4 h + r, and the column.
template <typename L>
__device__ __forceinline__ int state_column(int t)
{
    const int l = threadIdx.x % WAVE, w = threadIdx.x / WAVE, n = l % 16;
    return L::NT == 2 ? 32 * w + 8 * (n >> 2) + 4 * t + (n & 3) : 16 * w + n;
}

// Values of a segment's state of one tile, in the order in which lanes hold them.
template <typename L>
constexpr int64_t state_values()
{
    return (int64_t)L::DK * L::N;
}

// ONLY: the segments' own states (from 0) to the workspace, of all but the last of a sequence; no results.
template <typename T, typename L, bool ONLY>
__global__ __launch_bounds__(L::THREADS, L::BLOCKS) void attention_walk_kernel(Sequences seq, Segments segments, int heads,
                                                                               const float* __restrict__ log_decay, Passes passes, int tiles)
{
    constexpr int C = L::C, DK = L::DK, N = L::N, NT = L::NT, PL = L::PL, PS = L::PS, RT = C / 16, KS = C / 32, KD = DK / 32;
    constexpr int UD = DK / UNIT, UN = N / UNIT, UC = C / UNIT;
    __shared__ __align__(16) char lds[ONLY ? PL * (L::AB + L::V) : L::LDS];
    __shared__ Spoiled<L> spoiled;
    char* const tb = lds;
    char* const tc = tb + PL * L::AB;
    char* const ta = ONLY ? nullptr : tc + PL * L::V;
    char* const tp = ONLY ? nullptr : ta + PL * L::AB;
    const int l = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, g = l / 16;
    const Pass& p = passes.p[blockIdx.y];
    const int s = p.backwards ? 1 : 0;
    if constexpr (!ONLY)
        for (int i = threadIdx.x; i < PS * L::P / 16; i += L::THREADS) ((uint4*)tp)[i] = make_uint4(0, 0, 0, 0);
    clear_spoiled(spoiled);
    int chunk = 0;

    const int64_t work = segments.count * heads * tiles;
    for (int64_t item = blockIdx.x; item < work; item += gridDim.x)
    {
        const int tile = (int)(item % tiles), head = (int)(item / tiles % heads);
        const int64_t at = item / tiles / heads;
        const Segment part = segment_at(seq, segments, at);
        const int64_t n_all = part.n;
        const bool last = part.first + n_all >= part.q.length;
        const int col0 = tile * N, cols = p.cols;
        const int64_t row0 = seq.offsets ? part.q.start : part.q.batch * seq.tokens;
        if (part.q.none)
        {
            if constexpr (!ONLY)
                if (p.out)
                    for (int64_t i = threadIdx.x; i < n_all * N; i += L::THREADS)
                    {
                        const int64_t row = row0 + part.first + i / N;
                        const int c = col0 + (int)(i % N);
                        if (c >= cols) continue;
                        if (p.out32)
                            p.out32[(row * heads + head) * cols + c] = 0.0f;
                        else
                            ((T*)p.out)[(row * heads + head) * cols + c] = (T)0.0f;
                    }
            continue;
        }
        // A sequence without rows has one segment (number 0), which hands its state on.
        if (ONLY ? last || n_all == 0 : n_all == 0 && part.number != 0) continue;

        const float lg = log_decay_of(log_decay, head), lg2 = lg * 1.4426950408889634f;
        auto power = [&](int n) { return __builtin_amdgcn_exp2f(lg2 * (float)n); };
        const Decay chunk_decay(lg, C);
        const float update = p.update, read = p.read;
        // e^(i - j) of two tiles of rows `d` apart, in a lane's place; e^(i + 1 - s); e^(7 - v) of a lane's 8 rows of c.
        float near[RT][4], far[RT], tail[UNIT];
        if constexpr (!ONLY)
        {
#pragma unroll
            for (int d = 0; d < RT; ++d)
            {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                {
                    const int gap = 16 * d + l % 16 - 4 * g - r;
                    near[d][r] = gap < 0 ? 0.0f : power(gap) * (update * read);
                }
                far[d] = power(16 * d + l % 16 + 1 - s) * read;
            }
        }
#pragma unroll
        for (int v = 0; v < UNIT; ++v) tail[v] = power(UNIT - 1 - v) * update;

        // The state: from the workspace, as lanes hold it, or the pass's first.
        f32x4 S[KD][2][NT];
        const int64_t state0 = (part.q.batch * heads + head) * p.dim * cols;
        const bool joined = !ONLY && part.number > 0;
        const float* __restrict__ begin = joined ? passes.states[blockIdx.y] + (((at - 1) * heads + head) * tiles + tile) * state_values<L>() : nullptr;
#pragma unroll
        for (int u = 0; u < KD; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                {
                    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (joined)
                    {
                        x = *(const f32x4*)(begin + ((((int64_t)wave * KD + u) * 2 + h) * NT + t) * WAVE * 4 + l * 4);
                    }
                    else if (!ONLY && p.first.p)
                    {
                        const int c = col0 + state_column<L>(t);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                        {
                            const int d = 32 * u + 8 * g + 4 * h + r;
                            if (d < p.dim && c < cols) x[r] = p.first.p[state0 + d * p.first.row_stride + c * p.first.col_stride];
                        }
                    }
                    S[u][h][t] = x;
                }

        // Position 0's rows; the rows of later positions follow, or come before it where time runs backwards.
        const int64_t dir = s ? -1 : 1, t0 = part.q.start + (s ? part.q.length - 1 - part.first : part.first);
        auto row_base = [&](const TokenRows& r) {
            return (const T*)r.p + (seq.offsets ? 0 : part.q.batch * r.batch_stride) + t0 * r.token_stride + head / r.share * r.head_stride;
        };
        const T* __restrict__ pa = ONLY ? nullptr : row_base(p.a);
        const T* __restrict__ pb = row_base(p.b);
        const T* __restrict__ pc = row_base(p.c);
        const int64_t sa = dir * p.a.token_stride, sb = dir * p.b.token_stride, sc = dir * p.c.token_stride;
        TileLoad<T, L, DK> la, lb;
        TileLoad<T, L, N> lc;
        auto load = [&](int64_t first) {
            const int n = (int)(n_all - first < C ? n_all - first : C);
            if constexpr (!ONLY) la.load(pa + first * sa, sa, n, 0, p.dim);
            lb.load(pb + first * sb, sb, n, 0, p.dim);
            lc.load(pc + first * sc, sc, n, col0, cols);
        };
        if (n_all > 0) load(0);
        for (int64_t first = 0; first < n_all; first += C)
        {
            const int n = (int)(n_all - first < C ? n_all - first : C);
            ++chunk;
            __syncthreads();
            if constexpr (!ONLY) la.template store<false>(ta, [](int, int) {});
            lb.template store<true>(tb, [&](int r, int c) {
                spoiled.any = chunk;
                spoiled.dim[c] = 1;
                atomicMin(&spoiled.row, r);
            });
            lc.template store<true>(tc, [&](int r, int c) {
                spoiled.any = chunk;
                atomicMin(&spoiled.col[c], r);
            });
            if (first + C < n_all) load(first + C);
            __syncthreads();

            f32x4 o[RT][NT] = {};
            if constexpr (!ONLY)
            {
                // Scores of the wave's rows, decayed, in terms to LDS.
#pragma unroll
                for (int rt0 = 0; rt0 < RT; rt0 += L::W)
                {
                    const int rt = rt0 + wave;
                    if (rt >= RT) continue;
                    bf16x8 fa[KD][PL];
#pragma unroll
                    for (int k = 0; k < KD; ++k)
#pragma unroll
                        for (int i = 0; i < PL; ++i) fa[k][i] = row_fragment<UD>(ta + i * L::AB, 16 * rt, k);
#pragma unroll
                    for (int ct = 0; ct < RT; ++ct)
                    {
                        if (ct > rt) continue;
                        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int k = 0; k < KD; ++k)
#pragma unroll
                            for (int j = 0; j < PL; ++j)
                            {
                                const bf16x8 fb = row_fragment<UD>(tb + j * L::AB, 16 * ct, k);
#pragma unroll
                                for (int i = 0; i < PL; ++i)
                                    if (i + j <= 2) x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, fa[k][i], x, 0, 0, 0);
                            }
                        float v[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                        {
                            float w = 0.0f;
#pragma unroll
                            for (int d = 0; d < RT; ++d) w = rt - ct == d ? near[d][r] : w;
                            // What lies above the diagonal is no product with 0: a query's infinity stays in its row.
                            v[r] = rt == ct && l % 16 - 4 * g - r < 0 ? 0.0f : x[r] * w;
                        }
                        __bf16 term[PS][4];
                        split<PS, false>(v, term);
#pragma unroll
                        for (int i = 0; i < PS; ++i)
                            *(bf16x4*)(tp + i * L::P + unit_byte<UC>(16 * rt + l % 16, 2 * ct + (g >> 1)) + 8 * (g & 1)) = term_vector<bf16x4>(term, i);
                    }
                }
                // a S, with the state's terms as they lie in the lanes.
#pragma unroll
                for (int u = 0; u < KD; ++u)
                {
                    bf16x8 fs[NT][PS];
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                    {
                        float v[UNIT];
#pragma unroll
                        for (int j = 0; j < UNIT; ++j) v[j] = S[u][j / 4][t][j % 4];
                        __bf16 term[PS][UNIT];
                        split<PS, false>(v, term);
#pragma unroll
                        for (int i = 0; i < PS; ++i) fs[t][i] = term_vector<bf16x8>(term, i);
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int i = 0; i < PL; ++i)
                        {
                            const bf16x8 fa = row_fragment<UD>(ta + i * L::AB, 16 * rt, u);
#pragma unroll
                            for (int t = 0; t < NT; ++t)
#pragma unroll
                                for (int j = 0; j < PS; ++j)
                                    if (i + j < PS) o[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fs[t][j], fa, o[rt][t], 0, 0, 0);
                        }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[rt][t] *= far[rt];
                __syncthreads();
            }

            // Scores times c, and the state after the chunk.
            const bool whole = n == C;
            const Decay decay = whole ? chunk_decay : Decay(lg, n);
#pragma unroll
            for (int u = 0; u < KD; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) S[u][h][t][r] = decay.of(S[u][h][t][r]);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
            {
                bf16x8 fc[NT][PL], fd[NT][3];
                // e^(n - 1 + s - j) of the lane's last row j = 32 ks + 8 g + 7 (rows behind the chunk's end are 0).
                const int past = n - 1 + s - (32 * ks + 8 * g + 7);
                const float base = power(past);
#pragma unroll
                for (int t = 0; t < NT; ++t)
                {
                    float v[UNIT] = {};
#pragma unroll
                    for (int i = 0; i < PL; ++i)
                    {
                        fc[t][i] = NT == 2 ? column_fragment<UN>(tc + i * L::V, 32 * ks, 4 * wave + (l & 3), t)
                                           : column_fragment<UN>(tc + i * L::V, 32 * ks, 2 * wave + ((l & 3) >> 1), l & 1);
#pragma unroll
                        for (int j = 0; j < UNIT; ++j) v[j] += (float)fc[t][i][j];
                    }
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) v[j] = past >= 0 ? v[j] * (tail[j] * base) : past + 7 - j >= 0 ? v[j] * (power(past + 7 - j) * update) : 0.0f;
                    __bf16 term[3][UNIT];
                    split<3, false>(v, term);
#pragma unroll
                    for (int i = 0; i < 3; ++i) fd[t][i] = term_vector<bf16x8>(term, i);
                }
                if constexpr (!ONLY)
                {
#pragma unroll
                    for (int rt = 2 * ks; rt < RT; ++rt)
#pragma unroll
                        for (int j = 0; j < PS; ++j)
                        {
                            const bf16x8 fp = row_fragment<UC>(tp + j * L::P, 16 * rt, ks);
#pragma unroll
                            for (int t = 0; t < NT; ++t)
#pragma unroll
                                for (int i = 0; i < PL; ++i)
                                    if (i + j < PS) o[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fc[t][i], fp, o[rt][t], 0, 0, 0);
                        }
                }
#pragma unroll
                for (int u = 0; u < KD; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < PL; ++i)
                        {
                            const bf16x8 fb = column_fragment<UD>(tb + i * L::AB, 32 * ks, 4 * u + (l & 3), h);
#pragma unroll
                            for (int t = 0; t < NT; ++t)
#pragma unroll
                                for (int j = 0; j < 3; ++j)
                                    if (i + j <= 2) S[u][h][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, fd[t][j], S[u][h][t], 0, 0, 0);
                        }
            }
            if (spoiled.any == chunk)
            {
                const float nan = __builtin_nanf("");
#pragma unroll
                for (int t = 0; t < NT; ++t)
                {
                    const int by = spoiled.col[state_column<L>(t)];
#pragma unroll
                    for (int u = 0; u < KD; ++u)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (by < C || spoiled.dim[32 * u + 8 * g + 4 * h + r]) S[u][h][t][r] = nan;
                    if constexpr (!ONLY)
                    {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                        {
                            const int from = min(spoiled.row, spoiled.col[NT == 2 ? 32 * wave + 8 * g + 4 * t + r : 16 * wave + 4 * g + r]);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt)
                                if (16 * rt + l % 16 >= from) o[rt][t][r] = nan;
                        }
                    }
                }
                __syncthreads();
                clear_spoiled(spoiled);
            }
            if constexpr (!ONLY)
            {
                if (p.out)
                {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                    {
                        const int i = 16 * rt + l % 16;
                        if (i >= n) continue;
                        const int64_t pos = part.first + first + i, row = row0 + (s ? part.q.length - 1 - pos : pos);
                        const int c = col0 + (NT == 2 ? 32 * wave + 8 * g : 16 * wave + 4 * g);
                        const int64_t to = (row * heads + head) * cols + c;
                        float v[UNIT] = {};
#pragma unroll
                        for (int j = 0; j < 4 * NT; ++j) v[j] = o[rt][j / 4][j % 4];
                        const int valid = min(cols - c, 4 * NT);
                        if (p.out32)
                            store_unit(p.out32 + to, valid, v);
                        else
                            store_unit((T*)p.out + to, valid, v);
                    }
                }
            }
        }

        if (ONLY)
        {
            float* __restrict__ end = passes.states[blockIdx.y] + ((at * heads + head) * tiles + tile) * state_values<L>();
#pragma unroll
            for (int u = 0; u < KD; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t = 0; t < NT; ++t) *(f32x4*)(end + ((((int64_t)wave * KD + u) * 2 + h) * NT + t) * WAVE * 4 + l * 4) = S[u][h][t];
        }
        else if (last && p.last.p)
        {
#pragma unroll
            for (int u = 0; u < KD; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                        {
                            const int d = 32 * u + 8 * g + 4 * h + r, c = col0 + state_column<L>(t);
                            if (d < p.dim && c < cols) p.last.p[state0 + d * p.last.row_stride + c * p.last.col_stride] = S[u][h][t][r];
                        }
        }
    }
}

// Turns the segments' own states into the states after them, sequence by sequence: one value of a tile's state a thread.
template <typename L>
__global__ __launch_bounds__(BLOCK) void attention_join_kernel(Sequences seq, Segments segments, int heads, const float* __restrict__ log_decay,
                                                               Passes passes, int tiles)
{
    constexpr int VALUES = (int)state_values<L>(), BLOCKS = (VALUES + BLOCK - 1) / BLOCK;
    const Pass& p = passes.p[blockIdx.y];
    const int64_t spans = seq.offsets ? seq.count : seq.count, work = spans * heads * tiles * BLOCKS;
    for (int64_t item = blockIdx.x; item < work; item += gridDim.x)
    {
        const int block = (int)(item % BLOCKS), tile = (int)(item / BLOCKS % tiles), head = (int)(item / BLOCKS / tiles % heads);
        const int64_t q = item / BLOCKS / tiles / heads;
        int64_t length = seq.tokens, at = q * segments.each;
        if (seq.offsets)
        {
            const int64_t a = offset_at(seq, q), b = offset_at(seq, q + 1);
            length = b > a ? b - a : 0;
            at = a / segments.rows + q + 1;
        }
        const int64_t count = (length + segments.rows - 1) / segments.rows - 1;  // all but the last
        const int e = block * BLOCK + threadIdx.x;
        if (count <= 0 || e >= VALUES) continue;
        // The value's place: see attention_walk_kernel's workspace.
        const int r = e % 4, l = e / 4 % WAVE, t = e / 4 / WAVE % L::NT, h = e / 4 / WAVE / L::NT % 2, u = e / 4 / WAVE / L::NT / 2 % (L::DK / 32);
        const int w = e / 4 / WAVE / L::NT / 2 / (L::DK / 32), n = l % 16, d = 32 * u + 8 * (l / 16) + 4 * h + r;
        const int c = tile * L::N + (L::NT == 2 ? 32 * w + 8 * (n >> 2) + 4 * t + (n & 3) : 16 * w + n);
        const Decay decay(log_decay_of(log_decay, head), (double)segments.rows);
        float x = 0.0f;
        if (p.first.p && d < p.dim && c < p.cols)
            x = p.first.p[(q * heads + head) * p.dim * p.cols + d * p.first.row_stride + c * p.first.col_stride];
        const int64_t stride = (int64_t)heads * tiles * VALUES;
        float* __restrict__ state = passes.states[blockIdx.y] + ((at * heads + head) * tiles + tile) * VALUES + e;
        constexpr int AHEAD = 8;
        for (int64_t i = 0; i < count; i += AHEAD)
        {
            float own[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) own[k] = state[(i + k < count ? i + k : count - 1) * stride];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
            {
                if (i + k >= count) break;
                x = decay.of(x) + own[k];
                state[(i + k) * stride] = x;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Launches.
// ------------------------------------------------------------------------------------------------

// f(the shape of a pass): as few columns as hold the pass's, up to 128 a workgroup.
template <typename T, typename F>
hipError_t by_walk(const Pass& p, F&& f)
{
#define MCA_WALK(DK, W, NT) return f(Walk<T, DK, W, NT>())
#define MCA_WALKS(DK)                        \
    do                                       \
    {                                        \
        if (p.cols <= 64) MCA_WALK(DK, 4, 1); \
        MCA_WALK(DK, 4, 2);                  \
    } while (0)
    if (p.dim <= 64 && p.cols <= 32)
    {
        if (p.dim <= 32)
        {
            if (p.cols <= 16) MCA_WALK(32, 1, 1);
            MCA_WALK(32, 2, 1);
        }
        if (p.cols <= 16) MCA_WALK(64, 1, 1);
        MCA_WALK(64, 2, 1);
    }
    if (p.dim <= 32) MCA_WALKS(32);
    if (p.dim <= 64) MCA_WALKS(64);
    if (p.dim <= 128) MCA_WALKS(128);
    MCA_WALKS(256);
#undef MCA_WALKS
#undef MCA_WALK
}

template <typename L>
int tiles_of(const Pass& p)
{
    return (p.cols + L::N - 1) / L::N;
}

// Rows of a segment. Splitting a sequence costs a second read of b and c and its states' way through memory, so it is split only where
// there are fewer walks than the chip holds, into segments of 8 chunks at least.
template <typename L>
Segments plan_segments(const Sequences& seq, int64_t walks)
{
    constexpr int64_t TARGET = 512, LEAST = 8;
    const int64_t chunks = (seq.tokens + L::C - 1) / L::C;
    // Packed rows may be one sequence.
    int64_t per = walks >= TARGET ? chunks : (chunks * walks + TARGET - 1) / TARGET;
    per = per < LEAST ? LEAST : per;
    if (per >= chunks) per = chunks < 1 ? 1 : chunks;
    return segments_of(seq, per * L::C);
}

template <typename L>
Segments plan_of(const Sequences& seq, int heads, const Pass& p, int count)
{
    return plan_segments<L>(seq, (seq.offsets ? 1 : seq.count) * (int64_t)heads * tiles_of<L>(p) * count);
}

template <typename L>
bool joins(const Sequences& seq, const Segments& s)
{
    return seq.tokens > s.rows;
}

template <typename L>
size_t walk_states(const Sequences& seq, int heads, const Pass& p, int count)
{
    const Segments s = plan_of<L>(seq, heads, p, count);
    return joins<L>(seq, s) ? align_up((size_t)(s.count * heads * tiles_of<L>(p) * state_values<L>()) * sizeof(float)) : 0;
}

template <typename T>
size_t linear_attention_workspace(const Sequences& seq, int heads, const Pass* passes, int count)
{
    size_t bytes = 0;
    for (int i = 0; i < count; ++i)
        (void)by_walk<T>(passes[i], [&](auto walk) {
            bytes += walk_states<decltype(walk)>(seq, heads, passes[i], count);
            return hipSuccess;
        });
    return bytes;
}

template <typename T>
hipError_t linear_attention(const Sequences& seq, int heads, const float* log_decay, const Pass* passes, int count, void* workspace, hipStream_t stream)
{
    if ((seq.offsets ? seq.count + seq.tokens : seq.count) <= 0 || heads <= 0) return hipSuccess;
    char* ws = (char*)workspace;
    for (int i = 0; i < count;)
    {
        // Passes of the same shape go together.
        int together = 1;
        while (i + together < count && passes[i + together].dim == passes[i].dim && passes[i + together].cols == passes[i].cols) ++together;
        const hipError_t err = by_walk<T>(passes[i], [&](auto walk) {
            using L = decltype(walk);
            const Segments s = plan_of<L>(seq, heads, passes[i], count);
            const int tiles = tiles_of<L>(passes[i]);
            const bool split = joins<L>(seq, s);
            Passes all = {};
            for (int k = 0; k < together; ++k)
            {
                all.p[k] = passes[i + k];
                if (!split) continue;
                all.states[k] = (float*)ws;
                ws += walk_states<L>(seq, heads, passes[i + k], count);
            }
            const int64_t work = s.count * heads * tiles, most = 1 << 20;
            const dim3 grid((unsigned)(work < most ? work : most), together);
            if (split)
            {
                attention_walk_kernel<T, L, true><<<grid, L::THREADS, 0, stream>>>(seq, s, heads, log_decay, all, tiles);
                const int64_t values = seq.count * heads * tiles * ((state_values<L>() + BLOCK - 1) / BLOCK);
                if (values > 0)
                    attention_join_kernel<L><<<dim3((unsigned)(values < most ? values : most), together), BLOCK, 0, stream>>>(seq, s, heads, log_decay, all, tiles);
            }
            attention_walk_kernel<T, L, false><<<grid, L::THREADS, 0, stream>>>(seq, s, heads, log_decay, all, tiles);
            return hipGetLastError();
        });
        if (err != hipSuccess) return err;
        i += together;
    }
    return hipSuccess;
}

#define MCA_LINEAR_ATTENTION(T)                                                                                 \
    template size_t linear_attention_workspace<T>(const Sequences&, int, const Pass*, int);                     \
    template hipError_t linear_attention<T>(const Sequences&, int, const float*, const Pass*, int, void*, hipStream_t)

}  // namespace mca
