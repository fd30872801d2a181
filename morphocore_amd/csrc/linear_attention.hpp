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
// rows of its 16 columns in the accumulators of the state's own product. Long sequences are split into segments
// where there are too few heads to fill the chip: one launch sums every segment's state by itself, a second joins them (both
// read b and c only), then every segment starts from its state.
//
// Products. Operands of 16 bits are one bfloat16 term (bfloat16) or two (float16, exactly), float32 is three; scores, states and decayed rows
// of c, which are float32, are split into three, so that nothing is rounded to fewer bits before the result. (With two terms for scores and
// states, 2^-16 of each, one bfloat16 result in a hundred was its neighbour, 1.0e-4 of the results by norm instead of 4.3e-5; 32768 tokens of 32
// heads took 480 us instead of 515, 4 x 4096 of 16 with their gradients 500 instead of 550.) Products of terms whose places add up to more than
// 2 are left out: below 2^-22 of the magnitudes at the very most.
//
// Layouts. Of a 16 x 16 x 32 product lane l gives the first operand's row l % 16 and the second's column l % 16 with 8 values
// of the summed axis from 8 (l / 16) on, and gets column l % 16, rows 4 (l / 16) to + 3. The transposing LDS read takes a row's 4-value
// groups from wherever a lane points, so the state's 32 rows of two products are numbered such that a lane's two
// results are 8 neighbouring rows: the first operand of a S, with no exchange between lanes. Rows of the staged tiles are units of 8 values whose order
// changes from row to row, so that row and transposing reads both spread over the banks.
//
// Measured, bfloat16, heads of 128 x 128. 32768 tokens of 32 heads, 128 columns a workgroup, two a CU: 150 us for the segments' states, 12
// for the join and 350 to 360 for the results, where reading and writing alone take 255 and the instructions alone 328, of which 122 matrix and
// about 800 vector ones a wave and chunk, which hardly overlap on a SIMD. 4 x 4096 tokens of 16 heads, 64 columns a workgroup: 44, 7 and 124
// us; the backward's three passes in one launch 419, not split. float32 goes by chunks of 32 rows: 8 x 4096 tokens of 4 heads of 16 x 16 take
// 12, 6 and 21 us, bound by the 3 us that one chunk's steps take after another.
#pragma once

#include <cmath>

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

// A value that every lane has, in a scalar register.
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

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

    Decay() = default;
    __device__ __forceinline__ Decay(float log_decay, double n)
    {
        const double d = exp((double)log_decay * n);
        hi = uniform((float)d), lo = uniform(d < 1e30 ? (float)(d - (double)hi) : 0.0f);
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
// needs no sum over the spans before it (and leaves some numbers without rows). The state after a segment has a slot in the workspace,
// unless it is its sequence's last: of packed rows, that of its first row over `rows`, which the row of the next such segment, `rows` rows
// on at least, can't share. So the workspace doesn't grow with the number of short sequences.
struct Segments
{
    int64_t rows, count, each, slots;
};

inline Segments segments_of(const Sequences& s, int64_t rows)
{
    if (s.offsets) return Segments{rows, s.tokens / rows + s.count + 2, 0, s.tokens / rows};
    const int64_t each = s.tokens > 0 ? (s.tokens + rows - 1) / rows : 1;
    return Segments{rows, s.count * each, each, s.count * each};
}

struct Segment
{
    Rows1 q;
    int64_t first, n, number;  // rows [first, first + n) of the sequence, the number-th segment of it
};

// The slot of a sequence's first segment; the others' follow.
__device__ __forceinline__ int64_t first_slot(const Sequences& s, const Segments& g, int64_t sequence, int64_t start)
{
    return s.offsets ? start / g.rows : sequence * g.each;
}

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

// DK: rows of the state (the values of a and b), W waves of 16 columns each.
template <typename T, int DK_, int W_>
struct Walk
{
    static constexpr int DK = DK_, W = W_, N = 16 * W, THREADS = W * WAVE;
    static constexpr int PL = terms_of<T>(), PS = 3;  // terms of the operands, and of scores and states
    // Rows of a chunk: what two workgroups' tiles leave room for in a CU's 160 KB, or one's.
    static constexpr int C = PL == 3 || (PL == 2 && DK == 256) ? 32 : 64;
    static constexpr int AB = C * DK * 2, V = C * N * 2, P = C * C * 2;  // bytes of a term's tile
    static constexpr int OUT = C * N * (PL == 3 ? 4 : 2), A = PL * AB > OUT ? PL * AB : OUT;  // a's tile is out's too
    static constexpr int LDS = A + PL * AB + PL * V + PS * P;
    static constexpr int64_t ALL = LDS + (2 + N + DK) * 4 + 2 * W * 8;  // with what is spoiled, and the decays
    static constexpr int64_t CUS = 256, CU_LDS = 160 * 1024;
    // Where two workgroups' tiles fit, registers are kept to what lets two run: the next chunk is loaded late.
    static constexpr bool LATE = W == 8 && LDS <= 76 * 1024;
    static constexpr int WAVES = LATE ? 4 : W >= 4 ? 2 : 1;  // a SIMD, at least
    // Workgroups that a CU runs at once, by their tiles and registers (8 waves a CU, 16 where they are kept to that).
    static constexpr int64_t BY_LDS = CU_LDS / ALL, BY_WAVES = (LATE ? 16 : 8) / W, TOGETHER = BY_LDS < BY_WAVES ? BY_LDS : BY_WAVES;
};

// Where unit x (8 values) of row r lies in a tile of U units a row. The 16 lanes that read 16 bytes each at once have rows 0 to 3 and 12 to 15 of unit
// x and rows 4 to 11 of unit x ^ 1, or the other way round: in 64 banks they lie apart, as do 4 rows' units x to x + 3.
template <int U>
__device__ __forceinline__ int unit_place(int r, int x)
{
    const int a = (r >> 2) & 1, b = (r >> 3) & 1, turn = 2 * (a ^ b) + b;
    if constexpr (U >= 16) return x ^ (4 * (r & 3) + turn);
    if constexpr (U == 8) return x ^ (4 * ((r >> 1) & 1) + turn);
    if constexpr (U == 4) return x ^ turn;
    return x ^ b;
}

template <int U>
__device__ __forceinline__ int unit_byte(int r, int x)
{
    return (r * U + unit_place<U>(r, x)) * 16;
}

// A lane's byte in row l % 16 of a tile for 8 values of the summed axis, which lies along the rows: its part of the unit is lane / 16. Of row
// + 16 n the byte is 256 U n further, of unit + 4 k it is xor 64 k (unit_place's xor commutes).
template <int U>
__device__ __forceinline__ int row_place(int l)
{
    return unit_byte<U>(l % 16, l / 16);
}

__device__ __forceinline__ bf16x8 row_fragment(const char* tile, int place, int k) { return *(const bf16x8*)(tile + (place ^ (64 * k))); }

// The same where it lies across the rows, in one of the column's 4 values that lane % 16 / 4 stands for: the lane points at 4 values of row
// 8 (lane / 16) + lane / 4 % 4, and of the one 4 rows below, which is xor 32 by the units' order.
template <int U>
__device__ __forceinline__ int column_place(int l, int unit)
{
    return unit_byte<U>(8 * (l / 16) + ((l >> 2) & 3), unit);
}

template <int U>
__device__ __forceinline__ bf16x8 column_fragment(const char* tile, int place, int k)
{
    typedef __attribute__((address_space(3))) bf16x4* lds4;
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(tile + (place ^ (64 * k))));
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(tile + (place ^ (64 * k) ^ (U > 2 ? 32 : 0)) + 64 * U));
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
    int any;          // the last chunk's number that has some
    int row;          // its first row with such a b
    int col[L::N];    // the first row with such a c, by column
    int dim[L::DK];   // whether b has one in this place
};

// The thread's number, anew at each call where registers are few (SPARE): what follows from it would be kept through the walk otherwise, and
// spilled. 32768 tokens of 32 heads take 523 us instead of 577 so; where they aren't, forming it anew costs 2 to 5%.
template <bool SPARE>
__device__ __forceinline__ int thread_now()
{
    uint32_t t = threadIdx.x;
    if constexpr (SPARE)
    {
        asm volatile("" : "+v"(t));
        t &= 1023u;
    }
    return (int)t;
}

template <bool SPARE, typename L>
__device__ __forceinline__ void clear_spoiled(Spoiled<L>& s)
{
    const int thread = thread_now<SPARE>();
    for (int i = thread; i < L::N; i += L::THREADS) s.col[i] = L::C;
    for (int i = thread; i < L::DK; i += L::THREADS) s.dim[i] = 0;
    if (thread == 0) s.row = L::C, s.any = 0;
}

// A staged tile's values that are not finite: zeros in their place, and f(row, column) for each. (The first term tells: it is cut.)
template <typename L, int COLS, bool SPARE, typename F>
__device__ __forceinline__ void take_out_spoiled(char* tile, F&& f)
{
    constexpr int U = COLS / UNIT, BYTES = L::C * COLS * 2;
#pragma unroll 1
    for (int i = thread_now<SPARE>(); i < L::C * COLS; i += L::THREADS)
    {
        const int r = i / COLS, c = i % COLS, at = unit_byte<U>(r, c / UNIT) + c % UNIT * 2;
        if ((*(const uint16_t*)(tile + at) & 0x7f80u) != 0x7f80u) continue;
        for (int p = 0; p < L::PL; ++p) *(uint16_t*)(tile + p * BYTES + at) = 0;
        f(r, c);
    }
}

// A tile of C rows on its way from memory to LDS. The units of a thread lie in one column of the tile, STEP rows apart.
template <typename T, typename L, int COLS, bool SPARE>
struct TileLoad
{
    static constexpr int U = COLS / UNIT, UNITS = L::C * U, COUNT = (UNITS + L::THREADS - 1) / L::THREADS, STEP = L::THREADS / U;
    static_assert((UNITS % L::THREADS == 0 || COUNT == 1) && STEP * U == L::THREADS);
    RawUnit<T> raw[COUNT];

    // A row's last, partial unit is read as the 8 values that end with it, and moved down by this much. `left`: the values of a row that are
    // there from the tile's first, c0, on.
    static __device__ __forceinline__ int down(int thread, int c0, int left)
    {
        const int c = thread % U * UNIT;
        return left - c >= UNIT || left - c <= 0 || c0 + left < UNIT ? 0 : UNIT - (left - c);
    }

    // The thread's first unit of a tile whose first row begins at `base`, with value c0.
    static __device__ __forceinline__ const T* begin(const T* base, int64_t stride, int c0, int left)
    {
        const int thread = thread_now<SPARE>();
        return base + thread / U * stride + (thread % U * UNIT - down(thread, c0, left));
    }

    // The chunk at `at`, which goes on to the next one: n rows; whole: all of the tile is there.
    __device__ __forceinline__ void load(const T*& at, int64_t stride, bool whole, int n, int c0, int left)
    {
        if (whole)
        {
#pragma unroll
            for (int i = 0; i < COUNT; ++i, at += STEP * stride)
            {
                if (UNITS % L::THREADS == 0 || thread_now<SPARE>() < UNITS)
                    __builtin_memcpy(raw[i].d, at, sizeof(raw[i].d));
                else  // a thread without a unit, which spoiled() asks too
#pragma unroll
                    for (int k = 0; k < RawUnit<T>::DWORDS; ++k) raw[i].d[k] = 0;
            }
        }
        else
        {
            const int thread = thread_now<SPARE>(), r = thread / U, c = thread % U * UNIT;
            const bool few = c0 + left < UNIT;  // rows of fewer than 8 values
            const T* const first = at;
#pragma unroll
            for (int i = 0; i < COUNT; ++i, at += STEP * stride)
            {
#pragma unroll
                for (int k = 0; k < RawUnit<T>::DWORDS; ++k) raw[i].d[k] = 0;
                if (!few && c < left && r + i * STEP < n) __builtin_memcpy(raw[i].d, at, sizeof(raw[i].d));
            }
            if (few && c == 0)
            {
#pragma unroll 1
                for (int j = 0; j < left; ++j)
#pragma unroll
                    for (int i = 0; i < COUNT; ++i)
                    {
                        if (r + i * STEP >= n) continue;
                        constexpr int PER = 4 / (int)sizeof(T);
                        uint32_t v;
                        if constexpr (PER == 1)
                            v = __builtin_bit_cast(uint32_t, first[i * (STEP * stride) + j]);
                        else
                            v = (uint32_t)__builtin_bit_cast(uint16_t, first[i * (STEP * stride) + j]) << (16 * (j % 2));
#pragma unroll
                        for (int k = 0; k < RawUnit<T>::DWORDS; ++k) raw[i].d[k] |= j / PER == k ? v : 0;
                    }
            }
        }
        static_assert(COUNT * STEP == L::C || COUNT == 1);
        if (COUNT * STEP != L::C) at += (L::C - COUNT * STEP) * stride;
    }

    // Whether a value is not finite.
    __device__ __forceinline__ bool spoiled() const
    {
        bool any = false;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) any |= not_finite<T>(raw[i]);
        return any;
    }

    // full: no unit is partial.
    __device__ __forceinline__ void store(char* tile, bool full, int c0, int left)
    {
        constexpr int BYTES = L::C * COLS * 2;
        const int thread = thread_now<SPARE>();
        if (!full)
        {
            const int n = down(thread, c0, left);
#pragma unroll
            for (int i = 0; i < COUNT; ++i) raw[i].shift(n);
        }
#pragma unroll
        for (int i = 0; i < COUNT; ++i)
        {
            const int u = thread + i * L::THREADS, r = u / U, x = u % U;
            if (UNITS % L::THREADS && u >= UNITS) break;
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

// Values of a segment's state of one tile, in the order in which lanes hold them.
template <typename L>
constexpr int64_t state_values()
{
    return (int64_t)L::DK * L::N;
}

// 32 rows of a tile's state from or to memory, neighbouring values by neighbouring threads.
template <typename L, bool SPARE>
__device__ __forceinline__ void move_state(float* __restrict__ lds, const States& s, int64_t state0, int row, int rows, int col, int cols, bool in)
{
    const bool by_rows = s.row_stride == 1;
#pragma unroll 1
    for (int i = thread_now<SPARE>(); i < 32 * L::N; i += L::THREADS)
    {
        const int d = by_rows ? i % 32 : i / L::N, c = by_rows ? i / 32 : i % L::N;
        const bool there = row + d < rows && col + c < cols;
        float* __restrict__ p = s.p + state0 + (row + d) * s.row_stride + (col + c) * s.col_stride;
        if (in)
            lds[d * L::N + c] = there ? *p : 0.0f;
        else if (there)
            *p = lds[d * L::N + c];
    }
}

// ONLY: the segments' own states (from 0) to the workspace, of all but the last of a sequence; no results.
template <typename T, typename L, bool ONLY>
__global__ __launch_bounds__(L::THREADS, L::WAVES) void attention_walk_kernel(Sequences seq, Segments segments, int heads,
                                                                               const float* __restrict__ log_decay, Passes passes, int tiles)
{
    constexpr int C = L::C, DK = L::DK, N = L::N, PL = L::PL, PS = L::PS, RT = C / 16, KS = C / 32, KD = DK / 32;
    constexpr int UD = DK / UNIT, UN = N / UNIT, UC = C / UNIT;
    constexpr bool SPARE = L::LATE && !ONLY;
    __shared__ __align__(16) char lds[ONLY ? PL * (L::AB + L::V) : L::LDS];
    __shared__ Spoiled<L> spoiled;
    __shared__ Decay kept[2][L::W];  // the decays of a chunk, and of the segment's last one: each wave's own, to spare registers
    char* const tb = lds;
    char* const tc = tb + PL * L::AB;
    char* const ta = ONLY ? nullptr : tc + PL * L::V;
    char* const tp = ONLY ? nullptr : ta + L::A;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const Pass& p = passes.p[blockIdx.y];
    const int s = p.backwards ? 1 : 0;
    static_assert(32 * N * 4 <= PL * (L::AB + L::V));  // 32 rows of the state on their way, which the scores outlive
    if constexpr (!ONLY)
        for (int i = threadIdx.x; i < PS * L::P / 16; i += L::THREADS) ((uint4*)tp)[i] = make_uint4(0, 0, 0, 0);  // above the diagonal they stay so
    clear_spoiled<SPARE>(spoiled);
    int chunk = 0;

    const int64_t work = segments.count * heads * tiles;
    for (int64_t item = blockIdx.x; item < work; item += gridDim.x)
    {
        const int l = thread_now<true>() % WAVE, g = l / 16;
        const int tile = (int)(item % tiles), head = (int)(item / tiles % heads);
        const int64_t at = item / tiles / heads;
        const Segment part = segment_at(seq, segments, at);
        const int64_t n_all = part.n, slot = first_slot(seq, segments, part.q.batch, part.q.start) + part.number;
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

        // Position 0's rows; the rows of later positions follow, or come before it where time runs backwards.
        const int64_t dir = s ? -1 : 1, t0 = part.q.start + (s ? part.q.length - 1 - part.first : part.first);
        auto row_base = [&](const TokenRows& r) {
            return (const T*)r.p + (seq.offsets ? 0 : part.q.batch * r.batch_stride) + t0 * r.token_stride + head / r.share * r.head_stride;
        };
        const T* pa = ONLY ? nullptr : row_base(p.a);
        const T* pb = row_base(p.b);
        const T* pc = row_base(p.c);
        const int64_t sa = dir * p.a.token_stride, sb = dir * p.b.token_stride, sc = dir * p.c.token_stride;
        pa = ONLY ? nullptr : TileLoad<T, L, DK, SPARE>::begin(pa, sa, 0, p.dim);
        pb = TileLoad<T, L, DK, SPARE>::begin(pb, sb, 0, p.dim);
        pc = TileLoad<T, L, N, SPARE>::begin(pc + col0, sc, col0, cols - col0);
        const bool wide = p.dim == DK && col0 + N <= cols, full = p.dim % UNIT == 0, full_c = col0 + N <= cols || (cols - col0) % UNIT == 0;
        struct Stage
        {
            TileLoad<T, L, DK, SPARE> a, b;
            TileLoad<T, L, N, SPARE> c;
        } stage;
        const int chunks = (int)((n_all + C - 1) / C), rest = (int)(n_all - (int64_t)(chunks - 1) * C);  // and the last one's rows
        auto load = [&](Stage& st, int i) {
            const int n = i + 1 < chunks ? C : rest;
            const bool whole = wide && n == C;
            if constexpr (!ONLY) st.a.load(pa, sa, whole, n, 0, p.dim);
            st.b.load(pb, sb, whole, n, 0, p.dim);
            st.c.load(pc, sc, whole, n, col0, cols - col0);
        };
        if (chunks > 0) load(stage, 0);

        const float lg = uniform(log_decay_of(log_decay, head)), lg2 = uniform(lg * 1.4426950408889634f);
        auto power = [&](int n) { return __builtin_amdgcn_exp2f(lg2 * (float)n); };
        const float update = p.update, read = p.read;
        const float e1 = uniform(power(1)), e16 = uniform(power(16));
        kept[0][wave] = Decay(lg, C), kept[1][wave] = Decay(lg, (double)((n_all + C - 1) % C + 1));

        // The state: from the workspace, as lanes hold it, or the pass's first, 32 rows at a time through LDS.
        f32x4 S[KD][2] = {};
        const int64_t state0 = (part.q.batch * heads + head) * p.dim * cols;
        if (!ONLY && part.number > 0)
        {
            const float* __restrict__ begin = passes.states[blockIdx.y] + (((slot - 1) * heads + head) * tiles + tile) * state_values<L>();
#pragma unroll
            for (int u = 0; u < KD; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    S[u][h] = *(const f32x4*)(begin + (((int64_t)wave * KD + u) * 2 + h) * WAVE * 4 + l * 4);
        }
        else if (!ONLY && p.first.p)
        {
            __syncthreads();
#pragma unroll
            for (int u = 0; u < KD; ++u)
            {
                move_state<L, SPARE>((float*)lds, p.first, state0, 32 * u, p.dim, col0, cols, true);
                __syncthreads();
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r) S[u][h][r] = ((const float*)lds)[(8 * g + 4 * h + r) * N + (16 * wave + l % 16)];
                __syncthreads();
            }
        }

        // Where the next chunk's result goes.
        const int64_t out_step = dir * heads * cols;
        int64_t out0 = ((row0 + t0 - part.q.start) * heads + head) * cols + col0;
        for (int i0 = 0; i0 < chunks; ++i0)
        {
            const int n = i0 + 1 < chunks ? C : rest;
            ++chunk;
            // The lane's places in LDS follow from this copy anew in every chunk: kept from chunk to chunk they would fill the registers.
            // Where registers are few, in each of its parts.
            const int lane = thread_now<true>() % WAVE;
            auto lane_now = [&] { return SPARE ? thread_now<true>() % WAVE : lane; };
            auto column_n_of = [&](int l) { return column_place<UN>(l, 2 * wave + ((l >> 1) & 1)) + 8 * (l & 1); };
            __syncthreads();
            if constexpr (!ONLY) stage.a.store(ta, full, 0, p.dim);
            stage.b.store(tb, full, 0, p.dim);
            stage.c.store(tc, full_c, col0, cols - col0);
            if ((int)stage.b.spoiled() | (int)stage.c.spoiled()) spoiled.any = chunk;
            if ((ONLY || !L::LATE) && i0 + 1 < chunks) load(stage, i0 + 1);
            __syncthreads();
            const bool spoils = spoiled.any == chunk;
            if (spoils)
            {
                take_out_spoiled<L, DK, SPARE>(tb, [&](int r, int c) {
                    spoiled.dim[c] = 1;
                    atomicMin(&spoiled.row, r);
                });
                take_out_spoiled<L, N, SPARE>(tc, [&](int r, int c) { atomicMin(&spoiled.col[c], r); });
                __syncthreads();
            }

            f32x4 o[RT] = {};
            if constexpr (!ONLY)
            {
                // Scores, decayed, in terms to LDS: tiles of 16 x 16 on and below the diagonal, by the waves in turn.
                const int l = lane_now(), g = l / 16, row_d = row_place<UD>(l), score_c = unit_byte<UC>(l % 16, g >> 1) + 8 * (g & 1);
#pragma unroll
                for (int t0 = 0; t0 < RT * (RT + 1) / 2; t0 += L::W)
                {
                    const int index = t0 + wave;
                    if (index >= RT * (RT + 1) / 2) break;
                    const int rt = index < 1 ? 0 : index < 3 ? 1 : index < 6 ? 2 : 3, ct = index - rt * (rt + 1) / 2;
                    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < KD; ++k)
                    {
                        bf16x8 fa[PL], fb[PL];
#pragma unroll
                        for (int i = 0; i < PL; ++i)
                        {
                            fa[i] = row_fragment(ta + i * L::AB + rt * (256 * UD), row_d, k);
                            fb[i] = row_fragment(tb + i * L::AB + ct * (256 * UD), row_d, k);
                        }
#pragma unroll
                        for (int i = 0; i < PL; ++i)
#pragma unroll
                            for (int j = 0; j < PL; ++j)
                                if (i + j <= 2) x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], x, 0, 0, 0);
                    }
                    // e^(i - j), of the tile on the diagonal value by value (nothing above it: no product with 0, so that a query's infinity
                    // stays in its row), of others from the lane's last row on.
                    float v[4];
                    const int gap = 16 * (rt - ct) + l % 16 - 4 * g;
                    if (rt == ct)
                    {
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] = gap - r < 0 ? 0.0f : x[r] * (power(gap - r) * (update * read));
                    }
                    else
                    {
                        float near = power(gap - 3) * (update * read);
#pragma unroll
                        for (int r = 3; r >= 0; --r, near *= e1) v[r] = x[r] * near;
                    }
                    __bf16 term[PS][4];
                    split<PS, false>(v, term);
#pragma unroll
                    for (int i = 0; i < PS; ++i)
                        *(bf16x4*)(tp + i * L::P + rt * (256 * UC) + (score_c ^ (32 * ct))) = term_vector<bf16x4>(term, i);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (!ONLY)
            {
                // a S, with the state's terms as they lie in the lanes.
                const int l = lane_now(), row_d = row_place<UD>(l);
#pragma unroll
                for (int u = 0; u < KD; ++u)
                {
                    bf16x8 fa[RT][PL];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int i = 0; i < PL; ++i) fa[rt][i] = row_fragment(ta + i * L::AB + rt * (256 * UD), row_d, u);
                    {
                        float v[UNIT];
#pragma unroll
                        for (int j = 0; j < UNIT; ++j) v[j] = S[u][j / 4][j % 4];
                        __bf16 term[PS][UNIT];
                        split<PS, false>(v, term);
#pragma unroll
                        for (int j = 0; j < PS; ++j)
                        {
                            const bf16x8 fs = term_vector<bf16x8>(term, j);
#pragma unroll
                            for (int i = 0; i < PL; ++i)
                                if (i + j <= 2)
#pragma unroll
                                    for (int rt = 0; rt < RT; ++rt) o[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fs, fa[rt][i], o[rt], 0, 0, 0);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                float reach = power(l % 16 + 1 - s) * read;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt, reach *= e16)
                    o[rt] *= reach;
                __syncthreads();
            }

            const float nan = __builtin_nanf("");
            if constexpr (!ONLY)
            {
                // Scores times c, and out.
                const int l = lane_now(), g = l / 16, row_c = row_place<UC>(l), column_n = column_n_of(l);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                {
                    bf16x8 fc[PL];
#pragma unroll
                    for (int i = 0; i < PL; ++i) fc[i] = column_fragment<UN>(tc + i * L::V + ks * (512 * UN), column_n, 0);
#pragma unroll
                    for (int j = 0; j < PS; ++j)
#pragma unroll
                        for (int rt = 2 * ks; rt < RT; ++rt)
                        {
                            const bf16x8 fp = row_fragment(tp + j * L::P + rt * (256 * UC), row_c, ks);
#pragma unroll
                            for (int i = 0; i < PL; ++i)
                                if (i + j <= 2) o[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fc[i], fp, o[rt], 0, 0, 0);
                        }
                }
                if (spoils)
                {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                    {
                        const int from = min(spoiled.row, spoiled.col[16 * wave + 4 * g + r]);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
                            if (16 * rt + l % 16 >= from) o[rt][r] = nan;
                    }
                }
                typedef T Tx4 __attribute__((ext_vector_type(4)));
                constexpr int E = 16 / (int)sizeof(T), UO = N / E;
                const bool rows_at_once = !p.out32 && p.out;
                if (p.out32)
                {
                    const int c = col0 + 16 * wave + 4 * g;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                    {
                        if (16 * rt + l % 16 >= n) continue;
                        float* __restrict__ to = p.out32 + out0 + (16 * rt + l % 16) * out_step + 16 * wave + 4 * g;
                        if (c + 4 <= cols)
                            __builtin_memcpy(to, &o[rt], 16);
                        else
#pragma unroll
                            for (int j = 0; j < 3; ++j)
                                if (c + j < cols) to[j] = o[rt][j];
                    }
                }
                else if (rows_at_once)
                {
                    // Through a's tile, which nobody reads any more, so that whole rows go to memory at once.
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                    {
                        const Tx4 v = __builtin_convertvector(o[rt], Tx4);
                        __builtin_memcpy(ta + rt * (256 * UO) + unit_byte<UO>(l % 16, (16 * wave + 4 * g) / E) + (4 * g) % E * (int)sizeof(T), &v, sizeof(v));
                    }
                }
                // Before out's stores: loads behind them would be waited for with them.
                __builtin_amdgcn_sched_barrier(0);
                if (L::LATE && i0 + 1 < chunks) load(stage, i0 + 1);
                __builtin_amdgcn_sched_barrier(0);
                if (rows_at_once)
                {
                    __syncthreads();
                    T* __restrict__ out = (T*)p.out + out0;
                    const int thread = thread_now<SPARE>();
#pragma unroll
                    for (int i = 0; i < C * UO / L::THREADS; ++i)
                    {
                        const int u = thread + i * L::THREADS, r = u / UO, x = u % UO;
                        if (r >= n) break;
                        T* __restrict__ to = out + r * out_step + x * E;
                        const uint4 v = *(const uint4*)(ta + unit_byte<UO>(r, x));
                        if (col0 + (x + 1) * E <= cols)
                        {
                            __builtin_memcpy(to, &v, 16);
                        }
                        else
                        {
                            const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int j = 0; j < E - 1; ++j)
                                if (col0 + x * E + j < cols)
                                {
                                    if constexpr (sizeof(T) == 4)
                                        to[j] = __builtin_bit_cast(T, d[j]);
                                    else
                                        to[j] = __builtin_bit_cast(T, (uint16_t)(d[j / 2] >> (16 * (j % 2))));
                                }
                        }
                    }
                }
                out0 += C * out_step;
                __builtin_amdgcn_sched_barrier(0);
            }

            // The state after the chunk.
            const int l = lane_now(), g = l / 16, column_d = column_place<UD>(l, l & 3), column_n = column_n_of(l);
            const bool whole = n == C;
            const Decay decay = kept[i0 + 1 < chunks ? 0 : 1][wave];
#pragma unroll
            for (int u = 0; u < KD; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[u][h][r] = decay.of(S[u][h][r]);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
            {
                bf16x8 fd[3];
                // e^(n - 1 + s - j) of the lane's last row j = 32 ks + 8 g + 7 (rows behind the chunk's end are 0).
                const int past = n - 1 + s - (32 * ks + 8 * g + 7);
                {
                    float v[UNIT] = {};
#pragma unroll
                    for (int i = 0; i < PL; ++i)
                    {
                        const bf16x8 fc = column_fragment<UN>(tc + i * L::V + ks * (512 * UN), column_n, 0);
#pragma unroll
                        for (int j = 0; j < UNIT; ++j) v[j] += (float)fc[j];
                    }
                    if (whole)
                    {
                        float w = power(past) * update;
#pragma unroll
                        for (int j = UNIT - 1; j >= 0; --j, w *= e1) v[j] *= w;
                    }
                    else
                    {
#pragma unroll
                        for (int j = 0; j < UNIT; ++j) v[j] *= past + 7 - j >= 0 ? power(past + 7 - j) * update : 0.0f;
                    }
                    __bf16 term[3][UNIT];
                    split<3, false>(v, term);
#pragma unroll
                    for (int i = 0; i < 3; ++i) fd[i] = term_vector<bf16x8>(term, i);
                }
                // b's columns for 32 rows of the state at a time.
#pragma unroll
                for (int u = 0; u < KD; ++u)
                {
                    bf16x8 fb[2][PL];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < PL; ++i) fb[h][i] = column_fragment<UD>(tb + i * L::AB + ks * (512 * UD) + 8 * h, column_d, u);
#pragma unroll
                    for (int j = 0; j < 3; ++j)
#pragma unroll
                        for (int i = 0; i < PL; ++i)
                            if (i + j <= 2)
#pragma unroll
                                for (int h = 0; h < 2; ++h) S[u][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[h][i], fd[j], S[u][h], 0, 0, 0);
                    if (L::LATE || u % 2) __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (spoils)
            {
                const int by = spoiled.col[16 * wave + l % 16];
#pragma unroll
                for (int u = 0; u < KD; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (by < C || spoiled.dim[32 * u + 8 * g + 4 * h + r]) S[u][h][r] = nan;
                __syncthreads();
                clear_spoiled<SPARE>(spoiled);
            }
        }

        if (ONLY)
        {
            float* __restrict__ end = passes.states[blockIdx.y] + ((slot * heads + head) * tiles + tile) * state_values<L>();
#pragma unroll
            for (int u = 0; u < KD; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *(f32x4*)(end + (((int64_t)wave * KD + u) * 2 + h) * WAVE * 4 + l * 4) = S[u][h];
        }
        else if (last && p.last.p)
        {
            __syncthreads();
#pragma unroll
            for (int u = 0; u < KD; ++u)
            {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r) ((float*)lds)[(8 * g + 4 * h + r) * N + (16 * wave + l % 16)] = S[u][h][r];
                __syncthreads();
                move_state<L, SPARE>((float*)lds, p.last, state0, 32 * u, p.dim, col0, cols, false);
                __syncthreads();
            }
        }
    }
}

// Turns the segments' own states into the states after them, sequence by sequence: 4 values of a tile's state a thread.
template <typename L>
__global__ __launch_bounds__(BLOCK) void attention_join_kernel(Sequences seq, Segments segments, int heads, const float* __restrict__ log_decay,
                                                               Passes passes, int tiles)
{
    constexpr int QUADS = (int)state_values<L>() / 4, BLOCKS = (QUADS + BLOCK - 1) / BLOCK;
    const Pass& p = passes.p[blockIdx.y];
    const int64_t work = seq.count * heads * tiles * BLOCKS;
    for (int64_t item = blockIdx.x; item < work; item += gridDim.x)
    {
        const int block = (int)(item % BLOCKS), tile = (int)(item / BLOCKS % tiles), head = (int)(item / BLOCKS / tiles % heads);
        const int64_t q = item / BLOCKS / tiles / heads;
        int64_t length = seq.tokens, start = 0;
        if (seq.offsets)
        {
            const int64_t end = offset_at(seq, q + 1);
            start = offset_at(seq, q);
            length = end > start ? end - start : 0;
            if (length <= segments.rows) continue;
        }
        const int64_t count = (length + segments.rows - 1) / segments.rows - 1;  // all but the last
        const int e = block * BLOCK + threadIdx.x;
        if (e >= QUADS) continue;
        const int64_t stride = (int64_t)heads * tiles * QUADS;
        f32x4* __restrict__ state = (f32x4*)passes.states[blockIdx.y] + ((first_slot(seq, segments, q, start) * heads + head) * tiles + tile) * QUADS + e;
        constexpr int AHEAD = 8;
        f32x4 own[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) own[k] = state[(k < count ? k : count - 1) * stride];
        // The values' place: see attention_walk_kernel's workspace.
        const int l = e % WAVE, h = e / WAVE % 2, u = e / WAVE / 2 % (L::DK / 32), w = e / WAVE / 2 / (L::DK / 32);
        const int d = 32 * u + 8 * (l / 16) + 4 * h, c = tile * L::N + 16 * w + l % 16;
        const Decay decay(log_decay_of(log_decay, head), (double)segments.rows);
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p.first.p && c < p.cols)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (d + r < p.dim) x[r] = p.first.p[(q * heads + head) * p.dim * p.cols + (d + r) * p.first.row_stride + c * p.first.col_stride];
        for (int64_t i = 0; i < count;)
        {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
            {
                if (i + k >= count) break;
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = decay.of(x[r]) + own[k][r];
                state[(i + k) * stride] = x;
            }
            i += AHEAD;
            if (i >= count) break;
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) own[k] = state[(i + k < count ? i + k : count - 1) * stride];
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Launches.
// ------------------------------------------------------------------------------------------------

template <typename L>
int tiles_of(const Pass& p)
{
    return (p.cols + L::N - 1) / L::N;
}

// How long sequences are split: the rows of a segment, and an estimate of the time that it takes.
struct Plan
{
    Segments segments;
    double cost;
};

// The estimate, in half the time that two workgroups of 128 columns on a CU take for a chunk each: a chunk takes n workgroups of W waves
// together 0.3 + 0.106 n W, a CU takes its workgroups in rounds of as many as it runs at once, and a workgroup's own cost (its first loads,
// its state) is that of 2 + W / 2 chunks; where sequences are split, the first launch adds 0.4 of the second's time and the join 2. The
// lengths of packed sequences are not known here: their mean length, each rounded up to a chunk more, counts for the rounds, and one of 32
// times the mean for what goes on behind them.
template <typename L>
Plan plan_of(const Sequences& seq, int heads, const Pass& p)
{
    constexpr double OWN = 2.0 + 0.5 * L::W, JOIN = 2.0;
    auto chunk = [](int64_t workgroups) { return workgroups ? 0.3 + 0.106 * (double)workgroups * L::W : 0.0; };
    const int64_t walks = (seq.offsets ? 1 : seq.count) * (int64_t)heads * tiles_of<L>(p) * p.together;
    const int64_t chunks = seq.tokens > 0 ? (seq.tokens + L::C - 1) / L::C : 1;
    const int64_t longest = !seq.offsets || seq.count <= 32 ? chunks : (32 * (chunks / seq.count + 1) < chunks ? 32 * (chunks / seq.count + 1) : chunks);
    int64_t best = chunks;
    double least = 1e300;
    auto consider = [&](int64_t size) {
        const int64_t parts = (chunks + size - 1) / size, items = walks * (seq.offsets ? parts + seq.count : parts);
        const int64_t each = (items + L::CUS - 1) / L::CUS, rounds = each / L::TOGETHER, rest = each % L::TOGETHER;
        const double most = (double)(size < longest ? size : longest);
        const double mean = seq.offsets ? fmin(most, (double)(chunks + seq.count) / (double)(parts + seq.count)) : most;
        const double time = (mean + OWN) * ((double)rounds * chunk(L::TOGETHER) + chunk(rest)) + (most - mean) * chunk(rounds > 0 ? L::TOGETHER : rest);
        const double cost = size >= chunks ? time : 1.4 * time + JOIN;
        if (cost < least) least = cost, best = size;
    };
    consider(chunks);
    for (int64_t size = chunks - chunks / 8; size > 16; size = size - size / 8) consider(size);
    for (int64_t size = chunks <= 16 ? chunks - 1 : 16; size >= 2; --size) consider(size);
    return Plan{segments_of(seq, best * L::C), least};
}

// f(the shape of a pass): as few columns a workgroup as hold the pass's. Of more than 64, 128 where two such workgroups don't fit a CU (the
// scores would be formed twice: 88 us instead of 67, forwards, for 4999 tokens of 6 heads of 96 x 77 in float16) and for sequences of one chunk, whose
// scores are most of the work (500 of 33 tokens of 8 heads of 64 x 128 in bfloat16: 84 us by 128, 125 by 64; 2000 of 60 of 16 heads of 128 x 128: 1100
// and 1190), otherwise 128 or 64 by the estimate: 32768 tokens of 32 heads of 128 x 128 in bfloat16 take 516 us by 128 and 612 by 64; 12001 of 41
// sequences take 185 and 182.
template <typename T, typename F>
hipError_t by_walk(const Sequences& seq, int heads, const Pass& p, F&& f)
{
#define MCA_WALK(DK, W) return f(Walk<T, DK, W>())
#define MCA_WALKS(DK)                                                                                                            \
    do                                                                                                                           \
    {                                                                                                                            \
        if (p.cols <= 64) MCA_WALK(DK, 4);                                                                                       \
        if (Walk<T, DK, 8>::LATE && seq.tokens > Walk<T, DK, 8>::C &&                                                            \
            plan_of<Walk<T, DK, 4>>(seq, heads, p).cost < plan_of<Walk<T, DK, 8>>(seq, heads, p).cost)                           \
            MCA_WALK(DK, 4);                                                                                                     \
        MCA_WALK(DK, 8);                                                                                                         \
    } while (0)
    if (p.dim <= 64 && p.cols <= 32)
    {
        if (p.dim <= 32)
        {
            if (p.cols <= 16) MCA_WALK(32, 1);
            MCA_WALK(32, 2);
        }
        if (p.cols <= 16) MCA_WALK(64, 1);
        MCA_WALK(64, 2);
    }
    if (p.dim <= 32) MCA_WALKS(32);
    if (p.dim <= 64) MCA_WALKS(64);
    if (p.dim <= 128) MCA_WALKS(128);
    MCA_WALKS(256);
#undef MCA_WALKS
#undef MCA_WALK
}

inline bool joins(const Sequences& seq, const Segments& s) { return seq.tokens > s.rows; }

// Bytes of the segments' states of a pass.
template <typename L>
size_t walk_states(const Sequences& seq, int heads, const Pass& p)
{
    const Segments s = plan_of<L>(seq, heads, p).segments;
    return joins(seq, s) ? align_up((size_t)(s.slots * heads * tiles_of<L>(p) * state_values<L>()) * sizeof(float)) : 0;
}

template <typename T>
size_t linear_attention_workspace(const Sequences& seq, int heads, const Pass* passes, int count)
{
    size_t bytes = 0;
    for (int i = 0; i < count; ++i)
        (void)by_walk<T>(seq, heads, passes[i], [&](auto walk) {
            bytes += walk_states<decltype(walk)>(seq, heads, passes[i]);
            return hipSuccess;
        });
    return bytes;
}

template <typename T>
hipError_t linear_attention(const Sequences& seq, int heads, const float* log_decay, const Pass* passes, int count, void* workspace,
                            hipStream_t stream)
{
    if ((seq.offsets ? seq.count + seq.tokens : seq.count) <= 0 || heads <= 0) return hipSuccess;
    char* ws = (char*)workspace;
    for (int i = 0; i < count;)
    {
        // Passes of the same shape go together.
        int together = 1;
        while (i + together < count && passes[i + together].dim == passes[i].dim && passes[i + together].cols == passes[i].cols) ++together;
        const hipError_t err = by_walk<T>(seq, heads, passes[i], [&](auto walk) {
            using L = decltype(walk);
            const Segments s = plan_of<L>(seq, heads, passes[i]).segments;
            const int tiles = tiles_of<L>(passes[i]);
            const bool split = joins(seq, s);
            Passes all = {};
            for (int k = 0; k < together; ++k)
            {
                all.p[k] = passes[i + k];
                if (!split) continue;
                all.states[k] = (float*)ws;
                ws += walk_states<L>(seq, heads, passes[i + k]);
            }
            const int64_t work = s.count * heads * tiles, most = 1 << 20;
            const dim3 grid((unsigned)(work < most ? work : most), together);
            if (split)
            {
                attention_walk_kernel<T, L, true><<<grid, L::THREADS, 0, stream>>>(seq, s, heads, log_decay, all, tiles);
                const int64_t values = seq.count * heads * tiles * ((state_values<L>() / 4 + BLOCK - 1) / BLOCK);
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
