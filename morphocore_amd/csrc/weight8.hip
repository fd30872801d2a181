// The weight gradient of a linear layer from its packed input:
//   grad_weight[n, k] = sum over the rows m of grad_y[m, n] * value(codes[m, k]).
//
// A matrix product over the rows on the bfloat16 matrix instructions. A packed value (4 significant bits
// times a power of two) is exact in bfloat16, and grad_y is split by truncation into as many bfloat16 terms
// as its significand takes: bfloat16 itself, float16 two, float32 three; every product is then exact (but for
// what a float32 value below 2^-110 has under bfloat16's smallest, 2^-133) and the sums are float32. Three bfloat16
// products still run several times as fast as one float32 product.
//
// Both operands lie with the summed axis as the slow one, so a wave reads its fragments from LDS with the
// transposing read (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 columns and each gets a column). A row
// of a staged tile is stored in groups of 16 columns (32 bytes), whose order changes from row to row so that
// the 4 rows of two neighbouring groups, which 32 lanes read at once, lie in different banks. Tiles are double-buffered in LDS: the next rows'
// loads are issued before the products of the present ones and stored after them. Codes become bfloat16 on
// the way into LDS, once for the workgroup.
//
// Rows are split over workgroups where the output has too few tiles for the 256 CUs; each split writes its
// float32 sums to a slot, and the slots are added in a fixed order (no atomics: the same result every time).
//
// Measured: 8192 x 4096 x 4096 (rows, out, columns) bfloat16 248 us among other work, 1109 TFLOP/s (234 to 244 launched back to
// back), where the library's bfloat16 product of 8192^3, the fastest measured, runs at 1202 and its product of these operands
// unpacked takes 287 us; back to back float16 452 to 463 us (1187 to 1216 TFLOP/s of bfloat16 products), float32 667 to 681 us
// (1211 to 1237). 524288 x 64 x 64 float32 36 us (4.5 TB/s), bound by HBM, and 6 for the slots. Tiles in between are bound by
// latency: 5003 x 1111 x 777 float16 32 us and 6.
#include "block8.hpp"
#include "launch.hpp"
#include "mixer.hpp"

namespace mca
{

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// bfloat16 terms of a grad_y value.
template <typename T>
constexpr int planes_of()
{
    return std::is_same_v<T, float> ? 3 : std::is_same_v<T, _Float16> ? 2 : 1;
}

// N x K outputs of a workgroup, M rows staged at a time, D steps of loads in flight, waves along N and K.
template <int N_, int K_, int M_, int D_, int WN_, int WK_>
struct WeightTile
{
    static constexpr int N = N_, K = K_, M = M_, D = D_, WN = WN_, WK = WK_;
    static constexpr int THREADS = WN * WK * WAVE;
    static constexpr int FN = N / WN / 32, FK = K / WK / 32;  // 32 x 32 fragments of a wave
};

// The place of column group g (of 16) in row m of a staged tile of C columns.
template <int C>
__device__ __forceinline__ int group_place(int g, int m)
{
    return C >= 128 ? g ^ (2 * (m & 3)) : g ^ (m & 2);
}

// Byte of column c (a multiple of 8) of row m in a staged tile of C columns.
template <int C>
__device__ __forceinline__ int tile_byte(int m, int c)
{
    return m * (C * 2) + group_place<C>(c / 16, m) * 32 + (c & 8) * 2;
}

// A lane's 8 values of the summed axis (rows m0 + 8 (lane / 32) ..) for column c0 + lane % 32.
template <int C>
__device__ __forceinline__ bf16x8 read_fragment(const char* tile, int m0, int c0)
{
    const int l = threadIdx.x % WAVE, r = (l / 4) & 3;
    const int group = group_place<C>(c0 / 16 + ((l / 16) & 1), r);
    const char* p = tile + (m0 + 8 * (l / 32) + r) * (C * 2) + group * 32 + (l & 3) * 8;
    typedef __attribute__((address_space(3))) bf16x4* lds4;
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)p);
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(p + 4 * C * 2));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The bfloat16 terms of 8 values, each the leading 8 bits of what the ones before leave.
template <typename T, int P>
__device__ __forceinline__ void split_unit(const RawUnit<T>& raw, bf16x8 (&term)[P])
{
    if constexpr (P == 1)
    {
        term[0] = __builtin_bit_cast(bf16x8, raw);
    }
    else
    {
#pragma unroll
        for (int j = 0; j < UNIT; ++j)
        {
            float v = raw[j];
#pragma unroll
            for (int i = 0; i < P; ++i)
            {
                const uint32_t bits = __float_as_uint(v) & 0xffff0000u;
                term[i][j] = __builtin_bit_cast(__bf16, (uint16_t)(bits >> 16));
                if (i + 1 == P) break;
                const float rest = v - __uint_as_float(bits);
                // An infinity is its own first term; what it leaves must be no NaN. (Of float16 the rest is at most 65504, and
                // for the NaN that an infinity leaves the median is -65504, which the infinite products swallow.)
                if constexpr (std::is_same_v<T, _Float16>)
                    v = __builtin_amdgcn_fmed3f(rest, -65504.0f, 65504.0f);
                else
                    v = i == 0 && fabsf(v) == __builtin_inff() ? 0.0f : rest;
            }
        }
    }
}

// One tile of the sums over rows [m0, m1), m0 = split * split_rows, to out + split * out_rows * cols.
//
// Every load is made, of an address within the arrays: rows past m1 read row m1 - 1 (grad_y's then count
// as 0; a value of that row that is not finite has already made its column so), and the last tile of an
// axis is moved back to end with it, its repeated outputs left to the tile before. What no tile covers
// whole (fewer columns than a tile's, packed columns that are no multiple of 8) reads the row's last 8
// values for a partial unit and moves them down; columns past the end hold anything, since they only
// reach outputs that are not stored. ANY: arrays of fewer than 8 columns, read value by value.
template <typename T, typename OT, typename L, bool ANY>
__global__ __launch_bounds__(L::THREADS) void grad_weight8_kernel(const T* __restrict__ gy, int64_t gys, const uint8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ scales, OT* __restrict__ out, int64_t rows,
                                                                  int64_t split_rows, int out_rows, int cols, int tiles_n, int tiles_k)
{
    constexpr int P = planes_of<T>(), THREADS = L::THREADS;
    constexpr int A_BYTES = L::M * L::N * 2, B_BYTES = L::M * L::K * 2, BUFFER = P * A_BYTES + B_BYTES;
    constexpr int UA = L::N / UNIT, UB = L::K / UNIT;               // units of a row
    constexpr int NA = L::M * UA / THREADS, NB = L::M * UB / THREADS;  // units of a thread
    static_assert(NA * THREADS == L::M * UA && NB * THREADS == L::M * UB);
    __shared__ __align__(16) char lds[2][BUFFER];

    const int tiles = tiles_n * tiles_k, work = xcd_work_index(blockIdx.x, gridDim.x);
    const int split = work / tiles, tile = work % tiles;
    const int first_n = tile / tiles_k * L::N, first_k = tile % tiles_k * L::K, nb = blocks_of(cols);
    const int n0 = max(0, min(first_n, out_rows - L::N)), k0 = max(0, min(first_k, units_of(cols) * UNIT - L::K));
    const int64_t m0 = split * split_rows;
    const int mrows = (int)((m0 + split_rows < rows ? m0 + split_rows : rows) - m0);
    const T* __restrict__ gy0 = gy + m0 * gys;
    const uint8_t* __restrict__ codes0 = codes + m0 * cols;
    const uint8_t* __restrict__ scales0 = scales + m0 * nb;
    const bool part_n = out_rows < L::N && out_rows % UNIT;

    struct Stage
    {
        RawUnit<T> a[NA];
        uint2 b[NB];
        uint32_t s[NB];
    };
    // Whole steps: a thread's units lie in one column, STEP_A (STEP_B) rows apart.
    constexpr int STEP_A = THREADS / UA, STEP_B = THREADS / UB;
    static_assert(STEP_A * UA == THREADS && STEP_B * UB == THREADS);
    const T* __restrict__ pa = gy0 + (int64_t)(threadIdx.x / UA) * gys + min(n0 + (int)threadIdx.x % UA * UNIT, out_rows - UNIT);
    const int col_b = k0 + (int)threadIdx.x % UB * UNIT;
    const uint8_t* __restrict__ pb = codes0 + (int64_t)(threadIdx.x / UB) * cols + min(col_b, cols - UNIT);
    const int down_b = 8 * min(max(col_b - (cols - UNIT), 0), UNIT - 1);
    const uint8_t* __restrict__ ps = scales0 + (int64_t)(threadIdx.x / UB) * nb + min(col_b / MX_BLOCK, nb - 1);
    auto load = [&](auto whole, int m, Stage& st) {
        if (decltype(whole)::value || (!ANY && m + L::M <= mrows))
        {
            const T* __restrict__ a = pa + m * gys;
            const uint8_t* __restrict__ b = pb + (int64_t)m * cols;
            const uint8_t* __restrict__ s = ps + (int64_t)m * nb;
#pragma unroll
            for (int i = 0; i < NA; ++i) __builtin_memcpy(st.a[i].d, a + (int64_t)(i * STEP_A) * gys, sizeof(st.a[i].d));
#pragma unroll
            for (int i = 0; i < NB; ++i)
            {
                __builtin_memcpy(&st.b[i], b + (int64_t)(i * STEP_B) * cols, sizeof(st.b[i]));
                st.s[i] = s[(int64_t)(i * STEP_B) * nb];
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < NA; ++i)
        {
            const int u = threadIdx.x + i * THREADS, c = n0 + u % UA * UNIT, row = min(m + u / UA, mrows - 1);
            if constexpr (ANY)
                load_raw(gy0 + row * gys + c, c, out_rows - c, st.a[i]);
            else
                __builtin_memcpy(st.a[i].d, gy0 + row * gys + min(c, out_rows - UNIT), sizeof(st.a[i].d));
        }
#pragma unroll
        for (int i = 0; i < NB; ++i)
        {
            const int u = threadIdx.x + i * THREADS, c = k0 + u % UB * UNIT;
            const int64_t row = min(m + u / UB, mrows - 1);
            if constexpr (ANY)
                st.b[i] = load_codes(codes0 + row * cols + c, c, cols - c);
            else
                __builtin_memcpy(&st.b[i], codes0 + row * cols + min(c, cols - UNIT), sizeof(st.b[i]));
            st.s[i] = scales0[row * nb + min(c / MX_BLOCK, nb - 1)];
        }
    };
    // whole: rows and columns are all there.
    auto store = [&](auto whole, int m, Stage& st, char* buffer) {
        constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
        for (int i = 0; i < NA; ++i)
        {
            const int u = threadIdx.x + i * THREADS;
            RawUnit<T>& raw = st.a[i];
            if (!WHOLE && !ANY && part_n) raw.shift(min(max(n0 + u % UA * UNIT - (out_rows - UNIT), 0), UNIT - 1));
            if (!WHOLE && m + L::M > mrows)
            {
#pragma unroll
                for (int j = 0; j < RawUnit<T>::DWORDS; ++j) raw.d[j] = m + u / UA < mrows ? raw.d[j] : 0;
            }
            bf16x8 term[P];
            split_unit<T, P>(raw, term);
#pragma unroll
            for (int q = 0; q < P; ++q) *(bf16x8*)(buffer + q * A_BYTES + tile_byte<L::N>(u / UA, u % UA * UNIT)) = term[q];
        }
#pragma unroll
        for (int i = 0; i < NB; ++i)
        {
            const int u = threadIdx.x + i * THREADS;
            const float scale = scale_of(st.s[i]);
            uint64_t q = (uint64_t)st.b[i].y << 32 | st.b[i].x;
            if constexpr (!ANY) q >>= down_b;
            typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
            const bf16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)q, scale, false);
            const bf16x2 v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)q, scale, true);
            const bf16x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)(q >> 32), scale, false);
            const bf16x2 v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)(q >> 32), scale, true);
            const bf16x8 v = {v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
            *(bf16x8*)(buffer + P * A_BYTES + tile_byte<L::K>(u / UB, u % UB * UNIT)) = v;
        }
    };

    const int wave = threadIdx.x / WAVE, wn = wave / L::WK * (L::N / L::WN), wk = wave % L::WK * (L::K / L::WK);
    // The first terms' sums; float32's further terms have sums of their own, so that the rounding of the large
    // ones does not swallow them.
    constexpr int SUMS = P == 3 ? 2 : 1;
    f32x16 acc[SUMS][L::FN][L::FK] = {};
    auto products = [&](const char* buffer) {
        // The fragments of the next 16 rows (and the next term) are read while the present ones are multiplied.
        constexpr int S = L::M / 16 * P;  // sets of A fragments, small terms first
        bf16x8 fa[2][L::FN], fb[2][L::FK];
        auto read = [&](int t) {
            const int i = t / P * 16, q = P - 1 - t % P;
            if (t % P == 0)
#pragma unroll
                for (int k = 0; k < L::FK; ++k) fb[t / P % 2][k] = read_fragment<L::K>(buffer + P * A_BYTES, i, wk + 32 * k);
#pragma unroll
            for (int n = 0; n < L::FN; ++n) fa[t % 2][n] = read_fragment<L::N>(buffer + q * A_BYTES, i, wn + 32 * n);
        };
        read(0);
#pragma unroll
        for (int t = 0; t < S; ++t)
        {
            if (t + 1 < S) read(t + 1);
            const int sum = t % P < P - 1 ? SUMS - 1 : 0;
#pragma unroll
            for (int n = 0; n < L::FN; ++n)
#pragma unroll
                for (int k = 0; k < L::FK; ++k)
                    acc[sum][n][k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[t % 2][n], fb[t / P % 2][k], acc[sum][n][k], 0, 0, 0);
            // Two reads to a product, so that neither unit waits for the other's burst.
            if (t + 1 < S)
            {
#pragma unroll
                for (int g = 0; g < L::FN * L::FK; ++g)
                {
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                }
            }
        }
    };
    // Before step m (in lds[turn]): step m + M is in st[d + 1], for the other buffer when the products are done,
    // and st[d], which step m has left, is free for step m + D M.
    using Whole = std::true_type;
    using Any = std::false_type;
    Stage st[L::D];
#pragma unroll
    for (int d = 0; d < L::D; ++d) load(Any(), d * L::M, st[d]);
    store(Any(), 0, st[0], lds[0]);
    __syncthreads();
    int turn = 0, m = 0;
    if (!ANY && !part_n)
        while (m + 2 * L::D * L::M <= mrows)  // no branch between the loads, products and stores of a step
        {
#pragma unroll
            for (int d = 0; d < L::D; ++d, m += L::M, turn ^= 1)
            {
                load(Whole(), m + L::D * L::M, st[d]);
                __builtin_amdgcn_sched_barrier(0);  // the loads first: the compiler would move them to their use
                products(lds[turn]);
                store(Whole(), m + L::M, st[(d + 1) % L::D], lds[turn ^ 1]);
                __syncthreads();
            }
        }
    while (m < mrows)
    {
#pragma unroll
        for (int d = 0; d < L::D; ++d, turn ^= 1)
        {
            if (m + L::D * L::M < mrows) load(Any(), m + L::D * L::M, st[d]);
            products(lds[turn]);
            m += L::M;
            if (m >= mrows) break;
            store(Any(), m, st[(d + 1) % L::D], lds[turn ^ 1]);
            __syncthreads();
        }
    }

    // A lane holds column lane % 32 and rows 8 (r / 4) + 4 (lane / 32) + r % 4 of a fragment.
    const int l = threadIdx.x % WAVE;
    OT* __restrict__ o = out + (int64_t)split * out_rows * cols;
#pragma unroll
    for (int n = 0; n < L::FN; ++n)
#pragma unroll
        for (int k = 0; k < L::FK; ++k)
        {
            const int col = k0 + wk + 32 * k + l % 32;
            if (col < first_k || col >= cols) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r)
            {
                const int row = n0 + wn + 32 * n + 8 * (r / 4) + 4 * (l / 32) + r % 4;
                float v = acc[0][n][k][r];
                if constexpr (SUMS == 2) v += acc[1][n][k][r];
                if (row >= first_n && row < out_rows) o[(int64_t)row * cols + col] = (OT)v;
            }
        }
}

using WideTile = WeightTile<256, 256, 32, 2, 2, 4>;
using TallTile = WeightTile<128, 256, 32, 2, 2, 4>;
using MiddleTile = WeightTile<128, 128, 32, 2, 4, 2>;
using SmallTile = WeightTile<64, 64, 64, 2, 2, 2>;

struct WeightPlan
{
    int tile;  // 0 wide, 1 tall, 2 middle, 3 small
    int tiles_n, tiles_k, splits;
    int64_t split_rows;
};

// What a row of a workgroup's sums takes, in ns: of one workgroup alone on its CU, and of each of several (at most
// per_cu). Measured over shapes from 64 x 64 to 4096 x 4096. Larger tiles read and convert less for a product:
// 8192 x 4096 x 4096 takes 234 us of bfloat16 with wide tiles, 292 with tall and 339 with middle ones; 452 of float16 with
// tall and 534 with middle ones; 667 against 834 of float32, whose conversion costs most. 4096 x 4096 x 2048 of bfloat16
// has too few wide tiles for the CUs: 77 us with tall ones, 91 with middle ones. The wide one's registers hold
// bfloat16's operands only.
struct TileCost
{
    int side_n, side_k, step, per_cu;
    double alone, shared;
};
constexpr TileCost TILE_COST[3][4] = {
    {{256, 256, 32, 1, 30.0, 30.0}, {128, 256, 32, 1, 18.0, 18.0}, {128, 128, 32, 2, 13.0, 9.0}, {64, 64, 64, 4, 6.5, 5.2}},  // bfloat16
    {{}, {128, 256, 32, 1, 30.0, 30.0}, {128, 128, 32, 2, 21.0, 16.5}, {64, 64, 64, 3, 12.0, 7.6}},                         // float16
    {{}, {128, 256, 32, 1, 43.0, 43.0}, {128, 128, 32, 1, 27.0, 27.0}, {64, 64, 64, 2, 17.0, 9.5}},                         // float32
};
constexpr int NUM_CU = 256;
// Bytes of slots written and read a ns, rows a split sums at least, and at most (a split counts its rows in 32 bits).
constexpr double SLOT_RATE = 3200.0;
constexpr int64_t SPLIT_ROWS = 48, SPLIT_MOST = 1 << 30;

// The tile and the number of splits of the least estimated time: rounds of workgroups over the CUs, and the
// slots' way to memory and back. The estimate picks within 2% of the best of all on average over 41
// measured shapes; one rule of thumb (the largest tile, splits up to two workgroups a CU) was 35% off
// (2048 x 2048 x 2048 bfloat16: 52 us against 27 with middle tiles unsplit; 16384 x 512 x 512: 40 against 27 with small ones).
// The slots have one rate here, though their sum's loads come in whole rounds of its threads (17 slots cost what 128 do), so
// between 17 and 128 splits it can pick a slower plan: 20000 x 128 x 1000 float32 39 us with the middle tile's 32 splits, 36
// with the small one's 16.
static WeightPlan weight_plan(int planes, int64_t rows, int out, int cols)
{
    WeightPlan best{};
    double best_ns = 0.0;
    for (int t = planes == 1 ? 0 : 1; t < 4; ++t)
    {
        const TileCost& c = TILE_COST[planes - 1][t];
        // Tiles wider than an axis leave the branch-free loop.
        if (t < 3 && (out < c.side_n || cols < c.side_k)) continue;
        const int tiles_n = (out + c.side_n - 1) / c.side_n, tiles_k = (cols + c.side_k - 1) / c.side_k;
        const int64_t tiles = (int64_t)tiles_n * tiles_k;
        for (int64_t wanted = 1; wanted <= 1024; wanted = wanted < 4 ? wanted + 1 : wanted % 3 ? wanted / 2 * 3 : wanted / 3 * 4)
        {
            if (wanted > 1 && (rows / wanted < SPLIT_ROWS || tiles * wanted > 16 * NUM_CU)) break;
            int64_t per = ((rows + wanted - 1) / wanted + c.step - 1) / c.step * c.step;
            per = per < SPLIT_MOST ? per : SPLIT_MOST;
            const int64_t splits = (rows + per - 1) / per, groups = tiles * splits, round = (int64_t)NUM_CU * c.per_cu;
            auto round_ns = [&](int64_t n) {
                const double on_cu = (double)((n + NUM_CU - 1) / NUM_CU), each = c.shared * on_cu;
                return (double)per * (each > c.alone ? each : c.alone);
            };
            double ns = (double)(groups / round) * round_ns(round) + (groups % round ? round_ns(groups % round) : 0.0);
            if (splits > 1) ns += 2000.0 + (double)splits * out * cols * 8.0 / SLOT_RATE;
            if (best.splits && ns >= best_ns) continue;
            best_ns = ns;
            best = WeightPlan{t, tiles_n, tiles_k, (int)splits, per};
        }
    }
    return best;
}

template <typename T>
size_t grad_weight8_workspace(int64_t rows, int out, int cols)
{
    if (rows <= 0 || out <= 0 || cols <= 0) return 0;
    const WeightPlan p = weight_plan(planes_of<T>(), rows, out, cols);
    return p.splits > 1 ? align_up((size_t)p.splits * out * cols * sizeof(float)) : 0;
}

template <typename T, typename OT>
static hipError_t weight_launch(const WeightPlan& p, const T* gy, int64_t gys, const uint8_t* codes, const uint8_t* scales, OT* out, int64_t rows,
                                int out_rows, int cols, hipStream_t stream)
{
    const unsigned grid = (unsigned)((int64_t)p.tiles_n * p.tiles_k * p.splits);
    auto run = [&](auto tile, auto any) {
        using L = decltype(tile);
        grad_weight8_kernel<T, OT, L, decltype(any)::value>
            <<<grid, L::THREADS, 0, stream>>>(gy, gys, codes, scales, out, rows, p.split_rows, out_rows, cols, p.tiles_n, p.tiles_k);
        return hipGetLastError();
    };
    if (out_rows < UNIT || cols < UNIT) return run(SmallTile(), std::true_type());
    if constexpr (planes_of<T>() == 1)
        if (p.tile == 0) return run(WideTile(), std::false_type());
    if (p.tile == 1) return run(TallTile(), std::false_type());
    return p.tile == 2 ? run(MiddleTile(), std::false_type()) : run(SmallTile(), std::false_type());
}

template <typename T, typename OT>
hipError_t grad_weight8(const T* grad_y, int64_t gy_stride, const uint8_t* codes, const uint8_t* scales, OT* grad_weight, int64_t rows,
                        int out, int cols, void* workspace, hipStream_t stream)
{
    if (out <= 0 || cols <= 0) return hipSuccess;
    if (rows <= 0) return sum_slots_async<OT>(nullptr, 0, (int64_t)out * cols, grad_weight, stream);
    const WeightPlan p = weight_plan(planes_of<T>(), rows, out, cols);
    if ((int64_t)p.tiles_n * p.tiles_k * p.splits > 0x7fffffff) return hipErrorInvalidValue;
    if (p.splits == 1) return weight_launch<T, OT>(p, grad_y, gy_stride, codes, scales, grad_weight, rows, out, cols, stream);
    const hipError_t err = weight_launch<T, float>(p, grad_y, gy_stride, codes, scales, (float*)workspace, rows, out, cols, stream);
    if (err != hipSuccess) return err;
    return sum_slots_async<OT>((const float*)workspace, p.splits, (int64_t)out * cols, grad_weight, stream);
}

// Q threads a group of 4 columns, each summing every Q-th slot, 8 loads in flight without a branch between them: the
// last group is moved back to end with the columns and leaves those before its own to its neighbour. The threads'
// sums are added in thread order.
template <typename OT, int Q>
__global__ __launch_bounds__(BLOCK) void sum_slots_kernel(const float* __restrict__ part, int nslots, int64_t n, OT* __restrict__ out)
{
    constexpr int GROUPS = BLOCK / Q, COLS = GROUPS * 4, U = Q > 1 ? 8 : 2;
    __shared__ Acc sums[Q * COLS], four[Q / 4 * COLS + 1];
    const int g = threadIdx.x % GROUPS, q = threadIdx.x / GROUPS;
    const int64_t own = ((int64_t)blockIdx.x * GROUPS + g) * 4, j = own + 4 <= n ? own : n < 4 ? 0 : n - 4;
    Acc s[4] = {};
    for (int b = q; b < nslots; b += U * Q)
    {
        float v[U][4];
        if (n >= 4)
        {
#pragma unroll
            for (int u = 0; u < U; ++u) __builtin_memcpy(v[u], part + (int64_t)min(b + u * Q, nslots - 1) * n + j, sizeof(v[u]));
        }
        else
        {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[u][k] = part[(int64_t)min(b + u * Q, nslots - 1) * n + min(k, (int)n - 1)];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += b + u * Q < nslots ? (Acc)v[u][k] : Acc(0);
    }
    if constexpr (Q > 1)
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[q * COLS + g * 4 + k] = s[k];
        __syncthreads();
        const int tc = threadIdx.x % COLS, tq = threadIdx.x / COLS;
        four[tq * COLS + tc] = ((sums[4 * tq * COLS + tc] + sums[(4 * tq + 1) * COLS + tc]) + sums[(4 * tq + 2) * COLS + tc]) +
                               sums[(4 * tq + 3) * COLS + tc];
        __syncthreads();
        // A thread a column.
        const int64_t first = (int64_t)blockIdx.x * COLS + tc / 4 * 4, c = (first + 4 <= n ? first : n < 4 ? 0 : n - 4) + tc % 4;
        if (tq != 0 || c < first || c >= n) return;
        Acc t = Acc(0);
#pragma unroll
        for (int i = 0; i < Q / 4; ++i) t += four[i * COLS + tc];
        out[c] = (OT)t;
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (j + k >= own && j + k < n) out[j + k] = (OT)s[k];
}

template <typename OT>
hipError_t sum_slots_async(const float* part, int nslots, int64_t n, OT* out, hipStream_t stream)
{
    if (n <= 0) return hipSuccess;
    auto blocks = [&](int columns) { return (unsigned)((n + columns - 1) / columns); };
    if (nslots <= 16)
        sum_slots_kernel<OT, 1><<<blocks(4 * BLOCK), BLOCK, 0, stream>>>(part, nslots, n, out);
    else if (nslots <= 256)
        sum_slots_kernel<OT, 16><<<blocks(64), BLOCK, 0, stream>>>(part, nslots, n, out);
    else if (n <= 1024)
        sum_slots_kernel<OT, 256><<<blocks(4), BLOCK, 0, stream>>>(part, nslots, n, out);
    else
        sum_slots_kernel<OT, 64><<<blocks(16), BLOCK, 0, stream>>>(part, nslots, n, out);
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
