// The shapes that linear attention's passes take, on the host: reads lines of
//   type (0 float32, 1 float16, 2 bfloat16), packed (0 or 1), sequences, tokens, heads, dim, columns, passes of this shape together
// and writes for each: state rows, waves, whether the next chunk is loaded late, rows of a chunk, rows of a segment, whether sequences are split, the estimated cost.
#include <cstdio>

#include "../morphocore_amd/csrc/linear_attention.hpp"

template <typename T>
static void plan(const mca::Sequences& seq, int heads, const mca::Pass& p)
{
    (void)mca::by_walk<T>(seq, heads, p, [&](auto walk) {
        using L = decltype(walk);
        const mca::Plan plan = mca::plan_of<L>(seq, heads, p);
        printf("%d %d %d %d %lld %d %.17g\n", L::DK, L::W, (int)L::LATE, L::C, (long long)plan.segments.rows, (int)mca::joins(seq, plan.segments), plan.cost);
        return hipSuccess;
    });
}

int main()
{
    int type, packed, heads, dim, cols, together;
    long long count, tokens;
    while (scanf("%d %d %lld %lld %d %d %d %d", &type, &packed, &count, &tokens, &heads, &dim, &cols, &together) == 8)
    {
        const mca::Sequences seq = {packed ? (const void*)&type : nullptr, false, count, tokens};
        mca::Pass p = {};
        p.dim = dim, p.cols = cols, p.together = together;
        if (type == 0)
            plan<float>(seq, heads, p);
        else if (type == 1)
            plan<_Float16>(seq, heads, p);
        else
            plan<__bf16>(seq, heads, p);
    }
}
