// Where the products of dense matrices (csrc/dense.h) read groups of 16 bytes through registers, by that file's own arithmetic on the host: no group of a step that is taken to be whole may
// pass the end of its matrix.  Compiled for the host alone.
#include <cstdio>
#include <cstdlib>

#include "dense.h"

using so_dense::Side;

static long checked = 0;

// The steps of a contraction as long as 32 bits count.
template <class S>
static void count(const char *what)
{
    for (uint64_t depth = (1ull << 32) - 2 * S::BK; depth < 1ull << 32; ++depth) {
        S side;
        side.own = 1;
        side.ld = (size_t)depth;
        side.depth = (uint32_t)depth;
        const uint64_t steps = (depth + S::BK - 1) / S::BK;
        if (side.steps() != steps || side.whole((uint32_t)steps - 1) != (depth % S::BK == 0)) {
            std::printf("%s: %u steps of a contraction of %llu\n", what, side.steps(), (unsigned long long)depth);
            std::exit(1);
        }
    }
}

// An operand of `own` entries of its own index and `depth` of the contraction, its rows `ld` apart.
template <class S, bool ACROSS>
static void check(uint32_t own, size_t ld, uint32_t depth, const char *what)
{
    S side;
    side.own = own;
    side.ld = ld;
    side.depth = depth;
    const uint32_t steps = side.steps();
    const size_t end = ACROSS ? (depth - 1) * ld + own : (own - 1) * ld + depth;
    for (uint32_t step = 0; step < steps; ++step) {
        if (!side.whole(step)) {
            if (step + 2 < steps) {
                std::printf("%s: step %u of %u is not whole: own %u, stride %zu, depth %u\n", what, step, steps, own, ld, depth);
                std::exit(1);
            }
            continue;
        }
        for (uint32_t q = 0; q < (uint32_t)(S::ROWS * S::PER); ++q) {
            ++checked;
            const size_t from = side.begin(step) + side.place(q);
            if (from + S::V > end) {
                std::printf("%s: step %u, group %u ends at %zu of %zu: own %u, stride %zu, depth %u\n", what, step, q, from + S::V, end, own, ld, depth);
                std::exit(1);
            }
        }
    }
}

template <class T, bool ACROSS, int LEN, int KB, int WAVES>
static void sweep(const char *what)
{
    typedef Side<T, ACROSS, LEN, KB, WAVES> S;
    const uint32_t step = S::BK;
    if (!ACROSS) count<S>(what);
    for (uint32_t own = 1; own <= (uint32_t)LEN + 9; own += own < 20 ? 1 : 7)
        for (uint32_t gap = 0; gap < 10; ++gap)
            for (uint32_t turns = 0; turns <= 2; ++turns)
                for (uint32_t rest = turns ? 0 : 1; rest < 12; ++rest) {
                    const uint32_t depth = turns * step + rest;
                    check<S, ACROSS>(own, (ACROSS ? own : depth) + gap, depth, what);
                }
}

template <class T>
static void sweeps(const char *type)
{
    std::printf("%s\n", type);
    // the tiles that are read through registers, and both sides of each
    sweep<T, true, 64, 256, 4>("X of 16 x 64");
    sweep<T, true, 64, 128, 4>("X of 32 x 64, 64 x 64");
    sweep<T, true, 128, 64, 4>("X of 128 x 128");
    sweep<T, false, 16, 256, 4>("A of 16 x 64");
    sweep<T, false, 32, 128, 4>("A of 32 x 64, half of 64 x 64");
    sweep<T, false, 64, 128, 4>("A of 64 x 64");
    sweep<T, false, 128, 64, 4>("A of 128 x 128");
}

int main()
{
    sweeps<float>("fp32");
    sweeps<_Float16>("fp16");
    sweeps<__bf16>("bf16");
    std::printf("%ld groups\n", checked);
    return checked ? 0 : 1;
}
