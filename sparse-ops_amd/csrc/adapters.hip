// Low-rank adapters of many requests: Y = base + scale_a B_a (A_a X), the adapter a of every column its own.
//
// Two launches.  Both take the columns 64 at a time and go over the adapters that occur among them, one after the other, or, where there are few such tiles, side by side: one tile of columns is multiplied as a
// whole with an adapter, and of the result those columns are kept that have it.  So the columns of a prompt, which share one, are read once, and of a batch of single tokens every adapter is.
#include "dense.h"

namespace {

using so_dense::f32x4;
using so_dense::Operand;
using so_dense::u32x4;

constexpr uint32_t kThreads = 256, kMostRank = 256, kCols = 64, kPad = 16, kFewColumns = 256, kResultPitch = kCols + 4;

// The adapters that occur in the 64 columns of a tile, by their first column.  Each of the four waves finds the columns of 16 of the 64 columns' adapters, and they meet in LDS, `masks` [64].
struct Which {
    uint32_t mine;                      // of `lane`'s column: its adapter
    uint64_t same;                      // and the columns that have the same one
    uint64_t having, none, firsts;      // columns with an adapter; columns that exist and have none; the first column of every adapter
    // The 64 columns from j0 on, of which those from `own` on count.
    __device__ __forceinline__ Which(const int32_t *which, uint64_t j0, uint64_t own, uint32_t C, uint32_t count, uint64_t *masks)
    {
        const uint32_t lane = threadIdx.x % 64u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
        const uint64_t c = j0 + lane;
        const bool counts = c >= own && c < C;
        mine = counts ? (uint32_t)which[c] : 0xffffffffu;
        const bool has = mine < count;                                   // a negative number is beyond all others
        having = __ballot(has);
        none = __ballot(counts && !has);
        uint64_t found = 0;
#pragma unroll 4                                                          // code that runs once is paid for by its length
        for (uint32_t i = 0; i < 16u; ++i) {
            const uint64_t columns = __ballot(mine == (uint32_t)__builtin_amdgcn_readlane((int)mine, (int)(wave * 16u + i)));
            found = lane == i ? columns : found;
        }
        if (lane < 16u) masks[wave * 16u + lane] = found;
        __syncthreads();
        same = masks[lane];
        firsts = __ballot(has && (same & ((1ull << lane) - 1ull)) == 0);
    }
    __device__ __forceinline__ uint32_t adapters() const { return (uint32_t)__builtin_popcountll(firsts); }
    // Whether lane's column is the first of an adapter, and the number of that.
    __device__ __forceinline__ bool begins() const { return firsts >> threadIdx.x % 64u & 1u; }
    __device__ __forceinline__ uint32_t number() const { return (uint32_t)__builtin_popcountll(firsts & ((1ull << threadIdx.x % 64u) - 1ull)); }
    // Adapter number i and its columns; no columns: there is none.
    struct Turn { uint32_t adapter; uint64_t columns; };
    __device__ __forceinline__ Turn turn(uint32_t i) const
    {
        const uint64_t it = __ballot(begins() && number() == i);
        if (!it) return {0, 0};
        const int at = __builtin_ctzll(it);
        return {(uint32_t)__builtin_amdgcn_readlane((int)mine, at),
                (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(same >> 32), at) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)same, at)};
    }
};

// How a call is cut: tiles of 64 columns, adapters of a tile side by side, parts of the features; the rows of Y that a workgroup takes.
struct Cut {
    uint32_t tiles, turns, parts, depth, rows, row_groups, padded;
    bool few;                // columns
    uint32_t strip;          // tiles of an XCD, 0: as they come
    uint32_t blocks(uint32_t each) const { return (strip ? 8u * strip : tiles) * each; }
};

// Which tile of columns a workgroup takes, and which of the tile's workgroups it is.  Workgroups go round-robin to the 8 XCDs; in strips neighbouring tiles are on the same one.
struct Spot {
    uint32_t tile, other;
    __device__ __forceinline__ Spot(const Cut &c)
    {
        const uint32_t in = c.strip ? blockIdx.x / 8u : blockIdx.x, w = c.strip ? c.strip : c.tiles;
        other = in / w;
        tile = in % w + (c.strip ? blockIdx.x % 8u * c.strip : 0u);
    }
};

template <class T> struct Call {
    const T *A, *B, *X, *base;
    T *Y;
    const float *scale;
    const int32_t *which;
    float *low;              // [parts][C][padded]: A x, an adapter's entries beyond its rank zeros
    size_t ldx, ldb, ldy;
    uint32_t m, n, C, count, rank;
    Cut cut;
};

// The launch's arguments lie in three lines of memory, and the first use of each waits for it: all at once, ahead of everything else.
template <class T>
__device__ __forceinline__ void fetch_arguments(const Call<T> &f)
{
    asm volatile("" : : "s"(f.A), "s"(f.scale), "s"(f.ldx), "s"(f.m), "s"(f.cut.rows));
}

// A x of one part of the features for the columns of the adapters in turn.  Bound by memory for many columns: 4096 features of 8192 bf16, 67 MB, rank 16, 19.3 us or 3.5 TB/s (15.8 where no tile has two adapters, and is
// read twice); by latency for few: 48 columns with 48 adapters fp16 5 us.
template <class T, class TILE, bool DIRECT>
__global__ __launch_bounds__(kThreads)
void adapters_in_kernel(Call<T> f)
{
    extern __shared__ char stage[];
    fetch_arguments(f);
    const Spot spot(f.cut);
    if (spot.tile >= f.cut.tiles) return;
    const uint32_t part = spot.other % f.cut.parts;
    const uint64_t j0 = (uint64_t)spot.tile * kCols;
    const size_t k0 = (size_t)part * f.cut.depth;
    const uint32_t depth = (uint32_t)min((size_t)f.cut.depth, f.n - k0), lane = threadIdx.x % 64u;
    const Which which(f.which, j0, j0, f.C, f.count, reinterpret_cast<uint64_t *>(stage));      // the ring comes later
    // a tile's second adapters first: few tiles have one, and they are not to begin when all others end
    for (uint32_t i = f.cut.turns - 1u - spot.other / f.cut.parts; i < which.adapters(); i += f.cut.turns) {
        const Which::Turn at = which.turn(i);
        for (uint32_t r0 = 0; r0 < f.rank; r0 += TILE::ROWS) {
            so_dense::Loop<T, TILE, false, true, false> loop;
            loop.template add<DIRECT>(stage, {{f.A + (size_t)at.adapter * f.rank * f.n + k0, f.n, f.rank, depth}}, r0, {f.X + k0 * f.ldx, f.ldx, f.C, depth}, j0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t col = threadIdx.x / 64u * 16u + 4u * (lane / 16u) + e;
                if (!(at.columns >> col & 1u)) continue;
                float *to = f.low + ((size_t)part * f.C + j0 + col) * f.cut.padded + r0 + lane % 16u;
#pragma unroll
                for (int i = 0; i < TILE::RT; ++i)
                    if (r0 + i * 16 < f.cut.padded) to[i * 16] = r0 + i * 16 + lane % 16u < f.rank ? loop.acc[i][0][e] : 0.0f;
            }
        }
    }
}

// What the kernels that make Y share.  The products' operand of a tile's 64 columns, every column's from its own adapter, lies in LDS; a wave multiplies 16 rows of an adapter's B with it and keeps the results of the
// columns that have that adapter.  Columns are dealt to the instructions so that a lane's results are 16 bytes of a row: in 16 bits column 8 g + 4 k + e of 32 is that of instruction k of two, lanes 16 g ..,
// result e.
template <class T>
struct Tile64 {
    static constexpr int V = so_elements<T>::V, RUNS = 16 / V;           // groups of 16 bytes that a lane has of a row
    static constexpr bool HALF = sizeof(T) == 2, SHIFTED = std::is_same<T, _Float16>::value;
    static constexpr bool THIRD = std::is_same<T, __bf16>::value;         // bf16 holds an fp32 sum in three numbers
    typedef typename so_elements<T>::plain group;
    typedef typename so_elements<T>::vec group_anywhere;
    // LDS: the operand [4][runs of 16][64 lanes], its third numbers [4][pairs of runs][64 lanes], what a column's results are multiplied with, the adapters and their columns
    static __host__ __device__ uint32_t operand_bytes(uint32_t runs) { return 4u * (runs + (THIRD ? (runs + 1u) / 2u : 0u)) * 1024u; }
    static __host__ __device__ uint32_t lds(uint32_t runs) { return operand_bytes(runs) + kCols * 4u + kCols * 12u; }

    const Call<T> &f;
    uint32_t runs, pairs, count;                                         // runs of 16 entries of rank, pairs of them; adapters
    u32x4 *operand, *third;
    float *factor;
    uint64_t *columns;
    uint32_t *adapter;
    uint64_t having, none;
    float scale;
    uint32_t held_adapter;
    uint64_t held_columns;
    __device__ __forceinline__ Tile64(const Call<T> &f_, char *lds) : f(f_)
    {
        runs = f.cut.padded / 16u;
        pairs = (runs + 1u) / 2u;
        operand = reinterpret_cast<u32x4 *>(lds);
        third = operand + 4u * runs * 64u;
        factor = reinterpret_cast<float *>(lds + operand_bytes(runs));
        columns = reinterpret_cast<uint64_t *>(factor + kCols);
        adapter = reinterpret_cast<uint32_t *>(columns + kCols);
    }
    // The adapters of the tile, and the scale of the column that this lane makes the operand of.  With barriers.
    __device__ __forceinline__ void list(uint64_t j0, uint64_t own)
    {
        const Which which(f.which, j0, own, f.C, f.count, columns);
        having = which.having;
        none = which.none;
        count = which.adapters();
        const uint32_t col = column(threadIdx.x / 64u, threadIdx.x % 16u), mine = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(col * 4u), (int)which.mine);
        scale = f.scale && having >> col & 1u ? f.scale[mine] : 1.0f;
        __syncthreads();                                                 // the masks are read
        if (threadIdx.x < 64u && which.begins()) {
            adapter[which.number()] = which.mine;
            columns[which.number()] = which.same;
        }
        __syncthreads();
        // lane i holds number i's: read from there they cost a few clocks, from LDS 130 each
        const uint32_t i = min(threadIdx.x % 64u, max(count, 1u) - 1u);
        held_adapter = adapter[i];
        held_columns = columns[i];
    }
    __device__ __forceinline__ uint32_t adapter_of(uint32_t i) const { return (uint32_t)__builtin_amdgcn_readlane((int)held_adapter, (int)i); }
    __device__ __forceinline__ uint64_t columns_of(uint32_t i) const
    {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(held_columns >> 32), (int)i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)held_columns, (int)i);
    }
    // The column of the tile that operand lane l of instruction k has, and the first of run p's
    static __device__ __forceinline__ uint32_t column(uint32_t k, uint32_t l) { return HALF ? k / 2u * 32u + l / 4u * 8u + k % 2u * 4u + l % 4u : k * 16u + l; }
    static __device__ __forceinline__ uint32_t first(int p, uint32_t g) { return HALF ? p * 32u + g * 8u : p * 16u + g * 4u; }
    // Which of instruction and result is column first(p, g) + e
    static __device__ __forceinline__ constexpr int instruction(int p, int e) { return HALF ? 2 * p + e / 4 : p; }

    // A x of the columns from j0 on as operand, wave k that of instruction k: entries of rank of a run of 16, of N parts at a time (behind the last one zeros).  The first ones can be asked for ahead of all else: a
    // column without an adapter has a place there too.
    template <int N> struct Sums { f32x4 s[N][V / 4]; };
    template <int N>
    __device__ __forceinline__ void ask(uint64_t j0, uint32_t run, uint32_t part, Sums<N> &a) const
    {
        const uint32_t lane = threadIdx.x % 64u, col = column(threadIdx.x / 64u, lane % 16u), g = lane / 16u;
        const float *from = f.low + min(j0 + col, (uint64_t)f.C - 1u) * f.cut.padded + (HALF ? g % 2u * 8u : g * 4u) + run * 16u;
        const size_t step = (size_t)f.C * f.cut.padded;
#pragma unroll
        for (uint32_t i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < V / 4; ++e) a.s[i][e] = part + i < f.cut.parts ? *reinterpret_cast<const f32x4 *>(from + (part + i) * step + e * 4) : f32x4{};
    }
    template <int HOLD, int N>
    __device__ __forceinline__ void gather(uint64_t j0, const Sums<N> &first) const
    {
        const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u, l = lane % 16u, g = lane / 16u, col = column(wave, l);
        const bool mine = having >> col & 1u;
        const auto low = [&](uint32_t run, float (&v)[V]) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = 0.0f;
            for (uint32_t p = 0; p < f.cut.parts; p += N) {
                Sums<N> a = first;
                if (run || p) ask(j0, run, p, a);
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] += a.s[i][e / 4][e % 4];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = mine ? v[e] : 0.0f;
        };
        // What entries are multiplied with on their way in, and results on theirs out: the adapter's scale; in fp16 a power of two that brings a column's largest finite entry to 2^14 .. 2^15, and the rest
        // behind the product.
        float in = scale, out = 1.0f;
        const auto choose = [&](float largest) {
            const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(largest), __float_as_uint(largest), false, false);
            const uint32_t top = max(h[0], h[1]) >> 23;                  // the largest's exponent, biased
            const int up = min(max(141 - (int)top, -100), 100);
            in = __uint_as_float((uint32_t)(127 + up) << 23);
            out = scale * __uint_as_float((uint32_t)(127 - up) << 23);
        };
        const auto put = [&](uint32_t run, const float (&v)[V]) {
            u32x4 &to = operand[(wave * runs + run) * 64u + lane];
            if constexpr (HALF) {
                // 16 entries as 32: lanes 0 .. 31 have them rounded to T, the others what that leaves, so that the product, with B's entries twice, has fp16's 22 bits and a
                // sign, half a step of fp32.  What bf16's 16 leave goes into an instruction of its own, of two runs, the second one's in lanes 32 .. 63: without it results that cancel lost bits.
                // It costs both launches of 4096 x 4096 x 8192, rank 16, 3 us of 53, rank 64 none of 100, rank 256, whose operand then leaves room for one workgroup a compute unit, 80 of 253; 48 requests none.
                group q, rest;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float w = v[e] * in;
                    const T high = (T)w;
                    const float left = __builtin_isinf((float)high) ? 0.0f : w - (float)high;
                    const T next = (T)left;
                    q[e] = g < 2u ? high : next;
                    rest[e] = (T)(left - (float)next);
                }
                to = __builtin_bit_cast(u32x4, q);
                if constexpr (THIRD) {
                    const bool mine_too = run % 2u == g / 2u;
                    if (mine_too || (run % 2u == 0 && run + 1u == runs)) third[(wave * pairs + run / 2u) * 64u + lane] = mine_too ? __builtin_bit_cast(u32x4, rest) : u32x4{};
                }
            } else {
                to = __builtin_bit_cast(u32x4, f32x4{v[0] * in, v[1] * in, v[2] * in, v[3] * in});
            }
        };
        if constexpr (SHIFTED) {
            // the first HOLD runs stay in registers between the two passes
            float held[HOLD][V], v[V], largest = 0.0f;
            const auto see = [&](float entry) { largest = fmaxf(largest, fabsf(entry) < INFINITY ? fabsf(entry) : 0.0f); };
#pragma unroll
            for (uint32_t run = 0; run < HOLD; ++run)
                if (run < runs) {
                    low(run, held[run]);
#pragma unroll
                    for (int e = 0; e < V; ++e) see(held[run][e]);
                }
            for (uint32_t run = HOLD; run < runs; ++run) {
                low(run, v);
#pragma unroll
                for (int e = 0; e < V; ++e) see(v[e]);
            }
            choose(largest);
            if (g == 0) factor[col] = out;
#pragma unroll
            for (uint32_t run = 0; run < HOLD; ++run)
                if (run < runs) put(run, held[run]);
            for (uint32_t run = HOLD; run < runs; ++run) {
                low(run, v);
                put(run, v);
            }
        } else {
            float v[V];
            for (uint32_t run = 0; run < runs; ++run) {
                low(run, v);
                put(run, v);
            }
        }
    }
    // A run of 16 entries of rank of a row of adapter a's B, asked for without a branch, and made what it is once it has come.  EVEN: the rank is a multiple of a group, so that groups are whole.  Else they reach into
    // the next row, and groups that would reach beyond the end of all are those that end there, to be moved down; what lies beyond the rank is cleared.
    template <bool EVEN> struct Run {
        u32x4 w;
        uint32_t down;                                                   // halves of words (not EVEN)
    };
    __device__ __forceinline__ uint32_t rank_of(uint32_t run) const { return run * 16u + (HALF ? threadIdx.x % 32u / 16u * 8u : threadIdx.x % 64u / 16u * 4u); }      // this lane's first
    template <bool EVEN>
    __device__ __forceinline__ Run<EVEN> load_b(uint32_t a, uint64_t row, uint32_t run) const
    {
        const size_t from = ((size_t)a * f.m + row) * f.rank;
        const uint32_t r = rank_of(run);
        Run<EVEN> b;
        b.down = 0;
        if constexpr (EVEN) {
            b.w = __builtin_bit_cast(u32x4, *reinterpret_cast<const group_anywhere *>(f.B + from + min(r, f.rank - V)));
        } else {
            const size_t want = from + (r < f.rank ? r : 0u), end = (size_t)f.count * f.m * f.rank, have = min(want, end - min(end, (size_t)V));
            b.w = __builtin_bit_cast(u32x4, *reinterpret_cast<const group_anywhere *>(f.B + have));
            b.down = (uint32_t)(want - have) * (HALF ? 1u : 2u);
        }
        return b;
    }
    template <bool EVEN>
    __device__ __forceinline__ u32x4 settle(const Run<EVEN> &b, uint32_t run) const
    {
        const uint32_t r = rank_of(run);
        u32x4 w = b.w;
        if constexpr (EVEN) return r < f.rank ? w : u32x4{};
        if (b.down & 4u) w = u32x4{w[2], w[3], 0, 0};
        if (b.down & 2u) w = u32x4{w[1], w[2], w[3], 0};
        if constexpr (HALF)
            if (b.down & 1u) w = u32x4{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16};
        const uint32_t left = r < f.rank ? f.rank - r : 0u;
        constexpr uint32_t E = HALF ? 2 : 1;                             // entries of a word
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) w[i] = left >= (i + 1u) * E ? w[i] : left > i * E ? w[i] & 0xffffu : 0u;
        return w;
    }
    __device__ __forceinline__ float add(float product, uint32_t col, float to) const { return SHIFTED ? fmaf(product, factor[col], to) : product + to; }
    // The operand of a single run can stay in registers.
    struct Kept { u32x4 first[4], third[THIRD ? 4 : 1]; };
    __device__ __forceinline__ void take(Kept &t) const
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            t.first[k] = operand[k * runs * 64u + threadIdx.x % 64u];
            if constexpr (THIRD) t.third[k] = third[k * pairs * 64u + threadIdx.x % 64u];
        }
    }
    // acc += runs from `run` on, an even number if there are several, of 16 rows of B
    template <int RC, bool EVEN>
    __device__ __forceinline__ void multiply(const Run<EVEN> (&b)[RC], uint32_t run, const Kept &t, f32x4 (&acc)[4]) const
    {
        u32x4 before = {};
#pragma unroll
        for (int c = 0; c < RC; ++c)
            if (RC == 1 || run + c < runs) {
                const u32x4 w = settle(b[c], run + c);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = so_dense::multiply<T>(w, RC == 1 ? t.first[k] : operand[(k * runs + run + c) * 64u + threadIdx.x % 64u], acc[k]);
                if constexpr (THIRD) {
                    // a pair's second run's entries of B for lanes 32 .. 63; where there is none they meet zeros
                    const bool last = RC == 1 || run + c + 1u == runs;
                    if (c % 2 || last) {
                        u32x4 both = w;
                        if (c % 2 && threadIdx.x % 64u < 32u) both = before;
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[k] = so_dense::multiply<T>(both, RC == 1 ? t.third[k] : third[(k * pairs + (run + c) / 2u) * 64u + threadIdx.x % 64u], acc[k]);
                    }
                    before = w;
                }
            }
    }
};

// Y of many columns.  A workgroup takes 64 of them and a run of rows, a wave 16 rows at a time, one adapter after the other (few tiles have two); the next products' entries of B and the next 16 rows' base are on their
// way while these are worked on.  Bound by memory: 4096 x 8192 bf16 with a base, 134 MB, 34.6 us or 3.9 TB/s.  Registers for as many waves as come without spilling.
template <class T, int RC, bool BASE, bool EVEN>
__global__ __launch_bounds__(kThreads, (std::is_same<T, __bf16>::value && RC <= 2 ? 4 : RC <= 2 ? 3 : 2))
void adapters_out_kernel(Call<T> f)
{
    typedef Tile64<T> Shared;
    constexpr int V = Shared::V, RUNS = Shared::RUNS;
    constexpr bool HALF = Shared::HALF;
    typedef typename Shared::group group;
    typedef typename Shared::group_anywhere group_anywhere;
    extern __shared__ char lds[];
    fetch_arguments(f);
    const Spot spot(f.cut);
    if (spot.tile >= f.cut.tiles) return;
    const uint32_t tile = spot.tile, part = spot.other, lane = threadIdx.x % 64u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), l = lane % 16u, g = lane / 16u;
    // The last tile's columns end at C.  Those that the tile before it has too are written by both, the same bits, or, in place, where that would add twice, by that one alone.
    const uint64_t j0 = min((uint64_t)tile * kCols, (uint64_t)f.C - kCols), row_begin = (uint64_t)part * f.cut.rows, row_end = min(row_begin + f.cut.rows, (uint64_t)f.m);
    Shared at(f, lds);
    typename Shared::template Sums<4> sums;
    at.ask(j0, 0, 0, sums);
    at.list(j0, f.base == f.Y ? (uint64_t)tile * kCols : j0);
    at.template gather<RC>(j0, sums);
    __syncthreads();
    typename Shared::Kept whole;
    if constexpr (RC == 1) at.take(whole);
    const uint32_t blocks = (at.runs + RC - 1u) / RC;
    typedef typename Shared::template Run<EVEN> Run;
    const auto load_b = [&](uint32_t a, uint64_t row, uint32_t block, Run (&b)[RC]) {
#pragma unroll
        for (int c = 0; c < RC; ++c) b[c] = at.template load_b<EVEN>(a, min(row, row_end - 1u), block * RC + c);
    };
    const auto load_base = [&](uint64_t row, group (&r)[RUNS]) {
        if constexpr (BASE)
#pragma unroll
            for (int p = 0; p < RUNS; ++p) r[p] = *reinterpret_cast<const group_anywhere *>(f.base + min(row, row_end - 1u) * f.ldb + j0 + Shared::first(p, g));
    };
    const uint64_t counts = at.having | at.none;
    group r[RUNS], next[RUNS];
    Run b[RC], next_b[RC];
    uint64_t row = row_begin + wave * 16u + l;
    load_base(row, r);
    if (at.count) load_b(at.adapter_of(0), row, 0, b);
    for (uint64_t from = row_begin + wave * 16u; from < row_end; from += 64u, row += 64u) {
        load_base(row + 64u, next);
        float v[RUNS][V];
#pragma unroll
        for (int p = 0; p < RUNS; ++p)
#pragma unroll
            for (int e = 0; e < V; ++e) v[p][e] = BASE ? (float)r[p][e] : 0.0f;
        for (uint32_t i = 0; i < at.count; ++i) {
            f32x4 acc[4] = {};
            for (uint32_t block = 0; block < (RC == 4 ? blocks : 1u); ++block) {
                const bool end = RC < 4 || block + 1u == blocks, more = i + 1u < at.count;      // then the next adapter's first, or the first one's of the next 16 rows
                load_b(at.adapter_of(end ? (more ? i + 1u : 0u) : i), end && !more ? row + 64u : row, end ? 0u : block + 1u, next_b);
                at.template multiply<RC, EVEN>(b, block * RC, whole, acc);
#pragma unroll
                for (int c = 0; c < RC; ++c) b[c] = next_b[c];
            }
            const uint64_t has = at.columns_of(i);
#pragma unroll
            for (int p = 0; p < RUNS; ++p)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const uint32_t col = Shared::first(p, g) + e;
                    const float sum = at.add(acc[Shared::instruction(p, e)][e % 4], col, v[p][e]);
                    v[p][e] = has >> col & 1u ? sum : v[p][e];
                }
        }
        if (row < row_end)
#pragma unroll
            for (int p = 0; p < RUNS; ++p) {
                T *to = f.Y + row * f.ldy + j0 + Shared::first(p, g);
                if (counts == ~0ull) so_group_store(to, V, v[p]);
                else
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (counts >> (Shared::first(p, g) + e) & 1u) to[e] = (T)v[p][e];
            }
#pragma unroll
        for (int p = 0; p < RUNS; ++p) r[p] = next[p];
    }
}

// Y of few columns, each perhaps with an adapter of its own.  A workgroup takes 16 rows at a time; the adapters are dealt to its waves, DEEP of a wave on their way at a time; results meet in LDS, and Y is written in
// groups.  Bound by latency, a chain of loads, and by the length of its code: eleven adapters of a wave at once, in 34 KB of code, were no faster than three.  4096 x 48, 48 adapters, rank 16 fp16: 8.3 us.
template <class T, int RC, bool EVEN>
__global__ __launch_bounds__(kThreads)
void adapters_out_few_kernel(Call<T> f)
{
    typedef Tile64<T> Shared;
    constexpr int V = Shared::V;
    constexpr bool HALF = Shared::HALF;
    constexpr uint32_t PITCH = kResultPitch, GROUPS = 16u * kCols / V, DEEP = RC == 4 ? 2 : 3;
    extern __shared__ char lds[];
    fetch_arguments(f);
    float *results = reinterpret_cast<float *>(lds + Shared::lds(f.cut.padded / 16u));
    const uint32_t tile = blockIdx.x % f.cut.tiles, part = blockIdx.x / f.cut.tiles, lane = threadIdx.x % 64u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), l = lane % 16u, g = lane / 16u;
    const uint64_t j0 = (uint64_t)tile * kCols, row_begin = (uint64_t)part * f.cut.rows, row_end = min(row_begin + f.cut.rows, (uint64_t)f.m);
    Shared at(f, lds);
    typename Shared::template Sums<8> sums;
    at.ask(j0, 0, 0, sums);
    const uint32_t blocks = (at.runs + RC - 1u) / RC, out_row = threadIdx.x / (kCols / V), out_col = threadIdx.x % (kCols / V) * V;
    const auto left_of = [&](uint64_t from) { return threadIdx.x < GROUPS && from + out_row < row_end && j0 + out_col < f.C ? (uint32_t)min((uint64_t)V, f.C - j0 - out_col) : 0u; };
    at.list(j0, j0);
    typedef typename Shared::template Run<EVEN> Run;
    Run b[DEEP][RC];
    const auto load_b = [&](uint32_t i, uint64_t row, uint32_t block, Run (&to)[RC]) {
        // behind the last one that one again: without a branch, so that it is known how many are on their way
#pragma unroll
        for (int c = 0; c < RC; ++c) to[c] = at.template load_b<EVEN>(at.adapter_of(min(i, at.count - 1u)), min(row, row_end - 1u), block * RC + c);
    };
    const auto load_first = [&](uint64_t row) {
#pragma unroll
        for (uint32_t i = 0; i < DEEP; ++i)
            load_b(wave + i * 4u, row, 0, b[i]);
    };
    if (at.count) load_first(row_begin + l);
    at.template gather<RC>(j0, sums);
    __syncthreads();
    typename Shared::Kept whole;
    if constexpr (RC == 1) at.take(whole);
    for (uint64_t from = row_begin; from < row_end; from += 16u) {
        const uint64_t row = from + l;
        const uint32_t left = left_of(from);
        typename Shared::group base = {};
        if (left && f.base) base = so_group_load(f.base + (from + out_row) * f.ldb + j0 + out_col, left);
        f32x4 mine[4] = {};                                              // results of the columns of this wave's adapters, and which they are
        uint64_t columns = 0;
        const auto multiply = [&](uint32_t i, Run (&own)[RC]) {
            f32x4 acc[4] = {};
            at.template multiply<RC, EVEN>(own, 0, whole, acc);
            if constexpr (RC == 4)
                for (uint32_t block = 1; block < blocks; ++block) {
                    load_b(i, row, block, own);
                    at.template multiply<RC, EVEN>(own, block * RC, whole, acc);
                }
            load_b(i + DEEP * 4u, row, 0, own);
            const uint64_t has = at.columns_of(i);
            columns |= has;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t bits = (uint32_t)(has >> (HALF ? k / 2 * 32u + g * 8u + k % 2 * 4u : k * 16u + g * 4u));
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[k][e] = bits >> e & 1u ? acc[k][e] : mine[k][e];
            }
        };
        for (uint32_t i = wave; i < at.count; i += DEEP * 4u)
#pragma unroll
            for (uint32_t d = 0; d < DEEP; ++d)
                if (i + d * 4u < at.count) multiply(i + d * 4u, b[d]);
        if (at.count && from + 16u < row_end) load_first(row + 16u);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t c0 = HALF ? k / 2 * 32u + g * 8u + k % 2 * 4u : k * 16u + g * 4u;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (columns >> (c0 + e) & 1u) results[l * PITCH + c0 + e] = mine[k][e];
        }
        __syncthreads();
        if (left) {
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] = (float)base[e];                                   // zero without a base
                if (at.having >> (out_col + e) & 1u) v[e] = at.add(results[out_row * PITCH + out_col + e], out_col + e, v[e]);
            }
            so_group_store(f.Y + (from + out_row) * f.ldy + j0 + out_col, left, v);
        }
        __syncthreads();
    }
}

Cut cut_of(const so_ctx *ctx, int type, uint32_t m, uint32_t n, uint32_t C, uint32_t count, uint32_t rank)
{
    const uint32_t step = (rank <= 16 ? 256u : 128u) / (uint32_t)so_type_bytes(type);      // of the first launch
    const uint64_t cus = (uint64_t)ctx->compute_units;
    Cut c = {};
    c.tiles = so_ceil_div(C, kCols);
    // a tile may have as many adapters as columns, and a workgroup without one ends at once; where a request ends and the next begins a tile has two
    c.turns = (uint32_t)std::min<uint64_t>(std::min({C, kCols, std::max(count, 1u)}), std::max<uint64_t>(2, cus / 2 / c.tiles));
    c.padded = so_ceil_div(rank, kPad) * kPad;
    // Parts of the features: of a rank beyond 16 the second launch takes 8 at a time of every 16 entries, one wait each (16 columns of 4096 x 4096, rank 64 fp16: 8 parts 21.3 us, 16 26.4; one column, rank 16 fp16: 12.2 and
    // 12.0).
    const uint64_t most = std::max<uint64_t>(1, so_ceil_div(n, 2 * step)), want = std::max<uint64_t>(1, 2 * cus / ((uint64_t)c.tiles * c.turns));
    c.parts = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(most, std::max<uint64_t>(want, c.tiles < cus ? 4 : 1)), rank <= 16 ? 16 : 8);
    c.depth = so_ceil_div(so_ceil_div(n, c.parts), step) * step;
    c.parts = so_ceil_div(n, c.depth);
    // With few columns the second launch deals adapters to waves, 16 rows at a time, else rows (us of the second launch, 4096 rows, rank 16 fp16, by rows / by adapters, of 1, 8 and 64 requests: 128 columns 5.3 / 6.6,
    // 6.7 / 6.8, 19 / 11.5; 256 columns 5.8 / 10.5, 6.2 / 10.8, 13 / 14; 512 columns of one 6.5 / 16).  Which requests there are is known on the device alone, so that the rule goes by the columns: below 256 it
    // spares many requests 8 us at the price of 1 to 4 of few, from 256 on rows are faster for any.  Of rows a workgroup takes as many as leave four workgroups a compute unit, two of a larger rank, whose operand takes
    // longer to gather.
    c.few = C < kFewColumns;
    const uint64_t rows = (uint64_t)m * c.tiles / ((c.few ? 8 : rank <= 16 ? 4 : 2) * cus);
    c.rows = c.few ? 16u * (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(rows / 16, 16)) : 64u * (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(rows / 64, 8));
    c.row_groups = so_ceil_div(m, c.rows);
    return c;
}

// Of the workspace: A x, and behind it a group of B's where that has no more.
size_t low_floats(const Cut &c, uint32_t C) { return (size_t)c.parts * C * c.padded; }
size_t bytes_of(const Cut &c, uint32_t C) { return low_floats(c, C) * sizeof(float) + 16; }

// All of B, less than a group of 16 bytes, as one.
template <class T>
__global__ void adapters_small_kernel(const T *B, uint32_t entries, T *to)
{
    if (threadIdx.x < so_elements<T>::V) to[threadIdx.x] = threadIdx.x < entries ? B[threadIdx.x] : (T)0.0f;
}

so_status workspace(so_ctx *ctx, const char *who, size_t bytes)
{
    SO_REQUIRE(!ctx->capturing || (ctx->mm_part && ctx->mm_part->bytes >= bytes),
               "%s: the context's workspace must grow, which cannot be done while a graph is being recorded (call so_adapters_reserve, or launch this shape once, before recording)", who);
    return so_matmul_workspace(ctx, bytes, 4);
}

template <class T, class TILE>
so_status launch_in(so_ctx *ctx, const Call<T> &f, bool direct)
{
    const auto kernel = direct ? adapters_in_kernel<T, TILE, true> : adapters_in_kernel<T, TILE, false>;
    SO_HIP(so_allow_big_lds(ctx, (const void *)kernel));
    kernel<<<f.cut.blocks(f.cut.parts * f.cut.turns), kThreads, TILE::lds, ctx->stream>>>(f);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

template <class T>
so_status run(so_ctx *ctx, Call<T> f)
{
    // Of many tiles each XCD gets a strip where rows do not all begin at a line of memory of 128 bytes: tiles side by side share their last lines.  4096 x 4096, rank 16
    // bf16, 5003 columns: 52.6 us, as they come 58.6; 8192 in rows of 8200: 48.6 and 52.9.
    const uint64_t bits = (uintptr_t)f.X | (uintptr_t)f.base | (uintptr_t)f.Y | (f.ldx | f.ldb | f.ldy) * sizeof(T);
    f.cut.strip = bits % 128 && f.cut.tiles >= 64 ? so_ceil_div(f.cut.tiles, 8) : 0;      // fewer would not go to the XCDs evenly
    const uint64_t most = (uint64_t)f.cut.tiles + 7, in = most * f.cut.parts * f.cut.turns, out = most * f.cut.row_groups;
    SO_REQUIRE(so_grid_fits(std::max(in, out), kThreads), "so_adapters: %u x %u is too large for one launch", f.m, f.C);
    if (const uint64_t entries = (uint64_t)f.m * f.rank * f.count; entries > 0 && (uint64_t)f.m * f.rank < 8 && entries < (uint64_t)so_elements<T>::V) {
        T *to = (T *)(f.low + low_floats(f.cut, f.C));
        adapters_small_kernel<T><<<1, 64, 0, ctx->stream>>>(f.B, (uint32_t)entries, to);
        f.B = to;
    }
    if (f.count) {
        const Operand<T> a = {f.A, f.n, f.rank, f.n}, x = {f.X, f.ldx, f.C, f.n};
        const bool direct = a.direct() && x.direct();
        so_status s;
        if (f.rank <= 16) s = launch_in<T, so_dense::Tile<1, 1, 1, 4, 256, 3>>(ctx, f, direct);
        else if (f.rank <= 32) s = launch_in<T, so_dense::Tile<2, 1, 1, 4, 128, 4>>(ctx, f, direct);
        else s = launch_in<T, so_dense::Tile<4, 1, 1, 4, 128, 4>>(ctx, f, direct);
        if (s != SO_OK) return s;
    }
    const uint32_t bytes = Tile64<T>::lds(f.cut.padded / 16) + (f.cut.few ? 16u * kResultPitch * 4u : 0u);
    const auto launch = [&](auto kernel) {
        const hipError_t e = bytes > 40 * 1024 ? so_allow_big_lds(ctx, (const void *)kernel) : hipSuccess;
        if (e == hipSuccess) kernel<<<f.cut.blocks(f.cut.row_groups), kThreads, bytes, ctx->stream>>>(f);
        return e;
    };
    const auto with = [&](auto rc) {
        constexpr int RC = decltype(rc)::value;
        const bool even = f.rank % so_elements<T>::V == 0;
        if (f.cut.few) return launch(even ? adapters_out_few_kernel<T, RC, true> : adapters_out_few_kernel<T, RC, false>);
        if (f.base) return launch(even ? adapters_out_kernel<T, RC, true, true> : adapters_out_kernel<T, RC, true, false>);
        return launch(even ? adapters_out_kernel<T, RC, false, true> : adapters_out_kernel<T, RC, false, false>);
    };
    const hipError_t e = f.rank <= 16 ? with(std::integral_constant<int, 1>()) : f.rank <= 32 ? with(std::integral_constant<int, 2>()) : with(std::integral_constant<int, 4>());
    SO_HIP(e);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

} // namespace

extern "C" so_status so_adapters_reserve(so_ctx *ctx, int type, uint32_t m, uint32_t n, uint32_t C, uint32_t rank)
{
    SO_REQUIRE(ctx != nullptr, "so_adapters_reserve: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_adapters_reserve: unknown element type %d", type);
    SO_REQUIRE(rank >= 1 && rank <= kMostRank, "so_adapters_reserve: rank %u is not 1 .. %u", rank, kMostRank);
    SO_REQUIRE(!ctx->capturing, "so_adapters_reserve: a graph is being recorded");
    if (m == 0 || n == 0 || C == 0) return SO_OK;
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    return workspace(ctx, "so_adapters_reserve", bytes_of(cut_of(ctx, type, m, n, C, 1, rank), C));
}

extern "C" so_status so_adapters(so_ctx *ctx, int type, uint32_t m, uint32_t n, uint32_t C, uint32_t count, uint32_t rank, const void *dA, const void *dB, const float *dScale,
                                 const int32_t *dWhich, const void *dX, size_t x_stride, const void *dBase, size_t base_stride, void *dY, size_t y_stride)
{
    SO_REQUIRE(ctx != nullptr, "so_adapters: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_adapters: unknown element type %d", type);
    SO_REQUIRE(rank >= 1 && rank <= kMostRank, "so_adapters: rank %u is not 1 .. %u", rank, kMostRank);
    SO_REQUIRE(count <= 0x7fffffffu, "so_adapters: %u adapters are too many", count);
    if (m == 0 || C == 0) return SO_OK;
    SO_REQUIRE(n > 0, "so_adapters: no input features");
    SO_REQUIRE(dX && dY && dWhich && (count == 0 || (dA && dB)), "so_adapters: null tensor");
    SO_REQUIRE(x_stride >= C && y_stride >= C && (!dBase || base_stride >= C), "so_adapters: a stride is shorter than a row");
    SO_REQUIRE(dY != dX && dY != dA && dY != dB && dY != (const void *)dWhich && dY != (const void *)dScale, "so_adapters: the result is an input");
    SO_REQUIRE(dY != dBase || y_stride == base_stride, "so_adapters: in place needs one stride");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const Cut c = cut_of(ctx, type, m, n, C, count, rank);
    if (const so_status s = workspace(ctx, "so_adapters", bytes_of(c, C)); s != SO_OK) return s;
    so_status status = SO_OK;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        status = run<T>(ctx, {(const T *)dA, (const T *)dB, (const T *)dX, (const T *)dBase, (T *)dY, dScale, dWhich, (float *)ctx->mm_part->p, x_stride, base_stride, y_stride, m, n, C, count, rank, c});
    });
    return status;
}
