// What the layer norm's forward pass and gradient share: how [F x B] is cut into tiles of columns and parts of the features, and the sums over them.
#pragma once
#include <type_traits>

#include "elements.h"
#include "lane_moves.h"
#include "so_internal.h"

namespace so_norm {

constexpr int kThreads = 256;      // of a workgroup that takes a part of the features

// op(value of the lane that differs in a bit above the LC lanes of a row) for each such bit of the lane number: the rows of a wave, pair by pair.  other(v): the partner's v.
template <int LC, class F>
__device__ __forceinline__ void over_rows(F &&f)
{
    static_assert(LC == 1 || LC == 2 || LC == 4 || LC == 8, "lanes of a row");
    const uint32_t lane = threadIdx.x % 64u;
    if constexpr (LC <= 1) f([](float v) { return so_lanes::across<1>(v); });
    if constexpr (LC <= 2) f([](float v) { return so_lanes::across<2>(v); });
    if constexpr (LC <= 4) f([](float v) { return so_lanes::across<4>(v); });
    f([](float v) { return so_lanes::across<8>(v); });
    f([lane](float v) {
        const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(lane & 16u ? h[0] : h[1]);
    });
    f([lane](float v) {
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(lane & 32u ? h[0] : h[1]);
    });
}

// The sum of v over the LC lanes of a row, in all of them.
template <int LC>
__device__ __forceinline__ float sum_lanes(float v)
{
    if constexpr (LC > 1) v += so_lanes::across<1>(v);
    if constexpr (LC > 2) v += so_lanes::across<2>(v);
    if constexpr (LC > 4) v += so_lanes::across<4>(v);
    return v;
}

// N values per thread summed over all rows of the workgroup's tile, in all its threads.  `lds` holds (NT / 64 + 1) * LC * N floats that nothing else is using.
template <int NT, int LC, int N>
__device__ __forceinline__ void sum_tile(float (&v)[N], float *lds)
{
    constexpr int WAVES = NT / 64;
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u;
    over_rows<LC>([&](auto other) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += other(v[i]);
    });
    if (lane < LC)
#pragma unroll
        for (int i = 0; i < N; ++i) lds[(wave * LC + lane) * N + i] = v[i];
    __syncthreads();
    float *total = lds + WAVES * LC * N;
    if (threadIdx.x < LC * N) {
        float s[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s[w] = lds[w * LC * N + threadIdx.x];
#pragma unroll
        for (int step = WAVES / 2; step; step /= 2)
#pragma unroll
            for (int w = 0; w < step; ++w) s[w] += s[w + step];
        total[threadIdx.x] = s[0];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = total[lane % LC * N + i];
}

// Where a thread stands: its column group and its first row.
template <class T, int LC, int RPT, int NT, bool FULL>      // FULL: all columns of the tile exist
struct Place {
    static constexpr int V = so_elements<T>::V, RL = NT / LC, RS = RL * RPT;         // rows a pass of the workgroup, rows of a part
    uint32_t part, tile, c0, left, row0, rows, features;                             // left: columns of the group that exist; rows: of the part
    __device__ __forceinline__ Place(uint32_t F, uint32_t B, uint32_t tile_, uint32_t part_)
    {
        tile = tile_;
        part = part_;
        const uint64_t c = (uint64_t)tile * (LC * V) + threadIdx.x % LC * V;
        left = FULL ? (uint32_t)V : c >= B ? 0u : min(B - (uint32_t)c, (uint32_t)V);
        c0 = (uint32_t)c;
        row0 = part * RS;
        rows = min(F - row0, (uint32_t)RS);
        features = F;
    }
    __device__ __forceinline__ uint32_t row(int k) const { return (uint32_t)k * RL + threadIdx.x / LC; }      // inside the part
    __device__ __forceinline__ bool in(int k) const { return row(k) < rows && (FULL || left); }
    __device__ __forceinline__ uint32_t held() const { return rows > threadIdx.x / LC ? (rows - threadIdx.x / LC + RL - 1u) / RL : 0u; }   // rows of this thread
    __device__ __forceinline__ uint32_t held_by_wave(uint32_t w) const                                        // rows of wave w, of each of its columns
    {
        constexpr uint32_t WR = 64 / LC;
        const uint32_t rest = rows % RL;
        return rows / RL * WR + (rest > w * WR ? min(rest - w * WR, WR) : 0u);
    }
    // Those of two matrices, row by row.
    __device__ __forceinline__ void load(typename so_elements<T>::plain (&x)[RPT], typename so_elements<T>::plain (&y)[RPT], const T *X, size_t ldx, const T *Y, size_t ldy) const
    {
        if constexpr (FULL) {
            const T *p = X + (size_t)row0 * ldx + c0, *q = Y + (size_t)row0 * ldy + c0;
            const uint32_t first = threadIdx.x / LC, last = rows - 1u;
#pragma unroll
            for (int k = 0; k < RPT; ++k) {
                x[k] = so_group_load(p + (row(k) < rows ? first * ldx + k * (RL * ldx) : last * ldx), left, true);
                y[k] = so_group_load(q + (row(k) < rows ? first * ldy + k * (RL * ldy) : last * ldy), left, true);
            }
        } else {
            load(x, X, ldx);
            load(y, Y, ldy);
        }
    }
    // The rows of a matrix that this thread holds, requested one after the other.  A full tile's without a branch: behind the last row that one again, so that the compiler
    // can count which have come and a row is worked on while those after it are on their way (behind branches it waits for all).
    __device__ __forceinline__ void load(typename so_elements<T>::plain (&x)[RPT], const T *X, size_t ld) const
    {
        const size_t step = (size_t)RL * ld;
        if constexpr (FULL) {
            const T *p = X + (size_t)row0 * ld + c0;
            const size_t first = (size_t)(threadIdx.x / LC) * ld, last = (size_t)(rows - 1u) * ld;
#pragma unroll
            for (int k = 0; k < RPT; ++k) x[k] = so_group_load(p + (row(k) < rows ? first + k * step : last), left, true);
        } else {
            const T *p = X + (size_t)(row0 + row(0)) * ld + c0;
            const uint32_t wide = so_group_wide_rows<T>(left, features, ld) - min(so_group_wide_rows<T>(left, features, ld), row0);
#pragma unroll
            for (int k = 0; k < RPT; ++k)
                if (in(k)) x[k] = so_group_load(p + k * step, left, row(k) < wide);
        }
    }
};

// Of the held rows, what `from` has for them.  To be asked for before X: the compiler does not know whether these requests are made.
template <class T, int LC, int RPT, int NT, bool FULL>
__device__ __forceinline__ void load_rows(const Place<T, LC, RPT, NT, FULL> &at, float (&v)[RPT], const float *from, float without)
{
#pragma unroll
    for (int k = 0; k < RPT; ++k) v[k] = without;
    if (from)
#pragma unroll
        for (int k = 0; k < RPT; ++k) v[k] = from[at.row0 + min(at.row(k), at.rows - 1u)];
}

// Which tile (.x) and part a workgroup takes: the tiles of the same rows side by side, so that the chip walks through the matrix as it lies in memory.  (The parts of a tile first, or
// a run of tiles for each XCD: 4096 x 8192 bf16, gradient of both passes 68 us this way, 81 and 96.)
__device__ __forceinline__ uint2 tile_and_part(uint32_t tiles) { return make_uint2(blockIdx.x % tiles, blockIdx.x / tiles); }

// f(a compile-time truth value): whether all LC * V columns of the tile exist, the same for the whole workgroup.
template <int COLS, class F>
__device__ __forceinline__ void by_fullness(uint32_t tile, uint32_t B, F &&f)
{
    if ((uint64_t)(tile + 1u) * COLS <= B) f(std::true_type());
    else f(std::false_type());
}

// Every thread takes each kThreads / COLS-th part of a column of the tile, take(part, column of B), the first one as it is (s where there is none), and add(s, value) adds the others to it; the shares of a column are added in the threads below
// COLS, which get the sum.  meanwhile() asks for other things once the first values are on their way.  `lds` holds kThreads values.
template <int COLS, class Value, class Take, class Add, class Meanwhile>
__device__ __forceinline__ Value join_parts(Value *lds, uint32_t first, uint32_t B, uint32_t parts, Value s, Take &&take, Add &&add, Meanwhile &&meanwhile)
{
    constexpr uint32_t SHARES = kThreads / COLS;
    const uint32_t col = threadIdx.x % COLS, share = threadIdx.x / COLS;
    const uint64_t c = (uint64_t)first + col;
    const uint32_t end = c < B ? parts : 0u;
    Value v[4];
    const auto ask = [&](uint32_t p) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p + i * SHARES < end) v[i] = take(p + i * SHARES, (uint32_t)c);
    };
    ask(share);
    meanwhile();
    if (share < end) s = v[0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
        if (share + i * SHARES < end) add(s, v[i]);
    for (uint32_t p = share + 4u * SHARES; p < end; p += 4u * SHARES) {
        ask(p);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p + i * SHARES < end) add(s, v[i]);
    }
    lds[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < COLS)
        for (uint32_t i = 1; i < SHARES && i < parts; ++i) add(s, lds[i * COLS + col]);
    return s;
}

constexpr int kRows = 4;      // rows a thread holds of a part

// Every workgroup that writes results joins the parts of its columns, which grow with the features as the workgroups do: where a thread would have more than kJoin of them, groups of as many
// are joined to one each first, until it has not.  At once / in groups, us: fp32 40960 x 32, 40 parts a thread, 12.5 / 14.4 (groups of 32); 65536 x 32, 64 parts, 16.3 / 16.8; 65536 x 256 57 / 42;
// 802816 x 32, 784 parts, 579 / 53, three times the matrix at a copy's rate 49.
constexpr uint32_t kJoin = 48;
constexpr uint32_t group_of(uint32_t columns) { return kJoin * (kThreads / columns); }

// How [F x B] is cut: lanes of a row, tiles of columns, parts of the features.
struct Cut {
    uint32_t lanes, tiles, parts, columns;      // columns of a tile
    uint64_t groups;
    size_t cols_bytes, rows_bytes;              // cols: of the parts, behind them their groups
};
static inline Cut cut_of(int type, uint32_t F, uint32_t B)
{
    const uint32_t V = 16u / (uint32_t)so_type_bytes(type);
    Cut c;
    c.lanes = B <= V ? 1 : B <= 2 * V ? 2 : B <= 4 * V ? 4 : 8;
    c.columns = c.lanes * V;
    c.tiles = so_ceil_div(B, c.columns);
    c.parts = so_ceil_div(F, kThreads / c.lanes * kRows);
    c.groups = (uint64_t)c.tiles * c.parts;
    c.cols_bytes = ((size_t)c.parts + (c.parts > group_of(c.columns) ? so_ceil_div(c.parts, group_of(c.columns)) : 0u)) * B * sizeof(float2);
    c.rows_bytes = (size_t)c.tiles * F * sizeof(float2);
    return c;
}

// What the workgroups that write results join: arrays of B, each of so many rows of X.
struct Parts {
    float2 *at;
    uint32_t count, rows;
};
// The parts of a cut in cols, group by group by launch(workgroups, parts, their groups), until they are few enough.
template <class F>
Parts few_parts(const Cut &c, uint32_t features, uint32_t B, float2 *cols, F &&launch)
{
    const uint32_t group = group_of(c.columns);
    Parts p = {cols, c.parts, std::min(features, kThreads / c.lanes * kRows)};
    float2 *to = cols + (size_t)c.parts * B;
    while (p.count > group) {
        const Parts next = {to, so_ceil_div(p.count, group), (uint32_t)std::min<uint64_t>(features, (uint64_t)p.rows * group)};
        launch(c.tiles * next.count, p, next.at);
        to = p.at;
        p = next;
    }
    return p;
}

template <class F>
void for_lanes(uint32_t lanes, F &&f)
{
    if (lanes == 1) f(std::integral_constant<int, 1>());
    else if (lanes == 2) f(std::integral_constant<int, 2>());
    else if (lanes == 4) f(std::integral_constant<int, 4>());
    else f(std::integral_constant<int, 8>());
}

// Of the kernels that take parts, and of the one that holds all features with as many lanes a row as it chooses.
static inline bool ranges_fit(const Cut &c, uint32_t joiners = 0) { return so_grid_fits(c.groups + joiners + 64, kThreads); }

static inline so_status workspace(so_ctx *ctx, const char *who, size_t bytes)
{
    SO_REQUIRE(!ctx->capturing || (ctx->mm_part && ctx->mm_part->bytes >= bytes),
               "%s: the context's workspace must grow, which cannot be done while a graph is being recorded (call so_layer_norm_reserve, or launch this shape "
               "once, before recording)", who);
    return so_matmul_workspace(ctx, bytes, 4);
}

} // namespace so_norm

// csrc/layer_norm_grad.hip: workspace that the gradient of F x B takes.
size_t so_norm_grad_bytes(const so_ctx *ctx, int type, uint32_t F, uint32_t B);
