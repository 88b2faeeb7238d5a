// Layer norm over the features of [F x B] activations (batch contiguous) and its gradient.  Statistics, sums and all arithmetic in fp32 whatever the element type;
// one rounding, of the result.
//
//   mean_b = sum_f x / F,  rstd_b = 1 / sqrt(sum_f (x - mean)^2 / F + eps),  y = (x - mean) rstd gamma_f + beta_f
//   g = dy gamma, h = (x - mean) rstd:  dx = rstd (g - sum_f g / F - h sum_f (g h) / F),  dgamma_f = sum_b dy h,  dbeta_f = sum_b dy
//
// A workgroup takes a tile of columns (LC lanes of 16 bytes a row) and a part of the features, and holds it in registers.  The parts' sums go through the context's workspace, and a second
// launch of the same shape joins them and writes the result.  Sums are taken in the same order on every launch: no atomics.
#include <type_traits>

#include "elements.h"
#include "lane_moves.h"
#include "so_internal.h"

namespace {

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

// Mean m and sum of squared deviations q of two sets of na and nb values from those of each: with t = mb - ma, m = ma + t nb / (na + nb), q = qa + qb + t^2 na nb / (na + nb).  No
// difference of large sums is taken, so a column far from zero keeps its variance.
struct Share { float to, sq; };      // nb / (na + nb), na nb / (na + nb)
__device__ __forceinline__ Share share_of(float na, float nb)
{
    const float sum = na + nb, to = sum > 0.0f ? nb * __builtin_amdgcn_rcpf(sum) : 0.0f;
    return {to, na * to};
}
__device__ __forceinline__ void join(float2 &a, float2 b, Share s)
{
    const float t = b.x - a.x;
    a.x = fmaf(t, s.to, a.x);
    a.y = fmaf(t * t, s.sq, a.y + b.y);
}

// Where a thread stands: its column group and its first row.
template <class T, int LC, int RPT, int NT, bool FULL>      // FULL: all columns of the tile exist
struct Place {
    static constexpr int V = so_elements<T>::V, RL = NT / LC, RS = RL * RPT;         // rows a pass of the workgroup, rows of a part
    uint32_t part, tile, c0, left, row0, rows, features;                             // left: columns of the group that exist; rows: of the part
    __device__ __forceinline__ Place(uint32_t F, uint32_t B, uint32_t parts, uint32_t id)
    {
        tile = id / parts;
        part = id - tile * parts;
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
    // The rows of a matrix that this thread holds, requested one after the other.
    __device__ __forceinline__ void load(typename so_elements<T>::plain (&x)[RPT], const T *X, size_t ld) const
    {
        const T *p = X + (size_t)(row0 + row(0)) * ld + c0;
        const size_t step = (size_t)RL * ld;
        const uint32_t wide = FULL ? 0u : so_group_wide_rows<T>(left, features, ld) - min(so_group_wide_rows<T>(left, features, ld), row0);
#pragma unroll
        for (int k = 0; k < RPT; ++k)
            if (in(k)) x[k] = so_group_load(p + k * step, left, FULL || row(k) < wide);
    }
};

// done(column of the tile, its mean and sum of squared deviations over the rows of the workgroup), in one thread for each column: a thread's own rows first, in one pass as
// they come, as differences from the first of them, then the rows of a wave pair by pair, then the waves.  A thread holds 32 rows at most, and the value that it counts from is one
// of them: the squares that cancel are at most as many times what is left, so the sum keeps all but 5 of its bits wherever the column lies and whatever sticks out of it.  `lds` holds NT / 64 * LC * V values.
template <class T, int LC, int RPT, int NT, bool FULL, class Done>
__device__ __forceinline__ void tile_moments(const Place<T, LC, RPT, NT, FULL> &at, typename so_elements<T>::plain (&x)[RPT], float2 *lds, Done &&done)
{
    constexpr int V = so_elements<T>::V, WAVES = NT / 64;
    static_assert(WAVES == 4 || WAVES == 8 || WAVES == 16, "lanes that a value is passed between");
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u;
    float2 s[V];
    float n = (float)at.held(), from[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        from[e] = at.in(0) ? (float)x[0][e] : 0.0f;
        s[e] = make_float2(0.0f, 0.0f);
    }
#pragma unroll
    for (int k = 1; k < RPT; ++k)
        if (at.in(k))
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float t = (float)x[k][e] - from[e];
                s[e].x += t;
                s[e].y = fmaf(t, t, s[e].y);
            }
    const float per = n > 0.0f ? 1.0f / n : 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float off = s[e].x * per, q = fmaf(-s[e].x, off, s[e].y);
        s[e] = make_float2(from[e] + off, q < 0.0f ? 0.0f : q);                      // NaN stays
    }
    if constexpr (V == 8)
#pragma unroll
        for (int k = 0; k < RPT; ++k) so_group_afresh(x[k]);
    over_rows<LC>([&](auto other) {
        const float nb = other(n);
        const Share w = share_of(n, nb);
#pragma unroll
        for (int e = 0; e < V; ++e) join(s[e], make_float2(other(s[e].x), other(s[e].y)), w);
        n += nb;
    });
    if (lane < LC)
#pragma unroll
        for (int e = 0; e < V; ++e) lds[(wave * LC + lane) * V + e] = s[e];
    __syncthreads();
    // a column's waves in neighbouring lanes
    static_assert(LC * V * WAVES <= NT, "a lane for every column and wave");
    if (threadIdx.x < LC * V * WAVES) {
        const uint32_t w = threadIdx.x % WAVES;
        float2 all = lds[w * (LC * V) + threadIdx.x / WAVES];
        n = (float)at.held_by_wave(w);
        const auto pair = [&](auto distance) {
            constexpr int D = decltype(distance)::value;
            const float nb = so_lanes::across<D>(n);
            join(all, make_float2(so_lanes::across<D>(all.x), so_lanes::across<D>(all.y)), share_of(n, nb));
            n += nb;
        };
        pair(std::integral_constant<int, 1>());
        pair(std::integral_constant<int, 2>());
        if constexpr (WAVES > 4) pair(std::integral_constant<int, 4>());
        if constexpr (WAVES > 8) pair(std::integral_constant<int, 8>());
        if (w == 0) done(threadIdx.x / WAVES, all);
    }
}

// y of the held rows, with the columns' mean and 1 / deviation in `st` for all threads; gamma(k), beta(k): of the k-th of them.
template <class T, int LC, int RPT, int NT, bool FULL, class Gamma, class Beta>
__device__ __forceinline__ void write_rows(const Place<T, LC, RPT, NT, FULL> &at, const typename so_elements<T>::plain (&x)[RPT], const float2 *st, Gamma &&gamma, Beta &&beta, T *Y, size_t ldy)
{
    constexpr int V = so_elements<T>::V;
    if (!FULL && !at.left) return;
    T *y0 = Y + (size_t)(at.row0 + at.row(0)) * ldy + at.c0;
    const size_t step = (size_t)Place<T, LC, RPT, NT, FULL>::RL * ldy;
    float2 c[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        c[e] = st[threadIdx.x % LC * V + e];
        c[e].x *= -c[e].y;
    }
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.in(k)) {
            const float ga = gamma(k), be = beta(k);
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = fmaf(fmaf((float)x[k][e], c[e].y, c[e].x), ga, be);
            so_group_store(y0 + k * step, at.left, y);
        }
}

template <class T, int LC, int RPT, int NT, bool FULL>
__device__ __forceinline__ void load_rows(const Place<T, LC, RPT, NT, FULL> &at, float (&v)[RPT], const float *from, float without)
{
#pragma unroll
    for (int k = 0; k < RPT; ++k) v[k] = from && at.in(k) ? from[at.row0 + at.row(k)] : without;
}

// f(a compile-time truth value): whether all LC * V columns of the tile exist, the same for the whole workgroup.
template <int COLS, class F>
__device__ __forceinline__ void by_fullness(uint32_t tile, uint32_t B, F &&f)
{
    if ((uint64_t)(tile + 1u) * COLS <= B) f(std::true_type());
    else f(std::false_type());
}

// All features of a tile of columns in one workgroup's registers: X is read once.  The tiles go to the XCDs in runs of neighbours, which share cache lines where LC is less than 8.
template <class T, int LC, int RPT, int NT>
__global__ __launch_bounds__(NT)
void norm_whole_kernel(uint32_t F, uint32_t B, uint32_t tiles, uint32_t per_xcd, const T *X, size_t ldx, const float *__restrict__ gamma, const float *__restrict__ beta, float eps, T *Y,
                       size_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out)
{
    constexpr int V = so_elements<T>::V;
    // gamma and beta are asked for with X: those of a thread's rows where there are registers for them, else all features' in turn, for LDS
    constexpr bool OWN = RPT <= 8;
    constexpr int TURNS = OWN ? 1 : RPT / LC > 0 ? RPT / LC : 1;
    extern __shared__ float2 lds[];                              // tile_moments's, the columns' results, gamma and beta [F] unless OWN
    float2 *const st = lds + NT / 64 * LC * V, *const params = st + LC * V;
    const uint32_t id = (blockIdx.x % 8u) * per_xcd + blockIdx.x / 8u;
    if (id >= tiles) return;
    by_fullness<LC * V>(id, B, [&](auto full) {
        const Place<T, LC, RPT, NT, decltype(full)::value> at(F, B, 1, id);
        typename so_elements<T>::plain x[RPT];
        float ga[OWN ? RPT : TURNS] = {}, be[OWN ? RPT : TURNS] = {};
        at.load(x, X, ldx);
        if constexpr (OWN) {
            load_rows(at, ga, gamma, 1.0f);
            load_rows(at, be, beta, 0.0f);
        } else {
#pragma unroll
            for (int i = 0; i < TURNS; ++i) {
                const uint32_t f = threadIdx.x + i * NT;
                ga[i] = gamma && f < F ? gamma[f] : 1.0f;
                be[i] = beta && f < F ? beta[f] : 0.0f;
            }
        }
        tile_moments(at, x, lds, [&](uint32_t col, float2 all) {
            const float rstd = 1.0f / sqrtf(all.y / (float)F + eps);
            st[col] = make_float2(all.x, rstd);
            const uint64_t c = (uint64_t)id * (LC * V) + col;
            if (c < B) {
                if (mean_out) mean_out[c] = all.x;
                if (rstd_out) rstd_out[c] = rstd;
            }
        });
        if constexpr (!OWN)
#pragma unroll
            for (int i = 0; i < TURNS; ++i)
                if (threadIdx.x + i * NT < F) params[threadIdx.x + i * NT] = make_float2(ga[i], be[i]);
        __syncthreads();
        write_rows(at, x, st, [&](int k) { return OWN ? ga[k % (OWN ? RPT : TURNS)] : params[at.row(k)].x; }, [&](int k) { return OWN ? be[k % (OWN ? RPT : TURNS)] : params[at.row(k)].y; }, Y,
                   ldy);
    });
}

// Mean and sum of squared deviations of every column of a part.
template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_parts_kernel(uint32_t F, uint32_t B, uint32_t parts, const T *X, size_t ldx, float2 *__restrict__ cols)
{
    constexpr int V = so_elements<T>::V;
    __shared__ float2 lds[kThreads / 64 * LC * V];
    by_fullness<LC * V>(blockIdx.x / parts, B, [&](auto full) {
        const Place<T, LC, RPT, kThreads, decltype(full)::value> at(F, B, parts, blockIdx.x);
        typename so_elements<T>::plain x[RPT];
        at.load(x, X, ldx);
        tile_moments(at, x, lds, [&](uint32_t col, float2 all) {
            const uint64_t c = (uint64_t)at.tile * (LC * V) + col;
            if (c < B) cols[(size_t)at.part * B + c] = all;
        });
    });
}

// Every thread takes each kThreads / COLS-th part of a column of the tile, take(part, column of B), and add(s, value) adds it to s; the shares of a column are added in the threads below
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
    for (uint32_t p = share; p < end; p += 4u * SHARES) {
        if (p != share) ask(p);
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

template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_apply_kernel(uint32_t F, uint32_t B, uint32_t parts, const T *X, size_t ldx, const float2 *__restrict__ cols, const float *__restrict__ gamma,
                       const float *__restrict__ beta, float eps, T *Y, size_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out)
{
    constexpr int COLS = LC * so_elements<T>::V;
    struct Moments { float2 s; float n; };
    __shared__ Moments lds[kThreads];
    __shared__ float2 st[COLS];
    by_fullness<COLS>(blockIdx.x / parts, B, [&](auto full) {
        using At = Place<T, LC, RPT, kThreads, decltype(full)::value>;
        const At at(F, B, parts, blockIdx.x);
        typename so_elements<T>::plain x[RPT];
        float ga[RPT], be[RPT];
        const uint32_t first = at.tile * COLS;
        const Moments all = join_parts<COLS>(lds, first, B, parts, Moments{make_float2(0.0f, 0.0f), 0.0f},
                                             [&](uint32_t p, uint32_t c) { return Moments{cols[(size_t)p * B + c], (float)min(F - p * At::RS, (uint32_t)At::RS)}; },
                                             [](Moments &a, const Moments &b) { join(a.s, b.s, share_of(a.n, b.n)); a.n += b.n; },
                                             [&] {
                                                 at.load(x, X, ldx);
                                                 load_rows(at, ga, gamma, 1.0f);
                                                 load_rows(at, be, beta, 0.0f);
                                             });
        if (threadIdx.x < COLS) {
            const float rstd = 1.0f / sqrtf(all.s.y / (float)F + eps);
            st[threadIdx.x] = make_float2(all.s.x, rstd);
            const uint64_t c = (uint64_t)first + threadIdx.x;
            if (at.part == 0 && c < B) {
                if (mean_out) mean_out[c] = all.s.x;
                if (rstd_out) rstd_out[c] = rstd;
            }
        }
        __syncthreads();
        write_rows(at, x, st, [&](int k) { return ga[k]; }, [&](int k) { return be[k]; }, Y, ldy);
    });
}

// Of a part and a tile: sum_f g and sum_f g h of every column, sum_b dy h and sum_b dy of every row.
template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_grad_parts_kernel(uint32_t F, uint32_t B, uint32_t parts, const T *X, size_t ldx, const T *Dy, size_t lddy, const float *__restrict__ gamma,
                            const float *__restrict__ mean, const float *__restrict__ rstd, float2 *__restrict__ cols, float2 *__restrict__ rows)
{
    constexpr int V = so_elements<T>::V;
    __shared__ float lds[(kThreads / 64 + 1) * LC * 2 * V];
    const Place<T, LC, RPT, kThreads, false> at(F, B, parts, blockIdx.x);
    typename so_elements<T>::plain x[RPT], dy[RPT];
    float ga[RPT];
    at.load(x, X, ldx);
    at.load(dy, Dy, lddy);
    load_rows(at, ga, gamma, 1.0f);
    float me[V], rs[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        me[e] = (uint32_t)e < at.left ? mean[at.c0 + e] : 0.0f;
        rs[e] = (uint32_t)e < at.left ? rstd[at.c0 + e] : 0.0f;
    }
    float s[2 * V] = {};
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
        float dga = 0.0f, dbe = 0.0f;
        const bool in = at.row(k) < at.rows;
        const uint32_t f = at.row0 + at.row(k);
        if (in && at.left) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if ((uint32_t)e < at.left) {
                    const float d = (float)dy[k][e], h = ((float)x[k][e] - me[e]) * rs[e], dh = d * h;
                    dbe += d;
                    dga += dh;
                    s[e] = fmaf(d, ga[k], s[e]);
                    s[V + e] = fmaf(dh, ga[k], s[V + e]);
                }
        }
        if (rows) {
            dga = sum_lanes<LC>(dga);
            dbe = sum_lanes<LC>(dbe);
            if (in && threadIdx.x % LC == 0) rows[(size_t)at.tile * F + f] = make_float2(dga, dbe);
        }
    }
    if (!cols) return;
    sum_tile<kThreads, LC>(s, lds);
    if (threadIdx.x < LC)
#pragma unroll
        for (int e = 0; e < V; ++e)
            if ((uint32_t)e < at.left) cols[(size_t)at.part * B + at.c0 + e] = make_float2(s[e], s[V + e]);
}

// dx of a part and a tile; the workgroups behind those join the rows' sums over the tiles, 64 rows each.
template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_grad_apply_kernel(uint32_t F, uint32_t B, uint32_t parts, uint32_t tiles, uint32_t workers, const T *X, size_t ldx, const T *Dy, size_t lddy,
                            const float *__restrict__ gamma, const float *__restrict__ mean, const float *__restrict__ rstd, const float2 *__restrict__ cols,
                            const float2 *__restrict__ rows, T *Dx, size_t lddx, float *__restrict__ dgamma, float *__restrict__ dbeta)
{
    constexpr int V = so_elements<T>::V;
    __shared__ float2 lds[kThreads], joined[LC * V];
    if (blockIdx.x >= workers) {
        const uint64_t f = (uint64_t)(blockIdx.x - workers) * 64u + threadIdx.x % 64u;
        float2 s = make_float2(0.0f, 0.0f);
        if (f < F)
            for (uint32_t t = threadIdx.x / 64u; t < tiles; t += kThreads / 64) {
                const float2 r = rows[(size_t)t * F + f];
                s.x += r.x;
                s.y += r.y;
            }
        lds[threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.x < 64u && f < F) {
#pragma unroll
            for (int w = 1; w < kThreads / 64; ++w) {
                s.x += lds[w * 64 + threadIdx.x].x;
                s.y += lds[w * 64 + threadIdx.x].y;
            }
            if (dgamma) dgamma[f] = s.x;
            if (dbeta) dbeta[f] = s.y;
        }
        return;
    }
    const Place<T, LC, RPT, kThreads, false> at(F, B, parts, blockIdx.x);
    T *dx0 = Dx + (size_t)at.row0 * lddx + at.c0;
    typename so_elements<T>::plain x[RPT], dy[RPT];
    float ga[RPT];
    at.load(x, X, ldx);
    at.load(dy, Dy, lddy);
    load_rows(at, ga, gamma, 1.0f);
    const float2 all = join_parts<LC * V>(lds, at.tile * (LC * V), B, parts, make_float2(0.0f, 0.0f), [&](uint32_t p, uint32_t c) { return cols[(size_t)p * B + c]; },
                                          [](float2 &a, float2 b) { a.x += b.x; a.y += b.y; }, [] {});
    if (threadIdx.x < LC * V) joined[threadIdx.x] = make_float2(all.x / (float)F, all.y / (float)F);
    __syncthreads();
    if (!at.left) return;
    float me[V], rs[V];
    float2 st[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        me[e] = (uint32_t)e < at.left ? mean[at.c0 + e] : 0.0f;
        rs[e] = (uint32_t)e < at.left ? rstd[at.c0 + e] : 0.0f;
        st[e] = joined[threadIdx.x % LC * V + e];
    }
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.row(k) < at.rows) {
            float out[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float h = ((float)x[k][e] - me[e]) * rs[e];
                out[e] = (fmaf((float)dy[k][e], ga[k], -st[e].x) - h * st[e].y) * rs[e];
            }
            so_group_store(dx0 + (size_t)at.row(k) * lddx, at.left, out);
        }
}

constexpr int kRows = 8;      // rows a thread holds of a part
constexpr uint32_t kWholeMost = 16384;      // rows by lanes of a row that a workgroup holds whole: 256 KB, and twice the rows that it takes

// How [F x B] is cut: lanes of a row, tiles of columns, parts of the features.
struct Cut {
    uint32_t lanes, tiles, parts;
    uint64_t groups;
    size_t cols_bytes, rows_bytes;
};
Cut cut_of(int type, uint32_t F, uint32_t B)
{
    const uint32_t V = 16u / (uint32_t)so_type_bytes(type);
    Cut c;
    c.lanes = B <= V ? 1 : B <= 2 * V ? 2 : B <= 4 * V ? 4 : 8;
    c.tiles = so_ceil_div(B, c.lanes * V);
    c.parts = so_ceil_div(F, kThreads / c.lanes * kRows);
    c.groups = (uint64_t)c.tiles * c.parts;
    c.cols_bytes = (size_t)c.parts * B * sizeof(float2);
    c.rows_bytes = (size_t)c.tiles * F * sizeof(float2);
    return c;
}

template <class F>
void for_lanes(uint32_t lanes, F &&f)
{
    if (lanes == 1) f(std::integral_constant<int, 1>());
    else if (lanes == 2) f(std::integral_constant<int, 2>());
    else if (lanes == 4) f(std::integral_constant<int, 4>());
    else f(std::integral_constant<int, 8>());
}

// A workgroup that holds all features: lanes of a row, rows a thread, threads.  None: lanes 0.
struct Whole { uint32_t lanes, rows, threads; };
Whole whole_of(const so_ctx *ctx, int type, uint32_t F, uint32_t B)
{
    const uint32_t V = 16u / (uint32_t)so_type_bytes(type), cus = (uint32_t)ctx->compute_units;
    uint32_t lanes = 8;
    while (lanes > 1 && so_ceil_div(B, lanes * V) < cus) lanes /= 2;
    const int asked = ctx->tune.norm_lanes;
    if (asked == 0) return {0, 0, 0};
    if (asked == 1 || asked == 2 || asked == 4 || asked == 8) lanes = (uint32_t)asked;
    while (lanes > 1 && F > kWholeMost / lanes) lanes /= 2;
    if (F > kWholeMost / 2) return {0, 0, 0};
    const uint32_t per = F * lanes;                               // threads at a row each
    const bool few = so_ceil_div(B, lanes * V) < cus;
    // One launch and one reading against two: it is the slower one only where long columns leave most compute units without a tile or give them 16 bytes of a row each (a cache line a
    // row and workgroup, in and out).  Whole / in parts, us: fp32 1024 x 1024 6.3 / 7.1, 4096 x 16 7.2 / 8.0, 4096 x 256 9.8 / 7.5, 4096 x 1024 16.7 / 11.3, 4096 x 4096 23.7 / 37.9;
    // bf16 2048 x 64 8.1 / 7.6, 4096 x 1024 13.4 / 9.1, 2048 x 16384 26 / 37, 8192 x 4096 35 / 42.
    if (asked < 0 && F > 1024 && (uint64_t)F * B > 98304 && (few || lanes == 1)) return {0, 0, 0};
    uint32_t threads = per <= 512 ? 256 : few && per <= 8192 ? 1024 : per <= 4096 ? 256 : 512, rows = 1;
    while (rows * threads < per) rows *= 2;
    return {lanes, rows, threads};
}

template <class F>
void for_whole(const Whole &w, F &&f)
{
    const auto rows = [&](auto lanes, auto threads) {
        constexpr int NT = decltype(threads)::value;
        if constexpr (NT == 512) {
            if (w.rows == 16) f(lanes, std::integral_constant<int, 16>(), threads);
            else f(lanes, std::integral_constant<int, 32>(), threads);
        } else {
            if (w.rows == 1) f(lanes, std::integral_constant<int, 1>(), threads);
            else if (w.rows == 2) f(lanes, std::integral_constant<int, 2>(), threads);
            else if (w.rows == 4) f(lanes, std::integral_constant<int, 4>(), threads);
            else if (NT == 1024 || w.rows == 8) f(lanes, std::integral_constant<int, 8>(), threads);
            else if constexpr (NT == 256) f(lanes, std::integral_constant<int, 16>(), threads);
        }
    };
    for_lanes(w.lanes, [&](auto lanes) {
        if (w.threads == 256) rows(lanes, std::integral_constant<int, 256>());
        else if (w.threads == 512) rows(lanes, std::integral_constant<int, 512>());
        else rows(lanes, std::integral_constant<int, 1024>());
    });
}

bool ranges_fit(const Cut &c, uint32_t F) { return c.groups + so_ceil_div(F, 64) < (1ull << 31); }

so_status workspace(so_ctx *ctx, const char *who, size_t bytes)
{
    SO_REQUIRE(!ctx->capturing || (ctx->mm_part && ctx->mm_part->bytes >= bytes),
               "%s: the context's workspace must grow, which cannot be done while a graph is being recorded (call so_layer_norm_reserve, or launch this shape "
               "once, before recording)", who);
    return so_matmul_workspace(ctx, bytes, 4);
}

} // namespace

extern "C" so_status so_layer_norm_reserve(so_ctx *ctx, int type, uint32_t F, uint32_t B)
{
    SO_REQUIRE(ctx != nullptr, "so_layer_norm_reserve: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_layer_norm_reserve: unknown element type %d", type);
    SO_REQUIRE(!ctx->capturing, "so_layer_norm_reserve: a graph is being recorded");
    if (F == 0 || B == 0) return SO_OK;
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const Cut c = cut_of(type, F, B);
    SO_REQUIRE(ranges_fit(c, F), "so_layer_norm_reserve: %u x %u is too large for one launch", F, B);
    return workspace(ctx, "so_layer_norm_reserve", c.cols_bytes + c.rows_bytes);
}

extern "C" so_status so_layer_norm(so_ctx *ctx, int type, uint32_t F, uint32_t B, const void *dX, size_t x_stride, const float *dGamma, const float *dBeta,
                                   float eps, void *dY, size_t y_stride, float *dMean, float *dRstd)
{
    SO_REQUIRE(ctx != nullptr, "so_layer_norm: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_layer_norm: unknown element type %d", type);
    SO_REQUIRE(eps >= 0.0f, "so_layer_norm: eps is negative or not a number");
    if (B == 0) return SO_OK;
    SO_REQUIRE(F > 0, "so_layer_norm: no features");
    SO_REQUIRE(dX && dY, "so_layer_norm: null tensor");
    SO_REQUIRE(x_stride >= B && y_stride >= B, "so_layer_norm: a stride is shorter than a row");
    SO_REQUIRE(dX != dY || x_stride == y_stride, "so_layer_norm: in place needs one stride");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const Cut c = cut_of(type, F, B);
    SO_REQUIRE(ranges_fit(c, F), "so_layer_norm: %u x %u is too large for one launch", F, B);
    if (const Whole w = whole_of(ctx, type, F, B); w.lanes) {
        const uint32_t tiles = so_ceil_div(B, w.lanes * (16u / (uint32_t)so_type_bytes(type))), per_xcd = so_ceil_div(tiles, 8);
        hipError_t allowed = hipSuccess;
        so_for_type(type, [&](auto t) {
            using T = decltype(t);
            for_whole(w, [&](auto lanes, auto rows, auto threads) {
                constexpr int LC = decltype(lanes)::value, RPT = decltype(rows)::value, NT = decltype(threads)::value;
                const uint32_t lds = ((NT / 64 + 1) * LC * so_elements<T>::V + (RPT <= 8 ? 0u : F)) * (uint32_t)sizeof(float2);
                const auto kernel = norm_whole_kernel<T, LC, RPT, NT>;
                if (lds > 48u * 1024u) allowed = so_allow_big_lds(ctx, (const void *)kernel);
                if (allowed == hipSuccess) kernel<<<per_xcd * 8, NT, lds, ctx->stream>>>(F, B, tiles, per_xcd, (const T *)dX, x_stride, dGamma, dBeta, eps, (T *)dY, y_stride, dMean, dRstd);
            });
        });
        SO_HIP(allowed);
        SO_LAUNCH_CHECK();
        return SO_OK;
    }
    if (const so_status s = workspace(ctx, "so_layer_norm", c.cols_bytes); s != SO_OK) return s;
    float2 *cols = (float2 *)ctx->mm_part->p;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        for_lanes(c.lanes, [&](auto lanes) {
            constexpr int LC = decltype(lanes)::value;
            norm_parts_kernel<T, LC, kRows><<<(uint32_t)c.groups, kThreads, 0, ctx->stream>>>(F, B, c.parts, (const T *)dX, x_stride, cols);
            norm_apply_kernel<T, LC, kRows><<<(uint32_t)c.groups, kThreads, 0, ctx->stream>>>(F, B, c.parts, (const T *)dX, x_stride, cols, dGamma, dBeta, eps, (T *)dY, y_stride,
                                                                                               dMean, dRstd);
        });
    });
    SO_LAUNCH_CHECK();
    return SO_OK;
}

extern "C" so_status so_layer_norm_grad(so_ctx *ctx, int type, uint32_t F, uint32_t B, const void *dX, size_t x_stride, const void *dDy, size_t dy_stride,
                                        const float *dGamma, const float *dMean, const float *dRstd, void *dDx, size_t dx_stride, float *dDgamma, float *dDbeta)
{
    SO_REQUIRE(ctx != nullptr, "so_layer_norm_grad: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_layer_norm_grad: unknown element type %d", type);
    SO_REQUIRE(F > 0 || B == 0, "so_layer_norm_grad: no features");
    if (B == 0) {                                                                    // sums over no columns
        if (F && dDgamma)
            if (const so_status s = so_fill_zero(ctx, dDgamma, (size_t)F * sizeof(float)); s != SO_OK) return s;
        if (F && dDbeta)
            if (const so_status s = so_fill_zero(ctx, dDbeta, (size_t)F * sizeof(float)); s != SO_OK) return s;
        return SO_OK;
    }
    SO_REQUIRE(dX && dDy && dMean && dRstd, "so_layer_norm_grad: null tensor");
    SO_REQUIRE(x_stride >= B && dy_stride >= B && (!dDx || dx_stride >= B), "so_layer_norm_grad: a stride is shorter than a row");
    SO_REQUIRE((dDx != dX || dx_stride == x_stride) && (dDx != dDy || dx_stride == dy_stride), "so_layer_norm_grad: in place needs one stride");
    const bool params = dDgamma || dDbeta;
    if (!dDx && !params) return SO_OK;
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const Cut c = cut_of(type, F, B);
    SO_REQUIRE(ranges_fit(c, F), "so_layer_norm_grad: %u x %u is too large for one launch", F, B);
    if (const so_status s = workspace(ctx, "so_layer_norm_grad", c.cols_bytes + c.rows_bytes); s != SO_OK) return s;
    float2 *cols = (float2 *)ctx->mm_part->p, *rows = params ? cols + (size_t)c.parts * B : nullptr;
    const uint32_t workers = dDx ? (uint32_t)c.groups : 0, joiners = params ? so_ceil_div(F, 64) : 0;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        for_lanes(c.lanes, [&](auto lanes) {
            constexpr int LC = decltype(lanes)::value;
            norm_grad_parts_kernel<T, LC, kRows><<<(uint32_t)c.groups, kThreads, 0, ctx->stream>>>(F, B, c.parts, (const T *)dX, x_stride, (const T *)dDy, dy_stride, dGamma, dMean,
                                                                                                    dRstd, dDx ? cols : nullptr, rows);
            norm_grad_apply_kernel<T, LC, kRows><<<workers + joiners, kThreads, 0, ctx->stream>>>(F, B, c.parts, c.tiles, workers, (const T *)dX, x_stride, (const T *)dDy, dy_stride,
                                                                                                   dGamma, dMean, dRstd, cols, rows, (T *)dDx, dx_stride, dDgamma, dDbeta);
        });
    });
    SO_LAUNCH_CHECK();
    return SO_OK;
}
