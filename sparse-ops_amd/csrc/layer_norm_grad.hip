// The layer norm's gradient on [F x B] activations, in fp32 whatever the element type, one rounding at the end: with g = dy gamma, h = (x - mean) rstd,
//
//   dx = rstd (g - sum_f g / F - h sum_f (g h) / F),  dgamma_f = sum_b dy h,  dbeta_f = sum_b dy
//
// dx needs two sums down every column, dgamma and dbeta two sums along every row; 1 / deviation is taken out of the former.  A batch of a few columns is one workgroup's, in one launch.
// Otherwise two launches cut the matrix into tiles of 1, 2, 4 or 8 lanes of 16 bytes a row and parts of 1024, 512, 256 or 128 features: the first takes the sums of a tile and a part, the
// second adds a tile's parts and writes dx, and its last workgroups add a row's tiles.  All sums are taken in the same order on every call: no atomics.
//
// What bounds it: X and dY come twice, since a workgroup's registers do not hold a tile's columns; 4096 x 8192 bf16 takes 67 us, 34.6 + 33.8, where the 335 MB that it then moves take
// 53 at a large copy's rate of 6.35 TB/s (32 for one reading).  The second launch runs at 6 TB/s, the first, all reading, at 3.9: its 21 vector instructions an element are 18 us of it.  More
// than a third of them are sums over lanes and the way out, once for every four rows of a thread.
#include "layer_norm.h"

using namespace so_norm;

namespace {

// 16 rows from 16 * `group` on: their sums over `parts` arrays of F in `rows`, 16 threads a row.  `lds` holds kThreads values.
__device__ __forceinline__ void join_rows(float2 *lds, uint32_t group, uint32_t F, uint32_t parts, const float2 *__restrict__ rows, float *__restrict__ dgamma, float *__restrict__ dbeta)
{
    const uint64_t f = (uint64_t)group * 16u + threadIdx.x % 16u;
    float2 s = make_float2(0.0f, 0.0f);
    if (f < F)
        for (uint32_t p = threadIdx.x / 16u; p < parts; p += 64u) {
            float2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = p + 16u * i < parts ? rows[(size_t)(p + 16u * i) * F + f] : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s.x += v[i].x;
                s.y += v[i].y;
            }
        }
    lds[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < 16u && f < F) {
        for (uint32_t i = 1; i < 16u && i < parts; ++i) {
            s.x += lds[i * 16u + threadIdx.x].x;
            s.y += lds[i * 16u + threadIdx.x].y;
        }
        if (dgamma) dgamma[f] = s.x;
        if (dbeta) dbeta[f] = s.y;
    }
}

// What a thread knows of its columns.
template <int V>
struct Columns {
    float rs[V], me[V];
    __device__ __forceinline__ Columns(const float *mean, const float *rstd, uint32_t c0, uint32_t left)
    {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            rs[e] = me[e] = 0.0f;
            if ((uint32_t)e < left) {
                rs[e] = rstd[c0 + e];
                me[e] = mean[c0 + e];
            }
        }
    }
};

// The held rows' part of the column sums, s[e] += g and s[V + e] += g (x - mean), and of the row sums.  Columns that do not exist count for neither: what was read there may be
// anything.
template <class T, int LC, int RPT, int NT, bool FULL, class Gamma, class Row>
__device__ __forceinline__ void add_rows(const Place<T, LC, RPT, NT, FULL> &at, const typename so_elements<T>::plain (&x)[RPT], const typename so_elements<T>::plain (&dy)[RPT],
                                         Gamma &&gamma, const Columns<so_elements<T>::V> &c, float (&s)[2 * so_elements<T>::V], Row &&row)
{
    constexpr int V = so_elements<T>::V;
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
        float dga = 0.0f, dbe = 0.0f;
        const float ga = gamma(k);
        if (at.in(k))
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const bool there = FULL || (uint32_t)e < at.left;
                const float d = there ? (float)dy[k][e] : 0.0f, t = there ? (float)x[k][e] - c.me[e] : 0.0f, dt = d * t;
                dbe += d;
                dga = fmaf(dt, c.rs[e], dga);
                s[e] = fmaf(d, ga, s[e]);
                s[V + e] = fmaf(dt, ga, s[V + e]);
            }
        row(k, dga, dbe);
    }
}

// dx of the held rows; a column's sums over F in s, the second times 1 / deviation twice.
template <class T, int LC, int RPT, int NT, bool FULL, class Gamma>
__device__ __forceinline__ void write_grads(const Place<T, LC, RPT, NT, FULL> &at, const typename so_elements<T>::plain (&x)[RPT], const typename so_elements<T>::plain (&dy)[RPT],
                                            Gamma &&gamma, const Columns<so_elements<T>::V> &c, const float (&s)[2 * so_elements<T>::V], T *Dx, size_t lddx)
{
    constexpr int V = so_elements<T>::V;
    if (!FULL && !at.left) return;
    T *p = Dx + (size_t)(at.row0 + at.row(0)) * lddx + at.c0;
    const size_t step = (size_t)Place<T, LC, RPT, NT, FULL>::RL * lddx;
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.in(k)) {
            const float ga = gamma(k);
            float out[V];
#pragma unroll
            for (int e = 0; e < V; ++e) out[e] = fmaf(c.me[e] - (float)x[k][e], s[V + e], fmaf((float)dy[k][e], ga, -s[e])) * c.rs[e];
            so_group_store(p + k * step, at.left, out);
        }
}

// A batch of one tile of columns, all features in one workgroup's registers: one launch, one reading.
template <class T, int LC, int RPT, int NT>
__global__ __launch_bounds__(NT)
void norm_grad_one_kernel(uint32_t F, uint32_t B, const T *X, size_t ldx, const T *Dy, size_t lddy, const float *__restrict__ gamma, const float *__restrict__ mean,
                          const float *__restrict__ rstd, T *Dx, size_t lddx, float *__restrict__ dgamma, float *__restrict__ dbeta)
{
    constexpr int V = so_elements<T>::V;
    __shared__ float lds[(NT / 64 + 1) * LC * 2 * V];
    by_fullness<LC * V>(0, B, [&](auto full) {
        const Place<T, LC, RPT, NT, decltype(full)::value> at(F, B, 0, 0);
        typename so_elements<T>::plain x[RPT], dy[RPT];
        float ga[RPT];
        load_rows(at, ga, gamma, 1.0f);
        const auto gamma_of = [&](int k) { return ga[k]; };
        const Columns<V> c(mean, rstd, at.c0, at.left);
        at.load(x, dy, X, ldx, Dy, lddy);
        float s[2 * V] = {};
        add_rows(at, x, dy, gamma_of, c, s, [&](int k, float a, float b) {
            a = sum_lanes<LC>(a);
            b = sum_lanes<LC>(b);
            if (at.row(k) < F && threadIdx.x % LC == 0) {
                if (dgamma) dgamma[at.row(k)] = a;
                if (dbeta) dbeta[at.row(k)] = b;
            }
        });
        if (!Dx) return;
        sum_tile<NT, LC>(s, lds);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            s[e] /= (float)F;
            s[V + e] = s[V + e] / (float)F * c.rs[e] * c.rs[e];
        }
        write_grads(at, x, dy, gamma_of, c, s, Dx, lddx);
    });
}

// Of a part and a tile: the column sums and the row sums.
template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_grad_parts_kernel(uint32_t F, uint32_t B, uint32_t tiles, const T *X, size_t ldx, const T *Dy, size_t lddy, const float *__restrict__ gamma,
                            const float *__restrict__ mean, const float *__restrict__ rstd, float2 *__restrict__ cols, float2 *__restrict__ rows)
{
    constexpr int V = so_elements<T>::V;
    __shared__ float lds[(kThreads / 64 + 1) * LC * 2 * V];
    const uint2 which = tile_and_part(tiles);
    by_fullness<LC * V>(which.x, B, [&](auto full) {
        const Place<T, LC, RPT, kThreads, decltype(full)::value> at(F, B, which.x, which.y);
        typename so_elements<T>::plain x[RPT], dy[RPT];
        float ga[RPT];
        load_rows(at, ga, gamma, 1.0f);
        const Columns<V> c(mean, rstd, at.c0, at.left);
        at.load(x, dy, X, ldx, Dy, lddy);
        float s[2 * V] = {};
        add_rows(at, x, dy, [&](int k) { return ga[k]; }, c, s, [&](int k, float a, float b) {
            if (!rows) return;
            a = sum_lanes<LC>(a);
            b = sum_lanes<LC>(b);
            if (at.row(k) < at.rows && threadIdx.x % LC == 0) rows[(size_t)at.tile * F + at.row0 + at.row(k)] = make_float2(a, b);
        });
        if (!cols) return;
        sum_tile<kThreads, LC>(s, lds);
        if (threadIdx.x < LC)
#pragma unroll
            for (int e = 0; e < V; ++e)
                if ((uint32_t)e < at.left) cols[(size_t)at.part * B + at.c0 + e] = make_float2(s[e], s[V + e]);
    });
}

// The sums of a column over parts, from part `first` on.
template <int COLS, class Meanwhile>
__device__ __forceinline__ float2 join_sums(float2 *lds, uint32_t column, uint32_t B, uint32_t first, uint32_t parts, const float2 *__restrict__ cols, Meanwhile &&meanwhile)
{
    return join_parts<COLS>(lds, column, B, parts, make_float2(0.0f, 0.0f), [&](uint32_t p, uint32_t c) { return cols[(size_t)(first + p) * B + c]; },
                            [](float2 &a, float2 b) { a.x += b.x; a.y += b.y; }, meanwhile);
}

// A group of parts to one.
template <int COLS>
__global__ __launch_bounds__(kThreads)
void norm_grad_group_kernel(uint32_t B, uint32_t parts, uint32_t tiles, const float2 *__restrict__ cols, float2 *__restrict__ out)
{
    __shared__ float2 lds[kThreads];
    const uint2 which = tile_and_part(tiles);
    const uint32_t first = which.y * group_of(COLS);
    const float2 all = join_sums<COLS>(lds, which.x * COLS, B, first, min(parts - first, group_of(COLS)), cols, [] {});
    const uint64_t c = (uint64_t)which.x * COLS + threadIdx.x;
    if (threadIdx.x < COLS && c < B) out[(size_t)which.y * B + c] = all;
}

// dx of a part and a tile; the workgroups behind those join the rows' sums over the tiles.
template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_grad_apply_kernel(uint32_t F, uint32_t B, uint32_t parts, uint32_t tiles, uint32_t workers, const T *X, size_t ldx, const T *Dy, size_t lddy,
                            const float *__restrict__ gamma, const float *__restrict__ mean, const float *__restrict__ rstd, const float2 *__restrict__ cols,
                            const float2 *__restrict__ rows, T *Dx, size_t lddx, float *__restrict__ dgamma, float *__restrict__ dbeta)
{
    constexpr int V = so_elements<T>::V, COLS = LC * V;
    __shared__ float2 lds[kThreads], joined[COLS];
    if (blockIdx.x >= workers) {
        join_rows(lds, blockIdx.x - workers, F, tiles, rows, dgamma, dbeta);
        return;
    }
    const uint2 which = tile_and_part(tiles);
    by_fullness<COLS>(which.x, B, [&](auto full) {
        const Place<T, LC, RPT, kThreads, decltype(full)::value> at(F, B, which.x, which.y);
        typename so_elements<T>::plain x[RPT], dy[RPT];
        float ga[RPT];
        const float2 all = join_sums<COLS>(lds, at.tile * COLS, B, 0, parts, cols, [&] {
            load_rows(at, ga, gamma, 1.0f);
            at.load(x, dy, X, ldx, Dy, lddy);
        });
        if (threadIdx.x < COLS) joined[threadIdx.x] = make_float2(all.x / (float)F, all.y / (float)F);
        __syncthreads();
        const Columns<V> c(mean, rstd, at.c0, at.left);
        float s[2 * V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float2 j = joined[threadIdx.x % LC * V + e];
            s[e] = j.x;
            s[V + e] = j.y * c.rs[e] * c.rs[e];
        }
        write_grads(at, x, dy, [&](int k) { return ga[k]; }, c, s, Dx, lddx);
    });
}

// One workgroup for everything: lanes of a row, rows a thread, threads.  None: lanes 0.  In one workgroup / in parts, us, on one X and dY that stay in the caches: fp32 64 x 1 3.3 / 5.7, 2048 x 1 5.7 / 7.5, 256 x 16 4.7 / 5.9,
// 1024 x 16 6.4 / 6.3; bf16 256 x 16 4.4 / 6.0, 1024 x 1 7.7 / 9.0, 784 x 16 7.6 / 7.1.  (With all features held for any batch, one reading instead of two, a workgroup for every tile
// of 32 bytes a row took longer than the two launches: 4096 x 8192 bf16 93 us, 67 in parts: each cache line goes to four compute units, and nothing is loaded while a tile is worked on.)
struct One { uint32_t lanes, rows, threads; };
One one_of(const so_ctx *ctx, int type, uint32_t F, uint32_t B)
{
    const uint32_t V = 16u / (uint32_t)so_type_bytes(type);
    uint32_t lanes = 1;
    while (lanes < 8 && B > lanes * V) lanes *= 2;
    if (ctx->tune.norm_lanes == 0 || B > lanes * V || (uint64_t)F * lanes * V > 8192) return {0, 0, 0};
    const uint32_t per = F * lanes, threads = per <= 512 ? 256 : 1024;
    return {lanes, so_ceil_div(per, threads), threads};
}

// As for_whole: 16-bit types have a row a thread of 1024 at most.
template <int V, class F>
void for_one(const One &w, F &&f)
{
    for_lanes(w.lanes, [&](auto lanes) {
        const std::integral_constant<int, 1> one;
        const std::integral_constant<int, 2> two;
        const std::integral_constant<int, 256> few;
        const std::integral_constant<int, 1024> many;
        if (w.threads == 256) {
            if (w.rows == 1) f(lanes, one, few);
            else f(lanes, two, few);
        } else {
            if (V == 8 || w.rows == 1) f(lanes, one, many);
            else if constexpr (V == 4) f(lanes, two, many);
        }
    });
}

} // namespace

size_t so_norm_grad_bytes(const so_ctx *ctx, int type, uint32_t F, uint32_t B)
{
    if (one_of(ctx, type, F, B).lanes) return 0;
    const Cut c = cut_of(type, F, B);
    return c.cols_bytes + c.rows_bytes;
}

extern "C" so_status so_layer_norm_grad(so_ctx *ctx, int type, uint32_t F, uint32_t B, const void *dX, size_t x_stride, const void *dDy, size_t dy_stride,
                                        const float *dGamma, const float *dMean, const float *dRstd, void *dDx, size_t dx_stride, float *dDgamma, float *dDbeta)
{
    SO_REQUIRE(ctx != nullptr, "so_layer_norm_grad: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_layer_norm_grad: unknown element type %d", type);
    SO_REQUIRE(F > 0 || B == 0, "so_layer_norm_grad: no features");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
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
    SO_REQUIRE(!dDgamma || (dDgamma != dDbeta && dDgamma != dGamma), "so_layer_norm_grad: aliased parameter gradients");
    SO_REQUIRE(!dDbeta || dDbeta != dGamma, "so_layer_norm_grad: aliased parameter gradients");
    const bool params = dDgamma || dDbeta;
    if (!dDx && !params) return SO_OK;
    const Cut c = cut_of(type, F, B);
    SO_REQUIRE(ranges_fit(c, so_ceil_div(F, 16)), "so_layer_norm_grad: %u x %u is too large for one launch", F, B);
    if (const One w = one_of(ctx, type, F, B); w.lanes) {
        so_for_type(type, [&](auto t) {
            using T = decltype(t);
            for_one<so_elements<T>::V>(w, [&](auto lanes, auto held, auto threads) {
                constexpr int LC = decltype(lanes)::value, RPT = decltype(held)::value, NT = decltype(threads)::value;
                norm_grad_one_kernel<T, LC, RPT, NT><<<1, NT, 0, ctx->stream>>>(F, B, (const T *)dX, x_stride, (const T *)dDy, dy_stride, dGamma, dMean, dRstd, (T *)dDx, dx_stride,
                                                                                dDgamma, dDbeta);
            });
        });
        SO_LAUNCH_CHECK();
        return SO_OK;
    }
    if (const so_status s = workspace(ctx, "so_layer_norm_grad", so_norm_grad_bytes(ctx, type, F, B)); s != SO_OK) return s;
    float2 *cols = (float2 *)ctx->mm_part->p, *rows = params ? cols + c.cols_bytes / sizeof(float2) : nullptr;
    const uint32_t workers = dDx ? (uint32_t)c.groups : 0, joiners = params ? so_ceil_div(F, 16) : 0;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        for_lanes(c.lanes, [&](auto lanes) {
            constexpr int LC = decltype(lanes)::value;
            norm_grad_parts_kernel<T, LC, kRows><<<(uint32_t)c.groups, kThreads, 0, ctx->stream>>>(F, B, c.tiles, (const T *)dX, x_stride, (const T *)dDy, dy_stride, dGamma, dMean,
                                                                                                    dRstd, dDx ? cols : nullptr, rows);
            Parts p = {cols, c.parts, 0};
            if (dDx)
                p = few_parts(c, F, B, cols, [&](uint32_t workgroups, const Parts &from, float2 *to) {
                    norm_grad_group_kernel<LC * so_elements<T>::V><<<workgroups, kThreads, 0, ctx->stream>>>(B, from.count, c.tiles, from.at, to);
                });
            norm_grad_apply_kernel<T, LC, kRows><<<workers + joiners, kThreads, 0, ctx->stream>>>(F, B, p.count, c.tiles, workers, (const T *)dX, x_stride, (const T *)dDy, dy_stride,
                                                                                                   dGamma, dMean, dRstd, p.at, rows, (T *)dDx, dx_stride, dDgamma, dDbeta);
        });
    });
    SO_LAUNCH_CHECK();
    return SO_OK;
}
