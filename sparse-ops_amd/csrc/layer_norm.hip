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

constexpr int kThreads = 256, kWaves = kThreads / 64;

// Columns of a tile are LC lanes of V; the lanes of a wave beyond that are rows.  The sum of v over the rows of the wave, in all its lanes.
template <int LC>
__device__ __forceinline__ float sum_rows(float v)
{
    static_assert(LC == 1 || LC == 2 || LC == 4 || LC == 8, "lanes of a row");
    {
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
    }
    {
        const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
    }
    if constexpr (LC <= 8) v += so_lanes::across<8>(v);
    if constexpr (LC <= 4) v += so_lanes::across<4>(v);
    if constexpr (LC <= 2) v += so_lanes::across<2>(v);
    if constexpr (LC <= 1) v += so_lanes::across<1>(v);
    return v;
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

// N values per thread summed over all rows of the workgroup's tile, in all its threads.  `lds` holds kWaves * LC * N floats that no thread uses between the
// barrier before the call and the one after it.
template <int LC, int N>
__device__ __forceinline__ void sum_tile(float (&v)[N], float *lds)
{
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u, lc = lane % LC;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sum_rows<LC>(v[i]);
    if (lane < LC)
#pragma unroll
        for (int i = 0; i < N; ++i) lds[(wave * LC + lane) * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) s += lds[(w * LC + lc) * N + i];
        v[i] = s;
    }
    __syncthreads();
}

// Where a thread stands: its column group and its first row.
template <class T, int LC, int RPT>
struct Place {
    static constexpr int V = so_elements<T>::V, RL = kThreads / LC, RS = RL * RPT;   // rows a pass of the workgroup, rows of a part
    uint32_t part, tile, c0, left, row0, rows;                                       // left: columns of the group that exist; rows: of the part
    __device__ __forceinline__ Place(uint32_t F, uint32_t B, uint32_t parts, uint32_t id)
    {
        tile = id / parts;
        part = id - tile * parts;
        const uint64_t c = (uint64_t)tile * (LC * V) + threadIdx.x % LC * V;
        left = c >= B ? 0u : min(B - (uint32_t)c, (uint32_t)V);
        c0 = (uint32_t)c;
        row0 = part * RS;
        rows = min(F - row0, (uint32_t)RS);
    }
    __device__ __forceinline__ uint32_t row(int k) const { return (uint32_t)k * RL + threadIdx.x / LC; }      // inside the part
};

// Mean and sum of squared deviations of every column of a part: the mean of the held values first, then the deviations from it, whose own mean corrects the
// first (a sum of many values far from zero rounds; a sum of deviations does not).
template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_parts_kernel(uint32_t F, uint32_t B, uint32_t parts, const T *X, size_t ldx, float2 *__restrict__ cols)
{
    constexpr int V = so_elements<T>::V;
    __shared__ float lds[kWaves * LC * 2 * V];
    const Place<T, LC, RPT> at(F, B, parts, blockIdx.x);
    const T *x0 = X + (size_t)at.row0 * ldx + at.c0;
    typename so_elements<T>::plain x[RPT];
    float m[V] = {};
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.row(k) < at.rows && at.left) x[k] = so_group_load(x0 + (size_t)at.row(k) * ldx, at.left);
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.row(k) < at.rows && at.left)
#pragma unroll
            for (int e = 0; e < V; ++e) m[e] += (float)x[k][e];
    sum_tile<LC>(m, lds);
    const float n = (float)at.rows;
#pragma unroll
    for (int e = 0; e < V; ++e) m[e] /= n;
    float d[2 * V] = {};
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.row(k) < at.rows && at.left)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float t = (float)x[k][e] - m[e];
                d[e] += t;
                d[V + e] = fmaf(t, t, d[V + e]);
            }
    sum_tile<LC>(d, lds);
    if (threadIdx.x < LC)
#pragma unroll
        for (int e = 0; e < V; ++e)
            if ((uint32_t)e < at.left) {
                const float off = d[e] / n;
                const float m2 = d[V + e] - off * d[e];
                cols[(size_t)at.part * B + at.c0 + e] = make_float2(m[e] + off, m2 < 0.0f ? 0.0f : m2);      // NaN stays
            }
}

// The columns of a tile from their parts: f(column of the tile, its number) gives two floats that end up in LDS for all threads.
template <int COLS, class F>
__device__ __forceinline__ void join_columns(float2 (&joined)[COLS], uint32_t first, uint32_t B, F &&f)
{
    if (threadIdx.x < COLS) {
        const uint64_t c = (uint64_t)first + threadIdx.x;
        joined[threadIdx.x] = c < B ? f((uint32_t)c) : make_float2(0.0f, 0.0f);
    }
    __syncthreads();
}

template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_apply_kernel(uint32_t F, uint32_t B, uint32_t parts, const T *X, size_t ldx, const float2 *__restrict__ cols, const float *__restrict__ gamma,
                       const float *__restrict__ beta, float eps, T *Y, size_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out)
{
    constexpr int V = so_elements<T>::V, RS = Place<T, LC, RPT>::RS;
    __shared__ float2 joined[LC * V];
    const Place<T, LC, RPT> at(F, B, parts, blockIdx.x);
    const T *x0 = X + (size_t)at.row0 * ldx + at.c0;
    T *y0 = Y + (size_t)at.row0 * ldy + at.c0;
    typename so_elements<T>::plain x[RPT];
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.row(k) < at.rows && at.left) x[k] = so_group_load(x0 + (size_t)at.row(k) * ldx, at.left);
    join_columns(joined, at.tile * (LC * V), B, [&](uint32_t c) {
        float sum = 0.0f;
        for (uint32_t s = 0; s < parts; ++s) sum = fmaf((float)min(F - s * RS, (uint32_t)RS), cols[(size_t)s * B + c].x, sum);
        const float mean = sum / (float)F;
        float m2 = 0.0f;
        for (uint32_t s = 0; s < parts; ++s) {
            const float2 p = cols[(size_t)s * B + c];
            const float off = p.x - mean;
            m2 += fmaf((float)min(F - s * RS, (uint32_t)RS) * off, off, p.y);
        }
        const float rstd = 1.0f / sqrtf(m2 / (float)F + eps);
        if (at.part == 0) {
            if (mean_out) mean_out[c] = mean;
            if (rstd_out) rstd_out[c] = rstd;
        }
        return make_float2(mean, rstd);
    });
    if (!at.left) return;
    float2 st[V];
#pragma unroll
    for (int e = 0; e < V; ++e) st[e] = joined[threadIdx.x % LC * V + e];
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.row(k) < at.rows) {
            const uint32_t f = at.row0 + at.row(k);
            const float ga = gamma ? gamma[f] : 1.0f, be = beta ? beta[f] : 0.0f;
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = fmaf(((float)x[k][e] - st[e].x) * st[e].y, ga, be);
            so_group_store(y0 + (size_t)at.row(k) * ldy, at.left, y);
        }
}

// Of a part and a tile: sum_f g and sum_f g h of every column, sum_b dy h and sum_b dy of every row.
template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_grad_parts_kernel(uint32_t F, uint32_t B, uint32_t parts, const T *X, size_t ldx, const T *Dy, size_t lddy, const float *__restrict__ gamma,
                            const float *__restrict__ mean, const float *__restrict__ rstd, float2 *__restrict__ cols, float2 *__restrict__ rows)
{
    constexpr int V = so_elements<T>::V;
    __shared__ float lds[kWaves * LC * 2 * V];
    const Place<T, LC, RPT> at(F, B, parts, blockIdx.x);
    const T *x0 = X + (size_t)at.row0 * ldx + at.c0, *dy0 = Dy + (size_t)at.row0 * lddy + at.c0;
    typename so_elements<T>::plain x[RPT], dy[RPT];
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.row(k) < at.rows && at.left) {
            x[k] = so_group_load(x0 + (size_t)at.row(k) * ldx, at.left);
            dy[k] = so_group_load(dy0 + (size_t)at.row(k) * lddy, at.left);
        }
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
            const float ga = gamma ? gamma[f] : 1.0f;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if ((uint32_t)e < at.left) {
                    const float d = (float)dy[k][e], h = ((float)x[k][e] - me[e]) * rs[e], dh = d * h;
                    dbe += d;
                    dga += dh;
                    s[e] = fmaf(d, ga, s[e]);
                    s[V + e] = fmaf(dh, ga, s[V + e]);
                }
        }
        if (rows) {
            dga = sum_lanes<LC>(dga);
            dbe = sum_lanes<LC>(dbe);
            if (in && threadIdx.x % LC == 0) rows[(size_t)at.tile * F + f] = make_float2(dga, dbe);
        }
    }
    if (!cols) return;
    sum_tile<LC>(s, lds);
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
    __shared__ float2 joined[LC * V > kThreads ? LC * V : kThreads];
    if (blockIdx.x >= workers) {
        const uint64_t f = (uint64_t)(blockIdx.x - workers) * 64u + threadIdx.x % 64u;
        float2 s = make_float2(0.0f, 0.0f);
        if (f < F)
            for (uint32_t t = threadIdx.x / 64u; t < tiles; t += kWaves) {
                const float2 r = rows[(size_t)t * F + f];
                s.x += r.x;
                s.y += r.y;
            }
        joined[threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.x < 64u && f < F) {
#pragma unroll
            for (int w = 1; w < kWaves; ++w) {
                s.x += joined[w * 64 + threadIdx.x].x;
                s.y += joined[w * 64 + threadIdx.x].y;
            }
            if (dgamma) dgamma[f] = s.x;
            if (dbeta) dbeta[f] = s.y;
        }
        return;
    }
    const Place<T, LC, RPT> at(F, B, parts, blockIdx.x);
    const T *x0 = X + (size_t)at.row0 * ldx + at.c0, *dy0 = Dy + (size_t)at.row0 * lddy + at.c0;
    T *dx0 = Dx + (size_t)at.row0 * lddx + at.c0;
    typename so_elements<T>::plain x[RPT], dy[RPT];
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.row(k) < at.rows && at.left) {
            x[k] = so_group_load(x0 + (size_t)at.row(k) * ldx, at.left);
            dy[k] = so_group_load(dy0 + (size_t)at.row(k) * lddy, at.left);
        }
    float2(&columns)[LC * V] = reinterpret_cast<float2(&)[LC * V]>(joined);
    join_columns(columns, at.tile * (LC * V), B, [&](uint32_t c) {
        float2 s = make_float2(0.0f, 0.0f);
        for (uint32_t p = 0; p < parts; ++p) {
            const float2 q = cols[(size_t)p * B + c];
            s.x += q.x;
            s.y += q.y;
        }
        return make_float2(s.x / (float)F, s.y / (float)F);
    });
    if (!at.left) return;
    float me[V], rs[V];
    float2 st[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        me[e] = (uint32_t)e < at.left ? mean[at.c0 + e] : 0.0f;
        rs[e] = (uint32_t)e < at.left ? rstd[at.c0 + e] : 0.0f;
        st[e] = columns[threadIdx.x % LC * V + e];
    }
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.row(k) < at.rows) {
            const float ga = gamma ? gamma[at.row0 + at.row(k)] : 1.0f;
            float out[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float h = ((float)x[k][e] - me[e]) * rs[e];
                out[e] = (fmaf((float)dy[k][e], ga, -st[e].x) - h * st[e].y) * rs[e];
            }
            so_group_store(dx0 + (size_t)at.row(k) * lddx, at.left, out);
        }
}

constexpr int kRows = 8;      // rows a thread holds

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
