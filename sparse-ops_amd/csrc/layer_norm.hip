// Layer norm over the features of [F x B] activations (batch contiguous).  Statistics and all arithmetic in fp32 whatever the element type; one rounding, of the result.
//
//   mean_b = sum_f x / F,  rstd_b = 1 / sqrt(sum_f (x - mean)^2 / F + eps),  y = (x - mean) rstd gamma_f + beta_f
//
// A workgroup holds a tile of columns, LC lanes of 16 bytes a row, in registers: all features, in one launch that reads X once, or a part of them, whose moments go through the
// context's workspace to a second launch of the same shape.  Sums are taken in the same order on every launch: no atomics.
#include "layer_norm.h"

using namespace so_norm;

namespace {

// Mean m and sum of squared deviations q of two sets of na and nb values from those of each: with t = mb - ma, m = ma + t nb / (na + nb), q = qa + qb + t^2 na nb / (na + nb).  No
// difference of large sums is taken, so a column far from zero keeps its variance.  The share is taken before the square: beside an empty set (mean 0) t is the column's own size, whose
// square fp32 need not hold.
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
    a.y = fmaf(t * s.sq, t, a.y + b.y);
}

// What a column's mean and sum of squared deviations give: its mean and 1 / deviation.  An infinity or NaN in it leaves the mean no finite number in any order of the joins, and where it
// is an infinity (one row a thread) the squares may still be 0: x - x makes both results NaN then, and adds zero otherwise.
__device__ __forceinline__ float2 results_of(float2 all, uint32_t F, float eps)
{
    const float none = all.x - all.x;
    return make_float2(all.x + none, 1.0f / sqrtf(all.y / (float)F + eps) + none);
}

// done(column of the tile, its mean and sum of squared deviations over the rows of the workgroup), in one thread for each column: a thread's own rows first, their mean in one pass as
// they come, as differences from the first of them, then the deviations from it out of the registers; then the rows of a wave pair by pair, then the waves.  (Squares of the differences
// from the first row in the same pass, less the share of its own, cancel where that row sticks out: 4096 x 8192 bf16 34.8 us instead of 35.6, 4096 x 4096 fp32 32.3 instead of 32.8,
// and 1 / deviation off by up to 350 roundings where one feature carries a column; 21 now.)  `lds` holds NT / 64 * LC * V values.
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
            for (int e = 0; e < V; ++e) s[e].x += (float)x[k][e] - from[e];
    const float per = n > 0.0f ? 1.0f / n : 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) from[e] = s[e].x = fmaf(s[e].x, per, from[e]);
    if constexpr (V == 8)
#pragma unroll
        for (int k = 0; k < RPT; ++k) so_group_afresh(x[k]);
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.in(k))
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float t = (float)x[k][e] - from[e];
                s[e].y = fmaf(t, t, s[e].y);
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
    for (int e = 0; e < V; ++e) c[e] = st[threadIdx.x % LC * V + e];
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (at.in(k)) {
            const float ga = gamma(k), be = beta(k);
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = fmaf(((float)x[k][e] - c[e].x) * c[e].y, ga, be);
            so_group_store(y0 + k * step, at.left, y);
        }
}

// All features of a tile of columns in one workgroup's registers: X is read once.  The tiles go to the XCDs in runs of neighbours, which share cache lines where LC is less than 8.
// Bound by the memory where there are tiles enough, in three phases that do not overlap, since a compute unit holds one large tile: 4096 x 8192 bf16 35.6 us, 3.8 TB/s (a copy 21); by instructions
// where not: 4096 x 1 fp32 5.3 us, of which the 530 vector instructions of each of 16 waves on four SIMDs take 3.5, most of them joins of four columns, three of which do not exist.
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
        const Place<T, LC, RPT, NT, decltype(full)::value> at(F, B, id, 0);
        typename so_elements<T>::plain x[RPT];
        float ga[OWN ? RPT : TURNS] = {}, be[OWN ? RPT : TURNS] = {};
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
        at.load(x, X, ldx);
        tile_moments(at, x, lds, [&](uint32_t col, float2 all) {
            const float2 of = st[col] = results_of(all, F, eps);
            const uint64_t c = (uint64_t)id * (LC * V) + col;
            if (c < B) {
                if (mean_out) mean_out[c] = of.x;
                if (rstd_out) rstd_out[c] = of.y;
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

// Mean and sum of squared deviations of every column of a part; then the parts joined and the result.  4096 x 256 fp32 3.0 + 4.2 us, one workgroup a compute unit.
template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_parts_kernel(uint32_t F, uint32_t B, uint32_t tiles, const T *X, size_t ldx, float2 *__restrict__ cols)
{
    constexpr int V = so_elements<T>::V;
    __shared__ float2 lds[kThreads / 64 * LC * V];
    const uint2 which = tile_and_part(tiles);
    by_fullness<LC * V>(which.x, B, [&](auto full) {
        const Place<T, LC, RPT, kThreads, decltype(full)::value> at(F, B, which.x, which.y);
        typename so_elements<T>::plain x[RPT];
        at.load(x, X, ldx);
        tile_moments(at, x, lds, [&](uint32_t col, float2 all) {
            const uint64_t c = (uint64_t)at.tile * (LC * V) + col;
            if (c < B) cols[(size_t)at.part * B + c] = all;
        });
    });
}

struct Moments { float2 s; float n; };
// Those of a column over parts of `per` rows each, the last one fewer, from part `first` on.
template <int COLS, class Meanwhile>
__device__ __forceinline__ Moments join_moments(Moments *lds, uint32_t column, uint32_t F, uint32_t B, uint32_t first, uint32_t parts, uint32_t per, const float2 *__restrict__ cols,
                                                Meanwhile &&meanwhile)
{
    return join_parts<COLS>(lds, column, B, parts, Moments{make_float2(0.0f, 0.0f), 0.0f},
                            [&](uint32_t p, uint32_t c) { return Moments{cols[(size_t)(first + p) * B + c], (float)min(F - (first + p) * per, per)}; },
                            // (Of two joined none is empty but the second: a thread's first part is taken as it is, lanes and waves hold the first rows of a tile first.  Beside an
                            // empty first one the share would be the hardware's reciprocal of nb times nb, which need not be 1, and a column of one value not keep it as its mean.)
                            [](Moments &a, const Moments &b) { join(a.s, b.s, share_of(a.n, b.n)); a.n += b.n; },
                            meanwhile);
}

// A group of parts to one.
template <int COLS>
__global__ __launch_bounds__(kThreads)
void norm_group_kernel(uint32_t F, uint32_t B, uint32_t parts, uint32_t per, uint32_t tiles, const float2 *__restrict__ cols, float2 *__restrict__ out)
{
    __shared__ Moments lds[kThreads];
    const uint2 which = tile_and_part(tiles);
    const uint32_t first = which.y * group_of(COLS);
    const Moments all = join_moments<COLS>(lds, which.x * COLS, F, B, first, min(parts - first, group_of(COLS)), per, cols, [] {});
    const uint64_t c = (uint64_t)which.x * COLS + threadIdx.x;
    if (threadIdx.x < COLS && c < B) out[(size_t)which.y * B + c] = all.s;
}

template <class T, int LC, int RPT>
__global__ __launch_bounds__(kThreads)
void norm_apply_kernel(uint32_t F, uint32_t B, uint32_t parts, uint32_t per, uint32_t tiles, const T *X, size_t ldx, const float2 *__restrict__ cols, const float *__restrict__ gamma,
                       const float *__restrict__ beta, float eps, T *Y, size_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out)
{
    constexpr int COLS = LC * so_elements<T>::V;
    __shared__ Moments lds[kThreads];
    __shared__ float2 st[COLS];
    const uint2 which = tile_and_part(tiles);
    by_fullness<COLS>(which.x, B, [&](auto full) {
        using At = Place<T, LC, RPT, kThreads, decltype(full)::value>;
        const At at(F, B, which.x, which.y);
        typename so_elements<T>::plain x[RPT];
        float ga[RPT], be[RPT];
        const uint32_t first = at.tile * COLS;
        const Moments all = join_moments<COLS>(lds, first, F, B, 0, parts, per, cols, [&] {
            load_rows(at, ga, gamma, 1.0f);
            load_rows(at, be, beta, 0.0f);
            at.load(x, X, ldx);
        });
        if (threadIdx.x < COLS) {
            const float2 of = st[threadIdx.x] = results_of(all.s, F, eps);
            const uint64_t c = (uint64_t)first + threadIdx.x;
            if (at.part == 0 && c < B) {
                if (mean_out) mean_out[c] = of.x;
                if (rstd_out) rstd_out[c] = of.y;
            }
        }
        __syncthreads();
        write_rows(at, x, st, [&](int k) { return ga[k]; }, [&](int k) { return be[k]; }, Y, ldy);
    });
}

constexpr uint32_t kWholeMost = 16384;      // rows by lanes of a row that a workgroup holds whole: 256 KB; and twice the rows that it takes

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
    // row and workgroup, in and out).  Whole / in parts, us, on one X that stays in the caches where they hold it: fp32 1024 x 1024 6.0 / 6.4, 8192 x 1 6.7 / 7.2, 4096 x 256 9.8 / 6.6, 4096 x 1024 17 / 11, 4096 x 4096 23 / 34; bf16 512 x 1024
    // 4.7 / 6.4, 1024 x 1024 7.6 / 6.6, 2048 x 16 6.8 / 6.6, 4096 x 1 8.3 / 7.5, 2048 x 16384 25 / 39, 8192 x 4096 34 / 40.
    if (lanes == 1 && F * V * V > 131072) return {0, 0, 0};
    if (asked < 0 && (few || lanes == 1) && F * V > 4096 && (uint64_t)F * B > 65536) return {0, 0, 0};
    // 1024 threads where only latency counts, which with more lanes a row is in parts
    const uint32_t threads = per <= 512 ? 256 : lanes == 1 && (few || per > 4096 / V) ? 1024 : per <= 4096 ? 256 : 512;
    uint32_t rows = 1;
    while (rows * threads < per) rows *= 2;
    return {lanes, rows, threads};
}

// f(lanes, rows, threads) as compile-time numbers, for those that whole_of chooses with 16 / V bytes an element.
template <int V, class F>
void for_whole(const Whole &w, F &&f)
{
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 8> eight;
    const std::integral_constant<int, 16> sixteen;
    const std::integral_constant<int, 256> few;
    const std::integral_constant<int, 512> more;
    const std::integral_constant<int, 1024> most;
    const auto more_lanes = [&](auto lanes) {
        if (w.threads == 512) {
            if (w.rows == 16) f(lanes, sixteen, more);
            else f(lanes, std::integral_constant<int, 32>(), more);
        } else {
            if (w.rows == 1) f(lanes, one, few);
            else if (w.rows == 2) f(lanes, two, few);
            else if (w.rows == 4) f(lanes, four, few);
            else if (w.rows == 8) f(lanes, eight, few);
            else f(lanes, sixteen, few);
        }
    };
    if (w.lanes == 2) more_lanes(two);
    else if (w.lanes == 4) more_lanes(four);
    else if (w.lanes == 8) more_lanes(eight);
    else if (w.threads == 256) {
        if (w.rows == 1) f(one, one, few);
        else if (V == 8 || w.rows == 2) f(one, two, few);
        else if constexpr (V == 4) f(one, four, few);
    } else {
        if (w.rows == 1) f(one, one, most);
        else if (V == 8 || w.rows == 2) f(one, two, most);
        else if constexpr (V == 4) {
            if (w.rows == 4) f(one, four, most);
            else f(one, eight, most);
        }
    }
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
    SO_REQUIRE(ranges_fit(c), "so_layer_norm_reserve: %u x %u is too large for one launch", F, B);
    return workspace(ctx, "so_layer_norm_reserve", std::max(c.cols_bytes, so_norm_grad_bytes(ctx, type, F, B)));
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
    SO_REQUIRE(!dMean || dMean != dRstd, "so_layer_norm: one array for both statistics");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const Cut c = cut_of(type, F, B);
    SO_REQUIRE(ranges_fit(c), "so_layer_norm: %u x %u is too large for one launch", F, B);
    if (const Whole w = whole_of(ctx, type, F, B); w.lanes) {
        const uint32_t tiles = so_ceil_div(B, w.lanes * (16u / (uint32_t)so_type_bytes(type))), per_xcd = so_ceil_div(tiles, 8);
        SO_REQUIRE(so_grid_fits((uint64_t)per_xcd * 8, w.threads), "so_layer_norm: %u x %u is too large for one launch", F, B);      // fewer lanes forced, more tiles
        hipError_t allowed = hipSuccess;
        so_for_type(type, [&](auto t) {
            using T = decltype(t);
            for_whole<so_elements<T>::V>(w, [&](auto lanes, auto rows, auto threads) {
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
            norm_parts_kernel<T, LC, kRows><<<(uint32_t)c.groups, kThreads, 0, ctx->stream>>>(F, B, c.tiles, (const T *)dX, x_stride, cols);
            const Parts p = few_parts(c, F, B, cols, [&](uint32_t workgroups, const Parts &from, float2 *to) {
                norm_group_kernel<LC * so_elements<T>::V><<<workgroups, kThreads, 0, ctx->stream>>>(F, B, from.count, from.rows, c.tiles, from.at, to);
            });
            norm_apply_kernel<T, LC, kRows><<<(uint32_t)c.groups, kThreads, 0, ctx->stream>>>(F, B, p.count, p.rows, c.tiles, (const T *)dX, x_stride, p.at, dGamma, dBeta, eps, (T *)dY,
                                                                                               y_stride, dMean, dRstd);
        });
    });
    SO_LAUNCH_CHECK();
    return SO_OK;
}
