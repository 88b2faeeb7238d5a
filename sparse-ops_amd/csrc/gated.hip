// The gated feed-forward block: both projections, the activation and the product, and their gradients.
#include "dense.h"
#include "gate.h"

namespace {

using so_dense::f32x4;
using so_dense::Grid;
using so_dense::Operand;

constexpr int kThreads = 256;

template <class T> struct Forward {
    const T *Wg, *Wu, *X, *G0, *U0;
    T *H, *G, *U;
    size_t ldw, ldx, ld0, ldh, ldg;
    uint32_t m, n, B;
    int act;
};

// The results of V neighbouring columns of a row from its two sums.
template <class T>
__device__ __forceinline__ void finish(const Forward<T> &f, uint64_t row, uint64_t col, float (&g)[so_elements<T>::V], float (&u)[so_elements<T>::V])
{
    constexpr int V = so_elements<T>::V;
    if (row >= f.m || col >= f.B) return;
    const uint32_t left = (uint32_t)min((uint64_t)V, f.B - col);
    if (f.G0) {
        const auto v = so_group_load(f.G0 + row * f.ld0 + col, left);
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] += (float)v[e];
    }
    if (f.U0) {
        const auto v = so_group_load(f.U0 + row * f.ld0 + col, left);
#pragma unroll
        for (int e = 0; e < V; ++e) u[e] += (float)v[e];
    }
    if (f.G) so_group_store(f.G + row * f.ldg + col, left, g);
    if (f.U) so_group_store(f.U + row * f.ldg + col, left, u);
    so_gate::apply<V>(f.act, g, u);
    so_group_store(f.H + row * f.ldh + col, left, g);
}

// A tile of both projections: half of its rows are the gate's, half the other's, so that every wave holds both sums of its part of H.
template <class T, class TILE, bool DIRECT>
__global__ __launch_bounds__(TILE::THREADS)
void gated_kernel(Forward<T> f, Grid grid)
{
    extern __shared__ char stage[];
    const auto spot = so_dense::spot_of(grid);
    if (spot.none) return;
    so_dense::Loop<T, TILE, false, true, true> loop;
    const uint64_t i0 = (uint64_t)spot.m * (TILE::ROWS / 2), j0 = (uint64_t)spot.c * TILE::COLS;
    loop.template add<DIRECT>(stage, {{f.Wg, f.ldw, f.m, f.n}, {f.Wu, f.ldw, f.m, f.n}}, i0, {f.X, f.ldx, f.B, f.n}, j0);
    __syncthreads();
    const uint64_t row0 = i0 + threadIdx.x / 64u / TILE::WC * (TILE::RT / 2 * 16);
    loop.template out<2>(stage, [&](int i, uint32_t r, uint32_t c, float (&v)[2][so_elements<T>::V]) { finish(f, row0 + i * 16 + r, j0 + c, v[0], v[1]); });
}

template <class T>
__global__ __launch_bounds__(kThreads)
void gated_slopes_kernel(uint32_t m, uint32_t B, int act, const T *G, const T *U, size_t ldg, const T *dH, size_t ldh, T *dG, T *dU, size_t ldd)
{
    const uint64_t at = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    if (at >= (uint64_t)m * B) return;
    const uint64_t row = at / B, col = at % B;
    const auto s = so_gate::value_and_slope(act, (float)G[row * ldg + col]);
    const float u = (float)U[row * ldg + col], h = (float)dH[row * ldh + col];
    if (dG) dG[row * ldd + col] = (T)(h * u * s.slope);
    if (dU) dU[row * ldd + col] = (T)(h * s.value);
}

// Y = A[0] B[0] + A[1] B[1], or either's rows one after the other where the result has two parts (Y2 is not null).
template <class T> struct Product {
    Operand<T> A[2], B[2];
    T *Y, *Y2;
    size_t ldy;
    uint32_t rows, cols, terms;      // of one part; products to add
};

template <class T, class TILE, bool AX, bool BX, bool DIRECT>
__global__ __launch_bounds__(TILE::THREADS)
void product_kernel(Product<T> p, Grid grid)
{
    extern __shared__ char stage[];
    const auto spot = so_dense::spot_of(grid);
    if (spot.none) return;
    const uint32_t each = (p.rows + TILE::ROWS - 1u) / TILE::ROWS, second = spot.m >= each ? 1u : 0u;
    so_dense::Loop<T, TILE, AX, BX, false> loop;
    const uint64_t i0 = (uint64_t)(spot.m - second * each) * TILE::ROWS, j0 = (uint64_t)spot.c * TILE::COLS;
    for (uint32_t t = 0; t < p.terms; ++t) loop.template add<DIRECT>(stage, {p.A[second + t]}, i0, p.B[second + t], j0);
    __syncthreads();
    T *Y = second ? p.Y2 : p.Y;
    const uint64_t row0 = i0 + threadIdx.x / 64u / TILE::WC * (TILE::RT * 16);
    loop.template out<1>(stage, [&](int i, uint32_t r, uint32_t c, float (&v)[1][so_elements<T>::V]) {
        const uint64_t row = row0 + i * 16 + r, col = j0 + c;
        if (row < p.rows && col < p.cols) so_group_store(Y + row * p.ldy + col, (uint32_t)min((uint64_t)so_elements<T>::V, p.cols - col), v[0]);
    });
}

// Tiles, by rows and columns of the result (of both projections together in the forward pass).
typedef so_dense::Tile<8, 4, 2, 4, 64, 4> Large;        // 256 x 256
typedef so_dense::Tile<4, 4, 2, 2, 64, 4> Middle;       // 128 x 128
typedef so_dense::Tile<2, 2, 2, 2, 128, 4> Small;       // 64 x 64
typedef so_dense::Tile<2, 1, 2, 2, 128, 5> Narrow;      // 64 x 32

// f(a tile, whether operands go past the registers): the largest that gives every compute unit a workgroup.  fp32 has no use for the largest: its products take four times as long, and 128 x 128 feeds them.
template <class T, class F>
so_status for_tile(const so_ctx *ctx, uint64_t rows, uint64_t cols, bool direct, F &&f)
{
    const uint64_t cus = (uint64_t)ctx->compute_units;
    const auto tiles = [&](uint32_t r, uint32_t c) { return (uint64_t)so_ceil_div(rows, r) * so_ceil_div(cols, c); };
    const bool middle = cols > 64 && tiles(128, 128) >= cus;
    if (!direct) return middle ? f(Middle(), std::false_type()) : f(Small(), std::false_type());
    if constexpr (sizeof(T) == 2)
        if (cols > 128 && tiles(256, 256) >= cus) return f(Large(), std::true_type());
    if (middle) return f(Middle(), std::true_type());
    if (cols > 32) return f(Small(), std::true_type());
    return f(Narrow(), std::true_type());
}

template <class TILE, class Kernel, class Arg>
so_status launch_tiles(so_ctx *ctx, const char *who, Kernel kernel, const Arg &arg, uint64_t mgroups, uint64_t cgroups)
{
    SO_REQUIRE(so_grid_fits(mgroups * cgroups + 8, TILE::THREADS), "%s: the result is too large for one launch", who);
    const Grid g = so_dense::grid_of(mgroups, cgroups);
    SO_HIP(so_allow_big_lds(ctx, (const void *)kernel));
    kernel<<<g.groups(), TILE::THREADS, TILE::lds, ctx->stream>>>(arg, g);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

template <class T>
so_status forward(so_ctx *ctx, const Forward<T> &f)
{
    const Operand<T> g = {f.Wg, f.ldw, f.m, f.n}, u = {f.Wu, f.ldw, f.m, f.n}, x = {f.X, f.ldx, f.B, f.n};
    return for_tile<T>(ctx, 2 * (uint64_t)f.m, f.B, g.direct() && u.direct() && x.direct(), [&](auto t, auto direct) {
        typedef decltype(t) TILE;
        return launch_tiles<TILE>(ctx, "so_gated", gated_kernel<T, TILE, decltype(direct)::value>, f, so_ceil_div(f.m, TILE::ROWS / 2), so_ceil_div(f.B, TILE::COLS));
    });
}

template <class T, bool AX, bool BX>
so_status product(so_ctx *ctx, const Product<T> &p)
{
    const uint32_t parts = p.Y2 ? 2 : 1;
    bool direct = true;
    for (uint32_t i = 0; i < std::max(parts, p.terms); ++i) direct = direct && p.A[i].direct() && p.B[i].direct();
    return for_tile<T>(ctx, (uint64_t)parts * p.rows, p.cols, direct, [&](auto t, auto past) {
        typedef decltype(t) TILE;
        return launch_tiles<TILE>(ctx, "so_gated_grad", product_kernel<T, TILE, AX, BX, decltype(past)::value>, p, (uint64_t)parts * so_ceil_div(p.rows, TILE::ROWS), so_ceil_div(p.cols, TILE::COLS));
    });
}

size_t grad_bytes(int type, uint32_t m, uint32_t B) { return 2 * (size_t)m * B * so_type_bytes(type); }

so_status workspace(so_ctx *ctx, const char *who, size_t bytes)
{
    SO_REQUIRE(!ctx->capturing || (ctx->mm_part && ctx->mm_part->bytes >= bytes),
               "%s: the context's workspace must grow, which cannot be done while a graph is being recorded (call so_gated_reserve, or launch this shape once, before recording)", who);
    return so_matmul_workspace(ctx, bytes, 4);
}

} // namespace

extern "C" so_status so_gated_reserve(so_ctx *ctx, int type, uint32_t m, uint32_t n, uint32_t B)
{
    SO_REQUIRE(ctx != nullptr, "so_gated_reserve: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_gated_reserve: unknown element type %d", type);
    SO_REQUIRE(!ctx->capturing, "so_gated_reserve: a graph is being recorded");
    if (m == 0 || B == 0) return SO_OK;
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    return workspace(ctx, "so_gated_reserve", grad_bytes(type, m, B));
}

extern "C" so_status so_gated(so_ctx *ctx, int type, uint32_t m, uint32_t n, uint32_t B, const void *dWg, const void *dWu, size_t w_stride, const void *dX, size_t x_stride, int act,
                              const void *dG0, const void *dU0, size_t g0_stride, void *dH, size_t h_stride, void *dG, void *dU, size_t g_stride)
{
    SO_REQUIRE(ctx != nullptr, "so_gated: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_gated: unknown element type %d", type);
    SO_REQUIRE(so_gate::known(act), "so_gated: unknown activation %d", act);
    if (m == 0 || B == 0) return SO_OK;
    SO_REQUIRE(n > 0, "so_gated: no input features");
    SO_REQUIRE(dWg && dWu && dX && dH, "so_gated: null tensor");
    SO_REQUIRE(w_stride >= n && x_stride >= B && h_stride >= B, "so_gated: a stride is shorter than a row");
    SO_REQUIRE(!(dG0 || dU0) || g0_stride >= B, "so_gated: a stride is shorter than a row");
    SO_REQUIRE(!(dG || dU) || g_stride >= B, "so_gated: a stride is shorter than a row");
    for (const void *result : {(const void *)dH, (const void *)dG, (const void *)dU})
        SO_REQUIRE(!result || (result != dWg && result != dWu && result != dX), "so_gated: a result is an input");
    SO_REQUIRE(dH != dG && dH != dU && (!dG || dG != dU), "so_gated: one array for two results");
    SO_REQUIRE(dH != dG0 && dH != dU0 && (!dG || dG != dU0) && (!dU || dU != dG0), "so_gated: a result is an input");
    SO_REQUIRE(!((dG && dG == dG0) || (dU && dU == dU0)) || g_stride == g0_stride, "so_gated: in place needs one stride");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    so_status status = SO_OK;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        status = forward<T>(ctx, {(const T *)dWg, (const T *)dWu, (const T *)dX, (const T *)dG0, (const T *)dU0, (T *)dH, (T *)dG, (T *)dU, w_stride, x_stride, g0_stride, h_stride, g_stride,
                                  m, n, B, act});
    });
    return status;
}

extern "C" so_status so_gated_grad(so_ctx *ctx, int type, uint32_t m, uint32_t n, uint32_t B, const void *dWg, const void *dWu, size_t w_stride, const void *dX, size_t x_stride, int act,
                                   const void *dG, const void *dU, size_t g_stride, const void *dDh, size_t dh_stride, void *dDx, size_t dx_stride, void *dDwg, void *dDwu,
                                   size_t dw_stride, void *dDg, void *dDu, size_t dg_stride)
{
    SO_REQUIRE(ctx != nullptr, "so_gated_grad: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_gated_grad: unknown element type %d", type);
    SO_REQUIRE(so_gate::known(act), "so_gated_grad: unknown activation %d", act);
    const bool weights = dDwg || dDwu;
    if (!dDx && !weights && !dDg && !dDu) return SO_OK;
    SO_REQUIRE(n > 0, "so_gated_grad: no input features");
    SO_REQUIRE(!weights || dw_stride >= n, "so_gated_grad: a stride is shorter than a row");
    SO_REQUIRE(!dDx || dx_stride >= B, "so_gated_grad: a stride is shorter than a row");
    const size_t e = so_type_bytes(type);
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const uint64_t slopes = so_ceil_div((uint64_t)m * B, kThreads);
    SO_REQUIRE((uint64_t)m * B < (1ull << 32) - kThreads, "so_gated_grad: %u x %u is too large for one launch", m, B);
    if (m > 0 && B > 0) {
        SO_REQUIRE(dG && dU && dDh, "so_gated_grad: null tensor");
        SO_REQUIRE(!dDx || (dWg && dWu), "so_gated_grad: null weights");
        SO_REQUIRE(!weights || dX, "so_gated_grad: null input");
        SO_REQUIRE(g_stride >= B && dh_stride >= B && (!dDx || w_stride >= n) && (!weights || x_stride >= B), "so_gated_grad: a stride is shorter than a row");
        SO_REQUIRE(!(dDg || dDu) || dg_stride >= B, "so_gated_grad: a stride is shorter than a row");
    }
    void *results[] = {dDx, dDwg, dDwu, dDg, dDu};
    for (int i = 0; i < 5; ++i) {
        if (!results[i]) continue;
        for (int j = 0; j < i; ++j) SO_REQUIRE(results[i] != results[j], "so_gated_grad: one array for two results");
        SO_REQUIRE(results[i] != dWg && results[i] != dWu && results[i] != dX, "so_gated_grad: a result is an input");
        for (const void *in : {dG, dU, dDh})
            SO_REQUIRE(results[i] != in || (i >= 3 && dg_stride == (in == dDh ? dh_stride : g_stride)), "so_gated_grad: a result is an input, or in place with two strides");
    }
    so_status status = SO_OK;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        T *g = (T *)dDg, *u = (T *)dDu;
        size_t ldg = dg_stride, ldu = dg_stride;
        if ((!g || !u) && (dDx || weights) && m && B) {
            status = workspace(ctx, "so_gated_grad", grad_bytes(type, m, B));
            if (status != SO_OK) return;
            T *w = (T *)ctx->mm_part->p;
            if (!g || !u) g = w, u = w + (size_t)m * B, ldg = ldu = B;
        }
        if (m && B) gated_slopes_kernel<T><<<(uint32_t)slopes, kThreads, 0, ctx->stream>>>(m, B, act, (const T *)dG, (const T *)dU, g_stride, (const T *)dDh, dh_stride, g, u, ldg);
        if (dDx && B)
            status = product<T, true, true>(ctx, {{{(const T *)dWg, w_stride, n, m}, {(const T *)dWu, w_stride, n, m}}, {{g, ldg, B, m}, {u, ldu, B, m}}, (T *)dDx, nullptr, dx_stride, n, B, 2});
        const Operand<T> x = {(const T *)dX, x_stride, n, B}, dg = {g, ldg, m, B}, du = {u, ldu, m, B};
        if (status == SO_OK && m && dDwg && dDwu) status = product<T, false, false>(ctx, {{dg, du}, {x, x}, (T *)dDwg, (T *)dDwu, dw_stride, m, n, 1});
        else if (status == SO_OK && m && weights) status = product<T, false, false>(ctx, {{dDwg ? dg : du, du}, {x, x}, (T *)(dDwg ? dDwg : dDwu), nullptr, dw_stride, m, n, 1});
        if (status != SO_OK) return;
        if ((dDg && g != (T *)dDg) || (dDu && u != (T *)dDu)) {      // one of the two asked for
            gated_slopes_kernel<T><<<(uint32_t)slopes, kThreads, 0, ctx->stream>>>(m, B, act, (const T *)dG, (const T *)dU, g_stride, (const T *)dDh, dh_stride, (T *)dDg, (T *)dDu, dg_stride);
        }
    });
    (void)e;
    if (status != SO_OK) return status;
    SO_LAUNCH_CHECK();
    return SO_OK;
}
