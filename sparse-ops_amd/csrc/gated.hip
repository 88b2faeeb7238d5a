// The gated feed-forward block: both projections, the activation and the product, and their gradients.
#include "gate.h"

namespace {

constexpr int kTile = 64, kDeep = 16, kThreads = 256;

// One operand of a product: entry (i, k) at p[i * ld + k], or at p[k * ld + i] where it lies across the contraction.
template <class T> struct Operand { const T *p; size_t ld; };

// acc[a][b] += sum over k of A(row 4 ty + a, k) B(column 4 tx + b, k), from tiles of 64 x 16 of both in LDS.
template <class T, bool AX, bool BX>
__device__ void add_product(float (&acc)[4][4], Operand<T> A, Operand<T> B, uint64_t i0, uint64_t rows, uint64_t j0, uint64_t cols, uint32_t K, float (*a)[kTile + 1], float (*b)[kTile + 1])
{
    const uint32_t ty = threadIdx.x / 16u, tx = threadIdx.x % 16u;
    const auto bring = [&](auto across, const Operand<T> &M, uint64_t at, uint64_t end, uint32_t k0, float (*to)[kTile + 1]) {
        for (uint32_t e = threadIdx.x; e < kTile * kDeep; e += kThreads) {
            const uint32_t i = decltype(across)::value ? e % kTile : e / kDeep, k = decltype(across)::value ? e / kTile : e % kDeep;
            float v = 0.0f;
            if (at + i < end && (uint64_t)k0 + k < K) v = (float)(decltype(across)::value ? M.p[((size_t)k0 + k) * M.ld + at + i] : M.p[(size_t)(at + i) * M.ld + k0 + k]);
            to[k][i] = v;
        }
    };
    for (uint32_t k0 = 0; k0 < K; k0 += kDeep) {
        __syncthreads();
        bring(std::integral_constant<bool, AX>(), A, i0, rows, k0, a);
        bring(std::integral_constant<bool, BX>(), B, j0, cols, k0, b);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[r][c] = fmaf(a[k][4 * ty + r], b[k][4 * tx + c], acc[r][c]);
    }
}

template <class T> struct Forward {
    const T *Wg, *Wu, *X, *G0, *U0;
    T *H, *G, *U;
    size_t ldw, ldx, ld0, ldh, ldg;
    uint32_t m, n, B;
    int act;
};

template <class T>
__global__ __launch_bounds__(kThreads)
void gated_kernel(Forward<T> f)
{
    __shared__ float a[kDeep][kTile + 1], b[kDeep][kTile + 1];
    const uint32_t across = (f.B + kTile - 1u) / kTile;
    const uint64_t i0 = (uint64_t)(blockIdx.x / across) * kTile, j0 = (uint64_t)(blockIdx.x % across) * kTile;
    float g[4][4] = {}, u[4][4] = {};
    add_product<T, false, true>(g, {f.Wg, f.ldw}, {f.X, f.ldx}, i0, f.m, j0, f.B, f.n, a, b);
    add_product<T, false, true>(u, {f.Wu, f.ldw}, {f.X, f.ldx}, i0, f.m, j0, f.B, f.n, a, b);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint64_t row = i0 + threadIdx.x / 16u * 4u + r, col = j0 + threadIdx.x % 16u * 4u + c;
            if (row >= f.m || col >= f.B) continue;
            const float gs = g[r][c] + (f.G0 ? (float)f.G0[row * f.ld0 + col] : 0.0f), us = u[r][c] + (f.U0 ? (float)f.U0[row * f.ld0 + col] : 0.0f);
            f.H[row * f.ldh + col] = (T)(so_gate::value(f.act, gs) * us);
            if (f.G) f.G[row * f.ldg + col] = (T)gs;
            if (f.U) f.U[row * f.ldg + col] = (T)us;
        }
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

// Y = A1 B1 (+ A2 B2).
template <class T, bool AX, bool BX>
__global__ __launch_bounds__(kThreads)
void product_kernel(Operand<T> A1, Operand<T> B1, Operand<T> A2, Operand<T> B2, uint32_t rows, uint32_t cols, uint32_t K, T *Y, size_t ldy)
{
    __shared__ float a[kDeep][kTile + 1], b[kDeep][kTile + 1];
    const uint32_t across = (cols + kTile - 1u) / kTile;
    const uint64_t i0 = (uint64_t)(blockIdx.x / across) * kTile, j0 = (uint64_t)(blockIdx.x % across) * kTile;
    float acc[4][4] = {};
    add_product<T, AX, BX>(acc, A1, B1, i0, rows, j0, cols, K, a, b);
    if (A2.p) add_product<T, AX, BX>(acc, A2, B2, i0, rows, j0, cols, K, a, b);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint64_t row = i0 + threadIdx.x / 16u * 4u + r, col = j0 + threadIdx.x % 16u * 4u + c;
            if (row < rows && col < cols) Y[row * ldy + col] = (T)acc[r][c];
        }
}

uint64_t tiles(uint32_t rows, uint32_t cols) { return (uint64_t)so_ceil_div(rows, kTile) * so_ceil_div(cols, kTile); }

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
    SO_REQUIRE(so_grid_fits(tiles(m, B), kThreads), "so_gated: %u x %u is too large for one launch", m, B);
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        gated_kernel<T><<<(uint32_t)tiles(m, B), kThreads, 0, ctx->stream>>>({(const T *)dWg, (const T *)dWu, (const T *)dX, (const T *)dG0, (const T *)dU0, (T *)dH, (T *)dG, (T *)dU, w_stride,
                                                                             x_stride, g0_stride, h_stride, g_stride, m, n, B, act});
    });
    SO_LAUNCH_CHECK();
    return SO_OK;
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
    SO_REQUIRE((uint64_t)m * B < (1ull << 32) - kThreads && so_grid_fits(tiles(n, B), kThreads) && so_grid_fits(tiles(m, n), kThreads), "so_gated_grad: %u x %u x %u is too large for one launch", m, n, B);
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
            product_kernel<T, true, true><<<(uint32_t)tiles(n, B), kThreads, 0, ctx->stream>>>({(const T *)dWg, w_stride}, {g, ldg}, {(const T *)dWu, w_stride}, {u, ldu}, n, B, m, (T *)dDx, dx_stride);
        if (dDwg && m) product_kernel<T, false, false><<<(uint32_t)tiles(m, n), kThreads, 0, ctx->stream>>>({g, ldg}, {(const T *)dX, x_stride}, {nullptr, 0}, {nullptr, 0}, m, n, B, (T *)dDwg, dw_stride);
        if (dDwu && m) product_kernel<T, false, false><<<(uint32_t)tiles(m, n), kThreads, 0, ctx->stream>>>({u, ldu}, {(const T *)dX, x_stride}, {nullptr, 0}, {nullptr, 0}, m, n, B, (T *)dDwu, dw_stride);
        if ((dDg && g != (T *)dDg) || (dDu && u != (T *)dDu)) {      // one of the two asked for
            gated_slopes_kernel<T><<<(uint32_t)slopes, kThreads, 0, ctx->stream>>>(m, B, act, (const T *)dG, (const T *)dU, g_stride, (const T *)dDh, dh_stride, (T *)dDg, (T *)dDu, dg_stride);
        }
    });
    (void)e;
    if (status != SO_OK) return status;
    SO_LAUNCH_CHECK();
    return SO_OK;
}
