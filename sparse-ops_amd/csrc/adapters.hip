// Low-rank adapters of many requests: Y = base + scale_a B_a (A_a X), the adapter a of every column its own.
#include "elements.h"
#include "so_internal.h"

namespace {

constexpr uint32_t kThreads = 256, kMostRank = 256;

// T [rank x C] = scale_a A_a X, in fp32: a workgroup takes one entry of rank for 64 columns, its waves a quarter of the features each.
template <class T>
__global__ __launch_bounds__(kThreads)
void adapters_in_kernel(uint32_t n, uint32_t C, uint32_t count, uint32_t rank, const T *A, const float *scale, const int32_t *which, const T *X, size_t ldx, float *low)
{
    __shared__ float sums[4][64];
    const uint32_t r = blockIdx.x % rank, lane = threadIdx.x % 64u, wave = threadIdx.x / 64u;
    const uint64_t c = (uint64_t)(blockIdx.x / rank) * 64u + lane;
    const int32_t a = c < C ? which[c] : -1;
    const bool has = a >= 0 && (uint32_t)a < count;
    float s = 0.0f;
    if (has)
        for (uint32_t k = wave; k < n; k += 4) s = fmaf((float)A[((size_t)a * rank + r) * n + k], (float)X[(size_t)k * ldx + c], s);
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && has) low[(size_t)r * C + c] = (sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane]) * (scale ? scale[a] : 1.0f);
}

template <class T>
__global__ __launch_bounds__(kThreads)
void adapters_out_kernel(uint32_t m, uint32_t C, uint32_t count, uint32_t rank, const T *B, const int32_t *which, const float *low, const T *base, size_t ldb, T *Y, size_t ldy)
{
    const uint64_t at = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    if (at >= (uint64_t)m * C) return;
    const uint64_t row = at / C, c = at % C;
    const int32_t a = which[c];
    float s = 0.0f;
    if (a >= 0 && (uint32_t)a < count)
        for (uint32_t r = 0; r < rank; ++r) s = fmaf((float)B[((size_t)a * m + row) * rank + r], low[(size_t)r * C + c], s);
    Y[row * ldy + c] = (T)((base ? (float)base[row * ldb + c] : 0.0f) + s);
}

so_status workspace(so_ctx *ctx, const char *who, size_t bytes)
{
    SO_REQUIRE(!ctx->capturing || (ctx->mm_part && ctx->mm_part->bytes >= bytes),
               "%s: the context's workspace must grow, which cannot be done while a graph is being recorded (call so_adapters_reserve, or launch this shape once, before recording)", who);
    return so_matmul_workspace(ctx, bytes, 4);
}

size_t low_bytes(uint32_t C, uint32_t rank) { return (size_t)C * rank * sizeof(float); }

} // namespace

extern "C" so_status so_adapters_reserve(so_ctx *ctx, int type, uint32_t m, uint32_t n, uint32_t C, uint32_t rank)
{
    SO_REQUIRE(ctx != nullptr, "so_adapters_reserve: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_adapters_reserve: unknown element type %d", type);
    SO_REQUIRE(rank >= 1 && rank <= kMostRank, "so_adapters_reserve: rank %u is not 1 .. %u", rank, kMostRank);
    SO_REQUIRE(!ctx->capturing, "so_adapters_reserve: a graph is being recorded");
    if (m == 0 || C == 0) return SO_OK;
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    return workspace(ctx, "so_adapters_reserve", low_bytes(C, rank));
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
    SO_REQUIRE(so_grid_fits((uint64_t)so_ceil_div(C, 64) * rank, kThreads) && (uint64_t)m * C < (1ull << 32) - kThreads, "so_adapters: %u x %u is too large for one launch", m, C);
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    if (const so_status s = workspace(ctx, "so_adapters", low_bytes(C, rank)); s != SO_OK) return s;
    float *low = (float *)ctx->mm_part->p;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        adapters_in_kernel<T><<<so_ceil_div(C, 64) * rank, kThreads, 0, ctx->stream>>>(n, C, count, rank, (const T *)dA, dScale, dWhich, (const T *)dX, x_stride, low);
        adapters_out_kernel<T><<<so_ceil_div((uint64_t)m * C, kThreads), kThreads, 0, ctx->stream>>>(m, C, count, rank, (const T *)dB, dWhich, low, (const T *)dBase, base_stride, (T *)dY, y_stride);
    });
    SO_LAUNCH_CHECK();
    return SO_OK;
}
