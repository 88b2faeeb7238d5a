// Products with a microscaled 4-bit matrix (csrc/mxfp4.h): with a batch of columns on the scaled matrix cores, with one vector in fp32.
#include "mxfp4.h"

#include <type_traits>

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int J>
__device__ __forceinline__ f32x16 mx_mfma(so_u32x4 x, uint32_t sx, so_u32x4 w, uint32_t sw, f32x16 acc)
{
    const i32x8 a = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0}, b = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc, 4, 4, J, (int)sx, J, (int)sw);
}

// Y tile of MT x CT tiles of 32 x 32, WK waves that share the blocks between them, a unit of 8 each in turn; their sums meet in LDS.  X's columns are the instruction's
// first operand, so that a lane holds one row of W and four neighbouring columns of Y in each four registers.
template <class T, int MT, int CT, int WK, int ACT>
__global__ __launch_bounds__(64 * WK)
void mx_matmul_kernel(const so_u32x4 *__restrict__ Wc, const uint32_t *__restrict__ Ws, const so_u32x4 *__restrict__ Xc, const uint32_t *__restrict__ Xs, uint32_t m, uint32_t C,
                      uint32_t units, uint32_t wtiles, uint32_t xtiles, uint32_t mgroups, uint32_t per_xcd, uint32_t groups, const float *__restrict__ bias, T *__restrict__ Y, size_t ldy)
{
    constexpr int V = so_elements<T>::V, PITCH = CT * 32 + 4;
    extern __shared__ float lds[];                                   // [WK][MT * 32][PITCH]
    // Workgroups go round-robin to the 8 XCDs: each gets neighbouring tiles, rows of W first, whose columns of X then stay in one L2.
    const uint32_t id = (blockIdx.x % 8u) * per_xcd + blockIdx.x / 8u;
    if (id >= groups) return;
    const uint32_t mg = id % mgroups, cg = id / mgroups;
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u;
    const so_u32x4 *wc[MT], *xc[CT];
    const uint32_t *ws[MT], *xs[CT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const size_t t = min(mg * MT + i, wtiles - 1u);              // a tile that is not there: the last one again, not stored
        wc[i] = Wc + t * units * 256 + lane;
        ws[i] = Ws + t * units * 64 + lane;
    }
#pragma unroll
    for (int i = 0; i < CT; ++i) {
        const size_t t = min(cg * CT + i, xtiles - 1u);
        xc[i] = Xc + t * units * 256 + lane;
        xs[i] = Xs + t * units * 64 + lane;
    }
    f32x16 acc[MT][CT] = {};
    for (uint32_t u = wave; u < units; u += WK) {
        so_u32x4 w[MT][4], x[CT][4];
        uint32_t sw[MT], sx[CT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            sw[i] = ws[i][(size_t)u * 64];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i][j] = wc[i][(size_t)u * 256 + j * 64];
        }
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            sx[i] = xs[i][(size_t)u * 64];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = xc[i][(size_t)u * 256 + j * 64];
        }
        const auto step = [&](auto byte) {
            constexpr int J = decltype(byte)::value;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int k = 0; k < CT; ++k) acc[i][k] = mx_mfma<J>(x[k][J], sx[k], w[i][J], sw[i], acc[i][k]);
        };
        step(std::integral_constant<int, 0>());
        step(std::integral_constant<int, 1>());
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
    }
    float *mine = lds + (size_t)wave * MT * 32 * PITCH;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < CT; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 v = {acc[i][k][4 * q], acc[i][k][4 * q + 1], acc[i][k][4 * q + 2], acc[i][k][4 * q + 3]};
                *reinterpret_cast<f32x4 *>(mine + (i * 32 + lane % 32u) * PITCH + k * 32 + 8 * q + 4 * (lane / 32u)) = v;
            }
    __syncthreads();
    constexpr int GR = CT * 32 / V;                                  // groups of 16 bytes in a row of the tile
    for (uint32_t g = threadIdx.x; g < MT * 32 * GR; g += 64 * WK) {
        const uint32_t r = g / GR, c = g % GR * V;
        const uint64_t row = (uint64_t)mg * (MT * 32) + r, col = (uint64_t)cg * (CT * 32) + c;
        if (row >= m || col >= C) continue;
        const float b = bias ? bias[row] : 0.0f;
        float y[V];
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            f32x4 s = *reinterpret_cast<const f32x4 *>(lds + r * PITCH + c + e);
#pragma unroll
            for (int w = 1; w < WK; ++w) s += *reinterpret_cast<const f32x4 *>(lds + ((size_t)w * MT * 32 + r) * PITCH + c + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[e + i] = so_epilogue<ACT>(s[i] + b);
        }
        so_group_store(Y + row * ldy + col, (uint32_t)min((uint64_t)V, C - col), y);
    }
}

struct Workspace { size_t codes, scales; };
Workspace workspace_of(const so_mxfp4 *W, uint32_t C)
{
    const size_t tiles = so_ceil_div(C, kMxTile);
    return {tiles * W->blocks * kMxTile * sizeof(so_u32x4), tiles * (W->blocks / kMxUnit) * 64 * sizeof(uint32_t)};
}

so_status reserve(so_ctx *ctx, const char *who, const so_mxfp4 *W, uint32_t C)
{
    const Workspace s = workspace_of(W, C);
    SO_REQUIRE(!ctx->capturing || (ctx->mm_part && ctx->mm_part->bytes >= s.codes + s.scales),
               "%s: the context's workspace must grow, which cannot be done while a graph is being recorded (call so_mxfp4_matmul_reserve, or launch this shape "
               "once, before recording)", who);
    return so_matmul_workspace(ctx, s.codes + s.scales, 4);
}

template <class T, int MT, int CT, int WK, int ACT>
so_status launch(so_ctx *ctx, const so_mxfp4 *W, const so_u32x4 *codes, const uint32_t *scales, uint32_t C, const float *bias, T *Y, size_t ldy)
{
    const uint32_t xtiles = so_ceil_div(C, kMxTile), mgroups = so_ceil_div(W->tiles, MT);
    const uint64_t groups = (uint64_t)mgroups * so_ceil_div(xtiles, CT);
    SO_REQUIRE(groups < (1ull << 30), "so_mxfp4_matmul: %u x %u output is too large for one launch", W->m, C);
    const uint32_t per_xcd = so_ceil_div(groups, 8);
    constexpr uint32_t bytes = WK * MT * 32 * (CT * 32 + 4) * sizeof(float);
    const auto kernel = mx_matmul_kernel<T, MT, CT, WK, ACT>;
    if (bytes > 48 * 1024) SO_HIP(so_allow_big_lds(ctx, (const void *)kernel));
    kernel<<<per_xcd * 8, 64 * WK, bytes, ctx->stream>>>(W->d_codes, W->d_scales, codes, scales, W->m, C, W->blocks / kMxUnit, W->tiles, xtiles, mgroups, per_xcd, (uint32_t)groups,
                                                        bias, Y, ldy);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

constexpr int kVecThreads = 512, kVecWaves = kVecThreads / 64;
constexpr uint32_t kVecChunk = 8192;         // entries of x in LDS at a time

// y = W x + bias with x in fp32: a workgroup takes RT tiles of 32 rows, its waves a unit of 8 blocks each in turn.  A lane multiplies one block of a row with x from LDS, which
// the rows share, as whole numbers of halves, and the block's sum with its scale.
template <int RT>
__global__ __launch_bounds__(kVecThreads)
void mx_matvec_kernel(const so_u32x4 *__restrict__ Wc, const uint32_t *__restrict__ Ws, const float *__restrict__ x, uint32_t m, uint32_t n, uint32_t units, uint32_t tiles,
                      const float *__restrict__ bias, float *__restrict__ y)
{
    __shared__ f32x4 xs[kVecChunk / 4];
    __shared__ float part[kVecWaves][RT * 32];
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u;
    const so_u32x4 *wc[RT];
    const uint32_t *ws[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const size_t t = min(blockIdx.x * RT + i, tiles - 1u);
        wc[i] = Wc + t * units * 256 + lane;
        ws[i] = Ws + t * units * 64 + lane;
    }
    float acc[RT] = {};
    constexpr uint32_t CU = kVecChunk / 256;                         // units of a chunk
    for (uint32_t u0 = 0; u0 < units; u0 += CU) {
        const uint32_t here = min(units - u0, CU);
        if (u0) __syncthreads();
        for (uint32_t k = threadIdx.x; k < here * 256; k += kVecThreads) {
            const uint64_t at = (uint64_t)u0 * 256 + k;
            reinterpret_cast<float *>(xs)[k] = at < n ? x[at] : 0.0f;
        }
        __syncthreads();
        for (uint32_t u = wave; u < here; u += kVecWaves) {
            so_u32x4 w[RT][4];
            uint32_t sc[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                sc[i] = ws[i][(size_t)(u0 + u) * 64];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[i][j] = wc[i][(size_t)(u0 + u) * 256 + j * 64];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 *xp = xs + (u * 8 + 2 * j + lane / 32u) * 8;
                float sum[RT] = {};
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 a = xp[2 * g], b = xp[2 * g + 1];
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][j][g], 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][j][g], 1.0f, 1);
                        const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][j][g], 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][j][g], 1.0f, 3);
                        sum[i] = fmaf(p0[0], a[0], sum[i]);
                        sum[i] = fmaf(p0[1], a[1], sum[i]);
                        sum[i] = fmaf(p1[0], a[2], sum[i]);
                        sum[i] = fmaf(p1[1], a[3], sum[i]);
                        sum[i] = fmaf(p2[0], b[0], sum[i]);
                        sum[i] = fmaf(p2[1], b[1], sum[i]);
                        sum[i] = fmaf(p3[0], b[2], sum[i]);
                        sum[i] = fmaf(p3[1], b[3], sum[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const uint32_t s = sc[i] >> (8 * j) & 255u;
                    acc[i] = fmaf(sum[i], s == 255u ? __builtin_nanf("") : so_mx_power(s), acc[i]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i]), __float_as_uint(acc[i]), false, false);
        const float s = __uint_as_float(h[0]) + __uint_as_float(h[1]);
        if (lane < 32u) part[wave][i * 32 + lane] = s;
    }
    __syncthreads();
    const uint64_t row = (uint64_t)blockIdx.x * (RT * 32) + threadIdx.x;
    if (threadIdx.x < RT * 32 && row < m) {
        float s = part[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < kVecWaves; ++w) s += part[w][threadIdx.x];
        y[row] = bias ? s + bias[row] : s;
    }
}

} // namespace

extern "C" so_status so_mxfp4_matmul_reserve(so_ctx *ctx, const so_mxfp4 *W, uint32_t C)
{
    SO_REQUIRE(ctx != nullptr && W != nullptr, "so_mxfp4_matmul_reserve: null handle");
    SO_REQUIRE(!ctx->capturing, "so_mxfp4_matmul_reserve: a graph is being recorded");
    if (C == 0) return SO_OK;
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    return reserve(ctx, "so_mxfp4_matmul_reserve", W, C);
}

extern "C" so_status so_mxfp4_matmul(so_ctx *ctx, const so_mxfp4 *W, int type, const void *dX, size_t x_stride, uint32_t C, const float *dBias, void *dY, size_t y_stride, int act)
{
    SO_REQUIRE(ctx != nullptr && W != nullptr, "so_mxfp4_matmul: null handle");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_mxfp4_matmul: unknown element type %d", type);
    SO_REQUIRE(act >= SO_ACT_NONE && act <= SO_ACT_TANH, "so_mxfp4_matmul: unknown activation %d", act);
    if (C == 0) return SO_OK;
    SO_REQUIRE(dX && dY && dX != dY, "so_mxfp4_matmul: null or aliased tensor");
    SO_REQUIRE(x_stride >= C && y_stride >= C, "so_mxfp4_matmul: a stride is shorter than a row");
    SO_REQUIRE((uint64_t)W->blocks * C < (1ull << 38), "so_mxfp4_matmul: %u x %u input is too large for one launch", W->n, C);
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    if (const so_status s = reserve(ctx, "so_mxfp4_matmul", W, C); s != SO_OK) return s;
    so_u32x4 *codes = (so_u32x4 *)ctx->mm_part->p;
    uint32_t *scales = (uint32_t *)((char *)codes + workspace_of(W, C).codes);
    if (const so_status s = so_mx_quantize_columns(ctx, type, dX, x_stride, W->n, C, codes, scales); s != SO_OK) return s;
    const bool large = (uint64_t)so_ceil_div(W->tiles, 2) * so_ceil_div(C, 64) >= (uint64_t)ctx->compute_units;
    so_status status = SO_OK;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        const auto with = [&](auto a) {
            constexpr int ACT = decltype(a)::value;
            status = large ? launch<T, 2, 2, 4, ACT>(ctx, W, codes, scales, C, dBias, (T *)dY, y_stride) : launch<T, 1, 1, 8, ACT>(ctx, W, codes, scales, C, dBias, (T *)dY, y_stride);
        };
        if (act == SO_ACT_RELU) with(std::integral_constant<int, SO_ACT_RELU>());
        else if (act == SO_ACT_SIGMOID) with(std::integral_constant<int, SO_ACT_SIGMOID>());
        else if (act == SO_ACT_TANH) with(std::integral_constant<int, SO_ACT_TANH>());
        else with(std::integral_constant<int, SO_ACT_NONE>());
    });
    return status;
}

extern "C" so_status so_mxfp4_matvec(so_ctx *ctx, const so_mxfp4 *W, const float *dx, const float *dBias, float *dy)
{
    SO_REQUIRE(ctx != nullptr && W != nullptr, "so_mxfp4_matvec: null handle");
    SO_REQUIRE(dx && dy && dx != dy, "so_mxfp4_matvec: null or aliased vector");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const uint32_t units = W->blocks / kMxUnit;
    if (W->tiles >= 2 * (uint32_t)ctx->compute_units)
        mx_matvec_kernel<2><<<so_ceil_div(W->tiles, 2), kVecThreads, 0, ctx->stream>>>(W->d_codes, W->d_scales, dx, W->m, W->n, units, W->tiles, dBias, dy);
    else
        mx_matvec_kernel<1><<<W->tiles, kVecThreads, 0, ctx->stream>>>(W->d_codes, W->d_scales, dx, W->m, W->n, units, W->tiles, dBias, dy);
    SO_LAUNCH_CHECK();
    return SO_OK;
}
