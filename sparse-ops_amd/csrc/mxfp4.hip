// Microscaled 4-bit floating point (csrc/mxfp4.h): quantisation and its way back on caller-owned arrays, the weights' handle, and the quantisation of a product's activations.
#include "lane_moves.h"
#include "mxfp4.h"

#include <new>
#include <type_traits>

namespace {

constexpr int kBlock = 256;

// Row-major to codes and scales.  A lane takes 16 bytes of a row, a block is 8 lanes of fp32 or 4 of a 16-bit type; a block that the row ends in is filled with zeros.
// Bound by the memory: 8192 x 8192 bf16, 170 MB, 39 us, and 27 us back, together 5.2 TB/s where a copy reaches 6.35
// (the first of them also writes back what is still in the caches).  Four groups a lane, asked for at once, 42 us; a short division for the row and half the instructions 39.
template <class T>
__global__ __launch_bounds__(kBlock)
void mx_quantize_kernel(const T *__restrict__ X, size_t ldx, uint32_t cols, uint32_t groups, uint64_t total, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales)
{
    constexpr int V = so_elements<T>::V, L = 32 / V;
    for (uint64_t u = (uint64_t)blockIdx.x * kBlock + threadIdx.x; u < total; u += (uint64_t)gridDim.x * kBlock) {
        const uint64_t row = u / groups;
        const uint32_t g = (uint32_t)(u - row * groups), c = g * V;
        typename so_elements<T>::plain x = {};
        if (c < cols) x = so_group_load(X + row * ldx + c, cols - c);
        float f[V];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            f[e] = (float)x[e];
            top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
        }
        top = so_lanes::reduce<L>(top, so_lanes::Max());          // groups and total are multiples of L: all lanes of a block are here
        const uint32_t s = so_mx_scale(top);
        const float scale = so_mx_power(s);
        if constexpr (V == 4) {
            const float v[8] = {f[0], f[1], f[2], f[3], 0.0f, 0.0f, 0.0f, 0.0f};
            reinterpret_cast<uint16_t *>(codes)[u] = s == 255u ? 0 : (uint16_t)so_mx_codes(v, scale);
        } else {
            reinterpret_cast<uint32_t *>(codes)[u] = s == 255u ? 0 : so_mx_codes(f, scale);
        }
        if (u % L == 0) scales[u / L] = (uint8_t)s;
    }
}

// And back: 8192 x 8192 bf16 27 us, the memory.
template <class T>
__global__ __launch_bounds__(kBlock)
void mx_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, uint32_t cols, uint32_t groups, uint64_t total, T *__restrict__ Y, size_t ldy)
{
    constexpr int V = so_elements<T>::V, L = 32 / V;
    for (uint64_t u = (uint64_t)blockIdx.x * kBlock + threadIdx.x; u < total; u += (uint64_t)gridDim.x * kBlock) {
        const uint64_t row = u / groups;
        const uint32_t g = (uint32_t)(u - row * groups), c = g * V;
        const uint32_t s = scales[u / L];
        const uint32_t w = V == 4 ? reinterpret_cast<const uint16_t *>(codes)[u] : reinterpret_cast<const uint32_t *>(codes)[u];
        const float scale = so_mx_power(s);
        float f[V];
        const auto pair = [&](auto byte) {
            constexpr int I = decltype(byte)::value;
            const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, I);
            f[2 * I] = s == 255u ? __builtin_nanf("") : p[0];
            f[2 * I + 1] = s == 255u ? __builtin_nanf("") : p[1];
        };
        pair(std::integral_constant<int, 0>());
        pair(std::integral_constant<int, 1>());
        if constexpr (V == 8) {
            pair(std::integral_constant<int, 2>());
            pair(std::integral_constant<int, 3>());
        }
        if (c < cols) so_group_store(Y + row * ldy + c, cols - c, f);
    }
}

// Row-major codes and scales into tiles, once for a matrix; a thread takes 16 bytes of the result (16384 x 16384 61 us: the rows' 16 bytes a cache line each come through the L2 again).
__global__ __launch_bounds__(kBlock)
void mx_tile_kernel(const so_u32x4 *__restrict__ src, const uint8_t *__restrict__ src_scales, uint32_t m, uint32_t real, uint32_t units, uint64_t total, so_u32x4 *__restrict__ codes,
                    uint8_t *__restrict__ scales)
{
    const uint64_t at = (uint64_t)blockIdx.x * kBlock + threadIdx.x;           // [tile][unit][operand][lane]
    if (at >= total) return;
    const uint32_t lane = (uint32_t)(at % 64u), operand = (uint32_t)(at / 64u % 4u);
    const uint64_t tu = at / 256u, tile = tu / units;
    const uint32_t b = (uint32_t)(tu - tile * units) * kMxUnit + operand / 2u * 4u + lane / 16u;
    const uint64_t row = tile * kMxTile + operand % 2u * 16u + lane % 16u;
    const bool in = row < m && b < real;
    so_u32x4 v = {0u, 0u, 0u, 0u};
    if (in) v = src[row * real + b];
    codes[at] = v;
    scales[so_mx_scale_at(row, b, units)] = in ? src_scales[row * real + b] : kMxZero;
}

// The word of the lane whose number differs in bit 3, 4 or 5, joined with this one's by max.
__device__ __forceinline__ uint32_t max_over_rows(uint32_t v)
{
    v = max(v, so_lanes::word_across<8>(v));
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(b[0], b[1]);
}

// X [n x C] into tiles of columns.  A wave takes one block of 32 rows and 8 lanes of columns, 128 bytes a row: a lane 4 rows of 16 bytes, the largest magnitude of a column
// meets across its 8 lanes.  (One lane a column with its 32 rows, four blocks one after the other, left most of the chip idle: 2777 x 101 fp16 38.5 us.)
// Bound by the memory and the launch: 8192 x 2048 bf16, 42 MB, 12 us; 14 us with the workgroups of one column after the other.
template <class T>
__global__ __launch_bounds__(kBlock)
void mx_columns_kernel(const T *__restrict__ X, size_t ldx, uint32_t n, uint32_t C, uint32_t units, uint32_t across, so_u32x4 *__restrict__ codes, uint8_t *__restrict__ scales)
{
    constexpr int V = so_elements<T>::V;
    const uint32_t quad = blockIdx.x / across, group = blockIdx.x - quad * across, b = quad * 4u + threadIdx.x / 64u;     // as X lies in memory
    const uint32_t lane = threadIdx.x % 64u, r = lane / 8u;
    const uint64_t c = ((uint64_t)group * 8u + lane % 8u) * V, k0 = (uint64_t)b * 32u + r * 4u;
    const uint32_t left = c >= C ? 0u : (uint32_t)min((uint64_t)V, C - c);
    const T *p = X + k0 * ldx + c;
    const uint32_t wide = so_group_wide_rows<T>(left, n, ldx);     // what stands behind a row's end goes into columns that are not stored
    typename so_elements<T>::plain x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (k0 + i < n && left) x[i] = so_group_load(p + (size_t)i * ldx, left, k0 + i < wide);
        else x[i] = typename so_elements<T>::plain{};
    float f[4][V];
    uint32_t top[V] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            f[i][e] = (float)x[i][e];
            top[e] = max(top[e], __float_as_uint(f[i][e]) & 0x7fffffffu);
        }
    const bool padding = (uint64_t)b * 32u >= n;
    uint32_t w[V], own = 0;                                      // 4 codes of every column; the scale of column r % V
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const uint32_t s = so_mx_scale(max_over_rows(top[e]));
        const float scale = so_mx_power(s);
        w[e] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0][e], f[1][e], scale, 0);
        w[e] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[e], f[2][e], f[3][e], scale, 1);
        if (s == 255u) w[e] = 0;
        own = r % V == (uint32_t)e ? s : own;
    }
    // Columns against lanes, a bit of both at a time: in the end a lane has column r % V, its 32 codes (16-bit types) or the 16 of its half of the lanes.
    uint32_t two[V / 2];
#pragma unroll
    for (int p = 0; p < V / 2; ++p) {
        const uint32_t keep = r % 2u ? w[2 * p + 1] : w[2 * p], other = so_lanes::word_across<8>(r % 2u ? w[2 * p] : w[2 * p + 1]);
        two[p] = r % 2u ? other | keep << 16 : keep | other << 16;
    }
    const uint64_t col = c + r % V;
    const bool mine = r % V < left;
    const auto a0 = __builtin_amdgcn_permlane16_swap(two[0], two[1], false, false);
    if constexpr (V == 4) {
        if (mine) reinterpret_cast<uint2 *>(codes)[so_mx_code_at(col, b, units) * 2u + r / 4u] = make_uint2(a0[0], a0[1]);
        if (mine && r < 4u) scales[so_mx_scale_at(col, b, units)] = padding ? kMxZero : own;
    } else {
        const auto a1 = __builtin_amdgcn_permlane16_swap(two[2], two[3], false, false);
        const auto lo = __builtin_amdgcn_permlane32_swap(a0[0], a1[0], false, false), hi = __builtin_amdgcn_permlane32_swap(a0[1], a1[1], false, false);
        const so_u32x4 v = {lo[0], hi[0], lo[1], hi[1]};
        if (mine) {
            codes[so_mx_code_at(col, b, units)] = v;
            scales[so_mx_scale_at(col, b, units)] = padding ? kMxZero : own;
        }
    }
}

// Groups of 16 bytes, of a row (whole blocks) and of all.
struct Flat { uint64_t groups, total; };
template <class T>
Flat flat(uint32_t rows, uint32_t cols)
{
    const uint64_t groups = (uint64_t)so_ceil_div(cols, 32) * (32 / so_elements<T>::V);
    return {groups, groups * rows};
}

uint32_t grid_of(uint64_t total) { return (uint32_t)std::min<uint64_t>((total + kBlock - 1) / kBlock, 1u << 20); }

} // namespace

extern "C" so_status so_mxfp4_quantize(so_ctx *ctx, int type, const void *dX, size_t x_stride, uint32_t rows, uint32_t cols, uint8_t *dCodes, uint8_t *dScales)
{
    SO_REQUIRE(ctx != nullptr, "so_mxfp4_quantize: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_mxfp4_quantize: unknown element type %d", type);
    if (rows == 0 || cols == 0) return SO_OK;
    SO_REQUIRE(dX && dCodes && dScales, "so_mxfp4_quantize: null array");
    SO_REQUIRE(x_stride >= cols, "so_mxfp4_quantize: a stride is shorter than a row");
    SO_REQUIRE(((uintptr_t)dCodes & 15) == 0, "so_mxfp4_quantize: codes are not 16-byte aligned");
    SO_REQUIRE(cols <= 0xffffffe0u, "so_mxfp4_quantize: too many columns");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        const Flat f = flat<T>(rows, cols);
        mx_quantize_kernel<T><<<grid_of(f.total), kBlock, 0, ctx->stream>>>((const T *)dX, x_stride, cols, (uint32_t)f.groups, f.total, dCodes, dScales);
    });
    SO_LAUNCH_CHECK();
    return SO_OK;
}

extern "C" so_status so_mxfp4_dequantize(so_ctx *ctx, const uint8_t *dCodes, const uint8_t *dScales, uint32_t rows, uint32_t cols, int type, void *dY, size_t y_stride)
{
    SO_REQUIRE(ctx != nullptr, "so_mxfp4_dequantize: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_mxfp4_dequantize: unknown element type %d", type);
    if (rows == 0 || cols == 0) return SO_OK;
    SO_REQUIRE(dY && dCodes && dScales, "so_mxfp4_dequantize: null array");
    SO_REQUIRE(y_stride >= cols, "so_mxfp4_dequantize: a stride is shorter than a row");
    SO_REQUIRE(((uintptr_t)dCodes & 15) == 0, "so_mxfp4_dequantize: codes are not 16-byte aligned");
    SO_REQUIRE(cols <= 0xffffffe0u, "so_mxfp4_dequantize: too many columns");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        const Flat f = flat<T>(rows, cols);
        mx_dequantize_kernel<T><<<grid_of(f.total), kBlock, 0, ctx->stream>>>(dCodes, dScales, cols, (uint32_t)f.groups, f.total, (T *)dY, y_stride);
    });
    SO_LAUNCH_CHECK();
    return SO_OK;
}

extern "C" so_status so_mxfp4_create(so_ctx *ctx, const uint8_t *dCodes, const uint8_t *dScales, uint32_t m, uint32_t n, so_mxfp4 **out)
{
    SO_REQUIRE(ctx != nullptr, "so_mxfp4_create: ctx is null");
    SO_REQUIRE(out != nullptr, "so_mxfp4_create: out is null");
    *out = nullptr;
    SO_REQUIRE(m > 0 && n > 0, "so_mxfp4_create: an empty matrix");
    SO_REQUIRE(dCodes && dScales, "so_mxfp4_create: null array");
    SO_REQUIRE(((uintptr_t)dCodes & 15) == 0, "so_mxfp4_create: codes are not 16-byte aligned");
    SO_REQUIRE(n <= 0xffffff00u && m <= 0xffffffe0u, "so_mxfp4_create: %u x %u is too large", m, n);
    SO_REQUIRE(!ctx->capturing, "so_mxfp4_create: not allowed while a graph is being recorded");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    std::unique_ptr<so_mxfp4> W(new (std::nothrow) so_mxfp4());
    if (!W) { so_set_error("host allocation failed"); return SO_ERR_OOM; }
    W->m = m;
    W->n = n;
    W->blocks = so_mx_blocks(n);
    W->tiles = so_ceil_div(m, kMxTile);
    const uint64_t total = (uint64_t)W->tiles * W->blocks * kMxTile;                 // threads, and 16 bytes of codes each
    SO_REQUIRE(so_grid_fits(total / kBlock, kBlock), "so_mxfp4_create: %u x %u is too large for one launch", m, n);
    W->device = ctx->device;
    SO_HIP(hipMalloc(&W->d_blob, total * 17));
    W->d_codes = (so_u32x4 *)W->d_blob;
    W->d_scales = (uint32_t *)(W->d_codes + total);
    mx_tile_kernel<<<so_ceil_div(total, kBlock), kBlock, 0, ctx->stream>>>((const so_u32x4 *)dCodes, dScales, m, so_ceil_div(n, 32), W->blocks / kMxUnit, total, W->d_codes, (uint8_t *)W->d_scales);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);                      // from here on other contexts may use it
    if (e != hipSuccess) {
        (void)hipFree(W->d_blob);
        so_set_error("so_mxfp4_create: %s", hipGetErrorString(e));
        return SO_ERR_HIP;
    }
    *out = W.release();
    return SO_OK;
}

extern "C" so_status so_mxfp4_free(so_ctx *ctx, so_mxfp4 *W)
{
    if (!W) return SO_OK;
    SO_REQUIRE(!ctx || !ctx->capturing, "so_mxfp4_free: not allowed while a graph is being recorded");
    if (ctx && ctx->stream) (void)hipStreamSynchronize(ctx->stream);
    (void)hipFree(W->d_blob);
    delete W;
    return SO_OK;
}

extern "C" so_status so_mxfp4_dims(const so_mxfp4 *W, uint32_t *m, uint32_t *n)
{
    SO_REQUIRE(W != nullptr, "so_mxfp4_dims: handle is null");
    if (m) *m = W->m;
    if (n) *n = W->n;
    return SO_OK;
}

so_status so_mx_quantize_columns(so_ctx *ctx, int type, const void *dX, size_t x_stride, uint32_t n, uint32_t C, so_u32x4 *codes, uint32_t *scales)
{
    const uint32_t blocks = so_mx_blocks(n);
    so_status status = SO_OK;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        const uint32_t across = so_ceil_div(C, 8 * so_elements<T>::V);
        const uint64_t groups = (uint64_t)across * (blocks / 4);
        if (!so_grid_fits(groups, kBlock)) {
            so_set_error("so_mxfp4_matmul: %u x %u input is too large for one launch", n, C);
            status = SO_ERR_INVALID;
        } else if (codes) {
            mx_columns_kernel<T><<<(uint32_t)groups, kBlock, 0, ctx->stream>>>((const T *)dX, x_stride, n, C, blocks / kMxUnit, across, codes, (uint8_t *)scales);
        }
    });
    if (status != SO_OK) return status;
    SO_LAUNCH_CHECK();
    return SO_OK;
}
