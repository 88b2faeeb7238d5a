// Products with a microscaled 4-bit matrix (csrc/mxfp4.h): with a batch of columns on the scaled matrix cores, with one vector in fp32.
#include "mxfp4.h"

#include <type_traits>

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// 16 x 16 x 128 with both operands in 4 bits; X's columns are the first operand, so that a lane holds row l % 16 of W and the neighbouring columns 4 (l / 16) .. + 3 of Y.  On values as
// they come this instruction reaches 7.35 PFLOP/s, 32 x 32 x 64 6.6: the chip's power is what bounds both (zeros: 9.8 for the latter).
template <int JX, int JW>
__device__ __forceinline__ f32x4 mx_mfma(so_u32x4 x, uint32_t sx, so_u32x4 w, uint32_t sw, f32x4 acc)
{
    const i32x8 a = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0}, b = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, JX, (int)sx, JW, (int)sw);
}

// f(0), f(1), ... as compile-time numbers.
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(F &&f)
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>());
        each<N, I + 1>(f);
    }
}

// The activation of a sum, as so_epilogue but that a ReLU keeps NaN: a block that is not a number marks all results that it goes into.
template <int ACT>
__device__ __forceinline__ float mx_epilogue(float v)
{
    if constexpr (ACT == SO_ACT_RELU) return v <= 0.0f ? 0.0f : v;
    else return so_epilogue<ACT>(v);
}

// Which tile of the output a workgroup takes.  Workgroups go round-robin to the 8 XCDs; each XCD gets neighbouring tiles of a strip four tiles of columns wide, so that its L2 is
// asked for few rows of W and few columns of X.
struct MxTile { uint32_t m, c; bool none; };
__device__ __forceinline__ MxTile mx_tile_of(uint32_t mgroups, uint32_t cgroups, uint32_t per_xcd)
{
    const uint32_t id = (blockIdx.x % 8u) * per_xcd + blockIdx.x / 8u;
    if (id >= mgroups * cgroups) return {0, 0, true};
    const uint32_t strip = id / (4u * mgroups), wide = min(4u, cgroups - strip * 4u), in = id - strip * 4u * mgroups;
    return {in / wide, strip * 4u + in % wide, false};
}

// A tile of Y of 16 MH x 16 CH, WK waves that share the blocks between them, a unit of 8 each in turn, straight from memory to registers; their sums meet in LDS.
// Bound by the caches, which bring a workgroup (rows + columns) n / 2 bytes, and by loads that the products wait for: 4096 x 4096 x 256 fp32 on 64 x 64 8.4 us (17 MB from memory, 71 from the
// L2s and half as much again for units that are asked for twice), 3001 x 2777 x 101 fp16 on 32 x 32 5.1.
template <class T, int MH, int CH, int WK, int ACT>
__global__ __launch_bounds__(64 * WK)
void mx_matmul_kernel(const so_u32x4 *__restrict__ Wc, const uint32_t *__restrict__ Ws, const so_u32x4 *__restrict__ Xc, const uint32_t *__restrict__ Xs, uint32_t m, uint32_t C,
                      uint32_t units, uint32_t wtiles, uint32_t xtiles, uint32_t mgroups, uint32_t cgroups, uint32_t per_xcd, const float *__restrict__ bias, T *__restrict__ Y,
                      size_t ldy)
{
    constexpr int V = so_elements<T>::V, PITCH = CH * 16 + 4, MW = (MH + 1) / 2, CW = (CH + 1) / 2;
    static_assert((MH == 1 || MH % 2 == 0) && (CH == 1 || CH % 2 == 0), "half a tile of 32, or whole ones");
    extern __shared__ f32x4 sums[];                                  // [WK][MH * 16][PITCH / 4]
    const MxTile tile = mx_tile_of(mgroups, cgroups, per_xcd);
    if (tile.none) return;
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u;
    // half a tile: its operands begin 64 lanes further, and its scales are the upper half of the words
    const uint32_t mhalf = MH == 1 ? tile.m % 2u : 0u, chalf = CH == 1 ? tile.c % 2u : 0u;
    const so_u32x4 *wc[MW], *xc[CW];
    const uint32_t *ws[MW], *xs[CW];
#pragma unroll
    for (int i = 0; i < MW; ++i) {
        const size_t t = min(MH == 1 ? tile.m / 2u : tile.m * MW + i, wtiles - 1u);              // a tile that is not there: the last one again, not stored
        wc[i] = Wc + t * units * 256 + mhalf * 64u + lane;
        ws[i] = Ws + t * units * 64 + lane;
    }
#pragma unroll
    for (int i = 0; i < CW; ++i) {
        const size_t t = min(CH == 1 ? tile.c / 2u : tile.c * CW + i, xtiles - 1u);
        xc[i] = Xc + t * units * 256 + chalf * 64u + lane;
        xs[i] = Xs + t * units * 64 + lane;
    }
    struct Unit {
        so_u32x4 w[2][MH], x[2][CH];
        uint32_t sw[MW], sx[CW];
    };
    const auto load = [&](Unit &t, uint32_t u) {
#pragma unroll
        for (int i = 0; i < MW; ++i) t.sw[i] = ws[i][(size_t)u * 64] >> mhalf * 16u;
#pragma unroll
        for (int i = 0; i < CW; ++i) t.sx[i] = xs[i][(size_t)u * 64] >> chalf * 16u;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int i = 0; i < MH; ++i) t.w[q][i] = wc[i / 2][(size_t)u * 256 + q * 128 + i % 2 * 64];
#pragma unroll
            for (int i = 0; i < CH; ++i) t.x[q][i] = xc[i / 2][(size_t)u * 256 + q * 128 + i % 2 * 64];
        }
    };
    f32x4 acc[MH][CH] = {};
    const auto multiply = [&](const Unit &t) {
        each<2>([&](auto q) {
            each<CH>([&](auto k) {
                each<MH>([&](auto i) {
                    constexpr int Q = decltype(q)::value, K = decltype(k)::value, I = decltype(i)::value;
                    acc[I][K] = mx_mfma<K % 2 * 2 + Q, I % 2 * 2 + Q>(t.x[Q][K], t.sx[K / 2], t.w[Q][I], t.sw[I / 2], acc[I][K]);
                });
            });
        });
    };
    // Two units in registers; behind the last one that one again, for nothing (a third of the loads where a wave has two units).  As compiled, a unit's loads are asked for behind most of
    // the products of the one before it, not ahead of them, so that little of their way is hidden.
    const uint32_t turns = wave < units ? (units - wave + WK - 1u) / WK : 0u;
    if (turns) {
        const uint32_t last = wave + (turns - 1u) * WK;
        Unit a, b;
        load(a, wave);
        for (uint32_t t = 0; t + 1u < turns; t += 2u) {
            load(b, wave + (t + 1u) * WK);
            multiply(a);
            load(a, min(wave + (t + 2u) * WK, last));
            multiply(b);
        }
        if (turns % 2u) multiply(a);
    }
    f32x4 *mine = sums + wave * MH * 16 * (PITCH / 4);
#pragma unroll
    for (int i = 0; i < MH; ++i)
#pragma unroll
        for (int k = 0; k < CH; ++k) mine[(i * 16 + lane % 16u) * (PITCH / 4) + k * 4 + lane / 16u] = acc[i][k];
    __syncthreads();
    constexpr int GR = CH * 16 / V;                                  // groups of 16 bytes in a row of the tile
    for (uint32_t g = threadIdx.x; g < MH * 16 * GR; g += 64 * WK) {
        const uint32_t r = g / GR, c = g % GR * V;
        const uint64_t row = (uint64_t)tile.m * (MH * 16) + r, col = (uint64_t)tile.c * (CH * 16) + c;
        if (row >= m || col >= C) continue;
        const float add = bias ? bias[row] : 0.0f;
        float y[V];
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            f32x4 s = sums[r * (PITCH / 4) + (c + e) / 4];
#pragma unroll
            for (int w = 1; w < WK; ++w) s += sums[(w * MH * 16 + r) * (PITCH / 4) + (c + e) / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[e + i] = mx_epilogue<ACT>(s[i] + add);
        }
        so_group_store(Y + row * ldy + col, (uint32_t)min((uint64_t)V, C - col), y);
    }
}

// The same for large products: a tile of (16 MH WM) x (16 CH WC), its waves WM x WC, each MH x CH operands.  Half a unit (128 entries a row) of W and of X at a time goes to LDS as it
// lies in memory, in a ring of four, each wave bringing as many tiles of 32 rows as the others.
// Half a unit of the 256 x 256 tile is 1024 clocks of the matrix cores and as many of LDS, 770 of reading and 256 of filling; they overlap in part, at the clock that the chip's power leaves:
// 8192 x 8192 x 2048 bf16 62 us, the matrix cores busy 64% of it (4.4 PFLOP/s).  Without matrix instructions it is 38 us, without LDS 48; with waves of 128 x 128, which read a third
// less, 77, since a single wave a SIMD waits for what it reads.
template <class T, int MH, int CH, int WM, int WC, int ACT>
__global__ __launch_bounds__(64 * WM * WC)
void mx_matmul_staged_kernel(const so_u32x4 *__restrict__ Wc, const uint32_t *__restrict__ Ws, const so_u32x4 *__restrict__ Xc, const uint32_t *__restrict__ Xs, uint32_t m, uint32_t C,
                             uint32_t units, uint32_t wtiles, uint32_t xtiles, uint32_t mgroups, uint32_t cgroups, uint32_t per_xcd, const float *__restrict__ bias, T *__restrict__ Y,
                             size_t ldy)
{
    constexpr int V = so_elements<T>::V, WT = MH * WM / 2, XT = CH * WC / 2, WAVES = WM * WC, EACH = WT / WAVES;
    static_assert(WT == XT && WT % WAVES == 0, "a wave brings as many tiles of W and of X as every other");
    constexpr uint32_t RING = 4, X0 = WT * 2048, STAGE = (WT + XT) * 2048, S0 = RING * STAGE, SCALES = (WT + XT) * 256;
    extern __shared__ char stage[];
    const MxTile tile = mx_tile_of(mgroups, cgroups, per_xcd);
    if (tile.none) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), lane = threadIdx.x % 64u;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)stage;
    // Request P of this wave for half h, of W's codes, X's codes and, in the even halves, their scales for each of its tiles.
    const auto request = [&](uint32_t h, auto piece) {
        constexpr int P = decltype(piece)::value, I = P % EACH, KIND = P / EACH;                 // kinds 0, 1: W; 2, 3: X; 4, 5: scales
        const uint32_t t = I * WAVES + wave;
        const size_t at = (KIND < 2 || KIND == 4 ? (size_t)min(tile.m * WT + t, wtiles - 1u) : (size_t)min(tile.c * XT + t, xtiles - 1u)) * units;   // not there: the last one again, not stored
        if constexpr (KIND < 4) {
            const uint32_t to = lds0 + h % RING * STAGE + (KIND < 2 ? 0u : X0) + t * 2048u + KIND % 2 * 1024u;
            const char *src = reinterpret_cast<const char *>(KIND < 2 ? Wc : Xc) + at * 4096 + (size_t)h * 2048 + KIND % 2 * 1024;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(lane * 16u), "s"(src) : "memory", "m0");
        } else {
            const uint32_t to = lds0 + S0 + h / 2u % RING * SCALES + ((KIND == 4 ? 0u : WT) + t) * 256u;
            const char *src = reinterpret_cast<const char *>(KIND == 4 ? Ws : Xs) + (at + h / 2u) * 256;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(to), "v"(lane * 4u), "s"(src) : "memory", "m0");
        }
    };
    const auto bring = [&](uint32_t h, auto odd) { each<(decltype(odd)::value ? 4 : 6) * EACH>([&](auto piece) { request(h, piece); }); };
    constexpr int ASKS = 10 * EACH;                                  // requests of two halves, one of them with scales
    // All but the last ASKS (or 0) requests have come in LDS, and all waves are done with what they read before.
    const auto meet = [&](auto more) {
        if constexpr (decltype(more)::value) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(ASKS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
    };
    const uint32_t wm = wave / WC, wc = wave % WC;
    struct Scales { uint32_t w[MH / 2], x[CH / 2]; };
    const auto scales = [&](Scales &s, uint32_t u) {
        const char *from = stage + S0 + u % RING * SCALES + lane * 4;
#pragma unroll
        for (int i = 0; i < MH / 2; ++i) s.w[i] = *reinterpret_cast<const uint32_t *>(from + (wm * (MH / 2) + i) * 256);
#pragma unroll
        for (int k = 0; k < CH / 2; ++k) s.x[k] = *reinterpret_cast<const uint32_t *>(from + (WT + wc * (CH / 2) + k) * 256);
    };
    const auto wat = [&](uint32_t h, int i) { return *reinterpret_cast<const so_u32x4 *>(stage + h % RING * STAGE + (wm * MH + i) * 1024 + lane * 16); };
    const auto xat = [&](uint32_t h, int k) { return *reinterpret_cast<const so_u32x4 *>(stage + h % RING * STAGE + X0 + (wc * CH + k) * 1024 + lane * 16); };
    f32x4 acc[MH][CH] = {};
    so_u32x4 w[2][MH], x[CH];
    Scales e, next;
    const uint32_t halves = 2u * units;
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> odd;
    bring(0, even);
    bring(1, odd);
    if (halves > 2u) {
        bring(2, even);
        bring(3, odd);
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"(ASKS + 4 * EACH) : "memory");
    } else {
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" : : : "memory");
    }
    scales(e, 0);
#pragma unroll
    for (int i = 0; i < MH; ++i) w[0][i] = wat(0, i);
#pragma unroll
    for (int k = 0; k < CH; ++k) x[k] = xat(0, k);
    // Half h's products; the operands of half h + 1 take the places of those that have been multiplied for the last time.  Behind the last half they are read from a place of the
    // ring that holds an older one, and not used.
    const auto half = [&](uint32_t h, auto q, auto wait, auto more) {
        constexpr int Q = decltype(q)::value;
        meet(wait);                                                  // half h + 1 is there, the two after it may be on their way; half h is in registers
        if constexpr (Q == 1) scales(next, (h + 1u) / 2u);
#pragma unroll
        for (int i = 0; i < MH; ++i) w[1 - Q][i] = wat(h + 1u, i);
        __builtin_amdgcn_sched_barrier(0);
        each<CH>([&](auto k) {
            constexpr int K = decltype(k)::value;
            each<MH>([&](auto i) {
                constexpr int I = decltype(i)::value;
                acc[I][K] = mx_mfma<K % 2 * 2 + Q, I % 2 * 2 + Q>(x[K], e.x[K / 2], w[Q][I], e.w[I / 2], acc[I][K]);
            });
            x[K] = xat(h + 1u, K);
            // The requests for half h + 4, into the place of half h, one after each group of products: all at once they hold up every wave of the workgroup at the same time.
            constexpr int PIECES = (Q == 1 ? 4 : 6) * EACH, FROM = K * PIECES / CH, TO = (K + 1) * PIECES / CH;
            if constexpr (decltype(more)::value && TO > FROM)
                each<TO - FROM>([&](auto i) { request(h + 4u, std::integral_constant<int, FROM + decltype(i)::value>()); });
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (Q == 1) e = next;
    };
    const std::true_type yes;
    const std::false_type no;
    uint32_t h = 0;
    for (; h + 4u < halves; h += 2u) {
        half(h, even, yes, yes);
        half(h + 1u, odd, yes, yes);
    }
    if (h + 2u < halves) {                                           // the last unit but one: nothing left to ask for
        half(h, even, yes, no);
        half(h + 1u, odd, no, no);
        h += 2u;
    }
    half(h, even, no, no);
    half(h + 1u, odd, no, no);
    __syncthreads();
    // Out through LDS, each wave in a part of its own, 32 rows at a time: a lane's four columns of one row become 16 bytes of a row that 8 or 16 lanes store together.
    constexpr int COLS = CH * 16, PITCH = COLS + 4, LANES = COLS / V, ROWS = 64 / LANES;
    float *mine = reinterpret_cast<float *>(stage) + wave * 32 * PITCH;
    const uint64_t col = (uint64_t)tile.c * (XT * 32) + wc * COLS + lane % LANES * V;
#pragma unroll
    for (int i = 0; i < MH; i += 2) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 0; k < CH; ++k) *reinterpret_cast<f32x4 *>(mine + (j * 16 + lane % 16u) * PITCH + k * 16 + 4 * (lane / 16u)) = acc[i + j][k];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += ROWS) {
            const uint32_t r = r0 + lane / LANES;
            const uint64_t row = (uint64_t)tile.m * (WT * 32) + (wm * MH + i) * 16 + r;
            float y[V];
#pragma unroll
            for (int f = 0; f < V; f += 4) {
                const f32x4 s = *reinterpret_cast<const f32x4 *>(mine + r * PITCH + lane % LANES * V + f);
#pragma unroll
                for (int k = 0; k < 4; ++k) y[f + k] = s[k];
            }
            if (row >= m || col >= C) continue;
            const float add = bias ? bias[row] : 0.0f;
#pragma unroll
            for (int f = 0; f < V; ++f) y[f] = mx_epilogue<ACT>(y[f] + add);
            so_group_store(Y + row * ldy + col, (uint32_t)min((uint64_t)V, C - col), y);
        }
        __builtin_amdgcn_wave_barrier();
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

struct Groups { uint32_t m, c, per_xcd; };
Groups groups_of(const so_mxfp4 *W, uint32_t C, uint32_t rows, uint32_t cols)
{
    const uint32_t m = so_ceil_div(W->m, rows), c = so_ceil_div(C, cols);
    return {m, c, so_ceil_div((uint64_t)m * c, 8)};
}

template <class T, int MH, int CH, int WK, int ACT>
so_status launch(so_ctx *ctx, const so_mxfp4 *W, const so_u32x4 *codes, const uint32_t *scales, uint32_t C, const float *bias, T *Y, size_t ldy)
{
    const Groups g = groups_of(W, C, MH * 16, CH * 16);
    constexpr uint32_t bytes = WK * MH * 16 * (CH * 16 + 4) * sizeof(float);
    const auto kernel = mx_matmul_kernel<T, MH, CH, WK, ACT>;
    if (bytes > 48 * 1024) SO_HIP(so_allow_big_lds(ctx, (const void *)kernel));
    kernel<<<g.per_xcd * 8, 64 * WK, bytes, ctx->stream>>>(W->d_codes, W->d_scales, codes, scales, W->m, C, W->blocks / kMxUnit, W->tiles, so_ceil_div(C, kMxTile), g.m, g.c, g.per_xcd,
                                                          bias, Y, ldy);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

template <class T, int MH, int CH, int WM, int WC, int ACT>
so_status launch_staged(so_ctx *ctx, const so_mxfp4 *W, const so_u32x4 *codes, const uint32_t *scales, uint32_t C, const float *bias, T *Y, size_t ldy)
{
    const Groups g = groups_of(W, C, MH * WM * 16, CH * WC * 16);
    constexpr uint32_t bytes = std::max<uint32_t>(4 * (MH * WM + CH * WC) / 2 * (2048 + 256), WM * WC * 32 * (CH * 16 + 4) * sizeof(float));
    const auto kernel = mx_matmul_staged_kernel<T, MH, CH, WM, WC, ACT>;
    SO_HIP(so_allow_big_lds(ctx, (const void *)kernel));
    kernel<<<g.per_xcd * 8, 64 * WM * WC, bytes, ctx->stream>>>(W->d_codes, W->d_scales, codes, scales, W->m, C, W->blocks / kMxUnit, W->tiles, so_ceil_div(C, kMxTile), g.m, g.c, g.per_xcd,
                                                               bias, Y, ldy);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

// The forms, by tile: rows and columns of Y.  Up to 64 x 64 the waves of a workgroup share the blocks.
struct Form { uint32_t rows, cols; const char *name; };
constexpr Form kForms[] = {{16, 16, "mx-16x16"}, {32, 16, "mx-32x16"}, {32, 32, "mx-32x32"}, {64, 32, "mx-64x32"}, {64, 64, "mx-64x64"}, {64, 64, "mx-64x64-four"}, {128, 128, "mx-128x128"},
                           {256, 256, "mx-256x256"}};
constexpr int kFormCount = 8;

// The largest tile that gives every compute unit a workgroup: a larger one asks the caches for less, a smaller one leaves none idle.  From a sweep over m of 64 .. 8192, n of 512 .. 8192
// and C of 1 .. 2048 (fp32, with the quantisation; us), this form / the next smaller: 8192 x 8192 x 2048 256 x 256 76.3 / 96.3, 4096 x 8192 x 1024 128 x 128 36.9 / 37.6, 4096 x 8192 x 512
// 64 x 64 on four waves 22.4 / 25.3 on eight, 4096 x 8192 x 256 64 x 64 15.0 / 19.1, 2048 x 8192 x 256 64 x 32 11.6 / 12.6, 1024 x 8192 x 256 32 x 32 9.3 / 10.6, 2048 x 8192 x 64 32 x 16
// 8.0 / 8.7; with half as many workgroups as compute units the larger loses by as much (4096 x 8192 x 2048: 256 x 256 61.5, 128 x 128 56.3).
// None half of whose columns would do: 32768 x 4096 x 8 32 x 16 15.4, 64 x 64 on four waves 17.2, 128 x 128 20.0; 65536 x 4096 x 32 32 x 32 27.0, 128 x 128 29.9.
int choose_form(const so_ctx *ctx, uint32_t m, uint32_t C)
{
    const uint64_t cus = (uint64_t)ctx->compute_units;
    const auto tiles = [&](int f) { return (uint64_t)so_ceil_div(m, kForms[f].rows) * so_ceil_div(C, kForms[f].cols); };
    const auto rounds = [](uint64_t tiles, uint64_t at_once) { return (tiles + at_once - 1) / at_once; };
    const auto wide = [&](int f) { return C <= kForms[f].cols / 2; };
    if (tiles(6) >= cus && !wide(6)) {
        // one tile of 256 x 256 a compute unit at a time takes 0.78 of what its four quarters take, two of those at a time
        return !wide(7) && 4.0 * (double)rounds(tiles(7), cus) <= 1.28 * 2.0 * (double)rounds(tiles(6), 2 * cus) ? 7 : 6;
    }
    if (tiles(5) >= 2 * cus && !wide(5)) return 5;
    for (int f = 4; f > 0; --f)
        if (tiles(f) >= cus && !wide(f)) return f;
    return 0;
}

constexpr uint32_t kVecChunk = 16384;        // entries of x in LDS at a time
constexpr uint32_t kVecThreads = 512;

// y = W x + bias with x in fp32: a workgroup takes H halves of a tile, 16 rows each, its waves a unit of 8 blocks each in turn.  A lane multiplies one block of a row with x from LDS, which
// the rows share, and the block's sum with its scale.  Bound by the vector instructions, a conversion for two products, where few workgroups run (64 x 8192 4.5 us), and by the reading of
// the codes where many do (16384 x 16384, 143 MB: 29.2 us, 4.9 TB/s).
template <int H>
__global__ __launch_bounds__(kVecThreads)
void mx_matvec_kernel(const so_u32x4 *__restrict__ Wc, const uint32_t *__restrict__ Ws, const float *__restrict__ x, uint32_t m, uint32_t n, uint32_t units, uint32_t tiles,
                      const float *__restrict__ bias, float *__restrict__ y)
{
    constexpr uint32_t NT = kVecThreads, WAVES = NT / 64, CU = kVecChunk / 256;        // units of a chunk
    constexpr int S = H > 1 ? H / 2 : 1;                             // words of scales, one for two halves
    extern __shared__ f32x4 xs[];                                    // a chunk of x, behind it the waves' sums
    float *part = reinterpret_cast<float *>(xs) + min(units, CU) * 256;      // [WAVES][H * 16]
    const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u, odd = H == 1 ? blockIdx.x % 2u : 0u;
    const so_u32x4 *wc[S];
    const uint32_t *ws[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const size_t t = min(H == 1 ? blockIdx.x / 2u : blockIdx.x * S + i, tiles - 1u);
        wc[i] = Wc + t * units * 256 + odd * 64 + lane;
        ws[i] = Ws + t * units * 64 + lane;
    }
    struct Unit {
        so_u32x4 w[H][2];
        uint32_t s[S];
    };
    const auto load = [&](Unit &t, uint32_t u) {
#pragma unroll
        for (int i = 0; i < S; ++i) t.s[i] = ws[i][(size_t)u * 64];
#pragma unroll
        for (int i = 0; i < H; ++i)
#pragma unroll
            for (int q = 0; q < 2; ++q) t.w[i][q] = wc[i / 2][(size_t)u * 256 + q * 128 + i % 2 * 64];
    };
    float acc[H] = {};
    const auto multiply = [&](const Unit &t, uint32_t u) {           // u: of the chunk
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const f32x4 *xp = xs + (u * 8 + 4 * q + lane / 16u) * 8;
            float sum[H] = {};
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 a = xp[2 * g], b = xp[2 * g + 1];
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    const uint32_t c = t.w[i][q][g];
                    float &s = sum[i];
                    const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
                    const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
                    s = fmaf(p0[0], a[0], s);
                    s = fmaf(p0[1], a[1], s);
                    s = fmaf(p1[0], a[2], s);
                    s = fmaf(p1[1], a[3], s);
                    s = fmaf(p2[0], b[0], s);
                    s = fmaf(p2[1], b[1], s);
                    s = fmaf(p3[0], b[2], s);
                    s = fmaf(p3[1], b[3], s);
                }
            }
#pragma unroll
            for (int i = 0; i < H; ++i) {
                const uint32_t s = t.s[i / 2] >> (16 * (i % 2 + odd) + 8 * q) & 255u;
                acc[i] = fmaf(sum[i], s == 255u ? __builtin_nanf("") : so_mx_power(s), acc[i]);
            }
        }
    };
    for (uint32_t u0 = 0; u0 < units; u0 += CU) {
        const uint32_t here = min(units - u0, CU), turns = wave < here ? (here - wave + WAVES - 1u) / WAVES : 0u;
        // Two units in registers, the first ones on their way while x is; behind the last one that one again, for nothing.  As compiled, the next two are asked for together behind the products
        // of both, and waited for in part at the next turn's beginning.
        const uint32_t last = wave + (turns ? turns - 1u : 0u) * WAVES;
        Unit a, b;
        if (turns) {
            load(a, u0 + wave);
            load(b, u0 + min(wave + WAVES, last));
        }
        if (u0) __syncthreads();
        // x in groups of 16 bytes, four of them on their way (one float after the other took 37.5 us for 16384 x 16384, eight at once 31.7), what lies behind x as zeros
        for (uint32_t k0 = threadIdx.x; k0 < here * 64; k0 += 4 * NT) {
            f32x4 v[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint64_t at = (uint64_t)u0 * 256 + (k0 + i * NT) * 4u;
                v[i] = f32x4{};
                if (k0 + i * NT < here * 64 && at < n) v[i] = so_group_load(x + at, (uint32_t)min(n - at, (uint64_t)4));
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (k0 + i * NT < here * 64) xs[k0 + i * NT] = v[i];
        }
        __syncthreads();
        for (uint32_t t = 0; t + 1u < turns; t += 2u) {
            multiply(a, wave + t * WAVES);
            load(a, u0 + min(wave + (t + 2u) * WAVES, last));
            multiply(b, wave + (t + 1u) * WAVES);
            load(b, u0 + min(wave + (t + 3u) * WAVES, last));
        }
        if (turns % 2u) multiply(a, last);
    }
#pragma unroll
    for (int i = 0; i < H; ++i) {                                    // the four blocks of a row lie 16 lanes apart
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i]), __float_as_uint(acc[i]), false, false);
        const float s = __uint_as_float(a[0]) + __uint_as_float(a[1]);
        const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(s), __float_as_uint(s), false, false);
        if (lane < 16u) part[wave * (H * 16) + i * 16 + lane] = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    }
    __syncthreads();
    const uint64_t row = (uint64_t)blockIdx.x * (H * 16) + threadIdx.x;
    if (threadIdx.x < H * 16 && row < m) {
        float s[WAVES];
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) s[w] = part[w * (H * 16) + threadIdx.x];
#pragma unroll
        for (uint32_t step = WAVES / 2; step; step /= 2)
#pragma unroll
            for (uint32_t w = 0; w < step; ++w) s[w] += s[w + step];
        y[row] = bias ? s[0] + bias[row] : s[0];
    }
}

// 16 rows a workgroup up to one tile a compute unit, which leaves fewer of them idle, else 32, which share what is read of x (us, 16 / 32): 1024 x 1024 2.9 / 3.2, 1024 x 4096 3.7 / 4.7,
// 1000 x 16384 7.6 / 10.8, 8192 x 8192 9.3 / 10.0, 12000 x 12000 19.1 / 19.4, 16384 x 8192 17.2 / 14.9, 16384 x 1000 5.3 / 4.4.  (64 rows, or 1024 threads, were faster nowhere by 3%.)
template <int H>
so_status launch_matvec(so_ctx *ctx, const so_mxfp4 *W, const float *dx, const float *dBias, float *dy)
{
    const uint32_t units = W->blocks / kMxUnit, lds = (std::min(units * 256u, kVecChunk) + kVecThreads / 64 * H * 16) * (uint32_t)sizeof(float);
    const auto kernel = mx_matvec_kernel<H>;
    if (lds > 48 * 1024) SO_HIP(so_allow_big_lds(ctx, (const void *)kernel));
    kernel<<<so_ceil_div(W->m, H * 16), kVecThreads, lds, ctx->stream>>>(W->d_codes, W->d_scales, dx, W->m, W->n, units, W->tiles, dBias, dy);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

} // namespace

extern "C" so_status so_mxfp4_matmul_reserve(so_ctx *ctx, const so_mxfp4 *W, uint32_t C)
{
    SO_REQUIRE(ctx != nullptr && W != nullptr, "so_mxfp4_matmul_reserve: null handle");
    SO_REQUIRE(!ctx->capturing, "so_mxfp4_matmul_reserve: a graph is being recorded");
    if (C == 0) return SO_OK;
    SO_REQUIRE(W->device == ctx->device, "so_mxfp4_matmul_reserve: the matrix lies on another device");
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
    SO_REQUIRE(W->device == ctx->device, "so_mxfp4_matmul: the matrix lies on another device");
    const Form &form = kForms[ctx->tune.mxfp4_form >= 1 && ctx->tune.mxfp4_form <= kFormCount ? ctx->tune.mxfp4_form - 1 : choose_form(ctx, W->m, C)];
    SO_REQUIRE(so_grid_fits((uint64_t)so_ceil_div(W->m, form.rows) * so_ceil_div(C, form.cols) + 8, 512), "so_mxfp4_matmul: %u x %u output is too large for one launch", W->m, C);
    if (const so_status s = so_mx_quantize_columns(ctx, type, dX, x_stride, W->n, C, nullptr, nullptr); s != SO_OK) return s;      // whether it can be done
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    if (const so_status s = reserve(ctx, "so_mxfp4_matmul", W, C); s != SO_OK) return s;
    so_u32x4 *codes = (so_u32x4 *)ctx->mm_part->p;
    uint32_t *scales = (uint32_t *)((char *)codes + workspace_of(W, C).codes);
    if (const so_status s = so_mx_quantize_columns(ctx, type, dX, x_stride, W->n, C, codes, scales); s != SO_OK) return s;
    ctx->last_kernel = form.name;
    so_status status = SO_OK;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        const auto with = [&](auto a) {
            constexpr int ACT = decltype(a)::value;
            T *y = (T *)dY;
            const auto run = [&](auto kernel) { status = kernel(ctx, W, codes, scales, C, dBias, y, y_stride); };
            switch (&form - kForms) {
            case 0: run(launch<T, 1, 1, 8, ACT>); break;
            case 1: run(launch<T, 2, 1, 8, ACT>); break;
            case 2: run(launch<T, 2, 2, 8, ACT>); break;
            case 3: run(launch<T, 4, 2, 8, ACT>); break;
            case 4: run(launch<T, 4, 4, 8, ACT>); break;
            case 5: run(launch<T, 4, 4, 4, ACT>); break;
            case 6: run(launch_staged<T, 4, 4, 2, 2, ACT>); break;
            default: run(launch_staged<T, 4, 8, 4, 2, ACT>); break;
            }
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
    SO_REQUIRE(W->device == ctx->device, "so_mxfp4_matvec: the matrix lies on another device");
    SO_REQUIRE(so_grid_fits(W->tiles, kVecThreads), "so_mxfp4_matvec: %u rows are too many for one launch", W->m);
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    return W->tiles <= (uint32_t)ctx->compute_units ? launch_matvec<1>(ctx, W, dx, dBias, dy) : launch_matvec<2>(ctx, W, dx, dBias, dy);
}
