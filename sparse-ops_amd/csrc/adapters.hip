// Low-rank adapters of many requests: Y = base + scale_a B_a (A_a X), the adapter a of every column its own.
//
// Two launches.  Both take the columns 64 at a time and go over the adapters that occur among them, one after the other, or, where there are few such tiles, side by side: one tile of columns is multiplied as a
// whole with an adapter, and of the result those columns are kept that have it.  So the columns of a prompt, which share one, are read once, and of a batch of single tokens every adapter is.
#include "dense.h"
#include "lane_moves.h"

namespace {

using so_dense::f32x4;
using so_dense::Operand;
using so_dense::u32x4;

constexpr uint32_t kThreads = 256, kMostRank = 256, kCols = 64, kPad = 16;

// Adapters in turn: the one of `lane`'s column, or none, and those that occur in the 64 columns of a tile by their first column.
struct Which {
    uint32_t mine;
    bool has;
    uint64_t none;           // columns that exist and have no adapter
    __device__ __forceinline__ Which(const int32_t *which, uint64_t j0, uint32_t C, uint32_t count)
    {
        const uint64_t c = j0 + threadIdx.x % 64u;
        mine = c < C ? (uint32_t)which[c] : 0xffffffffu;
        has = mine < count;                                              // a negative number is beyond all others
        none = __ballot(c < C && !has);
    }
    // The adapter that is number `turn` of the tile, and its columns; no columns: there is none.
    struct Turn { uint32_t adapter; uint64_t columns; };
    __device__ __forceinline__ Turn turn(uint32_t turn) const
    {
        uint64_t left = __ballot(has);
        for (; left; --turn) {
            const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)mine, __builtin_ctzll(left));
            const uint64_t columns = __ballot(has && mine == a);
            if (turn == 0) return {a, columns};
            left &= ~columns;
        }
        return {0, 0};
    }
};

// How a call is cut: tiles of 64 columns, turns side by side, parts of the features; the rows of Y that a workgroup takes.
struct Cut { uint32_t tiles, turns, parts, depth, rows, row_groups, padded; };

template <class T> struct Call {
    const T *A, *B, *X, *base;
    T *Y;
    const float *scale;
    const int32_t *which;
    float *low;              // [parts][C][padded]: A x, an adapter's entries beyond its rank zeros
    size_t ldx, ldb, ldy;
    uint32_t m, n, C, count, rank;
    Cut cut;
};

// A x of one part of the features for the columns of the adapters in turn.
template <class T, class TILE, bool DIRECT>
__global__ __launch_bounds__(kThreads)
void adapters_in_kernel(Call<T> f)
{
    extern __shared__ char stage[];
    const uint32_t tile = blockIdx.x % f.cut.tiles, part = blockIdx.x / f.cut.tiles % f.cut.parts;
    const uint64_t j0 = (uint64_t)tile * kCols;
    const size_t k0 = (size_t)part * f.cut.depth;
    const uint32_t depth = (uint32_t)min((size_t)f.cut.depth, f.n - k0), lane = threadIdx.x % 64u;
    const Which which(f.which, j0, f.C, f.count);
    for (uint32_t turn = blockIdx.x / f.cut.tiles / f.cut.parts;; turn += f.cut.turns) {
        const Which::Turn at = which.turn(turn);
        if (!at.columns) return;
        for (uint32_t r0 = 0; r0 < f.rank; r0 += TILE::ROWS) {
            so_dense::Loop<T, TILE, false, true, false> loop;
            loop.template add<DIRECT>(stage, {{f.A + (size_t)at.adapter * f.rank * f.n + k0, f.n, f.rank, depth}}, r0, {f.X + k0 * f.ldx, f.ldx, f.C, depth}, j0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t col = threadIdx.x / 64u * 16u + 4u * (lane / 16u) + e;
                if (!(at.columns >> col & 1u)) continue;
                float *to = f.low + ((size_t)part * f.C + j0 + col) * f.cut.padded + r0 + lane % 16u;
#pragma unroll
                for (int i = 0; i < TILE::RT; ++i)
                    if (r0 + i * 16 < f.cut.padded) to[i * 16] = r0 + i * 16 + lane % 16u < f.rank ? loop.acc[i][0][e] : 0.0f;
            }
        }
    }
}

// Y for the columns of the adapters in turn, and of those that have none.  A wave takes 16 rows at a time; the products' operand of 64 columns stays in registers, RC times 16 entries of rank.  Columns are
// dealt to the instructions so that a lane's results are 16 bytes of a row: in 16 bits column 8 g + 4 k + e is that of instruction k (of two), lanes 16 g .., result e.
template <class T, int RC>
__global__ __launch_bounds__(kThreads)
void adapters_out_kernel(Call<T> f)
{
    constexpr int V = so_elements<T>::V, RUNS = 16 / V;                  // groups of 16 bytes that a lane has of a row
    constexpr bool HALF = sizeof(T) == 2;
    typedef typename so_elements<T>::plain group;
    const uint32_t tile = blockIdx.x % f.cut.tiles, part = blockIdx.x / f.cut.tiles % f.cut.row_groups, lane = threadIdx.x % 64u, l = lane % 16u, g = lane / 16u;
    const uint64_t j0 = (uint64_t)tile * kCols, row0 = (uint64_t)part * f.cut.rows, row_end = min(row0 + f.cut.rows, (uint64_t)f.m);
    const Which which(f.which, j0, f.C, f.count);
    // the column of the tile that operand lane l of instruction k has, and the first of run p's
    const auto column = [&](int k) { return HALF ? k / 2 * 32u + l / 4u * 8u + k % 2 * 4u + l % 4u : k * 16u + l; };
    const auto first = [&](int p) { return HALF ? p * 32u + g * 8u : p * 16u + g * 4u; };
    const auto store = [&](uint64_t row, int p, uint64_t columns, const float (&v)[V]) {
        const uint32_t bits = (uint32_t)(columns >> first(p)) & ((1u << V) - 1u);
        T *to = f.Y + row * f.ldy + j0 + first(p);
        if (bits == (1u << V) - 1u) so_group_store(to, V, v);
        else
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (bits >> e & 1u) to[e] = (T)v[e];
    };
    struct Row { group base[RUNS]; };
    const auto load_base = [&](uint64_t row, Row &r) {
#pragma unroll
        for (int p = 0; p < RUNS; ++p) {
            r.base[p] = group{};
            const uint64_t c = j0 + first(p);
            if (f.base && row < row_end && c < f.C) r.base[p] = so_group_load(f.base + row * f.ldb + c, (uint32_t)min((uint64_t)V, f.C - c));
        }
    };
    uint32_t turn = blockIdx.x / f.cut.tiles / f.cut.row_groups;
    if (turn == 0 && which.none && f.base != f.Y)
        for (uint64_t row = row0 + threadIdx.x / 64u * 16u + l; row < row_end; row += 64u) {
            Row r;
            load_base(row, r);
#pragma unroll
            for (int p = 0; p < RUNS; ++p) {
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = (float)r.base[p][e];
                store(row, p, which.none, v);
            }
        }
    for (;; turn += f.cut.turns) {
        const Which::Turn at = which.turn(turn);
        if (!at.columns) return;
        const T *B = f.B + (size_t)at.adapter * f.m * f.rank;
        const float scale = f.scale ? f.scale[at.adapter] : 1.0f;
        const uint32_t blocks = (f.cut.padded + RC * 16u - 1u) / (RC * 16u);
        // the entries of rank that this lane has of a run of 16, of instruction k's column
        const auto low = [&](int k, uint32_t run, float (&v)[V]) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = 0.0f;
            const uint32_t col = column(k);
            if (run * 16u >= f.cut.padded || !(at.columns >> col & 1u)) return;
            const float *from = f.low + (j0 + col) * f.cut.padded + run * 16u + (HALF ? g % 2u * 8u : g * 4u);
            for (uint32_t p = 0; p < f.cut.parts; ++p, from += (size_t)f.C * f.cut.padded)
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    const f32x4 s = *reinterpret_cast<const f32x4 *>(from + e);
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[e + c] += s[c];
                }
        };
        // In fp16 a column's entries are taken times a power of two that brings the largest to 2^14 .. 2^15; by[k][e]: what result e of instruction k is multiplied with.
        float shift[4] = {1.0f, 1.0f, 1.0f, 1.0f}, by[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (std::is_same<T, _Float16>::value) {
                float largest = 0.0f;
                for (uint32_t run = 0; run * 16u < f.cut.padded; ++run) {
                    float v[V];
                    low(k, run, v);
#pragma unroll
                    for (int e = 0; e < V; ++e) largest = fmaxf(largest, fabsf(v[e]));
                }
                const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(largest), __float_as_uint(largest), false, false);
                const uint32_t top = max(h[0], h[1]) >> 23;              // the largest's exponent, biased
                const int up = top >= 255u ? 0 : min(max(141 - (int)top, -100), 100);
                shift[k] = __uint_as_float((uint32_t)(127 + up) << 23);
                const float down = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
                for (int e = 0; e < 4; ++e) by[k][e] = __uint_as_float((uint32_t)__builtin_amdgcn_ds_bpermute((int)(4u * g + e) * 4, (int)__float_as_uint(down)));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) by[k][e] = 1.0f;
            }
        }
        u32x4 t[4][RC];
        const auto operand = [&](uint32_t block) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int c = 0; c < RC; ++c) {
                    float v[V];
                    low(k, block * RC + c, v);
                    if constexpr (HALF) {
                        // 16 entries as 32: lanes 0 .. 31 have them rounded to T, the others what that leaves, so that the product, with B's entries twice, has them to 2^-16
                        group r;
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float w = v[e] * shift[k];
                            const T high = (T)w;
                            r[e] = g < 2u ? high : __builtin_isinf((float)high) ? (T)0.0f : (T)(w - (float)high);
                        }
                        t[k][c] = __builtin_bit_cast(u32x4, r);
                    } else {
                        t[k][c] = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
                    }
                }
        };
        const auto load_b = [&](uint64_t row, uint32_t block, u32x4 (&b)[RC]) {
#pragma unroll
            for (int c = 0; c < RC; ++c) {
                const uint32_t r = (block * RC + c) * 16u + (HALF ? g % 2u * 8u : g * 4u);
                b[c] = u32x4{};
                if (row < row_end && r < f.rank) b[c] = __builtin_bit_cast(u32x4, so_group_load(B + (size_t)row * f.rank + r, min(f.rank - r, (uint32_t)V)));
            }
        };
        if (blocks == 1) operand(0);
        Row r, next;
        u32x4 b[RC], next_b[RC];
        uint64_t row = row0 + threadIdx.x / 64u * 16u + l;
        load_base(row, r);
        load_b(row, 0, b);
        for (uint64_t at_row = row0 + threadIdx.x / 64u * 16u; at_row < row_end; at_row += 64u, row += 64u) {
            load_base(row + 64u, next);
            if (blocks == 1) load_b(row + 64u, 0, next_b);
            f32x4 acc[4] = {};
            for (uint32_t block = 0; block < blocks; ++block) {
                if (blocks > 1) {
                    operand(block);
                    load_b(row, block, b);
                }
#pragma unroll
                for (int c = 0; c < RC; ++c)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[k] = so_dense::multiply<T>(b[c], t[k][c], acc[k]);
            }
            if (row < row_end)
#pragma unroll
                for (int p = 0; p < RUNS; ++p) {
                    float v[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int k = HALF ? 2 * p + e / 4 : p;
                        v[e] = fmaf(acc[k][e % 4] * by[k][e % 4], scale, (float)r.base[p][e]);
                    }
                    store(row, p, at.columns, v);
                }
            r = next;
#pragma unroll
            for (int c = 0; c < RC; ++c) b[c] = next_b[c];
        }
    }
}

Cut cut_of(const so_ctx *ctx, int type, uint32_t m, uint32_t n, uint32_t C, uint32_t rank)
{
    const uint32_t step = (rank <= 16 ? 256u : 128u) / (uint32_t)so_type_bytes(type);      // of the first launch
    const uint64_t cus = (uint64_t)ctx->compute_units;
    Cut c;
    c.tiles = so_ceil_div(C, kCols);
    // Up to two tiles a compute unit side by side in turns: a tile may have as many adapters as columns, and a workgroup without one ends at once
    c.turns = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(std::min(C, kCols), cus / 2 / c.tiles));
    c.padded = so_ceil_div(rank, kPad) * kPad;
    const uint64_t most = std::max<uint64_t>(1, so_ceil_div(n, 2 * step)), want = std::max<uint64_t>(1, 2 * cus / ((uint64_t)c.tiles * c.turns));
    c.parts = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(most, std::max<uint64_t>(want, c.tiles < cus ? 4 : 1)), 16);
    c.depth = so_ceil_div(so_ceil_div(n, c.parts), step) * step;
    c.parts = so_ceil_div(n, c.depth);
    // rows of a workgroup: 64 times as many as leave four workgroups a compute unit
    const uint64_t rows = (uint64_t)so_ceil_div(m, 64) * c.tiles * c.turns / (4 * cus);
    c.rows = 64u * (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(rows, 16));
    c.row_groups = so_ceil_div(m, c.rows);
    return c;
}

size_t low_bytes(const Cut &c, uint32_t C) { return (size_t)c.parts * C * c.padded * sizeof(float); }

so_status workspace(so_ctx *ctx, const char *who, size_t bytes)
{
    SO_REQUIRE(!ctx->capturing || (ctx->mm_part && ctx->mm_part->bytes >= bytes),
               "%s: the context's workspace must grow, which cannot be done while a graph is being recorded (call so_adapters_reserve, or launch this shape once, before recording)", who);
    return so_matmul_workspace(ctx, bytes, 4);
}

template <class T, class TILE>
so_status launch_in(so_ctx *ctx, const Call<T> &f, bool direct)
{
    const auto kernel = direct ? adapters_in_kernel<T, TILE, true> : adapters_in_kernel<T, TILE, false>;
    SO_HIP(so_allow_big_lds(ctx, (const void *)kernel));
    kernel<<<f.cut.tiles * f.cut.parts * f.cut.turns, kThreads, TILE::lds, ctx->stream>>>(f);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

template <class T>
so_status run(so_ctx *ctx, Call<T> f)
{
    const uint64_t in = (uint64_t)f.cut.tiles * f.cut.parts * f.cut.turns, out = (uint64_t)f.cut.tiles * f.cut.row_groups * f.cut.turns;
    SO_REQUIRE(so_grid_fits(std::max(in, out), kThreads), "so_adapters: %u x %u is too large for one launch", f.m, f.C);
    if (f.count) {
        const Operand<T> a = {f.A, f.n, f.rank, f.n}, x = {f.X, f.ldx, f.C, f.n};
        const bool direct = a.direct() && x.direct();
        so_status s;
        if (f.rank <= 16) s = launch_in<T, so_dense::Tile<1, 1, 1, 4, 256, 3>>(ctx, f, direct);
        else if (f.rank <= 32) s = launch_in<T, so_dense::Tile<2, 1, 1, 4, 128, 4>>(ctx, f, direct);
        else s = launch_in<T, so_dense::Tile<4, 1, 1, 4, 128, 4>>(ctx, f, direct);
        if (s != SO_OK) return s;
    }
    const auto kernel = f.rank <= 16 ? adapters_out_kernel<T, 1> : f.rank <= 32 ? adapters_out_kernel<T, 2> : adapters_out_kernel<T, 4>;
    kernel<<<(uint32_t)out, kThreads, 0, ctx->stream>>>(f);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

} // namespace

extern "C" so_status so_adapters_reserve(so_ctx *ctx, int type, uint32_t m, uint32_t n, uint32_t C, uint32_t rank)
{
    SO_REQUIRE(ctx != nullptr, "so_adapters_reserve: ctx is null");
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, "so_adapters_reserve: unknown element type %d", type);
    SO_REQUIRE(rank >= 1 && rank <= kMostRank, "so_adapters_reserve: rank %u is not 1 .. %u", rank, kMostRank);
    SO_REQUIRE(!ctx->capturing, "so_adapters_reserve: a graph is being recorded");
    if (m == 0 || n == 0 || C == 0) return SO_OK;
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    return workspace(ctx, "so_adapters_reserve", low_bytes(cut_of(ctx, type, m, n, C, rank), C));
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
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const Cut c = cut_of(ctx, type, m, n, C, rank);
    if (const so_status s = workspace(ctx, "so_adapters", low_bytes(c, C)); s != SO_OK) return s;
    so_status status = SO_OK;
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        status = run<T>(ctx, {(const T *)dA, (const T *)dB, (const T *)dX, (const T *)dBase, (T *)dY, dScale, dWhich, (float *)ctx->mm_part->p, x_stride, base_stride, y_stride, m, n, C, count, rank, c});
    });
    return status;
}
