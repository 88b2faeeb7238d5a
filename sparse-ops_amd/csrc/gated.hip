// The gated feed-forward block: both projections, the activation and the product, and their gradients.
#include "dense.h"
#include "gate.h"
#include "lane_moves.h"

namespace {

using so_dense::f32x4;
using so_dense::Grid;
using so_dense::Operand;

constexpr int kThreads = 256;

// A long contraction over few tiles of the result is dealt to workgroups piece by piece: each piece's sums go to the workspace as [piece][row][column], fp32, and are added up in order by a kernel of their own.
// dX of 145 x 89 from 2 x 6578 terms in fp32, 6 to 15 tiles: 300 us as a whole, 16 in pieces and 4 to join them.
struct Pieces {
    float *to;                       // null: no pieces
    uint32_t cuts, depth;            // of one product: how many, and of how many terms
    size_t pitch;
    __device__ __forceinline__ float *at(uint64_t row, uint64_t col) const { return to + row * pitch + col; }
};

// The piece of an operand that begins at k0, its rows along the contraction or across.
template <class T, bool ACROSS>
__device__ __forceinline__ Operand<T> piece_of(const Operand<T> &o, uint32_t k0, uint32_t depth)
{
    return {o.p + (ACROSS ? k0 * o.ld : k0), o.ld, o.own, min(depth, o.depth - k0)};
}

// V neighbouring sums of a row from its pieces, `between` rows apart.
template <int V>
__device__ __forceinline__ void join(const Pieces &p, uint32_t count, uint64_t between, uint64_t row, uint64_t col, float (&v)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.0f;
    constexpr uint32_t AHEAD = 32 / V;
    for (uint32_t i = 0; i < count; i += AHEAD) {
        f32x4 w[AHEAD][V / 4];
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j)
#pragma unroll
            for (int e = 0; e < V; e += 4) w[j][e / 4] = *reinterpret_cast<const f32x4 *>(p.at(row + min(i + j, count - 1u) * between, col + e));
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += i + j < count ? w[j][e / 4][e % 4] : 0.0f;
    }
}

template <int V>
__device__ __forceinline__ void keep(const Pieces &p, uint64_t row, uint64_t col, const float (&v)[V])
{
#pragma unroll
    for (int e = 0; e < V; e += 4) *reinterpret_cast<f32x4 *>(p.at(row, col + e)) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
}

template <class T> struct Forward {
    const T *Wg, *Wu, *X, *G0, *U0;
    T *H, *G, *U;
    size_t ldw, ldx, ld0, ldh, ldg;
    uint32_t m, n, B;
    int act;
    Pieces pieces;
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
    so_gate::apply<T, V>(f.act, g, u);
    so_group_store(f.H + row * f.ldh + col, left, g);
}

// A tile of both projections: half of its rows are the gate's, half the other's, so that every wave holds both sums of its part of H, and activation and
// product are its epilogue.  8192 x 4096 (m x n) in 16 bits: 4096 columns 440 to 467 us, 1.18 to 1.25 PFLOP/s, where both products alone, as one of 16384 rows, take a library 405: the matrix cores are busy 59 % of the
// clocks that the chip's power leaves them, and the rest is LDS and its filling; 24 columns 23 us, the weights at 5.9 TB/s (27 on data that is in no cache).  2777 x 1531 x 203 fp32: 55.6 us, 65 % of the clocks, without
// the 5.8 that joining its pieces takes.
template <class T, class TILE, bool DIRECT>
__global__ __launch_bounds__(TILE::THREADS)
void gated_kernel(Forward<T> f, Grid grid)
{
    extern __shared__ char stage[];
    const auto spot = so_dense::spot_of(grid);
    if (spot.none) return;
    so_dense::Loop<T, TILE, false, true, true> loop;
    constexpr bool PIECES = TILE::ROWS < 256;                            // of the largest tile there are enough
    const bool pieces = PIECES && f.pieces.to;
    const uint32_t each = (f.m + TILE::ROWS / 2 - 1u) / (TILE::ROWS / 2), piece = pieces ? spot.m / each : 0u, k0 = piece * f.pieces.depth;
    const uint64_t i0 = (uint64_t)(spot.m - piece * each) * (TILE::ROWS / 2), j0 = (uint64_t)spot.c * TILE::COLS;
    const Operand<T> g = {f.Wg, f.ldw, f.m, f.n}, u = {f.Wu, f.ldw, f.m, f.n}, x = {f.X, f.ldx, f.B, f.n};
    if constexpr (!PIECES) loop.template add<DIRECT>(stage, {g, u}, i0, x, j0);
    else loop.template add<DIRECT>(stage, {piece_of<T, false>(g, k0, f.pieces.depth), piece_of<T, false>(u, k0, f.pieces.depth)}, i0, piece_of<T, true>(x, k0, f.pieces.depth), j0);
    __syncthreads();
    const uint64_t row0 = i0 + threadIdx.x / 64u / TILE::WC * (TILE::RT / 2 * 16);
    loop.template out<2>(stage, [&](int i, uint32_t r, uint32_t c, float (&v)[2][so_elements<T>::V]) {
        const uint64_t row = row0 + i * 16 + r, col = j0 + c;
        if (!pieces) return finish(f, row, col, v[0], v[1]);
        if (row >= f.m || col >= f.B) return;
        keep(f.pieces, piece * 2u * (uint64_t)f.m + row, col, v[0]);
        keep(f.pieces, (piece * 2u + 1u) * (uint64_t)f.m + row, col, v[1]);
    });
}

// Both sums from their pieces, and what follows them.  Bound by memory: 5.8 us for two pieces of 2777 x 203 fp32.
template <class T>
__global__ __launch_bounds__(kThreads)
void gated_join_kernel(Forward<T> f, uint32_t groups)
{
    constexpr int V = so_elements<T>::V;
    const uint32_t at = blockIdx.x * kThreads + threadIdx.x, row = at / groups, col = at % groups * V;      // a launch has fewer than 2^32 threads
    if (row >= f.m) return;
    float g[V], u[V];
    join(f.pieces, f.pieces.cuts, 2u * (uint64_t)f.m, row, col, g);
    join(f.pieces, f.pieces.cuts, 2u * (uint64_t)f.m, (uint64_t)row + f.m, col, u);
    finish(f, row, col, g, u);
}

// One column: a wave takes R rows of both projections, 64 lanes a group of 16 bytes each, and holds a panel of kPanel groups a lane of X in registers for them.  Bound by memory: 16384 x 4096 bf16,
// 268 MB, 43 us or 6.1 TB/s (52 in a loop over inputs that no cache holds).
constexpr int kPanel = 8;
template <class T, int R>
__global__ __launch_bounds__(kThreads)
void gated_token_kernel(Forward<T> f)
{
    constexpr int V = so_elements<T>::V;
    typedef typename so_elements<T>::plain group;
    const uint32_t lane = threadIdx.x % 64u, groups = f.n / V, rest = f.n % V;
    const uint64_t row0 = ((uint64_t)blockIdx.x * (kThreads / 64) + threadIdx.x / 64u) * R;
    if (row0 >= f.m) return;
    const T *wg[R], *wu[R];
    float g[R], u[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint64_t row = min(row0 + r, (uint64_t)f.m - 1u);          // not there: the last one again, not stored
        wg[r] = f.Wg + row * f.ldw;
        wu[r] = f.Wu + row * f.ldw;
        g[r] = u[r] = 0.0f;
    }
    const auto panel = [&](uint32_t q0, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        group x[kPanel];
        uint32_t at[kPanel];
#pragma unroll
        for (int c = 0; c < kPanel; ++c) {
            const uint32_t q = q0 + c * 64u + lane;
            at[c] = (WHOLE ? q : min(q, groups - 1u)) * V;               // not there: the last one again, as zeros
            if (f.ldx == 1) x[c] = *reinterpret_cast<const typename so_elements<T>::vec *>(f.X + at[c]);
            else
#pragma unroll
                for (int e = 0; e < V; ++e) x[c][e] = f.X[(size_t)(at[c] + e) * f.ldx];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            group a[kPanel], b[kPanel];
#pragma unroll
            for (int c = 0; c < kPanel; ++c) {
                a[c] = *reinterpret_cast<const typename so_elements<T>::vec *>(wg[r] + at[c]);
                b[c] = *reinterpret_cast<const typename so_elements<T>::vec *>(wu[r] + at[c]);
            }
#pragma unroll
            for (int c = 0; c < kPanel; ++c) {
                float p = 0.0f, q = 0.0f;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    p = fmaf((float)a[c][e], (float)x[c][e], p);
                    q = fmaf((float)b[c][e], (float)x[c][e], q);
                }
                const bool there = WHOLE || q0 + c * 64u + lane < groups;
                g[r] += there ? p : 0.0f;
                u[r] += there ? q : 0.0f;
            }
        }
    };
    uint32_t q0 = 0;
    for (; q0 + 64u * kPanel <= groups; q0 += 64u * kPanel) panel(q0, std::true_type());
    if (q0 < groups) panel(q0, std::false_type());
    if (lane < rest) {
        const size_t k = (size_t)groups * V + lane;
        const float x = (float)f.X[k * f.ldx];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            g[r] = fmaf((float)wg[r][k], x, g[r]);
            u[r] = fmaf((float)wu[r][k], x, u[r]);
        }
    }
    float mine[1] = {}, other[1] = {};                                   // of row row0 + lane
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float p = so_lanes::reduce<64>(g[r], so_lanes::Sum()), q = so_lanes::reduce<64>(u[r], so_lanes::Sum());
        if (lane == r) mine[0] = p, other[0] = q;
    }
    const uint64_t row = row0 + lane;
    if (lane >= R || row >= f.m) return;
    if (f.G0) mine[0] += (float)f.G0[row * f.ld0];
    if (f.U0) other[0] += (float)f.U0[row * f.ld0];
    if (f.G) f.G[row * f.ldg] = (T)mine[0];
    if (f.U) f.U[row * f.ldg] = (T)other[0];
    so_gate::apply<T, 1>(f.act, mine, other);
    f.H[row * f.ldh] = (T)mine[0];
}

// A matrix with its rows at multiples of 16 bytes: 1003 x 331 fp16 in 2.2 us, where a product that takes it as it lies, through registers, takes half as long again.
template <class T> struct Rows {
    const T *X;
    size_t ldx;
    uint32_t rows, cols, groups, blocks;     // groups of a row; workgroups, 0: nothing to do
    T *Y;
    size_t ldy;
    __device__ __forceinline__ void copy(uint32_t at) const
    {
        constexpr int V = so_elements<T>::V;
        const uint32_t row = at / groups, col = at % groups * V;
        if (row >= rows) return;
        const auto v = so_group_load(X + row * ldx + col, min((uint32_t)V, cols - col));
        *reinterpret_cast<typename so_elements<T>::vec *>(Y + row * ldy + col) = v;      // zeros behind the row's end
    }
};
template <class T>
__global__ __launch_bounds__(kThreads)
void align_rows_kernel(Rows<T> x)
{
    x.copy(blockIdx.x * kThreads + threadIdx.x);
}

// The gradients of the two sums, to either or both of two places (the caller's and the products').  A thread takes a group of 16 bytes of a row; groups of whole rows follow one another.  It reads what it
// needs before it writes, so that the caller's may be the inputs.  In 16 bits both are rounded to the type, which the products take operands of: as any 16-bit gradient that is handed on, and as the caller gets them.
// It makes the results' errors 1.4 times what rounding them alone makes (8192 x 4096 x 4096: bf16 2.4e-3 for 1.7e-3 of the norm, fp16 3.0e-4 for 2.1e-4); two numbers for each would double the products, 860 of 930 us.  The first workgroups align X for the products, where that is to be done.  Bound by memory: 8192 x 4096 bf16, 335 MB, 54 us or 6.2 TB/s.
template <class T> struct Place {
    T *g, *u;
    size_t ld;
};
template <class T> struct Slopes {
    const T *G, *U, *dH;
    size_t ldg, ldh;
    uint32_t m, B, groups;           // groups of a row
    int act;
    Place<T> to[2];
};
template <class T>
__global__ __launch_bounds__(kThreads)
void gated_slopes_kernel(Slopes<T> s, Rows<T> x)
{
    constexpr int V = so_elements<T>::V;
    if (blockIdx.x < x.blocks) return x.copy(blockIdx.x * kThreads + threadIdx.x);
    const uint32_t at = (blockIdx.x - x.blocks) * kThreads + threadIdx.x, row = at / s.groups, col = at % s.groups * V;
    if (row >= s.m) return;
    const uint32_t left = min((uint32_t)V, s.B - col);
    const auto gv = so_group_load(s.G + row * s.ldg + col, left), uv = so_group_load(s.U + row * s.ldg + col, left), hv = so_group_load(s.dH + row * s.ldh + col, left);
    float g[V], u[V];
    so_gate::with_slope<sizeof(T) == 2>(s.act, [&](auto both) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const so_gate::Both b = both((float)gv[e]);
            g[e] = (float)hv[e] * (float)uv[e] * b.slope;
            u[e] = (float)hv[e] * b.value;
        }
    });
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (s.to[i].g) so_group_store(s.to[i].g + row * s.to[i].ld + col, left, g);
        if (s.to[i].u) so_group_store(s.to[i].u + row * s.to[i].ld + col, left, u);
    }
}

// Y = A[0] B[0] + A[1] B[1], or either's rows one after the other where the result has two parts (Y2 is not null).  The three gradients of 8192 x 4096 x
// 4096 bf16: 430 us dX, both operands turned on their way out of LDS, and 430 both weights', 1.28 PFLOP/s each; the matrix cores are busy 63 to 65 % of the clocks.
template <class T> struct Product {
    Operand<T> A[2], B[2];
    T *Y, *Y2;
    size_t ldy;
    uint32_t rows, cols, terms;      // of one part; products to add
    Pieces pieces;                   // of either product in turn
};

template <class T, class TILE, bool AX, bool BX, bool DIRECT>
__global__ __launch_bounds__(TILE::THREADS)
void product_kernel(Product<T> p, Grid grid)
{
    extern __shared__ char stage[];
    const auto spot = so_dense::spot_of(grid);
    if (spot.none) return;
    const uint32_t each = (p.rows + TILE::ROWS - 1u) / TILE::ROWS, tiles = p.Y2 ? 2u * each : each;
    constexpr bool PIECES = TILE::ROWS < 256;                            // of the largest tile there are enough
    const bool pieces = PIECES && p.pieces.to;
    const uint32_t piece = pieces ? spot.m / tiles : 0u, m = spot.m - piece * tiles, second = m >= each ? 1u : 0u;
    so_dense::Loop<T, TILE, AX, BX, false> loop;
    const uint64_t i0 = (uint64_t)(m - second * each) * TILE::ROWS, j0 = (uint64_t)spot.c * TILE::COLS;
    const uint32_t term = pieces ? piece / p.pieces.cuts : 0u, k0 = (piece - term * p.pieces.cuts) * p.pieces.depth;
    for (uint32_t t = term; t < (pieces ? term + 1u : p.terms); ++t) {
        if constexpr (PIECES) loop.template add<DIRECT>(stage, {piece_of<T, AX>(p.A[second + t], k0, p.pieces.depth)}, i0, piece_of<T, BX>(p.B[second + t], k0, p.pieces.depth), j0);
        else loop.template add<DIRECT>(stage, {p.A[second + t]}, i0, p.B[second + t], j0);
    }
    __syncthreads();
    T *Y = second ? p.Y2 : p.Y;
    const uint64_t row0 = i0 + threadIdx.x / 64u / TILE::WC * (TILE::RT * 16), kept = (tiles == each ? piece : 2u * piece + second) * (uint64_t)p.rows;
    loop.template out<1>(stage, [&](int i, uint32_t r, uint32_t c, float (&v)[1][so_elements<T>::V]) {
        const uint64_t row = row0 + i * 16 + r, col = j0 + c;
        if (row >= p.rows || col >= p.cols) return;
        if (pieces) keep(p.pieces, kept + row, col, v[0]);
        else so_group_store(Y + row * p.ldy + col, (uint32_t)min((uint64_t)so_elements<T>::V, p.cols - col), v[0]);
    });
}

template <class T>
__global__ __launch_bounds__(kThreads)
void product_join_kernel(Product<T> p, uint32_t groups, uint32_t parts)
{
    constexpr int V = so_elements<T>::V;
    const uint32_t at = blockIdx.x * kThreads + threadIdx.x, row = at / groups, col = at % groups * V;
    if (row >= (uint64_t)parts * p.rows) return;
    float v[V];
    join(p.pieces, p.terms * p.pieces.cuts, (uint64_t)parts * p.rows, row, col, v);
    T *Y = row >= p.rows ? p.Y2 + (row - p.rows) * p.ldy : p.Y + row * p.ldy;
    so_group_store(Y + col, min((uint32_t)V, p.cols - col), v);
}

// Tiles, by rows and columns of the result (of both projections together in the forward pass).
typedef so_dense::Tile<8, 4, 2, 4, 64, 4> T256x256;
typedef so_dense::Tile<4, 4, 2, 2, 64, 4> T128x128;
typedef so_dense::Tile<4, 2, 1, 4, 128, 3> T64x128;
typedef so_dense::Tile<2, 2, 2, 2, 128, 4> T64x64;
typedef so_dense::Tile<2, 1, 1, 4, 256, 3, true> T32x64;
typedef so_dense::Tile<2, 1, 1, 2, 256, 4, true> T32x32;

// A KiB of the contraction of one tile on every compute unit, and of one more tile, in us, for elements of 2 and of 4 bytes: operands past the registers, both of them across the contraction (dX's), and by way of the
// registers (two tiles only).  Measured with 256, 512, 768 and 1024 tiles of each form and contractions of 4 and 8 KiB: 64 x 128 in 16 bits, say, takes 2.8, 4.7, 7.6 and 9.6 us a KiB.  A turn
// of tiles takes 1.5 us besides, and a unit stores its results at 20 bytes a ns.
struct Rate { float first, other; };
struct Form { uint32_t rows, cols; const char *name; Rate along[2], across[2], any[2]; };
constexpr Form kForms[] = {
    {32, 32, "gated-32x32", {{1.4f, 1.4f}, {2.6f, 2.1f}}, {{1.1f, 1.2f}, {2.4f, 2.2f}}, {}},
    {32, 64, "gated-32x64", {{1.6f, 1.4f}, {2.8f, 2.1f}}, {{1.6f, 1.2f}, {2.7f, 2.4f}}, {}},
    {64, 64, "gated-64x64", {{1.9f, 1.4f}, {4.6f, 3.9f}}, {{2.3f, 1.3f}, {4.8f, 4.1f}}, {{3.2f, 1.2f}, {5.7f, 3.7f}}},
    {64, 128, "gated-64x128", {{2.8f, 2.3f}, {9.4f, 7.8f}}, {{3.6f, 2.1f}, {10.5f, 8.2f}}, {}},
    {128, 128, "gated-128x128", {{5.7f, 4.6f}, {18.0f, 15.5f}}, {{4.8f, 3.2f}, {16.2f, 15.1f}}, {{6.5f, 4.2f}, {18.8f, 14.5f}}},
    {256, 256, "gated-256x256", {{13.0f, 13.0f}, {}}, {{11.5f, 11.6f}, {}}, {}},
};
constexpr int kFormCount = 6;

// How a result of `rows` x `cols` is made of `terms` products of `depth` each: the tile, and in how many pieces; what takes least by the rates above.  Not half of a tile's
// columns would do: fewer of the weights' rows a workgroup keep more of them on their way (24 columns of 8192 x 4096 fp16: 32 x 32 27 us, 64 x 64 33).  The pieces' sums are written and read at 4 TB/s, by a launch of 3 us.
struct Plan {
    bool direct;
    int form;
    uint32_t cuts, depth;
    size_t pitch, bytes;             // of the pieces in the workspace, 0: none
    Pieces pieces(void *at) const { return {bytes ? (float *)at : nullptr, cuts, depth, pitch}; }
};
Plan plan_of(const so_ctx *ctx, int type, bool direct, uint64_t rows, uint32_t cols, uint32_t terms, uint32_t depth)
{
    Plan p = {direct, 2, 1, depth, (cols + 7u) / 8u * (size_t)8, 0};
    const uint32_t size = (uint32_t)so_type_bytes(type), units = (uint32_t)ctx->compute_units;
    const float length = (float)terms * (float)depth * (float)size / 1024.0f;
    const int forced = ctx->tune.gated_form < 1 || ctx->tune.gated_form > kFormCount ? -1 : std::min(ctx->tune.gated_form - 1, size == 4 ? 4 : 5);
    uint32_t pieces = 1;
    float least = INFINITY;
    for (int f = 0; f < kFormCount; ++f) {
        const Rate rate = (!direct ? kForms[f].any : terms == 2 ? kForms[f].across : kForms[f].along)[size / 4u];
        if (rate.first == 0.0f || (direct && (forced >= 0 ? f != forced : f && cols <= kForms[f].cols / 2))) continue;
        const uint64_t tiles = (uint64_t)so_ceil_div(rows, kForms[f].rows) * so_ceil_div(cols, kForms[f].cols);
        // pieces of a KiB at least, as long as there are fewer than three for every unit
        for (uint32_t n = 1; n <= 32 && (n == 1 || ((float)n <= length && tiles * n < 3ull * units && f < 5)); n += n < terms ? terms - n : terms) {
            const float turns = (float)((tiles * n + units - 1) / units);
            const float results = (float)(kForms[f].rows * kForms[f].cols) * (n > 1 ? 4.0f : (float)size);
            const float time = (rate.first + (turns - 1.0f) * rate.other) * length / (float)n + turns * (1.5f + results / 20000.0f) + (n > 1 ? 3.0f + (float)n * (0.25f + (float)rows * (float)p.pitch * 2e-6f) : 0.0f);
            if (time < least) {
                least = time;
                p.form = f;
                pieces = n;
            }
        }
    }
    if (pieces == 1) return p;
    const uint64_t step = 256u / size;                                   // whole steps of the smallest tile
    p.depth = (uint32_t)std::min<uint64_t>(so_ceil_div(so_ceil_div(depth, pieces / terms), step) * step, depth);
    p.cuts = so_ceil_div(depth, p.depth);
    p.bytes = (uint64_t)p.cuts * terms * rows * p.pitch * sizeof(float);
    return p;
}

// f(a tile, whether operands go past the registers)
template <class T, class F>
so_status for_tile(so_ctx *ctx, const Plan &p, F &&f)
{
    ctx->last_kernel = kForms[p.form].name;
    if (!p.direct) {
        ctx->last_kernel = p.form == 4 ? "gated-128x128-any" : "gated-64x64-any";
        return p.form == 4 ? f(T128x128(), std::false_type()) : f(T64x64(), std::false_type());
    }
    switch (p.form) {
    case 0: return f(T32x32(), std::true_type());
    case 1: return f(T32x64(), std::true_type());
    case 2: return f(T64x64(), std::true_type());
    case 3: return f(T64x128(), std::true_type());
    case 4: return f(T128x128(), std::true_type());
    default:
        if constexpr (sizeof(T) == 2) return f(T256x256(), std::true_type());
        return SO_ERR_INVALID;
    }
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

so_status workspace(so_ctx *ctx, const char *who, size_t bytes)
{
    SO_REQUIRE(!ctx->capturing || (ctx->mm_part && ctx->mm_part->bytes >= bytes),
               "%s: the context's workspace must grow, which cannot be done while a graph is being recorded (call so_gated_reserve, or launch this shape once, before recording)", who);
    return so_matmul_workspace(ctx, bytes, 4);
}

// Bytes of a matrix in the workspace, its rows at multiples of 16 bytes.
size_t stride_of(uint32_t cols) { return (cols + 7u) / 8u * (size_t)8; }
size_t bytes_of(int type, uint32_t rows, uint32_t cols) { return rows * stride_of(cols) * so_type_bytes(type); }
template <class T> bool direct_there(uint32_t cols) { return Operand<T>{nullptr, stride_of(cols), 0, 0}.direct(); }

template <class T> uint64_t blocks_of(uint32_t rows, uint32_t groups) { return ((uint64_t)rows * groups + kThreads - 1) / kThreads; }

template <class T, bool AX, bool BX>
so_status product(so_ctx *ctx, const Product<T> &p, const Plan &plan)
{
    const uint32_t parts = p.Y2 ? 2 : 1;
    const so_status status = for_tile<T>(ctx, plan, [&](auto t, auto past) {
        typedef decltype(t) TILE;
        return launch_tiles<TILE>(ctx, "so_gated_grad", product_kernel<T, TILE, AX, BX, decltype(past)::value>, p,
                                  (uint64_t)(plan.bytes ? p.terms * plan.cuts : 1u) * parts * so_ceil_div(p.rows, TILE::ROWS), so_ceil_div(p.cols, TILE::COLS));
    });
    if (status != SO_OK || !plan.bytes) return status;
    const uint32_t groups = so_ceil_div(p.cols, so_elements<T>::V);
    const uint64_t blocks = ((uint64_t)parts * p.rows * groups + kThreads - 1) / kThreads;
    SO_REQUIRE(so_grid_fits(blocks, kThreads), "so_gated_grad: the result is too large for one launch");
    product_join_kernel<T><<<(uint32_t)blocks, kThreads, 0, ctx->stream>>>(p, groups, parts);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

// *m as what it is in the workspace at `to`, aligned; -> what makes it that.
template <class T>
Rows<T> align_rows(Operand<T> *m, uint32_t rows, uint32_t cols, void *to)
{
    const uint32_t groups = so_ceil_div(cols, so_elements<T>::V);
    const Rows<T> r = {m->p, m->ld, rows, cols, groups, (uint32_t)blocks_of<T>(rows, groups), (T *)to, stride_of(cols)};
    m->p = (const T *)to;
    m->ld = stride_of(cols);
    return r;
}
template <class T> bool align_fits(uint32_t rows, uint32_t cols) { return so_grid_fits(blocks_of<T>(rows, so_ceil_div(cols, so_elements<T>::V)), kThreads); }

template <class T>
so_status slopes(so_ctx *ctx, Slopes<T> s, const Rows<T> &x)
{
    s.groups = so_ceil_div(s.B, so_elements<T>::V);
    const uint64_t blocks = blocks_of<T>(s.m, s.groups);
    SO_REQUIRE(so_grid_fits(blocks + x.blocks, kThreads), "so_gated_grad: %u x %u is too large for one launch", s.m, s.B);
    gated_slopes_kernel<T><<<(uint32_t)blocks + x.blocks, kThreads, 0, ctx->stream>>>(s, x);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

template <class T>
so_status forward(so_ctx *ctx, int type, Forward<T> f)
{
    if (f.B == 1) {
        // four rows a wave where that leaves every compute unit eight waves: X is read once for them
        const uint32_t waves = 8u * (uint32_t)ctx->compute_units, rows = f.m / 4u >= waves ? 4u : f.m / 2u >= waves ? 2u : 1u, blocks = so_ceil_div(f.m, rows * (kThreads / 64));
        SO_REQUIRE(so_grid_fits(blocks, kThreads), "so_gated: %u rows are too many for one launch", f.m);
        const auto kernel = rows == 4 ? gated_token_kernel<T, 4> : rows == 2 ? gated_token_kernel<T, 2> : gated_token_kernel<T, 1>;
        ctx->last_kernel = "gated-token";
        kernel<<<blocks, kThreads, 0, ctx->stream>>>(f);
        SO_LAUNCH_CHECK();
        return SO_OK;
    }
    const Operand<T> g = {f.Wg, f.ldw, f.m, f.n}, u = {f.Wu, f.ldw, f.m, f.n};
    Operand<T> x = {f.X, f.ldx, f.B, f.n};
    const bool align = g.direct() && u.direct() && !x.direct() && direct_there<T>(f.B);
    const Plan plan = plan_of(ctx, type, g.direct() && u.direct() && (align || x.direct()), 2 * (uint64_t)f.m, f.B, 1, f.n);
    const size_t aligned = align ? bytes_of(type, f.n, f.B) : 0;
    if (align || plan.bytes)
        if (const so_status s = workspace(ctx, "so_gated", aligned + plan.bytes); s != SO_OK) return s;
    if (align) {
        SO_REQUIRE(align_fits<T>(f.n, f.B), "so_gated: %u x %u is too large for one launch", f.n, f.B);
        const Rows<T> r = align_rows(&x, f.n, f.B, ctx->mm_part->p);
        align_rows_kernel<T><<<r.blocks, kThreads, 0, ctx->stream>>>(r);
        SO_LAUNCH_CHECK();
        f.X = x.p;
        f.ldx = x.ld;
    }
    f.pieces = plan.pieces(plan.bytes ? (char *)ctx->mm_part->p + aligned : nullptr);
    const so_status status = for_tile<T>(ctx, plan, [&](auto t, auto past) {
        typedef decltype(t) TILE;
        return launch_tiles<TILE>(ctx, "so_gated", gated_kernel<T, TILE, decltype(past)::value>, f, (uint64_t)plan.cuts * so_ceil_div(f.m, TILE::ROWS / 2), so_ceil_div(f.B, TILE::COLS));
    });
    if (status != SO_OK || !plan.bytes) return status;
    const uint32_t groups = so_ceil_div(f.B, so_elements<T>::V);
    const uint64_t blocks = blocks_of<T>(f.m, groups);
    SO_REQUIRE(so_grid_fits(blocks, kThreads), "so_gated: %u x %u is too large for one launch", f.m, f.B);
    gated_join_kernel<T><<<(uint32_t)blocks, kThreads, 0, ctx->stream>>>(f, groups);
    SO_LAUNCH_CHECK();
    return SO_OK;
}

// The three gradients from dG and dU, either of which may have to go to the caller too.
struct Gradients {
    void *dX, *dWg, *dWu;
    size_t ldx, ldw;
};
template <class T>
so_status backward(so_ctx *ctx, int type, Slopes<T> s, uint32_t n, const Operand<T> (&W)[2], Operand<T> x, const Gradients &r)
{
    const uint32_t m = s.m, B = s.B;
    const bool weights = r.dWg || r.dWu, products = r.dX || weights;
    so_status status = SO_OK;
    Operand<T> d[2] = {{s.to[0].g, s.to[0].ld, B, m}, {s.to[0].u, s.to[0].ld, B, m}};
    const uint32_t parts = r.dWg && r.dWu ? 2u : 1u;
    const bool to_workspace = products && !(s.to[0].g && s.to[0].u && d[0].direct() && d[1].direct()), align = weights && !x.direct() && direct_there<T>(B);
    const bool direct = to_workspace ? direct_there<T>(B) : d[0].direct() && d[1].direct();
    const Plan dx = plan_of(ctx, type, direct && W[0].direct() && W[1].direct(), n, B, 2, m);
    const Plan dw = plan_of(ctx, type, direct && (align || x.direct()), (uint64_t)parts * m, n, 1, B);
    char *pieces = nullptr;
    Rows<T> rows = {};
    if (m && B) {
        const size_t each = to_workspace ? bytes_of(type, m, B) : 0, aligned = align ? bytes_of(type, n, B) : 0;
        const size_t bytes = 2 * each + aligned + std::max(r.dX ? dx.bytes : 0, weights ? dw.bytes : 0);
        if (bytes) {
            if ((status = workspace(ctx, "so_gated_grad", bytes)) != SO_OK) return status;
            char *at = (char *)ctx->mm_part->p;
            if (to_workspace) {
                s.to[1] = {(T *)at, (T *)(at + each), stride_of(B)};
                for (int i = 0; i < 2; ++i) d[i] = {(const T *)(at + i * each), stride_of(B), B, m};
            }
            SO_REQUIRE(!align || align_fits<T>(n, B), "so_gated_grad: %u x %u is too large for one launch", n, B);
            if (align) rows = align_rows(&x, n, B, at + 2 * each);
            pieces = at + 2 * each + aligned;
        }
        if ((status = slopes(ctx, s, rows)) != SO_OK) return status;
    }
    if (r.dX && B) status = product<T, true, true>(ctx, {{W[0], W[1]}, {d[0], d[1]}, (T *)r.dX, nullptr, r.ldx, n, B, 2, dx.pieces(pieces)}, dx);
    if (status != SO_OK || !weights || !m) return status;
    const Operand<T> along = {x.p, x.ld, n, B}, g = {d[0].p, d[0].ld, m, B}, u = {d[1].p, d[1].ld, m, B};
    if (parts == 2) return product<T, false, false>(ctx, {{g, u}, {along, along}, (T *)r.dWg, (T *)r.dWu, r.ldw, m, n, 1, dw.pieces(pieces)}, dw);
    return product<T, false, false>(ctx, {{r.dWg ? g : u, u}, {along, along}, (T *)(r.dWg ? r.dWg : r.dWu), nullptr, r.ldw, m, n, 1, dw.pieces(pieces)}, dw);
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
    size_t pieces = 0;
    for (const bool direct : {false, true}) {
        pieces = std::max(pieces, plan_of(ctx, type, direct, 2 * (uint64_t)m, B, 1, n).bytes);
        pieces = std::max(pieces, plan_of(ctx, type, direct, n, B, 2, m).bytes);
        for (const uint64_t rows : {(uint64_t)m, 2 * (uint64_t)m}) pieces = std::max(pieces, plan_of(ctx, type, direct, rows, n, 1, B).bytes);
    }
    return workspace(ctx, "so_gated_reserve", 2 * bytes_of(type, m, B) + bytes_of(type, n, B) + pieces);
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
        status = forward<T>(ctx, type, {(const T *)dWg, (const T *)dWu, (const T *)dX, (const T *)dG0, (const T *)dU0, (T *)dH, (T *)dG, (T *)dU, w_stride, x_stride, g0_stride, h_stride, g_stride,
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
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
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
        status = backward<T>(ctx, type, {(const T *)dG, (const T *)dU, (const T *)dDh, g_stride, dh_stride, m, B, 0, act, {{(T *)dDg, (T *)dDu, dg_stride}, {nullptr, nullptr, 0}}}, n,
                             {{(const T *)dWg, w_stride, n, m}, {(const T *)dWu, w_stride, n, m}}, {(const T *)dX, x_stride, n, B}, {dDx, dDwg, dDwu, dx_stride, dw_stride});
    });
    return status;
}
