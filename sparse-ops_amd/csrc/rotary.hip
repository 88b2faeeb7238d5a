// Rotary positions of queries and keys, with a norm of every head ahead of them, and the gradient.
#include "layer_norm.h"

namespace {

constexpr uint32_t kMostFeatures = 512;

struct Shape {
    uint32_t heads_q, heads, D, B, rot;
    int pairs;                          // SO_ROTARY_PAIRS
    uint32_t tiles, per, groups_q, groups;      // tiles of columns; heads of a workgroup; groups of them, first the queries'
    uint32_t strip;                             // tiles of an XCD, 0: as they come
    uint32_t blocks() const { return (strip ? 8u * strip : tiles) * groups; }
};

// The rows of a head that a thread holds: pair p is two features that are turned together, or two neighbours of those behind them.
__device__ __forceinline__ uint2 rows_of(const Shape &s, uint32_t p)
{
    const uint32_t half = s.rot / 2u;
    if (p >= half) return make_uint2(s.rot + 2u * (p - half), s.rot + 2u * (p - half) + 1u);
    return s.pairs ? make_uint2(2u * p, 2u * p + 1u) : make_uint2(p, p + half);
}

// cos and sin of pos * freq, times the amplitude.  The turns pos * freq / (2 pi) are rounded three times in fp64, the constant among them, by 2^-53 of themselves at most each, and the whole ones are taken off there: an
// angle is off by |pos freq| 2^-54 turns at most, less than fp32 can tell (2^-25 of a turn) up to |pos freq| = 2^29, and by 2^-23 of a turn at a position of 2^31 and a frequency of 1.  Frequencies above 1 are taken, and
// cost in proportion.  For results of 16 bits the vector unit's sine and cosine of what is left do: over half a turn to either side they are off by 2^-22.9 at most.
template <bool HALF>
__device__ __forceinline__ float2 turn_of(int32_t pos, double turns, float amplitude)
{
    const double t = (double)pos * turns;
    const float left = (float)(t - rint(t));
    float c, s;
    if constexpr (HALF) {
        c = __builtin_amdgcn_cosf(left);
        s = __builtin_amdgcn_sinf(left);
    } else {
        sincospif(2.0f * left, &s, &c);
    }
    return make_float2(amplitude * c, amplitude * s);
}

// 1 / sqrt(v), also where v is below the least normal number, which the vector unit takes for 0
__device__ __forceinline__ float inverse_root(float v)
{
    const bool small = v < 0x1p-100f;
    return __builtin_amdgcn_rsqf(small ? v * 0x1p100f : v) * (small ? 0x1p50f : 1.0f);
}

constexpr double kTurnsPerRadian = 0.15915494309189533577;

// y = turn(gain * x * rstd), rstd = 1 / sqrt(mean(x^2) + eps) of a head's D features; turn takes (u, v) to (u cos - v sin, v cos + u sin).  One read and one write of every element: memory bounds
// it.  32 + 8 heads of 128 x 8192 bf16, 168 MB, take 38.6 us or 4.4 TB/s (a layer norm of as many bytes runs at 3.9); one column 4.8 us, a launch.  With fp64 multiples and the library's sine for
// every type it was 50 us, and with two pairs a thread and 256 threads, of 136 registers, 45.
// What forward pass and gradient share: a workgroup of NT threads takes LC * V columns of `per` heads, one after the other; a thread PPT pairs of a head's features, for which it keeps the turns of its columns.
template <class T, int LC, int PPT, int NT>
struct Seat {
    static constexpr int V = so_elements<T>::V, RL = NT / LC;
    typedef typename so_elements<T>::plain group;
    uint32_t at, tile, c0, left, first, last, wide; // its number; columns; heads first .. last - 1
    bool query;
    uint2 row[PPT];                                 // inside a head
    bool has[PPT], two[PPT], turned[PPT];
    __device__ __forceinline__ Seat(const Shape &s, size_t ld)
    {
        // Workgroups go round-robin to the 8 XCDs.  With strips neighbouring tiles, which share the lines of memory that rows' tiles end in, are on the same one: the gradient of 24 + 8 heads of 96 x 4099 fp16 with neighbours on
        // different ones reads 98 MB instead of 50 and takes 30.6 us instead of 26.8.
        const uint32_t in = s.strip ? blockIdx.x / 8u : blockIdx.x, wide_of = s.strip ? s.strip : s.tiles, g = in / wide_of;
        tile = in % wide_of + (s.strip ? blockIdx.x % 8u * s.strip : 0u);
        at = g * s.tiles + tile;
        query = g < s.groups_q;
        first = query ? g * s.per : s.heads_q + (g - s.groups_q) * s.per;
        last = min(first + s.per, query ? s.heads_q : s.heads);
        const uint64_t c = (uint64_t)tile * (LC * V) + threadIdx.x % LC * V;
        left = c >= s.B ? 0u : (uint32_t)min((uint64_t)s.B - c, (uint64_t)V);
        c0 = (uint32_t)c;
        wide = so_group_wide_rows<T>(left, s.heads * s.D, ld);
#pragma unroll
        for (int k = 0; k < PPT; ++k) {
            row[k] = rows_of(s, threadIdx.x / LC + k * RL);
            has[k] = left && row[k].x < s.D;
            two[k] = left && row[k].y < s.D;
            turned[k] = threadIdx.x / LC + k * RL < s.rot / 2u;
        }
    }
    __device__ __forceinline__ void turns(const Shape &s, const int32_t *pos, const float *freq, float amplitude, float2 (&t)[PPT][V]) const
    {
        int32_t p[V];
#pragma unroll
        for (int e = 0; e < V; ++e) p[e] = s.rot && (uint32_t)e < left ? pos[c0 + e] : 0;
#pragma unroll
        for (int k = 0; k < PPT; ++k) {
            const uint32_t i = threadIdx.x / LC + k * RL;
            const double f = turned[k] ? (double)freq[i] * kTurnsPerRadian : 0.0;
#pragma unroll
            for (int e = 0; e < V; ++e) t[k][e] = turned[k] ? turn_of<sizeof(T) == 2>(p[e], f, amplitude) : make_float2(1.0f, 0.0f);
        }
    }
    __device__ __forceinline__ void load(const Shape &s, uint32_t head, const T *X, size_t ld, group (&x)[PPT][2]) const
    {
#pragma unroll
        for (int k = 0; k < PPT; ++k) {
            const uint32_t r0 = head * s.D + row[k].x, r1 = head * s.D + row[k].y;
            x[k][0] = group{};
            x[k][1] = group{};
            if (has[k]) x[k][0] = so_group_load(X + (size_t)r0 * ld + c0, left, r0 < wide);
            if (two[k]) x[k][1] = so_group_load(X + (size_t)r1 * ld + c0, left, r1 < wide);
        }
    }
};

template <class T, int LC, int PPT, int NT, bool NORM>
__global__ __launch_bounds__(NT)
void rotary_kernel(Shape s, const T *X, size_t ldx, const float *gain_q, const float *gain_k, float eps, const int32_t *pos, const float *freq, float amplitude, float direction, T *Y, size_t ldy,
                   float *rstd)
{
    constexpr int V = so_elements<T>::V;
    __shared__ float lds[(NT / 64 + 1) * LC * V];
    const Seat<T, LC, PPT, NT> at(s, ldx);
    if (at.tile >= s.tiles) return;
    typename so_elements<T>::plain x[PPT][2], next[PPT][2];
    at.load(s, at.first, X, ldx, x);
    float2 turn[PPT][V];
    at.turns(s, pos, freq, amplitude, turn);
    const float *gain = at.query ? gain_q : gain_k;
    float2 g[PPT];
#pragma unroll
    for (int k = 0; k < PPT; ++k) {
        g[k] = make_float2(1.0f, 1.0f);
        if (NORM && gain && at.has[k]) g[k].x = gain[at.row[k].x];
        if (NORM && gain && at.two[k]) g[k].y = gain[at.row[k].y];
    }
    for (uint32_t head = at.first; head < at.last; ++head) {
        if (head + 1u < at.last) at.load(s, head + 1u, X, ldx, next);
        float r[V];
#pragma unroll
        for (int e = 0; e < V; ++e) r[e] = 0.0f;
        if constexpr (NORM) {
#pragma unroll
            for (int k = 0; k < PPT; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) r[e] = fmaf((float)x[k][1][e], (float)x[k][1][e], fmaf((float)x[k][0][e], (float)x[k][0][e], r[e]));
            so_norm::sum_tile<NT, LC, V>(r, lds);
#pragma unroll
            for (int e = 0; e < V; ++e) r[e] = inverse_root(fmaf(r[e], 1.0f / (float)s.D, eps));
            if (rstd && threadIdx.x < LC)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if ((uint32_t)e < at.left) rstd[(size_t)head * s.B + at.c0 + e] = r[e];
        }
#pragma unroll
        for (int k = 0; k < PPT; ++k) {
            float a[V], b[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float u = NORM ? (float)x[k][0][e] * r[e] * g[k].x : (float)x[k][0][e], v = NORM ? (float)x[k][1][e] * r[e] * g[k].y : (float)x[k][1][e];
                const float c = turn[k][e].x, d = direction * turn[k][e].y;
                a[e] = at.turned[k] ? fmaf(u, c, -(v * d)) : u;      // not a turn by nothing, which would make NaN of what lies beside an infinity
                b[e] = at.turned[k] ? fmaf(v, c, u * d) : v;
            }
            if (at.has[k]) so_group_store(Y + (size_t)(head * s.D + at.row[k].x) * ldy + at.c0, at.left, a);
            if (at.two[k]) so_group_store(Y + (size_t)(head * s.D + at.row[k].y) * ldy + at.c0, at.left, b);
        }
#pragma unroll
        for (int k = 0; k < PPT; ++k) x[k][0] = next[k][0], x[k][1] = next[k][1];
    }
}

// With norms: h = turn^-1(dY); dX = rstd (gain h - n mean(gain h n)), n = x rstd, and of every workgroup its share of the gains' gradients sum(h n), [tiles * groups][D], which the kernel below adds
// up in a fixed order.  24 + 8 heads of 96 x 4099 fp16, 75 MB: 25.9 us and 4.7 for the shares; with the next head in registers ahead, which leaves one workgroup a compute unit, 47, and with h
// kept instead of turned back again after the sum, 38.
template <class T, int LC, int PPT, int NT>
__global__ __launch_bounds__(NT, PPT == 1 ? 4 : 1)
void rotary_grad_kernel(Shape s, const T *X, size_t ldx, const T *dY, size_t ldd, const float *gain_q, const float *gain_k, const float *rstd, const int32_t *pos, const float *freq, float amplitude,
                        T *dX, size_t ldo, float *shares)
{
    constexpr int V = so_elements<T>::V;
    typedef typename so_elements<T>::plain group;
    __shared__ float lds[(NT / 64 + 1) * LC * V];
    const Seat<T, LC, PPT, NT> at(s, ldx);
    if (at.tile >= s.tiles) return;
    const uint32_t wide_d = so_group_wide_rows<T>(at.left, s.heads * s.D, ldd);
    Seat<T, LC, PPT, NT> of_dy = at;
    of_dy.wide = wide_d;
    float2 turn[PPT][V];
    at.turns(s, pos, freq, amplitude, turn);
    const float *gain = at.query ? gain_q : gain_k;
    float2 g[PPT], sum[PPT];
#pragma unroll
    for (int k = 0; k < PPT; ++k) {
        g[k] = make_float2(1.0f, 1.0f);
        sum[k] = make_float2(0.0f, 0.0f);
        if (gain && at.has[k]) g[k].x = gain[at.row[k].x];
        if (gain && at.two[k]) g[k].y = gain[at.row[k].y];
    }
    for (uint32_t head = at.first; head < at.last; ++head) {
        group x[PPT][2], d[PPT][2];
        at.load(s, head, X, ldx, x);
        of_dy.load(s, head, dY, ldd, d);
        float r[V];
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const float *from = rstd + (size_t)head * s.B + at.c0 + e;
            const auto w = so_group_load(from, at.left > (uint32_t)e ? at.left - e : 0u, at.left >= e + 4u);
#pragma unroll
            for (int j = 0; j < 4; ++j) r[e + j] = w[j];
        }
        float dot[V];
#pragma unroll
        for (int e = 0; e < V; ++e) dot[e] = 0.0f;
        // the gradients of the products, turned back
        const auto back = [&](int k, int e) {
            const float u = (float)d[k][0][e], v = (float)d[k][1][e];
            if (!at.turned[k]) return make_float2(u, v);
            return make_float2(fmaf(u, turn[k][e].x, v * turn[k][e].y), fmaf(v, turn[k][e].x, -(u * turn[k][e].y)));
        };
#pragma unroll
        for (int k = 0; k < PPT; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 y = back(k, e);
                const float p = y.x * ((float)x[k][0][e] * r[e]), q = y.y * ((float)x[k][1][e] * r[e]);
                if ((uint32_t)e < at.left) {
                    sum[k].x += p;
                    sum[k].y += q;
                }
                dot[e] += fmaf(p, g[k].x, q * g[k].y);
            }
        if (!dX) continue;
        so_norm::sum_tile<NT, LC, V>(dot, lds);
#pragma unroll
        for (int k = 0; k < PPT; ++k) {
            for (int i = 0; i < 2; ++i) so_group_afresh(x[k][i]), so_group_afresh(d[k][i]);      // converted again: the fp32 values would take 32 registers a pair
            float p[V], q[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 y = back(k, e);
                const float mean = dot[e] * (1.0f / (float)s.D);
                p[e] = r[e] * fmaf(y.x, g[k].x, -(((float)x[k][0][e] * r[e]) * mean));
                q[e] = r[e] * fmaf(y.y, g[k].y, -(((float)x[k][1][e] * r[e]) * mean));
            }
            if (at.has[k]) so_group_store(dX + (size_t)(head * s.D + at.row[k].x) * ldo + at.c0, at.left, p);
            if (at.two[k]) so_group_store(dX + (size_t)(head * s.D + at.row[k].y) * ldo + at.c0, at.left, q);
        }
    }
    if (!shares) return;
#pragma unroll
    for (int k = 0; k < PPT; ++k) {
        const float p = so_norm::sum_lanes<LC>(sum[k].x), q = so_norm::sum_lanes<LC>(sum[k].y);
        if (threadIdx.x % LC == 0) {                                 // the first of a row's lanes: its columns exist where any do
            if (at.has[k]) shares[(size_t)at.at * s.D + at.row[k].x] = p;
            if (at.two[k]) shares[(size_t)at.at * s.D + at.row[k].y] = q;
        }
    }
}

// The shares of the queries' workgroups and of the keys' to one gradient each: 16 features a workgroup, 16 runs of shares, eight of a run on their way at a time (one at a time: 25 us for 455).
__global__ __launch_bounds__(256)
void rotary_gains_kernel(uint32_t D, uint32_t shares_q, uint32_t shares, uint32_t blocks, const float *from, float *gain_q, float *gain_k)
{
    __shared__ float sums[16][17];
    const bool query = blockIdx.x < blocks;
    float *out = query ? gain_q : gain_k;
    const uint32_t d = blockIdx.x % blocks * 16u + threadIdx.x % 16u, run = threadIdx.x / 16u, end = query ? shares_q : shares;
    float s = 0.0f;
    if (d < D)
        for (uint32_t p = (query ? 0u : shares_q) + run; p < end; p += 128u) {
            float v[8];                                                  // eight on their way at a time
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) v[i] = p + i * 16u < end ? from[(size_t)(p + i * 16u) * D + d] : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
    sums[run][threadIdx.x % 16u] = s;
    __syncthreads();
    if (run || d >= D || !out) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sums[i][threadIdx.x];
    out[d] = s;
}

// Lanes of a row and threads, and the pairs of a thread: 32 lanes down a head of up to 64 features, 64 of one of up to 256, 128 of a larger one, 64 where a row is one group.
struct Cut { uint32_t lanes, threads, pairs; };
Cut cut_of(int type, uint32_t D, uint32_t B)
{
    const uint32_t V = 16u / (uint32_t)so_type_bytes(type), pairs = (D + 1u) / 2u;
    Cut c;
    c.lanes = B <= V ? 1 : pairs > 128 ? 4 : B <= 2 * V ? 2 : B <= 4 * V ? 4 : 8;
    c.threads = c.lanes == 1 ? 64 : pairs > 128 ? 512 : (pairs > 32 ? 64 : 32) * c.lanes;
    const uint32_t each = so_ceil_div(pairs, c.threads / c.lanes);
    c.pairs = each <= 1 ? 1 : each <= 2 ? 2 : 4;
    return c;
}

Shape shape_of(const so_ctx *ctx, const Cut &c, int type, uint32_t heads_q, uint32_t heads_k, uint32_t D, uint32_t B, uint32_t rot, int layout)
{
    Shape s = {heads_q, heads_q + heads_k, D, B, rot, layout == SO_ROTARY_PAIRS, 0, 1, 0, 0, 0};
    s.tiles = so_ceil_div(B, c.lanes * (16u / (uint32_t)so_type_bytes(type)));
    // The turns are worked out once for all heads of a workgroup, and the next head is on its way while one is turned: as many heads a workgroup as all there are, dealt to two workgroups of 512
    // threads on every compute unit.  32 + 8 heads of 128 x 8192 bf16, 10 a workgroup: 38.6 us; 5: 43; 2: 45; 20: 45.  The gradient of 24 + 8 heads of 96 x 4099 fp16, 5 a workgroup: 33 us (27.7 with strips); 4: 37;
    // 1: 43; 10: 39.
    const uint64_t room = (uint64_t)ctx->compute_units * (1024u / c.threads);
    s.per = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(((uint64_t)s.tiles * s.heads + room - 1u) / room, s.heads));
    s.groups_q = so_ceil_div(heads_q, s.per);
    s.groups = s.groups_q + so_ceil_div(heads_k, s.per);
    return s;
}

// Of many tiles each XCD gets a strip, where rows do not all begin at a line of memory of 128 bytes; where they do, as they come: 38.6 us of rotary positions of 32 + 8 heads of 128 x 8192 bf16, in strips 40.7.
void place(Shape &s, int type, std::initializer_list<const void *> arrays, std::initializer_list<size_t> strides)
{
    uint64_t bits = 0;
    for (const void *p : arrays) bits |= (uintptr_t)p;
    for (const size_t n : strides) bits |= n * so_type_bytes(type);
    s.strip = bits % 128 && s.tiles >= 64 ? so_ceil_div(s.tiles, 8) : 0;      // fewer would not go to the XCDs evenly
}

size_t share_bytes(const Shape &s) { return (size_t)s.tiles * s.groups * s.D * sizeof(float); }

template <class F>
void for_cut(const Cut &c, F &&f)
{
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const auto with = [&](auto lanes) {
        constexpr int N = decltype(lanes)::value;
        const std::integral_constant<int, 64 * N> threads;
        if (c.threads == 32 * N) f(lanes, one, std::integral_constant<int, 32 * N>());
        else if (c.pairs == 1) f(lanes, one, threads);
        else f(lanes, two, threads);
    };
    if (c.lanes == 1) {
        const std::integral_constant<int, 64> threads;
        if (c.pairs == 1) f(one, one, threads);
        else if (c.pairs == 2) f(one, two, threads);
        else f(one, std::integral_constant<int, 4>(), threads);
    } else if (c.lanes == 2) with(two);
    else if (c.lanes == 8) with(std::integral_constant<int, 8>());
    else if (c.threads == 512) f(std::integral_constant<int, 4>(), two, std::integral_constant<int, 512>());
    else with(std::integral_constant<int, 4>());
}

so_status workspace(so_ctx *ctx, const char *who, size_t bytes)
{
    SO_REQUIRE(!ctx->capturing || (ctx->mm_part && ctx->mm_part->bytes >= bytes),
               "%s: the context's workspace must grow, which cannot be done while a graph is being recorded (call so_head_rotary_reserve, or launch this shape once, before recording)", who);
    return so_matmul_workspace(ctx, bytes, 4);
}

bool launch_fits(const Shape &s, const Cut &c) { return so_grid_fits(((uint64_t)s.tiles + 7) * s.groups, c.threads) && (uint64_t)s.heads * s.D < (1ull << 32); }

} // namespace

#define SO_ROTARY_CHECKS(who)                                                                                               \
    SO_REQUIRE(ctx != nullptr, who ": ctx is null");                                                                        \
    SO_REQUIRE(type >= SO_F32 && type <= SO_BF16, who ": unknown element type %d", type);                                   \
    SO_REQUIRE(D >= 1 && D <= kMostFeatures, who ": %u features a head are not 1 .. %u", D, kMostFeatures);                 \
    SO_REQUIRE((uint64_t)heads_q + heads_k < (1ull << 32) / kMostFeatures, who ": too many heads")

extern "C" so_status so_head_rotary_reserve(so_ctx *ctx, int type, uint32_t heads_q, uint32_t heads_k, uint32_t D, uint32_t B)
{
    SO_ROTARY_CHECKS("so_head_rotary_reserve");
    SO_REQUIRE(!ctx->capturing, "so_head_rotary_reserve: a graph is being recorded");
    if (heads_q + heads_k == 0 || B == 0) return SO_OK;
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    return workspace(ctx, "so_head_rotary_reserve", share_bytes(shape_of(ctx, cut_of(type, D, B), type, heads_q, heads_k, D, B, 0, SO_ROTARY_HALVES)));
}

extern "C" so_status so_head_rotary(so_ctx *ctx, int type, uint32_t heads_q, uint32_t heads_k, uint32_t D, uint32_t B, const void *dX, size_t x_stride, int norm, const float *dGainQ,
                                    const float *dGainK, float eps, const int32_t *dPos, const float *dFreq, uint32_t rot, float amplitude, int layout, void *dY, size_t y_stride, float *dRstd)
{
    SO_ROTARY_CHECKS("so_head_rotary");
    SO_REQUIRE(rot % 2 == 0 && rot <= D, "so_head_rotary: %u features to turn are not an even number of 0 .. %u", rot, D);
    SO_REQUIRE(layout == SO_ROTARY_HALVES || layout == SO_ROTARY_PAIRS, "so_head_rotary: unknown layout %d", layout);
    SO_REQUIRE(!norm || eps >= 0.0f, "so_head_rotary: eps is negative or not a number");
    if (heads_q + heads_k == 0 || B == 0) return SO_OK;
    SO_REQUIRE(dX && dY, "so_head_rotary: null tensor");
    SO_REQUIRE(rot == 0 || (dPos && dFreq), "so_head_rotary: null positions or frequencies");
    SO_REQUIRE(x_stride >= B && y_stride >= B, "so_head_rotary: a stride is shorter than a row");
    SO_REQUIRE(dX != dY || x_stride == y_stride, "so_head_rotary: in place needs one stride");
    SO_REQUIRE(!norm || !dRstd || (dRstd != dX && dRstd != dY), "so_head_rotary: a result is an input, or one array for both results");
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const Cut c = cut_of(type, D, B);
    Shape s = shape_of(ctx, c, type, heads_q, heads_k, D, B, rot, layout);
    place(s, type, {dX, dY}, {x_stride, y_stride});
    SO_REQUIRE(launch_fits(s, c), "so_head_rotary: %u x %u is too large for one launch", s.heads * D, B);
    so_for_type(type, [&](auto t) {
        using T = decltype(t);
        for_cut(c, [&](auto lanes, auto pairs, auto threads) {
            constexpr int LC = decltype(lanes)::value, PPT = decltype(pairs)::value, NT = decltype(threads)::value;
            const auto kernel = norm ? rotary_kernel<T, LC, PPT, NT, true> : rotary_kernel<T, LC, PPT, NT, false>;
            kernel<<<s.blocks(), NT, 0, ctx->stream>>>(s, (const T *)dX, x_stride, dGainQ, dGainK, eps, dPos, dFreq, amplitude, 1.0f, (T *)dY, y_stride, dRstd);
        });
    });
    SO_LAUNCH_CHECK();
    return SO_OK;
}

extern "C" so_status so_head_rotary_grad(so_ctx *ctx, int type, uint32_t heads_q, uint32_t heads_k, uint32_t D, uint32_t B, const void *dX, size_t x_stride, const void *dDy, size_t dy_stride,
                                         int norm, const float *dGainQ, const float *dGainK, const float *dRstd, const int32_t *dPos, const float *dFreq, uint32_t rot, float amplitude,
                                         int layout, void *dDx, size_t dx_stride, float *dDgainQ, float *dDgainK)
{
    SO_ROTARY_CHECKS("so_head_rotary_grad");
    SO_REQUIRE(rot % 2 == 0 && rot <= D, "so_head_rotary_grad: %u features to turn are not an even number of 0 .. %u", rot, D);
    SO_REQUIRE(layout == SO_ROTARY_HALVES || layout == SO_ROTARY_PAIRS, "so_head_rotary_grad: unknown layout %d", layout);
    const bool gains = norm && (dDgainQ || dDgainK), any = heads_q + heads_k > 0 && B > 0;
    if (!gains && (!dDx || !any)) return SO_OK;
    if (any) {
        SO_REQUIRE(dDy && (!norm || dX), "so_head_rotary_grad: null tensor");
        SO_REQUIRE(!norm || dRstd, "so_head_rotary_grad: null factors");
        SO_REQUIRE(rot == 0 || (dPos && dFreq), "so_head_rotary_grad: null positions or frequencies");
        SO_REQUIRE((!norm || x_stride >= B) && dy_stride >= B && (!dDx || dx_stride >= B), "so_head_rotary_grad: a stride is shorter than a row");
        SO_REQUIRE(!dDx || ((dDx != dDy || dx_stride == dy_stride) && (!norm || dDx != dX || dx_stride == x_stride)), "so_head_rotary_grad: in place needs one stride");
    }
    if (gains) {
        SO_REQUIRE(!dDgainQ || dDgainQ != dDgainK, "so_head_rotary_grad: one array for two results");
        for (const void *result : {(const void *)dDgainQ, (const void *)dDgainK})
            SO_REQUIRE(!result || (result != dX && result != dDy && result != dDx && result != dRstd && result != dGainQ && result != dGainK && result != dFreq),
                       "so_head_rotary_grad: a result is an input, or one array for two results");
    }
    const so_on_device on(ctx->device);
    SO_HIP(on.status);
    const Cut c = cut_of(type, D, std::max(B, 1u));
    Shape s = shape_of(ctx, c, type, heads_q, heads_k, D, B, rot, layout);
    place(s, type, {norm ? dX : nullptr, dDy, dDx}, {norm ? x_stride : 0, dy_stride, dDx ? dx_stride : 0});
    SO_REQUIRE(launch_fits(s, c), "so_head_rotary_grad: %u x %u is too large for one launch", s.heads * D, B);
    float *shares = nullptr;
    if (gains && any) {
        if (const so_status st = workspace(ctx, "so_head_rotary_grad", share_bytes(s)); st != SO_OK) return st;
        shares = (float *)ctx->mm_part->p;
    }
    if (any)
        so_for_type(type, [&](auto t) {
            using T = decltype(t);
            for_cut(c, [&](auto lanes, auto pairs, auto threads) {
                constexpr int LC = decltype(lanes)::value, PPT = decltype(pairs)::value, NT = decltype(threads)::value;
                if (norm)
                    rotary_grad_kernel<T, LC, PPT, NT><<<s.blocks(), NT, 0, ctx->stream>>>(s, (const T *)dX, x_stride, (const T *)dDy, dy_stride, dGainQ, dGainK, dRstd, dPos, dFreq,
                                                                                                     amplitude, (T *)dDx, dx_stride, shares);
                else
                    rotary_kernel<T, LC, PPT, NT, false><<<s.blocks(), NT, 0, ctx->stream>>>(s, (const T *)dDy, dy_stride, nullptr, nullptr, 0.0f, dPos, dFreq, amplitude, -1.0f, (T *)dDx,
                                                                                                       dx_stride, nullptr);
            });
        });
    if (gains) {
        const uint32_t blocks = so_ceil_div(D, 16);
        rotary_gains_kernel<<<2 * blocks, 256, 0, ctx->stream>>>(D, s.tiles * s.groups_q, s.tiles * s.groups, blocks, shares, dDgainQ, dDgainK);
    }
    SO_LAUNCH_CHECK();
    return SO_OK;
}
