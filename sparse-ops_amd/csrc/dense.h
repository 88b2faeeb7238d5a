// Products of dense matrices on the matrix cores, in tiles of the result: the operands go to LDS a step of the contraction at a time, in a ring, past the registers where they are aligned.
//
// Y[i][j] = sum_k A(i, k) B(j, k).  An operand's entry (i, k) lies at p[i * ld + k] ("along" the contraction) or at p[k * ld + i] ("across" it), and goes to LDS as it lies.  A lane of
// v_mfma_f32_16x16x32 takes 8 entries in 16 bits that follow one another in k: along, one read of 16 bytes; across, two transposing reads of 4 rows each.  v_mfma_f32_16x16x4_f32 takes one
// entry; which k it stands for is free as long as both operands agree, so that a lane's four reads along are one of 16 bytes: lanes 16 g .. hold k = 4 g + s in instruction s.
#pragma once
#include <type_traits>

#include "elements.h"
#include "so_internal.h"

namespace so_dense {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// acc += B A^T for 16 columns and 16 rows over 64 bytes of k: a lane gets row l % 16 and columns 4 (l / 16) .. + 3.
template <class T>
__device__ __forceinline__ f32x4 multiply(u32x4 a, u32x4 b, f32x4 acc)
{
    if constexpr (std::is_same<T, float>::value) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(y[s], x[s], acc, 0, 0, 0);
        return acc;
    } else {
        typedef typename so_elements<T>::plain group;
        const group x = __builtin_bit_cast(group, a), y = __builtin_bit_cast(group, b);
        if constexpr (std::is_same<T, __bf16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(y, x, acc, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_f16(y, x, acc, 0, 0, 0);
    }
}

// A matrix as an operand: `own` entries of its own index, `depth` of the contraction.
template <class T> struct Operand {
    const T *p;
    size_t ld;
    uint32_t own, depth;
    // Whether it can go to LDS past the registers: groups of 16 bytes, and the offsets of a step's 256 rows at most in 31 bits.
    bool direct() const { return ((uintptr_t)p | ld * sizeof(T)) % 16 == 0 && (uint64_t)ld * sizeof(T) * 256 < (1ull << 31); }
};

// LEN entries of an operand's own index times KB bytes of the contraction in LDS, brought by WAVES waves.
template <class T, bool ACROSS, int LEN, int KB, int WAVES>
struct Side {
    static constexpr int E = sizeof(T), V = 16 / E, BK = KB / E;
    static constexpr int ROWS = ACROSS ? BK : LEN, PER = ACROSS ? LEN * E / 16 : KB / 16, PITCH = PER * 16;      // rows in LDS, their groups of 16 bytes and bytes
    static constexpr int BYTES = ROWS * PITCH, ASKS = ROWS * PER / 64 / WAVES;                                   // requests of a wave, 64 groups each
    static_assert(ASKS * 64 * WAVES == ROWS * PER, "every wave brings as many groups as the others");

    // A row's groups are exchanged by an exclusive or, so that lanes that read at the same place of neighbouring rows meet in different banks: along, 16 rows of one group (8 of rows of 128 bytes, pairs of rows of 64); across, in 16 bits
    // 16 rows (4 neighbours, of 4 eights) of 32 bytes, in 32 bits 4 rows (each fourth) of 64 bytes.
    static __host__ __device__ __forceinline__ uint32_t swap(uint32_t row)
    {
        if constexpr (!ACROSS) return PER == 16 ? row & 15u : PER == 8 ? row & 7u : row >> 1 & 3u;
        else if constexpr (E == 2) return PER >= 16 ? ((row & 3u) | (row >> 1 & 4u)) << 1 : PER == 8 ? ((row >> 1 & 1u) | (row >> 2 & 2u)) << 1 : PER == 4 ? (row >> 3 & 1u) << 1 : 0u;
        else return PER >= 16 ? (row >> 2 & 3u) << 2 : PER == 8 ? (row >> 2 & 1u) << 2 : 0u;
    }

    const T *at;             // entry (i0, 0)
    size_t ld;
    uint32_t own, depth;     // from i0 on
    uint32_t from[ASKS];     // byte offsets of this lane's groups, of a step
    __device__ __forceinline__ void start(const Operand<T> &m, uint64_t i0)
    {
        at = m.p + (ACROSS ? i0 : i0 * m.ld);
        ld = m.ld;
        own = (uint32_t)(m.own - i0);
        depth = m.depth;
        const uint32_t wave = threadIdx.x / 64u, lane = threadIdx.x % 64u;
#pragma unroll
        for (int a = 0; a < ASKS; ++a) {
            const uint32_t q = (a * WAVES + wave) * 64u + lane, row = q / PER;
            from[a] = row * (uint32_t)(ld * E) + (q % PER ^ swap(row)) * 16u;
        }
    }
    __host__ __device__ __forceinline__ uint32_t steps() const { return depth / BK + (depth % BK ? 1u : 0u); }
    // Whether a step is all there, so that its groups can be read whole.  Across, the group at a row's end holds what lies behind it, entries of no use that nothing depends on: the rows below have to be as many as it
    // reaches into, one where a row's stride is a group at least, seven of a single 16-bit column without gaps.
    __host__ __device__ __forceinline__ bool whole(uint32_t step) const
    {
        const uint64_t end = (uint64_t)(step + 1u) * BK;
        return end <= depth && (!ACROSS || own >= (uint32_t)LEN || own % V == 0 || (depth - end) * ld >= V - own % V);
    }
    // Request `piece` of this wave for such a step, or all of them, straight to LDS at `to`.  Whole rows beyond `own` are kept off by the buffer's size.
    __device__ __forceinline__ void bring(uint32_t step, uint32_t to, int piece) const
    {
        const char *base = reinterpret_cast<const char *>(at) + (ACROSS ? (size_t)step * BK * ld : (size_t)step * BK) * E;
        const uint64_t left = ((uint64_t)(ACROSS ? depth - step * BK - 1u : own - 1u) * ld + (ACROSS ? own : depth - step * BK)) * E;
        const u32x4 buffer = {(uint32_t)(uintptr_t)base, (uint32_t)((uintptr_t)base >> 32) & 0xffffu, (uint32_t)min(left, (uint64_t)0xfffffffcu), 0x00020000u};
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(to + (piece * WAVES + wave) * 1024u), "v"(from[piece]), "s"(buffer) : "memory", "m0");
    }
    __device__ __forceinline__ void bring(uint32_t step, uint32_t to) const
    {
#pragma unroll
        for (int p = 0; p < ASKS; ++p) bring(step, to, p);
    }
    // Group q of any step, to a register: what does not exist is zero.
    __device__ __forceinline__ u32x4 group(uint32_t step, uint32_t q) const
    {
        const uint32_t row = q / PER, group = q % PER ^ swap(row);
        const uint64_t k = (uint64_t)step * BK + (ACROSS ? row : group * V), i = ACROSS ? group * V : row;
        const uint64_t end = ACROSS ? own : depth, along = ACROSS ? i : k;
        if (!((ACROSS ? k < depth : i < own) && along < end)) return u32x4{};
        return __builtin_bit_cast(u32x4, so_group_load(at + (ACROSS ? (size_t)k * ld + i : (size_t)i * ld + k), (uint32_t)min(end - along, (uint64_t)V)));
    }
    static __device__ __forceinline__ uint32_t group_of(uint32_t a) { return (a * WAVES + threadIdx.x / 64u) * 64u + threadIdx.x % 64u; }
    // Where a step begins, from `at` on, and where behind that group q of one that is whole is read.  Rows, or groups of a row, that do not exist are replaced by others that do, for nothing.
    __host__ __device__ __forceinline__ size_t begin(uint32_t step) const { return ACROSS ? (size_t)step * BK * ld : (size_t)step * BK; }
    __host__ __device__ __forceinline__ size_t place(uint32_t q) const
    {
        const uint32_t row = q / PER, group = q % PER ^ swap(row);
        const uint32_t i = ACROSS ? (group * V < own ? group * V : 0u) : (row < own ? row : own - 1u), k = ACROSS ? row : group * V;
        return ACROSS ? (size_t)k * ld + i : (size_t)i * ld + k;
    }
    // The groups of a step that is whole, at any address.
    __device__ __forceinline__ void take(uint32_t step, u32x4 (&r)[ASKS]) const
    {
        const T *from = at + begin(step);
#pragma unroll
        for (int a = 0; a < ASKS; ++a) r[a] = __builtin_bit_cast(u32x4, *reinterpret_cast<const typename so_elements<T>::vec *>(from + place(group_of(a))));
    }
    static __device__ __forceinline__ void put(char *to, const u32x4 (&r)[ASKS])
    {
#pragma unroll
        for (int a = 0; a < ASKS; ++a) *reinterpret_cast<u32x4 *>(to + group_of(a) * 16u) = r[a];
    }
    // One after the other, in as few registers as can be.
    __device__ __forceinline__ void settle(uint32_t step, char *to) const
    {
#pragma unroll 1
        for (uint32_t a = 0; a < ASKS; ++a) *reinterpret_cast<u32x4 *>(to + group_of(a) * 16u) = group(step, group_of(a));
    }

    // What a lane reads of tiles of 16 entries, from tile `first` (a multiple of TILES) on: get(slot, T, Q) is tile first + T's operand of the step's 64-byte run Q.
    template <int TILES>
    struct Reader {
        static_assert((TILES & (TILES - 1)) == 0, "a tile's place differs from the first's in bits of its own");
        uint32_t base[ACROSS ? 1 : KB / 64];
        __device__ __forceinline__ void start(uint32_t first)
        {
            const uint32_t l = threadIdx.x % 16u, g = threadIdx.x % 64u / 16u;
            if constexpr (!ACROSS) {
#pragma unroll
                for (int q = 0; q < KB / 64; ++q) base[q] = (first * 16u + l) * PITCH + ((4u * q + g) ^ swap(l)) * 16u;
            } else {
                const uint32_t row = E == 2 ? 8u * g + l / 4u : 4u * g;
                base[0] = row * PITCH + (first * (E == 2 ? 32u : 64u) ^ swap(row) * 16u) + (E == 2 ? l % 4u * 8u : l * 4u);
            }
        }
        __device__ __forceinline__ u32x4 get(const char *slot, int t, int q) const
        {
            if constexpr (!ACROSS) {
                return *reinterpret_cast<const u32x4 *>(slot + base[q] + t * 16 * PITCH);
            } else if constexpr (E == 2) {
                typedef __attribute__((address_space(3))) s16x4 place;
                const uint32_t p = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)slot + (base[0] ^ t * 32u);
                const s16x4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place *)(p + q * 32 * PITCH)), high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place *)(p + (q * 32 + 4) * PITCH));
                struct Two { s16x4 a, b; } both = {low, high};
                return __builtin_bit_cast(u32x4, both);
            } else {
                u32x4 r;
#pragma unroll
                for (int s = 0; s < 4; ++s) r[s] = *reinterpret_cast<const uint32_t *>(slot + (base[0] ^ t * 64u) + (q * 16 + s) * PITCH);
                return r;
            }
        }
    };
};

// A tile of the result: WM x WC waves of RT x CT tiles of 16 x 16 each, KB bytes of the contraction a step, RING steps in LDS.  With HALVES the rows are those of two operands, half of each wave's
// from either.  TURNED: workgroups begin at different steps, so that they do not all ask for the same places of their rows (and with them for the same channels of the memory) at the same time.
template <int RT_, int CT_, int WM_, int WC_, int KB_, int RING_, bool TURNED_ = false>
struct Tile {
    static constexpr bool TURNED = TURNED_;
    static constexpr int RT = RT_, CT = CT_, WM = WM_, WC = WC_, KB = KB_, RING = RING_, WAVES = WM * WC, THREADS = WAVES * 64, ROWS = RT * WM * 16, COLS = CT * WC * 16;
    static constexpr int OUT_PITCH = CT * 16 + 4;                    // floats of a row on its way out, in a part of LDS of each wave's own: 32 rows of one result, or 16 of two
    static constexpr uint32_t lds = std::max((ROWS + COLS) * KB * RING, WAVES * 32 * OUT_PITCH * 4);
};

template <class T, class TILE, bool AX, bool BX, bool HALVES>
struct Loop {
    static constexpr int RT = TILE::RT, CT = TILE::CT, WM = TILE::WM, WC = TILE::WC, KB = TILE::KB, RING = TILE::RING, WAVES = TILE::WAVES, PARTS = HALVES ? 2 : 1;
    static_assert(!HALVES || (!AX && RT % 2 == 0), "two operands with rows along the contraction");
    typedef Side<T, AX, TILE::ROWS / PARTS, KB, WAVES> SideA;
    typedef Side<T, BX, TILE::COLS, KB, WAVES> SideB;
    static constexpr uint32_t B0 = SideA::BYTES * PARTS, STAGE = B0 + SideB::BYTES;
    static constexpr int ASKS = SideA::ASKS * PARTS + SideB::ASKS;

    f32x4 acc[RT][CT];
    __device__ __forceinline__ Loop()
    {
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int k = 0; k < CT; ++k) acc[i][k] = f32x4{};
    }
    SideA a[PARTS];
    SideB b;
    typename SideA::template Reader<RT> ra;
    typename SideB::template Reader<CT> rb;
    __device__ __forceinline__ void start(const Operand<T> (&A)[PARTS], uint64_t i0, const Operand<T> &B, uint64_t j0)
    {
#pragma unroll
        for (int h = 0; h < PARTS; ++h) a[h].start(A[h], i0);
        b.start(B, j0);
        const uint32_t wave = threadIdx.x / 64u;
        ra.start(wave / WC * (RT / PARTS));
        rb.start(wave % WC * CT);
    }
    __device__ __forceinline__ u32x4 row_tile(const char *slot, int i, int q) const { return ra.get(slot + (HALVES && i >= RT / 2 ? SideA::BYTES : 0), HALVES ? i % (RT / 2) : i, q); }
    struct Taken { u32x4 a[PARTS][SideA::ASKS], b[SideB::ASKS]; };
    __device__ __forceinline__ void take(uint32_t step, Taken &w) const
    {
#pragma unroll
        for (int h = 0; h < PARTS; ++h) a[h].take(step, w.a[h]);
        b.take(step, w.b);
    }
    static __device__ __forceinline__ void put(char *slot, const Taken &w)
    {
#pragma unroll
        for (int h = 0; h < PARTS; ++h) SideA::put(slot + h * SideA::BYTES, w.a[h]);
        SideB::put(slot + B0, w.b);
    }
    __device__ __forceinline__ void settle(uint32_t step, char *slot) const
    {
#pragma unroll
        for (int h = 0; h < PARTS; ++h) a[h].settle(step, slot + h * SideA::BYTES);
        b.settle(step, slot + B0);
    }
    // How many steps are whole: all or all but the last of aligned operands, whose strides are a group at least; else all but the last two at least, since a step has more rows than a group has entries.
    __device__ __forceinline__ uint32_t whole_of(uint32_t steps) const
    {
        uint32_t whole = steps;
        for (int i = 0; i < 2; ++i) whole -= whole && !(a[0].whole(whole - 1u) && b.whole(whole - 1u)) ? 1u : 0u;
        return whole;
    }

    // acc += the product of rows from i0 on (of both operands, with HALVES) and columns from j0 on, both operands aligned.  All steps go straight to LDS, but for a last one that is not whole.
    // A run (64 bytes of k) is multiplied from registers while the next one's operands are read: those of the rows into a second set, those of the columns into the places that have been multiplied
    // for the last time.  Once a step's last run is in registers its place in the ring is free for the step that comes RING later, whose requests go out one by one between the products.
    __device__ __forceinline__ void add_direct(char *stage)
    {
        constexpr int Q = KB / 64;
        static_assert(Q == 1 || Q == 2 || Q == 4, "runs of a step");
        const uint32_t steps = b.steps(), lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)stage;
        const uint32_t whole = whole_of(steps);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");      // what an earlier call has in LDS is read
        if (!steps) return;
        const uint32_t first = TILE::TURNED && whole ? blockIdx.x % whole : 0u;
        const auto nth = [&](uint32_t step) {                            // of the whole steps
            if constexpr (!TILE::TURNED) return step;
            else return step + first >= whole ? step + first - whole : step + first;
        };
        const auto bring_all = [&](uint32_t step) {
#pragma unroll
            for (int h = 0; h < PARTS; ++h) a[h].bring(nth(step), lds0 + step % RING * STAGE + h * SideA::BYTES);
            b.bring(nth(step), lds0 + step % RING * STAGE + B0);
        };
        for (uint32_t s = 0; s < RING && s < whole; ++s) bring_all(s);
        if (whole < steps && whole < RING) settle(whole, stage + whole % RING * STAGE);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
        u32x4 x[2][RT], y[CT];
#pragma unroll
        for (int i = 0; i < RT; ++i) x[0][i] = row_tile(stage, i, 0);
#pragma unroll
        for (int k = 0; k < CT; ++k) y[k] = rb.get(stage + B0, k, 0);
        // Run `run` of a step; SET: which set of the rows' operands it has.  STREAM: the step that comes RING later exists, and all before it.
        const auto multiply_run = [&](uint32_t step, auto run, auto set, auto stream) {
            constexpr int R = decltype(run)::value, SET = decltype(set)::value, NEXT = (R + 1) % Q;
            constexpr bool STREAM = decltype(stream)::value, END = R + 1 == Q;
            if constexpr (END) {
                // the next step is there, and all waves have this one in registers
                if constexpr (STREAM) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(ASKS * (RING - 2)) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
                if constexpr (!STREAM) {
                    if (whole < steps && step + RING == whole) settle(whole, stage + step % RING * STAGE);
                    if (step + RING < whole) bring_all(step + RING);
                }
            }
            const char *next = stage + (END ? step + 1u : step) % RING * STAGE;      // behind the last step: an older one, for nothing
#pragma unroll
            for (int i = 0; i < RT; ++i) x[1 - SET][i] = row_tile(next, i, NEXT);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < CT; ++k) {
#pragma unroll
                for (int i = 0; i < RT; ++i) acc[i][k] = multiply<T>(x[SET][i], y[k], acc[i][k]);
                y[k] = rb.get(next + B0, k, NEXT);
                if constexpr (END && STREAM) {
                    const uint32_t to = lds0 + step % RING * STAGE;
#pragma unroll
                    for (int p = k * ASKS / CT; p < (k + 1) * ASKS / CT; ++p) {
                        if (p < SideA::ASKS * PARTS) a[p / SideA::ASKS].bring(nth(step + RING), to + p / SideA::ASKS * SideA::BYTES, p % SideA::ASKS);
                        else b.bring(nth(step + RING), to + B0, p - SideA::ASKS * PARTS);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const std::integral_constant<int, 0> zero;
        const std::integral_constant<int, 1> one;
        const std::integral_constant<int, 2> two;
        const std::integral_constant<int, 3> three;
        const std::true_type yes;
        const std::false_type no;
        const auto multiply_step = [&](uint32_t step, auto stream) {
            multiply_run(step, zero, zero, stream);
            if constexpr (Q >= 2) multiply_run(step, one, one, stream);
            if constexpr (Q == 4) {
                multiply_run(step, two, zero, stream);
                multiply_run(step, three, one, stream);
            }
        };
        uint32_t s = 0;
        if constexpr (Q > 1) {
            for (; s + RING < whole; ++s) multiply_step(s, yes);
            for (; s < steps; ++s) multiply_step(s, no);
        } else {
            for (; s + 1u + RING < whole; s += 2u) {
                multiply_run(s, zero, zero, yes);
                multiply_run(s + 1u, zero, one, yes);
            }
            for (; s < steps; s += 2u) {
                multiply_run(s, zero, zero, no);
                if (s + 1u < steps) multiply_run(s + 1u, zero, one, no);
            }
        }
    }

    // The same for operands at any address, by way of registers: three steps are on their way there, two in LDS.
    __device__ __forceinline__ void add_any(char *stage)
    {
        const uint32_t steps = b.steps(), whole = whole_of(steps);
        __syncthreads();
        if (!steps) return;
        Taken w[3];
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if ((uint32_t)i < whole) take(i, w[i]);
        const auto compute = [&](uint32_t step) {
            const char *slot = stage + step % 2u * STAGE;
#pragma unroll
            for (int q = 0; q < KB / 64; ++q) {
                u32x4 x[RT], y[CT];
#pragma unroll
                for (int i = 0; i < RT; ++i) x[i] = row_tile(slot, i, q);
#pragma unroll
                for (int k = 0; k < CT; ++k) y[k] = rb.get(slot + B0, k, q);
#pragma unroll
                for (int k = 0; k < CT; ++k)
#pragma unroll
                    for (int i = 0; i < RT; ++i) acc[i][k] = multiply<T>(x[i], y[k], acc[i][k]);
            }
        };
        // Step s from its registers to LDS, the one three later to them; the other half of LDS, which the step before it is read from, is free behind the barrier of the next turn.
        const auto turn = [&](uint32_t s, Taken &own, auto more) {
            put(stage + s % 2u * STAGE, own);
            __syncthreads();
            if constexpr (decltype(more)::value) take(s + 3u, own);
            compute(s);
        };
        uint32_t s = 0;
        for (; s + 5u < whole; s += 3u) {
            turn(s, w[0], std::true_type());
            turn(s + 1u, w[1], std::true_type());
            turn(s + 2u, w[2], std::true_type());
        }
        for (; s < whole; s += 3u) {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (s + i < whole) {
                    put(stage + (s + i) % 2u * STAGE, w[i]);
                    __syncthreads();
                    if (s + i + 3u < whole) take(s + i + 3u, w[i]);
                    compute(s + i);
                }
        }
        for (uint32_t rest = whole; rest < steps; ++rest) {
            settle(rest, stage + rest % 2u * STAGE);
            __syncthreads();
            compute(rest);
        }
    }
    template <bool DIRECT>
    __device__ __forceinline__ void add(char *stage, const Operand<T> (&A)[PARTS], uint64_t i0, const Operand<T> &B, uint64_t j0)
    {
        start(A, i0, B, j0);
        if constexpr (DIRECT) add_direct(stage);
        else add_any(stage);
    }
    // f(i, row, column, values) for each group of V neighbouring results of tile i of the wave's N x RT / N tiles of rows, i running over RT / N, by way of LDS: rows within a tile of 16, columns within the
    // workgroup's; the values of tile i, of tile i + RT / N and so on.  One copy of f's code, whatever RT is.
    template <int N, class F>
    __device__ __forceinline__ void out(char *stage, F &&f) const
    {
        constexpr int V = so_elements<T>::V, PITCH = TILE::OUT_PITCH, LANES = CT * 16 / V, ROWS = 64 / LANES, EACH = RT / N;
        float *mine = reinterpret_cast<float *>(stage) + threadIdx.x / 64u * 32u * PITCH;
        const uint32_t lane = threadIdx.x % 64u;
#pragma unroll 1
        for (int i = 0; i < EACH; ++i) {
#pragma unroll
            for (int t = 0; t < EACH; ++t)
                if (t == i) {
#pragma unroll
                    for (int j = 0; j < N; ++j)
#pragma unroll
                        for (int k = 0; k < CT; ++k) *reinterpret_cast<f32x4 *>(mine + (j * 16 + lane % 16u) * PITCH + k * 16 + 4 * (lane / 16u)) = acc[j * EACH + t][k];
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int r0 = 0; r0 < 16; r0 += ROWS < 16 ? ROWS : 16) {
                const uint32_t r = r0 + lane / LANES;
                float v[N][V];
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < V; e += 4) {
                        const f32x4 s = *reinterpret_cast<const f32x4 *>(mine + (j * 16 + r % 16u) * PITCH + lane % LANES * V + e);
#pragma unroll
                        for (int c = 0; c < 4; ++c) v[j][e + c] = s[c];
                    }
                if (r < 16u) f(i, r, (uint32_t)(threadIdx.x / 64u % WC) * (CT * 16) + lane % LANES * V, v);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
};

// Which tile of the result a workgroup takes.  Workgroups go round-robin to the 8 XCDs; each XCD gets neighbouring tiles of a strip four tiles of columns wide, so that its L2 is asked for few rows of A and
// few columns of B.
struct Grid {
    uint32_t mgroups, cgroups, per_xcd;
    uint32_t groups() const { return per_xcd * 8u; }
};
static inline Grid grid_of(uint64_t mgroups, uint64_t cgroups) { return {(uint32_t)mgroups, (uint32_t)cgroups, so_ceil_div(mgroups * cgroups, 8)}; }
struct Spot { uint32_t m, c; bool none; };
__device__ __forceinline__ Spot spot_of(const Grid &g)
{
    const uint32_t id = (blockIdx.x % 8u) * g.per_xcd + blockIdx.x / 8u;
    if (id >= g.mgroups * g.cgroups) return {0, 0, true};
    const uint32_t strip = id / (4u * g.mgroups), wide = min(4u, g.cgroups - strip * 4u), in = id - strip * 4u * g.mgroups;
    return {in / wide, strip * 4u + in % wide, false};
}

} // namespace so_dense
