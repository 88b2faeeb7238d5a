// Element types of the operators that take more than fp32 (SO_F32, SO_F16, SO_BF16): groups of 16 bytes in memory, fp32 in registers.  A group may start at
// any element: gfx950 loads and stores 16 bytes at any address, so a row stride that is no multiple of a group needs no path of its own.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

#include "sparseops_hip.h"

template <class T> struct so_elements;
template <> struct so_elements<float> {
    static constexpr int V = 4;                                                      // elements of a group
    typedef float plain __attribute__((ext_vector_type(4)));
    typedef plain vec __attribute__((aligned(4)));
};
template <> struct so_elements<_Float16> {
    static constexpr int V = 8;
    typedef _Float16 plain __attribute__((ext_vector_type(8)));
    typedef plain vec __attribute__((aligned(2)));
};
template <> struct so_elements<__bf16> {
    static constexpr int V = 8;
    typedef __bf16 plain __attribute__((ext_vector_type(8)));
    typedef plain vec __attribute__((aligned(2)));
};

static inline size_t so_type_bytes(int type) { return type == SO_F32 ? 4 : 2; }

// The group at p as it is in memory; `left` elements of it (1 .. V) are the caller's.  `wide`: all V may be read, whatever the others are; else they are zero.
template <class T>
__device__ __forceinline__ typename so_elements<T>::plain so_group_load(const T *p, uint32_t left, bool wide)
{
    constexpr int V = so_elements<T>::V;
    typename so_elements<T>::plain v;
    if (wide) {
        v = *reinterpret_cast<const typename so_elements<T>::vec *>(p);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)0.0f;
#pragma unroll
        for (int e = 0; e < V - 1; ++e)
            if ((uint32_t)e < left) v[e] = p[e];
    }
    return v;
}
template <class T>
__device__ __forceinline__ typename so_elements<T>::plain so_group_load(const T *p, uint32_t left)
{
    return so_group_load(p, left, left >= (uint32_t)so_elements<T>::V);
}

// The same group, of which the compiler does not know that it has converted it before: it would keep the fp32 values, twice the registers, for the next use.
template <class G>
__device__ __forceinline__ void so_group_afresh(G &g)
{
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    words w = __builtin_bit_cast(words, g);
    asm volatile("" : "+v"(w));
    g = __builtin_bit_cast(G, w);
}

// How many rows of a matrix of `rows`, from the first on, the group of `left` elements at their end may be read whole from: what lies behind a row's end is then the
// matrix's own, the rows below it.
template <class T>
__device__ __forceinline__ uint32_t so_group_wide_rows(uint32_t left, uint32_t rows, size_t stride)
{
    constexpr uint32_t V = so_elements<T>::V;
    if (left >= V) return rows;
    const uint32_t s = (uint32_t)min(stride, (size_t)V), below = (V - left + s - 1u) / s;
    return rows > below ? rows - below : 0u;
}

// The first `left` elements of a group, whole or in pieces of 4, 2 and 1; fp32 values are rounded to nearest even.  Stored for the next reader: past the caches (nontemporal) a layer norm of
// 4096 x 8192 bf16 on data from memory takes 29 us instead of 34.5, but a second one that reads its result 71 instead of 50 for the two.
template <class T>
__device__ __forceinline__ void so_group_store(T *p, uint32_t left, const float (&f)[so_elements<T>::V])
{
    constexpr int V = so_elements<T>::V;
    typename so_elements<T>::plain v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)f[e];
    if (left >= (uint32_t)V) {
        *reinterpret_cast<typename so_elements<T>::vec *>(p) = v;
        return;
    }
    typedef T pair __attribute__((ext_vector_type(2)));
    typedef pair pair_anywhere __attribute__((aligned(sizeof(T))));
    typedef T quad __attribute__((ext_vector_type(4)));
    typedef quad quad_anywhere __attribute__((aligned(sizeof(T))));
    if constexpr (V == 8)
        if (left & 4u) *reinterpret_cast<quad_anywhere *>(p) = quad{v[0], v[1], v[2], v[3]};
    if (left & 2u) {
        pair q = {v[0], v[1]};
        if constexpr (V == 8)
            if (left & 4u) q = pair{v[4], v[5]};
        *reinterpret_cast<pair_anywhere *>(p + (left & 4u)) = q;
    }
    if (left & 1u) {
        T q = v[0];
        if (left & 2u) q = v[2];
        if constexpr (V == 8) {
            if ((left & 6u) == 4u) q = v[4];
            if ((left & 6u) == 6u) q = v[6];
        }
        p[left & 6u] = q;
    }
}

// f(T()) for an element type by its number; false for an unknown one.
template <class F>
static inline bool so_for_type(int type, F &&f)
{
    if (type == SO_F32) f(float());
    else if (type == SO_F16) f((_Float16)0.0f);
    else if (type == SO_BF16) f((__bf16)0.0f);
    else return false;
    return true;
}
