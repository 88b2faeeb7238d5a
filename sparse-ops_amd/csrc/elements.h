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

// The group at p as it is in memory; `left` elements of it (1 .. V) are the caller's to read, the others are zero.
template <class T>
__device__ __forceinline__ typename so_elements<T>::plain so_group_load(const T *p, uint32_t left)
{
    constexpr int V = so_elements<T>::V;
    typename so_elements<T>::plain v;
    if (left >= (uint32_t)V) {
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

// The first `left` elements of a group; fp32 values are rounded to nearest even.
template <class T>
__device__ __forceinline__ void so_group_store(T *p, uint32_t left, const float (&f)[so_elements<T>::V])
{
    constexpr int V = so_elements<T>::V;
    typename so_elements<T>::plain v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)f[e];
    if (left >= (uint32_t)V) {
        *reinterpret_cast<typename so_elements<T>::vec *>(p) = v;
    } else {
#pragma unroll
        for (int e = 0; e < V - 1; ++e)
            if ((uint32_t)e < left) p[e] = v[e];
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
