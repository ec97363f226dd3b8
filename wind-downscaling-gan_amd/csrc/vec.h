// vec.h — several adjacent elements in one request, at any element's address (layernorm.hip, adamw.hip).
// Rows and tensors may start anywhere (odd widths, views into wider buffers), so no alignment beyond the element's own is promised;
// the global memory path of this target takes such requests whole.
//
// Pointers are cast to global memory: one that comes out of a table in memory would otherwise be followed by flat requests, which also
// wait for the LDS counter.
//
// STREAM: the request is marked as not to be used again (non-temporal), for tensors that the caches cannot hold until their next use.
#pragma once
#include "common.h"

#define WDG_GLOBAL __attribute__((address_space(1)))

template <class T, int V>
struct WdgVec {
    T e[V];
};
template <int BYTES, int ALIGN>
struct WdgWords;      // BYTES that are aligned to ALIGN
template <> struct WdgWords<16, 4> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct WdgWords<16, 2> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct WdgWords<8, 4> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(4))); };
template <> struct WdgWords<8, 2> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct WdgWords<4, 4> { typedef unsigned type; };
template <> struct WdgWords<4, 2> { typedef unsigned type __attribute__((aligned(2))); };
template <> struct WdgWords<2, 2> { typedef unsigned short type; };
// the widest request that divides BYTES
constexpr int wdg_request(int bytes) { return bytes % 16 == 0 ? 16 : bytes % 8 == 0 ? 8 : bytes % 4 == 0 ? 4 : 2; }

template <class T, int V, bool STREAM = false>
__device__ __forceinline__ WdgVec<T, V> wdg_vec_load(const T* p) {
    constexpr int W = wdg_request(sizeof(WdgVec<T, V>)), N = sizeof(WdgVec<T, V>) / W;
    typedef typename WdgWords<W, sizeof(T)>::type words;
    const WDG_GLOBAL words* g = (const WDG_GLOBAL words*)p;
    WdgVec<T, V> v;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        words w;
        if constexpr (STREAM) w = __builtin_nontemporal_load(g + i);
        else w = g[i];
        __builtin_memcpy((char*)&v + i * W, &w, W);
    }
    return v;
}
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ void wdg_vec_store(T* p, const WdgVec<T, V>& v) {
    constexpr int W = wdg_request(sizeof(WdgVec<T, V>)), N = sizeof(WdgVec<T, V>) / W;
    typedef typename WdgWords<W, sizeof(T)>::type words;
    WDG_GLOBAL words* g = (WDG_GLOBAL words*)p;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        words w;
        __builtin_memcpy(&w, (const char*)&v + i * W, W);
        if constexpr (STREAM) __builtin_nontemporal_store(w, g + i);
        else g[i] = w;
    }
}
