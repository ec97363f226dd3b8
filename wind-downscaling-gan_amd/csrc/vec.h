// vec.h — several adjacent elements in one request, at any element's address (layernorm.hip, adamw.hip).
// Rows and tensors may start anywhere (odd widths, views into wider buffers), so no alignment beyond the element's own is promised;
// the global memory path of this target takes such requests whole.
#pragma once
#include "common.h"

template <class T, int V>
struct WdgVec {
    T e[V];
};
template <class T, int V>
__device__ __forceinline__ WdgVec<T, V> wdg_vec_load(const T* p) {
    WdgVec<T, V> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <class T, int V>
__device__ __forceinline__ void wdg_vec_store(T* p, const WdgVec<T, V>& v) {
    __builtin_memcpy(p, &v, sizeof(v));
}
