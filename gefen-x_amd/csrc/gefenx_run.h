// gefenx_run.h -- runs of elements that a lane moves at a time.
#pragma once

#include "gefenx_device.h"

namespace gx {

// W consecutive elements (8 bytes or more) at any alignment of their type, streamed (reads: unless
// told otherwise); the end of an array, where fewer than W are left, by elements (reads fill up with
// `beyond`, nothing is written past it).
template <class T, int W> struct Run { T e[W]; };

template <class T, int W, bool STREAM = true>
__device__ __forceinline__ Run<T, W> load_run(const T* base, int64_t left, T beyond = T(0)) {
    typedef uint32_t V __attribute__((ext_vector_type(W * sizeof(T) / 4), aligned(sizeof(T))));
    static_assert(W * sizeof(T) >= 8, "vectors of two words and more");
    Run<T, W> r;
    if (left >= W) {
        if constexpr (STREAM) {
            const auto v = __builtin_nontemporal_load(GX_GLOBAL_AS(const V, base));
            __builtin_memcpy(&r, &v, sizeof(r));
        } else {
            const V v = *GX_GLOBAL_AS(const V, base);
            __builtin_memcpy(&r, &v, sizeof(r));
        }
    } else {
#pragma unroll
        for (int k = 0; k < W; ++k) r.e[k] = k < left ? *gbl(base + k) : beyond;
    }
    return r;
}

template <class T, int W>
__device__ __forceinline__ void store_run(T* base, int64_t left, const Run<T, W>& r) {
    typedef uint32_t V __attribute__((ext_vector_type(W * sizeof(T) / 4), aligned(sizeof(T))));
    if (left >= W) {
        V v;
        __builtin_memcpy(&v, &r, sizeof(r));
        __builtin_nontemporal_store(v, GX_GLOBAL_AS(V, base));
    } else {
#pragma unroll
        for (int k = 0; k < W; ++k)
            if (k < left) *gbl(base + k) = r.e[k];
    }
}

}  // namespace gx
