// Shared helpers of the trained-block operators (dmn_layernorm.hip, dmn_linear.hip, dmn_clip.hip): element types, 16-byte
// vectors of them at any element alignment, reductions over a workgroup.
#pragma once
#include "../../include/dmn.h"
#include "dmn_common.h"

typedef _Float16 f16;

template <typename T> struct Pack {
    static constexpr int N = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
};

// 16 bytes from / to an address that is aligned to the element only. gfx950 takes any alignment in one global
// instruction; a row of an odd width costs at most one more cache line per wave.
template <typename T> __device__ __forceinline__ typename Pack<T>::vec load16(const T* p) {
    typename Pack<T>::vec v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
template <typename T> __device__ __forceinline__ void store16(T* p, typename Pack<T>::vec v) { __builtin_memcpy(p, &v, 16); }

// The vector at element `at` of a row of `n` elements: elements behind the row's end read as zero (their addresses are
// clamped to the row, so nothing outside it is touched). at < n.
template <typename T> __device__ __forceinline__ typename Pack<T>::vec load16_tail(const T* row, int at, int n) {
    typename Pack<T>::vec v;
    if (at + Pack<T>::N <= n) return load16(row + at);
#pragma unroll
    for (int i = 0; i < Pack<T>::N; ++i) {
        const T e = row[at + i < n ? at + i : n - 1];
        v[i] = at + i < n ? e : (T)0.f;
    }
    return v;
}
template <typename T> __device__ __forceinline__ void store16_tail(T* row, int at, int n, typename Pack<T>::vec v) {
    if (at + Pack<T>::N <= n) {
        store16(row + at, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < Pack<T>::N; ++i)
        if (at + i < n) row[at + i] = v[i];
}

// Pack<A>::N-independent read of Pack<T>::N consecutive parameters of type A as float (A is T or float).
template <typename T, typename A> __device__ __forceinline__ void load_params(const A* p, int at, int n, float* out) {
#pragma unroll
    for (int i = 0; i < Pack<T>::N; i += Pack<A>::N) {
        if (at + i < n) {
            const auto v = load16_tail(p, at + i, n);
#pragma unroll
            for (int j = 0; j < Pack<A>::N; ++j)
                if (i + j < Pack<T>::N) out[i + j] = (float)v[j];
        } else {
#pragma unroll
            for (int j = 0; j < Pack<A>::N; ++j)
                if (i + j < Pack<T>::N) out[i + j] = 0.f;
        }
    }
}

// Sum over aligned groups of W lanes (8..64), every lane of the group receives it; fixed order. Every lane of the wave
// must be active.
template <int W> __device__ __forceinline__ float group_sum(float v) {
    static_assert(W == 8 || W == 16 || W == 32 || W == 64, "lanes per group");
    if constexpr (W == 8) {
        v += dpp_move<0xB1>(v);
        v += dpp_move<0x4E>(v);
        v += dpp_move<0x141>(v);
        return v;
    } else {
        return seg_sum(v, W);
    }
}

inline size_t block_align256(size_t n) { return (n + 255) & ~(size_t)255; }

#define DMN_BLOCK_LAUNCH_CHECK()                                                                                      \
    do {                                                                                                              \
        hipError_t _e = hipGetLastError();                                                                            \
        if (_e != hipSuccess) {                                                                                       \
            dmn_set_error("kernel launch failed: %s (%s:%d)", hipGetErrorString(_e), __FILE__, __LINE__);             \
            return DMN_ERR_HIP;                                                                                       \
        }                                                                                                             \
    } while (0)
