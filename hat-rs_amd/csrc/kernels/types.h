// Element types of the operators on device tensors: fp32, fp16, bf16, each read into
// fp32 and rounded to nearest once when written.
#pragma once
#include "common.h"

typedef _Float16 f16;
typedef __bf16 bf16;

// N consecutive elements, moved as one load or store where N * sizeof(T) allows.
template <class T, int N>
struct Vec {
    typedef T type __attribute__((ext_vector_type(N)));
};
template <class T>
struct Vec<T, 1> {
    typedef T type;
};

template <class T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[N])
{
    const auto u = *(const typename Vec<T, N>::type*)p;
    if constexpr (N == 1) {
        v[0] = (float)u;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)u[i];
    }
}

template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[N])
{
    typename Vec<T, N>::type u;
    if constexpr (N == 1) {
        u = (T)v[0];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = (T)v[i];
    }
    *(typename Vec<T, N>::type*)p = u;
}
