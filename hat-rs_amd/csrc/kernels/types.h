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

// N consecutive elements at byte offset off + base of a buffer descriptor: zeros past its
// end, where stores are dropped, so that a row's last moves need no branch.
template <class T, int N>
__device__ __forceinline__ typename Vec<T, N>::type buffer_load_raw(__amdgpu_buffer_rsrc_t r, unsigned off, unsigned base)
{
    typedef typename Vec<T, N>::type U;
    if constexpr (sizeof(T) * N == 16)
        return __builtin_bit_cast(U, __builtin_amdgcn_raw_buffer_load_b128(r, off, base, 0));
    else if constexpr (sizeof(T) * N == 8)
        return __builtin_bit_cast(U, __builtin_amdgcn_raw_buffer_load_b64(r, off, base, 0));
    else if constexpr (sizeof(T) * N == 4)
        return __builtin_bit_cast(U, __builtin_amdgcn_raw_buffer_load_b32(r, off, base, 0));
    else
        return __builtin_bit_cast(U, __builtin_amdgcn_raw_buffer_load_b16(r, off, base, 0));
}

template <class T, int N>
__device__ __forceinline__ void to_float(const typename Vec<T, N>::type& u, float (&v)[N])
{
    if constexpr (N == 1) {
        v[0] = (float)u;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)u[i];
    }
}

template <class T, int N>
__device__ __forceinline__ void buffer_load_vec(__amdgpu_buffer_rsrc_t r, unsigned off, unsigned base, float (&v)[N])
{
    to_float<T, N>(buffer_load_raw<T, N>(r, off, base), v);
}

template <class T, int N>
__device__ __forceinline__ void buffer_store_vec(__amdgpu_buffer_rsrc_t r, unsigned off, unsigned base, const float (&v)[N])
{
    typename Vec<T, N>::type u;
    if constexpr (N == 1) {
        u = (T)v[0];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = (T)v[i];
    }
    if constexpr (sizeof(T) * N == 16)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, u), r, off, base, 0);
    else if constexpr (sizeof(T) * N == 4)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, u), r, off, base, 0);
    else
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, u), r, off, base, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00027000);
}
