// Element types and vector accesses of libartread.so.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef _Float16 f16;
typedef __bf16 bf16;

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T from_f32(float x) { return (T)x; }   // to nearest, ties to even

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec {
    T x[N];
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// N elements from an address aligned to min(16, their bytes)
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) { return *(const Vec<T, N>*)p; }
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec_nt(const T* p) {
    if constexpr (sizeof(T) * N == 16) {
        const u32x4 v = __builtin_nontemporal_load((const u32x4*)p);
        return __builtin_bit_cast(Vec<T, N>, v);
    } else {
        return *(const Vec<T, N>*)p;
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& v) { *(Vec<T, N>*)p = v; }
template <typename T, int N>
__device__ __forceinline__ void store_vec_nt(T* p, const Vec<T, N>& v) {
    if constexpr (sizeof(T) * N == 16)
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4*)p);
    else
        *(Vec<T, N>*)p = v;
}
