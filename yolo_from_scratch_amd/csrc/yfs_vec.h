// 16-byte vectors of fp32, bf16 or fp16 elements at any element alignment, widened to fp32 in registers.
// gfx950 loads and stores 16 bytes at any address, so rows of odd widths need no second code path: only the vector that
// crosses the end of a row is taken element by element.
#pragma once
#include <hip/hip_runtime.h>

template <typename T, int VE = 16 / (int)sizeof(T)>
__device__ __forceinline__ void load_vec(const T* p, long long n, float (&v)[VE]) {   // n = elements left in the row
    T t[VE];
    if (n >= VE) {
        __builtin_memcpy(t, p, 16);
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = (float)t[j];
    } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = j < n ? (float)p[j] : 0.0f;
    }
}

template <typename T, int VE>
__device__ __forceinline__ void store_vec(T* p, long long n, const float (&v)[VE]) {
    if (n >= VE) {
        T t[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) t[j] = (T)v[j];
        __builtin_memcpy(p, t, 16);
    } else {
#pragma unroll
        for (int j = 0; j < VE; ++j)
            if (j < n) p[j] = (T)v[j];
    }
}

// VE fp32 values (16-byte loads), or `none` where there is no tensor
template <int VE>
__device__ __forceinline__ void load_vec_or(const float* p, long long c, long long n, float (&v)[VE], float none) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = none;
    } else if (n >= VE) {
        __builtin_memcpy(v, p + c, VE * 4);
    } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = j < n ? p[c + j] : 0.0f;
    }
}

// 8 elements of any of the three types; n = elements left in the row
template <typename T>
__device__ __forceinline__ void load_vec8(const T* p, long long n, float (&v)[8]) {
    T t[8];
    if (n >= 8) {
        __builtin_memcpy(t, p, 8 * sizeof(T));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.0f;
    }
}
