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

// The elements c .. c + VE - 1 of a row of n.  ODD false: n is a multiple of VE.  ODD true: `whole` says that the vectors of all lanes
// of the wave lie inside the row, so that the one that crosses its end costs the others nothing.
template <bool ODD, typename T, int VE = 16 / (int)sizeof(T)>
__device__ __forceinline__ void load_row(const T* row, int c, int n, bool whole, T (&t)[VE]) {
    if (ODD && whole) __builtin_memcpy(t, row + c, 16);
    else if (ODD ? c + VE <= n : c < n) __builtin_memcpy(t, row + c, 16);
    else {
#pragma unroll
        for (int j = 0; j < VE; ++j) t[j] = ODD && c + j < n ? row[c + j] : (T)0.0f;
    }
}
template <bool ODD, typename T, int VE>
__device__ __forceinline__ void store_row(T* row, int c, int n, bool whole, const float (&v)[VE]) {
    T t[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) t[j] = (T)v[j];
    if (ODD && whole) __builtin_memcpy(row + c, t, 16);
    else if (ODD ? c + VE <= n : c < n) __builtin_memcpy(row + c, t, 16);
    else if (ODD) {
#pragma unroll
        for (int j = 0; j < VE; ++j)
            if (c + j < n) row[c + j] = t[j];
    }
}

template <typename T, int VE>
__device__ __forceinline__ void store_vec(T* p, long long n, const float (&v)[VE]) {
    if (n >= VE) {
        T t[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) t[j] = (T)v[j];
        __builtin_memcpy(p, t, VE * sizeof(T));
    } else {
#pragma unroll
        for (int j = 0; j < VE; ++j)
            if (j < n) p[j] = (T)v[j];
    }
}

// VE fp32 values at c .. of n, or `none` where there is no tensor
template <int VE>
__device__ __forceinline__ void load_vec_or(const float* p, long long c, long long n, float (&v)[VE], float none) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = none;
    } else if (c + VE <= n) {
        __builtin_memcpy(v, p + c, VE * 4);
    } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = c + j < n ? p[c + j] : 0.0f;
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

// The same past the caches: for an operand that is read once and would push out of them what the next kernels read
typedef __attribute__((ext_vector_type(4), aligned(1), may_alias)) int yfs_int4_any;
template <typename T>
__device__ __forceinline__ void load_vec8_once(const T* p, long long n, float (&v)[8]) {
    if (n < 8) {
        load_vec8(p, n, v);
        return;
    }
    T t[8];
    yfs_int4_any raw[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __builtin_nontemporal_load((const yfs_int4_any*)p + i);
    __builtin_memcpy(t, raw, sizeof(t));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
}

// 16 bytes of a row as they lie in memory: what a kernel keeps in registers between two passes over a long row.  fence() before the
// second pass, or the widened values of the first are kept instead, twice the registers of a 16-bit row.
typedef __attribute__((ext_vector_type(4))) int yfs_int4;
template <bool ODD, typename T>
__device__ __forceinline__ yfs_int4 load_raw(const T* row, int c, int n, bool whole) {
    constexpr int VE = 16 / sizeof(T);
    yfs_int4 r = {0, 0, 0, 0};
    if ((ODD && whole) || (ODD ? c + VE <= n : c < n)) __builtin_memcpy(&r, row + c, 16);
    else if (ODD && c < n) {
        T t[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) t[j] = c + j < n ? row[c + j] : (T)0.0f;
        __builtin_memcpy(&r, t, 16);
    }
    return r;
}
template <typename T, int VE = 16 / (int)sizeof(T)>
__device__ __forceinline__ void widen_raw(const yfs_int4& r, float (&v)[VE]) {
    T t[VE];
    __builtin_memcpy(t, &r, 16);
#pragma unroll
    for (int j = 0; j < VE; ++j) v[j] = (float)t[j];
}
template <int N>
__device__ __forceinline__ void fence(yfs_int4 (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(r[i]));
}
