// elem.h — one value of a tensor that is 16-bit or f32: the type, and its way from and to f32.
#pragma once
#include "common.h"

template <bool F32>
struct Elem;
template <>
struct Elem<true> {
    typedef float T;
    static __device__ __forceinline__ float get(const float *p) { return *p; }
    static __device__ __forceinline__ void put(float *p, float v) { *p = v; }
};
template <>
struct Elem<false> {
    typedef a16_t T;
    static __device__ __forceinline__ float get(const a16_t *p) { return a2f(*p); }
    static __device__ __forceinline__ void put(a16_t *p, float v) { *p = f2a(v); }
};
