// Element types of the grouped-row operators (key order, table lookup, grouped products): conversions to and from the
// 32-bit arithmetic type, and vector loads and stores of 2 to 16 bytes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace qmlb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// BYTES consecutive bytes as one access
template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };

template <typename T, int VEC>
struct Pack {
    union {
        typename Word<VEC * (int)sizeof(T)>::type word;
        T item[VEC];
    };
    __device__ __forceinline__ Pack() {}
};

template <typename T, int VEC>
__device__ __forceinline__ void load_f32(const T *p, float (&v)[VEC]) {
    Pack<T, VEC> k;
    k.word = *reinterpret_cast<const typename Word<VEC * (int)sizeof(T)>::type *>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(k.item[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_f32(T *p, const float (&v)[VEC]) {
    Pack<T, VEC> k;
#pragma unroll
    for (int i = 0; i < VEC; ++i) k.item[i] = from_f32<T>(v[i]);
    *reinterpret_cast<typename Word<VEC * (int)sizeof(T)>::type *>(p) = k.word;
}

inline int dtype_size(int dtype) { return dtype == QMLB_F32 ? 4 : (dtype == QMLB_F16 || dtype == QMLB_BF16 ? 2 : 0); }

// Largest power of two of at most 16 bytes that divides a row of `row_bytes` bytes and every given address, at least the
// element size: the width of the accesses that can follow the rows.
inline int access_bytes(size_t row_bytes, int element, const void *a, const void *b = nullptr) {
    const uintptr_t bits = (uintptr_t)row_bytes | (uintptr_t)a | (uintptr_t)b;
    int w = 16;
    while (w > element && (bits & (uintptr_t)(w - 1))) w >>= 1;
    return w;
}

}  // namespace qmlb
