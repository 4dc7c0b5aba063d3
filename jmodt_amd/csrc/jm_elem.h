// jm_elem.h — element types of the row operators that take float32, bfloat16 or float16 rows (rows8.hip, adapters.hip): loads and
// stores of 8 consecutive elements at element alignment, and the 16 x 16 matrix step on fragments of 8 contraction elements a lane.
#pragma once
#include "jm_common.h"

namespace jm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int TY> struct Elem;      // JM_F32, JM_BF16, JM_F16
template <> struct Elem<JM_F32> { typedef float T; typedef f32x8 V8; };
template <> struct Elem<JM_BF16> { typedef __bf16 T; typedef bf16x8 V8; };
template <> struct Elem<JM_F16> { typedef _Float16 T; typedef f16x8 V8; };

// 8 consecutive elements, aligned to one element only (global memory takes any address; row strides are the caller's)
template <typename V, typename T>
__device__ __forceinline__ V load8(const T* p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <typename V, typename T>
__device__ __forceinline__ void store8(T* p, const V& v) {
    __builtin_memcpy(p, &v, sizeof(V));
}
// elements 0 .. n - 1 of the 8, zeros behind them (n <= 0: all zeros, nothing is read)
template <typename V, typename T>
__device__ __forceinline__ V load8_tail(const T* p, int n) {
    V v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        T t = (T)0.f;
        if (e < n) t = p[e];
        v[e] = t;
    }
    return v;
}
template <typename V, typename T>
__device__ __forceinline__ V load8_upto(const T* p, int n) { return n >= 8 ? load8<V>(p) : load8_tail<V>(p, n); }

// D (16 x 16) += A (16 x 32) B (32 x 16): lane l holds row / column l % 16 and contraction elements 8 (l / 16) .. + 7 of both
// operands; D: column l % 16, rows 4 (l / 16) .. + 3.  In float32 the step is eight 16 x 16 x 4 products, the e-th of which
// contracts element e of the four lane groups (the order of the contraction is free as long as both operands share it).
__device__ __forceinline__ f32x4 mma16(f32x4 c, const f32x8& a, const f32x8& b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mma16(f32x4 c, const bf16x8& a, const bf16x8& b) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(f32x4 c, const f16x8& a, const f16x8& b) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// the upper (lower) halves of two words as one: half of a | half of b << 16
__device__ __forceinline__ unsigned pack_hi(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ unsigned pack_lo(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }

}  // namespace jm
