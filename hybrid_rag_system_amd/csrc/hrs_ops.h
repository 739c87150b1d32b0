// Shared by the encoder-layer operators (hrs_linear.hip, hrs_attention.hip, hrs_norm.hip): element types, matrix
// instructions, waits, activations.
#pragma once
#include <stdlib.h>

#include "hrs_internal.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct vec_of;
template <>
struct vec_of<__bf16> {
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 x4 __attribute__((ext_vector_type(4)));
    typedef __bf16 x2 __attribute__((ext_vector_type(2)));
};
template <>
struct vec_of<_Float16> {
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    typedef _Float16 x4 __attribute__((ext_vector_type(4)));
    typedef _Float16 x2 __attribute__((ext_vector_type(2)));
};

// D[16 rows of a][16 rows of b] += a b^T over 32 of the depth: lane l gives row l % 16, depth (l / 16) * 8 .. + 7 of either
// operand and holds rows (l / 16) * 4 .. + 3 of column l % 16 of D.
__device__ __forceinline__ f32x4 mfma16(vec_of<__bf16>::x8 a, vec_of<__bf16>::x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(vec_of<_Float16>::x8 a, vec_of<_Float16>::x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// The same for 32 x 32 over 16 of the depth: lane l gives row l % 32, depth (l / 32) * 8 .. + 7 and holds rows
// 8 g + 4 (l / 32) + i (register 4 g + i) of column l % 32.
__device__ __forceinline__ f32x16 mfma32(vec_of<__bf16>::x8 a, vec_of<__bf16>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(vec_of<_Float16>::x8 a, vec_of<_Float16>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// c + v[0] + v[1] in fp32
__device__ __forceinline__ float add_pair(vec_of<__bf16>::x2 v, float c) {
    const vec_of<__bf16>::x2 one = {(__bf16)1.f, (__bf16)1.f};
    return __builtin_amdgcn_fdot2_f32_bf16(v, one, c, false);
}
__device__ __forceinline__ float add_pair(vec_of<_Float16>::x2 v, float c) {
    const vec_of<_Float16>::x2 one = {(_Float16)1.f, (_Float16)1.f};
    return __builtin_amdgcn_fdot2(v, one, c, false);
}

// v over the wave's lanes
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Every earlier load of this wave has arrived, every earlier LDS access of it is done; then the workgroup's barrier.
__device__ __forceinline__ void wait_all_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 8 elements at p, of which the first n (<= 8) exist; the rest are zero.  p need only be aligned to an element: the
// hardware takes a 16-byte global load at any address.
template <typename T>
__device__ __forceinline__ typename vec_of<T>::x8 load8_any(const T* p, int n) {
    typename vec_of<T>::x8 v;
    if (n >= 8) {
        __builtin_memcpy(&v, p, 16);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (T)0.f;
    }
    return v;
}

// Consecutive workgroups go round the 8 XCDs, each with an L2 of its own: renumbered so that an XCD has a consecutive run.
__device__ __forceinline__ int spread_over_xcds(int block, int grid) {
    const int x = block & 7, q = grid >> 3, r = grid & 7;
    return x * q + (x < r ? x : r) + (block >> 3);
}

// ---- activations -----------------------------------------------------------------------------------
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4, ACT_TANH = 5 };

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_hw(float x) { return __builtin_amdgcn_rcpf(x); }

// x Phi(x) = max(x, 0) - |x| Phi(-|x|), with Phi(-a) = exp(-a^2 / 2) erfcx(a / sqrt 2) / 2 and the scaled complement as
// t (c0 + c1 t + .. + c4 t^4), t = 1 / (1 + 0.375 a): a least-maximum fit of the relative error over 0 <= a <= 13.5
// (2.9e-5; the result is within 3.4e-5 of its own size on both sides of zero, a fifteenth of an fp16 half-step).  Two
// transcendental and ten ordinary operations.
__device__ __forceinline__ float gelu_f(float x) {
    const float a = fabsf(fminf(x, 20.f));  // (e is 0 from 20 on, and 0 * inf would be NaN where x is inf)
    const float t = rcp_hw(fmaf(0.375f, a, 1.f));
    float q = fmaf(-0.0909841f, t, 0.20104071f);
    q = fmaf(q, t, 0.08297601f);
    q = fmaf(q, t, 0.15791951f);
    q = fmaf(q, t, 0.14904118f);
    const float e = exp2_hw(x * x * -0.72134752f);
    return fmaf(-a, t * q * e, fmaxf(x, 0.f));
}
__device__ __forceinline__ float sigmoid_f(float x) { return rcp_hw(1.f + exp2_hw(x * -1.44269504f)); }
// tanh = 1 - 2 / (1 + e^2x) loses its leading digits near zero, where three terms of the series are exact to 2e-7
__device__ __forceinline__ float tanh_f(float x) {
    const float big = fmaf(-2.f, rcp_hw(1.f + exp2_hw(x * 2.88539008f)), 1.f);
    const float s = x * x;
    const float small = x * fmaf(s, fmaf(s, 0.13333333f, -0.33333333f), 1.f);
    return s < 0.01f ? small : big;
}
// As in the formulas, an infinite argument of gelu, gelu_tanh or silu below zero gives NaN (0 * inf).
template <int ACT>
__device__ __forceinline__ float activate(float x) {
    if constexpr (ACT == ACT_RELU) return x > 0.f ? x : (x != x ? x : 0.f);
    if constexpr (ACT == ACT_GELU) return gelu_f(x);
    if constexpr (ACT == ACT_GELU_TANH) return x * sigmoid_f(x * fmaf(x * x, 0.07135481f, 1.59576912f));
    if constexpr (ACT == ACT_SILU) return x * sigmoid_f(x);
    if constexpr (ACT == ACT_TANH) return tanh_f(x);
    return x;
}

// Selects `device` for the calling thread and puts the thread's own device back at the end of the scope.
struct hrs_device_scope {
    int before = -1;
    hipError_t err;
    explicit hrs_device_scope(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) {
            err = hipSetDevice(device);
        } else {
            before = -1;
        }
    }
    ~hrs_device_scope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};
