// Element types and scalar functions shared by the token-sequence kernels (token embedding, causal convolution, selective
// scan, gradient clipping).  Storage is fp32, bf16 or fp16 (JOVA_F32 / JOVA_BF16 / JOVA_F16); arithmetic is fp32.
#pragma once
#include "common.h"
#include "jova_hip.h"

typedef __bf16 bf16_t;
typedef _Float16 fp16_t;

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
// one rounding to nearest-even when the value leaves the registers (identity for fp32)
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }

static inline size_t jova_dtype_size(int dtype) { return dtype == JOVA_F32 ? 4 : 2; }
static inline bool jova_dtype_ok(int dtype) { return dtype == JOVA_F32 || dtype == JOVA_BF16 || dtype == JOVA_F16; }

// a value of a small parameter whose type is known only at run time (weights of the convolution)
__device__ __forceinline__ float ld_any(const void* p, int dtype, long long i) {
    if (dtype == JOVA_F32) return ((const float*)p)[i];
    if (dtype == JOVA_BF16) return (float)((const bf16_t*)p)[i];
    return (float)((const fp16_t*)p)[i];
}
__device__ __forceinline__ void st_any(void* p, int dtype, long long i, float v) {
    if (dtype == JOVA_F32) ((float*)p)[i] = v;
    else if (dtype == JOVA_BF16) ((bf16_t*)p)[i] = (bf16_t)v;
    else ((fp16_t*)p)[i] = (fp16_t)v;
}

constexpr float LOG2E_F = 1.4426950408889634f;
constexpr float LN2_F = 0.6931471805599453f;

// 1 / (1 + e^-v): v_exp_f32 and v_rcp_f32 are one ulp each; e^-v = inf gives 0, NaN stays NaN
__device__ __forceinline__ float sigmoid_f(float v) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E_F * v));
}
// log(1 + e^v) = max(v, 0) + log1p(e), e = e^-|v| in (0, 1], and log1p(e) = 2 atanh(s) with s = e / (2 + e) <= 1/3, so small
// results keep their relative accuracy (a plain log(1 + e) loses it: steps of 1e-3 are ordinary inputs of the scan).  atanh(s)/s
// is a polynomial of degree 4 in s^2, fitted for the smallest largest relative error on [0, 1/9]: 8e-9, an eighth of fp32's.
__device__ __forceinline__ float softplus_f(float v) {
    const float e = __builtin_amdgcn_exp2f(-LOG2E_F * fabsf(v));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float p = fmaf(0.14089167f, q, 0.13980301f);
    p = fmaf(p, q, 0.20012455f);
    p = fmaf(p, q, 0.33333158f);
    p = fmaf(p * q, s, s);
    return fmaf(2.f, p, v > 0.f ? v : 0.f);
}

// LDS accesses of a wave's lanes on either side stay on theirs (the hardware keeps a wave's LDS operations in order)
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
__device__ __forceinline__ void wave_order() {
    wave_fence();
    __builtin_amdgcn_wave_barrier();
}
