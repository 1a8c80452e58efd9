// vx_i8.hpp — rows of 8-bit integers with a scale each, and what becomes of a
// product's whole-number sums.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../vx_kargs.h"

typedef int i4v __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));

// The scale of a row whose largest magnitude is m (as bits: NaN above infinity
// above all numbers) and what its values are multiplied with to give codes. A row
// below 2^-100 is zeros; one with a NaN or an infinity has the scale NaN, which
// reaches every product of the row.
__device__ __forceinline__ float vx_i8_scale(uint32_t m, float& r) {
    if (m >= 0x7F800000u) {
        r = 0.f;
        return __builtin_nanf("");
    }
    const float f = __builtin_bit_cast(float, m);
    if (f < 0x1p-100f) {
        r = 0.f;
        return 0.f;
    }
    r = 127.0f / f;
    return f / 127.0f;
}
__device__ __forceinline__ uint32_t vx_i8_code(float x, float r) {
    // (NaN, or infinity times 0: the lower bound, under a scale that is NaN)
    return (uint32_t)(int)__builtin_amdgcn_fmed3f(__builtin_rintf(x * r), -127.f, 127.f) & 255u;
}
__device__ __forceinline__ uint32_t vx_i8_codes(f4v x, float r) {
    return vx_i8_code(x.x, r) | vx_i8_code(x.y, r) << 8 | vx_i8_code(x.z, r) << 16 | vx_i8_code(x.w, r) << 24;
}
__device__ __forceinline__ uint32_t vx_abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t vx_max4(uint32_t m, f4v x) {
    return max(max(m, max(vx_abs_bits(x.x), vx_abs_bits(x.y))), max(vx_abs_bits(x.z), vx_abs_bits(x.w)));
}

// sum * sx * sw with three roundings of half a step each, for scales of any size:
// mantissas are multiplied, the powers of two added and put on at the end.
struct vx_i8_scaled {
    float m;
    int e;
    __device__ __forceinline__ explicit vx_i8_scaled(float s) : m(__builtin_amdgcn_frexp_mantf(s)), e(__builtin_amdgcn_frexp_expf(s)) {}
};
__device__ __forceinline__ float vx_i8_value(int sum, vx_i8_scaled x, vx_i8_scaled w) {
    return __builtin_amdgcn_ldexpf((float)sum * (x.m * w.m), x.e + w.e);
}

// ---- activations of the gate (vx_act)
// 1 / (1 + e^-y): 2^p with p = y log2(e) as a rounded product and what that left
// out (whose share of the result is its share of p times ln 2), and a reciprocal
// made better by one Newton step: 2 steps of f32 off at most.
__device__ __forceinline__ float vx_sigmoid(float y) {
    const float p = y * -1.44269504f;
    const float left = __builtin_fmaf(y, -1.44269504f, -p) + y * -1.92596299e-8f;
    float e = __builtin_amdgcn_exp2f(p);
    e = e < __builtin_inff() ? __builtin_fmaf(e, left * 0.693147182f, e) : e;
    const float d = 1.f + e;
    const float r = __builtin_amdgcn_rcpf(d);
    return d < 0x1p126f ? __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.f), r) : r;
}
__device__ __forceinline__ float vx_act(uint32_t act, float g) {
    if (act == 0) return g * vx_sigmoid(g);                                                                          // silu
    if (act == 1) return g * vx_sigmoid(1.5957691216f * __builtin_fmaf(0.044715f * g * g, g, g));                    // gelu, by tanh
    if (act == 2) return 0.5f * g * erfcf(g * -0.70710678118f);                                                      // gelu
    return g > 0.f ? g : g == g ? 0.f : g;                                                                           // relu
}

// Four neighbouring channels of a token.
__device__ __forceinline__ void vx_i8_store4(const vx_i8_args& a, uint32_t t, uint32_t n, f4v v) {
    if (t >= a.T || n >= a.N) return;
    float* p = a.out + (int64_t)t * a.os[0] + (int64_t)n * a.os[1];
    if (a.out_vec && n + 4 <= a.N) {
        *(f4v*)p = v;
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (n + i < a.N) p[i * a.os[1]] = v[i];
}
__device__ __forceinline__ f4v vx_i8_scales4(const float* s, uint32_t n, uint32_t N) {
    f4v v;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) v[i] = s[min(n + i, N - 1u)];
    return v;
}
template <bool GATED>
__device__ __forceinline__ void vx_i8_finish4(const vx_i8_args& a, uint32_t t, uint32_t n, float sx, i4v g, i4v u, f4v sg, f4v su) {
    const vx_i8_scaled x(sx);
    f4v v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = vx_i8_value(g[i], x, vx_i8_scaled(sg[i]));
        if constexpr (GATED) v[i] = vx_act(a.act, v[i]) * vx_i8_value(u[i], x, vx_i8_scaled(su[i]));
    }
    vx_i8_store4(a, t, n, v);
}
