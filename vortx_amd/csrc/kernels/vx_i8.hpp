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

// sum * sx * sw for scales of any size: mantissas are multiplied, the powers of two
// added and put on at the end. Three roundings, of the sum (if 2^24 or more), of the
// mantissas' product and of the result, 2^-24 each, relatively: the first two may be
// a step of the result each, 2.5 in all (1.95 measured, 1.4 with sums below 2^24).
struct vx_i8_scaled {
    float m;
    int e;
    __device__ __forceinline__ explicit vx_i8_scaled(float s) : m(__builtin_amdgcn_frexp_mantf(s)), e(__builtin_amdgcn_frexp_expf(s)) {}
};
__device__ __forceinline__ float vx_i8_value(int sum, vx_i8_scaled x, vx_i8_scaled w) {
    return __builtin_amdgcn_ldexpf((float)sum * (x.m * w.m), x.e + w.e);
}

// ---- activations of the gate (vx_act)
// g / (1 + e^-y), for y of g's sign: 2^p with p = y log2(e) as a rounded product and
// what that left out (whose share of the result is its share of p times ln 2), and a
// reciprocal made better by one Newton step. At most 6 2^-24 off, relatively: 3 of
// e^-y, 1 each of the sum, the reciprocal and the product. From p = 64 on (where 1 no
// longer counts) 2^-64 of the sum is formed and put on after the product, so that
// no factor leaves the normal numbers before the result does. Past 126 either way
// y changes nothing any more (g e^-126 rounds to 0), and is 126, so that p and what
// it left out are finite.
__device__ __forceinline__ float vx_gate(float g, float y) {
#pragma clang fp contract(off)  // (p - 64 of the rounded product)
    y = __builtin_amdgcn_fmed3f(y, -126.f, 126.f);  // (NaN too: g is one then)
    const float p = y * -1.44269504f;
    const float left = __builtin_fmaf(y, -1.92596299e-8f, __builtin_fmaf(y, -1.44269504f, -p));
    const bool far = p > 64.f;
    const float one = far ? 0x1p-64f : 1.f;
    float e = __builtin_amdgcn_exp2f(far ? p - 64.f : p);
    e = __builtin_fmaf(e, left * 0.693147182f, e);
    const float d = one + e;
    const float r = __builtin_amdgcn_rcpf(d);
    return g * __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.f), r) * one;
}
// Gates below -126 are as -126: nothing, also where the product has left f32's range.
// (N together: the branch is taken once, and their chains overlap. A prompt's gated
// product 2011 x 11008 x 4096 207 us with four, 212 with one after the other.)
template <int N>
__device__ __forceinline__ void vx_act(uint32_t act, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] < -126.f ? -126.f : v[i];
    if (act == 0) {  // silu
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = vx_gate(v[i], v[i]);
    } else if (act == 1) {  // gelu, by tanh
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = vx_gate(v[i], 1.5957691216f * __builtin_fmaf(0.044715f * v[i] * v[i], v[i], v[i]));
    } else if (act == 2) {  // gelu
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.5f * v[i] * erfcf(v[i] * -0.70710678118f);
    } else {  // relu
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] > 0.f ? v[i] : v[i] == v[i] ? 0.f : v[i];
    }
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
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = vx_i8_value(g[i], x, vx_i8_scaled(sg[i]));
    if constexpr (GATED) {
        vx_act(a.act, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= vx_i8_value(u[i], x, vx_i8_scaled(su[i]));
    }
    vx_i8_store4(a, t, n, f4v{v[0], v[1], v[2], v[3]});
}
