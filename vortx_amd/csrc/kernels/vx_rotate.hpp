// vx_rotate.hpp — rows of heads normed and rotated, four dims a lane.
//
// Everything between the load and the store is f64 and rounded once: a key's
// codes in the cache follow from the result, and next to a border between two
// codes f32 sums of another order would give another code. The f64 units carry
// it: a value takes some 10 operations, 8000 tokens of 48 heads of 128 0.5 G of
// them, 13 us of the card's f64 rate beside 80 us of HBM traffic. A row's dims lie in one
// wave, which loads all of them (its partners' too) before it stores any, so a
// row may be overwritten in place.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../vx_kargs.h"

typedef float vx_r4 __attribute__((ext_vector_type(4)));

// sin and cos of a: multiples of pi / 2 taken out by fused multiply-adds with
// pi / 2 as the sum of two doubles, then the Taylor series to x^17 and x^16 on
// [-pi / 4, pi / 4] (the next terms are below 2^-58).
__device__ __forceinline__ void vx_sin_cos(double a, double& s, double& c) {
    const double n = __builtin_rint(a * 0.63661977236758134308);
    double x = __builtin_fma(n, -1.57079632679489655800, a);
    x = __builtin_fma(n, -6.12323399573676603587e-17, x);
    const double z = x * x;
    double p = 1.0 / 355687428096000.0, q = 1.0 / 20922789888000.0;
    p = __builtin_fma(p, z, -1.0 / 1307674368000.0);
    q = __builtin_fma(q, z, -1.0 / 87178291200.0);
    p = __builtin_fma(p, z, 1.0 / 6227020800.0);
    q = __builtin_fma(q, z, 1.0 / 479001600.0);
    p = __builtin_fma(p, z, -1.0 / 39916800.0);
    q = __builtin_fma(q, z, -1.0 / 3628800.0);
    p = __builtin_fma(p, z, 1.0 / 362880.0);
    q = __builtin_fma(q, z, 1.0 / 40320.0);
    p = __builtin_fma(p, z, -1.0 / 5040.0);
    q = __builtin_fma(q, z, -1.0 / 720.0);
    p = __builtin_fma(p, z, 1.0 / 120.0);
    q = __builtin_fma(q, z, 1.0 / 24.0);
    p = __builtin_fma(p, z, -1.0 / 6.0);
    q = __builtin_fma(q, z, -0.5);
    p = __builtin_fma(p * z, x, x);
    q = __builtin_fma(q, z, 1.0);
    const int k = (int)(n - 4.0 * __builtin_floor(n * 0.25));  // quadrant, for any n
    s = k & 1 ? q : p;
    c = k & 1 ? p : q;
    if (k & 2) s = -s;
    if ((k + 1) & 2) c = -c;
}

template <int CTRL>
__device__ __forceinline__ double vx_dpp64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over aligned groups of LANES lanes, the same in every lane of one.
template <int LANES>
__device__ __forceinline__ double vx_sum_lanes(double v) {
    v += vx_dpp64<0xB1>(v);
    v += vx_dpp64<0x4E>(v);
    v += vx_dpp64<0x141>(v);
    v += vx_dpp64<0x140>(v);
    if constexpr (LANES > 16) v += __shfl_xor(v, 16);
    if constexpr (LANES > 32) v += __shfl_xor(v, 32);
    return v;
}

// Cosines and signed sines of a lane's dims d .. d + 3: dim e becomes x[e] c[e] + partner s[e].
struct vx_turn {
    double c[4], s[4];
    uint32_t on;  // bit e: dim d + e is rotated
    __device__ __forceinline__ vx_turn(const vx_rotate_args& a, uint32_t t, uint32_t d) {
        on = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = s[e] = 0;
        if (d >= a.rotated) return;
        const double pos = a.positions[t];
        const uint32_t half = a.rotated / 2;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if (a.pairs && (e & 1)) {  // (the pair's other half: d is a multiple of 4)
                c[e] = c[e - 1];
                s[e] = -s[e - 1];
                if (d + e < a.rotated) on |= 1u << e;
                continue;
            }
            const uint32_t i = d + e;
            if (i >= a.rotated) continue;
            const bool second = !a.pairs && i >= half;
            vx_sin_cos(pos * a.freqs[a.pairs ? i / 2 : second ? i - half : i], s[e], c[e]);
            if (!second) s[e] = -s[e];
            on |= 1u << e;
        }
    }
};

// Dims d .. d + 3 of a row at p (element stride sd) and, if nothing else holds them, their partners.
__device__ __forceinline__ void vx_rotate_load(const vx_rotate_args& a, const float* p, int64_t sd, uint32_t d, vx_r4& x, vx_r4& y) {
    x = y = vx_r4{};
    if (d >= a.dim) return;
    const uint32_t half = a.rotated / 2;
    if (a.vec) {
        x = *(const vx_r4*)(p + d);
        if (!a.pairs && d < a.rotated) y = *(const vx_r4*)(p + (d < half ? d + half : d - half));
        return;
    }
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t i = d + e;
        if (i >= a.dim) continue;
        x[e] = p[i * sd];
        if (!a.pairs && i < a.rotated) y[e] = p[(i < half ? i + half : i - half) * sd];
    }
}

// The row's dims d .. d + 3, of which x and the partners y are loaded; w: the row's norm weight or null.
template <int LANES>
__device__ __forceinline__ vx_r4 vx_rotate_row(const vx_rotate_args& a, const vx_turn& t, const float* w, uint32_t d, vx_r4 x, vx_r4 y) {
    double v[4], u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = x[e];
    vx_r4 wx = {1.f, 1.f, 1.f, 1.f}, wy = wx;
    if (w) {
        int64_t one = 1;
        vx_rotate_load(a, w, one, d, wx, wy);
    }
    if (a.norm) {
        double m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) m = __builtin_fma(v[e], v[e], m);
        const double inv = 1.0 / __builtin_sqrt(vx_sum_lanes<LANES>(m) / a.dim + (double)a.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = v[e] * inv * wx[e];
            u[e] = y[e] * inv * wy[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = y[e];
    }
    if (a.pairs) {
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = v[e ^ 1];
    }
    vx_r4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (float)(t.on >> e & 1u ? __builtin_fma(v[e], t.c[e], u[e] * t.s[e]) : v[e]);
    return r;
}

__device__ __forceinline__ void vx_rotate_store(const vx_rotate_args& a, float* p, int64_t sd, uint32_t d, vx_r4 r) {
    if (d >= a.dim) return;
    if (a.vec) {
        *(vx_r4*)(p + d) = r;
        return;
    }
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
        if (d + e < a.dim) p[(d + e) * sd] = r[e];
}

// The rows of part `block` of a.blocks: a group of LANES lanes has a token's angles for a.run heads.
template <int LANES>
__device__ __forceinline__ void vx_rotate_rows(const vx_rotate_args& a, uint32_t block) {
    constexpr uint32_t GROUPS = 256 / LANES;
    const uint32_t d = 4 * (threadIdx.x % LANES), H = a.heads[0] + a.heads[1];
    const uint64_t jobs = (uint64_t)a.tokens * a.chunks;
    for (uint64_t n = (uint64_t)block * GROUPS + threadIdx.x / LANES; n < jobs; n += (uint64_t)a.blocks * GROUPS) {
        const uint32_t t = (uint32_t)(n / a.chunks), h0 = (uint32_t)(n - (uint64_t)t * a.chunks) * a.run;
        const vx_turn turn(a, t, d);
        for (uint32_t h = h0; h < min(H, h0 + a.run); ++h) {
            const uint32_t i = h >= a.heads[0], head = i ? h - a.heads[0] : h;
            const float* p = a.x[i] + (int64_t)t * a.xs[i][0] + (int64_t)head * a.xs[i][1];
            const float* w = a.w[i] ? a.w[i] + (uint64_t)head * a.ws[i] : nullptr;
            vx_r4 x, y;
            vx_rotate_load(a, p, a.xs[i][2], d, x, y);
            const vx_r4 r = vx_rotate_row<LANES>(a, turn, w, d, x, y);
            vx_rotate_store(a, a.y[i] + (int64_t)t * a.ys[i][0] + (int64_t)head * a.ys[i][1], a.ys[i][2], d, r);
        }
    }
}
