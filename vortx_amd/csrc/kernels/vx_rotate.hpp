// vx_rotate.hpp — rows of heads normed and rotated, four dims a lane.
//
// A workgroup has its tokens' angles in LDS for all its heads. Everything between the
// load and the store is f64 and rounded once: a key's codes in the cache follow from
// the result, and next to a border between two codes f32 sums of another order would
// give another code. f64 multiply-adds run at f32's rate here, two thirds of the time
// that the rows take from and to memory: 8000 tokens of 32 heads of 128, normed, 65 us,
// 4.0 TB/s, where a large copy reaches 4.8. A row's dims lie in one wave, which loads
// all of them (its partners' too) before it stores any, so a row may be overwritten in
// place.
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

// 1 / sqrt(a), the instruction's estimate made better twice; 0 for infinity, NaN for 0.
__device__ __forceinline__ double vx_inverse_root(double a) {
    double y = __builtin_amdgcn_rsq(a);
    const double h = 0.5 * a;
#pragma unroll
    for (int i = 0; i < 2; ++i) y = y * __builtin_fma(-h * y, y, 1.5);
    return a < __builtin_inf() ? y : a == a ? 0.0 : a;
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

// Cosines and sines of some tokens' pairs, in LDS: each is computed by one thread and
// read by all heads. Pair i of a token lies at (i % 4) quarter + i / 4, so that lanes
// with four neighbouring pairs each read neighbouring places.
struct vx_angles {
    double2* at;
    uint32_t first, quarter;  // first token; a quarter of a token's places
    // of n tokens (those past the last one: as the last)
    __device__ __forceinline__ vx_angles(const vx_rotate_args& a, double2* lds, uint32_t t0, uint32_t n) : at(lds), first(t0), quarter((a.rotated / 2 + 3) / 4) {
        const uint32_t half = a.rotated / 2;
#pragma unroll 1
        for (uint32_t j = threadIdx.x; j < n * half; j += 256) {
            const uint32_t t = j / half, i = j - t * half;
            const double pos = a.positions[min(t0 + t, a.tokens - 1u)];
            double2 v;
            vx_sin_cos(pos * a.freqs[i], v.y, v.x);
            at[(t * 4 + i % 4) * quarter + i / 4] = v;
        }
        __syncthreads();
    }
    __device__ __forceinline__ double2 get(uint32_t t, uint32_t i) const { return at[((t - first) * 4 + i % 4) * quarter + i / 4]; }
};
constexpr uint32_t VX_ANGLE_TOKENS = 11;  // of a workgroup at most: eight, and three that a group of four may reach past them
constexpr uint32_t VX_ANGLE_PLACES = VX_ANGLE_TOKENS * 128;
#define VX_ROTATE_TOKENS(LANES) ((LANES) > 32 ? 4 : 8)  // of a workgroup, where there are many

// What a lane's dims d .. d + 3 of a token are made of: dim e becomes (x[e] c[e] +
// partner s[e]) times the row's norm, with the cosine and the signed sine times the norm weights.
struct vx_turn {
    double c[4], s[4];
    uint32_t on;  // bit e: dim d + e is rotated (otherwise the partner is left out: it may be infinite)
    __device__ __forceinline__ vx_turn(const vx_rotate_args& a, const vx_angles& g, uint32_t t, uint32_t d) : on(0) {
        const uint32_t half = a.rotated / 2;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            c[e] = 1.0;
            s[e] = 0.0;
            const uint32_t i = d + e;
            if (i >= a.rotated) continue;
            on |= 1u << e;
            const bool second = a.pairs ? e & 1 : i >= half;  // (d is a multiple of 4)
            const double2 v = g.get(t, a.pairs ? i / 2 : second ? i - half : i);
            c[e] = v.x;
            s[e] = second ? v.y : -v.y;
        }
    }
    // times the weights of the dims and of their partners
    __device__ __forceinline__ void weigh(const vx_rotate_args& a, vx_r4 x, vx_r4 y) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e] *= x[e];
            s[e] *= a.pairs ? x[e ^ 1] : y[e];
        }
    }
};

// Dims d .. d + 3 of a row at p (element stride sd) and, if nothing else holds them,
// their partners. VEC: fours of dims, and their partners, are 16-byte aligned everywhere.
template <bool VEC>
__device__ __forceinline__ void vx_rotate_load(const vx_rotate_args& a, const float* p, int64_t sd, uint32_t d, vx_r4& x, vx_r4& y) {
    x = y = vx_r4{};
    if (d >= a.dim) return;
    const uint32_t half = a.rotated / 2;
    if constexpr (VEC) {
        x = *(const vx_r4*)(p + d);
        if (!a.pairs && d < a.rotated) y = *(const vx_r4*)(p + (d < half ? d + half : d - half));
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t i = d + e;
            if (i >= a.dim) continue;
            x[e] = p[i * sd];
            if (!a.pairs && i < a.rotated) y[e] = p[(i < half ? i + half : i - half) * sd];
        }
    }
}

// The row's dims d .. d + 3, of which x and the partners y are loaded. (VEC: all four are rotated or none.)
template <int LANES, bool VEC>
__device__ __forceinline__ vx_r4 vx_rotate_row(const vx_rotate_args& a, const vx_turn& t, vx_r4 x, vx_r4 y) {
    double v[4], r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = x[e];
        r[e] = v[e] * t.c[e];
    }
    if (VEC ? t.on != 0 : true) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (VEC || t.on >> e & 1u) r[e] = __builtin_fma(a.pairs ? v[e ^ 1] : (double)y[e], t.s[e], r[e]);
    }
    if (a.norm) {
        double m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) m = __builtin_fma(v[e], v[e], m);
        const double inv = vx_inverse_root(__builtin_fma(vx_sum_lanes<LANES>(m), a.per_dim, (double)a.eps));
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] *= inv;
    }
    return vx_r4{(float)r[0], (float)r[1], (float)r[2], (float)r[3]};
}

template <bool VEC>
__device__ __forceinline__ void vx_rotate_store(const vx_rotate_args& a, float* p, int64_t sd, uint32_t d, vx_r4 r) {
    if (d >= a.dim) return;
    if constexpr (VEC) {
        *(vx_r4*)(p + d) = r;
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (d + e < a.dim) p[(d + e) * sd] = r[e];
    }
}

// Workgroup `job` of one part's rows: q.block_tokens tokens (one, or as many as a
// workgroup has groups of LANES lanes, eight at most), q.run heads of them. A group has
// one token, and two heads under way.
template <int LANES, bool VEC>
__device__ __forceinline__ void vx_rotate_rows(const vx_rotate_args& a, const vx_rotate_rows_args& q, uint32_t job, double2* lds) {
    constexpr uint32_t GROUPS = 256 / LANES;
    const uint32_t d = 4 * (threadIdx.x % LANES), g = threadIdx.x / LANES, n = q.block_tokens;
    const uint32_t t0 = job / q.chunks * n, h0 = job % q.chunks * q.run, end = min(h0 + q.run, q.heads);
    const vx_angles angles(a, lds, t0, n);
    const uint32_t t = t0 + (n > 1 ? g % VX_ROTATE_TOKENS(LANES) : 0u), step = n > 1 ? GROUPS / VX_ROTATE_TOKENS(LANES) : GROUPS;
    if (t >= a.tokens) return;
    vx_turn turn(a, angles, t, d);
    vx_r4 wx, wy;
    const bool each = q.w && q.ws;  // a weight for each head
    if (q.w && !each) {
        vx_rotate_load<VEC>(a, q.w, 1, d, wx, wy);
        turn.weigh(a, wx, wy);
    }
    const float* p = q.x + t * q.xs[0];
    float* o = q.y + t * q.ys[0];
#pragma unroll 1
    for (uint32_t h = h0 + (n > 1 ? g / VX_ROTATE_TOKENS(LANES) : g); h < end; h += 2 * step) {
        vx_r4 x[2], y[2];
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j)
            if (h + j * step < end) vx_rotate_load<VEC>(a, p + (h + j * step) * q.xs[1], q.xs[2], d, x[j], y[j]);
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) {
            const uint32_t k = h + j * step;
            if (k >= end) continue;
            vx_turn own = turn;
            if (each) {
                vx_rotate_load<VEC>(a, q.w + (uint64_t)k * q.ws, 1, d, wx, wy);
                own.weigh(a, wx, wy);
            }
            vx_rotate_store<VEC>(a, o + k * q.ys[1], q.ys[2], d, vx_rotate_row<LANES, VEC>(a, own, x[j], y[j]));
        }
    }
}
