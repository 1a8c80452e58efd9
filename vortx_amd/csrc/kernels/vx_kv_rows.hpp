// vx_kv_rows.hpp — rows into the quantized cache and out of it.
//
// Eight lanes take a block of 32 values of K and of V, four values each.
// Quantization of a block x: d = f16(max|x| / 127) and q = clamp(rint(x r),
// -127, 127) at 8 bits; d = f16(m / -8) with m the value of the largest
// magnitude (the positive one of two) and q = clamp(rint(x r), -8, 7) at 4,
// r = 1 / d or 0. A block with a NaN or an infinity, or one too large for d,
// has a d that is not finite and reads as NaN.
#pragma once
#include "vx_dpp.hpp"
#include "vx_kv.hpp"

#pragma clang fp contract(off)

__device__ __forceinline__ f4 vx_kv_get4(const float* p, int64_t sd, uint32_t d, bool vec) {
    if (vec) return *(const f4*)(p + d);
    return f4{p[d * sd], p[(d + 1) * sd], p[(d + 2) * sd], p[(d + 3) * sd]};
}

// f32 -> f16 of a value that is a rounded f32 (no folding into a mixed multiply)
__device__ __forceinline__ _Float16 vx_kv_half(float v) {
    asm("" : "+v"(v));
    return (_Float16)v;
}

// The scale of the block whose four values are x; r its reciprocal.
template <int BITS>
__device__ __forceinline__ _Float16 vx_kv_scale(f4 x, float& r) {
    float d;
    if constexpr (BITS == 8) {
        // as bit patterns: a NaN is larger than any number
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        auto up = [](uint32_t v, uint32_t o) { return max(v, o); };
        m = up(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
        m = up(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
        m = up(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));
        d = __builtin_bit_cast(float, m) / 127.0f;
    } else {
        // magnitude above, sign (1: positive) in the lowest bit: the largest value, the positive one of two
        uint32_t hi = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = __float_as_uint(x[i]);
            hi = max(hi, (u << 1) | (~u >> 31));
        }
        auto up = [](uint32_t v, uint32_t o) { return max(v, o); };
        hi = up(hi, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi, 0xB1, 0xF, 0xF, false));
        hi = up(hi, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi, 0x4E, 0xF, 0xF, false));
        hi = up(hi, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi, 0x141, 0xF, 0xF, false));
        const float a = __builtin_bit_cast(float, hi >> 1);
        d = ((hi & 1u) ? a : -a) / -8.0f;
    }
    _Float16 h = vx_kv_half(d);
    float f = (float)h;
    if (!(fabsf(f) < __builtin_inff())) h = (_Float16)(f = __builtin_nanf(""));
    r = f != 0.f ? 1.0f / f : 0.f;
    return h;
}

// Stored codes of four values, one a byte.
template <int BITS>
__device__ __forceinline__ uint32_t vx_kv_codes(f4 x, float r) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float y = __builtin_rintf(x[i] * r);  // (NaN: clamped to the lower bound)
        const int q = BITS == 8 ? (int)__builtin_amdgcn_fmed3f(y, -127.f, 127.f) + 128 : (int)__builtin_amdgcn_fmed3f(y, -8.f, 7.f) + 8;
        w |= ((uint32_t)q & (BITS == 8 ? 255u : 15u)) << (8 * i);
    }
    return w;
}

template <int NB, int BITS>
__device__ __forceinline__ uint32_t vx_kv_put_k(uint8_t* rec, uint32_t key, uint32_t b, uint32_t u, f4 x) {
    using P = vx_kv_part<NB, BITS>;
    float r;
    const _Float16 d = vx_kv_scale<BITS>(x, r);
    const uint32_t w = vx_kv_codes<BITS>(x, r);  // dims 32 b + 4 u + 0..3: of "lane" g = u / 2
    uint8_t* p = rec + P::at(b, (u >> 1) * 16 + key);
    if constexpr (BITS == 8) {
        *(uint32_t*)(p + 4 * (u & 1)) = w;
    } else {
        // dims 0..3 of the dword are nibbles 0 4 1 5, dims 4..7 nibbles 2 6 3 7
        const uint32_t n = (w & 15u) | ((w >> 8 & 15u) << 16) | ((w >> 16 & 15u) << 4) | ((w >> 24) << 20);
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)n, 0xB1, 0xF, 0xF, false);
        if ((u & 1) == 0) *(uint32_t*)p = n | (o << 8);
    }
    if (u == 0) *(_Float16*)(rec + P::VALS + ((key >> 2) * NB + b) * 8 + (key & 3) * 2) = d;
    return vx_kv_size(__builtin_bit_cast(uint16_t, d));
}

template <int NB, int BITS>
__device__ __forceinline__ uint32_t vx_kv_put_v(uint8_t* rec, uint32_t key, uint32_t b, uint32_t u, f4 x) {
    using P = vx_kv_part<NB, BITS>;
    float r;
    const _Float16 d = vx_kv_scale<BITS>(x, r);
    const uint32_t w = vx_kv_codes<BITS>(x, r);  // dims 32 b + 2 m + v: m = 2 u, 2 u + 1
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t) {
        uint8_t* p = rec + P::at(b, (key >> 2) * 16 + 2 * u + t);
        const uint32_t c = w >> (16 * t);
        if constexpr (BITS == 8) {
            p[key & 3] = (uint8_t)c;
            p[4 + (key & 3)] = (uint8_t)(c >> 8);
        } else {
            const uint32_t j = key & 3;
            p[(j >> 1) | ((j & 1) << 1)] = (uint8_t)((c & 15u) | ((c >> 8 & 15u) << 4));
        }
    }
    if (u == 0) *(_Float16*)(rec + P::VALS + ((key >> 2) * NB + b) * 8 + (key & 3) * 2) = d;
    return vx_kv_size(__builtin_bit_cast(uint16_t, d));
}

template <int NB, int KB, int VB>
__device__ __forceinline__ void vx_kv_write_rows(const vx_kv_rows_args& a) {
    using R = vx_kv_rec<NB, KB, VB>;
    constexpr uint32_t NP = NB == 3 ? 4 : NB;  // lanes of a row: 8 NP, a power of two
    const uint64_t units = (uint64_t)a.tokens * a.c.heads * NP;
    const uint32_t u = threadIdx.x & 7, b = (threadIdx.x >> 3) % NP;
    for (uint64_t n = (uint64_t)blockIdx.x * 32 + (threadIdx.x >> 3); n < units; n += (uint64_t)gridDim.x * 32) {
        const uint64_t th = n / NP;
        const uint32_t t = (uint32_t)(th / a.c.heads), h = (uint32_t)(th - (uint64_t)t * a.c.heads);
        const uint32_t slot = (uint32_t)a.slots[t];
        const uint32_t page = slot >> a.c.page_shift, key = slot & ((1u << a.c.page_shift) - 1u);
        if ((int32_t)slot < 0 || page >= a.c.pages) continue;  // (the same for the row's lanes)
        uint8_t* rec = a.c.base + vx_kv_page(a.c, page, h, R::BYTES) + (uint64_t)(key >> 4) * R::BYTES;
        uint32_t size = 0;  // of K above, of V below
        if (b < NB) {
            const uint32_t d = 32 * b + 4 * u;
            const f4 k = vx_kv_get4(a.k + (int64_t)t * a.ks[0] + (int64_t)h * a.ks[1], a.ks[2], d, a.vec);
            const f4 v = vx_kv_get4(a.v + (int64_t)t * a.vs[0] + (int64_t)h * a.vs[1], a.vs[2], d, a.vec);
            size = vx_kv_put_k<NB, KB>(rec, key & 15, b, u, k) << 16;
            size |= vx_kv_put_v<NB, VB>(rec + R::V, key & 15, b, u, v);
        }
#pragma unroll
        for (uint32_t o = 8; o < 8 * NP; o <<= 1) {
            const uint32_t w = (uint32_t)__shfl_xor((int)size, (int)o);
            size = max(size & 0xFFFF0000u, w & 0xFFFF0000u) | max(size & 255u, w & 255u);
        }
        if (u == 0 && b == 0) {
            rec[R::K_SIZES + (key & 15)] = (uint8_t)(size >> 16);
            rec[R::V_SIZES + (key & 15)] = (uint8_t)size;
        }
    }
}

__device__ __forceinline__ void vx_kv_set4(float* p, int64_t sd, uint32_t d, bool vec, f4 x) {
    if (vec) {
        *(f4*)(p + d) = x;
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) p[(d + i) * sd] = x[i];
}

template <int NB, int KB, int VB>
__device__ __forceinline__ void vx_kv_read_rows(const vx_kv_rows_args& a) {
    using PK = vx_kv_part<NB, KB>;
    using PV = vx_kv_part<NB, VB>;
    constexpr uint32_t REC = vx_kv_rec<NB, KB, VB>::BYTES;
    const uint64_t units = (uint64_t)a.tokens * a.c.heads * NB;
    const uint32_t u = threadIdx.x & 7;
    for (uint64_t n = (uint64_t)blockIdx.x * 32 + (threadIdx.x >> 3); n < units; n += (uint64_t)gridDim.x * 32) {
        const uint32_t b = (uint32_t)(n % NB);
        const uint64_t th = n / NB;
        const uint32_t t = (uint32_t)(th / a.c.heads), h = (uint32_t)(th - (uint64_t)t * a.c.heads);
        const uint32_t slot = (uint32_t)a.slots[t];
        const uint32_t page = slot >> a.c.page_shift, key = slot & ((1u << a.c.page_shift) - 1u);
        const bool in = (int32_t)slot >= 0 && page < a.c.pages;
        const uint32_t d = 32 * b + 4 * u, m = key & 15, sc = ((m >> 2) * NB + b) * 8 + (m & 3) * 2;
        const uint8_t* rec = a.c.base + vx_kv_page(a.c, in ? page : 0u, h, REC) + (in ? (uint64_t)(key >> 4) * REC : 0u);
        if (a.k) {
            f4 x = {};
            if (in) {
                const uint8_t* p = rec + PK::at(b, (u >> 1) * 16 + m);
                const float s = (float)*(const _Float16*)(rec + PK::VALS + sc);
                if constexpr (KB == 8) {
                    const uint32_t w = *(const uint32_t*)(p + 4 * (u & 1));
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = s * (float)((int)(w >> (8 * i) & 255u) - 128);
                } else {
                    const uint32_t w = *(const uint32_t*)p >> (8 * (u & 1));
                    constexpr int at[4] = {0, 16, 4, 20};
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = s * (float)((int)(w >> at[i] & 15u) - 8);
                }
            }
            vx_kv_set4(a.k + (int64_t)t * a.ks[0] + (int64_t)h * a.ks[1], a.ks[2], d, a.vec, x);
        }
        if (a.v) {
            f4 x = {};
            if (in) {
                const uint8_t* vrec = rec + PK::BYTES;
                const float s = (float)*(const _Float16*)(vrec + PV::VALS + sc);
                const uint32_t j = m & 3;
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    const uint8_t* p = vrec + PV::at(b, (m >> 2) * 16 + 2 * u + i);
                    if constexpr (VB == 8) {
                        x[2 * i] = s * (float)((int)p[j] - 128);
                        x[2 * i + 1] = s * (float)((int)p[4 + j] - 128);
                    } else {
                        const uint32_t w = p[(j >> 1) | ((j & 1) << 1)];
                        x[2 * i] = s * (float)((int)(w & 15u) - 8);
                        x[2 * i + 1] = s * (float)((int)(w >> 4) - 8);
                    }
                }
            }
            vx_kv_set4(a.v + (int64_t)t * a.vs[0] + (int64_t)h * a.vs[1], a.vs[2], d, a.vec, x);
        }
    }
}
