// vx_kv_rows.hpp — rows into the quantized cache and out of it.
//
// Eight lanes take a block of 32 values of K and of V, four values each, of one
// token, or of four whose slots are a record's group of four keys: their V bytes
// make up whole words, where one token's go byte by byte.
// 8000 tokens of 8 heads of 128 written and read back, K in 8 and V in 4 bits:
// 53.7 us token by token, by fours 42.8; 51000 tokens read back, both in 4 bits:
// 108 and 75.
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

// What a group of lanes does with its tokens, one or (many tokens) four: a token
// is taken alone, with the three after it where their slots are a record's group
// of four keys, or not at all where such a four before it has it.
struct vx_kv_tokens {
    uint32_t first, count;
    uint32_t fours, ones;  // bit i: token first + i
    __device__ __forceinline__ vx_kv_tokens(const vx_kv_rows_args& a, uint32_t n) : first(n), count(1), fours(0), ones(1) {
        if (!a.quads) return;
        first = 4 * n;
        count = min(4u, a.tokens - first);
        int32_t s[10];  // slots of tokens first - 3 to first + 6
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            const int64_t t = (int64_t)first + i - 3;
            s[i] = t >= 0 && t < a.tokens ? a.slots[t] : -1;
        }
        uint32_t lead = 0;  // bit i: the tokens from first - 3 + i on are such a four
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (s[i] >= 0 && (s[i] & 3) == 0 && s[i + 1] == s[i] + 1 && s[i + 2] == s[i] + 2 && s[i + 3] == s[i] + 3) lead |= 1u << i;
        fours = lead >> 3;
        ones = ~((lead | lead << 1 | lead << 2 | lead << 3) >> 3) & ((1u << count) - 1u);
    }
};

// Four tokens' scales, codes and sizes (a byte a token) of a block.
template <int BITS>
__device__ __forceinline__ void vx_kv_quantize4(const f4 (&x)[4], uint32_t (&w)[4], u2& d, uint32_t& lo, uint32_t& hi) {
    uint32_t h[4], e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float r;
        h[i] = __builtin_bit_cast(uint16_t, vx_kv_scale<BITS>(x[i], r));
        w[i] = vx_kv_codes<BITS>(x[i], r);
        e[i] = vx_kv_size(h[i]);
    }
    d = u2{h[0] | h[1] << 16, h[2] | h[3] << 16};
    lo = e[0] | e[1] << 16;  // sizes in halves, for packed maxima
    hi = e[2] | e[3] << 16;
}

template <int NP>
__device__ __forceinline__ uint32_t vx_kv_max_halves(uint32_t v) {
    typedef uint16_t us2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int o = 8; o < 8 * NP; o <<= 1) {
        const uint32_t w = (uint32_t)__shfl_xor((int)v, o);
        v = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, v), __builtin_bit_cast(us2, w)));
    }
    return v;
}

// Two size bytes (a half each) of a row whose block has sizes `own`, `least` at the least.
template <int NP>
__device__ __forceinline__ uint32_t vx_kv_row_sizes(uint32_t own, uint32_t least) {
    typedef uint16_t us2 __attribute__((ext_vector_type(2)));
    uint32_t top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, vx_kv_max_halves<NP>(own)), __builtin_bit_cast(us2, least)));
    // how far the block is below the largest one; not at all if it is all zeros
    const uint32_t lo = own & 0xFFFFu ? (top & 0xFFFFu) - (own & 0xFFFFu) : 0u, hi = own >> 16 ? (top >> 16) - (own >> 16) : 0u;
    if (__any((lo > VX_KV_APART) | (hi > VX_KV_APART))) {
        const uint32_t apart = vx_kv_max_halves<NP>(lo | hi << 16);
        top |= ((apart & 0xFFFFu) > VX_KV_APART ? 0x80u : 0u) | (apart >> 16 > VX_KV_APART ? 0x800000u : 0u);
    }
    return top;
}
__device__ __forceinline__ uint32_t vx_kv_bytes(uint32_t lo, uint32_t hi) { return (lo & 255u) | (lo >> 8 & 0xFF00u) | (hi & 255u) << 16 | (hi >> 16) << 24; }

// The dims 4 u + 2 p, + 1 of four keys (codes w, a byte a dim) as the record has them: V
template <int BITS>
__device__ __forceinline__ u2 vx_kv_v4(const uint32_t (&w)[4], int p) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = w[i] >> (16 * p) & 0xFFFFu;
    if constexpr (BITS == 8)
        return u2{(c[0] & 255u) | (c[1] & 255u) << 8 | (c[2] & 255u) << 16 | c[3] << 24,
                  c[0] >> 8 | (c[1] & 0xFF00u) | (c[2] >> 8) << 16 | (c[3] >> 8) << 24};
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = (c[i] | c[i] >> 4) & 255u;  // two nibbles
    return u2{c[0] | c[2] << 8 | c[1] << 16 | c[3] << 24, 0u};
}

template <int NB, int KB, int VB>
__device__ __forceinline__ void vx_kv_write_rows(const vx_kv_rows_args& a) {
    using R = vx_kv_rec<NB, KB, VB>;
    using PK = vx_kv_part<NB, KB>;
    using PV = vx_kv_part<NB, VB>;
    constexpr uint32_t NP = NB == 3 ? 4 : NB;  // lanes of a row: 8 NP, a power of two
    const uint64_t units = (uint64_t)a.groups * a.c.heads * NP;
    const uint32_t u = threadIdx.x & 7, b = (threadIdx.x >> 3) % NP;
    for (uint64_t n = (uint64_t)blockIdx.x * 32 + (threadIdx.x >> 3); n < units; n += (uint64_t)gridDim.x * 32) {
        const uint64_t th = n / NP;
        const uint32_t group = (uint32_t)(th / a.c.heads), h = (uint32_t)(th - (uint64_t)group * a.c.heads);
        const vx_kv_tokens run(a, group);
        const uint32_t d = 32 * b + 4 * u;
#pragma unroll 1
        for (uint32_t i = 0; i < run.count; ++i) {  // (the same for the row's lanes)
        const bool four = run.fours >> i & 1u;
        if (!four && !(run.ones >> i & 1u)) continue;
        const int64_t t = run.first + i;
        const uint32_t slot = (uint32_t)a.slots[t];
        const uint32_t page = slot >> a.c.page_shift, key = slot & ((1u << a.c.page_shift) - 1u), m = key & 15;
        if ((int32_t)slot < 0 || page >= a.c.pages) continue;
        uint8_t* rec = a.c.base + vx_kv_page(a.c, page, h, R::BYTES) + (uint64_t)(key >> 4) * R::BYTES;
        const float* kp = a.k + t * a.ks[0] + (int64_t)h * a.ks[1];
        const float* vp = a.v + t * a.vs[0] + (int64_t)h * a.vs[1];
        if (four) {
            uint32_t klo = 0, khi = 0, vlo = 0, vhi = 0;
            if (b < NB) {
                f4 x[4], y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = vx_kv_get4(kp + i * a.ks[0], a.ks[2], d, a.vec);
                    y[i] = vx_kv_get4(vp + i * a.vs[0], a.vs[2], d, a.vec);
                }
                uint32_t w[4];
                u2 sc;
                vx_kv_quantize4<KB>(x, w, sc, klo, khi);
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    uint8_t* p = rec + PK::at(b, (u >> 1) * 16 + m + i);
                    if constexpr (KB == 8) *(uint32_t*)(p + 4 * (u & 1)) = w[i];
                    else {
                        const uint32_t k4 = (w[i] & 15u) | ((w[i] >> 8 & 15u) << 16) | ((w[i] >> 16 & 15u) << 4) | ((w[i] >> 24) << 20);
                        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)k4, 0xB1, 0xF, 0xF, false);
                        if ((u & 1) == 0) *(uint32_t*)p = k4 | (o << 8);
                    }
                }
                if (u == 0) *(u2*)(rec + PK::VALS + ((m >> 2) * NB + b) * 8) = sc;
                vx_kv_quantize4<VB>(y, w, sc, vlo, vhi);
#pragma unroll
                for (uint32_t p = 0; p < 2; ++p) {
                    uint8_t* q = rec + R::V + PV::at(b, (m >> 2) * 16 + 2 * u + p);
                    const u2 v = vx_kv_v4<VB>(w, p);
                    if constexpr (VB == 8) *(u2*)q = v;
                    else *(uint32_t*)q = v.x;
                }
                if (u == 0) *(u2*)(rec + R::V + PV::VALS + ((m >> 2) * NB + b) * 8) = sc;
            }
            klo = vx_kv_row_sizes<NP>(klo, 0u), khi = vx_kv_row_sizes<NP>(khi, 0u);
            vlo = vx_kv_row_sizes<NP>(vlo, 0x00010001u), vhi = vx_kv_row_sizes<NP>(vhi, 0x00010001u);
            if (u == 0 && b == 0) {
                *(uint32_t*)(rec + R::K_SIZES + m) = vx_kv_bytes(klo, khi);
                *(uint32_t*)(rec + R::V_SIZES + m) = vx_kv_bytes(vlo, vhi);
            }
            continue;
        }
        uint32_t size = 0;  // of K above, of V below
        if (b < NB) {
            const f4 k = vx_kv_get4(kp, a.ks[2], d, a.vec), v = vx_kv_get4(vp, a.vs[2], d, a.vec);
            size = vx_kv_put_k<NB, KB>(rec, m, b, u, k) << 16;
            size |= vx_kv_put_v<NB, VB>(rec + R::V, m, b, u, v);
        }
        size = vx_kv_row_sizes<NP>(size, 1u);
        if (u == 0 && b == 0) {
            rec[R::K_SIZES + m] = (uint8_t)(size >> 16);
            rec[R::V_SIZES + m] = (uint8_t)size;
        }
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

// Dims 4 u .. of a key: K. One dword holds them (8 bits) or eight (4 bits).
template <int BITS>
__device__ __forceinline__ f4 vx_kv_k_values(uint32_t w, uint32_t u, float s) {
    f4 x;
    constexpr int at[4] = {0, 16, 4, 20};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = s * (float)(BITS == 8 ? (int)(w >> (8 * i) & 255u) - 128 : (int)(w >> (8 * (u & 1) + at[i]) & 15u) - 8);
    return x;
}
// Dims 4 u .. of key j of four: V, from the words of dims 4 u (+ 1) and 4 u + 2 (+ 1).
template <int BITS>
__device__ __forceinline__ f4 vx_kv_v_values(const u2 (&w)[2], uint32_t j, float s) {
    f4 x;
    const uint32_t sh = BITS == 8 ? 8 * j : 8 * ((j >> 1) | ((j & 1) << 1));
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        x[2 * p] = s * (float)(BITS == 8 ? (int)(w[p].x >> sh & 255u) - 128 : (int)(w[p].x >> sh & 15u) - 8);
        x[2 * p + 1] = s * (float)(BITS == 8 ? (int)(w[p].y >> sh & 255u) - 128 : (int)(w[p].x >> (sh + 4) & 15u) - 8);
    }
    return x;
}

template <int NB, int KB, int VB>
__device__ __forceinline__ void vx_kv_read_rows(const vx_kv_rows_args& a) {
    using R = vx_kv_rec<NB, KB, VB>;
    using PK = vx_kv_part<NB, KB>;
    using PV = vx_kv_part<NB, VB>;
    const uint64_t units = (uint64_t)a.groups * a.c.heads * NB;
    const uint32_t u = threadIdx.x & 7;
    for (uint64_t n = (uint64_t)blockIdx.x * 32 + (threadIdx.x >> 3); n < units; n += (uint64_t)gridDim.x * 32) {
        const uint32_t b = (uint32_t)(n % NB), d = 32 * b + 4 * u;
        const uint64_t th = n / NB;
        const uint32_t group = (uint32_t)(th / a.c.heads), h = (uint32_t)(th - (uint64_t)group * a.c.heads);
        const vx_kv_tokens run(a, group);
#pragma unroll 1
        for (uint32_t i = 0; i < run.count; ++i) {
        const bool four = run.fours >> i & 1u;
        if (!four && !(run.ones >> i & 1u)) continue;
        const int64_t t = run.first + i;
        const uint32_t slot = (uint32_t)a.slots[t];
        const uint32_t page = slot >> a.c.page_shift, key = slot & ((1u << a.c.page_shift) - 1u), m = key & 15;
        const bool in = (int32_t)slot >= 0 && page < a.c.pages;
        float* kp = a.k ? a.k + t * a.ks[0] + (int64_t)h * a.ks[1] : nullptr;
        float* vp = a.v ? a.v + t * a.vs[0] + (int64_t)h * a.vs[1] : nullptr;
        if (!in) {  // (a group of four lies outside as a whole: it is in one page)
            for (uint32_t i = 0; i < (four ? 4u : 1u); ++i) {
                if (kp) vx_kv_set4(kp + i * a.ks[0], a.ks[2], d, a.vec, f4{});
                if (vp) vx_kv_set4(vp + i * a.vs[0], a.vs[2], d, a.vec, f4{});
            }
            continue;
        }
        const uint8_t* rec = a.c.base + vx_kv_page(a.c, page, h, R::BYTES) + (uint64_t)(key >> 4) * R::BYTES;
        const uint32_t scales = ((m >> 2) * NB + b) * 8;
        const h4 ks = *(const h4*)(rec + PK::VALS + scales), vs = *(const h4*)(rec + R::V + PV::VALS + scales);
        u2 vw[2] = {};
        if (vp) {
#pragma unroll
            for (uint32_t p = 0; p < 2; ++p) {
                const uint8_t* q = rec + R::V + PV::at(b, (m >> 2) * 16 + 2 * u + p);
                if constexpr (VB == 8) vw[p] = *(const u2*)q;
                else vw[p].x = *(const uint32_t*)q;
            }
        }
        if (four) {  // (keys 4 g to 4 g + 3: m is the first)
            if (kp) {
                uint32_t w[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) w[i] = *(const uint32_t*)(rec + PK::at(b, (u >> 1) * 16 + m + i) + (KB == 8 ? 4 * (u & 1) : 0));
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) vx_kv_set4(kp + i * a.ks[0], a.ks[2], d, a.vec, vx_kv_k_values<KB>(w[i], u, (float)ks[i]));
            }
            if (vp) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) vx_kv_set4(vp + i * a.vs[0], a.vs[2], d, a.vec, vx_kv_v_values<VB>(vw, i, (float)vs[i]));
            }
            continue;
        }
        const uint32_t j = m & 3;
        const float kd = (float)(j & 2 ? (j & 1 ? ks.w : ks.z) : (j & 1 ? ks.y : ks.x)), vd = (float)(j & 2 ? (j & 1 ? vs.w : vs.z) : (j & 1 ? vs.y : vs.x));
        if (kp) {
            const uint32_t w = *(const uint32_t*)(rec + PK::at(b, (u >> 1) * 16 + m) + (KB == 8 ? 4 * (u & 1) : 0));
            vx_kv_set4(kp, a.ks[2], d, a.vec, vx_kv_k_values<KB>(w, u, kd));
        }
        if (vp) vx_kv_set4(vp, a.vs[2], d, a.vec, vx_kv_v_values<VB>(vw, j, vd));
        }
    }
}
