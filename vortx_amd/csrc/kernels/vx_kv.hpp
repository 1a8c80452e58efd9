// vx_kv.hpp — layout of the quantized key/value cache, and its decoding.
//
// A page holds page_tokens (a power of two >= 16) tokens of every key/value
// head: page p at base + p * page_bytes, in it head h's page_tokens / 16
// records, one per 16 tokens. A record is laid out as the 16 x 16 x 32 matrix
// instructions take its parts, so that attention loads fragments without a
// transpose and single tokens can still be written on their own:
//
//   K values | K scales | V values | V scales | K sizes | V sizes
//
// Values of one kind: "lane" l = 16 g + m (m, g in 0..15, 0..3) owns the
// values that lane l of a wave feeds to the matrix cores, LB = NB * 8 bytes
// (8 bits) or NB * 4 (4 bits) of them, NB = dim / 32, in pieces of 16 bytes
// (the last one may be shorter): piece p of all lanes, then piece p + 1.
// Lanes' bytes by 32-dim block b:
//   K  key m of the record, dims 32 b + 8 g + i, i = 0..7
//      8 bits: byte i of 8; 4 bits: nibble {0,4,1,5,2,6,3,7}[i] of a dword
//   V  dims 32 b + 2 m + v (v = 0, 1) of keys 4 g + j, j = 0..3
//      8 bits: byte 4 v + j; 4 bits: nibble v of byte {0,2,1,3}[j]
// Values are stored with 128 (8 bits) or 8 (4 bits) added. The orders inside
// a dword are those that masks and byte permutes unpack to pairs of f16.
// Scales: f16, [g][b][4]: of K for keys 4 g + j, of V the same. Sizes: a byte a
// key, 16 above the exponent of the largest of its scales (1 to 31; an f16
// below its normal numbers counts as 2^-15; where all are zero, K has 0 and V
// 1), with 128 added where another one that is not zero has an exponent more
// than VX_KV_APART lower, and 255 where one is not finite.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../vx_kargs.h"

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// a and b as two f16 terms each: hi rounds, lo what that left out. The empty
// asm keeps one rounding for both uses of hi: the compiler otherwise folds a
// multiply before it into v_fma_mixlo for one of them, which rounds once
// instead of twice, and lo is then off by hi's last place.
__device__ __forceinline__ void vx_two_terms(float a, float b, h2& hi, h2& lo) {
    uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), h2));
    asm("" : "+v"(u));
    hi = __builtin_bit_cast(h2, u);
    lo = __builtin_convertvector((f2{a - (float)hi.x, b - (float)hi.y}), h2);
}

// The same with -1.0 in a register: a multiply-add takes hi as it is (v_fma_mix).
__device__ __forceinline__ void vx_two_terms(float a, float b, float minus, h2& hi, h2& lo) {
    hi = __builtin_convertvector((f2{a, b}), h2);
    lo = __builtin_convertvector((f2{__builtin_fmaf((float)hi.x, minus, a), __builtin_fmaf((float)hi.y, minus, b)}), h2);
}

// w0 * d.x and w1 * d.y as two f16 terms each, lo from the exact product. `zero`
// is -0.0 in a register: a product written as a multiply-add takes the f16
// operand as it is (v_fma_mix), a multiplication would convert it first.
__device__ __forceinline__ void vx_two_terms(float w0, float w1, h2 d, float zero, h2& hi, h2& lo) {
    uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{__builtin_fmaf(w0, (float)d.x, zero),
                                                                         __builtin_fmaf(w1, (float)d.y, zero)}), h2));
    asm("" : "+v"(u));
    hi = __builtin_bit_cast(h2, u);
    lo = __builtin_convertvector((f2{__builtin_fmaf(w0, (float)d.x, -(float)hi.x), __builtin_fmaf(w1, (float)d.y, -(float)hi.y)}), h2);
}

// Bytes of a record's parts.
template <int NB, int BITS>
struct vx_kv_part {
    static constexpr uint32_t LB = NB * BITS;        // bytes per lane
    static constexpr uint32_t VALS = 64 * LB;        // values of 16 tokens
    static constexpr uint32_t SCALES = 32 * NB;      // scales of 16 tokens
    static constexpr uint32_t BYTES = VALS + SCALES;
    static constexpr uint32_t FULL = LB / 16, REST = LB % 16;  // pieces of 16 bytes, and what is left
    // offset of lane l's bytes of block b
    __host__ __device__ static constexpr uint32_t at(uint32_t b, uint32_t l) {
        const uint32_t o = b * BITS, p = o / 16;
        return p < FULL ? p * 1024 + l * 16 + o % 16 : FULL * 1024 + l * REST + o % 16;
    }
};

template <int NB, int KB, int VB>
struct vx_kv_rec {
    static constexpr uint32_t V = vx_kv_part<NB, KB>::BYTES, K_SIZES = V + vx_kv_part<NB, VB>::BYTES, V_SIZES = K_SIZES + 16,
                              BYTES = V_SIZES + 16;
};
constexpr uint32_t VX_KV_APART = 10;
__device__ __forceinline__ uint32_t vx_kv_size(uint32_t d) {  // of a scale's bits
    d &= 0x7FFFu;
    return d >= 0x7C00u ? 255u : d ? (d >> 10) + 1u : 0u;
}

__device__ __forceinline__ uint64_t vx_kv_page(const vx_kv_geom& c, uint32_t page, uint32_t head, uint32_t rec_bytes) {
    return page * c.page_bytes + (uint64_t)(head << (c.page_shift - 4)) * rec_bytes;
}

// A lane's bytes of a record's values, as dwords.
template <int NB, int BITS>
__device__ __forceinline__ void vx_kv_load(const uint8_t* p, uint32_t lane, uint32_t (&w)[NB * BITS / 4]) {
    using P = vx_kv_part<NB, BITS>;
#pragma unroll
    for (uint32_t i = 0; i < P::FULL; ++i) {
        const u4 v = *(const u4*)(p + i * 1024 + lane * 16);
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
    const uint32_t* r = (const uint32_t*)(p + P::FULL * 1024 + lane * P::REST);
#pragma unroll
    for (uint32_t i = 0; i < P::REST / 4; ++i) w[4 * P::FULL + i] = r[i];
}

// Four values as f16 from a dword of bytes (value + 128): the byte below a
// 0x64 is 1024 + byte in f16, and the subtraction is exact.
__device__ __forceinline__ void vx_unpack8(uint32_t w, h2& a, h2& b) {
    const h2 off = {(_Float16)1152.f, (_Float16)1152.f};
    a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
    b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
}

// Nibbles 0 and 4 (value + 8) of w as f16; of w >> 4 the next pair, and so on.
__device__ __forceinline__ h2 vx_unpack4(uint32_t w) {
    const h2 off = {(_Float16)1032.f, (_Float16)1032.f};
    return __builtin_bit_cast(h2, (w & 0x000F000Fu) | 0x64006400u) - off;
}
// Nibbles 1 and 5: 1024 + 16 n, brought down by one exact multiply-add.
__device__ __forceinline__ h2 vx_unpack4_high(uint32_t w) {
    const h2 m = {(_Float16)0.0625f, (_Float16)0.0625f}, off = {(_Float16)-72.f, (_Float16)-72.f};
    return __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & 0x00F000F0u) | 0x64006400u), m, off);
}

// The K fragment of block b: 8 values along the dim of the lane's key.
template <int NB, int BITS>
__device__ __forceinline__ h8 vx_kv_kfrag(const uint32_t (&w)[NB * BITS / 4], int b) {
    h2 p[4];
    if constexpr (BITS == 8) {
        vx_unpack8(w[2 * b], p[0], p[1]);
        vx_unpack8(w[2 * b + 1], p[2], p[3]);
    } else {
        p[0] = vx_unpack4(w[b]);
        p[1] = vx_unpack4_high(w[b]);
        p[2] = vx_unpack4(w[b] >> 8);
        p[3] = vx_unpack4_high(w[b] >> 8);
    }
    return h8{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
}

// The V half fragment of dim 32 b + 2 m + v: keys 4 g + 0..3.
template <int NB, int BITS>
__device__ __forceinline__ void vx_kv_vfrag(const uint32_t (&w)[NB * BITS / 4], int b, int v, h2& lo, h2& hi) {
    if constexpr (BITS == 8) {
        vx_unpack8(w[2 * b + v], lo, hi);
    } else if (v == 0) {
        lo = vx_unpack4(w[b]);
        hi = vx_unpack4(w[b] >> 8);
    } else {
        lo = vx_unpack4_high(w[b]);
        hi = vx_unpack4_high(w[b] >> 8);
    }
}
