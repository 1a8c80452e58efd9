// vx_attn_tile.hpp — attention of many query rows over the quantized cache.
//
// A workgroup takes 128 or 256 query rows of a sequence and key/value head, 32
// to a wave, and goes over their keys 32 at a time. The waves decode a tile of
// keys once into LDS, as operands of the 32 x 32 x 16 matrix instructions, while
// the tile before is computed from the other buffer:
// each value is scale x number, 19 bits, held as two f16 terms whose sum is
// exact: hi rounds the product, lo = fma(number, scale, -hi). The scales of each
// four keys are first brought below 2 by a power of two, which K's scores take
// back as a factor, and V's weights: w = exp2(score + e - M), so V of any
// magnitude fills f16's range, and the weights' sum takes w 2^-e. Four keys that
// are more than 2^10 apart, some of which a row may not see, have a power each
// (2 % of the time below; of 78 us for packed documents of dim 64, 7). Slots that
// were never written may hold anything: sizes above 31 are no key's, and a scale
// of V that its size does not allow is taken as 0.
// (With K as whole numbers, exact in one term, and its scales on the 32-dim
// products, a tile had 8 matrix instructions fewer and 64 multiply-adds and 32
// registers a wave more: 430 us where this took 415, 4096 causal tokens of
// 32 heads of 128.)
// q is two f16 terms (22 bits, a power of two per row), and so are the weights;
// of the product's terms the one of two lows is left out (2^-22). M follows the
// maximum of score + e by steps of more than 2^8 only: the weights have f16's
// range for that, and most tiles leave the sums O^T = V^T P^T unscaled. P^T is
// used in the registers S^T was left in: the order of keys within a
// contraction is free, and V is laid out to it.
// Bound: matrix and vector issue, which take turns more than they overlap (48
// 32-cycle matrix instructions and 330 vector ones a wave and tile at 128, 450
// with a cap): 4096 causal tokens of 32 heads of 128, capped, 428 us, 321
// TFLOP/s of attention, 960 of f16 products (matrix cores busy 44 %, vector
// issue 53 %).
#pragma once
#include "vx_attn.hpp"

typedef float f16v __attribute__((ext_vector_type(16)));

template <int NB, int KB, int VB, int WAVES>
struct vx_tile {
    using PK = vx_kv_part<NB, KB>;
    using PV = vx_kv_part<NB, VB>;
    using R = vx_kv_rec<NB, KB, VB>;
    static constexpr uint32_t REC = R::BYTES;
    static constexpr uint32_t THREADS = 64 * WAVES, ROWS = 32 * WAVES;
    static constexpr int ITEMS = (128 * NB + THREADS - 1) / THREADS;  // a thread's pieces of a tile: one lane's bytes of a block

    // tiles between barriers: two where LDS holds them, so that the waves of a
    // SIMD drift apart and one's matrix instructions run beside the other's softmax
    static constexpr int PERIOD = WAVES == 8 || NB <= 2 ? 2 : 1;

    struct tile {
        h8 k[NB * 2 * 2 * 64];  // [block][16 dims][hi, lo][half, key]
        h8 v[NB * 2 * 2 * 64];  // [block][16 keys][hi, lo][half, dim]
        f2 e[8];                // of four keys: 2^exponent of K's scales (negative: see key), exponent of V's
        f2 key[32];             // of keys far apart: what their own powers are to those, factor and difference
        uint32_t bad[8];        // their V scales that are not finite, bit 4 block + key
    };

    struct raw {  // a thread's pieces as loaded
        uint32_t k[ITEMS][KB / 4], v[ITEMS][VB / 4], d[ITEMS][2];
        uint16_t kd[ITEMS];
        uint32_t ke, e;  // sizes: of K for the four keys of key m, of V for keys 4 g
    };

    template <int BITS>
    static __device__ __forceinline__ void load_block(const uint8_t* p, int b, uint32_t lane, uint32_t (&w)[BITS / 4]) {
        const uint8_t* q = p + vx_kv_part<NB, BITS>::at(b, lane);
        if constexpr (BITS == 8) {
            const u2 v = *(const u2*)q;
            w[0] = v.x, w[1] = v.y;
        } else {
            w[0] = *(const uint32_t*)q;
        }
    }

    static constexpr uint32_t FAR = 10;  // f16 holds both terms of a key that is 2^10 below to 22 bits
    static __device__ __forceinline__ int power(uint32_t size) { return max((int)size - 16, -15); }  // (of no key: size 0)

    // the record of the 16 keys from key on; past the end the last one
    static __device__ __forceinline__ const uint8_t* record(const vx_attn_args& a, vx_scalar_i32 table, const uint8_t* base, int key, int last) {
        key = min(key, last);
        const uint32_t page = min((uint32_t)table[(uint32_t)key >> a.c.page_shift], a.c.pages - 1u);
        return base + page * a.c.page_bytes + (((uint32_t)key & ((1u << a.c.page_shift) - 1u)) >> 4) * REC;
    }

    static __device__ __forceinline__ void load(const vx_attn_args& a, vx_scalar_i32 table, const uint8_t* base, int k0, int last, raw& r) {
        const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), rec = wave & 1, lane = t & 63, m = lane & 15, g = lane >> 4;
        const uint8_t* p = record(a, table, base, k0 + 16 * (int)rec, last);
        const uint8_t* sc = p + PK::BYTES + PV::VALS + g * (8 * NB);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int b = (int)(wave >> 1) + WAVES / 2 * i;
            if (NB % (WAVES / 2) == 0 || b < NB) {
                load_block<KB>(p, b, lane, r.k[i]);
                load_block<VB>(p + PK::BYTES, b, lane, r.v[i]);
                const u2 d = *(const u2*)(sc + 8 * b);
                r.d[i][0] = d.x, r.d[i][1] = d.y;
                r.kd[i] = *(const uint16_t*)(p + PK::VALS + ((m >> 2) * NB + b) * 8 + (m & 3) * 2);
            }
        }
        r.ke = ((const uint32_t*)(p + R::K_SIZES))[m >> 2];
        r.e = ((const uint32_t*)(p + R::V_SIZES))[g];
    }

    // decodes a thread's pieces into the tile of the keys from k0 on
    static __device__ __forceinline__ void store(const vx_attn_args& a, vx_scalar_i32 table, const uint8_t* base, raw& r, tile& s, int k0, int last) {
        const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), rec = wave & 1, lane = t & 63, m = lane & 15, g = lane >> 4;
        uint32_t bad = 0;
        // largest of four sizes, and whether another is far below it
        auto largest = [](uint32_t e, bool& far) {
            typedef uint16_t us2 __attribute__((ext_vector_type(2)));
            const us2 lo = __builtin_bit_cast(us2, e & 0x00FF00FFu), hi = __builtin_bit_cast(us2, e >> 8 & 0x00FF00FFu);
            const us2 most = __builtin_elementwise_max(lo, hi), least = __builtin_elementwise_min(lo, hi);
            const uint32_t top = max((uint32_t)most.x, (uint32_t)most.y);
            far = top > min((uint32_t)least.x, (uint32_t)least.y) + FAR;
            return top;
        };
        bool far, kfar;
        uint32_t size = largest(r.e, far), ksize = largest(r.ke, kfar);
        auto below = [](uint32_t v) { return (_Float16)__builtin_ldexpf(1.f, -power(v)); };
        h2 f0, f1;  // what V's four keys and K's key are brought down by
        _Float16 fk;
        float sign = 1.f;
        // (seldom: out of the way of the rest, 2 us of 196, eight trees of 61 drafts)
        if (__builtin_expect(k0 + 32 > last + 1 || __any(far | kfar | (max(size, ksize) > 31u)), 0)) {
            // scales of keys that do not exist, which may be anything: 0; those that are not finite: 0, and noted
            const int valid = last + 1 - (k0 + 16 * (int)rec + 4 * (int)g);
            auto fix = [&](uint32_t d, int i) {
                if (valid <= 2 * i || (d & 0x7FFFu) >= 0x7C00u) d &= 0xFFFF0000u;
                if (valid <= 2 * i + 1 || (d >> 16 & 0x7FFFu) >= 0x7C00u) d &= 0x0000FFFFu;
                return d;
            };
#pragma unroll
            for (int n = 0; n < ITEMS; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) r.d[n][i] = fix(r.d[n][i], i);
            const uint32_t* sc = (const uint32_t*)(record(a, table, base, k0 + 16 * (int)rec, last) + PK::BYTES + PV::VALS + g * (8 * NB));
            uint32_t e[4] = {};
#pragma unroll 1
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t v = vx_kv_size(sc[2 * b + (i >> 1)] >> (16 * (i & 1)));
                    if (valid <= i) continue;
                    if (v == 255u) bad |= 1u << (4 * b + i);
                    else e[i] = max(e[i], v);
                }
            size = max(max(e[0], e[1]), max(e[2], e[3]));
            uint32_t least = size;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (valid > i) least = min(least, e[i]);
            far = size > least + FAR;
            uint32_t own[4], kown = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) own[i] = far ? e[i] : size;
            f0 = h2{below(own[0]), below(own[1])}, f1 = h2{below(own[2]), below(own[3])};
            // K's keys that do not exist, are not finite or were never written: the others' exponent
            const int kvalid = last + 1 - (k0 + 16 * (int)rec + 4 * (int)(m >> 2));
            ksize = 0;
            least = 255u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t v = r.ke >> (8 * i) & 255u;
                if (i < kvalid && v < 32u) {
                    ksize = max(ksize, v);
                    least = min(least, v);
                    if (i == (int)(m & 3)) kown = v;
                }
            }
            kfar = ksize > least + FAR;
            if (!kfar) kown = ksize;
            fk = below(kown);
            if (far | kfar) sign = -1.f;
            if (wave < 2 && (m >> 2) == g) {
                const uint32_t v = m & 2 ? (m & 1 ? own[3] : own[2]) : (m & 1 ? own[1] : own[0]);
                s.key[rec * 16 + m] = f2{__builtin_ldexpf(1.f, power(kown) - power(ksize)), (float)(power(v) - power(size))};
            }
        } else {
            const _Float16 f = below(size);
            f0 = f1 = h2{f, f};
            fk = below(ksize);
            // a scale of V above what the sizes say is of a key that was never
            // written, which no row sees: 0, so that its weights' zeros stay zeros
            typedef uint16_t us2 __attribute__((ext_vector_type(2)));
            us2 most = {};
#pragma unroll
            for (int n = 0; n < ITEMS; ++n)
#pragma unroll
                for (int i = 0; i < 2 && (NB % (WAVES / 2) == 0 || (int)(wave >> 1) + WAVES / 2 * n < NB); ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(us2, r.d[n][i] & 0x7FFF7FFFu));
            const uint32_t limit = max(size, 1u) << 10;
            if (__builtin_expect(__any(max((uint32_t)most.x, (uint32_t)most.y) >= limit), 0)) {
#pragma unroll
                for (int n = 0; n < ITEMS; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if ((r.d[n][i] & 0x7FFFu) >= limit) r.d[n][i] &= 0xFFFF0000u;
                        if ((r.d[n][i] >> 16 & 0x7FFFu) >= limit) r.d[n][i] &= 0x0000FFFFu;
                    }
            }
        }
        if (wave < 2 && m == 4 * g) s.e[rec * 4 + g] = f2{__builtin_ldexpf(sign, power(ksize)), (float)power(size)};
        if (wave < 2 && m == 0) s.bad[rec * 4 + g] = bad;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int b = (int)(wave >> 1) + WAVES / 2 * i;
            if (NB % (WAVES / 2) != 0 && b >= NB) break;
            h2 p[4];
            if constexpr (KB == 8) {
                vx_unpack8(r.k[i][0], p[0], p[1]);
                vx_unpack8(r.k[i][1], p[2], p[3]);
            } else {
                const uint32_t w = r.k[i][0];
                p[0] = vx_unpack4(w), p[1] = vx_unpack4_high(w), p[2] = vx_unpack4(w >> 8), p[3] = vx_unpack4_high(w >> 8);
            }
            const _Float16 rk = __builtin_bit_cast(_Float16, r.kd[i]) * fk;
            const h2 rk2 = {rk, rk};
            h2 kh[4], kl[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                kh[j] = p[j] * rk2;
                kl[j] = __builtin_elementwise_fma(p[j], rk2, -kh[j]);
            }
            // dims 16 (g / 2) + 8 (g % 2) ..: step g / 2, half g % 2
            h8* kat = &s.k[((b * 2 + (g >> 1)) * 2) * 64 + (g & 1) * 32 + 16 * rec + m];
            kat[0] = h8{kh[0].x, kh[0].y, kh[1].x, kh[1].y, kh[2].x, kh[2].y, kh[3].x, kh[3].y};
            kat[64] = h8{kl[0].x, kl[0].y, kl[1].x, kl[1].y, kl[2].x, kl[2].y, kl[3].x, kl[3].y};
            const uint32_t d0 = r.d[i][0], d1 = r.d[i][1];
            const h2 r0 = __builtin_bit_cast(h2, d0) * f0, r1 = __builtin_bit_cast(h2, d1) * f1;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                h2 x0, x1;
                if constexpr (VB == 8) {
                    vx_unpack8(r.v[i][v], x0, x1);
                } else {
                    const uint32_t w = r.v[i][0];
                    x0 = v ? vx_unpack4_high(w) : vx_unpack4(w);
                    x1 = v ? vx_unpack4_high(w >> 8) : vx_unpack4(w >> 8);
                }
                const h2 a0 = x0 * r0, a1 = x1 * r1;
                const h2 b0 = __builtin_elementwise_fma(x0, r0, -a0), b1 = __builtin_elementwise_fma(x1, r1, -a1);
                // row 16 v + m of the block's 32 (dim 2 m + v), half g % 2, keys' place g / 2
                h4* at = (h4*)&s.v[((b * 2 + rec) * 2) * 64 + (g & 1) * 32 + 16 * v + m] + (g >> 1);
                at[0] = h4{a0.x, a0.y, a1.x, a1.y};
                at[2 * 64] = h4{b0.x, b0.y, b1.x, b1.y};
            }
        }
    }

    struct shared {
        tile t[2 * PERIOD];
        int at[WAVES][32];
    };

    // Row block rb of sequence s and head kvh over the keys that range(lo, hi)
    // leaves of those its rows see; whole: the rows' results, else sums to partial `part`.
    template <class Range>
    static __device__ __forceinline__ void unit(const vx_attn_args& a, shared& shm, const vx_attn_seq& q, uint32_t s, uint32_t kvh,
                                                uint32_t rb, bool whole_unit, uint32_t part, Range range) {
        tile* sh = shm.t;
        const uint32_t lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t r0 = rb * ROWS;
        const uint32_t row = r0 + wave * 32 + n;
        const vx_attn_row w = vx_attn_row_of(a, q, s, kvh, row);
        const int tail = a.tree ? max(q.len - q.n, 0) : q.len;  // keys from here on: by the tree's bits
        const int last = q.len - 1;
        __syncthreads();  // (LDS may be another unit's still)
        // what the wave's rows see, and all of them; and the workgroup's
        int lo = w.hi > w.lo ? w.lo : 0x7FFFFFFF, hi = w.hi > w.lo ? w.hi : 0;
        int lo_all = row < q.rows ? w.lo : 0, hi_all = row < q.rows ? w.hi : 0x7FFFFFFF;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            lo = min(lo, __shfl_xor(lo, o));
            hi = max(hi, __shfl_xor(hi, o));
            lo_all = max(lo_all, __shfl_xor(lo_all, o));
            hi_all = min(hi_all, __shfl_xor(hi_all, o));
        }
        const bool rows_here = r0 + wave * 32 < q.rows;  // (the first row's wave: uniform)
        if (a.tree && rows_here) {
            lo = min(lo, tail);
            hi = q.len;
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
        lo_all = __builtin_amdgcn_readfirstlane(lo_all);
        hi_all = __builtin_amdgcn_readfirstlane(hi_all);
        int wg_lo, wg_hi;
        {
            int* b = (int*)&sh[0];
            if (lane == 0) b[wave] = lo, b[WAVES + wave] = hi;
            __syncthreads();
            wg_lo = b[0], wg_hi = b[WAVES];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) wg_lo = min(wg_lo, b[i]), wg_hi = max(wg_hi, b[WAVES + i]);
            __syncthreads();
        }
        wg_lo = __builtin_amdgcn_readfirstlane(wg_lo);
        wg_hi = __builtin_amdgcn_readfirstlane(wg_hi);
        if (wg_lo >= wg_hi) wg_lo = wg_hi = 0;  // nothing seen
        int kbeg = wg_lo, kend = wg_hi;
        range(kbeg, kend);
        kbeg &= ~31;
        if (kbeg >= kend) kbeg = kend = 0;

        h8 qh[NB][2], ql[NB][2];
        float fq;
        {
            uint32_t token, head;
            vx_attn_token(a, q, kvh, min(row, q.rows - 1u), token, head);  // (a row past the end: another's, never stored)
            const float* qp = a.q + (int64_t)token * a.qs[0] + (int64_t)head * a.qs[1];
            int64_t sd = a.qs[2];
            asm volatile("" : "+s"(sd));  // (else every address of the strided case is kept over all units)
            float x[NB][2][8], top = 0.f;
            bool fine = true;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t d = 32 * b + 16 * j + 8 * h;
                    if (a.vec) {
                        const f4 u = *(const f4*)(qp + d), v = *(const f4*)(qp + d + 4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[b][j][i] = u[i], x[b][j][4 + i] = v[i];
                    } else {
                        const float* p = qp + (int64_t)d * sd;
#pragma unroll
                        for (int i = 0; i < 8; ++i, p += sd) x[b][j][i] = *p;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        top = fmaxf(top, fabsf(x[b][j][i]));
                        fine = fine && fabsf(x[b][j][i]) < __builtin_inff();
                    }
                }
            if (!fine) top = __builtin_inff();
            top = fmaxf(top, __shfl_xor(top, 32));
            int e = 0;
            if (top > 0.f && top < __builtin_inff()) e = __builtin_amdgcn_frexp_expf(top);
            const float not_finite = top < __builtin_inff() ? 0.f : __builtin_nanf("");
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        h2 u, v;  // (below 2^15)
                        vx_two_terms(__builtin_ldexpf(x[b][j][i], 15 - e) + not_finite, __builtin_ldexpf(x[b][j][i + 1], 15 - e) + not_finite, u, v);
                        qh[b][j][i] = u.x, qh[b][j][i + 1] = u.y, ql[b][j][i] = v.x, ql[b][j][i + 1] = v.y;
                    }
            fq = __builtin_ldexpf(a.cap > 0.f ? a.scale / a.cap : a.scale * VX_LOG2E, e - 15);
        }

        f16v o[NB] = {};
        float M = -__builtin_inff(), l = 0.f;
        const vx_scalar_i32 table = (vx_scalar_i32)(a.table + (uint64_t)s * a.table_stride);
        const uint8_t* base = a.c.base + (uint64_t)(kvh << (a.c.page_shift - 4)) * REC;
        const float capl = a.cap * VX_LOG2E;
        float poly[5];
#pragma unroll
        for (int i = 0; i < 5; ++i) poly[i] = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(capl * VX_TANH[i])));

#pragma unroll
        for (int i = 0; i < PERIOD; ++i)
            if (kbeg + 32 * i < kend) {
                raw r;
                load(a, table, base, kbeg + 32 * i, last, r);
                store(a, table, base, r, sh[i], kbeg + 32 * i, last);
            }
        __syncthreads();
        uint32_t buf = 0;
        float minus = -1.f;
        asm("" : "+s"(minus));
        for (int k0 = kbeg; k0 < kend; k0 += 32, ++buf) {
            const tile& t = sh[buf % (2 * PERIOD)];
            raw r;
            const int kn = k0 + 32 * PERIOD;  // the tile that this one's turn decodes
            const bool more = kn < kend;
            if (more) load(a, table, base, kn, last, r);
            if (k0 < hi && k0 + 32 > lo) {
                __builtin_amdgcn_s_setprio(1);
                // scores: lane (n, h), register i: query n, key 8 (i / 4) + 4 h + i % 4
                // Operands are read from LDS two steps before the products that take
                // them; the barriers keep the compiler from moving the reads back
                // (vector and scalar arithmetic may cross them).
                f16v x = {};
                h8 kf[3][2];
                auto kread = [&](int u) {
                    kf[u % 3][0] = t.k[2 * u * 64 + lane];
                    kf[u % 3][1] = t.k[(2 * u + 1) * 64 + lane];
                };
                kread(0);
                kread(1);
#pragma unroll
                for (int u = 0; u < 2 * NB; ++u) {
                    const int b = u / 2, j = u % 2;
                    if (u + 2 < 2 * NB) kread(u + 2);
                    __builtin_amdgcn_sched_barrier(6);
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[u % 3][0], qh[b][j], x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[u % 3][0], ql[b][j], x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[u % 3][1], qh[b][j], x, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(6);
                }
                __builtin_amdgcn_s_setprio(0);
                float e[4], apart = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f2 ke = t.e[4 * (j / 2) + 2 * (j % 2) + (int)h];
                    const float f = fq * fabsf(ke.x);
                    e[j] = ke.y;
                    apart = fminf(apart, ke.x);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[4 * j + i] *= f;
                }
                // keys far apart: own(register, factor and difference)
                const bool far = __builtin_expect(__any(apart < 0.f), 0);
                auto each_own = [&](auto own) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (t.e[2 * j + (int)h].x < 0.f) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) own(4 * j + i, t.key[8 * j + 4 * (int)h + i]);
                        }
                };
                if (__builtin_expect(far, 0)) each_own([&](int i, f2 k) { x[i] *= k.x; });
                if (a.cap > 0.f) {
                    float big = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) big = fmaxf(big, fabsf(x[i]));
                    if (__any(!(big < 0.65f))) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = capl * vx_tanh(x[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {  // vx_tanh_small times capl
                            const float z = x[i] * x[i];
                            float p = __builtin_fmaf(z, poly[4], poly[3]);
                            p = __builtin_fmaf(z, p, poly[2]);
                            p = __builtin_fmaf(z, p, poly[1]);
                            p = __builtin_fmaf(z, p, poly[0]);
                            x[i] *= __builtin_fmaf(z, p, capl);
                        }
                    }
                }
                const bool whole = k0 >= lo_all && k0 + 32 <= hi_all && k0 + 32 <= tail;
                uint32_t see = 0xFFFFFFFFu;  // bit k: key k0 + 4 h + k
                if (!whole) see = vx_attn_sees(a, q, w, kvh, row, tail, k0, shm.at[wave]) >> (4 * h);
                if (a.slopes) {
                    if (a.tree && k0 + 32 > tail) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            x[i] = __builtin_fmaf(-w.slope, fabsf((float)(w.pos - shm.at[wave][8 * (i / 4) + i % 4 + 4 * h])), x[i]);
                    } else {
                        const float d0 = (float)(w.pos - (k0 + 4 * (int)h));
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(-w.slope, fabsf(d0 - (float)(8 * (i / 4) + i % 4)), x[i]);
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t v = (uint32_t)__builtin_amdgcn_sbfe((int)see, 8 * (i / 4) + i % 4, 1);
                        x[i] = __uint_as_float((v & __float_as_uint(x[i])) | (~v & 0xFF800000u));
                    }
                }
                if (__builtin_expect(far, 0)) each_own([&](int i, f2 k) { x[i] += k.y; });
                // running maximum of score + e: four keys at a time
                float top = -__builtin_inff();
                uint32_t bad = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = 4 * (j / 2) + 2 * (j % 2) + (int)h;
                    bad |= t.bad[at];
                    top = fmaxf(top, fmaxf(fmaxf(x[4 * j], x[4 * j + 1]), fmaxf(x[4 * j + 2], x[4 * j + 3])) + e[j]);
                }
                {
                    uint32_t u = __builtin_bit_cast(uint32_t, top), v = u;
                    vx_swap32(u, v);
                    top = fmaxf(__builtin_bit_cast(float, u), __builtin_bit_cast(float, v)) - 6.f;
                }
                if (__any(top > M + 8.f)) {
                    const float Mn = top > M + 8.f ? top : M;
                    const float al = __builtin_amdgcn_exp2f(Mn == -__builtin_inff() ? 0.f : M - Mn);
                    l *= al;
#pragma unroll
                    for (int b = 0; b < NB; ++b) o[b] *= al;
                    M = Mn;
                }
                const float Mr = M == -__builtin_inff() ? 0.f : M;
                h8 ph[2], pl[2];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float c = Mr - e[j];
                    float part = 0.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[4 * j + i] = __builtin_amdgcn_exp2f(x[4 * j + i] - c);
                        part += x[4 * j + i];
                    }
                    l = __builtin_fmaf(part, __builtin_ldexpf(1.f, -(int)e[j]), l);
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        h2 u, v;
                        vx_two_terms(x[4 * j + i], x[4 * j + i + 1], minus, u, v);
                        const int k = 4 * (j % 2) + i;
                        ph[j / 2][k] = u.x, ph[j / 2][k + 1] = u.y, pl[j / 2][k] = v.x, pl[j / 2][k + 1] = v.y;
                    }
                }
                if (__builtin_expect(far, 0))  // the weights' sum takes w 2^-e of the key's own e
                    each_own([&](int i, f2 k) { l += x[i] * __builtin_ldexpf(__builtin_ldexpf(1.f, -(int)k.y) - 1.f, -(int)e[i / 4]); });
                __builtin_amdgcn_s_setprio(1);
                h8 vf[3][2];
                auto vread = [&](int u) {
                    vf[u % 3][0] = t.v[2 * u * 64 + lane];
                    vf[u % 3][1] = t.v[(2 * u + 1) * 64 + lane];
                };
                vread(0);
                vread(1);
#pragma unroll
                for (int u = 0; u < 2 * NB; ++u) {
                    const int b = u / 2, j = u % 2;
                    if (u + 2 < 2 * NB) vread(u + 2);
                    __builtin_amdgcn_sched_barrier(6);
                    o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[u % 3][0], ph[j], o[b], 0, 0, 0);
                    o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[u % 3][0], pl[j], o[b], 0, 0, 0);
                    o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[u % 3][1], ph[j], o[b], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(6);
                }
                __builtin_amdgcn_s_setprio(0);
                if (__any(bad)) {
                    // values that are not finite, taken as zeros above: NaN for the rows that see their key
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint32_t keys = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j) keys |= (t.bad[4 * (j / 2) + 2 * (j % 2) + h] >> (4 * b) & 15u) << (8 * j);
                        const int hit = (keys & see) != 0u;
                        if (hit | __shfl_xor(hit, 32)) o[b] += __builtin_nanf("");  // (a lane has half of the keys, and half of the dims)
                    }
                }
            }
            if (more) store(a, table, base, r, sh[(buf + PERIOD) % (2 * PERIOD)], kn, last);
            if (PERIOD == 1 || buf % PERIOD == PERIOD - 1) __syncthreads();
        }

        // both halves' sums; registers 8 v + 4 p + i hold dims 32 b + 16 p + 8 h + 2 i + v
        l += __shfl_xor(l, 32);
        uint32_t r = r0 + (threadIdx.x >> 6) * 32 + (threadIdx.x & 31), token, head;
        if (r >= q.rows) return;
        vx_attn_token(a, q, kvh, r, token, head);
        constexpr uint32_t D = 32 * NB;
        const uint64_t at = (uint64_t)part * ROWS + wave * 32 + n;
        if (!whole_unit && h == 0) *(f2*)(a.part_ml + at * 2) = f2{M, l};
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const f4 v = {o[b][4 * p + 2 * u], o[b][8 + 4 * p + 2 * u], o[b][4 * p + 2 * u + 1], o[b][8 + 4 * p + 2 * u + 1]};
                    const uint32_t d = 32 * b + 16 * p + 8 * h + 4 * u;
                    if (whole_unit) vx_attn_put(a, token, head, d, v, l);
                    else *(f4*)(a.part_o + at * D + d) = v;
                }
    }

    // A workgroup a unit: heads fastest (a head's row blocks on one XCD where
    // heads are a multiple of 8), late rows first (causal: they have the most keys).
    static __device__ __forceinline__ void each(const vx_attn_args& a) {
        __shared__ shared sh;
        uint32_t id = blockIdx.x;
        const uint32_t kvh = id % a.c.heads;
        id /= a.c.heads;
        const uint32_t s = id % a.seqs, place = id / a.seqs;
        const vx_attn_seq q = vx_attn_sequence(a, s);
        const uint32_t blocks = (q.rows + ROWS - 1) / ROWS;
        if (place >= blocks) return;
        unit(a, sh, q, s, kvh, blocks - 1 - place, true, 0, [](int&, int&) {});
    }

    // Fewer units than the card has places: their keys dealt out evenly.
    static __device__ __forceinline__ void even(const vx_attn_args& a) {
        __shared__ shared sh;
        vx_attn_deal<THREADS, ROWS, 64, 4>(a, [&](const vx_attn_seq& q, uint32_t s, uint32_t kvh, uint32_t rb, bool whole, uint32_t part,
                                               int from, int to, bool end) {
            unit(a, sh, q, s, kvh, rb, whole, part, [&](int& lo, int& hi) {
                lo = max(lo, from);
                if (!end) hi = min(hi, to);
            });
        });
    }
};
