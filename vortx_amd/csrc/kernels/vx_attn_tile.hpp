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
// magnitude fills f16's range, and the weights' sum takes w 2^-e.
// That is exact while no scale but 0 is 2^15 below the largest of its four keys.
// K or V of a record (16 keys) in which some may be further apart (sizes of four
// keys by more than FAR, or the blocks of a key, which its size byte says), with a
// scale that is not finite, or never written is rough: the tile has its numbers
// as they are, and the scales beside them. The scores then take K's scales on
// each block's product; weight times V's scale goes block by block, by a power of
// two that each row has there (every tile rough: 4096 causal tokens take 1.35
// times as long where K is, 1.9 V, eight trees of 61 drafts 1.4 and 2.7).
// In records that are not rough a scale of V that its size does not allow is of a
// slot that was never written, which no row sees: 0, so that a weight of 0 times
// it is 0.
// (With K always as whole numbers, exact in one term, and its scales on the
// 32-dim products, a tile had 8 matrix instructions fewer and 64 multiply-adds
// and 32 registers a wave more: 430 us where this then took 415, 4096 causal
// tokens of 32 heads of 128.)
// q is two f16 terms (22 bits, a power of two per row), and so are the weights;
// of the product's terms the one of two lows is left out (2^-22). M follows the
// maximum of score + e by steps of more than 2^5 only: most tiles leave the sums
// O^T = V^T P^T unscaled. The largest weight is 2^10 to 2^15, so two terms, which
// end at 2^-24, leave out 2^-21 of a value beside others that its e, of another
// block or a key out of sight, says to be 2^14 larger than they are. P^T is
// used in the registers S^T was left in: the order of keys within a
// contraction is free, and V is laid out to it.
// Bound: matrix and vector issue, which take turns more than they overlap (48
// 32-cycle matrix instructions and 420 vector ones a wave and tile at 128, 480
// with a cap, units' beginnings and ends among them): 4096 causal tokens of 32
// heads of 128, capped, 424 to 465 us by the card, at 436 us 315 TFLOP/s of
// attention, 945 of f16 products (matrix cores busy 43 %, vector issue 54 %).
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
        _Float16 ks[NB][32], vs[NB][32];  // scales of rough records
        f2 e[8];                // of four keys: 2^exponent of K's scales, exponent of V's
        uint32_t rough[2];      // of a record: 1, K's numbers without their scales; 4, V's
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

    static constexpr uint32_t FAR = 4;
    static_assert(FAR + VX_KV_APART <= 14, "a scale 2^15 below the largest is no normal f16 beside it");
    static __device__ __forceinline__ int power(uint32_t size) { return max((int)size - 16, -15); }  // (of no key: size 0)

    // the record of the 16 keys from key on; past the end the last one
    static __device__ __forceinline__ const uint8_t* record(const vx_attn_args& a, vx_scalar_i32 table, const uint8_t* base, int key, int last) {
        key = min(key, last);
        const uint32_t page = min((uint32_t)table[(uint32_t)key >> a.c.page_shift], a.c.pages - 1u);
        return base + page * a.c.page_bytes + (((uint32_t)key & ((1u << a.c.page_shift) - 1u)) >> 4) * REC;
    }

    static __device__ __forceinline__ void load(const vx_attn_args& a, vx_scalar_i32 table, const uint8_t* base, int k0, int last, raw& r) {
        const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), rec = wave & 1, lane = t & 63, m = lane & 15, g = lane >> 4;
        if (NB < WAVES / 2 && (int)(wave >> 1) >= NB) return;
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
    static __device__ __forceinline__ void store(raw& r, tile& s, int k0, int last) {
        typedef uint16_t us2 __attribute__((ext_vector_type(2)));
        const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), rec = wave & 1, lane = t & 63, m = lane & 15, g = lane >> 4;
        if (NB < WAVES / 2 && (int)(wave >> 1) >= NB) return;  // (no pieces: packed documents of dim 64 82 us, with the rest done for nothing 87)
        // the largest of four sizes, and whether another one is far below it. 0 is no size: K's zeros are
        // exact beside any; a key of V's zeros has weight, which the others' exponent would take bits from
        auto largest = [](uint32_t e, bool& far) {
            const us2 lo = __builtin_bit_cast(us2, e & 0x00FF00FFu), hi = __builtin_bit_cast(us2, e >> 8 & 0x00FF00FFu), one = {1, 1};
            const us2 most = __builtin_elementwise_max(lo, hi), least = __builtin_elementwise_min(lo - one, hi - one);
            const uint32_t top = max((uint32_t)most.x, (uint32_t)most.y);
            far = top > min((uint32_t)least.x, (uint32_t)least.y) + 1u + FAR;
            return top;
        };
        // sizes of keys that do not exist (a sequence's last tile): none, so that what their slots hold makes no record
        // rough (eight trees of 61 drafts behind 300 keys 40 us, else up to 50)
        if (__builtin_expect(k0 + 32 > last + 1, 0)) {
            auto first = [](int n) { return n >= 4 ? 0xFFFFFFFFu : n > 0 ? (1u << (8 * n)) - 1u : 0u; };
            const int keys = last + 1 - (k0 + 16 * (int)rec);
            r.e &= first(keys - 4 * (int)g);
            r.ke &= first(keys - 4 * (int)(m >> 2));
        }
        bool far, kfar;
        uint32_t size = largest(r.e, far), ksize = largest(r.ke, kfar);
        // (a wave has the sizes of all of its record: waves of one record agree)
        const bool kr = __any(kfar | (ksize > 31u)), vr = __any(far | (size > 31u));
        if (__builtin_expect(kr, 0)) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int b = (int)(wave >> 1) + WAVES / 2 * i;
                if (NB % (WAVES / 2) != 0 && b >= NB) break;
                if (g == 0) s.ks[b][16 * rec + m] = __builtin_bit_cast(_Float16, r.kd[i]);
                r.kd[i] = 0x3C00;  // 1
            }
            ksize = 16;  // 2^0
        }
        if (__builtin_expect(vr, 0)) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int b = (int)(wave >> 1) + WAVES / 2 * i;
                if (NB % (WAVES / 2) != 0 && b >= NB) break;
                if (m == 0) *(u2*)&s.vs[b][16 * rec + 4 * g] = u2{r.d[i][0], r.d[i][1]};
                r.d[i][0] = r.d[i][1] = 0x3C003C00u;
            }
            size = 16;
        } else {
            us2 most = {};
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int j = 0; j < 2 && (NB % (WAVES / 2) == 0 || (int)(wave >> 1) + WAVES / 2 * i < NB); ++j)
                    most = __builtin_elementwise_max(most, __builtin_bit_cast(us2, r.d[i][j] & 0x7FFF7FFFu));
            const uint32_t limit = max(size, 1u) << 10;
            if (__builtin_expect(__any(max((uint32_t)most.x, (uint32_t)most.y) >= limit), 0)) {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if ((r.d[i][j] & 0x7FFFu) >= limit) r.d[i][j] &= 0xFFFF0000u;
                        if ((r.d[i][j] >> 16 & 0x7FFFu) >= limit) r.d[i][j] &= 0x0000FFFFu;
                    }
            }
        }
        // what V's four keys and K's key are brought down by
        auto below = [](uint32_t v) { return (_Float16)__builtin_ldexpf(1.f, -power(v)); };
        const _Float16 f = below(size), fk = below(ksize);
        const h2 fv = {f, f};
        if (wave < 2 && m == 4 * g) s.e[rec * 4 + g] = f2{__builtin_ldexpf(1.f, power(ksize)), (float)power(size)};
        if (wave < 2 && lane == 0) s.rough[rec] = (kr ? 1u : 0u) | (vr ? 4u : 0u);
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
            const h2 r0 = __builtin_bit_cast(h2, d0) * fv, r1 = __builtin_bit_cast(h2, d1) * fv;
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
        const int tail = a.tree ? q.tail : q.len;  // keys from here on: by the tree's bits
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
            lo = min(lo, max(tail, 0));
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
                store(r, sh[i], kbeg + 32 * i, last);
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
                const uint32_t rough = __builtin_amdgcn_readfirstlane(t.rough[0] | t.rough[1] << 1);  // K: bits 0, 1; V: 2, 3
                if (__builtin_expect(rough & 3u, 0)) {  // once more, block by block
                    x = f16v{};
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        __builtin_amdgcn_sched_barrier(0);  // (one block's products at a time: registers)
                        f16v y = {};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const h8 kh = t.k[(b * 4 + 2 * j) * 64 + lane], kl = t.k[(b * 4 + 2 * j + 1) * 64 + lane];
                            y = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[b][j], y, 0, 0, 0);
                            y = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[b][j], y, 0, 0, 0);
                            y = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[b][j], y, 0, 0, 0);
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const h4 d = *(const h4*)&t.ks[b][8 * j + 4 * h];
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[4 * j + i] = __builtin_fmaf(y[4 * j + i], rough >> (j / 2) & 1 ? (float)d[i] : 1.f, x[4 * j + i]);
                        }
                    }
                }
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f2 ke = t.e[4 * (j / 2) + 2 * (j % 2) + (int)h];
                    const float f = fq * ke.x;
                    e[j] = ke.y;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[4 * j + i] *= f;
                }
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
                // running maximum of score + e: four keys at a time
                float top = -__builtin_inff();
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    top = fmaxf(top, fmaxf(fmaxf(x[4 * j], x[4 * j + 1]), fmaxf(x[4 * j + 2], x[4 * j + 3])) + e[j]);
                {
                    uint32_t u = __builtin_bit_cast(uint32_t, top), v = u;
                    vx_swap32(u, v);
                    top = fmaxf(__builtin_bit_cast(float, u), __builtin_bit_cast(float, v)) - 10.f;
                }
                if (__any(top > M + 5.f)) {
                    const float Mn = top > M + 5.f ? top : M;
                    const float al = __builtin_amdgcn_exp2f(Mn == -__builtin_inff() ? 0.f : M - Mn);
                    l *= al;
#pragma unroll
                    for (int b = 0; b < NB; ++b) o[b] *= al;
                    M = Mn;
                }
                const float Mr = M == -__builtin_inff() ? 0.f : M;
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
                }
                // a weight times its scale, as two f16 terms of eight keys
                auto terms = [&](int j, h8& hi, h8& lo, auto value) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        h2 u, v;
                        vx_two_terms(value(8 * j + i), value(8 * j + i + 1), minus, u, v);
                        hi[i] = u.x, hi[i + 1] = u.y, lo[i] = v.x, lo[i + 1] = v.y;
                    }
                };
                if (__builtin_expect(rough >> 2, 0)) {
                    // 0 for what the row does not see, whose scale may be anything; never 0 for what it sees, whose NaN shows
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = see >> (8 * (i / 4) + i % 4) & 1 ? fmaxf(x[i], 0x1p-126f) : 0.f;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        asm volatile("" ::: "memory");  // (one block at a time: registers)
                        __builtin_amdgcn_sched_barrier(0);
                        h4 scales[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) scales[j] = *(const h4*)&t.vs[b][8 * j + 4 * h];
                        auto value = [&](int i) {
                            const float d = (float)scales[i / 4][i % 4];
                            return x[i] == 0.f ? 0.f : x[i] * (rough >> (2 + i / 8) & 1 ? d : 1.f);
                        };
                        float most = 0.f;
#pragma unroll
                        for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(value(i)));  // (not a NaN)
                        {
                            uint32_t u = __builtin_bit_cast(uint32_t, most), v = u;
                            vx_swap32(u, v);
                            most = fmaxf(__builtin_bit_cast(float, u), __builtin_bit_cast(float, v));
                        }
                        // (sums below 2^23 2^15 keys: no overflow with 2^55)
                        const int p = most > 0x1p-40f ? __builtin_amdgcn_frexp_expf(most) : -40;
                        o[b] *= __builtin_ldexpf(1.f, 15 - p);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            asm volatile("" ::: "memory");
                            h8 ph, pl;
                            terms(j, ph, pl, [&](int i) { return __builtin_ldexpf(value(i), 15 - p); });  // (below 2^15)
                            __builtin_amdgcn_sched_barrier(0);
                            const h8 vh = t.v[(b * 4 + 2 * j) * 64 + lane];
                            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph, o[b], 0, 0, 0);
                            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl, o[b], 0, 0, 0);
                            const h8 vl = t.v[(b * 4 + 2 * j + 1) * 64 + lane];
                            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph, o[b], 0, 0, 0);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        o[b] *= __builtin_ldexpf(1.f, p - 15);
                    }
                    // the usual products below then add nothing: in two branches the sums
                    // were copied, and 60 registers spilled
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = 0.f;
                }
                h8 ph[2], pl[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) terms(j, ph[j], pl[j], [&](int i) { return x[i]; });
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
            }
            if (more) store(r, sh[(buf + PERIOD) % (2 * PERIOD)], kn, last);
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
