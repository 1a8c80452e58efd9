// vx_attn_tile.hpp — attention of many query rows over the quantized cache.
//
// A workgroup takes 128 or 256 query rows of a sequence and key/value head, 32
// to a wave, and goes over their keys 32 at a time. The waves decode a tile of
// keys once into LDS, as operands of the 32 x 32 x 16 matrix instructions, while
// the tile before is computed from the other buffer:
//   K   the whole numbers, exact in f16; a block's scale is applied to its
//       32-dim product in f32 (S^T = K q^T: rows are keys, columns queries);
//   V   scale x number, 19 bits, as two f16 terms whose sum is exact: hi rounds
//       the product, lo = fma(number, scale, -hi). The scales of each four keys
//       are first brought to [1, 2) by a power of two 2^-e, and 2^e goes to the
//       weights: w = exp2(score + e - M), so V of any magnitude fills f16's
//       range, and the weights' sum takes w 2^-e.
// q is two f16 terms (22 bits, a power of two per row), and so are the weights;
// of the product's terms the one of two lows is left out (2^-22). M follows the
// maximum of score + e by steps of more than 2^8 only: the weights have f16's
// range for that, and most tiles leave the sums O^T = V^T P^T unscaled. P^T is
// used in the registers S^T was left in: the order of keys within a
// contraction is free, and V is laid out to it.
// Bound: about as many matrix as vector cycles a tile (28 32-cycle
// instructions a wave at 64, 40 at 128, beside the softmax).
#pragma once
#include "vx_attn.hpp"

typedef float f16v __attribute__((ext_vector_type(16)));

template <int NB, int KB, int VB, int WAVES>
struct vx_tile {
    using PK = vx_kv_part<NB, KB>;
    using PV = vx_kv_part<NB, VB>;
    static constexpr uint32_t REC = PK::BYTES + PV::BYTES;
    static constexpr uint32_t THREADS = 64 * WAVES, ROWS = 32 * WAVES;
    static constexpr int ITEMS = (128 * NB + THREADS - 1) / THREADS;  // a thread's pieces of a tile: one lane's bytes of a block

    struct tile {
        h8 k[NB * 4 * 32];      // [block][8-dim group][key]
        h8 v[NB * 2 * 2 * 64];  // [block][16 keys][hi, lo][half, dim]
        uint32_t ks[NB][16];    // K scales, f16 pairs of keys
        float e[8];             // exponents of four keys' V scales
        uint32_t bad[8];        // their V scales that are not finite, bit 4 block + key
    };

    struct raw {  // a thread's pieces as loaded
        uint32_t k[ITEMS][KB / 4], v[ITEMS][VB / 4], d[ITEMS][2];
        uint32_t vs[NB][2];  // V scales of its four keys
        uint32_t ks[2];
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

    // records of the 32 keys from k0 on; past the end the last one
    static __device__ __forceinline__ void load(const vx_attn_args& a, vx_scalar_i32 table, const uint8_t* base, int k0, int last, raw& r) {
        const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), rec = wave & 1, lane = t & 63, g = lane >> 4;
        const int key = min(k0 + 16 * (int)rec, last);
        const uint32_t page = min((uint32_t)table[(uint32_t)key >> a.c.page_shift], a.c.pages - 1u);
        const uint8_t* p = base + page * a.c.page_bytes + (((uint32_t)key & ((1u << a.c.page_shift) - 1u)) >> 4) * REC;
        const uint8_t* sc = p + PK::BYTES + PV::VALS + g * (8 * NB);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int b = (int)(wave >> 1) + WAVES / 2 * i;
            if (NB % (WAVES / 2) == 0 || b < NB) {
                load_block<KB>(p, b, lane, r.k[i]);
                load_block<VB>(p + PK::BYTES, b, lane, r.v[i]);
                const u2 d = *(const u2*)(sc + 8 * b);
                r.d[i][0] = d.x, r.d[i][1] = d.y;
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const u2 v = *(const u2*)(sc + 8 * b);
            r.vs[b][0] = v.x, r.vs[b][1] = v.y;
        }
        // K's scales: lanes 0.. of waves 0 and 1, four keys of a block each
        if (wave < 2 && lane < 4 * NB) {
            const u2 v = *(const u2*)(p + PK::VALS + lane * 8);
            r.ks[0] = v.x, r.ks[1] = v.y;
        }
    }

    // decodes a thread's pieces into the tile of the keys from k0 on
    static __device__ __forceinline__ void store(raw& r, tile& s, int k0, int last) {
        typedef uint16_t us2 __attribute__((ext_vector_type(2)));
        const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), rec = wave & 1, lane = t & 63, m = lane & 15, g = lane >> 4;
        uint32_t bad = 0;
        auto largest = [&] {
            us2 big = {0, 0};
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t d = VB == 4 ? r.vs[b][i] & 0x7FFF7FFFu : r.vs[b][i];  // (8 bits: never negative)
                    big = __builtin_elementwise_max(big, __builtin_bit_cast(us2, d));
                }
            return (uint32_t)max(big.x, big.y);
        };
        uint32_t big = largest();
        if (k0 + 32 > last + 1 || __any(big >= 0x7C00u)) {
            // scales of keys that do not exist, which may be anything: 0; those that are not finite: 0, and noted
            const int valid = last + 1 - (k0 + 16 * (int)rec + 4 * (int)g);
            auto fix = [&](uint32_t d, int i) {
                if (valid <= 2 * i || (d & 0x7FFFu) >= 0x7C00u) d &= 0xFFFF0000u;
                if (valid <= 2 * i + 1 || (d >> 16 & 0x7FFFu) >= 0x7C00u) d &= 0x0000FFFFu;
                return d;
            };
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t d = r.vs[b][i];
                    if (valid > 2 * i && (d & 0x7FFFu) >= 0x7C00u) bad |= 1u << (4 * b + 2 * i);
                    if (valid > 2 * i + 1 && (d >> 16 & 0x7FFFu) >= 0x7C00u) bad |= 2u << (4 * b + 2 * i);
                    r.vs[b][i] = fix(d, i);
                }
#pragma unroll
            for (int n = 0; n < ITEMS; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) r.d[n][i] = fix(r.d[n][i], i);
            big = largest();
        }
        const int e = (int)(big >> 10) - 15;
        if (wave < 2 && m == 0) {
            s.e[rec * 4 + g] = (float)e;
            s.bad[rec * 4 + g] = bad;
        }
        const _Float16 f = (_Float16)__builtin_ldexpf(1.f, -e);
        const h2 f2h = {f, f};
        if (wave < 2 && lane < 4 * NB) {  // [g][block] -> [block][pair of keys]
            const uint32_t kg = lane / NB, b = lane % NB;
            *(u2*)&s.ks[b][8 * rec + 2 * kg] = u2{r.ks[0], r.ks[1]};
        }
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
            s.k[(b * 4 + g) * 32 + 16 * rec + m] = h8{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
            const uint32_t d0 = r.d[i][0], d1 = r.d[i][1];
            const h2 r0 = __builtin_bit_cast(h2, d0) * f2h, r1 = __builtin_bit_cast(h2, d1) * f2h;
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

    static __device__ __forceinline__ void run(const vx_attn_args& a) {
        __shared__ tile sh[2];
        __shared__ int sh_at[WAVES][32];
        const uint32_t lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        // workgroup -> (row block, split, sequence, head): heads fastest (a head's
        // row blocks on one XCD where heads are a multiple of 8), late rows first
        // (causal: they have the most keys)
        uint32_t id = blockIdx.x;
        const uint32_t kvh = id % a.c.heads;
        id /= a.c.heads;
        const uint32_t s = id % a.seqs;
        id /= a.seqs;
        const uint32_t split = id % a.splits;
        const vx_attn_seq q = vx_attn_sequence(a, s);
        const uint32_t blocks = (q.rows + ROWS - 1) / ROWS, place = id / a.splits;
        if (place >= blocks) return;
        const uint32_t r0 = (blocks - 1 - place) * ROWS, row = r0 + wave * 32 + n;
        const vx_attn_row w = vx_attn_row_of(a, q, s, kvh, row);
        const int tail = a.tree ? max(q.len - q.n, 0) : q.len;  // keys from here on: by the tree's bits
        const int last = q.len - 1;
        // what the wave's rows see, and all of them; and the workgroup's
        int lo = w.valid && w.hi > w.lo ? w.lo : 0x7FFFFFFF, hi = w.valid && w.hi > w.lo ? w.hi : 0;
        int lo_all = w.valid ? w.lo : 0, hi_all = w.valid ? w.hi : 0x7FFFFFFF;
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
        hi = min(__builtin_amdgcn_readfirstlane(hi), last + 1);
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
        // this split's keys; the last one takes what is left
        const int64_t c0 = (int64_t)(wg_lo & ~31) + (int64_t)split * a.chunk;
        const int kbeg = (int)min(c0, (int64_t)wg_hi);
        const int kend = split + 1 == a.splits ? wg_hi : (int)min((int64_t)wg_hi, c0 + a.chunk);

        h8 qh[NB][2], ql[NB][2];
        float fq;
        {
            const float* qp = a.q + (int64_t)w.token * a.qs[0] + (int64_t)w.head * a.qs[1];
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
                        const float* p = qp + (int64_t)d * a.qs[2];
#pragma unroll
                        for (int i = 0; i < 8; ++i, p += a.qs[2]) x[b][j][i] = *p;
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
        for (int i = 0; i < 5; ++i) poly[i] = capl * VX_TANH[i];

        if (kbeg < kend) {
            raw r;
            load(a, table, base, kbeg, last, r);
            store(r, sh[0], kbeg, last);
        }
        __syncthreads();
        uint32_t buf = 0;
        float minus = -1.f;
        asm("" : "+s"(minus));
        for (int k0 = kbeg; k0 < kend; k0 += 32, buf ^= 1) {
            const tile& t = sh[buf];
            raw r;
            const bool more = k0 + 32 < kend;
            if (more) load(a, table, base, k0 + 32, last, r);
            if (k0 < hi && k0 + 32 > lo) {
                // scores: lane (n, h), register i: query n, key 8 (i / 4) + 4 h + i % 4
                f16v x = {};
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    f16v acc = {};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const h8 kf = t.k[(b * 4 + 2 * j + h) * 32 + n];
                        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[b][j], acc, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[b][j], acc, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const u2 sc = *(const u2*)&t.ks[b][i + 2 * h];
                        const uint32_t s0 = sc.x, s1 = sc.y;
                        const h2 d0 = __builtin_bit_cast(h2, s0), d1 = __builtin_bit_cast(h2, s1);
                        x[i] = __builtin_fmaf(acc[i], (float)d0.x, x[i]);
                        x[i + 1] = __builtin_fmaf(acc[i + 1], (float)d0.y, x[i + 1]);
                        x[i + 2] = __builtin_fmaf(acc[i + 2], (float)d1.x, x[i + 2]);
                        x[i + 3] = __builtin_fmaf(acc[i + 3], (float)d1.y, x[i + 3]);
                    }
                }
                x *= fq;
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
                if (whole) {
                    if (a.slopes) {
                        const float d0 = (float)(w.pos - (k0 + 4 * (int)h));
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(-w.slope, fabsf(d0 - (float)(8 * (i / 4) + i % 4)), x[i]);
                    }
                } else {
                    see = vx_attn_sees(a, q, w, tail, k0, sh_at[wave]) >> (4 * h);
                    const bool drafts = a.tree && k0 + 32 > tail;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = 8 * (i / 4) + i % 4;
                        if (a.slopes)
                            x[i] = __builtin_fmaf(-w.slope, fabsf((float)(w.pos - (drafts ? sh_at[wave][key + 4 * h] : k0 + key + 4 * (int)h))), x[i]);
                        x[i] = see >> key & 1u ? x[i] : -__builtin_inff();
                    }
                }
                // running maximum of score + e: four keys at a time
                float e[4], top = -__builtin_inff();
                uint32_t bad = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = 4 * (j / 2) + 2 * (j % 2) + (int)h;
                    e[j] = t.e[at];
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
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const h8 vh = t.v[((b * 2 + j) * 2) * 64 + lane], vl = t.v[((b * 2 + j) * 2 + 1) * 64 + lane];
                        o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph[j], o[b], 0, 0, 0);
                        o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl[j], o[b], 0, 0, 0);
                        o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[j], o[b], 0, 0, 0);
                    }
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
            if (more) store(r, sh[buf ^ 1], k0 + 32, last);
            __syncthreads();
        }

        // both halves' sums; registers 8 v + 4 p + i hold dims 32 b + 16 p + 8 h + 2 i + v
        l += __shfl_xor(l, 32);
        if (!w.valid) return;
        const uint64_t heads = a.c.heads * a.group;
        constexpr uint32_t D = 32 * NB;
        const uint64_t part = ((uint64_t)split * a.tokens + w.token) * heads + w.head;
        if (a.splits > 1 && h == 0) *(f2*)(a.part_ml + part * 2) = f2{M, l};
        if (a.splits > 1 && kbeg >= kend) return;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const f4 v = {o[b][4 * p + 2 * u], o[b][8 + 4 * p + 2 * u], o[b][4 * p + 2 * u + 1], o[b][8 + 4 * p + 2 * u + 1]};
                    const uint32_t d = 32 * b + 16 * p + 8 * h + 4 * u;
                    if (a.splits > 1) *(f4*)(a.part_o + part * D + d) = v;
                    else vx_attn_put(a, (uint32_t)w.token, (uint32_t)w.head, d, v, l);
                }
    }
};
