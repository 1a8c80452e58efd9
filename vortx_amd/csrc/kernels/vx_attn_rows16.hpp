// vx_attn_rows16.hpp — attention of up to 16 query rows (query heads of one
// key/value head, times tokens) over the quantized cache.
//
// Keys go over the rows of the 16 x 16 x 32 matrix instructions and queries
// over their columns: S^T = K q^T leaves lane (m, g) with the scores of query m
// for keys 4 g + 0..3 of 16, which is also how P^T goes into O^T = V^T P^T, so
// nothing crosses lanes but the maximum. q (f32) is two f16 terms after a
// power of two per row (22 bits); the cached whole numbers are exact in f16, a
// block's scale is applied to its 32-dim product in f32. P times a value's
// scale is two f16 terms again. The running maximum M is of score + e, e the
// exponent of the key's largest scale for V: then P times a scale fills f16's
// range whatever the magnitude of V.
// Each of four waves takes every fourth 32 keys, straight from memory to the
// registers that the matrix instructions read; their sums meet in LDS.
// Where a row sees a key whose blocks of V are more than 2^10 apart (its size byte
// says so), P times scale has a power of two for each row and block: under the
// one of its largest block a block 2^23 smaller would keep 14 bits.
// Bound: memory and vector instructions together. 32 sequences of 2400 to 8000
// keys, 32 heads over 8 of 128 in 8 bits: 80 us with the join, 4.4 TB/s of the
// cache (vector issue 43 %, matrix cores 11 %); one of 131000, 64 heads over 8,
// values in 4 bits, scores capped: 66 us, 3.3 TB/s (56 %, 12 %). Two waves a SIMD:
// a third one spills in the loop (120 us where this then took 78).
#pragma once
#include "vx_attn.hpp"

template <int NB, int KB, int VB>
struct vx_rows16 {
    using PK = vx_kv_part<NB, KB>;
    using PV = vx_kv_part<NB, VB>;
    using R = vx_kv_rec<NB, KB, VB>;
    static constexpr uint32_t REC = R::BYTES;
    static constexpr int KW = NB * KB / 4, VW = NB * VB / 4;

    struct raw_k {
        uint32_t w[2][KW];
        uint32_t s[2][NB][2];  // f16 pairs: keys 4 g, + 1; + 2, + 3
    };
    struct raw_v {
        uint32_t w[2][VW];
        uint32_t s[2][NB][2];
        uint32_t e[2];  // sizes, a byte a key
    };

    // the record of the 16 keys from key on; past the end the last one
    static __device__ __forceinline__ const uint8_t* record(const vx_attn_args& a, vx_scalar_i32 table, const uint8_t* base, int key, int last) {
        key = min(key, last);
        const uint32_t page = min((uint32_t)table[(uint32_t)key >> a.c.page_shift], a.c.pages - 1u);
        return base + page * a.c.page_bytes + (((uint32_t)key & ((1u << a.c.page_shift) - 1u)) >> 4) * REC;
    }

    static __device__ __forceinline__ void load_scales(const uint8_t* p, uint32_t g, uint32_t (&s)[NB][2]) {
        // (rows of 8 NB bytes: of three blocks every other one begins between two multiples of 16)
        typedef uint32_t row_u4 __attribute__((ext_vector_type(4), aligned(8)));
        static_assert(8 * NB % alignof(row_u4) == 0 && PK::VALS % alignof(row_u4) == 0 && PK::BYTES % alignof(row_u4) == 0 &&
                          PV::VALS % alignof(row_u4) == 0 && REC % alignof(row_u4) == 0,
                      "a row of scales is not aligned for its loads");
        p += g * (8 * NB);
#pragma unroll
        for (int b = 0; b + 1 < NB; b += 2) {
            const row_u4 v = *(const row_u4*)(p + 8 * b);
            s[b][0] = v.x, s[b][1] = v.y, s[b + 1][0] = v.z, s[b + 1][1] = v.w;
        }
        if constexpr (NB % 2 != 0) {
            const u2 v = *(const u2*)(p + 8 * (NB - 1));
            s[NB - 1][0] = v.x, s[NB - 1][1] = v.y;
        }
    }

    static __device__ __forceinline__ void load(const uint8_t* const (&at)[2], uint32_t lane, uint32_t g, raw_k& k) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            vx_kv_load<NB, KB>(at[t], lane, k.w[t]);
            load_scales(at[t] + PK::VALS, g, k.s[t]);
        }
    }
    static __device__ __forceinline__ void load(const uint8_t* const (&at)[2], uint32_t lane, uint32_t g, raw_v& v) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            vx_kv_load<NB, VB>(at[t] + PK::BYTES, lane, v.w[t]);
            load_scales(at[t] + PK::BYTES + PV::VALS, g, v.s[t]);
            v.e[t] = ((const uint32_t*)(at[t] + R::V_SIZES))[g];
        }
    }

    struct shared {
        float o[4][16][NB * 32 + 4];
        float ml[4][16][2];
        int at[4][32];
    };

    // Rows r0.. of sequence s and key/value head kvh over the keys that
    // range(lo, hi) gives for those that its rows see; the four waves' sums go to sh.
    template <class Range>
    static __device__ __forceinline__ bool unit(const vx_attn_args& a, shared& sh, const vx_attn_seq& q, uint32_t s, uint32_t kvh,
                                                uint32_t r0, Range range) {
        const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t row = r0 + m;
        const vx_attn_row w = vx_attn_row_of(a, q, s, kvh, row);
        const int tail = a.tree ? q.tail : q.len;  // keys from here on: by the tree's bits
        int lo = w.hi > w.lo ? w.lo : 0x7FFFFFFF, hi = w.hi > w.lo ? w.hi : 0;
        int lo_all = row < q.rows ? w.lo : 0, hi_all = row < q.rows ? w.hi : 0x7FFFFFFF;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            lo = min(lo, __shfl_xor(lo, o));
            hi = max(hi, __shfl_xor(hi, o));
            lo_all = max(lo_all, __shfl_xor(lo_all, o));
            hi_all = min(hi_all, __shfl_xor(hi_all, o));
        }
        if (a.tree) {
            lo = min(lo, max(tail, 0));
            hi = q.len;
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
        lo_all = __builtin_amdgcn_readfirstlane(lo_all);
        hi_all = __builtin_amdgcn_readfirstlane(hi_all);
        if (lo >= hi) lo = hi = 0;  // (lo of rows that see nothing is the largest int: 32 more would be negative)
        int kbeg = lo, kend = hi;
        range(kbeg, kend);
        if (kbeg >= kend) kbeg = kend = 0;

        // q: 8 dims of each block, two f16 terms
        h8 qh[NB], ql[NB];
        float fq;
        {
            float x[NB][8];
            uint32_t token, head;
            vx_attn_token(a, q, kvh, min(row, q.rows - 1u), token, head);  // (a row past the end: another's, never stored)
            const float* qp = a.q + (int64_t)token * a.qs[0] + (int64_t)head * a.qs[1];
            int64_t sd = a.qs[2];
            asm volatile("" : "+s"(sd));  // (else every address of the strided case is kept over all units)
            float top = 0.f;
            bool fine = true;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint32_t d = 32 * b + 8 * g;
                if (a.vec) {
                    const f4 u = *(const f4*)(qp + d), v = *(const f4*)(qp + d + 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[b][i] = u[i], x[b][4 + i] = v[i];
                } else {
                    const float* p = qp + (int64_t)d * sd;
#pragma unroll
                    for (int i = 0; i < 8; ++i, p += sd) x[b][i] = *p;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    top = fmaxf(top, fabsf(x[b][i]));
                    fine = fine && fabsf(x[b][i]) < __builtin_inff();
                }
            }
            top = vx_max_rows4(fine ? top : __builtin_inff());
            int e = 0;
            if (top > 0.f && top < __builtin_inff()) e = __builtin_amdgcn_frexp_expf(top);
            const float bad = top < __builtin_inff() ? 0.f : __builtin_nanf("");  // a row that is not finite: NaN
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    h2 hi, lo;  // (below 2^15)
                    vx_two_terms(__builtin_ldexpf(x[b][i], 15 - e) + bad, __builtin_ldexpf(x[b][i + 1], 15 - e) + bad, hi, lo);
                    qh[b][i] = hi.x, qh[b][i + 1] = hi.y, ql[b][i] = lo.x, ql[b][i + 1] = lo.y;
                }
            // score = product * fq in units of log2 (capped: as the argument of tanh)
            fq = __builtin_ldexpf(a.cap > 0.f ? a.scale / a.cap : a.scale * VX_LOG2E, e - 15);
        }

        f4 o[NB][2] = {};
        float M = -__builtin_inff(), l = 0.f;
        const vx_scalar_i32 table = (vx_scalar_i32)(a.table + (uint64_t)s * a.table_stride);
        const uint8_t* base = a.c.base + (uint64_t)(kvh << (a.c.page_shift - 4)) * REC;
        const int last = q.len - 1;
        const float capl = a.cap * VX_LOG2E;

        // K of the next keys is requested when these keys' registers are free,
        // V while the scores are computed
        raw_k rk;
        raw_v rv;
        const uint8_t *at[2], *next[2];
        const int kfirst = kbeg + 32 * (int)wave;
        if (kfirst < kend) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                at[t] = record(a, table, base, kfirst + 16 * t, last);
                next[t] = record(a, table, base, kfirst + 128 + 16 * t, last);
            }
            load(at, lane, g, rk);
        }
        float zero = -0.f;
        asm("" : "+s"(zero));
        for (int k0 = kfirst; k0 < kend; k0 += 128) {
            load(at, lane, g, rv);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                at[t] = next[t];
                next[t] = record(a, table, base, k0 + 256 + 16 * t, last);
            }
            float x[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f4 sum = {};
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const h8 kf = vx_kv_kfrag<NB, KB>(rk.w[t], b);
                    f4 acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[b], f4{}, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[b], acc, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const h2 d = __builtin_bit_cast(h2, rk.s[t][b][i >> 1]);
                        sum[i] = __builtin_fmaf(acc[i], (float)(i & 1 ? d.y : d.x), sum[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) x[t][i] = sum[i] * fq;
            }
            load(at, lane, g, rk);
            if (a.cap > 0.f) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][i] = capl * vx_tanh(x[t][i]);
            }
            const bool whole = k0 >= lo_all && k0 + 32 <= hi_all && k0 + 32 <= tail;
            if (whole) {
                if (a.slopes) {
                    const float d0 = (float)(w.pos - (k0 + 4 * (int)g));
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[t][i] = __builtin_fmaf(-w.slope, fabsf(d0 - (float)(16 * t + i)), x[t][i]);
                }
            } else {
                const uint32_t see = vx_attn_sees(a, q, w, kvh, row, tail, k0, sh.at[wave]) >> (4 * g);
                const bool drafts = a.tree && k0 + 32 > tail;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (a.slopes) {
                            const int key = 16 * t + 4 * (int)g + i;
                            x[t][i] = __builtin_fmaf(-w.slope, fabsf((float)(w.pos - (drafts ? sh.at[wave][key] : k0 + key))), x[t][i]);
                        }
                        const uint32_t v = 0u - (see >> (16 * t + i) & 1u);
                        x[t][i] = v ? x[t][i] : -__builtin_inff();
                        // a lane's scales are of its own row: what the row does not see, which
                        // may be anything, counts nowhere
#pragma unroll
                        for (int b = 0; b < NB; ++b) rv.s[t][b][i >> 1] &= v | (i & 1 ? 0x0000FFFFu : 0xFFFF0000u);
                        rv.e[t] &= v | ~(0xFFu << (8 * i));
                    }
            }
            // running maximum of score + exponent of V's scales
            float top = -__builtin_inff();
            // keys that a row sees whose blocks are far apart or not finite
            const bool rough = __any((rv.e[0] | rv.e[1]) & 0x80808080u);
            {
                if (__builtin_expect(rough, 0)) {  // the largest of the finite scales
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t e = 0;
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                const uint32_t d = vx_kv_size(rv.s[t][b][i >> 1] >> (16 * (i & 1)));
                                e = max(e, d == 255u ? 0u : d);
                            }
                            top = fmaxf(top, x[t][i] + (float)e);
                        }
                } else {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = fmaxf(top, x[t][i] + (float)(rv.e[t] >> (8 * i) & 255u));
                }
                top = vx_max_rows4(top - 29.f);  // P times scale below 2^14
            }
            const float Mn = fmaxf(M, top), Mr = Mn == -__builtin_inff() ? 0.f : Mn;
            if (__any(Mn != M)) {
                const float al = __builtin_amdgcn_exp2f(M - Mr);
                l *= al;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int v = 0; v < 2; ++v) o[b][v] *= al;
                M = Mn;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[t][i] = __builtin_amdgcn_exp2f(x[t][i] - Mr);
                    l += x[t][i];
                }
            auto vfrag = [&](int b, int v) {
                h2 v0, v1, v2, v3;
                vx_kv_vfrag<NB, VB>(rv.w[0], b, v, v0, v1);
                vx_kv_vfrag<NB, VB>(rv.w[1], b, v, v2, v3);
                return h8{v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
            };
            if (__builtin_expect(rough, 0)) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    __builtin_amdgcn_sched_barrier(0);  // (one block at a time: registers)
                    float most = 0.f;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const h2 d = __builtin_bit_cast(h2, rv.s[t][b][i >> 1]);
                            most = fmaxf(most, fabsf(x[t][i] * (float)(i & 1 ? d.y : d.x)));  // (not a NaN)
                        }
                    most = vx_max_rows4(most);
                    const int e = most > 0x1p-100f ? __builtin_amdgcn_frexp_expf(most) : -100;
                    h8 ph, pl;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            const h2 d = __builtin_bit_cast(h2, rv.s[t][b][i >> 1]);
                            h2 hi, lo;  // (below 2^15)
                            vx_two_terms(__builtin_ldexpf(x[t][i] * (float)d.x, 15 - e), __builtin_ldexpf(x[t][i + 1] * (float)d.y, 15 - e), hi, lo);
                            const int n = 4 * t + i;
                            ph[n] = hi.x, ph[n + 1] = hi.y, pl[n] = lo.x, pl[n + 1] = lo.y;
                        }
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const h8 vf = vfrag(b, v);
                        f4 acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, f4{}, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, acc, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[b][v][i] += __builtin_ldexpf(acc[i], e - 15);
                    }
                }
                continue;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                h8 ph, pl;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        h2 hi, lo;
                        vx_two_terms(x[t][i], x[t][i + 1], __builtin_bit_cast(h2, rv.s[t][b][i >> 1]), zero, hi, lo);
                        const int n = 4 * t + i;
                        ph[n] = hi.x, ph[n + 1] = hi.y, pl[n] = lo.x, pl[n + 1] = lo.y;
                    }
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const h8 vf = vfrag(b, v);
                    o[b][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, o[b][v], 0, 0, 0);
                    o[b][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, o[b][v], 0, 0, 0);
                }
            }
        }

        // lane (m, g) holds dims 32 b + 2 (4 g + i) + v of query m
        l = vx_sum_rows4(l);
        if (g == 0) {
            sh.ml[wave][m][0] = M;
            sh.ml[wave][m][1] = l;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) *(f2*)&sh.o[wave][m][32 * b + 8 * g + 2 * i] = f2{o[b][0][i], o[b][1][i]};
        __syncthreads();
        return kbeg < kend;
    }

    // The four waves' sums of a row, 4 dims.
    static __device__ __forceinline__ f4 total(const shared& sh, uint32_t row, uint32_t d, float& M, float& l) {
        M = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 4; ++i) M = fmaxf(M, sh.ml[i][row][0]);
        const float Mr = M == -__builtin_inff() ? 0.f : M;
        f4 t = {};
        l = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float c = __builtin_amdgcn_exp2f(sh.ml[i][row][0] - Mr);
            t += c * *(const f4*)&sh.o[i][row][d];
            l = __builtin_fmaf(c, sh.ml[i][row][1], l);
        }
        return t;
    }

    // Single tokens, small trees: the keys of the batch dealt out evenly. Against
    // equal splits of every sequence: 32 sequences of 2400 to 8000 keys 91 us, then 78 like this.
    static __device__ __forceinline__ void even(const vx_attn_args& a) {
        __shared__ shared sh;
        constexpr uint32_t D = 32 * NB;
        vx_attn_deal<256, 16, 128, 1>(a, [&](const vx_attn_seq& q, uint32_t s, uint32_t kvh, uint32_t rb, bool whole, uint32_t part, int from,
                                          int to, bool end) {
            const uint32_t r0 = rb * 16, rows = min(q.rows - r0, 16u);
            unit(a, sh, q, s, kvh, r0, [&](int& lo, int& hi) {
                lo = max(lo & ~31, from);
                if (!end) hi = min(hi, to);
            });
            for (uint32_t at = threadIdx.x; at < rows * (D / 4); at += 256) {
                const uint32_t r = at / (D / 4), d = 4 * (at % (D / 4));
                float M, l;
                const f4 v = total(sh, r, d, M, l);
                if (whole) {
                    uint32_t token, head;
                    vx_attn_token(a, q, kvh, r0 + r, token, head);
                    vx_attn_put(a, token, head, d, v, l);
                } else {
                    const uint64_t row = (uint64_t)part * 16 + r;
                    *(f4*)(a.part_o + row * D + d) = v;
                    if (d == 0) *(f2*)(a.part_ml + row * 2) = f2{M, l};
                }
            }
            __syncthreads();  // sh is the next unit's
        });
    }
};

// Joins the partial sums of a query row (vx_attn_deal): 16 to 64 lanes take its
// dims, four at a time, and the partials go over the groups of lanes, of a wave
// where a row has up to 8 of them (four rows a workgroup) and of the workgroup
// above (one row). One group a row took 90 us for 64 rows of 128 partials, this 11.
__device__ __forceinline__ void vx_attn_join_rows(const vx_attn_args& a) {
    __shared__ f4 sh_t[256];
    __shared__ f2 sh_ml[64];
    const uint32_t D = a.c.dim, lanes = D <= 64 ? 16 : D <= 128 ? 32 : 64;  // of a group
    const uint32_t span = a.parts > 8 ? 256 : 64;                          // threads of a row
    const uint32_t in = threadIdx.x % span, group = in / lanes, groups = span / lanes, d = 4 * (in % lanes);
    uint32_t id = blockIdx.x * (256 / span) + threadIdx.x / span;
    const uint32_t kvh = id % a.c.heads;
    id /= a.c.heads;
    const uint32_t s = id % a.seqs, r = id / a.seqs;
    const vx_attn_seq q = vx_attn_sequence(a, s);
    const uint32_t j = r / a.group, head = kvh * a.group + (r - j * a.group), rb = r / a.part_rows;
    bool valid = r < q.rows && d < D;
    u2 info = {0, 1};
    if (valid) info = *(const u2*)(a.info + 2 * (((uint64_t)s * a.row_blocks + rb) * a.c.heads + kvh));
    const uint32_t parts = info.y;
    valid = valid && parts > 1;  // (else the result is there)
    // partials 2 w or 2 w + 1, then 2 (w + 1), 2 (w + 2) ..
    auto row_of = [&](uint32_t i) { return (uint64_t)(i ? (info.x >> 1) * 2 + 2 * i : info.x) * a.part_rows + (r - rb * a.part_rows); };
    float M = -__builtin_inff(), l = 0.f;
    f4 t = {};
    if (valid) {
#pragma unroll 4
        for (uint32_t i = group; i < parts; i += groups) {
            const uint64_t row = row_of(i);
            const f2 ml = *(const f2*)(a.part_ml + row * 2);
            const f4 o = *(const f4*)(a.part_o + row * D + d);
            if (ml.y == 0.f) continue;  // nothing seen there (not so for a NaN)
            const float Mn = fmaxf(M, ml.x), c = __builtin_amdgcn_exp2f(M - Mn), k = __builtin_amdgcn_exp2f(ml.x - Mn);
            // (M is -inf before the first; a NaN in y may have -inf beside it, and stays)
            l = __builtin_fmaf(k, ml.y, c * l);
            t = c * t + k * o;
            M = Mn;
        }
    }
    sh_t[threadIdx.x] = t;
    if (in % lanes == 0) sh_ml[threadIdx.x / 16] = f2{M, l};
    __syncthreads();
    if (!valid || group) return;
    const uint32_t first = threadIdx.x;  // this row's first group is this thread's
    float Mt = M;
    for (uint32_t i = 1; i < groups; ++i) Mt = fmaxf(Mt, sh_ml[(first - in % lanes + i * lanes) / 16].x);
    const float Mr = Mt == -__builtin_inff() ? 0.f : Mt;
    const float c0 = __builtin_amdgcn_exp2f(M - Mr);
    t *= c0;
    l *= c0;
    for (uint32_t i = 1; i < groups; ++i) {
        const f2 ml = sh_ml[(first - in % lanes + i * lanes) / 16];
        const float c = __builtin_amdgcn_exp2f(ml.x - Mr);
        t += c * sh_t[first + i * lanes];
        l = __builtin_fmaf(c, ml.y, l);
    }
    vx_attn_put(a, (uint32_t)q.start + j, head, d, t, l);
}
