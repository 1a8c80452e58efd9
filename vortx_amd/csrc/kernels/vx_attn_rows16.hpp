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
// exponent of the largest scale that a lane's keys have for V: then P times
// a scale fills f16's range whatever the magnitude of V.
// Each of four waves takes every fourth 32 keys; their sums meet in LDS.
#pragma once
#include "vx_attn.hpp"

template <int NB, int KB, int VB>
struct vx_rows16 {
    using PK = vx_kv_part<NB, KB>;
    using PV = vx_kv_part<NB, VB>;
    static constexpr uint32_t REC = PK::BYTES + PV::BYTES;
    static constexpr int KW = NB * KB / 4, VW = NB * VB / 4;

    struct raw_k {
        uint32_t w[2][KW];
        h4 s[2][NB];
    };
    struct raw_v {
        uint32_t w[2][VW];
        h4 s[2][NB];
    };

    // the record of the 16 keys from key on; past the end the last one
    static __device__ __forceinline__ const uint8_t* record(const vx_attn_args& a, const int32_t* table, const uint8_t* base, int key, int last) {
        key = min(key, last);
        const uint32_t page = min((uint32_t)table[(uint32_t)key >> a.c.page_shift], a.c.pages - 1u);
        return base + page * a.c.page_bytes + (((uint32_t)key & ((1u << a.c.page_shift) - 1u)) >> 4) * REC;
    }

    static __device__ __forceinline__ void load_scales(const uint8_t* p, uint32_t g, h4 (&s)[NB]) {
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = ((const h4*)p)[g * NB + b];
    }

    static __device__ __forceinline__ void load(const uint8_t* const (&at)[2], uint32_t lane, uint32_t g, raw_k& k, raw_v& v) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            vx_kv_load<NB, KB>(at[t], lane, k.w[t]);
            load_scales(at[t] + PK::VALS, g, k.s[t]);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            vx_kv_load<NB, VB>(at[t] + PK::BYTES, lane, v.w[t]);
            load_scales(at[t] + PK::BYTES + PV::VALS, g, v.s[t]);
        }
    }

    static __device__ void run(const vx_attn_args& a) {
        __shared__ float sh_o[4][16][NB * 32 + 4];
        __shared__ float sh_ml[4][16][2];
        const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        // workgroup -> (row block, split, sequence, key/value head), heads fastest
        uint32_t id = blockIdx.x;
        const uint32_t kvh = id % a.c.heads;
        id /= a.c.heads;
        const uint32_t s = id % a.seqs;
        id /= a.seqs;
        const uint32_t split = id % a.splits, rb = id / a.splits;
        const vx_attn_seq q = vx_attn_sequence(a, s);
        const uint32_t rows = q.rows, r0 = rb * 16;
        if (r0 >= rows) return;
        const vx_attn_row w = vx_attn_row_of(a, q, s, kvh, r0 + m);
        const int tail = a.tree ? max(q.len - q.n, 0) : q.len;  // keys from here on: by the tree's bits
        int lo = w.valid && w.hi > w.lo ? w.lo : 0x7FFFFFFF, hi = w.valid && w.hi > w.lo ? w.hi : 0;
        int lo_all = w.valid ? w.lo : 0, hi_all = w.valid ? w.hi : 0x7FFFFFFF;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            lo = min(lo, __shfl_xor(lo, o));
            hi = max(hi, __shfl_xor(hi, o));
            lo_all = max(lo_all, __shfl_xor(lo_all, o));
            hi_all = min(hi_all, __shfl_xor(hi_all, o));
        }
        if (a.tree) {
            lo = min(lo, tail);
            hi = q.len;
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = min(__builtin_amdgcn_readfirstlane(hi), min(q.len, (int)(a.table_cols << a.c.page_shift)));
        lo_all = __builtin_amdgcn_readfirstlane(lo_all);
        hi_all = __builtin_amdgcn_readfirstlane(hi_all);
        // this split's keys; the last one takes what is left
        const int64_t c0 = (int64_t)(lo & ~31) + (int64_t)split * a.chunk;
        const int kbeg = (int)min(c0, (int64_t)hi);
        const int kend = split + 1 == a.splits ? hi : (int)min((int64_t)hi, c0 + a.chunk);

        // q: 8 dims of each block, two f16 terms
        h8 qh[NB], ql[NB];
        float fq;
        {
            float x[NB][8];
            const float* qp = a.q + (int64_t)w.token * a.qs[0] + (int64_t)w.head * a.qs[1];
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
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[b][i] = qp[(int64_t)(d + i) * a.qs[2]];
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
                    vx_two_terms(__builtin_ldexpf(x[b][i], 15 - e) + bad, 1.f, __builtin_ldexpf(x[b][i + 1], 15 - e) + bad, 1.f, hi, lo);
                    qh[b][i] = hi.x, qh[b][i + 1] = hi.y, ql[b][i] = lo.x, ql[b][i + 1] = lo.y;
                }
            // score = product * fq in units of log2 (capped: as the argument of tanh)
            fq = __builtin_ldexpf(a.cap > 0.f ? a.scale / a.cap : a.scale * VX_LOG2E, e - 15);
        }

        f4 o[NB][2] = {};
        float M = -__builtin_inff(), l = 0.f;
        const int32_t* table = a.table + (uint64_t)s * a.table_stride;
        const uint8_t* base = a.c.base + (uint64_t)(kvh << (a.c.page_shift - 4)) * REC;
        const int last = min(q.len, (int)(a.table_cols << a.c.page_shift)) - 1;
        const float capl = a.cap * VX_LOG2E;

        // records of the next keys are requested while these are computed, and
        // the page of the ones after those
        constexpr bool AHEAD = NB <= 4;  // (registers: larger heads fill them)
        raw_k rk;
        raw_v rv;
        const uint8_t* at[2];
        const int kfirst = kbeg + 32 * (int)wave;
        if (kfirst < kend) {
#pragma unroll
            for (int t = 0; t < 2; ++t) at[t] = record(a, table, base, kfirst + 16 * t, last);
            if (AHEAD) {
                load(at, lane, g, rk, rv);
#pragma unroll
                for (int t = 0; t < 2; ++t) at[t] = record(a, table, base, kfirst + 128 + 16 * t, last);
            }
        }
        for (int k0 = kfirst; k0 < kend; k0 += 128) {
            raw_k nk;
            raw_v nv;
            if (AHEAD) load(at, lane, g, nk, nv);
            else load(at, lane, g, rk, rv);
#pragma unroll
            for (int t = 0; t < 2; ++t) at[t] = record(a, table, base, k0 + (AHEAD ? 256 : 128) + 16 * t, last);
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
                    for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(acc[i], (float)rk.s[t][b][i], sum[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) x[t][i] = sum[i] * fq;
            }
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
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = k0 + 16 * t + 4 * (int)g + i;
                        float dist = fabsf((float)(w.pos - key));
                        bool v;
                        if (key < tail) v = key >= w.lo && key < w.hi;
                        else v = a.tree && vx_tree_sees(a, q, w, key, dist);
                        x[t][i] = v ? __builtin_fmaf(-w.slope, dist, x[t][i]) : -__builtin_inff();
                        // a lane's scales are of its own row: what the row does not see, which
                        // may be anything, counts nowhere
#pragma unroll
                        for (int b = 0; b < NB; ++b) rv.s[t][b][i] = v ? rv.s[t][b][i] : (_Float16)0.f;
                    }
            }
            // running maximum of score + exponent of V's scales
            float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
            {
                typedef uint16_t us2 __attribute__((ext_vector_type(2)));
                us2 big = {0, 0};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        typedef uint16_t us4 __attribute__((ext_vector_type(4)));
                        const us4 d = __builtin_bit_cast(us4, rv.s[t][b]) & (uint16_t)0x7FFF;
                        big = __builtin_elementwise_max(__builtin_elementwise_max(big, d.xy), d.zw);
                    }
                const int e = (int)(max(big.x, big.y) >> 10) - 15;
                top = vx_max_rows4(top + (float)(e - 13));  // P times scale below 2^14
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
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                h8 ph, pl;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        h2 hi, lo;
                        vx_two_terms(x[t][i], (float)rv.s[t][b][i], x[t][i + 1], (float)rv.s[t][b][i + 1], hi, lo);
                        const int n = 4 * t + i;
                        ph[n] = hi.x, ph[n + 1] = hi.y, pl[n] = lo.x, pl[n + 1] = lo.y;
                    }
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    h2 v0, v1, v2, v3;
                    vx_kv_vfrag<NB, VB>(rv.w[0], b, v, v0, v1);
                    vx_kv_vfrag<NB, VB>(rv.w[1], b, v, v2, v3);
                    const h8 vf = {v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
                    o[b][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, o[b][v], 0, 0, 0);
                    o[b][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, o[b][v], 0, 0, 0);
                }
            }
            if (AHEAD) {
                rk = nk;
                rv = nv;
            }
        }

        // the four waves' sums: lane (m, g) holds dims 32 b + 2 (4 g + i) + v of query m
        l = vx_sum_rows4(l);
        if (g == 0) {
            sh_ml[wave][m][0] = M;
            sh_ml[wave][m][1] = l;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(f2*)&sh_o[wave][m][32 * b + 8 * g + 2 * i] = f2{o[b][0][i], o[b][1][i]};
        __syncthreads();
        const uint32_t D = 32 * NB;
        const bool parts = a.splits > 1;
        for (uint32_t at = threadIdx.x; at < 16 * (D / 4); at += 256) {
            const uint32_t row = at / (D / 4), d = 4 * (at % (D / 4));
            if (r0 + row >= rows) break;  // (rows grow with at)
            float Mt = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 4; ++i) Mt = fmaxf(Mt, sh_ml[i][row][0]);
            const float Mr = Mt == -__builtin_inff() ? 0.f : Mt;
            f4 t = {};
            float lt = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float c = __builtin_amdgcn_exp2f(sh_ml[i][row][0] - Mr);
                t += c * *(const f4*)&sh_o[i][row][d];
                lt = __builtin_fmaf(c, sh_ml[i][row][1], lt);
            }
            const uint32_t j = (r0 + row) / a.group, token = (uint32_t)q.start + j, head = kvh * a.group + (r0 + row - j * a.group);
            if (parts) {
                const uint64_t at_row = ((uint64_t)split * a.tokens + token) * (a.c.heads * a.group) + head;
                if (kbeg < kend) *(f4*)(a.part_o + at_row * D + d) = t;
                if (d == 0) *(f2*)(a.part_ml + at_row * 2) = f2{Mt, lt};
            } else {
                const float r = lt == 0.f ? 0.f : 1.f / lt;  // nothing seen: zeros
                float* op = a.out + (int64_t)token * a.os[0] + (int64_t)head * a.os[1];
                if (a.vec) {
                    *(f4*)(op + d) = t * r;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) op[(int64_t)(d + i) * a.os[2]] = t[i] * r;
                }
            }
        }
    }
};

// Joins the splits of a query row: 16 to 64 lanes take its dims, four at a
// time, and the splits go over the groups of lanes, of a wave where there are
// up to 8 splits (four rows a workgroup) and of the workgroup above (one row).
// One group a row took 90 us for 64 rows of 128 splits, this 4.
__device__ __forceinline__ void vx_attn_join_rows(const vx_attn_args& a) {
    __shared__ f4 sh_t[256];
    __shared__ f2 sh_ml[64];
    const uint32_t D = a.c.dim, lanes = D <= 64 ? 16 : D <= 128 ? 32 : 64;  // of a group
    const uint32_t span = a.splits > 8 ? 256 : 64;                         // threads of a row
    const uint32_t in = threadIdx.x % span, group = in / lanes, groups = span / lanes, d = 4 * (in % lanes);
    uint32_t id = blockIdx.x * (256 / span) + threadIdx.x / span;
    const uint32_t kvh = id % a.c.heads;
    id /= a.c.heads;
    const uint32_t s = id % a.seqs, r = id / a.seqs;
    const vx_attn_seq q = vx_attn_sequence(a, s);
    const bool valid = r < q.rows && d < D;
    const uint32_t heads = a.c.heads * a.group, j = r / a.group, head = kvh * a.group + (r - j * a.group);
    const uint64_t stride = (uint64_t)a.tokens * heads, row = ((uint64_t)q.start + j) * heads + head;
    float M = -__builtin_inff(), l = 0.f;
    f4 t = {};
    if (valid) {
#pragma unroll 4
        for (uint32_t i = group; i < a.splits; i += groups) {
            const f2 ml = *(const f2*)(a.part_ml + (i * stride + row) * 2);
            if (ml.y == 0.f) continue;  // nothing seen there, and nothing written (not so for a NaN)
            const f4 o = *(const f4*)(a.part_o + (i * stride + row) * D + d);
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
    const float k = l == 0.f ? 0.f : 1.f / l;
    float* op = a.out + (int64_t)(q.start + j) * a.os[0] + (int64_t)head * a.os[1];
    if (a.vec) {
        *(f4*)(op + d) = t * k;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) op[(int64_t)(d + i) * a.os[2]] = t[i] * k;
    }
}
