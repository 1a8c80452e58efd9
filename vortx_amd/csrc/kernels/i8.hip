// i8.hip — products of 8-bit integers with a scale for each token and channel:
// out[t, n] = sx[t] sw[n] sum_k x[t, k] w[n, k], and act(x gate^T) (x up^T) of two.
//
// Sums are int32 on the int8 matrix cores, exact for any order, so every kernel and
// every way of splitting K gives the same bits. A matrix instruction takes 16 bytes
// a lane of both operands, 16 rows x 64 k; channels are its rows, tokens its
// columns, so that a lane ends with four neighbouring channels of a token.
#include "vx_i8.hpp"

// The largest of the 64 lanes' numbers, by lane moves (lanes without a source take part with 0).
__device__ __forceinline__ uint32_t vx_wave_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// ---------------------------------------------------------------- quantize
// A workgroup a row. C fours of each thread stay in registers between the two
// passes over a row (its largest value, its codes); what is longer is read again.
// Bound by memory, or by a row's latency where there are few: 4096 x 4096 16.0 us, 5.2
// TB/s; 100 x 11008 3.0 with 1024 threads a row (3.6 with 256; 17 x 65536 7.6 and 20).
template <int C, uint32_t THREADS>
__device__ __forceinline__ void vx_i8_quantize_row(const vx_i8_quant_args& a, uint32_t row, uint32_t* part) {
    const float* p = a.x + (int64_t)row * a.xs[0];
    int8_t* q = a.out + (uint64_t)row * a.row_stride;
    const uint32_t tid = threadIdx.x, K = a.cols;
    uint32_t m = 0;
    f4v keep[C > 0 ? C : 1];
    if constexpr (C > 0) {
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) {
            const uint32_t k = 4 * (c * THREADS + tid);
            keep[c] = k + 4 <= K ? *(const f4v*)(p + k) : f4v{};
        }
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) m = vx_max4(m, keep[c]);
        for (uint32_t k = 4 * (C * THREADS + tid); k + 4 <= K; k += 4 * THREADS) m = vx_max4(m, *(const f4v*)(p + k));
        if (tid < K % 4) m = max(m, vx_abs_bits(p[K / 4 * 4 + tid]));
    } else {
        for (uint32_t k = tid; k < K; k += THREADS) m = max(m, vx_abs_bits(p[(int64_t)k * a.xs[1]]));
    }
    m = vx_wave_max(m);
    if ((tid & 63) == 0) part[tid >> 6] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (uint32_t i = 0; i < THREADS / 64; ++i) m = max(m, part[i]);
    float r;
    const float d = vx_i8_scale(m, r);
    if (tid == 0) a.scales[row] = d;
    if constexpr (C > 0) {
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) {
            const uint32_t k = 4 * (c * THREADS + tid);
            if (k + 4 <= K) *(uint32_t*)(q + k) = vx_i8_codes(keep[c], r);
        }
        for (uint32_t k = 4 * (C * THREADS + tid); k + 4 <= K; k += 4 * THREADS) *(uint32_t*)(q + k) = vx_i8_codes(*(const f4v*)(p + k), r);
        if (tid < K % 4) q[K / 4 * 4 + tid] = (int8_t)vx_i8_code(p[K / 4 * 4 + tid], r);
    } else {
        for (uint32_t k = tid; k < K; k += THREADS) q[k] = (int8_t)vx_i8_code(p[(int64_t)k * a.xs[1]], r);
    }
}
#define VX_I8_QUANTIZE(name, C, THREADS)                                                                 \
    extern "C" __global__ __launch_bounds__(THREADS) void name(vx_i8_quant_args a) {                     \
        __shared__ uint32_t part[2][THREADS / 64];                                                                  \
        uint32_t flip = 0;                                                                               \
        for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1)                       \
            vx_i8_quantize_row<C, THREADS>(a, (uint32_t)row, part[flip]);                                         \
    }
VX_I8_QUANTIZE(vx_i8_quantize_c4, 4, 256)
VX_I8_QUANTIZE(vx_i8_quantize_c16, 16, 256)
VX_I8_QUANTIZE(vx_i8_quantize_long, 4, 1024)
VX_I8_QUANTIZE(vx_i8_quantize_any, 0, 256)

// Neighbouring numbers of an order in which each XCD (workgroups go to the eight in
// turn) has a run of its own: what workgroups of a run share stays in its L2.
__device__ __forceinline__ uint32_t vx_xcd_order(uint32_t id, uint32_t n) {
    const uint32_t each = n / 8, more = n % 8, x = id % 8, i = id / 8;
    return x * each + min(x, more) + i;
}

// A barrier for what is in LDS: loads from memory stay on their way.
__device__ __forceinline__ void vx_lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---------------------------------------------------------------- few tokens
// TT x 16 tokens by NT x 16 channels (of each matrix) a workgroup of eight waves,
// which have K's pieces of 64 U bytes in turn, straight from memory to the matrix
// cores; their sums meet in LDS at the end. Bound by what a CU takes from L2 and
// memory, about 37 GB/s: 11008 x 4096 by 16 tokens 16.1 us, 64 22.3, 128 28.7; 32
// tokens gated 26.2.
template <int TT, int NT, int U, bool GATED>
struct vx_i8_direct {
    static constexpr int G = GATED ? 2 : 1, A = NT * G;
    i4v wr[2][U][A], xr[2][U][TT];
    i4v acc[A][TT];

    static __device__ __forceinline__ i4v masked(i4v v, int32_t have) {  // the first `have` bytes
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int32_t n = have - 4 * i;
            v[i] = n >= 4 ? v[i] : n <= 0 ? 0 : v[i] & (int)((1u << (8 * n)) - 1u);
        }
        return v;
    }

    __device__ __forceinline__ void run(const vx_i8_args& a, uint8_t* lds) {
        const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, kg = lane >> 4;
        const uint32_t tile = vx_xcd_order(blockIdx.x, a.tiles_t * a.tiles_n);
        const uint32_t t0 = tile % a.tiles_t * (16 * TT), n0 = tile / a.tiles_t * (16 * NT);
        const int8_t* wp[A];
        const int8_t* xp[TT];
#pragma unroll
        for (int i = 0; i < A; ++i) {
            const uint32_t n = min(n0 + 16u * (i / G) + m, a.N - 1u);
            wp[i] = a.w[i % G] + (uint64_t)n * a.ws[i % G] + 16 * kg;
        }
#pragma unroll
        for (int j = 0; j < TT; ++j) xp[j] = a.x + (uint64_t)min(t0 + 16u * j + m, a.T - 1u) * a.xs + 16 * kg;
#pragma unroll
        for (int i = 0; i < A; ++i)
#pragma unroll
            for (int j = 0; j < TT; ++j) acc[i][j] = i4v{};
        constexpr uint32_t P = 64 * U;
        const uint32_t full = a.K / P;
        auto load = [&](int b, uint32_t c) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < A; ++i) wr[b][u][i] = *(const i4v*)(wp[i] + (uint64_t)c * P + 64 * u);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < TT; ++j) xr[b][u][j] = *(const i4v*)(xp[j] + (uint64_t)c * P + 64 * u);
        };
        auto multiply = [&](int b) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < A; ++i)
#pragma unroll
                    for (int j = 0; j < TT; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wr[b][u][i], xr[b][u][j], acc[i][j], 0, 0, 0);
            }
        };
        if (wave < full) load(0, wave);
        for (uint32_t c = wave; c < full; c += 16) {
            if (c + 8 < full) load(1, c + 8);
            multiply(0);
            if (c + 16 < full) load(0, c + 16);
            if (c + 8 < full) multiply(1);
        }
        // the rest of K, 64 bytes a wave; nothing past the 16 bytes that K ends in is read
        const uint32_t left = a.K - full * P;
        for (uint32_t s = (wave + 8u - full % 8u) % 8u; 64 * s < left; s += 8) {
            const uint32_t k = full * P + 64 * s;
            const int32_t have = (int32_t)a.K - (int32_t)(k + 16 * kg);
            i4v x[TT], w[A];
#pragma unroll
            for (int i = 0; i < A; ++i) w[i] = *(const i4v*)(wp[i] + (have > 0 ? (int64_t)k : -16 * (int64_t)kg));
#pragma unroll
            for (int j = 0; j < TT; ++j) x[j] = masked(*(const i4v*)(xp[j] + (have > 0 ? (int64_t)k : -16 * (int64_t)kg)), have);
#pragma unroll
            for (int i = 0; i < A; ++i)
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x[j], acc[i][j], 0, 0, 0);
        }
        // the eight waves' sums, eight fragments (of a product, or pairs of two) a round
        constexpr int F = NT * TT, R = GATED ? 4 : 8;
        i4v* sums = (i4v*)lds;
#pragma unroll
        for (int f0 = 0; f0 < F; f0 += R) {
            if (f0) __syncthreads();
#pragma unroll
            for (int f = f0; f < F && f < f0 + R; ++f)
#pragma unroll
                for (int g = 0; g < G; ++g) sums[(((f - f0) * G + g) * 8 + wave) * 64 + lane] = acc[f / TT * G + g][f % TT];
            __syncthreads();
            const uint32_t f = f0 + wave;
            if (wave < R && f < F) {
                i4v s[2] = {};
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int v = 0; v < 8; ++v) s[g] += sums[((wave * G + g) * 8 + v) * 64 + lane];
                const uint32_t t = t0 + 16 * (f % TT) + m, n = n0 + 16 * (f / TT) + 4 * kg;
                vx_i8_finish4<GATED>(a, t, n, a.xscale[min(t, a.T - 1u)], s[0], s[1], vx_i8_scales4(a.wscale[0], n, a.N),
                                     GATED ? vx_i8_scales4(a.wscale[1], n, a.N) : f4v{});
            }
        }
    }
};

extern __shared__ __align__(16) uint8_t vx_i8_lds[];
#define VX_I8_DIRECT(name, TT, NT, U, GATED)                                         \
    extern "C" __global__ __launch_bounds__(512) void name(vx_i8_args a) {           \
        vx_i8_direct<TT, NT, U, GATED> d;                                            \
        d.run(a, vx_i8_lds);                                                         \
    }
VX_I8_DIRECT(vx_i8_direct_t1, 1, 1, 2, false)
VX_I8_DIRECT(vx_i8_direct_t1_gated, 1, 1, 4, true)
VX_I8_DIRECT(vx_i8_direct_t2, 2, 2, 2, false)
VX_I8_DIRECT(vx_i8_direct_t2_gated, 2, 1, 2, true)
VX_I8_DIRECT(vx_i8_direct_t4, 4, 2, 2, false)
VX_I8_DIRECT(vx_i8_direct_t4_gated, 4, 1, 2, true)
VX_I8_DIRECT(vx_i8_direct_t4_wide, 4, 4, 1, false)
VX_I8_DIRECT(vx_i8_direct_t4_wide_gated, 4, 2, 1, true)

// ---------------------------------------------------------------- one to four tokens of f32
// A workgroup of 16 waves a CU. A wave reads a row of the weights as it lies in memory,
// 1 KB a load and four loads a step (of a gated product a row of each), DEPTH steps ahead
// over the ends of its rows, against x's codes in LDS on the dot-product units; a.split
// waves share a row where there are fewer rows than waves. x is quantized into LDS by
// each workgroup for itself, under its first loads, which saves the launch that would
// do it. Bound by HBM, the weights' bytes, and what a launch takes to begin; a step is
// kept short, because with 100 instructions more a kilobyte their issue was the bound.
// One token by 32000 x 4096 25.6 us, 5.1 TB/s; by 11008 x 4096 11.5 (gated 18.2; a row a
// wave and step of 8 KB, loads under conditions: 13.4 and 24); two tokens 12.6, four 15.9.
template <int TT, bool GATED, int DEPTH>
struct vx_i8_stream {
    static constexpr int G = GATED ? 2 : 1;

    // What a thread has of x: four values of every 4096 of a row, row after row; of a few they stay in registers.
    static constexpr uint32_t KEEP = 4;
    f4v kept[KEEP];
    static __device__ __forceinline__ f4v get(const vx_i8_args& a, uint32_t t, uint32_t k) {
        const float* p = a.xf + (int64_t)t * a.xfs[0];
        f4v v = {};
        if (a.xf_vec && k + 4 <= a.K) return *(const f4v*)(p + k);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (k + i < a.K) v[i] = p[(int64_t)(k + i) * a.xfs[1]];
        return v;
    }
    __device__ __forceinline__ void keep(const vx_i8_args& a, uint32_t each) {  // each: such fours of a row
#pragma unroll
        for (uint32_t j = 0; j < KEEP; ++j)
            if (j < each * a.T) kept[j] = get(a, j / each, (j % each) * 4096 + 4 * threadIdx.x);
    }
    // x's rows as codes in LDS, zeros from K to the next multiple of 4096; returns their scales.
    __device__ __forceinline__ const float* quantize(const vx_i8_args& a, uint8_t* lds, uint32_t each) {
        const uint32_t tid = threadIdx.x, end = (a.K + 4095) / 4096 * 4096;
        uint32_t* part = (uint32_t*)(lds + a.T * a.pitch);
        float* sx = (float*)(part + VX_I8_OWN_TOKENS * 16);
        const bool few = each * a.T <= KEEP;
        for (uint32_t t = 0; t < a.T; ++t) {
            uint32_t m = 0;
            if (few) {
#pragma unroll
                for (uint32_t j = 0; j < KEEP; ++j)
                    if (j / each == t) m = vx_max4(m, kept[j]);
            } else {
                for (uint32_t k = 4 * tid; k < a.K; k += 4096) m = vx_max4(m, get(a, t, k));
            }
            m = vx_wave_max(m);
            if ((tid & 63) == 0) part[t * 16 + (tid >> 6)] = m;
        }
        vx_lds_barrier();
        for (uint32_t t = 0; t < a.T; ++t) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) m = max(m, part[t * 16 + i]);
            float r;
            const float d = vx_i8_scale(m, r);
            if (tid == 0) sx[t] = d;
            auto put = [&](uint32_t k, f4v v) {
                if (k < end) *(uint32_t*)(lds + t * a.pitch + k) = k < a.K ? vx_i8_codes(v, r) : 0u;
            };
            if (few) {
#pragma unroll
                for (uint32_t j = 0; j < KEEP; ++j)
                    if (j / each == t) put((j % each) * 4096 + 4 * tid, kept[j]);
            } else {
                for (uint32_t k = 4 * tid; k < end; k += 4096) put(k, get(a, t, k));
            }
        }
        vx_lds_barrier();
        return sx;
    }

    static __device__ __forceinline__ int wave_sum(int v) {
        v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
        return __builtin_amdgcn_readlane(v, 63);
    }

    i4v w[DEPTH][G][4];
    int acc[G][TT];
    float sw[G];       // the row's scales
    uint32_t part[4];  // where this lane's pieces of a row's last step lie

    __device__ __forceinline__ void load(const vx_i8_args& a, int b, uint32_t row, uint32_t c, bool last) {
        row = min(row, a.N - 1u);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int8_t* p = a.w[g] + (uint64_t)row * a.ws[g] + 4096 * c;
            if (last) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[b][g][i] = *(const i4v*)(p + part[i]);
            } else {
                const uint32_t at = 16 * (threadIdx.x & 63);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[b][g][i] = *(const i4v*)(p + at + 1024 * i);
            }
        }
    }
    __device__ __forceinline__ void multiply(const uint8_t* x, uint32_t pitch, int b) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const i4v v = *(const i4v*)(x + t * pitch + 1024 * i);
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[g][t] = __builtin_amdgcn_sdot4(w[b][g][i][j], v[j], acc[g][t], false);
            }
    }
    // by scalar loads: the weights' loads are not waited for with them
    __device__ __forceinline__ void scales(const vx_i8_args& a, uint32_t row) {
        typedef const __attribute__((address_space(4))) float* scalars;
#pragma unroll
        for (int g = 0; g < G; ++g) sw[g] = ((scalars)(uintptr_t)a.wscale[g])[min(row, a.N - 1u)];
    }
    // The row's end: its sums meet, lane t writes token t's value.
    __device__ __forceinline__ void finish(const vx_i8_args& a, int* sums, uint32_t wave, uint32_t share, uint32_t row, uint32_t round, vx_i8_scaled x) {
        const uint32_t lane = threadIdx.x & 63;
        int s[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            s[g] = 0;
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const int v = wave_sum(acc[g][t]);
                if (lane == (uint32_t)t) s[g] = v;
                acc[g][t] = 0;
            }
        }
        if (a.split > 1) {  // (two places in turn: a place is written again behind the barrier after its reading)
            int* at = sums + round % 2 * (16 * G * TT);
#pragma unroll
            for (int g = 0; g < G; ++g)
                if (lane < TT) at[(wave * G + g) * TT + lane] = s[g];
            vx_lds_barrier();
#pragma unroll
            for (int g = 0; g < G; ++g) {
                s[g] = 0;
                for (uint32_t v = 0; v < a.split; ++v) s[g] += at[((wave - share + v) * G + g) * TT + min(lane, TT - 1u)];
            }
        }
        if (share == 0 && lane < a.T && row < a.N) {
            float v[1] = {vx_i8_value(s[0], x, vx_i8_scaled(sw[0]))};
            if constexpr (GATED) {
                vx_act(a.act, v);
                v[0] *= vx_i8_value(s[1], x, vx_i8_scaled(sw[1]));
            }
            a.out[lane * a.os[0] + row * a.os[1]] = v[0];
        }
    }

    __device__ __forceinline__ void run(const vx_i8_args& a, uint8_t* lds) {
        const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t per = 16 / a.split, share = wave % a.split;  // rows of a workgroup at a time; which part of its row
        const uint32_t hop = a.tiles_n * per, rounds = (a.N + hop - 1) / hop;
        const uint32_t fours = (a.K + 4095) / 4096, steps = (fours + a.split - 1) / a.split;  // of a row, and of a wave's share
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t at = 1024 * i + 16 * lane;
            part[i] = (fours - 1) * 4096 + at < a.K ? at : 0u;  // (past K: something of the row, times zeros)
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[g][t] = 0;
        // Loads arrive in the order of their requests: x goes before the weights, so that it is quantized while those
        // are on their way.
        if (fours * a.T <= KEEP) keep(a, fours);
        asm volatile("" ::: "memory");
        uint32_t row = blockIdx.x * per + wave / a.split, c = share, round = 0;  // the step at hand: 4096 bytes c of a row
        uint32_t row_l = row, c_l = share;                                      // and the next one to request
        // (past a row's share: its last ones again, and nothing comes of it; past the last row, the last row)
        auto request = [&](int b) {
            const uint32_t k = min(c_l, fours - 1u);
            load(a, b, row_l, k, k + 1 == fours);
            if ((c_l += a.split) >= steps * a.split) c_l = share, row_l = min(row_l + hop, a.N);
        };
        const uint32_t all = rounds * steps;
        const bool few = all < DEPTH;
        const float* sx;
        if (few) {
            request(0);
            asm volatile("" ::: "memory");
            sx = quantize(a, lds, fours);
        } else {
#pragma unroll
            for (int b = 0; b < DEPTH; ++b) request(b);
            asm volatile("" ::: "memory");
            sx = quantize(a, lds, fours);
        }
        const vx_i8_scaled scale(sx[min(lane, a.T - 1u)]);
        int* sums = (int*)(lds + a.x_bytes);  // [2][16 waves][G][TT], of rows that waves share
        auto take = [&](int b) {
            if (c < fours) multiply(lds + 16 * lane + 4096 * c, a.pitch, b);
            if ((c += a.split) < steps * a.split) return;
            finish(a, sums, wave, share, row, round, scale);
            c = share;
            row += hop;
            ++round;
            scales(a, row);
        };
        scales(a, row);
        if (few) {
            for (uint32_t q = 0; q < all; ++q) {
                take(0);
                if (q + 1 < all) request(0);
            }
            return;
        }
        uint32_t q = 0;
        for (; q + 2 * DEPTH <= all; q += DEPTH)
#pragma unroll
            for (int b = 0; b < DEPTH; ++b) {
                take(b);
                request(b);
            }
        const uint32_t left = all - q;  // DEPTH to 2 DEPTH - 1, the first DEPTH of them requested
#pragma unroll
        for (int b = 0; b < DEPTH; ++b) {
            take(b);
            if ((uint32_t)b + DEPTH < left) request(b);
        }
#pragma unroll
        for (int b = 0; b < DEPTH; ++b)
            if ((uint32_t)b + DEPTH < left) take(b);
    }
};
#define VX_I8_STREAM(name, TT, GATED, DEPTH)                                         \
    extern "C" __global__ __launch_bounds__(1024) void name(vx_i8_args a) {          \
        vx_i8_stream<TT, GATED, DEPTH> s;                                            \
        s.run(a, vx_i8_lds);                                                         \
    }
VX_I8_STREAM(vx_i8_stream_t1, 1, false, 2)
VX_I8_STREAM(vx_i8_stream_t1_gated, 1, true, 1)
VX_I8_STREAM(vx_i8_stream_t2, 2, false, 2)
VX_I8_STREAM(vx_i8_stream_t2_gated, 2, true, 1)
VX_I8_STREAM(vx_i8_stream_t4, 4, false, 2)
VX_I8_STREAM(vx_i8_stream_t4_gated, 4, true, 1)

// ---------------------------------------------------------------- many tokens
// Tiles of MT tokens by MN rows of weights (of a gated product half gate, half up,
// 16 and 16 in turn, so that a lane has both sums of an output), WT x WN waves, a
// workgroup one after the other. A stage is 128 bytes of K, whole cache lines, in two
// halves that a matrix instruction takes 64 bytes of; a unit is one operand of a stage,
// brought from memory straight into LDS, and five units go round: two are multiplied
// while three are on their way. The 16-byte pieces of a row are stored in an order that
// goes by the row, so that the lanes of a fragment (16 rows, one piece each) meet all
// banks. 4096 x 4096 x 11008 (tokens, channels, k) 158 us, 2330 TOP/s; 4096 x 11008 x
// 4096 205 us, 1800 (gated 414, 1785). A stage takes 1.7 us: the loads from memory take
// 1.4 of it by themselves (46 GB/s a CU), all else 1.3, of which the matrix instructions
// are 2048 cycles, 0.9 to 1.0, so that neither is the bound alone: it is how much of the
// one lies under the other. Counted over the last product, the matrix cores are busy 37 %
// of the cycles (45 % of those in which their CU has work: 688 tiles are 2.7 rounds), LDS
// with reads 14 %, without a bank conflict; a wave waits for data or the others 38 % of its time,
// and to issue 39 %. Beside the stages the stores, which all CUs make at the same time, 16 us
// a tile of each CU.
template <int MT, int MN, int WT, int WN, bool GATED, bool PART = false>
struct vx_i8_tile {
    static_assert(MT == MN, "units of one size");
    static constexpr int WAVES = WT * WN, THREADS = 64 * WAVES;
    static constexpr int FT = MT / (16 * WT), FN = MN / (16 * WN);  // fragments of a wave
    static constexpr uint32_t UNIT = 128 * MT, UNITS = 5;
    static constexpr int PIECES = MT / 8 / WAVES;  // loads of a wave and unit, 8 rows each
    static_assert(PIECES * WAVES * 8 == MT && PIECES == 4, "a wave loads 32 rows of a unit");

    // piece `c` (of eight) of row r within a unit
    static __device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) { return r * 128 + ((c ^ (r >> 1)) & 7) * 16; }

    const vx_i8_args& a;
    const uint32_t tid, lane, m, kg, wave;
    uint32_t K, S, last;  // columns (of the part), stages, where the last one begins
    uint32_t part_of;
    uint32_t off_w[PIECES], off_x[PIECES];  // within the operands' first stage
    i4v base_w[2], base_x;
    uint32_t t0, n0, lds0;

    static __device__ __forceinline__ i4v buffer(const int8_t* p) {  // without an end
        const uint64_t u = (uint64_t)(uintptr_t)p;
        return i4v{(int)__builtin_amdgcn_readfirstlane((int)(uint32_t)u), (int)(__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32)) & 0xFFFF), -1, 0x00027000};
    }
    __device__ __forceinline__ vx_i8_tile(const vx_i8_args& a_, uint8_t* lds)
        : a(a_), tid(threadIdx.x), lane(tid & 63), m(lane & 15), kg(lane >> 4), wave(__builtin_amdgcn_readfirstlane(tid >> 6)),
          K(a_.K), S((a_.K + 127) / 128), last(128 * (S - 1)), part_of(0),
          lds0(__builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds)) {}

    // The loads of tile `id` of all in their order.
    __device__ __forceinline__ void place(uint32_t id) {
        // in bands of eight tiles of tokens: the 32 tiles that an XCD works on at a time are 8 by 4,
        // so that its L2 takes 12 operands of a tile from farther away, where 16 by 2 takes 18
        uint32_t tile = vx_xcd_order(id, a.tiles_t * a.tiles_n * (PART ? a.split : 1u)), k0 = 0;
        if constexpr (PART) {  // (an XCD has whole parts where it can: its L2 then takes each column of x and of the weights once)
            part_of = tile / (a.tiles_t * a.tiles_n);
            tile -= part_of * a.tiles_t * a.tiles_n;
            k0 = part_of * a.chunk;
            K = min(a.K - k0, a.chunk);
            S = (K + 127) / 128;
            last = 128 * (S - 1);
        }
        const uint32_t band = tile / (8 * a.tiles_n), in = tile - band * 8 * a.tiles_n;
        const uint32_t high = min(8u, a.tiles_t - 8 * band);
        t0 = (8 * band + in % high) * MT;
        n0 = in / high * (GATED ? MN / 2 : MN);
        base_w[0] = buffer(a.w[0] + (uint64_t)n0 * a.ws[0] + k0);
        base_w[1] = GATED ? buffer(a.w[1] + (uint64_t)n0 * a.ws[1] + k0) : base_w[0];
        base_x = buffer(a.x + (uint64_t)t0 * a.xs + k0);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const uint32_t r = wave * 32 + 8 * p + lane / 8, c = piece(p);
            const uint32_t n = GATED ? n0 + r / 32 * 16 + r % 16 : n0 + r;  // (a piece is all gate or all up)
            const uint32_t w = (min(n, a.N - 1u) - n0) * (uint32_t)a.ws[GATED ? p / 2 : 0], x = (min(t0 + r, a.T - 1u) - t0) * (uint32_t)a.xs;
            off_w[p] = w + 16 * c;
            off_x[p] = x + 16 * c;
        }
    }
    // which piece of its row this lane has
    __device__ __forceinline__ uint32_t piece(int p) const { return ((lane & 7) ^ (4 * p + lane / 16)) & 7; }
    __device__ __forceinline__ void load(const uint32_t (&from)[PIECES], const i4v& b0, const i4v& b1, uint32_t slot, uint32_t k) {
        const uint32_t to = lds0 + slot * UNIT + wave * 4096;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(to + 1024 * p), "v"(from[p]), "s"(p / 2 ? b1 : b0), "s"(k) : "memory");
    }
    // Unit u of the tile: the weights of stage u / 2 or x. In the last stage pieces past K are the row's first (and count for nothing).
    __device__ __forceinline__ void request(uint32_t u, uint32_t slot) {
        const uint32_t s = u / 2;
        if (s >= S) return;
        const bool end = s + 1 == S && K % 128;
        uint32_t from[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const uint32_t k = 16 * piece(p);
            from[p] = (u & 1 ? off_x[p] : off_w[p]) + (end ? (last + k < K ? last : 0u - k) : 128 * s);
        }
        load(from, u & 1 ? base_x : base_w[0], u & 1 ? base_x : base_w[1], slot, 0);
    }

    __device__ __forceinline__ void run(uint8_t* lds) {
        const uint32_t wn = wave % WN * (16 * FN), wt = wave / WN * (16 * FT);
        const uint32_t tiles = a.tiles_t * a.tiles_n;
        i4v acc[FN][FT], x[2][FT], w[2][FN];
        auto fetch = [&](int b, uint32_t slot_w, uint32_t slot_x, uint32_t half) {
            const uint8_t *pw = lds + slot_w * UNIT, *px = lds + slot_x * UNIT;
#pragma unroll
            for (int j = 0; j < FT; ++j) x[b][j] = *(const i4v*)(px + at(wt + 16 * j + m, 4 * half + kg));
#pragma unroll
            for (int i = 0; i < FN; ++i) w[b][i] = *(const i4v*)(pw + at(wn + 16 * i + m, 4 * half + kg));
        };
        auto multiply = [&](int b) {
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[b][i], x[b][j], acc[i][j], 0, 0, 0);
        };
        // x past K in the last stage becomes zeros
        auto clear = [&](uint32_t slot) {
            const uint32_t have = K - last;
            if (have == 128) return;
            for (uint32_t i = tid; i < MT * 8; i += THREADS) {
                const uint32_t r = i / 8, c = i % 8;
#pragma unroll
                for (uint32_t d = 0; d < 4; ++d) {
                    const int32_t n = (int32_t)have - (int32_t)(16 * c + 4 * d);
                    uint32_t* q = (uint32_t*)(lds + slot * UNIT + at(r, c)) + d;
                    if (n < 4) *q = n <= 0 ? 0u : *q & ((1u << (8 * n)) - 1u);
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        };
        // all units but the last n requested are there, for all waves
        auto arrived = [](uint32_t n) {
            switch (n) {
                case 3: asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(3 * PIECES) : "memory"); break;
                case 2: asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(2 * PIECES) : "memory"); break;
                case 1: asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(PIECES) : "memory"); break;
                default: asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
        };
        auto next = [](uint32_t slot, uint32_t by) { return slot + by >= UNITS ? slot + by - UNITS : slot + by; };

        uint32_t id = blockIdx.x;
        place(id);
        for (uint32_t u = 0; u < UNITS; ++u) request(u, u);
        while (true) {
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FT; ++j) acc[i][j] = i4v{};
            // stage 0 is there (its units are the oldest requests; stores of the tile before may be among the newer ones)
            arrived(min(2 * S, UNITS) - 2);
            if (S == 1) clear(1);
            uint32_t at_w = 0, at_x = 1;  // slots of stage s
            fetch(0, at_w, at_x, 0);
            uint32_t s = 0;
            // While a half is multiplied, the next one is read. At the barrier every wave has the whole of
            // stage s in registers, stage s + 1 is there and the weights of s + 2 may be on their way; the two
            // free slots take x of s + 2 and the weights of s + 3.
            for (; s + 4 < S; ++s) {
                fetch(1, at_w, at_x, 1);
                multiply(0);
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(PIECES) : "memory");
                load(off_x, base_x, base_x, at_w, 128 * (s + 2));
                load(off_w, base_w[0], base_w[1], at_x, 128 * (s + 3));
                at_w = next(at_w, 2);
                at_x = next(at_x, 2);
                fetch(0, at_w, at_x, 0);
                multiply(1);
            }
            for (; s < S; ++s) {
                fetch(1, at_w, at_x, 1);
                multiply(0);
                if (s + 1 < S) {
                    arrived(min(2 * S, 2 * s + UNITS) - (2 * s + 4));
                    request(2 * s + UNITS, at_w);
                    request(2 * s + UNITS + 1, at_x);
                    at_w = next(at_w, 2);
                    at_x = next(at_x, 2);
                    if (s + 2 == S) clear(at_x);
                    fetch(0, at_w, at_x, 0);
                }
                multiply(1);
            }
            const uint32_t tt = t0 + wt + m, nn = n0 + (GATED ? wn / 2 : wn) + 4 * kg;
            if constexpr (PART) {
                const uint32_t pitch = (a.N + 3) / 4 * 4;
#pragma unroll
                for (int j = 0; j < FT; ++j)
#pragma unroll
                    for (int i = 0; i < FN; ++i) {
                        const uint32_t t = tt + 16 * j, n = nn + 16 * (GATED ? i / 2 : i), g = part_of * (GATED ? 2 : 1) + (GATED ? i & 1 : 0);
                        if (t < a.T && n < a.N) *(i4v*)(a.parts + ((uint64_t)g * a.T + t) * pitch + n) = acc[i][j];
                    }
                return;
            }
            // the results, under the first loads of the next tile (after the scales: loads end in order)
            float sx[FT];
            f4v sw[FN];
#pragma unroll
            for (int j = 0; j < FT; ++j) sx[j] = a.xscale[min(tt + 16 * j, a.T - 1u)];
#pragma unroll
            for (int i = 0; i < FN; ++i) sw[i] = vx_i8_scales4(a.wscale[GATED ? i & 1 : 0], nn + 16 * (GATED ? i / 2 : i), a.N);
#pragma unroll
            for (int j = 0; j < FT; ++j) asm volatile("" : "+v"(sx[j]));
#pragma unroll
            for (int i = 0; i < FN; ++i) asm volatile("" : "+v"(sw[i]));
            id += gridDim.x;
            const bool more = id < tiles;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (more) {
                place(id);
                for (uint32_t u = 0; u < UNITS; ++u) request(u, u);
            }
#pragma unroll
            for (int j = 0; j < FT; ++j)
#pragma unroll
                for (int i = 0; i < FN; i += GATED ? 2 : 1)
                    vx_i8_finish4<GATED>(a, tt + 16 * j, nn + 16 * (GATED ? i / 2 : i), sx[j], acc[i][j], GATED ? acc[i + 1][j] : i4v{}, sw[i],
                                         GATED ? sw[i + 1] : f4v{});
            if (!more) break;
        }
    }
};
#define VX_I8_TILE(name, threads, ...)                                                           \
    extern "C" __global__ __launch_bounds__(threads) void name(vx_i8_args a) {                   \
        using tile = vx_i8_tile<__VA_ARGS__>;                                                    \
        static_assert(tile::THREADS == threads, "waves of 64");                                  \
        __shared__ __align__(1024) uint8_t lds[tile::UNIT * tile::UNITS];                        \
        tile(a, lds).run(lds);                                                                   \
    }
VX_I8_TILE(vx_i8_tile256, 512, 256, 256, 2, 4, false)
VX_I8_TILE(vx_i8_tile256_gated, 512, 256, 256, 2, 4, true)
VX_I8_TILE(vx_i8_tile128, 256, 128, 128, 2, 2, false)
VX_I8_TILE(vx_i8_tile128_gated, 256, 128, 128, 2, 2, true)

// ---------------------------------------------------------------- a long K, few tiles
// Tiles of 128 over parts of K, whose sums a second launch joins: few tokens by few
// channels would otherwise leave CUs idle, or have all of them load the same rows.
VX_I8_TILE(vx_i8_part128, 256, 128, 128, 2, 2, false, true)
VX_I8_TILE(vx_i8_part128_gated, 256, 128, 128, 2, 2, true, true)

template <bool GATED>
__device__ __forceinline__ void vx_i8_join_rows(const vx_i8_args& a) {
    constexpr uint32_t G = GATED ? 2 : 1;
    const uint32_t fours = (a.N + 3) / 4;
    const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x, step = G * (uint64_t)a.T * fours;
    const uint32_t t = (uint32_t)(id / fours), n = 4 * (uint32_t)(id % fours);
    if (t >= a.T) return;
    const i4v* p = (const i4v*)a.parts + id;
    i4v s[2] = {};
#pragma unroll 4
    for (uint32_t q = 0; q < a.split; ++q)
#pragma unroll
        for (uint32_t g = 0; g < G; ++g) s[g] += p[q * step + g * (uint64_t)a.T * fours];
    vx_i8_finish4<GATED>(a, t, n, a.xscale[t], s[0], s[1], vx_i8_scales4(a.wscale[0], n, a.N), GATED ? vx_i8_scales4(a.wscale[1], n, a.N) : f4v{});
}
extern "C" __global__ __launch_bounds__(256) void vx_i8_join(vx_i8_args a) { vx_i8_join_rows<false>(a); }
extern "C" __global__ __launch_bounds__(256) void vx_i8_join_gated(vx_i8_args a) { vx_i8_join_rows<true>(a); }
