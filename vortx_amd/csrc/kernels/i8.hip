// i8.hip — products of 8-bit integers with a scale for each token and channel:
// out[t, n] = sx[t] sw[n] sum_k x[t, k] w[n, k], and act(x gate^T) (x up^T) of two.
//
// Sums are int32 on the int8 matrix cores, exact for any order, so every kernel and
// every way of splitting K gives the same bits. A matrix instruction takes 16 bytes
// a lane of both operands, 16 rows x 64 k; channels are its rows, tokens its
// columns, so that a lane ends with four neighbouring channels of a token.
#include "vx_i8.hpp"

// ---------------------------------------------------------------- quantize
// A workgroup a row. C fours of each thread stay in registers between the two
// passes over a row (its largest value, its codes); what is longer is read again.
template <int C>
__device__ __forceinline__ void vx_i8_quantize_row(const vx_i8_quant_args& a, uint32_t row, uint32_t* part) {
    const float* p = a.x + (int64_t)row * a.xs[0];
    int8_t* q = a.out + (uint64_t)row * a.row_stride;
    const uint32_t tid = threadIdx.x, K = a.cols;
    uint32_t m = 0;
    f4v keep[C > 0 ? C : 1];
    if constexpr (C > 0) {
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) {
            const uint32_t k = 4 * (c * 256 + tid);
            keep[c] = k + 4 <= K ? *(const f4v*)(p + k) : f4v{};
        }
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) m = vx_max4(m, keep[c]);
        for (uint32_t k = 4 * (C * 256 + tid); k + 4 <= K; k += 1024) m = vx_max4(m, *(const f4v*)(p + k));
        if (tid < K % 4) m = max(m, vx_abs_bits(p[K / 4 * 4 + tid]));
    } else {
        for (uint32_t k = tid; k < K; k += 256) m = max(m, vx_abs_bits(p[(int64_t)k * a.xs[1]]));
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    if ((tid & 63) == 0) part[tid >> 6] = m;
    __syncthreads();
    m = max(max(part[0], part[1]), max(part[2], part[3]));
    float r;
    const float d = vx_i8_scale(m, r);
    if (tid == 0) a.scales[row] = d;
    if constexpr (C > 0) {
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) {
            const uint32_t k = 4 * (c * 256 + tid);
            if (k + 4 <= K) *(uint32_t*)(q + k) = vx_i8_codes(keep[c], r);
        }
        for (uint32_t k = 4 * (C * 256 + tid); k + 4 <= K; k += 1024) *(uint32_t*)(q + k) = vx_i8_codes(*(const f4v*)(p + k), r);
        if (tid < K % 4) q[K / 4 * 4 + tid] = (int8_t)vx_i8_code(p[K / 4 * 4 + tid], r);
    } else {
        for (uint32_t k = tid; k < K; k += 256) q[k] = (int8_t)vx_i8_code(p[(int64_t)k * a.xs[1]], r);
    }
}
#define VX_I8_QUANTIZE(name, C)                                                                          \
    extern "C" __global__ __launch_bounds__(256) void name(vx_i8_quant_args a) {                         \
        __shared__ uint32_t part[2][4];                                                                  \
        uint32_t flip = 0;                                                                               \
        for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1)                       \
            vx_i8_quantize_row<C>(a, (uint32_t)row, part[flip]);                                         \
    }
VX_I8_QUANTIZE(vx_i8_quantize_c4, 4)
VX_I8_QUANTIZE(vx_i8_quantize_c16, 16)
VX_I8_QUANTIZE(vx_i8_quantize_any, 0)

// Neighbouring numbers of an order in which each XCD (workgroups go to the eight in
// turn) has a run of its own: what workgroups of a run share stays in its L2.
__device__ __forceinline__ uint32_t vx_xcd_order(uint32_t id, uint32_t n) {
    const uint32_t each = n / 8, more = n % 8, x = id % 8, i = id / 8;
    return x * each + min(x, more) + i;
}

// ---------------------------------------------------------------- few tokens
// TT x 16 tokens by NT x 16 channels (of each matrix) a workgroup of eight waves,
// which have K's pieces of 64 U bytes in turn, straight from memory to the matrix
// cores; their sums meet in LDS at the end. Bound by W's bytes. F32X: x comes as f32
// (its tokens at most 16) and every workgroup quantizes it for itself into LDS,
// under its first loads of W, which saves the launch that would do it.
template <int TT, int NT, int U, bool GATED, bool F32X>
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
        if constexpr (!F32X)
#pragma unroll
            for (int j = 0; j < TT; ++j) xp[j] = a.x + (uint64_t)min(t0 + 16u * j + m, a.T - 1u) * a.xs + 16 * kg;
        const uint32_t pitch = a.pitch;  // of x's rows in LDS
        const uint8_t* xl = lds + min(m, a.T - 1u) * pitch + 16 * kg;
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
            if constexpr (!F32X)
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < TT; ++j) xr[b][u][j] = *(const i4v*)(xp[j] + (uint64_t)c * P + 64 * u);
        };
        auto multiply = [&](int b, uint32_t c) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if constexpr (F32X) xr[b][u][0] = *(const i4v*)(xl + c * P + 64 * u);
#pragma unroll
                for (int i = 0; i < A; ++i)
#pragma unroll
                    for (int j = 0; j < TT; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wr[b][u][i], xr[b][u][j], acc[i][j], 0, 0, 0);
            }
        };
        if (wave < full) load(0, wave);
        float* sx = nullptr;
        if constexpr (F32X) sx = quantize(a, lds);
        for (uint32_t c = wave; c < full; c += 16) {
            if (c + 8 < full) load(1, c + 8);
            multiply(0, c);
            if (c + 16 < full) load(0, c + 16);
            if (c + 8 < full) multiply(1, c + 8);
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
            for (int j = 0; j < TT; ++j) {
                if constexpr (F32X) x[j] = *(const i4v*)(xl + k);  // (zeros past K)
                else x[j] = masked(*(const i4v*)(xp[j] + (have > 0 ? (int64_t)k : -16 * (int64_t)kg)), have);
            }
#pragma unroll
            for (int i = 0; i < A; ++i)
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x[j], acc[i][j], 0, 0, 0);
        }
        // the eight waves' sums, eight fragments (of a product, or pairs of two) a round
        constexpr int F = NT * TT, R = GATED ? 4 : 8;
        i4v* sums = (i4v*)(lds + (F32X ? a.x_bytes : 0));
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
                const float scale = F32X ? sx[min(m, a.T - 1u)] : a.xscale[min(t, a.T - 1u)];
                vx_i8_finish4<GATED>(a, t, n, scale, s[0], s[1], vx_i8_scales4(a.wscale[0], n, a.N),
                                     GATED ? vx_i8_scales4(a.wscale[1], n, a.N) : f4v{});
            }
        }
    }

    // x's rows as codes in LDS, zeros from K to the next multiple of 64; returns their scales.
    static __device__ __forceinline__ float* quantize(const vx_i8_args& a, uint8_t* lds) {
        const uint32_t tid = threadIdx.x, K = a.K;
        uint32_t* part = (uint32_t*)(lds + a.T * a.pitch);
        float* sx = (float*)(part + 8 * 16);
        const bool vec = a.xf_vec;
        auto get = [&](const float* p, uint32_t k) {
            f4v v = {};
            if (vec && k + 4 <= K) return *(const f4v*)(p + k);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (k + i < K) v[i] = p[(int64_t)(k + i) * a.xfs[1]];
            return v;
        };
        for (uint32_t t = 0; t < a.T; ++t) {
            const float* p = a.xf + (int64_t)t * a.xfs[0];
            uint32_t m = 0;
#pragma unroll 4
            for (uint32_t k = 4 * tid; k < K; k += 2048) m = vx_max4(m, get(p, k));
#pragma unroll
            for (int o = 32; o; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
            if ((tid & 63) == 0) part[t * 8 + (tid >> 6)] = m;
        }
        __syncthreads();
        const uint32_t end = (K + 63) / 64 * 64;
        for (uint32_t t = 0; t < a.T; ++t) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, part[t * 8 + i]);
            float r;
            const float d = vx_i8_scale(m, r);
            if (tid == 0) sx[t] = d;
            const float* p = a.xf + (int64_t)t * a.xfs[0];
#pragma unroll 4
            for (uint32_t k = 4 * tid; k < end; k += 2048) *(uint32_t*)(lds + t * a.pitch + k) = k < K ? vx_i8_codes(get(p, k), r) : 0u;
        }
        __syncthreads();
        return sx;
    }
};

extern __shared__ __align__(16) uint8_t vx_i8_lds[];
#define VX_I8_DIRECT(name, TT, NT, U, GATED, F32X)                                   \
    extern "C" __global__ __launch_bounds__(512) void name(vx_i8_args a) {           \
        vx_i8_direct<TT, NT, U, GATED, F32X> d;                                      \
        d.run(a, vx_i8_lds);                                                         \
    }
VX_I8_DIRECT(vx_i8_direct_x, 1, 1, 4, false, true)
VX_I8_DIRECT(vx_i8_direct_x_gated, 1, 1, 4, true, true)
VX_I8_DIRECT(vx_i8_direct_t1, 1, 1, 4, false, false)
VX_I8_DIRECT(vx_i8_direct_t1_gated, 1, 1, 4, true, false)
VX_I8_DIRECT(vx_i8_direct_t2, 2, 2, 2, false, false)
VX_I8_DIRECT(vx_i8_direct_t2_gated, 2, 1, 2, true, false)
VX_I8_DIRECT(vx_i8_direct_t4, 4, 2, 2, false, false)
VX_I8_DIRECT(vx_i8_direct_t4_gated, 4, 1, 2, true, false)

// ---------------------------------------------------------------- many tokens
// A tile of MT tokens by MN rows of weights (of a gated product half gate, half up,
// 16 and 16 in turn, so that a lane has both sums of an output), WT x WN waves. A
// stage is 64 bytes of K of both, brought from memory straight into LDS; four stages
// go round, three on their way while one is multiplied, with one barrier each. The
// 16-byte pieces of a row are stored in an order that goes by the row, so that the
// lanes of a fragment (16 rows, one piece each) meet all banks.
template <int MT, int MN, int WT, int WN, bool GATED>
struct vx_i8_tile {
    static constexpr int WAVES = WT * WN, THREADS = 64 * WAVES;
    static constexpr int FT = MT / (16 * WT), FN = MN / (16 * WN);  // fragments of a wave
    static constexpr uint32_t STAGE = 64 * (MT + MN), STAGES = 4;
    static constexpr int PIECES = (MT + MN) / 16 / WAVES;  // loads of a wave and stage, 16 rows each
    static_assert(PIECES * WAVES * 16 == MT + MN && (MN / 16) % PIECES == 0, "a wave's loads are all of one operand");

    // piece `c` (of four) of row r within a stage's operand
    static __device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) { return r * 64 + ((c ^ (r >> 1)) & 3) * 16; }

    static __device__ __forceinline__ void run(const vx_i8_args& a) {
        __shared__ __align__(1024) uint8_t lds[STAGE * STAGES];
        const uint32_t tid = threadIdx.x, lane = tid & 63, m = lane & 15, kg = lane >> 4;
        const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const uint32_t tile = vx_xcd_order(blockIdx.x, a.tiles_t * a.tiles_n);
        constexpr uint32_t CH = GATED ? MN / 2 : MN;  // channels of a tile
        const uint32_t t0 = tile % a.tiles_t * MT, n0 = tile / a.tiles_t * CH;
        // this wave's loads: 16 rows of the weights (first in LDS) or of x, four lanes a row
        uint32_t off[PIECES], cut[PIECES];  // of a stage inside K, and of the last one
        const uint32_t S = (a.K + 63) / 64, last = 64 * (S - 1);
        const uint32_t row0 = wave * PIECES * 16;
        const bool weights = row0 < MN;
        const int8_t* base[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const uint32_t r = row0 + 16 * p + lane / 4, c = ((lane & 3) ^ (r >> 1)) & 3;
            uint64_t row;
            if (weights) {
                const uint32_t g = GATED ? (row0 / 16 + p) & 1 : 0;  // (a piece is all gate or all up)
                const uint32_t n = GATED ? n0 + r / 32 * 16 + r % 16 : n0 + r;
                base[p] = a.w[g] + (uint64_t)n0 * a.ws[g];
                row = (uint64_t)(min(n, a.N - 1u) - n0) * a.ws[g];
            } else {
                base[p] = a.x + (uint64_t)t0 * a.xs;
                row = (uint64_t)(min(t0 + r - MN, a.T - 1u) - t0) * a.xs;
            }
            off[p] = (uint32_t)row + 16 * c;
            cut[p] = (uint32_t)row + (last + 16 * c < a.K ? last + 16 * c : 0u);
        }
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
        auto request = [&](uint32_t s) {
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const uint64_t b = (uint64_t)(uintptr_t)base[p];
                i4v rsrc;
                rsrc.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)b);
                rsrc.y = __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32) & 0xFFFF);
                rsrc.z = -1;
                rsrc.w = 0x00027000;
                const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + (s % STAGES) * STAGE + (row0 + 16 * p) * 64);
                const uint32_t v = s + 1 == S ? cut[p] : off[p], k = __builtin_amdgcn_readfirstlane(s + 1 == S ? 0u : 64 * s);
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                             :: "s"(to), "v"(v), "s"(rsrc), "s"(k) : "memory");
            }
        };
        i4v acc[FN][FT];
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FT; ++j) acc[i][j] = i4v{};
        const uint32_t wn = wave % WN * (16 * FN), wt = wave / WN * (16 * FT);
#pragma unroll
        for (uint32_t s = 0; s < STAGES - 1; ++s)
            if (s < S) request(s);
        for (uint32_t s = 0; s < S; ++s) {
            // stage s is there (later ones may be on their way), and no wave still reads the one before it
            if (s + 2 < S) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(2 * PIECES) : "memory");
            else if (s + 1 < S) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(PIECES) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (s + STAGES - 1 < S) request(s + STAGES - 1);
            uint8_t* stage = lds + (s % STAGES) * STAGE;
            if (s + 1 == S && a.K % 64) {  // x past K becomes zeros
                const uint32_t have = a.K % 64;
                for (uint32_t i = tid; i < MT * 4; i += THREADS) {
                    const uint32_t r = i / 4, c = i % 4;
                    uint8_t* p = stage + MN * 64 + at(r, c);
#pragma unroll
                    for (uint32_t w = 0; w < 4; ++w) {
                        const int32_t n = (int32_t)have - (int32_t)(16 * c + 4 * w);
                        uint32_t* q = (uint32_t*)p + w;
                        if (n < 4) *q = n <= 0 ? 0u : *q & ((1u << (8 * n)) - 1u);
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            i4v x[FT];
#pragma unroll
            for (int j = 0; j < FT; ++j) x[j] = *(const i4v*)(stage + MN * 64 + at(wt + 16 * j + m, kg));
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const i4v w = *(const i4v*)(stage + at(wn + 16 * i + m, kg));
#pragma unroll
                for (int j = 0; j < FT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x[j], acc[i][j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int j = 0; j < FT; ++j) {
            const uint32_t t = t0 + wt + 16 * j + m;
            const float sx = a.xscale[min(t, a.T - 1u)];
#pragma unroll
            for (int i = 0; i < FN; i += GATED ? 2 : 1) {
                const uint32_t n = n0 + (GATED ? (wn + 16 * i) / 2 : wn + 16 * i) + 4 * kg;
                vx_i8_finish4<GATED>(a, t, n, sx, acc[i][j], GATED ? acc[i + 1][j] : i4v{}, vx_i8_scales4(a.wscale[0], n, a.N),
                                     GATED ? vx_i8_scales4(a.wscale[1], n, a.N) : f4v{});
            }
        }
    }
};
#define VX_I8_TILE(name, MT, MN, WT, WN, GATED)                                                  \
    extern "C" __global__ __launch_bounds__(64 * WT * WN) void name(vx_i8_args a) {              \
        vx_i8_tile<MT, MN, WT, WN, GATED>::run(a);                                               \
    }
VX_I8_TILE(vx_i8_tile256, 256, 256, 2, 4, false)
VX_I8_TILE(vx_i8_tile256_gated, 256, 256, 2, 4, true)
VX_I8_TILE(vx_i8_tile128, 128, 128, 2, 2, false)
VX_I8_TILE(vx_i8_tile128_gated, 128, 128, 2, 2, true)
