// vx_attn.hpp — what the attention kernels share: a query row's bounds and
// masks, scores and their cap, and the order of the workgroups.
#pragma once
#include "vx_dpp.hpp"
#include "vx_kv.hpp"

// What is the same for a whole wave and no kernel writes comes by scalar loads.
typedef const __attribute__((address_space(4))) int32_t* vx_scalar_i32;

constexpr float VX_LOG2E = 1.44269504088896340736f;

// tanh to about two units in the last place: below 0.65 a minimax polynomial,
// above 1 - 2 / (1 + e^2|t|), which would cancel below.
constexpr float VX_TANH[5] = {-0.3333323001861572f, 0.1333041489124298f, -0.05366527661681175f, 0.020415181294083595f, -0.005468255840241909f};
__device__ __forceinline__ float vx_tanh_small(float t) {
    const float z = t * t;
    float p = __builtin_fmaf(z, VX_TANH[4], VX_TANH[3]);
    p = __builtin_fmaf(z, p, VX_TANH[2]);
    p = __builtin_fmaf(z, p, VX_TANH[1]);
    p = __builtin_fmaf(z, p, VX_TANH[0]);
    return __builtin_fmaf(z * t, p, t);
}
__device__ __forceinline__ float vx_tanh(float t) {
    const float a = fabsf(t), e = __builtin_amdgcn_exp2f(a * (2.f * VX_LOG2E));
    const float q = __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + e), 1.f);
    return a < 0.65f ? vx_tanh_small(t) : __builtin_copysignf(q, t);  // (NaN: q, which is NaN)
}

// Maximum / sum over the four 16-lane rows, in every lane.
__device__ __forceinline__ float vx_max_rows4(float v) {
    uint32_t a = __builtin_bit_cast(uint32_t, v), b = a;
    vx_swap16(a, b);
    v = fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    a = b = __builtin_bit_cast(uint32_t, v);
    vx_swap32(a, b);
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// A sequence of the batch: queries, keys and where they lie.
struct vx_attn_seq {
    int start, n, len;  // first query token, query tokens, keys
    uint32_t rows;      // query rows that are computed
};
__device__ __forceinline__ vx_attn_seq vx_attn_sequence(const vx_attn_args& a, uint32_t s) {
    vx_attn_seq q;
    const int T = (int)a.tokens;
    q.start = min(max(a.starts[s], 0), T);
    q.n = min(max(a.starts[s + 1], q.start), T) - q.start;
    q.len = min(max(a.lens[s], 0), (int)min(a.max_len, a.table_cols << a.c.page_shift));
    q.rows = min((uint32_t)q.n, a.max_queries) * a.group;
    return q;
}

// What a query row sees: the keys of [lo, hi), and for a tree of drafts those
// of [tail, len) whose bit is set.
struct vx_attn_row {
    bool valid;
    int token, head;  // of q and out
    int pos, lo, hi;
    float slope;      // times log2 e
};

// Number of drafts that a token's row of the tree sees.
__device__ __forceinline__ int vx_tree_count(const vx_attn_args& a, int token) {
    const uint32_t* w = a.tree + (uint64_t)token * a.tree_stride;
    int n = 0;
    for (uint32_t i = 0; i < a.tree_words; ++i) n += __builtin_popcount(w[i]);
    return n;
}

__device__ __forceinline__ vx_attn_row vx_attn_row_of(const vx_attn_args& a, const vx_attn_seq& q, uint32_t s, uint32_t kvh, uint32_t r) {
    vx_attn_row w;
    w.valid = r < q.rows;
    const uint32_t j = w.valid ? r / a.group : 0u;
    w.token = q.start + (int)j;
    w.head = (int)(kvh * a.group + (w.valid ? r - j * a.group : 0u));
    const int tail = q.len - q.n;
    if (!w.valid) {
        w.pos = w.lo = w.hi = 0;
        w.slope = 0.f;
        return w;
    }
    w.lo = 0;
    if (a.tree) {
        w.pos = tail + vx_tree_count(a, w.token) - 1;
        w.hi = max(tail, 0);
    } else {
        w.pos = tail + (int)j;
        w.hi = q.len;
        if (a.causal) w.hi = min(w.hi, max(w.pos + 1, a.prefix ? a.prefix[s] : 0));
    }
    if (a.first) w.lo = max(w.lo, a.first[w.token]);
    if (a.window) {
        w.lo = (int)max((int64_t)w.lo, (int64_t)w.pos - a.window + 1);
        w.hi = (int)min((int64_t)w.hi, (int64_t)w.pos + a.window);
    }
    w.hi = max(w.hi, w.lo);
    w.slope = a.slopes ? a.slopes[w.head] * VX_LOG2E : 0.f;
    return w;
}

// Which of the 32 keys from k0 on a row sees, a bit each: those of its
// interval before `tail`, and the drafts from there on by the tree's bits.
// at[i] becomes the position of key k0 + i where that is not k0 + i for all of
// them (slopes or a window over a tree; the wave's own 32 words of LDS).
__device__ __forceinline__ uint32_t vx_attn_sees(const vx_attn_args& a, const vx_attn_seq& q, const vx_attn_row& w, int tail, int k0, int* at) {
    auto from = [&](int key) { return key <= k0 ? 0xFFFFFFFFu : key - k0 > 31 ? 0u : 0xFFFFFFFFu << (key - k0); };  // keys >= key
    uint32_t see = from(w.lo) & ~from(min(w.hi, tail));
    if (a.tree && k0 + 32 > tail) {
        const int j0 = k0 - tail;  // first draft of the tile (above -32)
        uint32_t bits = 0;
        if (w.valid) {
            const uint32_t* row = a.tree + (uint64_t)w.token * a.tree_stride;
            const int i = j0 >> 5, sh = j0 & 31;
            const uint32_t w0 = i >= 0 && (uint32_t)i < a.tree_words ? row[i] : 0u;
            const uint32_t w1 = (uint32_t)(i + 1) < a.tree_words ? row[i + 1] : 0u;
            bits = (uint32_t)(((uint64_t)w1 << 32 | w0) >> sh);
        }
        bits &= from(tail) & ~from(q.len);
        if (a.slopes || a.window) {
            const int lane = threadIdx.x & 31, key = k0 + lane;
            int p = key;
            if (key >= tail && key < q.len) p = q.len - q.n + vx_tree_count(a, q.start + key - (q.len - q.n)) - 1;
            at[lane] = p;  // (both halves of the wave the same)
            __builtin_amdgcn_wave_barrier();
            if (a.window) {
#pragma unroll 1
                for (int i = 0; i < 32; ++i)
                    if ((uint32_t)abs(w.pos - at[i]) >= a.window) bits &= ~(1u << i);
            }
        }
        see |= bits;
    }
    return see;
}

// Four dims of a row's result: its sums over its weights' sum. Nothing seen: zeros.
__device__ __forceinline__ void vx_attn_put(const vx_attn_args& a, uint32_t token, uint32_t head, uint32_t d, f4 t, float l) {
    const float k = l == 0.f ? 0.f : 1.f / l;
    float* op = a.out + (int64_t)token * a.os[0] + (int64_t)head * a.os[1];
    if (a.vec) {
        *(f4*)(op + d) = t * k;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) op[(int64_t)(d + i) * a.os[2]] = t[i] * k;
    }
}
