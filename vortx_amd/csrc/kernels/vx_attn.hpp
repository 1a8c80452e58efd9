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
    int start, n, len;  // first query token, query tokens, keys in reach
    int tail;           // position of the first query (negative where there are more queries than keys)
    uint32_t rows;      // query rows that are computed
};
__device__ __forceinline__ vx_attn_seq vx_attn_sequence(const vx_attn_args& a, uint32_t s) {
    vx_attn_seq q;
    const int T = (int)a.tokens;
    q.start = min(max(a.starts[s], 0), T);
    q.n = min(max(a.starts[s + 1], q.start), T) - q.start;
    const int all = max(a.lens[s], 0);  // (positions go by it, whatever is in reach)
    q.len = min(all, (int)min(a.max_len, a.table_cols << a.c.page_shift));
    q.tail = all - q.n;
    q.rows = min((uint32_t)q.n, a.max_queries) * a.group;
    return q;
}

// What a query row sees: the keys of [lo, hi), and for a tree of drafts those
// of [tail, len) whose bit is set.
struct vx_attn_row {
    int pos, lo, hi;
    float slope;  // times log2 e
};

// Token and query head of a unit's row r (below q.rows). Computed again where
// they are needed: kept over the keys, they are registers that the sums want.
__device__ __forceinline__ void vx_attn_token(const vx_attn_args& a, const vx_attn_seq& q, uint32_t kvh, uint32_t r, uint32_t& token, uint32_t& head) {
    asm volatile("" : "+v"(r));
    const uint32_t j = r / a.group;
    token = (uint32_t)q.start + j;
    head = kvh * a.group + (r - j * a.group);
}

// Number of a sequence's `drafts` that a token's row of the tree sees.
__device__ __forceinline__ int vx_tree_count(const vx_attn_args& a, int token, int drafts) {
    const uint32_t* w = a.tree + (uint64_t)token * a.tree_stride;
    int n = 0;
    for (uint32_t i = 0; i < a.tree_words && drafts > 0; ++i, drafts -= 32)
        n += __builtin_popcount(drafts < 32 ? w[i] & ((1u << drafts) - 1u) : w[i]);
    return n;
}

__device__ __forceinline__ vx_attn_row vx_attn_row_of(const vx_attn_args& a, const vx_attn_seq& q, uint32_t s, uint32_t kvh, uint32_t r) {
    vx_attn_row w;
    if (r >= q.rows) {
        w.pos = w.lo = w.hi = 0;
        w.slope = 0.f;
        return w;
    }
    uint32_t token, head;
    vx_attn_token(a, q, kvh, r, token, head);
    w.lo = 0;
    if (a.tree) {
        w.pos = q.tail + vx_tree_count(a, (int)token, q.n) - 1;
        w.hi = min(max(q.tail, 0), q.len);
    } else {
        w.pos = q.tail + (int)token - q.start;
        w.hi = q.len;
        if (a.causal) w.hi = min(w.hi, max(w.pos + 1, a.prefix ? a.prefix[s] : 0));
    }
    if (a.first) w.lo = max(w.lo, a.first[token]);
    if (a.window) {
        w.lo = (int)max((int64_t)w.lo, (int64_t)w.pos - a.window + 1);
        w.hi = (int)min((int64_t)w.hi, (int64_t)w.pos + a.window);
    }
    w.hi = max(w.hi, w.lo);
    w.slope = a.slopes ? a.slopes[head] * VX_LOG2E : 0.f;
    return w;
}

// Which of the 32 keys from k0 on the unit's row r sees, a bit each: those of its
// interval before `tail`, and the drafts from there on by the tree's bits.
// at[i] becomes the position of key k0 + i where that is not k0 + i for all of
// them (slopes or a window over a tree; the wave's own 32 words of LDS).
__device__ __forceinline__ uint32_t vx_attn_sees(const vx_attn_args& a, const vx_attn_seq& q, const vx_attn_row& w, uint32_t kvh, uint32_t r, int tail, int k0, int* at) {
    auto from = [&](int key) { return key <= k0 ? 0xFFFFFFFFu : key - k0 > 31 ? 0u : 0xFFFFFFFFu << (key - k0); };  // keys >= key
    uint32_t see = from(w.lo) & ~from(min(w.hi, tail));
    if (a.tree && k0 + 32 > tail) {
        const int j0 = k0 - tail;  // first draft of the tile (above -32; drafts before key 0 have no key)
        uint32_t bits = 0;
        if (r < q.rows) {
            uint32_t token, head;
            vx_attn_token(a, q, kvh, r, token, head);
            const uint32_t* row = a.tree + (uint64_t)token * a.tree_stride;
            const int i = j0 >> 5, sh = j0 & 31;
            const uint32_t w0 = i >= 0 && (uint32_t)i < a.tree_words ? row[i] : 0u;
            const uint32_t w1 = (uint32_t)(i + 1) < a.tree_words ? row[i + 1] : 0u;
            bits = (uint32_t)(((uint64_t)w1 << 32 | w0) >> sh);
        }
        bits &= from(tail) & ~from(q.len);
        if (a.slopes || a.window) {
            const int lane = threadIdx.x & 31, key = k0 + lane;
            int p = key;
            if (key >= tail && key < q.len) p = q.tail + vx_tree_count(a, q.start + key - q.tail, q.n) - 1;
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
        int64_t sd = a.os[2];
        asm volatile("" : "+s"(sd));  // (else the addresses of all calls are kept over a kernel's units)
        op += d * sd;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i, op += sd) *op = t[i] * k;
    }
}

// Keys that the rows of row block rb (ROWS query rows) may see, by their
// positions alone, and how many steps of STEP keys they are: at least one where
// there is a row.
template <uint32_t ROWS, uint32_t STEP>
__device__ __forceinline__ uint32_t vx_attn_steps(const vx_attn_args& a, const vx_attn_seq& q, uint32_t s, uint32_t rb, int& lo) {
    const uint32_t r0 = rb * ROWS;
    lo = 0;
    if (r0 >= q.rows) return 0u;
    // (32 bits: lengths and windows are below 2^31 - 2^16, query tokens 2^30 at most)
    const int tail = q.tail;
    int p0 = tail - 1, p1 = q.len, from = 0, to = q.len;  // a tree's drafts are anywhere from there on
    if (!a.tree) {
        p0 = tail + (int)(r0 / a.group);
        p1 = tail + (int)((min(r0 + ROWS, q.rows) - 1) / a.group);
        if (a.causal) to = min(to, max(p1 + 1, a.prefix ? a.prefix[s] : 0));
        if (a.window && p1 < 0x7FFFFFFF - (int)a.window) to = min(to, p1 + (int)a.window);
    }
    if (a.window && p0 >= (int)a.window) from = p0 - (int)a.window + 1;
    lo = min(from, q.len) & ~31;
    return (uint32_t)max(1, (to - lo + (int)STEP - 1) / (int)STEP);
}

// Quotients of numbers that seldom need 64 bits.
__device__ __forceinline__ uint64_t vx_div(uint64_t a, uint64_t b) {
    return (a | b) >> 32 ? a / b : (uint64_t)((uint32_t)a / (uint32_t)b);
}

// The key steps of all units (row block, sequence, head) dealt out evenly, a
// run of them to each workgroup, whatever the lengths. Pair (s, rb) has c steps
// a head and its heads follow each other; a unit counts COST steps more, in
// front, for what it takes to begin and to end: without that the first row
// blocks of a causal prompt, many short units to a workgroup, took three times
// the others' time (8192 tokens, 8 heads over 2 of 128, 64-key steps: COST 0
// 548 us, 2 417, 4 413, 8 428). do_unit takes a unit's keys from..to (end: to its end). A
// unit that several workgroups share goes to partial sums:
// a workgroup's first unit is partial 2 w, its last, if another, 2 w + 1; info
// has a unit's first partial and their number, for the join.
template <uint32_t THREADS, uint32_t ROWS, uint32_t STEP, uint32_t COST, class Unit>
__device__ __forceinline__ void vx_attn_deal(const vx_attn_args& a, Unit do_unit) {
    __shared__ uint32_t sh_sum[THREADS / 64], sh_at[2];
    const uint32_t t = threadIdx.x, H = a.c.heads, RB = a.row_blocks, pairs = a.seqs * RB;
    const uint32_t per = (pairs + THREADS - 1) / THREADS;
    uint32_t mine = 0;
    for (uint32_t p = t * per; p < min((t + 1) * per, pairs); ++p) {
        int lo;
        const uint32_t s = p / RB;
        const uint32_t c = vx_attn_steps<ROWS, STEP>(a, vx_attn_sequence(a, s), s, p - s * RB, lo);
        mine += c ? c + COST : 0u;
    }
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(upto, o);
        if ((t & 63) >= (uint32_t)o) upto += v;
    }
    if ((t & 63) == 63) sh_sum[t >> 6] = upto;
    __syncthreads();
    uint32_t before = upto - mine, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < THREADS / 64; ++i) {
        if (i < t >> 6) before += sh_sum[i];
        all += sh_sum[i];
    }
    // workgroup w's run is [w total / G, (w + 1) total / G): step k is run (k G + G - 1) / total
    const uint64_t total = (uint64_t)all * H;
    const uint32_t G = (uint32_t)min((uint64_t)gridDim.x, total);  // (no run is empty)
    if (blockIdx.x >= G) return;
    uint64_t p = vx_div(blockIdx.x * total, G);
    const uint64_t end = vx_div((blockIdx.x + 1) * total, G);
    if (p >= end) return;
    auto run_of = [&](uint64_t k) { return vx_div(k * G + G - 1, total); };
    if (p >= (uint64_t)before * H && p < (uint64_t)(before + mine) * H) {
        uint32_t i = t * per, sum = before;
        for (;; ++i) {
            int lo;
            const uint32_t s = i / RB, c = vx_attn_steps<ROWS, STEP>(a, vx_attn_sequence(a, s), s, i - s * RB, lo);
            const uint32_t all_c = c ? c + COST : 0u;
            if (p < (uint64_t)(sum + all_c) * H) break;
            sum += all_c;
        }
        sh_at[0] = i;
        sh_at[1] = sum;
    }
    __syncthreads();
    uint32_t pair = __builtin_amdgcn_readfirstlane(sh_at[0]);
    uint64_t begin = (uint64_t)__builtin_amdgcn_readfirstlane(sh_at[1]) * H;  // first step of the pair
    bool first = true;
    while (p < end) {
        const uint32_t s = pair / RB, rb = pair - s * RB;
        const vx_attn_seq q = vx_attn_sequence(a, s);
        int klo;
        const uint32_t c = vx_attn_steps<ROWS, STEP>(a, q, s, rb, klo);
        if (!c || p >= begin + (uint64_t)(c + COST) * H) {
            begin += c ? (uint64_t)(c + COST) * H : 0u;
            ++pair;
            continue;
        }
        const uint32_t kvh = (uint32_t)vx_div(p - begin, c + COST);
        const uint64_t k0 = begin + (uint64_t)kvh * (c + COST) + COST;  // the unit's first step of keys
        if (k0 >= end) break;
        const uint32_t c0 = p > k0 ? (uint32_t)(p - k0) : 0u, c1 = (uint32_t)min((uint64_t)c, end - k0);
        const uint32_t parts = (uint32_t)(run_of(k0 + c - 1) - run_of(k0)) + 1;
        const uint32_t part = 2 * blockIdx.x + (first ? 0u : 1u);
        if (c0 == 0 && t == 0) *(u2*)(a.info + 2 * (pair * H + kvh)) = u2{part, parts};
        do_unit(q, s, kvh, rb, parts == 1, part, klo + (int)(c0 * STEP), klo + (int)(c1 * STEP), c1 == c);
        p = k0 + c1;
        first = false;
    }
}
