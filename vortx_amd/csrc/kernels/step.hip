// step.hip — what a step of a batch needs before its attention: the pages that
// sequences give back and take, the slots of their new tokens, and queries and
// keys normed and rotated.
#include "vx_kv_rows.hpp"
#include "vx_rotate.hpp"

// The first workgroups have the queries, the others the keys. _s: rows of any strides.
#define VX_ROTATE(L, S, VEC)                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void vx_rotate_l##L##S(vx_rotate_args a) {                      \
        __shared__ double2 angles[VX_ANGLE_PLACES];                                                              \
        const uint32_t keys = blockIdx.x >= a.part[0].blocks;                                                    \
        vx_rotate_rows<L, VEC>(a, a.part[keys], keys ? blockIdx.x - a.part[0].blocks : blockIdx.x, angles);      \
    }
VX_ROTATE(16, , true)
VX_ROTATE(32, , true)
VX_ROTATE(64, , true)
VX_ROTATE(16, _s, false)
VX_ROTATE(32, _s, false)
VX_ROTATE(64, _s, false)

// Keys and values written token by token, queries rotated by the first workgroups
// beside them; and of many tokens keys and values by fours, by themselves.
#define VX_ROTATE_KV(d, types, NB, LANES, KB, VB, S, VEC)                                                                      \
    extern "C" __global__ __launch_bounds__(256) void vx_rotate_kv_d##d##S##_##types(vx_kv_rotated_args a) {                   \
        __shared__ double2 angles[VX_ANGLE_PLACES];                                                                            \
        const uint32_t queries = a.t.part[0].blocks;                                                                           \
        if (blockIdx.x < queries) vx_rotate_rows<LANES, VEC>(a.t, a.t.part[0], blockIdx.x, angles);                            \
        else vx_kv_write_turned<NB, KB, VB, LANES, VEC>(a.r, a.t, blockIdx.x - queries, angles);                               \
    }
#define VX_ROTATE_KV4(d, types, NB, LANES, KB, VB)                                                                             \
    extern "C" __global__ __launch_bounds__(256) void vx_rotate_kv4_d##d##_##types(vx_kv_rotated_args a) {                     \
        __shared__ double2 angles[vx_kv_staged<NB>::PLACES];                                                                   \
        __shared__ __align__(16) float rows[vx_kv_staged<NB>::FLOATS];                                                         \
        vx_kv_write_staged<NB, KB, VB, LANES>(a.r, a.t, blockIdx.x, angles, rows);                                             \
    }
#define VX_ROTATE_KVS(d, NB, LANES)                                                                                            \
    VX_ROTATE_KV(d, k8v8, NB, LANES, 8, 8, , true) VX_ROTATE_KV(d, k8v4, NB, LANES, 8, 4, , true)                              \
    VX_ROTATE_KV(d, k4v8, NB, LANES, 4, 8, , true) VX_ROTATE_KV(d, k4v4, NB, LANES, 4, 4, , true)                              \
    VX_ROTATE_KV(d, k8v8, NB, LANES, 8, 8, _s, false) VX_ROTATE_KV(d, k8v4, NB, LANES, 8, 4, _s, false)                        \
    VX_ROTATE_KV(d, k4v8, NB, LANES, 4, 8, _s, false) VX_ROTATE_KV(d, k4v4, NB, LANES, 4, 4, _s, false)                        \
    VX_ROTATE_KV4(d, k8v8, NB, LANES, 8, 8) VX_ROTATE_KV4(d, k8v4, NB, LANES, 8, 4)                                            \
    VX_ROTATE_KV4(d, k4v8, NB, LANES, 4, 8) VX_ROTATE_KV4(d, k4v4, NB, LANES, 4, 4)
VX_ROTATE_KVS(64, 2, 16)
VX_ROTATE_KVS(96, 3, 32)
VX_ROTATE_KVS(128, 4, 32)
VX_ROTATE_KVS(256, 8, 64)

// Sums that stop at 2^31 - 1 (of numbers up to it).
__device__ __forceinline__ uint32_t vx_add_sat(uint32_t a, uint32_t b) { return min(a + b, 0x7FFFFFFFu); }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t vx_scan_step(uint32_t v) {
    return vx_add_sat(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}
// Sums over the lanes up to this one: rows of 16 by shifts, then the rows before.
__device__ __forceinline__ uint32_t vx_wave_scan(uint32_t v) {
    v = vx_scan_step<0x111, 0xF>(v);
    v = vx_scan_step<0x112, 0xF>(v);
    v = vx_scan_step<0x114, 0xF>(v);
    v = vx_scan_step<0x118, 0xF>(v);
    v = vx_scan_step<0x142, 0xA>(v);
    return vx_scan_step<0x143, 0xC>(v);
}

// Exclusive sums over the workgroup's threads of N numbers each, and their totals.
template <int N>
struct vx_sums {
    uint32_t before[N], total[N];
    __device__ __forceinline__ vx_sums(const uint32_t (&v)[N], uint32_t (*lds)[16], uint32_t waves) {
        const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        uint32_t s[N];
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = vx_wave_scan(v[i]);
        __syncthreads();  // (what lds held is read)
        if (lane == 63)
#pragma unroll
            for (int i = 0; i < N; ++i) lds[i][wave] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint32_t base = 0, all = 0;
            for (uint32_t w = 0; w < waves; ++w) {
                if (w == wave) base = all;
                all = vx_add_sat(all, lds[i][w]);
            }
            uint32_t own = (uint32_t)__shfl_up((int)s[i], 1);
            if (lane == 0) own = 0;
            before[i] = vx_add_sat(base, own);
            total[i] = all;
        }
    }
};

// Last index of first[0..n) whose entry is at most i (first[0] <= i).
__device__ __forceinline__ uint32_t vx_owner(const uint32_t* first, uint32_t n, uint32_t i) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (first[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Items 0 .. total shared out over n threads, a run of neighbours each; four are read
// before any of them is written. k: the item's sequence, looked up once (`first`: of
// each sequence) and then moved on by `read`.
template <class Read, class Write>
__device__ __forceinline__ void vx_shared_out(uint32_t total, uint32_t n, Read read, Write write, const uint32_t* first) {
    const uint32_t each = (total + n - 1) / n, begin = min(total, each * threadIdx.x), end = min(total, begin + each);
    if (begin >= end) return;
    uint32_t k = vx_owner(first, n, begin);
#pragma unroll 1
    for (uint32_t i = begin; i < end; i += 4) {
        int32_t v[4];
        uint32_t of[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            if (i + j < end) {
                v[j] = read(i + j, k);
                of[j] = k;
            }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            if (i + j < end) write(i + j, of[j], v[j]);
    }
}

// A sequence before and after the step.
struct vx_held {
    uint32_t have, want, old_pages, new_pages;  // want: have where it is to stay
    uint32_t gives, needs, tokens;
    bool fits;  // its table row holds what it wants (otherwise it takes no part)
    __device__ __forceinline__ vx_held(const vx_pages_args& a, uint32_t s) : have(0), want(0), old_pages(0), new_pages(0), tokens(0), fits(true) {
        if (s < a.seqs) {
            const uint64_t most = min((uint64_t)a.table_cols << a.page_shift, (uint64_t)0x7FFFFFFF);
            const int32_t len = a.lens[s], w = a.want[s];
            have = (uint32_t)min((uint64_t)max(len, 0), most);
            want = w < 0 ? have : (uint32_t)w;
            tokens = want > have ? want - have : 0u;
            fits = want <= most;
            const uint32_t round = (1u << a.page_shift) - 1u;
            old_pages = (have + round) >> a.page_shift;
            new_pages = fits ? (want + round) >> a.page_shift : old_pages;
        }
        gives = old_pages > new_pages ? old_pages - new_pages : 0u;
        needs = new_pages > old_pages ? new_pages - old_pages : 0u;
    }
};

// The whole step in one workgroup of a.threads, as many sequences at a time. It is
// bound by a chain: lengths, their sums, stack or table, what follows from it (32
// sequences, a token each, 4.2 us traced; 200 with 320000 new tokens 12.1, and 5.0 for
// the slots after it). It puts what sequences give back on the stack before any takes
// from it. (Sums alone would do: page i that is taken is page i that is given back, as
// long as there are such, and then comes the stack as it was. Many workgroups could
// share out a long step so.) A thread moves the pages and tokens of its own sequence
// where all have few, otherwise all threads share them out.
constexpr uint32_t VX_OWN_PAGES = 4, VX_OWN_TOKENS = 8;
extern "C" __global__ __launch_bounds__(1024) void vx_pages_resize(vx_pages_args a) {
    __shared__ uint32_t part[4][16];
    __shared__ uint32_t first[1024], row[1024], first_token[1024], state[1024];  // of the sequences at hand
    const uint32_t tid = threadIdx.x, n = a.threads, waves = n / 64;
    const uint32_t count = (uint32_t)max(0, min(*a.free_count, (int32_t)a.pages));
    const vx_held mine(a, tid);
    auto many = [](const vx_held& h) -> uint32_t { return h.gives > VX_OWN_PAGES || h.needs > VX_OWN_PAGES || h.tokens > VX_OWN_TOKENS; };
    // what all sequences give back, and all other sums of the first ones
    const uint32_t v0[4] = {mine.gives, mine.needs, mine.tokens, many(mine)};
    const vx_sums<4> sums0(v0, part, waves);
    uint32_t given = sums0.total[0];
    for (uint32_t s0 = n; s0 < a.seqs; s0 += n) {
        const uint32_t v[1] = {vx_held(a, s0 + tid).gives};
        given += vx_sums<1>(v, part, waves).total[0];
    }
    for (uint32_t s0 = 0, done = 0; given && s0 < a.seqs; s0 += n) {
        const vx_held h(a, s0 + tid);
        const uint32_t v[2] = {h.gives, many(h)};
        const vx_sums<2> sums(v, part, waves);
        const uint32_t top = count + given - 1u - done;
        if (!sums.total[1]) {
            for (uint32_t i = 0; i < h.gives; ++i) {
                const uint32_t at = top - (sums.before[0] + i);
                if (at < a.pages) a.free_pages[at] = a.table[(uint64_t)(s0 + tid) * a.table_stride + h.new_pages + i];
            }
        } else {
            first[tid] = sums.before[0];
            row[tid] = h.new_pages;
            __syncthreads();
            vx_shared_out(sums.total[0], n, [&](uint32_t i, uint32_t& k) {
                while (k + 1 < n && first[k + 1] <= i) ++k;
                return a.table[(uint64_t)(s0 + k) * a.table_stride + row[k] + (i - first[k])];
            }, [&](uint32_t i, uint32_t, int32_t page) {
                if (top - i < a.pages) a.free_pages[top - i] = page;
            }, first);
        }
        done += sums.total[0];
    }
    if (given) __syncthreads();
    const uint32_t room = min(count + given, a.pages);
    uint32_t asked = 0, taken = 0, token = 0;  // by the sequences before those at hand
    for (uint32_t s0 = 0; s0 < a.seqs; s0 += n) {
        const uint32_t s = s0 + tid;
        const vx_held h(a, s);
        const uint32_t v[4] = {0u, h.needs, h.tokens, many(h)};
        const vx_sums<4> sums = s0 ? vx_sums<4>(v, part, waves) : sums0;
        // (one that finds its pages has found them for all before it: those that are served take what is on top)
        const uint32_t lo = asked + sums.before[1], t0 = vx_add_sat(token, sums.before[2]);
        const bool served = h.fits && (h.needs == 0 || lo + h.needs <= room);
        if (s < a.seqs) {
            a.lens[s] = (int32_t)(served ? h.want : h.have);
            a.starts[s] = (int32_t)t0;
        }
        int32_t* table = a.table + (uint64_t)s * a.table_stride;
        if (!sums.total[3]) {
            for (uint32_t i = 0; served && i < h.needs; ++i) table[h.old_pages + i] = a.free_pages[room - 1u - (lo + i)];
            for (uint32_t i = 0; a.here && i < h.tokens && t0 + i < a.tokens; ++i) {
                const uint32_t p = h.have + i, page = p >> a.page_shift;
                int32_t slot = -1;
                if (served) {
                    const uint32_t id = (uint32_t)(page < h.old_pages ? table[page] : a.free_pages[room - 1u - (lo + page - h.old_pages)]);
                    slot = (int32_t)((id << a.page_shift) + (p & ((1u << a.page_shift) - 1u)));
                }
                a.slots[t0 + i] = slot;
                a.positions[t0 + i] = (int32_t)p;
            }
        } else {
            __syncthreads();  // (the arrays are free)
            first[tid] = sums.before[1];
            row[tid] = h.old_pages;
            first_token[tid] = sums.before[2];
            state[tid] = h.have | (served ? 0u : 0x80000000u);
            __syncthreads();
            vx_shared_out(min(sums.total[1], room - min(room, asked)), n, [&](uint32_t i, uint32_t& k) {
                while (k + 1 < n && first[k + 1] <= i) ++k;
                return a.free_pages[room - 1u - (asked + i)];
            }, [&](uint32_t i, uint32_t k, int32_t page) {
                if (!(state[k] >> 31)) a.table[(uint64_t)(s0 + k) * a.table_stride + row[k] + (i - first[k])] = page;
            }, first);
            for (uint32_t i = tid; a.here && i < sums.total[2] && (uint64_t)token + i < a.tokens; i += n) {
                const uint32_t k = vx_owner(first_token, n, i);
                const uint32_t p = (state[k] & 0x7FFFFFFFu) + (i - first_token[k]), page = p >> a.page_shift;
                int32_t slot = -1;
                if (!(state[k] >> 31)) {
                    const uint32_t id = (uint32_t)(page < row[k] ? a.table[(uint64_t)(s0 + k) * a.table_stride + page]
                                                                 : a.free_pages[room - 1u - (asked + first[k] + page - row[k])]);
                    slot = (int32_t)((id << a.page_shift) + (p & ((1u << a.page_shift) - 1u)));
                }
                a.slots[token + i] = slot;
                a.positions[token + i] = (int32_t)p;
            }
        }
        // what is taken ends with the last one that is served
        uint32_t top = h.needs && served ? lo + h.needs : 0u;
#pragma unroll
        for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        __syncthreads();
        if ((tid & 63) == 0) part[0][tid >> 6] = top;
        __syncthreads();
        for (uint32_t w = 0; w < waves; ++w) taken = max(taken, part[0][w]);
        asked = vx_add_sat(asked, sums.total[1]);
        token = vx_add_sat(token, sums.total[2]);
    }
    if (a.here)
        for (uint64_t i = (uint64_t)token + tid; i < a.tokens; i += n) {
            a.slots[i] = -1;
            a.positions[i] = 0;
        }
    if (tid == 0) {
        a.starts[a.seqs] = (int32_t)token;
        *a.free_count = (int32_t)(room - taken);
    }
}

// Slots and positions of many tokens, after vx_pages_resize: 1024 a workgroup, four a
// thread. The starts, or every few of them, are searched in LDS.
extern "C" __global__ __launch_bounds__(256) void vx_pages_slots(vx_pages_args a) {
    __shared__ uint32_t some[1024];
    const uint32_t every = (a.seqs + 1023) / 1024, there = every ? (a.seqs + every - 1) / every : 0;
    for (uint32_t i = threadIdx.x; i < there; i += 256) some[i] = (uint32_t)a.starts[i * every];
    __syncthreads();
    const uint32_t end = (uint32_t)a.starts[a.seqs];
    const uint64_t at = (uint64_t)blockIdx.x * 1024 + 4 * threadIdx.x;
    if (at >= a.tokens) return;
    int32_t slot[4], pos[4];
    uint32_t s = 0, first = 0, next = 0, base = 0;  // the sequence at hand: tokens first to next, the first at position base
    bool served = false;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t i = (uint32_t)at + j;
        slot[j] = -1;
        pos[j] = 0;
        if (i >= end) continue;
        if (i >= next) {
            const uint32_t k = vx_owner(some, there, i) * every;
            s = k + vx_owner((const uint32_t*)a.starts + k, min(every, a.seqs - k), i);
            first = (uint32_t)a.starts[s];
            next = (uint32_t)a.starts[s + 1];
            const uint32_t len = (uint32_t)a.lens[s];
            served = len == (uint32_t)a.want[s];  // (it has new tokens, so want was more than its length)
            base = served ? len - (next - first) : len;
        }
        const uint32_t p = base + (i - first);
        pos[j] = (int32_t)p;
        if (served) {
            const uint32_t id = (uint32_t)a.table[(uint64_t)s * a.table_stride + (p >> a.page_shift)];
            slot[j] = (int32_t)((id << a.page_shift) + (p & ((1u << a.page_shift) - 1u)));
        }
    }
    if (a.vec && at + 4 <= a.tokens) {
        *(int4*)(a.slots + at) = int4{slot[0], slot[1], slot[2], slot[3]};
        *(int4*)(a.positions + at) = int4{pos[0], pos[1], pos[2], pos[3]};
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
        if (at + j < a.tokens) {
            a.slots[at + j] = slot[j];
            a.positions[at + j] = pos[j];
        }
}
