// step.hip — what a step of a batch needs before its attention: the pages that
// sequences give back and take, the slots of their new tokens, and queries and
// keys normed and rotated.
#include "vx_kv_rows.hpp"
#include "vx_rotate.hpp"

#define VX_ROTATE(L) \
    extern "C" __global__ __launch_bounds__(256) void vx_rotate_l##L(vx_rotate_args a) { vx_rotate_rows<L>(a, blockIdx.x); }
VX_ROTATE(16)
VX_ROTATE(32)
VX_ROTATE(64)

// Queries rotated by the first workgroups, keys and values written by the others.
#define VX_ROTATE_KV(d, types, NB, LANES, KB, VB)                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void vx_rotate_kv_d##d##_##types(vx_kv_rotated_args a) {                          \
        if (blockIdx.x < a.t.blocks) vx_rotate_rows<LANES>(a.t, blockIdx.x);                                                       \
        else vx_kv_write_rows<NB, KB, VB>(a.r, vx_kv_turned_keys<LANES>{a.t}, blockIdx.x - a.t.blocks, gridDim.x - a.t.blocks);    \
    }
#define VX_ROTATE_KVS(d, NB, LANES)                                                                                                \
    VX_ROTATE_KV(d, k8v8, NB, LANES, 8, 8) VX_ROTATE_KV(d, k8v4, NB, LANES, 8, 4)                                                  \
    VX_ROTATE_KV(d, k4v8, NB, LANES, 4, 8) VX_ROTATE_KV(d, k4v4, NB, LANES, 4, 4)
VX_ROTATE_KVS(64, 2, 16)
VX_ROTATE_KVS(96, 3, 32)
VX_ROTATE_KVS(128, 4, 32)
VX_ROTATE_KVS(256, 8, 64)

// Sums that stop at 2^31 - 1 (of numbers up to it).
__device__ __forceinline__ uint32_t vx_add_sat(uint32_t a, uint32_t b) { return min(a + b, 0x7FFFFFFFu); }

// Exclusive sums over the 1024 threads of three numbers each, and their totals.
struct vx_sums3 {
    uint32_t before[3], total[3];
    __device__ __forceinline__ vx_sums3(const uint32_t (&v)[3], uint32_t (*lds)[17]) {
        uint32_t s[3] = {v[0], v[1], v[2]};
        const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (uint32_t o = 1; o < 64; o <<= 1)
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const uint32_t u = (uint32_t)__shfl_up((int)s[i], o);
                if (lane >= o) s[i] = vx_add_sat(s[i], u);
            }
        __syncthreads();  // (what lds held is read)
        if (lane == 63)
#pragma unroll
            for (int i = 0; i < 3; ++i) lds[i][wave] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            uint32_t w = lane < 16 ? lds[i][lane] : 0;
#pragma unroll
            for (uint32_t o = 1; o < 16; o <<= 1) {
                const uint32_t u = (uint32_t)__shfl_up((int)w, o);
                if (lane >= o) w = vx_add_sat(w, u);
            }
            total[i] = (uint32_t)__shfl((int)w, 15);
            const uint32_t base = wave ? (uint32_t)__shfl((int)w, (int)wave - 1) : 0u;
            uint32_t own = (uint32_t)__shfl_up((int)s[i], 1);
            if (lane == 0) own = 0;
            before[i] = vx_add_sat(base, own);
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

// A sequence before and after the step.
struct vx_held {
    uint32_t have, want, old_pages, new_pages;  // want: have where it is to stay, or cannot be served
    uint32_t tokens;
    bool fits;  // its table row holds what it wants
    __device__ __forceinline__ vx_held(const vx_pages_args& a, uint32_t s) : have(0), want(0), old_pages(0), new_pages(0), tokens(0), fits(true) {
        if (s >= a.seqs) return;
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
};

// The whole step in one workgroup, 1024 sequences at a time (bound by the chain
// of its loads: lengths, stack, table). What sequences give back has to be on the
// stack before any takes from it.
extern "C" __global__ __launch_bounds__(1024) void vx_pages_resize(vx_pages_args a) {
    __shared__ uint32_t part[3][17];
    __shared__ uint32_t first[1024], row[1024];  // of the chunk's sequences: first item, first table column
    const uint32_t tid = threadIdx.x;
    const uint32_t count = (uint32_t)max(0, min(*a.free_count, (int32_t)a.pages));
    // given back, in all
    uint32_t given = 0;
    for (uint32_t s0 = 0; s0 < a.seqs; s0 += 1024) {
        const vx_held h(a, s0 + tid);
        const uint32_t v[3] = {h.old_pages > h.new_pages ? h.old_pages - h.new_pages : 0u, 0u, 0u};
        const vx_sums3 sums(v, part);
        given += sums.total[0];
    }
    if (given) {
        uint32_t done = 0;
        for (uint32_t s0 = 0; s0 < a.seqs; s0 += 1024) {
            const vx_held h(a, s0 + tid);
            const uint32_t v[3] = {h.old_pages > h.new_pages ? h.old_pages - h.new_pages : 0u, 0u, 0u};
            const vx_sums3 sums(v, part);
            first[tid] = sums.before[0];
            row[tid] = h.new_pages;
            __syncthreads();
            for (uint32_t i = tid; i < sums.total[0]; i += 1024) {
                const uint32_t k = vx_owner(first, 1024, i);
                const uint32_t at = count + given - 1u - (done + i);
                if (at < a.pages) a.free_pages[at] = a.table[(uint64_t)(s0 + k) * a.table_stride + row[k] + (i - first[k])];
            }
            done += sums.total[0];
            __syncthreads();
        }
    }
    // taken, and the tokens
    const uint32_t room = min(count + given, a.pages);
    uint32_t asked = 0, taken = 0, token = 0;
    for (uint32_t s0 = 0; s0 < a.seqs; s0 += 1024) {
        const uint32_t s = s0 + tid;
        const vx_held h(a, s);
        const uint32_t need = h.new_pages > h.old_pages ? h.new_pages - h.old_pages : 0u;
        const uint32_t v[3] = {need, h.tokens, 0u};
        const vx_sums3 sums(v, part);
        const uint32_t lo = asked + sums.before[0];
        const bool served = h.fits && (need == 0 || lo + need <= room);
        first[tid] = sums.before[0];
        row[tid] = h.old_pages;
        if (s < a.seqs) {
            a.lens[s] = (int32_t)(served ? h.want : h.have);
            a.starts[s] = (int32_t)vx_add_sat(token, sums.before[1]);
        }
        // (those that are served come before all that are not: what they take is what fits)
        const uint32_t mine = need && served ? lo + need : 0u;
        __syncthreads();
        for (uint32_t i = tid; i < sums.total[0] && asked + i < room; i += 1024) {
            const uint32_t k = vx_owner(first, 1024, i);
            const uint32_t end = k + 1 < 1024 ? first[k + 1] : sums.total[0];
            if (asked + end > room) continue;
            a.table[(uint64_t)(s0 + k) * a.table_stride + row[k] + (i - first[k])] = a.free_pages[room - 1u - (asked + i)];
        }
        // the largest end of one that is served
        uint32_t top = mine;
#pragma unroll
        for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        __syncthreads();
        if ((tid & 63) == 0) part[0][tid >> 6] = top;
        __syncthreads();
        for (int i = 0; i < 16; ++i) taken = max(taken, part[0][i]);
        if (a.here) {
            first[tid] = sums.before[1];
            row[tid] = served ? h.have : h.have | 0x80000000u;
            __syncthreads();
            for (uint32_t i = tid; i < sums.total[1] && (uint64_t)token + i < a.tokens; i += 1024) {
                const uint32_t k = vx_owner(first, 1024, i);
                const uint32_t p = (row[k] & 0x7FFFFFFFu) + (i - first[k]);
                int32_t slot = -1;
                if (!(row[k] >> 31)) {
                    const uint32_t page = (uint32_t)a.table[(uint64_t)(s0 + k) * a.table_stride + (p >> a.page_shift)];
                    slot = (int32_t)((page << a.page_shift) + (p & ((1u << a.page_shift) - 1u)));
                }
                a.slots[token + i] = slot;
                a.positions[token + i] = (int32_t)p;
            }
            __syncthreads();
        }
        asked = vx_add_sat(asked, sums.total[0]);
        token = vx_add_sat(token, sums.total[1]);
    }
    if (a.here)
        for (uint64_t i = (uint64_t)token + tid; i < a.tokens; i += 1024) {
            a.slots[i] = -1;
            a.positions[i] = 0;
        }
    if (tid == 0) {
        a.starts[a.seqs] = (int32_t)token;
        *a.free_count = (int32_t)(room - taken);
    }
}

// Slots and positions of many tokens, after vx_pages_resize: 1024 consecutive ones a workgroup.
extern "C" __global__ __launch_bounds__(256) void vx_pages_slots(vx_pages_args a) {
    const uint32_t end = (uint32_t)a.starts[a.seqs];
#pragma unroll 1
    for (uint32_t j = 0; j < 4; ++j) {
        const uint64_t at = (uint64_t)blockIdx.x * 1024 + j * 256 + threadIdx.x;
        if (at >= a.tokens) return;
        const uint32_t i = (uint32_t)at;
        int32_t slot = -1, pos = 0;
        if (i < end) {
            const uint32_t s = vx_owner((const uint32_t*)a.starts, a.seqs, i);
            const uint32_t first = (uint32_t)a.starts[s], n = (uint32_t)a.starts[s + 1] - first;
            const uint32_t len = (uint32_t)a.lens[s], want = (uint32_t)a.want[s];
            const bool served = len == want;  // (it has new tokens, so want was more than its length)
            pos = (int32_t)((served ? len - n : len) + (i - first));
            if (served) {
                const uint32_t page = (uint32_t)a.table[(uint64_t)s * a.table_stride + ((uint32_t)pos >> a.page_shift)];
                slot = (int32_t)((page << a.page_shift) + ((uint32_t)pos & ((1u << a.page_shift) - 1u)));
            }
        }
        a.slots[i] = slot;
        a.positions[i] = pos;
    }
}
