// vx_attn.cpp — host side of the quantized key/value cache, what goes into it
// (pages, rotated rows) and the attention over it: checks, kernel choice, and how
// the work is split over workgroups.
#include <algorithm>
#include <cmath>

#include "vx_internal.hpp"
#include "vx_kargs.h"

namespace vx {

// Values of a block of 32 take 32 (8 bits) or 16 (4 bits) bytes, its scale 2.
static uint64_t token_bytes(uint32_t type, uint32_t dim) { return (uint64_t)(dim / 32u) * (type == VX_Q8_0 ? 34u : 18u); }

static int dim_index(uint32_t dim) { return dim == 64 ? 0 : dim == 96 ? 1 : dim == 128 ? 2 : dim == 256 ? 3 : -1; }

static int check_geometry(const vx_kv_cache* c, uint64_t* bytes) {
    if (!c) return fail(VX_ERR_INVALID, "null cache");
    if ((c->k_type != VX_Q8_0 && c->k_type != VX_Q4_0) || (c->v_type != VX_Q8_0 && c->v_type != VX_Q4_0))
        return fail(VX_ERR_INVALID, "cache types are VX_Q8_0 and VX_Q4_0");
    if (dim_index(c->dim) < 0) return fail(VX_ERR_UNSUPPORTED, "head dim is not 64, 96, 128 or 256");
    if (c->page_tokens < 16 || c->page_tokens > 65536 || (c->page_tokens & (c->page_tokens - 1)))
        return fail(VX_ERR_UNSUPPORTED, "page_tokens is not a power of two from 16 to 65536");
    if (c->heads == 0 || c->heads > 4096) return fail(VX_ERR_UNSUPPORTED, "cache heads are not 1 to 4096");
    if ((uint64_t)c->pages * c->page_tokens > (1ull << 31)) return fail(VX_ERR_UNSUPPORTED, "a cache has at most 2^31 slots");
    // (a byte more each: how large the scales are, vx_kv.hpp)
    *bytes = (uint64_t)c->pages * c->page_tokens * c->heads * (token_bytes(c->k_type, c->dim) + token_bytes(c->v_type, c->dim) + 2);
    return VX_OK;
}

static int check_cache(const vx_kv_cache* c, vx_kv_geom* g) {
    uint64_t need = 0;
    const int s = check_geometry(c, &need);
    if (s) return s;
    if (c->bytes < need) return fail(VX_ERR_INVALID, "cache buffer is smaller than vx_kv_cache_size");
    if (need && !c->base) return fail(VX_ERR_INVALID, "null cache base");
    if ((uintptr_t)c->base & 15u) return fail(VX_ERR_INVALID, "cache base is not 16-byte aligned");
    g->base = (uint8_t*)c->base;
    g->pages = c->pages;
    g->page_bytes = c->pages ? need / c->pages : 0;
    g->page_shift = 0;
    while ((1u << g->page_shift) < c->page_tokens) ++g->page_shift;
    g->heads = c->heads;
    g->dim = c->dim;
    return VX_OK;
}

// Kernel of this cache's head size and types: the lists go d64 k8v8, k8v4, k4v8, k4v4, d96 ...
static int kernel_of(const vx_kv_cache* c, const int* d) {
    return d[dim_index(c->dim)] + (c->k_type == VX_Q4_0 ? 2 : 0) + (c->v_type == VX_Q4_0 ? 1 : 0);
}
#define VX_DIMS(f) {K_vx_##f##_d64_k8v8, K_vx_##f##_d96_k8v8, K_vx_##f##_d128_k8v8, K_vx_##f##_d256_k8v8}
static const int kWrite[4] = VX_DIMS(kv_write), kRead[4] = VX_DIMS(kv_read), kRotateKv[4] = VX_DIMS(rotate_kv), kRotateKv4[4] = VX_DIMS(rotate_kv4), kEven16[4] = VX_DIMS(attn_even16),
                 kEach128[4] = VX_DIMS(attn_each128);
#undef VX_DIMS
#define VX_DIMS(f) {K_vx_##f##_d64_k8v8, K_vx_##f##_d96_k8v8, K_vx_##f##_d128_k8v8}
static const int kJoin[4] = {K_vx_attn_join_d64, K_vx_attn_join_d96, K_vx_attn_join_d128, K_vx_attn_join_d256};
static const int kEach256[3] = VX_DIMS(attn_each256);
#undef VX_DIMS
static const int kRotateKvStrided[4] = {K_vx_rotate_kv_d64_s_k8v8, K_vx_rotate_kv_d96_s_k8v8, K_vx_rotate_kv_d128_s_k8v8,
                                        K_vx_rotate_kv_d256_s_k8v8};
static const int kEvenTiles[4] = {K_vx_attn_even256_d64_k8v8, K_vx_attn_even256_d96_k8v8, K_vx_attn_even256_d128_k8v8,
                                  K_vx_attn_even128_d256_k8v8};

// A [tokens, heads, dim] view.
struct Rows {
    uintptr_t ptr;
    uint32_t tokens, heads;
    int64_t stride[3];
    bool vec;  // stride 1 along the dim, 16-byte aligned rows
};

static int rows_view(const void* base, const vx_layout* l, uint32_t dim, Rows* r, const char* name, bool written) {
    Canon c;
    const int s = canon_view(base, l, &c, name);
    if (s) return s;
    if (c.l.size[0] != 1 || c.l.size[3] != dim) return fail(VX_ERR_SHAPE, "a view of rows is [tokens, heads, dim] with the cache's dim");
    r->ptr = c.ptr;
    r->tokens = c.l.size[1];
    r->heads = c.l.size[2];
    for (int i = 0; i < 3; ++i) {
        r->stride[i] = c.l.stride[i + 1];
        if (written && c.l.size[i + 1] > 1 && r->stride[i] == 0)
            return fail(VX_ERR_INVALID, "a written view has a zero stride on a dimension of size > 1");
    }
    r->vec = r->stride[2] == 1 && (c.ptr & 15u) == 0 && (r->tokens == 1 || r->stride[0] % 4 == 0) &&
             (r->heads == 1 || r->stride[1] % 4 == 0);
    return VX_OK;
}

// Tokens by fours from so many on: 333 of 3 heads of 64 read back 4.25 us (one by one 4.15), 8000 of
// 8 heads of 128 written and read 42.8 (53.7). Fewer leave most of the card without work.
constexpr uint32_t VX_QUAD_TOKENS = 256;
// The arguments of a call on rows, and its workgroups (0: nothing to do).
static int plan_rows(const vx_kv_cache* cache, const vx_cview* k, const vx_cview* v, const int32_t* slots, bool write,
                     vx_kv_rows_args* out, uint32_t* grid) {
    vx_kv_rows_args& a = *out;
    *grid = 0;
    int s = check_cache(cache, &a.c);
    if (s) return s;
    if (write ? !k || !v : !k && !v) return fail(VX_ERR_INVALID, "null view");
    Rows r[2] = {};
    const vx_cview* views[2] = {k, v};
    a.vec = 1;
    for (int i = 0; i < 2; ++i) {
        if (!views[i]) continue;
        if ((s = rows_view(views[i]->base, &views[i]->layout, cache->dim, &r[i], i ? "v" : "k", !write))) return s;
        if (r[i].heads != cache->heads) return fail(VX_ERR_SHAPE, "k and v have the cache's heads");
        if (!r[i].vec) a.vec = 0;
    }
    if (k && v && r[0].tokens != r[1].tokens) return fail(VX_ERR_SHAPE, "k and v have different tokens");
    a.tokens = k ? r[0].tokens : r[1].tokens;
    if (a.tokens == 0) return VX_OK;
    if (!slots) return fail(VX_ERR_INVALID, "null slots");
    if ((uintptr_t)slots & 3u) return fail(VX_ERR_INVALID, "slots is not 4-byte aligned");
    if (cache->pages == 0 && write) return VX_OK;
    a.slots = slots;
    a.k = k ? (float*)r[0].ptr : nullptr;
    a.v = v ? (float*)r[1].ptr : nullptr;
    for (int i = 0; i < 3; ++i) {
        a.ks[i] = r[0].stride[i];
        a.vs[i] = r[1].stride[i];
    }
    a.quads = a.tokens >= VX_QUAD_TOKENS;
    a.groups = a.quads ? (a.tokens - 1) / 4 + 1 : a.tokens;
    const uint64_t units = (uint64_t)a.groups * cache->heads * (cache->dim == 96 ? 4 : cache->dim / 32);
    *grid = (uint32_t)std::min<uint64_t>((units + 31) / 32, 1u << 20);
    return VX_OK;
}

static int run_rows(vx_ctx ctx, vx_stream stream, const vx_kv_cache* cache, const vx_cview* k, const vx_cview* v,
                    const int32_t* slots, bool write) {
    clear_error();
    if (!ctx) return fail(VX_ERR_INVALID, "null ctx");
    vx_kv_rows_args a{};
    uint32_t grid = 0;
    if (const int s = plan_rows(cache, k, v, slots, write, &a, &grid)) return s;
    return launch_struct(ctx, kernel_of(cache, write ? kWrite : kRead), grid, 256, stream, &a);
}

static int check_rotation(const vx_rotation* r, uint32_t dim) {
    if (!r) return fail(VX_ERR_INVALID, "null rotation");
    if (r->reserved) return fail(VX_ERR_INVALID, "vx_rotation.reserved must be 0");
    if (r->flags & ~(uint32_t)(VX_ROTATE_PAIRS | VX_ROTATE_NORM)) return fail(VX_ERR_INVALID, "unknown rotation flags");
    if (r->rotated % 2) return fail(VX_ERR_SHAPE, "an even number of dims is rotated");
    if (r->rotated > dim) return fail(VX_ERR_SHAPE, "more dims are rotated than a head has");
    if (r->rotated && !r->freqs) return fail(VX_ERR_INVALID, "null freqs");
    if ((uintptr_t)r->freqs & 7u) return fail(VX_ERR_INVALID, "freqs is not 8-byte aligned");
    if (((uintptr_t)r->q_weight | (uintptr_t)r->k_weight) & 3u) return fail(VX_ERR_INVALID, "a norm weight is not 4-byte aligned");
    if (!(r->flags & VX_ROTATE_NORM)) {
        if (r->q_weight || r->k_weight) return fail(VX_ERR_INVALID, "norm weights without VX_ROTATE_NORM");
        return VX_OK;
    }
    if (!(r->eps >= 0.f) || !std::isfinite(r->eps)) return fail(VX_ERR_INVALID, "eps is negative or not finite");
    if ((r->q_weight && r->q_weight_stride && r->q_weight_stride < dim) || (r->k_weight && r->k_weight_stride && r->k_weight_stride < dim))
        return fail(VX_ERR_INVALID, "norm weights of heads overlap");
    return VX_OK;
}

// The arguments for rows q (0) and k (1); either view may be null, outputs too. vec:
// fours of dims, and their partners, are 16-byte aligned everywhere.
static int plan_rotation(const vx_mview* const (&outs)[2], const vx_cview* const (&ins)[2], uint32_t dim, const int32_t* positions,
                         const vx_rotation* how, vx_rotate_args* a, bool* vec) {
    static const char* const names[2][2] = {{"q", "q_out"}, {"k", "k_out"}};
    int s = check_rotation(how, dim);
    if (s) return s;
    const bool norm = how->flags & VX_ROTATE_NORM;
    const float* const weights[2] = {how->q_weight, how->k_weight};
    const uint32_t strides[2] = {how->q_weight_stride, how->k_weight_stride};
    a->pairs = how->flags & VX_ROTATE_PAIRS ? 1 : 0;
    a->norm = norm;
    a->dim = dim;
    a->per_dim = 1.0 / dim;
    a->rotated = how->rotated;
    a->eps = how->eps;
    a->freqs = how->freqs;
    a->positions = positions;
    *vec = dim % 4 == 0 && how->rotated % (a->pairs ? 4 : 8) == 0;
    bool first = true;
    for (int i = 0; i < 2; ++i) {
        if (!ins[i]) continue;
        vx_rotate_rows_args& p = a->part[i];
        Rows r, o;
        if ((s = rows_view(ins[i]->base, &ins[i]->layout, dim, &r, names[i][0], false))) return s;
        if (!first && r.tokens != a->tokens) return fail(VX_ERR_SHAPE, "q and k have different tokens");
        first = false;
        // (the kernels' counters go on to two steps past a run of heads, in 32 bits)
        if (r.heads > 0x7FFFFFFFu) return fail(VX_ERR_UNSUPPORTED, "2^31 heads and more");
        a->tokens = r.tokens;
        p.heads = r.heads;
        p.x = (const float*)r.ptr;
        p.w = norm ? weights[i] : nullptr;
        p.ws = strides[i];
        for (int j = 0; j < 3; ++j) p.xs[j] = r.stride[j];
        if (!r.vec || (p.w && (((uintptr_t)weights[i] & 15u) || strides[i] % 4))) *vec = false;
        if (!outs[i]) continue;
        if ((s = rows_view(outs[i]->base, &outs[i]->layout, dim, &o, names[i][1], true))) return s;
        if (o.tokens != r.tokens || o.heads != r.heads) return fail(VX_ERR_SHAPE, i ? "k and k_out have different shapes" : "q and q_out have different shapes");
        p.y = (float*)o.ptr;
        for (int j = 0; j < 3; ++j) p.ys[j] = o.stride[j];
        if (!o.vec) *vec = false;
    }
    if (how->rotated && a->tokens && (!positions || ((uintptr_t)positions & 3u)))
        return fail(VX_ERR_INVALID, "positions is null or not 4-byte aligned");
    return VX_OK;
}

static int lanes_index(uint32_t dim) { return dim <= 64 ? 0 : dim <= 128 ? 1 : 2; }

// Tokens and heads of a workgroup: `many` tokens and as many heads as leave the card
// full, whose angles are computed once for them; where there are few rows, one token
// and as many heads as its lanes take at once.
static void split_rows(int num_cus, uint32_t tokens, uint32_t dim, uint32_t many, vx_rotate_rows_args* p) {
    p->block_tokens = p->run = p->chunks = p->blocks = 0;
    if (!tokens || !p->heads) return;
    const uint64_t at_once = 16u >> lanes_index(dim), rows = (uint64_t)tokens * p->heads;
    p->block_tokens = rows / at_once >= (uint64_t)num_cus * 4 ? many : 1;
    const uint64_t groups = ((uint64_t)tokens + p->block_tokens - 1) / p->block_tokens;
    // (six workgroups a CU end about together, and each has its angles for more heads than with twelve: us, six / twelve /
    // three, 4097 tokens of 32 heads of 80 19.7 / 23.8 / 19.8; 8000 of 32 of 128 65 / 63 / 66, of 8 into the cache 46 / 59 / 44)
    const uint64_t most = std::max<uint64_t>(std::max<uint64_t>(1, at_once / p->block_tokens), groups * p->heads / ((uint64_t)num_cus * 6));
    p->chunks = (uint32_t)((p->heads + most - 1) / most);
    p->run = (p->heads + p->chunks - 1) / p->chunks;
    p->chunks = (p->heads + p->run - 1) / p->run;
    p->blocks = (uint32_t)(groups * p->chunks);
}

// One launch for tokens [t, t + n) of a part or of both: a workgroup is a job, so that
// calls beyond a grid's size go in pieces.
constexpr uint32_t VX_ROTATE_PIECE = 1u << 20;
static void move_rows(vx_rotate_args* a, uint32_t tokens) {  // on by so many tokens
    for (auto& p : a->part) {
        if (p.x) p.x += p.xs[0] * tokens;
        if (p.y) p.y += p.ys[0] * tokens;
    }
    if (a->positions) a->positions += tokens;
    a->tokens -= tokens;
}

static int run_rotate(vx_ctx ctx, vx_stream stream, const vx_mview* q_out, const vx_cview* q, const vx_mview* k_out, const vx_cview* k,
                      const int32_t* positions, const vx_rotation* how) {
    if (!q || !q_out) return fail(VX_ERR_INVALID, "null view");
    if (!k != !k_out) return fail(VX_ERR_INVALID, "k without k_out, or k_out without k");
    Canon c;
    int s = canon_view(q->base, &q->layout, &c, "q");
    if (s) return s;
    const uint32_t dim = c.l.size[3];
    if (dim == 0 || dim > 256) return fail(VX_ERR_UNSUPPORTED, "heads have 1 to 256 dims");
    vx_rotate_args a{};
    bool vec = false;
    if ((s = plan_rotation({q_out, k_out}, {q, k}, dim, positions, how, &a, &vec))) return s;
    while (a.tokens && !s) {
        vx_rotate_args one = a;
        one.tokens = std::min(a.tokens, VX_ROTATE_PIECE);
        for (auto& p : one.part) split_rows(ctx_cus(ctx), one.tokens, dim, dim > 128 ? 4 : 8, &p);
        s = launch_struct(ctx, (vec ? K_vx_rotate_l16 : K_vx_rotate_l16_s) + lanes_index(dim), one.part[0].blocks + one.part[1].blocks, 256, stream, &one);
        move_rows(&a, one.tokens);
    }
    return s;
}

static int run_write_rotated(vx_ctx ctx, vx_stream stream, const vx_kv_cache* cache, const vx_mview* q_out, const vx_cview* q,
                             const vx_cview* k, const vx_cview* v, const int32_t* positions, const int32_t* slots,
                             const vx_rotation* how) {
    if (!q != !q_out) return fail(VX_ERR_INVALID, "q without q_out, or q_out without q");
    vx_kv_rotated_args a{};
    uint32_t grid = 0;
    int s = plan_rows(cache, k, v, slots, true, &a.r, &grid);
    if (s) return s;
    bool vec = false;
    if ((s = plan_rotation({q_out, nullptr}, {q, k}, cache->dim, positions, how, &a.t, &vec))) return s;
    if (!grid) a.t.part[1].heads = 0;  // (a cache without pages)
    while (a.t.tokens && !s) {
        vx_kv_rotated_args one = a;
        vx_rotate_rows_args *qs = &one.t.part[0], *ks = &one.t.part[1];
        one.r.tokens = one.t.tokens = std::min(a.t.tokens, VX_ROTATE_PIECE);
        split_rows(ctx_cus(ctx), one.t.tokens, cache->dim, cache->dim > 128 ? 4 : 8, qs);
        split_rows(ctx_cus(ctx), one.t.tokens, cache->dim, 8, ks);
        one.r.quads = vec && ks->block_tokens == 8;
        one.r.groups = one.r.quads ? (one.r.tokens - 1) / 4 + 1 : one.r.tokens;
        if (one.r.quads) {
            ks->run = std::min(ks->run, VX_ROTATE_STAGE / (cache->dim * 11u));
            ks->chunks = (ks->heads + ks->run - 1) / ks->run;
            ks->blocks = (one.t.tokens + 7) / 8 * ks->chunks;
            s = launch_struct(ctx, kernel_of(cache, kRotateKv4), ks->blocks, 256, stream, &one);
            ks->blocks = 0;
            if (!s) s = launch_struct(ctx, K_vx_rotate_l16 + lanes_index(cache->dim), qs->blocks, 256, stream, &one.t);
        } else {
            s = launch_struct(ctx, kernel_of(cache, vec ? kRotateKv : kRotateKvStrided), qs->blocks + ks->blocks, 256, stream, &one);
        }
        move_rows(&a.t, one.t.tokens);
        a.r.k += a.r.ks[0] * one.t.tokens;
        a.r.v += a.r.vs[0] * one.t.tokens;
        a.r.slots += one.t.tokens;
    }
    return s;
}

// Slots in the workgroup that deals out the pages, up to so many tokens.
constexpr uint32_t VX_SLOTS_HERE = 4096;
static int run_resize(vx_ctx ctx, vx_stream stream, const vx_kv_pages* p, const int32_t* want, int32_t* starts, int32_t* slots,
                      int32_t* positions, uint32_t tokens) {
    if (!p) return fail(VX_ERR_INVALID, "null pages");
    if (p->reserved) return fail(VX_ERR_INVALID, "vx_kv_pages.reserved must be 0");
    if (p->page_tokens < 16 || p->page_tokens > 65536 || (p->page_tokens & (p->page_tokens - 1)))
        return fail(VX_ERR_UNSUPPORTED, "page_tokens is not a power of two from 16 to 65536");
    if ((uint64_t)p->pages * p->page_tokens > (1ull << 31)) return fail(VX_ERR_UNSUPPORTED, "a cache has at most 2^31 slots");
    if (p->table_stride < p->table_cols) return fail(VX_ERR_INVALID, "table_stride smaller than table_cols");
    if ((uint64_t)p->seqs * p->table_cols >= (1ull << 31) || p->seqs >= (1u << 31))
        return fail(VX_ERR_UNSUPPORTED, "a table has fewer than 2^31 entries");
    if (tokens > (1u << 30)) return fail(VX_ERR_UNSUPPORTED, "more than 2^30 tokens");
    if (!p->free_count || (p->pages && !p->free_pages) || (p->seqs && (!p->lens || !want || (p->table_cols && !p->table))))
        return fail(VX_ERR_INVALID, "null pages array");
    if (!starts || (tokens && (!slots || !positions))) return fail(VX_ERR_INVALID, "null output array");
    if (((uintptr_t)p->table | (uintptr_t)p->lens | (uintptr_t)p->free_pages | (uintptr_t)p->free_count | (uintptr_t)want |
         (uintptr_t)starts | (uintptr_t)slots | (uintptr_t)positions) & 3u)
        return fail(VX_ERR_INVALID, "an array is not 4-byte aligned");
    vx_pages_args a{};
    a.table = p->table;
    a.lens = p->lens;
    a.free_pages = p->free_pages;
    a.free_count = p->free_count;
    a.want = want;
    a.starts = starts;
    a.slots = slots;
    a.positions = positions;
    a.seqs = p->seqs;
    a.table_cols = p->table_cols;
    a.table_stride = p->table_stride;
    while ((1u << a.page_shift) < p->page_tokens) ++a.page_shift;
    a.pages = p->pages;
    a.tokens = tokens;
    a.here = tokens <= VX_SLOTS_HERE;
    a.vec = (((uintptr_t)slots | (uintptr_t)positions) & 15u) == 0;
    a.threads = p->seqs <= 256 && tokens <= 1024 ? 256 : 1024;
    if (const int s = launch_struct(ctx, K_vx_pages_resize, 1, a.threads, stream, &a)) return s;
    return a.here ? VX_OK : launch_struct(ctx, K_vx_pages_slots, (tokens + 1023) / 1024, 256, stream, &a);
}

// How a call is laid out: the kernel by the query rows of a sequence and head
// (16, 128 or 256 a workgroup), and whether a workgroup takes a unit (row block,
// sequence, head) each, or the keys of all units are dealt out evenly over the
// places that the card has for workgroups.
constexpr uint32_t VX_MOST_KEYS = (1u << 31) - 65536u;  // of a sequence
// Up to so many rows the 16-row kernel, whose row blocks read the keys again, is
// faster than the tiles of 128 and 256 rows, which decode them once. Trees of
// drafts, us, 16 rows / tiles:
//   dim 128, 1 sequence of 300 keys   120 rows 13.9 / 24.2   128 rows 13.9 / 24.5
//            1 of 1500                120      19.1 / 30.2   128      19.8 / 30.7   192 rows 22.1 / 37.0
//            1 of 20000               120      56.1 / 57.7   128      57.9 / 58.6   192      78.3 / 72.5
//            4 of up to 6000          120      47.0 / 50.1   128      56.1 / 60.2
//            8 of up to 12000         120       116 / 112    128       140 / 129    192       203 / 186
//            32 of up to 2000         120       112 / 105    128       105 / 95.9   192       162 / 151
//   dim 96,  1 of 1500                120      17.9 / 27.0   128      17.9 / 27.1
//            8 of up to 12000         120      89.8 / 105    128      96.4 / 115
//            32 of up to 2000         120      88.8 / 90.0   128       106 / 100
//   dim 64,  4 of up to 6000          128      37.1 / 42.2   192      57.0 / 61.0
//   dim 256, 4 of up to 6000          128       102 / 115    192       181 / 194
// So batches of many sequences lose up to a tenth just below the bound, and single ones win up to half.
static uint64_t rows16_most(uint32_t dim) { return dim == 96 || dim == 128 ? 128 : 192; }
// More units than places: a workgroup each (units of one length, or many of them,
// fill the card by themselves, and no partial sums are written). Us, a workgroup
// each / dealt out evenly: 512 units on 256 places, 4096 causal tokens of 32
// heads of 128, 398 / 462; 480, windows of 1000 in prompts of up to 2500, 116 /
// 133; 752 of dim 64, two prompts of up to 3000, 271 / 289. Up to as many: 256,
// four chunks behind histories of 900 to 3000, 259 / 255; 256, a prompt of 2000,
// 153 / 148.
constexpr uint64_t VX_EVEN_UNITS = 1;
struct AttnPlan {
    const int* kernel;
    uint32_t block, rows, row_blocks, grid, parts;
    bool even;
    uint64_t units;
    uint64_t info() const { return (units * 8 + 15) / 16 * 16; }  // bytes of the workspace before the partial sums
    uint64_t part_rows() const { return 2ull * grid * rows; }
    uint64_t bytes(uint32_t dim) const { return even ? info() + part_rows() * (dim + 2) * 4 : 0; }
};

static int plan_attention(int num_cus, const vx_kv_cache* c, const vx_attn_batch* b, const vx_attn_opts* o, uint32_t q_heads,
                          bool ws, AttnPlan* p) {
    const uint64_t group = q_heads / c->heads, queries = b->max_queries, rows = queries * group;
    // 256 rows a workgroup decode a tile of keys once where two of 128 do it twice; us, 256 / 128
    // rows, when both were dealt out: 4096 causal tokens, dim 128 383 / 430, dim 64 250 / 268; chunks behind histories 208 / 229;
    // trees of 244 rows 196 / 183, of 200 rows, 16 sequences, 313 / 312. (256 dims: see the kernels.)
    const bool wide = rows > 128 && c->dim <= 128;
    *p = AttnPlan{};
    // (a grid has below 2^32 threads, and the join 256 a row; one factor after the other: the products stay in 64 bits)
    constexpr uint64_t most_rows = 1ull << 24;
    if (rows >= most_rows || rows * b->seqs >= most_rows || rows * b->seqs * c->heads >= most_rows)
        return fail(VX_ERR_UNSUPPORTED, "attention: too many query rows (split the batch)");
    // (the keys are dealt out by their number of steps, which is counted in 32 bits)
    const uint64_t most = std::min<uint64_t>(b->max_len, (uint64_t)b->table_cols * c->page_tokens);
    const bool deal = ws && ((rows + 15) / 16) * b->seqs * (most / 64 + 8) < (1ull << 32);
    p->rows = rows <= rows16_most(c->dim) && deal ? 16 : wide ? 256 : 128;
    p->block = p->rows == 256 ? 512 : 256;
    const uint64_t places = (uint64_t)num_cus * (p->rows == 256 || c->dim > 128 ? 1 : 2);  // workgroups that the card holds
    const uint64_t rb = (rows + p->rows - 1) / p->rows;
    p->units = rb * b->seqs * c->heads;
    if (p->units >= (1ull << 23)) return fail(VX_ERR_UNSUPPORTED, "attention: too many query rows (split the batch)");
    p->row_blocks = (uint32_t)rb;
    p->even = deal && (p->rows == 16 || p->units <= VX_EVEN_UNITS * places);
    p->kernel = p->even ? (p->rows == 16 ? kEven16 : kEvenTiles) : p->rows == 128 ? kEach128 : kEach256;
    p->grid = (uint32_t)p->units;
    if (p->even) {
        uint64_t span = most;
        if (o && o->window) span = std::min<uint64_t>(span, 2ull * o->window + queries + 64);
        const uint64_t step = p->rows == 16 ? 128 : 64;
        p->grid = (uint32_t)std::max<uint64_t>(1, std::min(p->units * ((span + step - 1) / step + 1), places));
        p->parts = (uint32_t)(p->grid / std::max<uint64_t>(1, p->units)) + 2;
    }
    return VX_OK;
}

static int check_batch(const vx_kv_cache* c, const vx_attn_batch* b, const vx_attn_opts* o, uint32_t q_heads) {
    if (!b) return fail(VX_ERR_INVALID, "null batch");
    if (b->reserved) return fail(VX_ERR_INVALID, "vx_attn_batch.reserved must be 0");
    if (q_heads == 0 || q_heads % c->heads) return fail(VX_ERR_SHAPE, "query heads are not a multiple of the cache's heads");
    if (b->table_stride < b->table_cols) return fail(VX_ERR_INVALID, "table_stride smaller than table_cols");
    if (b->max_len > VX_MOST_KEYS) return fail(VX_ERR_UNSUPPORTED, "max_len is 2^31 - 2^16 at most");
    if (b->seqs && (!b->lens || !b->starts || (!b->table && b->table_cols))) return fail(VX_ERR_INVALID, "null batch array");
    if (((uintptr_t)b->lens | (uintptr_t)b->starts | (uintptr_t)b->table) & 3u)
        return fail(VX_ERR_INVALID, "a batch array is not 4-byte aligned");
    if (!o) return VX_OK;
    if (o->flags & ~(uint32_t)VX_ATTN_CAUSAL) return fail(VX_ERR_INVALID, "unknown attention flags");
    if (!std::isfinite(o->scale)) return fail(VX_ERR_INVALID, "scale is not finite");
    if (!(o->softcap >= 0.f) || !std::isfinite(o->softcap)) return fail(VX_ERR_INVALID, "softcap is negative or not finite");
    if (((uintptr_t)o->slopes | (uintptr_t)o->prefix | (uintptr_t)o->first) & 3u)
        return fail(VX_ERR_INVALID, "an option array is not 4-byte aligned");
    return VX_OK;
}

static int run_attention(vx_ctx ctx, vx_stream stream, const vx_mview* out, const vx_cview* q, const vx_kv_cache* cache,
                         const vx_attn_batch* batch, const vx_attn_opts* opts, const uint32_t* tree, uint32_t tree_words,
                         uint32_t tree_stride, void* ws, uint64_t ws_size) {
    vx_attn_args a{};
    int s = check_cache(cache, &a.c);
    if (s) return s;
    if (!out || !q) return fail(VX_ERR_INVALID, "null view");
    Rows ro, rq;
    if ((s = rows_view(out->base, &out->layout, cache->dim, &ro, "out", true))) return s;
    if ((s = rows_view(q->base, &q->layout, cache->dim, &rq, "q", false))) return s;
    if (ro.tokens != rq.tokens || ro.heads != rq.heads) return fail(VX_ERR_SHAPE, "q and out have different shapes");
    if ((s = check_batch(cache, batch, opts, rq.heads))) return s;
    if ((uintptr_t)ws & 15u) return fail(VX_ERR_INVALID, "workspace is not 16-byte aligned");
    if (rq.tokens > (1u << 30)) return fail(VX_ERR_UNSUPPORTED, "more than 2^30 query tokens");
    if (rq.tokens == 0 || batch->seqs == 0 || batch->max_queries == 0) return VX_OK;
    AttnPlan p;
    if ((s = plan_attention(ctx_cus(ctx), cache, batch, opts, rq.heads, ws != nullptr, &p))) return s;
    if (ws_size < p.bytes(cache->dim)) return fail(VX_ERR_INVALID, "workspace smaller than vx_attention_ws_size");
    a.q = (const float*)rq.ptr;
    a.out = (float*)ro.ptr;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = rq.stride[i];
        a.os[i] = ro.stride[i];
    }
    a.vec = rq.vec && ro.vec;
    a.table = batch->table;
    a.lens = batch->lens;
    a.starts = batch->starts;
    a.table_stride = batch->table_stride;
    a.table_cols = cache->pages ? (uint32_t)std::min<uint64_t>(batch->table_cols, ((1u << 31) - 1u) >> a.c.page_shift) : 0u;
    a.seqs = batch->seqs;
    a.tokens = rq.tokens;
    a.group = rq.heads / cache->heads;
    a.max_queries = batch->max_queries;
    a.max_len = batch->max_len;
    a.scale = opts && opts->scale != 0.f ? opts->scale : 1.f / std::sqrt((float)cache->dim);
    if (opts) {
        // score / cap and cap log2(e) must stay among f32's normal numbers: a cap that scores do not come
        // near changes none, and below 2^-64 no cap leaves a difference between keys
        a.cap = opts->softcap >= 0x1p64f ? 0.f : opts->softcap > 0.f ? std::max(opts->softcap, 0x1p-64f) : 0.f;
        a.slopes = opts->slopes;
        a.first = opts->first;
        a.window = opts->window >= VX_MOST_KEYS ? 0u : opts->window;  // (none that any key is outside of)
        if (!tree) {
            a.causal = opts->flags & VX_ATTN_CAUSAL;
            a.prefix = opts->prefix;
        }
    }
    a.tree = tree;
    a.tree_words = tree_words;
    a.tree_stride = tree_stride;
    a.row_blocks = p.row_blocks;
    a.part_rows = p.rows;
    a.parts = p.parts;
    a.info = (uint32_t*)ws;
    a.part_o = (float*)((char*)ws + p.info());
    a.part_ml = a.part_o + p.part_rows() * cache->dim;
    if ((s = launch_struct(ctx, kernel_of(cache, p.kernel), p.grid, p.block, stream, &a))) return s;
    if (p.even) {
        const uint64_t jobs = (uint64_t)batch->max_queries * a.group * batch->seqs * cache->heads;
        return launch_struct(ctx, kJoin[dim_index(cache->dim)], (uint32_t)(p.parts > 8 ? jobs : (jobs + 3) / 4), 256, stream, &a);
    }
    return VX_OK;
}

}  // namespace vx

extern "C" {

int vx_kv_cache_size(const vx_kv_cache* cache, uint64_t* bytes) {
    vx::clear_error();
    if (!bytes) return vx::fail(VX_ERR_INVALID, "null bytes");
    return vx::check_geometry(cache, bytes);
}

int vx_kv_write(vx_ctx ctx, vx_stream stream, const vx_kv_cache* cache, const vx_cview* k, const vx_cview* v,
                const int32_t* slots) {
    return vx::run_rows(ctx, stream, cache, k, v, slots, true);
}

int vx_kv_read(vx_ctx ctx, vx_stream stream, const vx_mview* k, const vx_mview* v, const vx_kv_cache* cache,
               const int32_t* slots) {
    vx_cview c[2];
    const vx_mview* views[2] = {k, v};
    for (int i = 0; i < 2; ++i)
        if (views[i]) c[i] = vx_cview{views[i]->base, views[i]->layout};
    return vx::run_rows(ctx, stream, cache, k ? &c[0] : nullptr, v ? &c[1] : nullptr, slots, false);
}

int vx_rotate(vx_ctx ctx, vx_stream stream, const vx_mview* q_out, const vx_cview* q, const vx_mview* k_out,
              const vx_cview* k, const int32_t* positions, const vx_rotation* how) {
    vx::clear_error();
    if (!ctx) return vx::fail(VX_ERR_INVALID, "null ctx");
    return vx::run_rotate(ctx, stream, q_out, q, k_out, k, positions, how);
}

int vx_kv_write_rotated(vx_ctx ctx, vx_stream stream, const vx_kv_cache* cache, const vx_mview* q_out, const vx_cview* q,
                        const vx_cview* k, const vx_cview* v, const int32_t* positions, const int32_t* slots,
                        const vx_rotation* how) {
    vx::clear_error();
    if (!ctx) return vx::fail(VX_ERR_INVALID, "null ctx");
    return vx::run_write_rotated(ctx, stream, cache, q_out, q, k, v, positions, slots, how);
}

int vx_kv_resize(vx_ctx ctx, vx_stream stream, const vx_kv_pages* pages, const int32_t* want, int32_t* starts,
                 int32_t* slots, int32_t* positions, uint32_t tokens) {
    vx::clear_error();
    if (!ctx) return vx::fail(VX_ERR_INVALID, "null ctx");
    return vx::run_resize(ctx, stream, pages, want, starts, slots, positions, tokens);
}

int vx_attention(vx_ctx ctx, vx_stream stream, const vx_mview* out, const vx_cview* q, const vx_kv_cache* cache,
                 const vx_attn_batch* batch, const vx_attn_opts* opts, void* workspace, uint64_t workspace_bytes) {
    vx::clear_error();
    if (!ctx) return vx::fail(VX_ERR_INVALID, "null ctx");
    return vx::run_attention(ctx, stream, out, q, cache, batch, opts, nullptr, 0, 0, workspace, workspace_bytes);
}

int vx_attention_tree(vx_ctx ctx, vx_stream stream, const vx_mview* out, const vx_cview* q, const vx_kv_cache* cache,
                      const vx_attn_batch* batch, const vx_attn_opts* opts, const uint32_t* tree, uint32_t tree_words,
                      uint32_t tree_stride, void* workspace, uint64_t workspace_bytes) {
    vx::clear_error();
    if (!ctx) return vx::fail(VX_ERR_INVALID, "null ctx");
    if (!tree || ((uintptr_t)tree & 3u)) return vx::fail(VX_ERR_INVALID, "tree is null or not 4-byte aligned");
    if (tree_stride < tree_words) return vx::fail(VX_ERR_INVALID, "tree_stride smaller than tree_words");
    if (batch && 32ull * tree_words < batch->max_queries) return vx::fail(VX_ERR_SHAPE, "tree_words too few for max_queries drafts");
    return vx::run_attention(ctx, stream, out, q, cache, batch, opts, tree, tree_words, tree_stride, workspace, workspace_bytes);
}

int vx_attention_ws_size(vx_ctx ctx, const vx_kv_cache* cache, const vx_attn_batch* batch, const vx_attn_opts* opts,
                         uint32_t tokens, uint32_t q_heads, uint64_t* bytes) {
    vx::clear_error();
    if (!ctx || !bytes) return vx::fail(VX_ERR_INVALID, "null ctx or bytes");
    *bytes = 0;
    uint64_t unused = 0;
    int s = vx::check_geometry(cache, &unused);
    if (s) return s;
    if ((s = vx::check_batch(cache, batch, opts, q_heads))) return s;
    if (!tokens || !batch->seqs || !batch->max_queries) return VX_OK;
    vx::AttnPlan p;
    if ((s = vx::plan_attention(vx::ctx_cus(ctx), cache, batch, opts, q_heads, true, &p))) return s;
    *bytes = p.bytes(cache->dim);
    return vx::need_kernel(ctx, vx::kernel_of(cache, p.kernel));
}

}  // extern "C"
