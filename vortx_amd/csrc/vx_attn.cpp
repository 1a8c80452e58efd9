// vx_attn.cpp — host side of the quantized key/value cache and the attention
// over it: checks, kernel choice, and how the keys are split over workgroups.
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
static const int kWrite[4] = VX_DIMS(kv_write), kRead[4] = VX_DIMS(kv_read), kEven16[4] = VX_DIMS(attn_even16),
                 kEach128[4] = VX_DIMS(attn_each128);
#undef VX_DIMS
#define VX_DIMS(f) {K_vx_##f##_d64_k8v8, K_vx_##f##_d96_k8v8, K_vx_##f##_d128_k8v8}
static const int kJoin[4] = {K_vx_attn_join_d64, K_vx_attn_join_d96, K_vx_attn_join_d128, K_vx_attn_join_d256};
static const int kEach256[3] = VX_DIMS(attn_each256);
#undef VX_DIMS
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
static int run_rows(vx_ctx ctx, vx_stream stream, const vx_kv_cache* cache, const vx_cview* k, const vx_cview* v,
                    const int32_t* slots, bool write) {
    clear_error();
    if (!ctx) return fail(VX_ERR_INVALID, "null ctx");
    vx_kv_rows_args a{};
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
    const uint32_t grid = (uint32_t)std::min<uint64_t>((units + 31) / 32, 1u << 20);
    return launch_struct(ctx, kernel_of(cache, write ? kWrite : kRead), grid, 256, stream, &a);
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
