// Calls that bring a step's pages, rotate rows and write them, on a HIP runtime
// that only counts: bad ones are refused and launch nothing, and every kernel of
// the step's code object is reached by some good one.
#include "hip_counts.hpp"

extern "C" {
extern const unsigned char vx_co_step[16];
const unsigned char vx_co_step[16] = {};
}

static vx_layout rows_of(uint32_t tokens, uint32_t heads, uint32_t dim) {
    vx_layout l = {};
    l.rank = 3;
    l.size[0] = tokens, l.size[1] = heads, l.size[2] = dim;
    l.stride[0] = heads * dim, l.stride[1] = dim, l.stride[2] = 1;
    return l;
}
static vx_cview in_of(uint32_t tokens, uint32_t heads, uint32_t dim) { return {(float*)0x100000, rows_of(tokens, heads, dim)}; }
static vx_mview out_of(uint32_t tokens, uint32_t heads, uint32_t dim) { return {(float*)0x200000, rows_of(tokens, heads, dim)}; }
static const int32_t* const kPos = (const int32_t*)0x3000;
static int refused(int status, int want) {
    const bool ok = status == want && launches == 0 && *vx_last_error_message();
    launches = 0;
    return ok;
}

int main() {
    vx_ctx ctx = nullptr;
    CHECK(vx_init(0, &ctx) == VX_OK);
    // ---- rotation
    vx_rotation how = {(const double*)0x8000, (const float*)0x9000, nullptr, 0, 0, 64, VX_ROTATE_NORM, 1e-6f, 0};
    vx_cview q = in_of(5, 8, 64), k = in_of(5, 2, 64), v = in_of(5, 2, 64);
    vx_mview qo = out_of(5, 8, 64), ko = out_of(5, 2, 64);
    auto rotate = [&](const vx_rotation& h) { return vx_rotate(ctx, nullptr, &qo, &q, &ko, &k, kPos, &h); };
    launches = 0;
    CHECK(refused(vx_rotate(nullptr, nullptr, &qo, &q, &ko, &k, kPos, &how), VX_ERR_INVALID));
    CHECK(refused(vx_rotate(ctx, nullptr, nullptr, &q, &ko, &k, kPos, &how), VX_ERR_INVALID));
    CHECK(refused(vx_rotate(ctx, nullptr, &qo, &q, nullptr, &k, kPos, &how), VX_ERR_INVALID));
    CHECK(refused(vx_rotate(ctx, nullptr, &qo, &q, &ko, nullptr, kPos, &how), VX_ERR_INVALID));
    CHECK(refused(vx_rotate(ctx, nullptr, &qo, &q, &ko, &k, nullptr, &how), VX_ERR_INVALID));
    CHECK(refused(vx_rotate(ctx, nullptr, &qo, &q, &ko, &k, (const int32_t*)0x3002, &how), VX_ERR_INVALID));
    CHECK(refused(vx_rotate(ctx, nullptr, &qo, &q, &ko, &k, kPos, nullptr), VX_ERR_INVALID));
    auto with = [&](auto change) {
        vx_rotation h = how;
        change(h);
        return rotate(h);
    };
    CHECK(refused(with([](vx_rotation& h) { h.rotated = 63; }), VX_ERR_SHAPE));
    CHECK(refused(with([](vx_rotation& h) { h.rotated = 66; }), VX_ERR_SHAPE));
    CHECK(refused(with([](vx_rotation& h) { h.freqs = nullptr; }), VX_ERR_INVALID));
    CHECK(refused(with([](vx_rotation& h) { h.freqs = (const double*)0x8004; }), VX_ERR_INVALID));
    CHECK(refused(with([](vx_rotation& h) { h.q_weight = (const float*)0x9001; }), VX_ERR_INVALID));
    CHECK(refused(with([](vx_rotation& h) { h.q_weight_stride = 63; }), VX_ERR_INVALID));
    CHECK(refused(with([](vx_rotation& h) { h.flags = 0; }), VX_ERR_INVALID));  // weights without a norm
    CHECK(refused(with([](vx_rotation& h) { h.flags = 4; }), VX_ERR_INVALID));
    CHECK(refused(with([](vx_rotation& h) { h.eps = -1.f; }), VX_ERR_INVALID));
    CHECK(refused(with([](vx_rotation& h) { h.eps = __builtin_nanf(""); }), VX_ERR_INVALID));
    CHECK(refused(with([](vx_rotation& h) { h.reserved = 1; }), VX_ERR_INVALID));
    k = in_of(5, 2, 32);
    CHECK(refused(rotate(how), VX_ERR_SHAPE));
    k = in_of(4, 2, 64), ko = out_of(4, 2, 64);
    CHECK(refused(rotate(how), VX_ERR_SHAPE));
    k = in_of(5, 2, 64), ko = out_of(5, 3, 64);
    CHECK(refused(rotate(how), VX_ERR_SHAPE));
    ko = out_of(5, 2, 64);
    qo.layout.stride[1] = 0;
    CHECK(refused(rotate(how), VX_ERR_INVALID));
    qo = out_of(5, 8, 64);
    q.base = nullptr;
    CHECK(refused(rotate(how), VX_ERR_INVALID));
    q = in_of(5, 8, 257), qo = out_of(5, 8, 257);
    CHECK(refused(rotate(how), VX_ERR_UNSUPPORTED));
    for (uint32_t dim : {1u, 64u, 80u, 256u}) {
        q = in_of(5, 8, dim), qo = out_of(5, 8, dim), k = in_of(5, 2, dim), ko = out_of(5, 2, dim);
        how.rotated = dim / 2 * 2;
        CHECK(rotate(how) == VX_OK && launches == 1);
        launches = 0;
        CHECK(vx_rotate(ctx, nullptr, &qo, &q, nullptr, nullptr, kPos, &how) == VX_OK && launches == 1);
        q.layout.stride[0] += 1;
        CHECK(rotate(how) == VX_OK && launches == 2);
        launches = 0;
    }
    q = in_of((1u << 21) + 5, 1, 64), qo = out_of((1u << 21) + 5, 1, 64);  // in pieces
    how.rotated = 64;
    CHECK(vx_rotate(ctx, nullptr, &qo, &q, nullptr, nullptr, kPos, &how) == VX_OK && launches == 3);
    launches = 0;
    q = in_of(0, 8, 64), qo = out_of(0, 8, 64), k = in_of(0, 2, 64), ko = out_of(0, 2, 64), how.rotated = 64;
    CHECK(rotate(how) == VX_OK && launches == 0);
    how.rotated = 0, how.freqs = nullptr;  // a norm alone
    q = in_of(5, 8, 64), qo = out_of(5, 8, 64);
    CHECK(vx_rotate(ctx, nullptr, &qo, &q, nullptr, nullptr, nullptr, &how) == VX_OK && launches == 1);
    launches = 0;
    // ---- into the cache
    how.rotated = 64, how.freqs = (const double*)0x8000;
    vx_kv_cache c = {(void*)0x10000, 1u << 30, 4, 16, 2, 64, VX_Q8_0, VX_Q8_0};
    k = in_of(5, 2, 64);
    auto write = [&](const int32_t* slots) { return vx_kv_write_rotated(ctx, nullptr, &c, &qo, &q, &k, &v, kPos, slots, &how); };
    CHECK(refused(write(nullptr), VX_ERR_INVALID));
    CHECK(refused(vx_kv_write_rotated(ctx, nullptr, &c, &qo, nullptr, &k, &v, kPos, kPos, &how), VX_ERR_INVALID));
    CHECK(refused(vx_kv_write_rotated(ctx, nullptr, &c, &qo, &q, nullptr, &v, kPos, kPos, &how), VX_ERR_INVALID));
    CHECK(refused(vx_kv_write_rotated(ctx, nullptr, &c, &qo, &q, &k, &v, nullptr, kPos, &how), VX_ERR_INVALID));
    CHECK(refused(vx_kv_write_rotated(ctx, nullptr, nullptr, &qo, &q, &k, &v, kPos, kPos, &how), VX_ERR_INVALID));
    q = in_of(4, 8, 64), qo = out_of(4, 8, 64);
    CHECK(refused(write(kPos), VX_ERR_SHAPE));
    q = in_of(5, 8, 96), qo = out_of(5, 8, 96);
    CHECK(refused(write(kPos), VX_ERR_SHAPE));
    for (uint32_t dim : {64u, 96u, 128u, 256u})
        for (uint32_t kt : {(uint32_t)VX_Q8_0, (uint32_t)VX_Q4_0})
            for (uint32_t vt : {(uint32_t)VX_Q8_0, (uint32_t)VX_Q4_0}) {
                c.dim = dim, c.k_type = kt, c.v_type = vt;
                q = in_of(5, 8, dim), qo = out_of(5, 8, dim), k = in_of(5, 2, dim), v = in_of(5, 2, dim);
                CHECK(write(kPos) == VX_OK && launches == 1);
                CHECK(vx_kv_write_rotated(ctx, nullptr, &c, nullptr, nullptr, &k, &v, kPos, kPos, &how) == VX_OK && launches == 2);
                k.layout.stride[0] += 1;  // rows that are not aligned
                CHECK(write(kPos) == VX_OK && launches == 3);
                q = in_of(9000, 8, dim), qo = out_of(9000, 8, dim), k = in_of(9000, 2, dim), v = in_of(9000, 2, dim);
                CHECK(write(kPos) == VX_OK && launches == 5);  // many: keys and values, then queries
                CHECK(vx_kv_write_rotated(ctx, nullptr, &c, nullptr, nullptr, &k, &v, kPos, kPos, &how) == VX_OK && launches == 6);
                k.layout.stride[0] += 1;
                CHECK(write(kPos) == VX_OK && launches == 7);
                launches = 0;
            }
    // ---- pages
    int32_t* at = (int32_t*)0x4000;
    vx_kv_pages p = {at, at, at, at, 3, 8, 8, 16, 100, 0};
    auto resize = [&](const vx_kv_pages& x, uint32_t tokens) { return vx_kv_resize(ctx, nullptr, &x, at, at, at, at, tokens); };
    auto pages = [&](auto change) {
        vx_kv_pages x = p;
        change(x);
        return resize(x, 10);
    };
    CHECK(refused(vx_kv_resize(nullptr, nullptr, &p, at, at, at, at, 10), VX_ERR_INVALID));
    CHECK(refused(vx_kv_resize(ctx, nullptr, nullptr, at, at, at, at, 10), VX_ERR_INVALID));
    CHECK(refused(vx_kv_resize(ctx, nullptr, &p, nullptr, at, at, at, 10), VX_ERR_INVALID));
    CHECK(refused(vx_kv_resize(ctx, nullptr, &p, at, nullptr, at, at, 10), VX_ERR_INVALID));
    CHECK(refused(vx_kv_resize(ctx, nullptr, &p, at, at, nullptr, at, 10), VX_ERR_INVALID));
    CHECK(refused(vx_kv_resize(ctx, nullptr, &p, at, at, at, nullptr, 10), VX_ERR_INVALID));
    CHECK(refused(vx_kv_resize(ctx, nullptr, &p, (int32_t*)0x4001, at, at, at, 10), VX_ERR_INVALID));
    CHECK(refused(resize(p, (1u << 30) + 1), VX_ERR_UNSUPPORTED));
    CHECK(refused(pages([](vx_kv_pages& x) { x.reserved = 1; }), VX_ERR_INVALID));
    CHECK(refused(pages([](vx_kv_pages& x) { x.page_tokens = 24; }), VX_ERR_UNSUPPORTED));
    CHECK(refused(pages([](vx_kv_pages& x) { x.page_tokens = 8; }), VX_ERR_UNSUPPORTED));
    CHECK(refused(pages([](vx_kv_pages& x) { x.pages = (1u << 27) + 1; }), VX_ERR_UNSUPPORTED));
    CHECK(refused(pages([](vx_kv_pages& x) { x.table_stride = 7; }), VX_ERR_INVALID));
    CHECK(refused(pages([](vx_kv_pages& x) { x.table = nullptr; }), VX_ERR_INVALID));
    CHECK(refused(pages([](vx_kv_pages& x) { x.lens = nullptr; }), VX_ERR_INVALID));
    CHECK(refused(pages([](vx_kv_pages& x) { x.free_pages = nullptr; }), VX_ERR_INVALID));
    CHECK(refused(pages([](vx_kv_pages& x) { x.free_count = nullptr; }), VX_ERR_INVALID));
    CHECK(refused(pages([](vx_kv_pages& x) { x.seqs = 1u << 16, x.table_cols = x.table_stride = 1u << 15; }), VX_ERR_UNSUPPORTED));
    CHECK(resize(p, 0) == VX_OK && launches == 1);
    CHECK(resize(p, 100000) == VX_OK && launches == 3);
    p.seqs = 0, p.table = p.lens = nullptr;
    CHECK(resize(p, 10) == VX_OK && launches == 4);
    for (const auto& e : names)
        for (const char* n : {"vx_pages", "vx_rotate"})
            if (!e.first.compare(0, std::strlen(n), n) && !launched.count(e.second)) std::printf("%s is never launched\n", e.first.c_str()), ++failures;
    CHECK(loads[vx_co_step] == 1 && vx_destroy(ctx) == VX_OK);
    if (!failures) std::printf("fine\n");
    return failures != 0;
}
