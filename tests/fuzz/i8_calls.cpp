// Products of 8-bit integers on a HIP runtime that only counts: bad calls are
// refused and launch nothing, and every kernel is reached by some good one.
#include "hip_counts.hpp"

extern "C" {
extern const unsigned char vx_co_i8[16];
const unsigned char vx_co_i8[16] = {};
}

static vx_layout matrix(uint32_t rows, uint32_t cols, uint32_t stride = 0) {
    vx_layout l = {};
    l.rank = 2;
    l.size[0] = rows, l.size[1] = cols;
    l.stride[0] = stride ? stride : cols, l.stride[1] = 1;
    return l;
}
static vx_i8_rows rows_of(uint32_t rows, uint32_t cols) { return {(void*)0x10000, (float*)0x20000, (cols + 15u) / 16u * 16u, rows, cols}; }
static int refused(int status, int want) {
    const bool ok = status == want && launches == 0 && *vx_last_error_message();
    launches = 0;
    return ok;
}

int main() {
    vx_ctx ctx = nullptr;
    CHECK(vx_init(0, &ctx) == VX_OK);
    void* ws = (void*)0x40000;
    const uint64_t enough = 1ull << 40;
    launches = 0;
    vx_i8_rows x = rows_of(5, 100), w = rows_of(40, 100), up = rows_of(40, 100);
    vx_mview o = {(float*)0x100000, matrix(5, 40)};
    vx_cview f = {(float*)0x200000, matrix(5, 100)};
    auto all = [&](int want) {  // every form of the call
        return refused(vx_gemm_i8(ctx, nullptr, &o, &x, &w), want) && refused(vx_gemm_i8_gated(ctx, nullptr, &o, &x, &w, &up, 0), want) &&
               refused(vx_gemm_i8_x(ctx, nullptr, &o, &f, &w, ws, enough), want) &&
               refused(vx_gemm_i8_gated_x(ctx, nullptr, &o, &f, &w, &up, 0, ws, enough), want);
    };
    CHECK(refused(vx_gemm_i8(nullptr, nullptr, &o, &x, &w), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8(ctx, nullptr, nullptr, &x, &w), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8(ctx, nullptr, &o, nullptr, &w), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8(ctx, nullptr, &o, &x, nullptr), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8_x(ctx, nullptr, &o, nullptr, &w, ws, enough), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8_gated(ctx, nullptr, &o, &x, &w, nullptr, 0), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8_gated_x(ctx, nullptr, &o, &f, &w, nullptr, 0, ws, enough), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8_gated(ctx, nullptr, &o, &x, &w, &up, 4), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8_x(ctx, nullptr, &o, &f, &w, nullptr, 0), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8_x(ctx, nullptr, &o, &f, &w, nullptr, enough), VX_ERR_INVALID));
    uint64_t bytes = 0;
    CHECK(vx_gemm_i8_ws_size(5, 100, &bytes) == VX_OK && bytes >= 5 * 104);
    CHECK(refused(vx_gemm_i8_x(ctx, nullptr, &o, &f, &w, ws, bytes - 1), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8_x(ctx, nullptr, &o, &f, &w, (void*)0x40008, bytes), VX_ERR_INVALID));
    CHECK(refused(vx_gemm_i8_ws_size(5, 100, nullptr), VX_ERR_INVALID));
    o.layout = matrix(4, 40);
    CHECK(all(VX_ERR_SHAPE));
    o.layout = matrix(5, 41);
    CHECK(all(VX_ERR_SHAPE));
    o.layout = matrix(5, 40);
    o.layout.stride[0] = 0;
    CHECK(all(VX_ERR_INVALID));
    o.layout = matrix(5, 40);
    o.base = nullptr;
    CHECK(all(VX_ERR_INVALID));
    o.base = (float*)0x100000;
    auto weights = [&](auto change, int want) {
        vx_i8_rows keep = w;
        change(w);
        const bool ok = all(want);
        w = keep;
        return ok;
    };
    CHECK(weights([](vx_i8_rows& r) { r.cols = 99; }, VX_ERR_SHAPE));
    CHECK(weights([](vx_i8_rows& r) { r.row_stride_bytes = 96; }, VX_ERR_INVALID));
    CHECK(weights([](vx_i8_rows& r) { r.row_stride_bytes = 104; }, VX_ERR_UNSUPPORTED));
    CHECK(weights([](vx_i8_rows& r) { r.base = (void*)0x10008; }, VX_ERR_UNSUPPORTED));
    CHECK(weights([](vx_i8_rows& r) { r.base = nullptr; }, VX_ERR_INVALID));
    CHECK(weights([](vx_i8_rows& r) { r.scales = nullptr; }, VX_ERR_INVALID));
    CHECK(weights([](vx_i8_rows& r) { r.scales = (float*)0x20002; }, VX_ERR_INVALID));
    up = rows_of(41, 100);
    CHECK(refused(vx_gemm_i8_gated(ctx, nullptr, &o, &x, &w, &up, 0), VX_ERR_SHAPE));
    up = rows_of(40, 116);
    CHECK(refused(vx_gemm_i8_gated(ctx, nullptr, &o, &x, &w, &up, 0), VX_ERR_SHAPE));
    for (uint32_t K : {0u, 131072u}) {
        x = rows_of(5, K), w = up = rows_of(40, K), f.layout = matrix(5, K);
        CHECK(all(VX_ERR_UNSUPPORTED));
    }
    // more outputs than a grid has workgroups
    x = rows_of(1u << 31, 16), w = up = rows_of(1u << 20, 16), o.layout = matrix(1u << 31, 1u << 20), f.layout = matrix(1u << 31, 16);
    CHECK(refused(vx_gemm_i8(ctx, nullptr, &o, &x, &w), VX_ERR_UNSUPPORTED));
    CHECK(refused(vx_gemm_i8_x(ctx, nullptr, &o, &f, &w, ws, enough), VX_ERR_UNSUPPORTED));
    x = rows_of(1, 16), w = up = rows_of(1u << 31, 16), o.layout = matrix(1, 1u << 31), f.layout = matrix(1, 16);
    CHECK(all(VX_ERR_UNSUPPORTED));
    x = rows_of(0, 16), w = up = rows_of(40, 16), o.layout = matrix(0, 40);
    CHECK(vx_gemm_i8(ctx, nullptr, &o, &x, &w) == VX_OK && vx_gemm_i8_gated(ctx, nullptr, &o, &x, &w, &up, 1) == VX_OK && launches == 0);
    // a workspace for so many tokens and columns does for fewer
    const uint32_t ts[] = {0, 1, 2, 4, 5, 16, 17, 127, 128, 129, 1024, 1025, 5000}, ks[] = {1, 100, 1023, 1024, 4096, 4097, 8192, 65536, 65537, 131071};
    for (size_t i = 0; i < 13; ++i)
        for (size_t j = 0; j < 10; ++j) {
            uint64_t here = 0, more = 0;
            CHECK(vx_gemm_i8_ws_size(ts[i], ks[j], &here) == VX_OK);
            if (i + 1 < 13) CHECK(vx_gemm_i8_ws_size(ts[i + 1], ks[j], &more) == VX_OK && more >= here);
            if (j + 1 < 10) CHECK(vx_gemm_i8_ws_size(ts[i], ks[j + 1], &more) == VX_OK && more >= here);
        }
    // quantizing
    w = rows_of(5, 100), f.layout = matrix(5, 100);
    CHECK(refused(vx_i8_quantize(nullptr, nullptr, &w, &f), VX_ERR_INVALID));
    CHECK(refused(vx_i8_quantize(ctx, nullptr, nullptr, &f), VX_ERR_INVALID));
    CHECK(refused(vx_i8_quantize(ctx, nullptr, &w, nullptr), VX_ERR_INVALID));
    w.row_stride_bytes = 104;
    CHECK(refused(vx_i8_quantize(ctx, nullptr, &w, &f), VX_ERR_UNSUPPORTED));
    w = rows_of(5, 99);
    CHECK(refused(vx_i8_quantize(ctx, nullptr, &w, &f), VX_ERR_SHAPE));
    f.layout.rank = 3;
    CHECK(refused(vx_i8_quantize(ctx, nullptr, &w, &f), VX_ERR_SHAPE));
    // every kernel
    for (uint32_t K : {100u, 5000u})
        for (uint32_t T : {1u, 2u, 3u, 5u, 16u, 17u, 40u, 70u, 100u, 130u, 200u, 300u, 600u, 3000u})
            for (uint32_t N : {40u, 500u, 2000u, 9000u})
                for (int vec = 0; vec < 2; ++vec) {
                    x = rows_of(T, K), w = up = rows_of(N, K), o.layout = matrix(T, N), f.layout = matrix(T, K, vec ? 0 : K + 1);
                    launches = 0;
                    CHECK(vx_gemm_i8(ctx, nullptr, &o, &x, &w) == VX_OK && launches == 1);
                    CHECK(vx_gemm_i8_gated(ctx, nullptr, &o, &x, &w, &up, 3) == VX_OK && launches == 2);
                    CHECK(vx_gemm_i8_ws_size(T, K, &bytes) == VX_OK);
                    for (int gated = 0; gated < 2; ++gated) {  // by itself, quantized before, or that and its parts joined after
                        launches = 0;
                        CHECK((gated ? vx_gemm_i8_gated_x(ctx, nullptr, &o, &f, &w, &up, 2, bytes ? ws : nullptr, bytes)
                                     : vx_gemm_i8_x(ctx, nullptr, &o, &f, &w, bytes ? ws : nullptr, bytes)) == VX_OK);
                        CHECK(bytes ? launches == 2 || (launches == 3 && T > 16 && K >= 1024) : launches == 1);
                    }
                }
    for (const auto& e : names)
        if (!e.first.compare(0, 5, "vx_i8") && !launched.count(e.second)) std::printf("%s is never launched\n", e.first.c_str()), ++failures;
    CHECK(loads[vx_co_i8] == 1 && vx_destroy(ctx) == VX_OK);
    if (!failures) std::printf("fine\n");
    return failures != 0;
}
