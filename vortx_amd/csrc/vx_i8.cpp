// vx_i8.cpp — host side of the products of 8-bit integers: checks and kernel choice.
#include <algorithm>

#include "vx_internal.hpp"
#include "vx_kargs.h"

namespace vx {

// Sums of K products of up to 128^2 stay within 31 bits.
constexpr uint32_t VX_I8_MOST_COLS = 131071;

static int check_rows(const vx_i8_rows* r) {
    if (!r) return fail(VX_ERR_INVALID, "null rows");
    if (r->row_stride_bytes < r->cols) return fail(VX_ERR_INVALID, "row_stride_bytes smaller than a row");
    if ((uintptr_t)r->base & 15u || r->row_stride_bytes % 16) return fail(VX_ERR_UNSUPPORTED, "rows of 8-bit integers are 16-byte aligned");
    if ((uintptr_t)r->scales & 3u) return fail(VX_ERR_INVALID, "scales is not 4-byte aligned");
    if (r->rows && (!r->scales || (r->cols && !r->base))) return fail(VX_ERR_INVALID, "null base or scales");
    return VX_OK;
}

// A [rows, cols] view of f32.
struct Matrix {
    uintptr_t ptr;
    uint32_t rows, cols;
    int64_t stride[2];
    bool vec;  // stride 1 along a row, 16-byte aligned rows
};
static int matrix_view(const void* base, const vx_layout* l, Matrix* m, const char* name, bool written) {
    Canon c;
    const int s = canon_view(base, l, &c, name);
    if (s) return s;
    if (c.l.size[0] != 1 || c.l.size[1] != 1) return fail(VX_ERR_SHAPE, "a view of rank 2 is expected");
    m->ptr = c.ptr;
    m->rows = c.l.size[2];
    m->cols = c.l.size[3];
    m->stride[0] = c.l.stride[2];
    m->stride[1] = c.l.stride[3];
    if (written)
        for (int i = 0; i < 2; ++i)
            if (c.l.size[i + 2] > 1 && m->stride[i] == 0) return fail(VX_ERR_INVALID, "a written view has a zero stride on a dimension of size > 1");
    m->vec = m->stride[1] == 1 && (c.ptr & 15u) == 0 && (m->rows == 1 || m->stride[0] % 4 == 0);
    return VX_OK;
}

static int quantize(vx_ctx ctx, vx_stream stream, const vx_i8_rows* out, const Matrix& x) {
    if (!out->rows) return VX_OK;
    vx_i8_quant_args a{};
    a.x = (const float*)x.ptr;
    a.xs[0] = x.stride[0];
    a.xs[1] = x.stride[1];
    a.out = (int8_t*)out->base;
    a.row_stride = out->row_stride_bytes;
    a.scales = out->scales;
    a.rows = out->rows;
    a.cols = out->cols;
    // rows of up to 4096 stay in 16 registers a thread; longer ones, where there are few, with 1024 threads, or in 64 registers
    const bool few = out->rows <= 2u * ctx_cus(ctx);
    const int k = !x.vec ? K_vx_i8_quantize_any : out->cols <= 4096 ? K_vx_i8_quantize_c4 : few ? K_vx_i8_quantize_long : K_vx_i8_quantize_c16;
    return launch_struct(ctx, k, std::min(out->rows, 1u << 20), k == K_vx_i8_quantize_long ? 1024 : 256, stream, &a);
}

static uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// x that a product quantizes itself (one launch, each workgroup for itself): one token of up to 65536 values, or up to
// four whose values stay in the workgroup's registers, 16 a thread (4096 values and up to four tokens, 8192 and two). By
// itself / by a launch before it, in a graph, us: 11008 x 4096, two tokens 12.6 / 14.5, four 15.9 / 14.8 (gated 19.6 / 22.4
// and 22.4 / 22.7); 4096 x 4096, two 7.9 / 8.6, three 9.2 / 8.5, four 9.9 / 8.7; 4096 x 11008, four 21.7 / 16.5. Three and
// four stay with it although one launch more takes them 1 us less: they need no workspace.
static bool own_x(uint32_t T, uint32_t K) {
    const uint64_t fours = (K + 4095ull) / 4096;
    return T == 1 ? fours <= 16 : T <= VX_I8_OWN_TOKENS && fours * T <= 4;
}

// x's rows and their scales, and behind them sums of parts of K (plan_gemm): 512 workgroups' tiles of 128 by 128. (Never less
// for more tokens or columns: a workspace is for up to so many.)
static uint64_t rows_bytes(uint32_t T, uint32_t K) { return own_x(T, K) ? 0 : up(K, 128) * T + up(4ull * T, 16); }
constexpr uint32_t VX_I8_PARTS_COLS = 1024;
static uint64_t parts_bytes(uint32_t T, uint32_t K) {
    return T <= 16 || K < VX_I8_PARTS_COLS ? 0 : std::min(T, 128u) * (512ull * 128 * 4);
}
static uint64_t ws_bytes(uint32_t T, uint32_t K) {
    K = std::min(K, VX_I8_MOST_COLS);  // (no product has more; sums of both ends would pass 64 bits)
    return rows_bytes(T, K) + parts_bytes(T, K);
}

struct I8Plan {
    int kernel;
    uint32_t tokens, channels;  // of a workgroup
    uint32_t block, lds, grid;  // grid: most workgroups, each then has several tiles (0: one each)
    uint32_t split, chunk;
};
// What a kernel takes is close to what a CU has to load, the rows of x and of the weights of all its workgroups, at
// some 37 GB/s from L2 (the kernels that go over tiles at 47, where the matrix cores are as long). Us, at 4096 columns:
//   128 x 4096 (N)   direct 96 rows 14.7   tiles of 128 256 rows 27     64 x 11008   direct 128 rows 22.3   tiles 256 rows 27
//   128 x 11008      direct 256 39.0       tiles 256 28.7             200 x 11008   direct 384 51.4        tiles 256 28.5
//   200 x 4096, 11008 columns: direct 128 42.1, tiles 256 61.2;  64 x 11008 gated: direct 256 41.6, tiles 256 31.5
// so that the least of them is taken, and of two the same the tiles of 128.
static I8Plan plan_gemm(int num_cus, const vx_i8_args& a, bool gated) {
    const int g = gated ? 1 : 0;
    const uint32_t both = gated ? 2 : 1;
    if (a.xf) {
        // a workgroup a CU; waves share rows where there are fewer of them than waves, 4096 bytes a step
        const uint32_t waves = (uint32_t)num_cus * 16;
        uint32_t split = 1;
        while (split < 16 && (uint64_t)a.N * split * 2 <= waves && split * 4096u < a.K) split *= 2;
        const uint32_t per = 16 / split, grid = std::min((uint32_t)num_cus, (a.N - 1) / per + 1);
        return {K_vx_i8_stream_t1 + 2 * (a.T > 2 ? 2 : (int)a.T - 1) + g, a.T, (a.N - 1) / grid + 1, 1024, a.x_bytes + 1024u, 0, split, 0};
    }
    struct Kernel { int kernel; uint32_t tokens, channels[2], block, at_once; };  // at_once: 0, or workgroups a CU that have several tiles
    static const Kernel kKernels[6] = {{K_vx_i8_direct_t1, 16, {16, 16}, 512, 0}, {K_vx_i8_direct_t2, 32, {32, 16}, 512, 0},
                                       {K_vx_i8_direct_t4, 64, {32, 16}, 512, 0}, {K_vx_i8_direct_t4_wide, 64, {64, 32}, 512, 0},
                                       {K_vx_i8_tile128, 128, {128, 64}, 256, 2}, {K_vx_i8_tile256, 256, {256, 128}, 512, 1}};
    auto cost = [&](const Kernel& k) {
        const uint64_t groups = (uint64_t)((a.T - 1) / k.tokens + 1) * ((a.N - 1) / k.channels[g] + 1);
        return (groups + num_cus - 1) / num_cus * (k.tokens + k.channels[g] * both);
    };
    const bool near = a.xs < (1u << 24) && a.ws[0] < (1u << 24) && a.ws[1] < (1u << 24);  // a tile's rows within 32 bits
    int best = a.T <= 16 ? 0 : a.T <= 32 ? 1 : 2;
    if (best == 2) {
        for (int i = 3; i < (near ? 6 : 4); ++i)
            if (cost(kKernels[i]) < cost(kKernels[best]) + (i == 4)) best = i;  // (of two the same: 512 x 11008 tiles of 128 50.8, of 256 59.2)
    }
    if (a.parts && near) {
        // Tiles of 128 over parts of K and a launch that joins their sums, against all of K: in bytes that a CU has to load,
        // where sums go to memory and back at half a CU's share of its rate and a launch takes as long as 150 KB.
        // With / without, x quantized before, us: 100 x 4096 by 11008 columns 25.5 / 36.3, 64 tokens 22.4 / 38, 256 34 / 52, 32
        // 20.8 / 27; where a part is not worth it (64 x 4096 by 4096 columns, 17.5) nothing changes.
        const uint64_t tiles = ((a.T - 1) / 128 + 1ull) * ((a.N - 1) / kKernels[4].channels[g] + 1), stages = (a.K + 127) / 128;
        uint64_t least = cost(kKernels[best]) * a.K;
        uint32_t parts = 0, chunk = 0;
        for (uint32_t n = 2; n <= 16 && tiles * n <= 2ull * num_cus && stages >= 4ull * n; ++n) {
            const uint64_t each = (stages + n - 1) / n * 128;
            if ((n - 1) * each >= a.K || n * (uint64_t)both * a.T * up(a.N, 4) * 4 > parts_bytes(a.T, a.K)) continue;
            const uint64_t bytes = (tiles * n + num_cus - 1) / num_cus * 256 * each + 16ull * n * both * a.T * a.N / num_cus + 150000;
            if (bytes < least) least = bytes, parts = n, chunk = (uint32_t)each;
        }
        if (parts) return {K_vx_i8_part128 + g, 128, kKernels[4].channels[g], 256, 0, 0, parts, chunk};
    }
    const Kernel& k = kKernels[best];
    const uint32_t fragments = k.tokens / 16 * (k.channels[g] / 16);  // (whose sums meet in LDS, eight products' at a time)
    return {k.kernel + g, k.tokens, k.channels[g], k.block, k.at_once ? 0u : std::min(fragments, gated ? 4u : 8u) * both * 8192u,
            (uint32_t)num_cus * k.at_once, 1, 0};
}

static int run_gemm(vx_ctx ctx, vx_stream stream, const vx_mview* out, const vx_i8_rows* xq, const vx_cview* xf, const vx_i8_rows* w,
                    const vx_i8_rows* up_w, uint32_t act, void* ws, uint64_t ws_size) {
    clear_error();
    if (!ctx) return fail(VX_ERR_INVALID, "null ctx");
    if (!out || (!xq && !xf)) return fail(VX_ERR_INVALID, "null view");
    Matrix o, x{};
    int s = matrix_view(out->base, &out->layout, &o, "out", true);
    if (s) return s;
    if ((s = check_rows(w)) || (up_w && (s = check_rows(up_w)))) return s;
    if (xq) {
        if ((s = check_rows(xq))) return s;
        x.rows = xq->rows;
        x.cols = xq->cols;
    } else if ((s = matrix_view(xf->base, &xf->layout, &x, "x", false))) {
        return s;
    }
    if (act > VX_ACT_RELU) return fail(VX_ERR_INVALID, "unknown activation");
    if (x.cols != w->cols || o.rows != x.rows || o.cols != w->rows || (up_w && (up_w->rows != w->rows || up_w->cols != w->cols)))
        return fail(VX_ERR_SHAPE, "incompatible shapes: out [T, N], x [T, K], weights [N, K]");
    if (w->cols == 0) return fail(VX_ERR_UNSUPPORTED, "rows of no columns");
    if (w->cols > VX_I8_MOST_COLS) return fail(VX_ERR_UNSUPPORTED, "more than 131071 columns");
    if ((uintptr_t)ws & 15u) return fail(VX_ERR_INVALID, "workspace is not 16-byte aligned");
    vx_i8_args a{};
    a.T = x.rows;
    a.N = w->rows;
    a.K = w->cols;
    if (xf && ws_size < ws_bytes(a.T, a.K)) return fail(VX_ERR_INVALID, "workspace smaller than vx_gemm_i8_ws_size");
    if (xf && ws_bytes(a.T, a.K) && !ws) return fail(VX_ERR_INVALID, "null workspace");
    if (a.T == 0 || a.N == 0) return VX_OK;
    const bool gated = up_w != nullptr;
    const vx_i8_rows* ws2[2] = {w, gated ? up_w : w};
    for (int i = 0; i < 2; ++i) {
        a.w[i] = (const int8_t*)ws2[i]->base;
        a.ws[i] = ws2[i]->row_stride_bytes;
        a.wscale[i] = ws2[i]->scales;
    }
    a.out = (float*)o.ptr;
    a.os[0] = o.stride[0];
    a.os[1] = o.stride[1];
    a.out_vec = o.vec;
    a.act = act;
    const bool own = xf && own_x(a.T, a.K);
    vx_i8_rows rows;
    if (xf && !own) {
        const uint64_t stride = up(a.K, 128);
        rows = vx_i8_rows{ws, (float*)((char*)ws + stride * a.T), stride, a.T, a.K};
        if (parts_bytes(a.T, a.K)) a.parts = (int32_t*)((char*)ws + rows_bytes(a.T, a.K));
        xq = &rows;
    }
    if (own) {
        a.xf = (const float*)x.ptr;
        a.xfs[0] = x.stride[0];
        a.xfs[1] = x.stride[1];
        a.xf_vec = x.vec;
        a.pitch = (uint32_t)up(a.K, 4096);
        const uint32_t rows_there = a.T == 3 ? 4 : a.T;  // (a kernel for four reads a fourth, and makes nothing of it)
        a.x_bytes = (uint32_t)up(rows_there * (uint64_t)a.pitch + VX_I8_OWN_TOKENS * (16 * 4 + 4), 16);
    } else {
        a.x = (const int8_t*)xq->base;
        a.xs = xq->row_stride_bytes;
        a.xscale = xq->scales;
    }
    const I8Plan p = plan_gemm(ctx_cus(ctx), a, gated);
    a.tiles_t = (a.T - 1) / p.tokens + 1;
    a.tiles_n = (a.N - 1) / p.channels + 1;
    a.split = p.split;
    a.chunk = p.chunk;
    if (a.N >= (1u << 31) || (uint64_t)a.tiles_t * a.tiles_n >= (1u << 22)) return fail(VX_ERR_UNSUPPORTED, "too many outputs (split the call)");
    if (xf && !own && (s = quantize(ctx, stream, &rows, x))) return s;
    const uint32_t tiles = a.tiles_t * a.tiles_n * (p.chunk ? p.split : 1u);
    if (p.chunk) {
        if ((s = launch_struct(ctx, p.kernel, tiles, p.block, stream, &a))) return s;
        return launch_struct(ctx, K_vx_i8_join + (gated ? 1 : 0), (uint32_t)((a.T * up(a.N, 4) / 4 + 255) / 256), 256, stream, &a);
    }
    return launch_struct(ctx, p.kernel, p.grid ? std::min(tiles, p.grid) : tiles, p.block, stream, &a, p.lds);
}

}  // namespace vx

extern "C" {

int vx_i8_quantize(vx_ctx ctx, vx_stream stream, const vx_i8_rows* out, const vx_cview* x) {
    vx::clear_error();
    if (!ctx) return vx::fail(VX_ERR_INVALID, "null ctx");
    if (!x) return vx::fail(VX_ERR_INVALID, "null view");
    vx::Matrix m;
    int s = vx::check_rows(out);
    if (s) return s;
    if ((s = vx::matrix_view(x->base, &x->layout, &m, "x", false))) return s;
    if (m.rows != out->rows || m.cols != out->cols) return vx::fail(VX_ERR_SHAPE, "x and out have different shapes");
    // (the kernels' counters go on to a step past a row's end, in 32 bits)
    if (m.cols > 0x7FFFFFFFu) return vx::fail(VX_ERR_UNSUPPORTED, "rows of 2^31 columns and more");
    return vx::quantize(ctx, stream, out, m);
}

int vx_gemm_i8_ws_size(uint32_t tokens, uint32_t cols, uint64_t* bytes) {
    vx::clear_error();
    if (!bytes) return vx::fail(VX_ERR_INVALID, "null bytes");
    *bytes = vx::ws_bytes(tokens, cols);
    return VX_OK;
}

int vx_gemm_i8(vx_ctx ctx, vx_stream stream, const vx_mview* out, const vx_i8_rows* x, const vx_i8_rows* w) {
    return vx::run_gemm(ctx, stream, out, x, nullptr, w, nullptr, 0, nullptr, 0);
}

int vx_gemm_i8_x(vx_ctx ctx, vx_stream stream, const vx_mview* out, const vx_cview* x, const vx_i8_rows* w, void* workspace,
                 uint64_t workspace_bytes) {
    return vx::run_gemm(ctx, stream, out, nullptr, x, w, nullptr, 0, workspace, workspace_bytes);
}

int vx_gemm_i8_gated(vx_ctx ctx, vx_stream stream, const vx_mview* out, const vx_i8_rows* x, const vx_i8_rows* gate,
                     const vx_i8_rows* up, uint32_t act) {
    if (!up) return vx::clear_error(), vx::fail(VX_ERR_INVALID, "null rows");
    return vx::run_gemm(ctx, stream, out, x, nullptr, gate, up, act, nullptr, 0);
}

int vx_gemm_i8_gated_x(vx_ctx ctx, vx_stream stream, const vx_mview* out, const vx_cview* x, const vx_i8_rows* gate,
                       const vx_i8_rows* up, uint32_t act, void* workspace, uint64_t workspace_bytes) {
    if (!up) return vx::clear_error(), vx::fail(VX_ERR_INVALID, "null rows");
    return vx::run_gemm(ctx, stream, out, nullptr, x, gate, up, act, workspace, workspace_bytes);
}

}  // extern "C"
