// The library's host code on a HIP runtime that only counts: which code objects
// are loaded when, by how many threads, and what is left at the end.
#include "hip_counts.hpp"

static int total() {
    int n = 0;
    for (auto& e : loads) n += e.second;
    return n;
}
static vx_kv_cache cache_of(uint32_t dim) {
    vx_kv_cache c = {(void*)0x10000, 1u << 30, 4, 16, 2, dim, VX_Q8_0, VX_Q8_0};
    return c;
}
static vx_layout rows_of(uint32_t dim, uint32_t heads) {
    vx_layout l = {};
    l.rank = 3;
    l.size[0] = 3, l.size[1] = heads, l.size[2] = dim;
    l.stride[0] = heads * dim, l.stride[1] = dim, l.stride[2] = 1;
    return l;
}
static int write(vx_ctx ctx, uint32_t dim) {
    const vx_kv_cache c = cache_of(dim);
    const vx_cview v = {(float*)0x100000, rows_of(dim, 2)};
    return vx_kv_write(ctx, nullptr, &c, &v, &v, (const int32_t*)0x2000);
}
static vx_attn_batch batch_of() {
    vx_attn_batch b = {};
    b.table = b.lens = b.starts = (const int32_t*)0x3000;
    b.seqs = 1, b.table_cols = b.table_stride = 4, b.max_queries = 3, b.max_len = 64;
    return b;
}
static int attend(vx_ctx ctx, uint32_t dim, void* ws, uint64_t bytes) {
    const vx_kv_cache c = cache_of(dim);
    const vx_cview q = {(float*)0x100000, rows_of(dim, 4)};
    const vx_mview o = {(float*)0x200000, rows_of(dim, 4)};
    const vx_attn_batch b = batch_of();
    return vx_attention(ctx, nullptr, &o, &q, &c, &b, nullptr, ws, bytes);
}

int main() {
    vx_ctx ctx = nullptr;
    CHECK(vx_init(0, &ctx) == VX_OK);
    CHECK(total() == 6 && live == 6);  // none of the attention's
    CHECK(write(ctx, 64) == VX_OK && total() == 7 && loads[vx_co_attn_d64] == 1 && launches == 1);
    CHECK(write(ctx, 64) == VX_OK && attend(ctx, 64, nullptr, 0) == VX_OK && total() == 7);
    const vx_kv_cache c = cache_of(128);
    const vx_attn_batch b = batch_of();
    uint64_t bytes = 0;
    CHECK(vx_attention_ws_size(ctx, &c, &b, nullptr, 3, 4, &bytes) == VX_OK && bytes && total() == 8);  // the plan loads
    CHECK(attend(ctx, 128, (void*)0x4000, bytes) == VX_OK && total() == 8 && launches == 5);              // (attention and its join)
    // a head size whose code is not there: an error, nothing launched, nothing left, and another try later
    const int before = live, launched = launches;
    fail_after = 7;
    CHECK(write(ctx, 96) == VX_ERR_NO_CODE_OBJECT && live == before && launches == launched);
    CHECK(std::strstr(vx_last_error_message(), "d96"));
    CHECK(write(ctx, 96) == VX_OK && live == before + 1);
    // the first use within a capture that allows stream work only
    strict = 1;
    CHECK(write(ctx, 256) == VX_OK && capture == hipStreamCaptureModeGlobal);
    strict = 0;
    CHECK(live == 10);
    // they are all contexts' of the device, and stay
    vx_ctx other = nullptr;
    CHECK(vx_init(0, &other) == VX_OK && live == 16);
    CHECK(write(other, 64) == VX_OK && write(other, 256) == VX_OK && attend(other, 128, nullptr, 0) == VX_OK && live == 16);
    CHECK(vx_destroy(other) == VX_OK && vx_destroy(ctx) == VX_OK && live == 4);
    CHECK(vx_init(0, &ctx) == VX_OK && live == 10);
    CHECK(write(ctx, 64) == VX_OK && live == 10);
    CHECK(vx_destroy(ctx) == VX_OK && live == 4);
    // threads whose first use is the same, each with a context of its own and all with one: another device
    live = launches = 0;
    loads.clear();
    CHECK(vx_init(1, &ctx) == VX_OK && total() == 6);
    std::vector<std::thread> threads;
    std::atomic<int> bad{0};
    for (int i = 0; i < 16; ++i)
        threads.emplace_back([&, i] {
            vx_ctx own = nullptr;
            bad += vx_init(1, &own) != VX_OK;
            for (int j = 0; j < 50; ++j) bad += write(j % 2 ? own : ctx, i % 2 ? 64 : 256) != VX_OK;
            bad += vx_destroy(own) != VX_OK;
        });
    for (auto& t : threads) t.join();
    CHECK(!bad && loads[vx_co_attn_d64] == 1 && loads[vx_co_attn_d256] == 1 && !loads[vx_co_attn_d128] && launches == 800);
    CHECK(vx_destroy(ctx) == VX_OK && live == 2);
    if (!failures) std::printf("fine\n");
    return failures != 0;
}
