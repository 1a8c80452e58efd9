// Every kernel of the cache and its attention is reached by some call, on a HIP
// runtime that only counts.
#include "hip_counts.hpp"

static vx_layout rows_of(uint32_t tokens, uint32_t heads, uint32_t dim) {
    vx_layout l = {};
    l.rank = 3;
    l.size[0] = tokens, l.size[1] = heads, l.size[2] = dim;
    l.stride[0] = heads * dim, l.stride[1] = dim, l.stride[2] = 1;
    return l;
}

int main() {
    vx_ctx ctx = nullptr;
    CHECK(vx_init(0, &ctx) == VX_OK);
    for (uint32_t dim : {64u, 96u, 128u, 256u})
        for (uint32_t kt : {(uint32_t)VX_Q8_0, (uint32_t)VX_Q4_0})
            for (uint32_t vt : {(uint32_t)VX_Q8_0, (uint32_t)VX_Q4_0}) {
                const vx_kv_cache c = {(void*)0x10000, 1u << 30, 64, 64, 8, dim, kt, vt};
                const vx_cview rows = {(float*)0x100000, rows_of(3, 8, dim)};
                const vx_mview back = {(float*)0x100000, rows_of(3, 8, dim)};
                CHECK(vx_kv_write(ctx, nullptr, &c, &rows, &rows, (const int32_t*)0x2000) == VX_OK);
                CHECK(vx_kv_read(ctx, nullptr, &back, &back, &c, (const int32_t*)0x2000) == VX_OK);
                for (uint32_t seqs : {1u, 100u})
                    for (uint32_t queries : {1u, 16u, 33u, 100u, 500u, 2000u})
                        for (bool space : {true, false}) {
                            const uint32_t tokens = seqs * queries;
                            const vx_cview q = {(float*)0x100000, rows_of(tokens, 32, dim)};
                            const vx_mview o = {(float*)0x200000, rows_of(tokens, 32, dim)};
                            vx_attn_batch b = {};
                            b.table = b.lens = b.starts = (const int32_t*)0x3000;
                            b.seqs = seqs, b.table_cols = b.table_stride = 64, b.max_queries = queries, b.max_len = 4096;
                            uint64_t bytes = 0;
                            CHECK(vx_attention_ws_size(ctx, &c, &b, nullptr, tokens, 32, &bytes) == VX_OK);
                            CHECK(vx_attention(ctx, nullptr, &o, &q, &c, &b, nullptr, space ? (void*)0x4000 : nullptr, space ? bytes : 0) == VX_OK);
                        }
            }
    int all = 0;
    for (const auto& e : names) {
        if (e.first.compare(0, 7, "vx_attn") && e.first.compare(0, 5, "vx_kv")) continue;
        ++all;
        if (!launched.count(e.second)) std::printf("%s is never launched\n", e.first.c_str()), ++failures;
    }
    CHECK(all > 0);
    CHECK(vx_destroy(ctx) == VX_OK);
    if (!failures) std::printf("fine\n");
    return failures != 0;
}
