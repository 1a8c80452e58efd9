// Which batches attention takes by their number of query rows, on a HIP runtime
// that only counts.
#include "hip_counts.hpp"

int main() {
    vx_ctx ctx = nullptr;
    CHECK(vx_init(0, &ctx) == VX_OK);
    const uint32_t heads = 4;
    const vx_kv_cache c = {(void*)0x10000, 1u << 30, 4, 16, heads, 64, VX_Q8_0, VX_Q8_0};
    struct { uint32_t seqs, queries, group; bool fine; } cases[] = {
        {1, 1, 1, true}, {1, (1u << 22) - 1, 1, true}, {1, 1u << 22, 1, false}, {(1u << 22) - 1, 1, 1, false},
        {1u << 20, 1, 2, true}, {1u << 20, 2, 2, false},
        // products that 64 bits do not hold
        {0x80000000u, 0x80000000u, 4, false}, {0x80000000u, 0x80000000u, 1, false}, {0x40000000u, 0x40000000u, 16, false},
        {1u << 10, 1u << 31, 1u << 29, false}, {1u << 30, 1u << 31, 1u << 9, false}, {1u << 31, 1u << 31, 1u << 8, false},
        {0xFFFFFFFFu, 0xFFFFFFFFu, 0x3FFFFFFFu, false}};
    for (const auto& k : cases) {
        vx_attn_batch b = {};
        b.table = b.lens = b.starts = (const int32_t*)0x3000;
        b.seqs = k.seqs, b.table_cols = b.table_stride = 4, b.max_queries = k.queries, b.max_len = 64;
        uint64_t bytes = 0;
        const int s = vx_attention_ws_size(ctx, &c, &b, nullptr, 1, heads * k.group, &bytes);
        if (s != (k.fine ? VX_OK : VX_ERR_UNSUPPORTED))
            std::printf("%u sequences, %u queries, group %u: status %d, %llu bytes\n", k.seqs, k.queries, k.group, s, (unsigned long long)bytes), ++failures;
    }
    CHECK(vx_destroy(ctx) == VX_OK);
    if (!failures) std::printf("fine\n");
    return failures != 0;
}
