// How many workgroups the library launches for rows into the cache, on a HIP
// runtime that only counts: up to the most tokens that a view can have.
#include "hip_counts.hpp"

int main() {
    vx_ctx ctx = nullptr;
    CHECK(vx_init(0, &ctx) == VX_OK);
    const vx_kv_cache c = {(void*)0x10000, 1u << 30, 4, 16, 1, 64, VX_Q8_0, VX_Q8_0};
    for (uint32_t tokens : {1u, 255u, 256u, 257u, 1000u, 0x7FFFFFFFu, 0x80000000u, 0xFFFFFFFCu, 0xFFFFFFFDu, 0xFFFFFFFFu}) {
        vx_layout l = {};
        l.rank = 3;
        l.size[0] = tokens, l.size[1] = 1, l.size[2] = 64;
        l.stride[2] = 1;  // the same row for every token
        const vx_cview v = {(float*)0x100000, l};
        const int before = launches;
        CHECK(vx_kv_write(ctx, nullptr, &c, &v, &v, (const int32_t*)0x2000) == VX_OK);
        // a group of tokens (one, or four from 256 on) is 2 of a workgroup's 32 units; the grid ends at 2^20
        const uint64_t groups = tokens < 256 ? tokens : (tokens + 3ull) / 4, need = (groups * 2 + 31) / 32;
        if (launches != before + 1 || last_grid != (need < (1u << 20) ? need : 1u << 20))
            std::printf("%u tokens: %d launches, grid %u\n", tokens, launches - before, last_grid), ++failures;
    }
    CHECK(vx_destroy(ctx) == VX_OK);
    if (!failures) std::printf("fine\n");
    return failures != 0;
}
