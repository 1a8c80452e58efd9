// Rows of 8-bit integers at the ends of their ranges, on a HIP runtime that only counts.
#include "hip_counts.hpp"

extern "C" {
extern const unsigned char vx_co_i8[16];
const unsigned char vx_co_i8[16] = {};
}

int main() {
    vx_ctx ctx = nullptr;
    CHECK(vx_init(0, &ctx) == VX_OK);
    // The quantizing kernels count a row's columns, and one step past them, in 32 bits. (One value, broadcast: no memory is needed.)
    for (uint32_t rows : {0u, 1u, 1000u})
        for (uint32_t cols : {0x7FFFFFFFu, 0x80000000u, 0xFFFFF000u, 0xFFFFFFF0u, 0xFFFFFFFFu})
            for (uint32_t along : {0u, 1u}) {
                const vx_i8_rows out = {(void*)0x10000, (float*)0x20000, 1ull << 32, rows, cols};
                vx_cview x = {(float*)0x200000, {}};
                x.layout.rank = 2;
                x.layout.size[0] = rows, x.layout.size[1] = cols;
                x.layout.stride[1] = along;
                launches = 0;
                const int s = vx_i8_quantize(ctx, nullptr, &out, &x);
                CHECK(cols > 0x7FFFFFFFu ? s == VX_ERR_UNSUPPORTED && launches == 0 && *vx_last_error_message() : s == VX_OK && launches == (rows ? 1 : 0));
            }
    // A workspace for so many tokens and columns does for fewer, to the ends of both.
    const uint32_t ends[] = {1, 4, 17, 128, 131071, 131072, 1u << 20, 0x7FFFFFFFu, 0xFFFFFF7Fu, 0xFFFFFF81u, 0xFFFFFFFFu};
    for (size_t i = 0; i < 11; ++i)
        for (size_t j = 0; j < 11; ++j) {
            uint64_t here = 0, more = 0;
            CHECK(vx_gemm_i8_ws_size(ends[i], ends[j], &here) == VX_OK);
            if (i + 1 < 11) {
                CHECK(vx_gemm_i8_ws_size(ends[i + 1], ends[j], &more) == VX_OK && more >= here);
            }
            if (j + 1 < 11) {
                CHECK(vx_gemm_i8_ws_size(ends[i], ends[j + 1], &more) == VX_OK && more >= here);
            }
        }
    CHECK(vx_destroy(ctx) == VX_OK);
    if (!failures) std::printf("fine\n");
    return failures != 0;
}
