// Rotation of very many heads and tokens, on a HIP runtime that only counts.
#include "hip_counts.hpp"

extern "C" {
extern const unsigned char vx_co_step[16];
const unsigned char vx_co_step[16] = {};
}

int main() {
    vx_ctx ctx = nullptr;
    CHECK(vx_init(0, &ctx) == VX_OK);
    // The kernels count heads, and two steps past a run of them, in 32 bits.
    for (uint32_t heads : {0x7FFFFFFFu, 0x80000000u, 0xFFFFFFF0u, 0xFFFFFFFFu})
        for (uint32_t dim : {1u, 2u, 64u}) {
            vx_layout l = {};
            l.rank = 3;
            l.size[0] = 1, l.size[1] = heads, l.size[2] = dim;
            l.stride[0] = 0, l.stride[1] = dim, l.stride[2] = 1;
            const vx_mview out = {(float*)0x100000, l};
            const vx_cview in = {(float*)0x100000, l};
            vx_rotation how = {};
            how.flags = VX_ROTATE_NORM;
            how.eps = 1e-6f;
            launches = 0;
            const int s = vx_rotate(ctx, nullptr, &out, &in, nullptr, nullptr, nullptr, &how);
            CHECK(heads > 0x7FFFFFFFu ? s == VX_ERR_UNSUPPORTED && launches == 0 && *vx_last_error_message() : s == VX_OK && launches == 1);
            vx_layout few = l;
            few.size[1] = 2;
            const vx_mview q_out = {(float*)0x100000, few};
            const vx_cview q = {(float*)0x100000, few};
            launches = 0;
            const int k = vx_rotate(ctx, nullptr, &q_out, &q, &out, &in, nullptr, &how);
            CHECK(heads > 0x7FFFFFFFu ? k == VX_ERR_UNSUPPORTED && launches == 0 && *vx_last_error_message() : k == VX_OK && launches == 1);
        }
    CHECK(vx_destroy(ctx) == VX_OK);
    if (!failures) std::printf("fine\n");
    return failures != 0;
}
