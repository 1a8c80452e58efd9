// vx_attn_kernels.hpp — the kernels of one head size (VX_NB blocks of 32), for
// each pair of cache types (k8v8: 8 bits for K and V, and so on).
#include "vx_attn_rows16.hpp"
#include "vx_attn_tile.hpp"
#include "vx_kv_rows.hpp"

#define VX_CAT(f, types) VX_NAME(f, types)
#define VX_KERNELS(types, KB, VB)                                                                              \
    extern "C" __global__ __launch_bounds__(256) void VX_CAT(kv_write, types)(vx_kv_rows_args a) {             \
        vx_kv_write_rows<VX_NB, KB, VB>(a);                                                                    \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(256) void VX_CAT(kv_read, types)(vx_kv_rows_args a) {              \
        vx_kv_read_rows<VX_NB, KB, VB>(a);                                                                     \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(256, VX_NB <= 4 ? 2 : 1) void VX_CAT(attn_even16, types)(vx_attn_args a) { \
        vx_rows16<VX_NB, KB, VB>::even(a);                                                                     \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(256, VX_NB <= 4 ? 2 : 1) void VX_CAT(attn_each128, types)(vx_attn_args a) { \
        vx_tile<VX_NB, KB, VB, 4>::each(a);                                                                    \
    }
// (heads of 256: eight waves' registers do not hold the sums, and four hold them
// with 15 to 23 registers in memory, dealt out 76 to 93; even256 of 128 has 17
// there, each128 up to 16)
#if VX_NB <= 4
#define VX_WIDE(types, KB, VB)                                                                                 \
    extern "C" __global__ __launch_bounds__(512, 2) void VX_CAT(attn_each256, types)(vx_attn_args a) {         \
        vx_tile<VX_NB, KB, VB, 8>::each(a);                                                                    \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(512, 2) void VX_CAT(attn_even256, types)(vx_attn_args a) {         \
        vx_tile<VX_NB, KB, VB, 8>::even(a);                                                                    \
    }
#else
#define VX_WIDE(types, KB, VB)                                                                                 \
    extern "C" __global__ __launch_bounds__(256) void VX_CAT(attn_even128, types)(vx_attn_args a) {            \
        vx_tile<VX_NB, KB, VB, 4>::even(a);                                                                    \
    }
#endif
VX_KERNELS(k8v8, 8, 8)
VX_KERNELS(k8v4, 8, 4)
VX_KERNELS(k4v8, 4, 8)
VX_KERNELS(k4v4, 4, 4)
VX_WIDE(k8v8, 8, 8)
VX_WIDE(k8v4, 8, 4)
VX_WIDE(k4v8, 4, 8)
VX_WIDE(k4v4, 4, 4)

extern "C" __global__ __launch_bounds__(256) void VX_JOIN(vx_attn_args a) { vx_attn_join_rows(a); }
