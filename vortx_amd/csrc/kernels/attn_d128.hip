// attn_d128.hip — the quantized cache and the attention over it, heads of 128.
#define VX_NB 4
#define VX_NAME(f, types) vx_##f##_d128_##types
#define VX_JOIN vx_attn_join_d128
#include "vx_attn_kernels.hpp"
