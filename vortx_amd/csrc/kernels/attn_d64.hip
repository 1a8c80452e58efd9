// attn_d64.hip — the quantized cache and the attention over it, heads of 64.
#define VX_NB 2
#define VX_NAME(f, types) vx_##f##_d64_##types
#define VX_JOIN vx_attn_join_d64
#include "vx_attn_kernels.hpp"
