// attn_d256.hip — the quantized cache and the attention over it, heads of 256.
#define VX_NB 8
#define VX_NAME(f, types) vx_##f##_d256_##types
#define VX_JOIN vx_attn_join_d256
#include "vx_attn_kernels.hpp"
