// attn_d96.hip — the quantized cache and the attention over it, heads of 96.
#define VX_NB 3
#define VX_NAME(f, types) vx_##f##_d96_##types
#define VX_JOIN vx_attn_join_d96
#include "vx_attn_kernels.hpp"
