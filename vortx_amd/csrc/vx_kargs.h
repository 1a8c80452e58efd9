/*
 * vx_kargs.h — kernel argument blocks shared by the host library (g++)
 * and the gfx950 kernels (hipcc). Each kernel takes one of these structs
 * by value; the host passes it to hipModuleLaunchKernel through
 * kernelParams, so the layout must be identical on both sides: only
 * fixed-width integers and pointers, naturally aligned.
 */
#ifndef VX_KARGS_H
#define VX_KARGS_H

#include <stdint.h>

#define VX_WG 256          /* threads per workgroup (4 wave64) */
#define VX_LDS_X_BYTES 65536 /* LDS budget for staged activations */

/* Dense f32 GEMM on canonical [n, c, rows, cols] operands. Base pointers
 * already include each view's element offset. Strides in elements. */
typedef struct vx_gemm_args {
    float* c;
    const float* a;
    const float* b;
    int64_t cs[4];
    int64_t as[4];
    int64_t bs[4];
    uint32_t batch_c;  /* size of dim 1; grid z = n * batch_c */
    uint32_t M, N, K;
    uint32_t tiles_m, tiles_n;
    float alpha, beta;  /* c = alpha * acc + beta * c (c not read when beta == 0) */
} vx_gemm_args;

/* Block-quantized GEMV / dequantize. */
typedef struct vx_gemv_args {
    const uint8_t* w;
    uint64_t row_stride;   /* bytes between rows of W */
    const float* x;        /* x[k, b] at x[k*xs_k + b*xs_b] */
    int64_t xs_k, xs_b;
    float* y;              /* y[m, b] at y[m*ys_m + b*ys_b] */
    int64_t ys_m, ys_b;
    uint32_t M, K, B;      /* B = batch columns handled by this launch */
    uint32_t nunits;       /* K / 64 (units of 64 weights) */
    uint32_t chunk_units;  /* units staged in LDS per chunk */
    uint32_t upitch;       /* LDS pitch (in float4) of one unit-column, odd */
    uint32_t x_vec;        /* 1: x has stride 1 along K and 16-byte aligned rows */
    uint32_t pad0;
} vx_gemv_args;

/* f32 GEMV (the N == 1 route of the GEMM op): y[m] = sum_k A[m,k] x[k]. */
typedef struct vx_gemv_f32_args {
    const float* a;
    int64_t as_m, as_k;
    const float* x;
    int64_t xs_k;
    float* y;
    int64_t ys_m;
    uint32_t M, K;
    uint32_t batch_c;
    float alpha, beta;  /* y = alpha * acc + beta * y (y not read when beta == 0) */
    uint32_t pad0;
    int64_t a_bs[2], x_bs[2], y_bs[2]; /* batch strides (dims n, c) */
} vx_gemv_f32_args;

/* Unsigned division by a fixed divisor d >= 1 (round-up multiplier m and
 * shift s; `one` marks d == 1). */
typedef struct vx_udiv {
    uint32_t m, s, one, pad;
} vx_udiv;

/* Strided -> contiguous copy of 4-byte elements over the canonical
 * [n, c, h, w] view (strides in elements, 64-bit). */
typedef struct vx_copy_args {
    uint32_t* dst;
    const uint32_t* src;
    const uint32_t* dev_offset; /* null, or a device u32 added to every source index */
    int64_t stride[4];
    uint32_t size[4];
    uint32_t total;             /* elements (< 2^32) */
    uint32_t pad0;
    vx_udiv dw, dh, dc;         /* divisions by size[3], size[2], size[1] */
} vx_copy_args;

/* f32 [M, K] -> quantized blocks (row i at out + i * row_stride). */
typedef struct vx_quant_args {
    const float* x;
    int64_t xs_m, xs_k;
    uint8_t* out;
    uint64_t row_stride;
    uint32_t M, K;
    uint32_t nblk;   /* blocks (Q4_K: super-blocks) per row */
    uint32_t x_vec;  /* 1: xs_k == 1 and 16-byte aligned rows */
} vx_quant_args;

/* Activation split x [K, B] f32 -> levels int8 [nblk][B][2][32] and scales
 * f32 [nblk][B][2] (the layout of vx_xq in include/vortx_hip.h). */
typedef struct vx_xq_args {
    const float* x;        /* x[k, b] at x[k*xs_k + b*xs_b] */
    int64_t xs_k, xs_b;
    int8_t* levels;
    float* scales;
    uint32_t K, B;
    uint32_t nblk;         /* K / 32 */
    uint32_t x_vec;        /* 1: xs_k == 1, 16-byte aligned columns */
} vx_xq_args;

/* Batched GEMV on split activations: y[m, b] = sum_k W[m, k] x[k, b]. */
typedef struct vx_gemv_xq_args {
    const uint8_t* w;
    uint64_t row_stride;   /* bytes between rows of W */
    const int8_t* levels;  /* the vx_xq levels of x */
    const float* scales;   /* the vx_xq scales of x */
    float* y;              /* y[m, b] at y[m*ys_m + b*ys_b] */
    int64_t ys_m, ys_b;
    uint32_t M, K, B;      /* B: columns of this launch, <= 16 */
    uint32_t nblk;         /* K / 32 */
    uint32_t nunits;       /* K / 64 */
    uint32_t ipr;          /* items (256 weights) per row, the last one possibly partial */
    uint32_t npass;        /* passes over K: ceil(ipr / (16 * items per wave)) */
    uint32_t xcols;        /* columns of the split x (its layout pitch) */
    uint32_t col0;         /* first split-x column of this launch (y is already offset) */
    uint32_t pad0;
    const float* x;        /* kernels that split x themselves (_fx): x[k, b] at x[k + b*xs_b] */
    int64_t xs_b;
} vx_gemv_xq_args;

/* Paged key/value cache (the layout of vx_kv.hpp). */
typedef struct vx_kv_geom {
    uint8_t* base;
    uint64_t page_bytes;
    uint32_t pages;
    uint32_t page_shift;   /* log2 of the tokens of a page, >= 4 */
    uint32_t heads;        /* key/value heads */
    uint32_t dim;
} vx_kv_geom;

/* Rows into the cache, and out of it. k / v of vx_kv_read may be null. */
typedef struct vx_kv_rows_args {
    vx_kv_geom c;
    float* k;              /* element (t, h, d) at k[t*ks[0] + h*ks[1] + d*ks[2]]; read only by vx_kv_write */
    float* v;
    int64_t ks[3], vs[3];
    const int32_t* slots;  /* [tokens]; one outside the cache is left out (write) or gives zeros (read) */
    uint32_t tokens;
    uint32_t vec;          /* 1: k and v have stride 1 along the dim and 16-byte aligned rows */
    uint32_t quads;        /* 1: tokens go by fours */
    uint32_t groups;       /* of tokens: one each, or four */
} vx_kv_rows_args;

/* Rows of heads, normed and rotated: the queries or the keys of a call. */
typedef struct vx_rotate_rows_args {
    const float* x;        /* element (t, h, d) at x[t*xs[0] + h*xs[1] + d*xs[2]] */
    float* y;              /* (null: keys on their way into the cache) */
    int64_t xs[3], ys[3];
    const float* w;        /* norm weight of head h, dim d at w[h*ws + d]; null: 1 */
    uint32_t ws;
    uint32_t heads;
    uint32_t block_tokens; /* tokens of a workgroup */
    uint32_t run;          /* heads of a workgroup */
    uint32_t chunks;       /* such runs a token */
    uint32_t blocks;       /* workgroups */
} vx_rotate_rows_args;
typedef struct vx_rotate_args {
    vx_rotate_rows_args part[2];  /* queries, keys */
    const double* freqs;   /* [rotated / 2] */
    const int32_t* positions;
    double per_dim;        /* 1 / dim */
    uint32_t tokens, dim, rotated;
    uint32_t pairs, norm;
    float eps;
} vx_rotate_args;

/* Floats of LDS for keys of eleven tokens that are turned before they are written. */
#define VX_ROTATE_STAGE 6144

/* Rows into the cache whose keys are normed and rotated on the way, and the queries beside them. */
typedef struct vx_kv_rotated_args {
    vx_kv_rows_args r;
    vx_rotate_args t;
} vx_kv_rotated_args;

/* Pages of sequences that grow and shrink, and the slots of their new tokens. */
typedef struct vx_pages_args {
    int32_t* table;
    int32_t* lens;
    int32_t* free_pages;
    int32_t* free_count;
    const int32_t* want;
    int32_t* starts;
    int32_t* slots;
    int32_t* positions;
    uint32_t seqs, table_cols, table_stride;
    uint32_t page_shift, pages;
    uint32_t tokens;       /* entries of slots and positions */
    uint32_t here;         /* 1: vx_pages_resize writes them, 0: vx_pages_slots after it */
    uint32_t threads;      /* of vx_pages_resize: a multiple of 64 up to 1024 */
    uint32_t vec;          /* 1: slots and positions are 16-byte aligned */
    uint32_t pad0;
} vx_pages_args;

/* Rows of f32 to 8-bit integers with a scale each. */
typedef struct vx_i8_quant_args {
    const float* x;        /* element (row, k) at x[row*xs[0] + k*xs[1]] */
    int64_t xs[2];
    int8_t* out;
    uint64_t row_stride;   /* bytes */
    float* scales;
    uint32_t rows, cols;
} vx_i8_quant_args;

/* Products of such rows: x [T, K] by w [N, K] (of a gated one, w[0] gate and w[1] up). */
typedef struct vx_i8_args {
    const int8_t* w[2];
    uint64_t ws[2];        /* bytes between rows */
    const float* wscale[2];
    const int8_t* x;
    uint64_t xs;
    const float* xscale;
    const float* xf;       /* kernels that quantize x themselves: element (t, k) at xf[t*xfs[0] + k*xfs[1]] */
    int64_t xfs[2];
    float* out;            /* element (t, n) at out[t*os[0] + n*os[1]] */
    int64_t os[2];
    uint32_t T, N, K;
    uint32_t act;
    uint32_t tiles_t, tiles_n;
    uint32_t out_vec;      /* 1: os[1] == 1 and fours of channels 16-byte aligned */
    uint32_t xf_vec;       /* 1: xfs[1] == 1 and 16-byte aligned rows */
    uint32_t pitch;        /* bytes between x's rows in LDS, of such kernels */
    uint32_t x_bytes;      /* of LDS that x, its maxima and scales take */
    uint32_t split;        /* waves of such a kernel that share a row of the weights: a power of two up to 16;
                            * of kernels for parts of K: how many, chunk columns each (a multiple of 128) */
    uint32_t chunk;
    int32_t* parts;        /* their sums, [split][gate, up][T][N up to a multiple of 4], 16-byte aligned */
} vx_i8_args;
#define VX_I8_OWN_TOKENS 4 /* of such kernels, at most */

/* Attention over the cache. Query row r = j * group + i of a sequence is its
 * j-th query token, i-th query head of the key/value head. */
typedef struct vx_attn_args {
    vx_kv_geom c;
    const float* q;        /* element (t, head, d) at q[t*qs[0] + head*qs[1] + d*qs[2]] */
    float* out;
    int64_t qs[3], os[3];
    const int32_t* table;  /* [seqs][table_stride]: page of each page_tokens keys */
    const int32_t* lens;   /* [seqs] */
    const int32_t* starts; /* [seqs + 1] */
    const float* slopes;   /* [query heads] or null */
    const int32_t* prefix; /* [seqs] or null */
    const int32_t* first;  /* [tokens] or null */
    const uint32_t* tree;  /* [tokens][tree_stride] or null */
    uint32_t* info;        /* [seqs][row blocks][heads] first partial and their number (vx_attn_deal) */
    float* part_o;         /* partial sums [partial][part_rows][dim] */
    float* part_ml;        /* [partial][part_rows][2] */
    uint32_t table_stride, table_cols;
    uint32_t seqs, tokens, group;
    uint32_t max_queries, max_len;
    uint32_t row_blocks;   /* of a sequence, part_rows query rows each */
    uint32_t part_rows;
    uint32_t parts;        /* about how many partials a unit has */
    uint32_t causal, window;
    uint32_t tree_stride, tree_words;
    float scale, cap;      /* cap 0: none */
    uint32_t vec;          /* 1: q and out have stride 1 along the dim and 16-byte aligned rows */
} vx_attn_args;

/* Bytes of the device scratch array of vx_gemv_q_noalloc (vx_scratch in
 * the GEMV code object): the largest activation split it can hold. */
#define VX_SCRATCH_BYTES (4u << 20)

#endif /* VX_KARGS_H */
