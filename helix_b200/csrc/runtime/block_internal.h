// block_internal.h -- what the runtime and the kernels of the block operators
// (helix_block.h) share.  Not installed, not part of the ABI.
#pragma once

#include <cstddef>
#include <cstdint>

#include "helix/helix_block.h"
#include "internal.h"

namespace hx {

// A row of the norm is cut into segments of 256 columns, one per warp and
// step: a lane holds 8 values of each of its warp's V segments.
struct NormShape {
    int v;     // segments per warp (kernel template: 1, 2 or 4)
    int wpr;   // warps per row
    int rpb;   // rows per block
};
NormShape norm_shape(const helix_rms_norm_desc& d);
int configure_norm();
// Gradient: slots of rows, each with its own partial sum of dweight.
struct NormGradPlan {
    NormShape shape;
    int       blocks;  // persistent grid
    int       slots;   // blocks * rpb
    size_t    total;   // scratch bytes: f32 [slots][n_col]
};
NormGradPlan norm_grad_plan(const helix_ctx* ctx, const helix_rms_norm_desc& d);

struct NormParams {
    int64_t     n_row;
    int32_t     n_col, wpr, rpb;
    float       eps, inv_col;  // inv_col: 1 / n_col
    int32_t     out_dtype, w_bf16;
    int64_t     ld_x, ld_res, ld_sum, ld_out, ld_scale;
    int64_t     ld_dout, ld_dsum, ld_dx, ld_dres;
    const void *x, *res, *w;
    void       *out, *sum;
    float      *scale, *rstd;
    const void *dout, *dsum;
    void       *dx, *dres;
    float      *partial;  // scratch [slots][n_col]
};

struct QuantParams {
    int64_t     n_row, n_col;
    int64_t     ld_x, ld_q, ld_scale;
    int32_t     n_tile_col;  // ceil(n_col / 128)
    int32_t     q_vec;       // rows of q can be written in 8-byte pieces
    const void* x;
    uint8_t*    q;
    float*      scale;
};

// One operand of the product as the kernel sees it.  P gives the rows of a
// tile (the MMA's M, 128 of them), Q its columns.
struct Mm8Operand {
    const float* scale;
    int64_t      ld_scale;
    int32_t      rows;
    int32_t      per;      // rows under one scale: 1 or 128
    bool         quads;    // rows of scale can be read in 16-byte pieces
};
// How one product runs.
struct Mm8Plan {
    bool pair;             // pairs of CTAs on tiles of 256 x bn (bn 128 or 256)
    bool swap;             // P is b (few rows of a: they become the columns)
    int  bn;               // columns of a tile
    int  splits;           // CTAs of a cluster that share a tile's blocks of k
};
struct Mm8Params {
    Mm8Operand p, q;
    int32_t    k_blocks, splits, tiles_q;
    int32_t    vec_out;    // rows of out can be written in 16-byte pieces
    int32_t    swap;
    int64_t    ld_out;
    void*      out;
    unsigned*  fault;
};
Mm8Plan mm8_plan(const helix_ctx* ctx, const helix_matmul8_desc& d);
int configure_mm8(helix_ctx* ctx);    // fills ctx->mm8_clusters
// a, b: operands as the caller laid them out.
int launch_mm8(const helix_ctx* ctx, const helix_matmul8_desc& d, const Mm8Plan& pl, Mm8Params p, const void* a,
               const void* b, void* stream);

struct GatedParams {
    int32_t        n_tok, n_seq, n_chan;
    int32_t        n_chunk;    // ceil(n_tok / HELIX_GATED_CHUNK)
    int32_t        cluster;    // CTAs that share a sequence's chunks
    int64_t        s_v, s_g, s_y, s_dy, s_dv, s_dg;
    int64_t        seq_v, seq_g, seq_y, seq_dy, seq_dv, seq_dg;
    int64_t        seq_h0, seq_h1, seq_dh1, seq_dh0;
    const void    *v, *g, *dy;
    void          *y, *dv, *dg;
    const float   *h0, *dh1;
    float         *h1, *dh0, *states;
    const int32_t* lengths;
    unsigned*      fault;
};
int configure_gated(helix_ctx* ctx);  // fills ctx->gated_clusters
// word (bf16): two channels of every token tensor can be accessed at once.
int launch_gated(const helix_ctx* ctx, const helix_gated_scan_desc& d, GatedParams p, bool word, void* stream);
int launch_gated_grad(const helix_ctx* ctx, const helix_gated_scan_desc& d, GatedParams p, bool word, void* stream);

// Kernel launchers (kernels/block_*.cu): cudaSuccess or the launch error.
// `vec`: every tensor (the quantiser: x) allows whole 16-byte accesses at
// 8-column boundaries.
int launch_norm(const helix_ctx* ctx, const helix_rms_norm_desc& d, const NormParams& p, bool vec, void* stream);
int launch_norm_grad(const helix_rms_norm_desc& d, const NormGradPlan& pl, const NormParams& p, bool vec,
                     float* dweight, void* stream);
int launch_quant(const helix_quant8_desc& d, const QuantParams& p, bool vec, void* stream);

}  // namespace hx
