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
    float       eps;
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
    const void* x;
    uint8_t*    q;
    float*      scale;
};

// Kernel launchers (kernels/block_*.cu): cudaSuccess or the launch error.
// `vec`: every tensor allows whole 16-byte accesses at 8-column boundaries.
int launch_norm(const helix_rms_norm_desc& d, const NormParams& p, bool vec, void* stream);
int launch_norm_grad(const helix_rms_norm_desc& d, const NormGradPlan& pl, const NormParams& p, bool vec,
                     float* dweight, void* stream);
int launch_quant(const helix_quant8_desc& d, const QuantParams& p, bool vec, void* stream);

}  // namespace hx
