/* helix_block.h -- the operators of a recurrent block around its scan.
 *
 * No counterpart in the reference, which holds the scan alone.  Everything
 * here follows the scan's contract (helix.h): a call is enqueued on `stream`
 * (a cudaStream_t; NULL = legacy default stream), never synchronises, never
 * allocates, and enqueues nothing when it returns an error; the message is in
 * helix_ctx_last_error().  Tensors are device memory on ctx's device, aligned
 * to their element size.  Strides are in elements; the innermost stride is 1.
 * An output may not overlap an input or another output, except where a
 * comment says "in place": then it is the same address, type and strides.
 *
 * 8-bit tensors are e4m3 floats (HELIX_E4M3) with one fp32 scale for each
 * group of HELIX_GROUP: a value is (float)q * scale, and
 *     scale = max(largest magnitude of the group, 2^-100) / 448,
 *     q     = value / scale rounded to nearest even,
 * where scale is within 2 units in its last place of that, and the quotient,
 * before it is rounded to 8 bits, within 4.
 * A group that holds a NaN or an infinity has that as its scale, and NaN (or
 * zero, for the finite values beside an infinity) as its q.
 */
#ifndef HELIX_BLOCK_H
#define HELIX_BLOCK_H

#include "helix/helix.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HELIX_GROUP 128

/* ------------------------------------------------------------------------ */
/* Root-mean-square norm with the residual's addition                       */
/* ------------------------------------------------------------------------ */

/* Per row, with s = x + residual in fp32:
 *     rstd = 1 / sqrt(mean(s^2) + eps),   n = s rstd weight
 * sum receives s rounded to sum_dtype; n is taken from the unrounded s. */
typedef struct {
    int64_t     n_row;
    int32_t     n_col;      /* 1 .. 16384                                      */
    float       eps;        /* >= 0                                            */
    helix_dtype x_dtype;    /* F32 or BF16: x; dout and dx of the gradient      */
    helix_dtype sum_dtype;  /* residual and sum, dsum and dres: F32, or x_dtype */
    helix_dtype out_dtype;  /* out: F32, BF16 or E4M3                           */
    helix_dtype w_dtype;    /* weight: F32 or BF16                              */
    int64_t     ld_x;       /* row strides: x                                   */
    int64_t     ld_res;     /* residual                                         */
    int64_t     ld_sum;     /* sum                                              */
    int64_t     ld_out;     /* out                                              */
    int64_t     ld_scale;   /* scale [n_row][ceil(n_col / 128)] f32             */
    int64_t     ld_dout;    /* gradient: dout, dsum, dx, dres                   */
    int64_t     ld_dsum;
    int64_t     ld_dx;
    int64_t     ld_dres;
} helix_rms_norm_desc;

/* Dense strides, every type F32, eps 1e-6. */
void helix_rms_norm_desc_init(helix_rms_norm_desc* d, int64_t n_row, int32_t n_col);

/* residual may be null (s = x).  sum may be null; in place of residual or of
 * x it is allowed.  scale is written when out_dtype is E4M3 (and required
 * then), rstd [n_row] f32 when not null. */
helix_status helix_rms_norm_encode(helix_ctx* ctx, void* stream, const helix_rms_norm_desc* d,
                                   helix_tensor x, helix_tensor residual, helix_tensor weight,
                                   helix_tensor out, helix_tensor scale, helix_tensor sum,
                                   helix_tensor rstd);

/* The gradient.  dout (x_dtype) is the gradient of n; rounding to 8 bits is
 * passed through.  dsum (sum_dtype, may be null) is the gradient that reaches
 * sum by another way.  With s = the stored sum (sum_dtype) and rstd as the
 * forward pass left them:
 *     ds = dsum + rstd (dout w - s rstd^2 mean(dout w s))
 *     dweight = sum over rows of dout s rstd         (f32, [n_col])
 * dx (x_dtype) and, when not null, dres (sum_dtype) both receive ds.  dx may
 * be in place of dout, dres in place of dsum.  The sum over rows is taken in
 * an order that depends on the sizes and the device alone.  Needs
 * helix_rms_norm_grad_scratch_size() bytes of 256-byte-aligned scratch. */
size_t       helix_rms_norm_grad_scratch_size(helix_ctx* ctx, const helix_rms_norm_desc* d);
helix_status helix_rms_norm_grad_encode(helix_ctx* ctx, void* stream, const helix_rms_norm_desc* d,
                                        helix_tensor dout, helix_tensor sum, helix_tensor rstd,
                                        helix_tensor weight, helix_tensor dsum, helix_tensor dx,
                                        helix_tensor dres, helix_tensor dweight,
                                        helix_tensor scratch);

/* ------------------------------------------------------------------------ */
/* Quantiser                                                                */
/* ------------------------------------------------------------------------ */

typedef enum {
    HELIX_SCALE_ROWS   = 0, /* one scale per row and 128 columns               */
    HELIX_SCALE_BLOCKS = 1, /* one scale per 128 rows and 128 columns          */
} helix_scale_form;

/* q = x, or x transposed, in 8 bits.  The groups are those of q: transposed,
 * HELIX_SCALE_ROWS puts 128 consecutive rows of x under one scale. */
typedef struct {
    int64_t          n_row;     /* of x                                        */
    int64_t          n_col;
    helix_dtype      x_dtype;   /* F32 or BF16                                 */
    helix_scale_form form;
    bool             transpose; /* q is [n_col][n_row], else [n_row][n_col]    */
    int64_t          ld_x;
    int64_t          ld_q;
    int64_t          ld_scale;  /* scale: [q rows, or their blocks][ceil(q columns / 128)] f32 */
} helix_quant8_desc;

/* Dense strides except ld_q, which is rounded up to 16 (what the product
 * needs of its operands). */
void         helix_quant8_desc_init(helix_quant8_desc* d, int64_t n_row, int64_t n_col,
                                    helix_scale_form form, bool transpose);
helix_status helix_quant8_encode(helix_ctx* ctx, void* stream, const helix_quant8_desc* d,
                                 helix_tensor x, helix_tensor q, helix_tensor scale);

/* ------------------------------------------------------------------------ */
/* Product of 8-bit matrices                                                */
/* ------------------------------------------------------------------------ */

/* out[i][j] = sum over blocks of 128 columns b of
 *     a_scale[i][b] b_scale[j or j / 128][b] sum_{k in b} a[i][k] b[j][k]
 * a [m][k] has its scales by rows (what the norm and the quantiser write),
 * b [n][k] by blocks (a weight) or by rows.  Products are exact; the tensor
 * cores sum a block's in fp32 and may truncate (within 16 x 2^-24 of the sum of
 * their magnitudes), blocks are scaled and summed in fp32 in an order that
 * depends on the sizes and the device alone, and out is rounded once.
 *
 * The gradients are two more such products: of a, the gradient of out (by
 * rows) with b transposed (blocks); of b, the gradient of out and a, both
 * transposed, by rows.  helix_quant8_encode lays all of them out.
 *
 * a and b are read in tiles: their bases must be 16-byte aligned and their
 * row strides multiples of 16 (HELIX_ERR_UNSUPPORTED_SHAPE otherwise). */
typedef struct {
    int32_t          m, n, k;
    helix_scale_form b_form;
    helix_dtype      out_dtype;  /* F32 or BF16                                 */
    int64_t          ld_a, ld_b, ld_out;
    int64_t          ld_a_scale, ld_b_scale;
} helix_matmul8_desc;

/* Dense strides except ld_a and ld_b, which are rounded up to 16; BF16 out. */
void         helix_matmul8_desc_init(helix_matmul8_desc* d, int32_t m, int32_t n, int32_t k,
                                     helix_scale_form b_form);
helix_status helix_matmul8_encode(helix_ctx* ctx, void* stream, const helix_matmul8_desc* d,
                                  helix_tensor a, helix_tensor a_scale, helix_tensor b,
                                  helix_tensor b_scale, helix_tensor out);

/* ------------------------------------------------------------------------ */
/* Gated linear recurrence                                                  */
/* ------------------------------------------------------------------------ */

#define HELIX_GATED_CHUNK 128

/* Per sequence and channel, with the gate f = 1 / (1 + exp(-g)) of every
 * token and a state of its own:
 *     h_t = f_t h_{t-1} + (1 - f_t) v_t,   y_t = h_t
 * from h0 (zeros when null) to h1, the state after the last token.  The
 * states are f32, the arithmetic fp32; v, g, y, dy, dv and dg are io_dtype.
 * Token tensors are [n_seq][n_tok][n_chan] with strides of their own for the
 * token and the sequence; those with the same strides may be slices of one
 * wider tensor.  States are [n_seq][n_chan].
 *
 * f and 1 - f are both known to (2 |g| + 14) 2^-24 of themselves (below 2^-126
 * they may count as 0 or as that), and what is left of a state or a gradient
 * after many tokens is as accurate relative to itself.  An infinite h0 or v
 * makes the states from there on infinite, an infinite dh1 or dy the gradients
 * before it, as the formula does: NaN where two of different sign meet, or
 * infinity and a difference h_{t-1} - v_t of zero.  NaN stays in its channel.
 *
 * lengths (int32, [n_seq], may be null) ends sequences early: tokens at or
 * past lengths[seq] (taken as 0 .. n_tok) leave the state as it is, whatever
 * v, g and dy hold there, and have y = dv = dg = 0.
 *
 * n_tok = 1 is the step of a decoder, h1 in place of h0. */
typedef struct {
    int32_t     n_tok, n_seq, n_chan;        /* at most 2^31 - 4097 tokens, 2^31 - 65 channels */
    helix_dtype io_dtype;                    /* F32 or BF16                     */
    int64_t     s_v, s_g, s_y;               /* token strides                   */
    int64_t     s_dy, s_dv, s_dg;
    int64_t     seq_v, seq_g, seq_y;         /* sequence strides                */
    int64_t     seq_dy, seq_dv, seq_dg;
    int64_t     seq_h0, seq_h1;
    int64_t     seq_dh1, seq_dh0;
} helix_gated_scan_desc;

/* Dense strides, F32. */
void helix_gated_scan_desc_init(helix_gated_scan_desc* d, int32_t n_tok, int32_t n_seq, int32_t n_chan);

/* Bytes of `states`: f32 [n_seq][ceil(n_tok / HELIX_GATED_CHUNK)][n_chan],
 * the state entering every chunk of tokens, which the gradient starts from. */
size_t helix_gated_scan_states_size(const helix_gated_scan_desc* d);

/* states may be null when no gradient follows.  h1 may be in place of h0. */
helix_status helix_gated_scan_encode(helix_ctx* ctx, void* stream, const helix_gated_scan_desc* d,
                                     helix_tensor v, helix_tensor g, helix_tensor h0,
                                     helix_tensor lengths, helix_tensor y, helix_tensor h1,
                                     helix_tensor states);

/* The gradient, from the forward pass's states.  dy is the gradient of y, dh1
 * (null: zeros) of h1; dh0 may be null.  With lam_t the gradient of h_t:
 *     lam_t = dy_t + f_{t+1} lam_{t+1},  lam_last = dy_last + dh1
 *     dv_t = (1 - f_t) lam_t,  dg_t = lam_t (h_{t-1} - v_t) f_t (1 - f_t)
 *     dh0 = f_0 lam_0
 * dv may be in place of dy, dh0 in place of dh1. */
helix_status helix_gated_scan_grad_encode(helix_ctx* ctx, void* stream, const helix_gated_scan_desc* d,
                                          helix_tensor dy, helix_tensor v, helix_tensor g,
                                          helix_tensor states, helix_tensor dh1, helix_tensor lengths,
                                          helix_tensor dv, helix_tensor dg, helix_tensor dh0);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* HELIX_BLOCK_H */
