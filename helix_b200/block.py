"""The operators of a recurrent block on torch tensors (include/helix/helix_block.h).

Each function maps its tensors onto one call of the C ABI on the tensors'
device and on `stream` (a torch.cuda.Stream, a raw handle, or None for torch's
current stream), and allocates the outputs and the scratch with torch.  There
is no compute here and no fallback: what the library refuses raises HelixError.

8-bit tensors are torch.float8_e4m3fn with an fp32 scale per 128 columns of a
row (or per 128 x 128 block); their rows are padded to whole 16 bytes, which is
what the product needs of its operands.
"""
from __future__ import annotations

import ctypes as C
from contextlib import nullcontext
from typing import NamedTuple, Optional

import torch

from . import Context, HelixError, _default_ctx, abi

_F32, _BF16, _F8, _I32 = torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.int32
_IO = {_F32: abi.HELIX_F32, _BF16: abi.HELIX_BF16}
_OUT = {**_IO, _F8: abi.HELIX_E4M3}
_HERE = nullcontext()
_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream(...).cuda_stream without the object


def _groups(n: int) -> int:
    return (n + abi.HELIX_GROUP - 1) // abi.HELIX_GROUP


def _t(t: Optional[torch.Tensor]) -> abi.Tensor:
    return abi.NULL_TENSOR if t is None else abi.Tensor(t.data_ptr(), 0)


def _dtype(name: str, dtype: torch.dtype, known=_IO) -> int:
    code = known.get(dtype)
    if code is None:
        raise TypeError(f"{name}: {dtype} is not supported")
    return code


def _matrix(name: str, t: torch.Tensor, shape) -> int:
    """Row stride of t seen as rows of its last dimension; raises when it is
    not that, or not of `shape`."""
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.is_contiguous():
        return shape[-1]
    if shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} needs unit stride along its last dimension")
    lead = [(n, s) for n, s in zip(shape[:-1], t.stride()[:-1]) if n != 1]
    for (_, s0), (n1, s1) in zip(lead, lead[1:]):
        if s0 != n1 * s1:
            raise ValueError(f"{name}: rows must be equally far apart")
    return lead[-1][1] if lead else shape[-1]


def _vector(name: str, t: torch.Tensor, n: int, dtype=None) -> None:
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a dense vector of {n}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}")


def _begin(ctx: Optional[Context], stream, first: torch.Tensor, *rest):
    """(context, stream handle, guard) of a call.  Outputs are allocated under
    the guard, so that the allocator ties them to the stream that writes them."""
    index = first.get_device()
    if index < 0:
        raise ValueError("tensors must be on a CUDA device")
    for t in rest:
        if t is not None and t.get_device() != index:
            raise ValueError("tensors are on different devices")
    if ctx is None:
        ctx = _default_ctx.get(index)
        if ctx is None:
            ctx = _default_ctx.setdefault(index, Context(index))
    current = _raw_stream(index)
    if stream is None:
        return ctx, current, _HERE
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=first.device)
    if stream.cuda_stream == current:
        return ctx, current, _HERE
    for t in (first, *rest):  # they may be freed before the stream gets to the call
        if t is not None:
            t.record_stream(stream)
    return ctx, stream.cuda_stream, torch.cuda.stream(stream)


def _check(ctx: Context, status: int) -> None:
    if status != abi.HELIX_OK:
        raise HelixError(status, ctx.last_error())


def _empty8(like: torch.Tensor, shape) -> torch.Tensor:
    """float8 tensor of `shape` whose rows start at multiples of 16 bytes."""
    cols = shape[-1]
    if cols % 16 == 0:
        return like.new_empty(shape, dtype=_F8)
    return like.new_empty((*shape[:-1], (cols + 15) // 16 * 16), dtype=_F8)[..., :cols]


class Norm(NamedTuple):
    """What rms_norm gives: out; its scales where it is in 8 bits; the sum
    (x itself without a residual); rstd where asked for."""
    out: torch.Tensor
    scale: Optional[torch.Tensor]
    sum: torch.Tensor
    rstd: Optional[torch.Tensor]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
             out_dtype: Optional[torch.dtype] = None, keep_rstd: bool = False, ctx: Optional[Context] = None,
             stream=None) -> Norm:
    """Root-mean-square norm over the last dimension of s = x + residual.

    out = s / sqrt(mean(s^2) + eps) * weight in out_dtype (x's by default);
    torch.float8_e4m3fn gives 8 bits with a scale per 128 columns.  sum is s
    in the residual's type.  keep_rstd keeps 1 / sqrt(...) per row for
    rms_norm_grad."""
    shape = x.shape
    cols = shape[-1]
    rows = x.numel() // cols if cols else 0
    tx = _dtype("x", x.dtype)
    ld_x = _matrix("x", x, shape)
    tr, ld_res = tx, cols
    if residual is not None:
        tr, ld_res = _dtype("residual", residual.dtype), _matrix("residual", residual, shape)
    _vector("weight", weight, cols)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    to = _dtype("out_dtype", out_dtype, _OUT)
    ctx, handle, guard = _begin(ctx, stream, x, residual, weight)
    total = scale = rstd = None
    with guard:
        if out_dtype == _F8:
            out = _empty8(x, shape)
            scale = x.new_empty((*shape[:-1], _groups(cols)), dtype=_F32)
            ld_out = (cols + 15) // 16 * 16
        else:
            out = x.new_empty(shape, dtype=out_dtype)
            ld_out = cols
        if residual is not None:
            total = residual.new_empty(shape)
        if keep_rstd:
            rstd = x.new_empty(shape[:-1], dtype=_F32)
    d = abi.RmsNormDesc(rows, cols, eps, tx, tr, to, _dtype("weight", weight.dtype), ld_x, ld_res, cols, ld_out,
                        _groups(cols))
    _check(ctx, ctx.lib.helix_rms_norm_encode(ctx.handle, handle, C.byref(d), _t(x), _t(residual), _t(weight),
                                              _t(out), _t(scale), _t(total), _t(rstd)))
    return Norm(out, scale, x if total is None else total, rstd)


def rms_norm_grad(dout: torch.Tensor, sum: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor,
                  dsum: Optional[torch.Tensor] = None, *, keep_dres: bool = False, ctx: Optional[Context] = None,
                  stream=None):
    """Gradient of rms_norm: (dx, dweight), or (dx, dweight, dres) with
    keep_dres.

    dout is the gradient of the norm's output in x's type (rounding to 8 bits
    is passed through), dsum the one that reaches sum by another way; sum and
    rstd are what the forward pass gave.  dx has dout's type and dres, the
    same gradient for the residual, sum's; dweight is f32."""
    shape = dout.shape
    cols = shape[-1]
    rows = dout.numel() // cols if cols else 0
    tx, ts = _dtype("dout", dout.dtype), _dtype("sum", sum.dtype)
    ld_dout, ld_sum, ld_dsum = _matrix("dout", dout, shape), _matrix("sum", sum, shape), cols
    if dsum is not None:
        if dsum.dtype != sum.dtype:
            raise TypeError("dsum must have sum's type")
        ld_dsum = _matrix("dsum", dsum, shape)
    if rstd.dtype != _F32 or rstd.shape != shape[:-1] or not rstd.is_contiguous():
        raise ValueError("rstd must be a dense float32 tensor with one value per row")
    _vector("weight", weight, cols)
    ctx, handle, guard = _begin(ctx, stream, dout, sum, rstd, weight, dsum)
    d = abi.RmsNormDesc(rows, cols, 0.0, tx, ts, tx, _dtype("weight", weight.dtype), 0, 0, ld_sum, 0, 0, ld_dout,
                        ld_dsum, cols, cols)
    lib, dres = ctx.lib, None
    nbytes = lib.helix_rms_norm_grad_scratch_size(ctx.handle, C.byref(d))
    with guard:
        dx = dout.new_empty(shape)
        dweight = dout.new_empty((cols,), dtype=_F32)
        if keep_dres and ts != tx:
            dres = sum.new_empty(shape)
        scratch = dout.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
    _check(ctx, lib.helix_rms_norm_grad_encode(ctx.handle, handle, C.byref(d), _t(dout), _t(sum), _t(rstd), _t(weight),
                                               _t(dsum), _t(dx), _t(dres), _t(dweight), _t(scratch)))
    if keep_dres:
        return dx, dweight, dx if dres is None else dres
    return dx, dweight


def quantize8(x: torch.Tensor, *, blocks: bool = False, transpose: bool = False, ctx: Optional[Context] = None,
              stream=None):
    """The matrix x, or x transposed, in 8 bits: (q, scale).

    One scale per 128 columns of each of q's rows, or per 128 x 128 block.
    transpose lays an operand out for the products of a backward pass: blocks
    of a weight, or (by rows) 128 tokens of a column under one scale."""
    if x.dim() != 2:
        raise ValueError("x must be a matrix")
    n_row, n_col = x.shape
    tx, ld_x = _dtype("x", x.dtype), _matrix("x", x, x.shape)
    rows, cols = (n_col, n_row) if transpose else (n_row, n_col)
    ctx, handle, guard = _begin(ctx, stream, x)
    with guard:
        q = _empty8(x, (rows, cols))
        scale = x.new_empty((_groups(rows) if blocks else rows, _groups(cols)), dtype=_F32)
    d = abi.Quant8Desc(n_row, n_col, tx, abi.HELIX_SCALE_BLOCKS if blocks else abi.HELIX_SCALE_ROWS, transpose, ld_x,
                       (cols + 15) // 16 * 16, _groups(cols))
    _check(ctx, ctx.lib.helix_quant8_encode(ctx.handle, handle, C.byref(d), _t(x), _t(q), _t(scale)))
    return q, scale


def matmul8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, *,
            out_dtype: torch.dtype = torch.bfloat16, ctx: Optional[Context] = None, stream=None) -> torch.Tensor:
    """a b^T of 8-bit matrices a (..., k) and b (n, k): (..., n) in out_dtype.

    a_scale (..., ceil(k / 128)); b_scale (ceil(n / 128), ceil(k / 128)) by
    blocks or (n, ceil(k / 128)) by rows.  Rows of a and b must start at
    multiples of 16 bytes, as rms_norm and quantize8 leave them."""
    if a.dtype != _F8 or b.dtype != _F8:
        raise TypeError("a and b must be torch.float8_e4m3fn")
    if a_scale.dtype != _F32 or b_scale.dtype != _F32:
        raise TypeError("scales must be torch.float32")
    if b.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError("b must be a matrix with as many columns as a")
    n, k = b.shape
    groups, lead = _groups(k), a.shape[:-1]
    rows = b_scale.shape == (n, groups)
    to = _dtype("out_dtype", out_dtype)
    strides = (_matrix("a", a, a.shape), _matrix("b", b, b.shape), n, _matrix("a_scale", a_scale, (*lead, groups)),
               _matrix("b_scale", b_scale, (n if rows else _groups(n), groups)))
    ctx, handle, guard = _begin(ctx, stream, a, a_scale, b, b_scale)
    with guard:
        out = a.new_empty((*lead, n), dtype=out_dtype)
    d = abi.Matmul8Desc(a.numel() // k if k else 0, n, k, abi.HELIX_SCALE_ROWS if rows else abi.HELIX_SCALE_BLOCKS, to,
                        *strides)
    _check(ctx, ctx.lib.helix_matmul8_encode(ctx.handle, handle, C.byref(d), _t(a), _t(a_scale), _t(b), _t(b_scale),
                                             _t(out)))
    return out


def _tokens(name: str, t: torch.Tensor, shape, dtype) -> tuple[int, int]:
    """(token stride, sequence stride) of a (sequences, tokens, channels) tensor."""
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}")
    s, k, c = t.stride()
    if c != 1 and shape[2] > 1:
        raise ValueError(f"{name} needs unit stride along the channels")
    return k, s


def _state(name: str, t: torch.Tensor, shape) -> int:
    if t.dtype != _F32:
        raise TypeError(f"{name} must be torch.float32")
    return _matrix(name, t, shape)


def gated_scan(v: torch.Tensor, g: torch.Tensor, h0: Optional[torch.Tensor] = None, *,
               lengths: Optional[torch.Tensor] = None, h1: Optional[torch.Tensor] = None, keep_states: bool = False,
               ctx: Optional[Context] = None, stream=None):
    """h_t = f_t h_{t-1} + (1 - f_t) v_t with f = sigmoid(g), per channel:
    (y, h1), or (y, h1, states) with keep_states (for gated_scan_grad).

    v and g are (sequences, tokens, channels) and may be slices of one wider
    tensor; h0 (sequences, channels) f32 is the state before the first token
    (zeros without), h1 the one after the last, written into the tensor given
    (h0 itself for a step in place) or a new one.  lengths (int32, one per
    sequence) ends sequences early: later tokens keep the state and have y 0."""
    if v.dim() != 3:
        raise ValueError("v must be (sequences, tokens, channels)")
    shape, dtype = v.shape, v.dtype
    seqs, toks, chans = shape
    io = _dtype("v", dtype)
    (s_v, seq_v), (s_g, seq_g) = _tokens("v", v, shape, dtype), _tokens("g", g, shape, dtype)
    if lengths is not None:
        _vector("lengths", lengths, seqs, _I32)
    seq_h0 = seq_h1 = chans
    if h0 is not None:
        seq_h0 = _state("h0", h0, (seqs, chans))
    if h1 is not None:
        seq_h1 = _state("h1", h1, (seqs, chans))
    ctx, handle, guard = _begin(ctx, stream, v, g, h0, lengths, h1)
    states = None
    with guard:
        y = v.new_empty(shape)
        if h1 is None:
            h1 = v.new_empty((seqs, chans), dtype=_F32)
        if keep_states:
            states = v.new_empty((seqs, -(-toks // abi.HELIX_GATED_CHUNK), chans), dtype=_F32)
    d = abi.GatedScanDesc(toks, seqs, chans, io, s_v, s_g, chans, 0, 0, 0, seq_v, seq_g, toks * chans, 0, 0, 0, seq_h0,
                          seq_h1)
    _check(ctx, ctx.lib.helix_gated_scan_encode(ctx.handle, handle, C.byref(d), _t(v), _t(g), _t(h0), _t(lengths),
                                                _t(y), _t(h1), _t(states)))
    return (y, h1, states) if keep_states else (y, h1)


def gated_scan_grad(dy: torch.Tensor, v: torch.Tensor, g: torch.Tensor, states: torch.Tensor,
                    dh1: Optional[torch.Tensor] = None, *, lengths: Optional[torch.Tensor] = None,
                    dv: Optional[torch.Tensor] = None, dg: Optional[torch.Tensor] = None,
                    ctx: Optional[Context] = None, stream=None):
    """Gradient of gated_scan: (dv, dg, dh0) from the gradients of y and of h1
    (zeros without), with the states the forward pass kept.  dv and dg are
    written into the tensors given (slices of one wider tensor, say) or new ones."""
    if v.dim() != 3:
        raise ValueError("v must be (sequences, tokens, channels)")
    shape, dtype = v.shape, v.dtype
    seqs, toks, chans = shape
    io = _dtype("v", dtype)
    (s_v, seq_v), (s_g, seq_g) = _tokens("v", v, shape, dtype), _tokens("g", g, shape, dtype)
    s_dy, seq_dy = _tokens("dy", dy, shape, dtype)
    if (states.dtype != _F32 or not states.is_contiguous()
            or states.shape != (seqs, -(-toks // abi.HELIX_GATED_CHUNK), chans)):
        raise ValueError("states must be what gated_scan(keep_states=True) gave")
    if lengths is not None:
        _vector("lengths", lengths, seqs, _I32)
    seq_dh1 = chans if dh1 is None else _state("dh1", dh1, (seqs, chans))
    ctx, handle, guard = _begin(ctx, stream, dy, v, g, states, dh1, lengths, dv, dg)
    with guard:
        dv = v.new_empty(shape) if dv is None else dv
        dg = v.new_empty(shape) if dg is None else dg
        dh0 = v.new_empty((seqs, chans), dtype=_F32)
    (s_dv, seq_dv), (s_dg, seq_dg) = _tokens("dv", dv, shape, dtype), _tokens("dg", dg, shape, dtype)
    d = abi.GatedScanDesc(toks, seqs, chans, io, s_v, s_g, 0, s_dy, s_dv, s_dg, seq_v, seq_g, 0, seq_dy, seq_dv,
                          seq_dg, 0, 0, seq_dh1, chans)
    _check(ctx, ctx.lib.helix_gated_scan_grad_encode(ctx.handle, handle, C.byref(d), _t(dy), _t(v), _t(g), _t(states),
                                                     _t(dh1), _t(lengths), _t(dv), _t(dg), _t(dh0)))
    return dv, dg, dh0
