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

from . import Context, HelixError, _ctx_for, _t, abi

_IO = {torch.float32: abi.HELIX_F32, torch.bfloat16: abi.HELIX_BF16}
_OUT = {**_IO, torch.float8_e4m3fn: abi.HELIX_E4M3}


def _groups(n: int) -> int:
    return -(-n // abi.HELIX_GROUP)


def _dtype(name: str, t: torch.Tensor, known=_IO) -> int:
    try:
        return known[t.dtype]
    except KeyError:
        raise TypeError(f"{name}: {t.dtype} is not supported") from None


def _matrix(name: str, t: torch.Tensor, shape=None) -> int:
    """Row stride of t seen as rows of its last dimension; raises when it is
    not that, or not of `shape`."""
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} needs unit stride along its last dimension")
    lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
    for (_, s0), (n1, s1) in zip(lead, lead[1:]):
        if s0 != n1 * s1:
            raise ValueError(f"{name}: rows must be equally far apart")
    return lead[-1][1] if lead else t.shape[-1]


def _vector(name: str, t: torch.Tensor, n: int, dtype=None) -> None:
    if t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a dense vector of {n}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}")


class _Call:
    """Where a call runs: the context, and the stream as a handle.  Outputs
    are allocated under `with call.alloc():`, so that the allocator ties them
    to the stream the call writes them on."""

    __slots__ = ("ctx", "handle", "other")

    def __init__(self, first: torch.Tensor, ctx: Optional[Context], stream, *tensors):
        dev = first.device
        if dev.type != "cuda":
            raise ValueError("tensors must be on a CUDA device")
        for t in tensors:
            if t is not None and t.device != dev:
                raise ValueError("tensors are on different devices")
        self.ctx = _ctx_for(first, ctx)
        self.other = None
        if stream is None:
            self.handle = torch.cuda.current_stream(dev).cuda_stream
            return
        if not hasattr(stream, "cuda_stream"):
            stream = torch.cuda.ExternalStream(int(stream), device=dev)
        self.handle = stream.cuda_stream
        if self.handle != torch.cuda.current_stream(dev).cuda_stream:
            self.other = stream
            for t in (first, *tensors):  # they may be freed before the stream gets to the call
                if t is not None:
                    t.record_stream(stream)

    def alloc(self):
        return torch.cuda.stream(self.other) if self.other is not None else nullcontext()

    def done(self, status: int) -> None:
        if status != abi.HELIX_OK:
            raise HelixError(status, self.ctx.last_error())


def _empty8(shape, device) -> torch.Tensor:
    """float8 tensor of `shape` whose rows start at multiples of 16 bytes."""
    cols = shape[-1]
    held = torch.empty((*shape[:-1], -(-cols // 16) * 16), dtype=torch.float8_e4m3fn, device=device)
    return held if held.shape[-1] == cols else held[..., :cols]


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
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    d = abi.RmsNormDesc()
    d.n_row, d.n_col, d.eps = rows, cols, eps
    d.x_dtype = _dtype("x", x)
    d.ld_x = _matrix("x", x)
    d.sum_dtype = d.x_dtype
    if residual is not None:
        d.sum_dtype = _dtype("residual", residual)
        d.ld_res = _matrix("residual", residual, x.shape)
    _vector("weight", weight, cols)
    d.w_dtype = _dtype("weight", weight)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    try:
        d.out_dtype = _OUT[out_dtype]
    except KeyError:
        raise TypeError(f"out_dtype {out_dtype} is not supported") from None
    call = _Call(x, ctx, stream, residual, weight)
    total = scale = rstd = None
    with call.alloc():
        if out_dtype == torch.float8_e4m3fn:
            out = _empty8(x.shape, x.device)
            scale = torch.empty((*x.shape[:-1], _groups(cols)), dtype=torch.float32, device=x.device)
            d.ld_scale = scale.shape[-1]
            d.ld_out = -(-cols // 16) * 16
        else:
            out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
            d.ld_out = cols
        if residual is not None:
            total = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
            d.ld_sum = cols
        if keep_rstd:
            rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    call.done(call.ctx.lib.helix_rms_norm_encode(call.ctx.handle, call.handle, C.byref(d), _t(x), _t(residual),
                                                 _t(weight), _t(out), _t(scale), _t(total), _t(rstd)))
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
    cols = dout.shape[-1]
    rows = dout.numel() // cols if cols else 0
    d = abi.RmsNormDesc()
    d.n_row, d.n_col = rows, cols
    d.x_dtype, d.sum_dtype = _dtype("dout", dout), _dtype("sum", sum)
    d.ld_dout, d.ld_sum = _matrix("dout", dout), _matrix("sum", sum, dout.shape)
    if dsum is not None:
        if dsum.dtype != sum.dtype:
            raise TypeError("dsum must have sum's type")
        d.ld_dsum = _matrix("dsum", dsum, dout.shape)
    if rstd.dtype != torch.float32 or tuple(rstd.shape) != tuple(dout.shape[:-1]) or not rstd.is_contiguous():
        raise ValueError("rstd must be a dense float32 tensor with one value per row")
    _vector("weight", weight, cols)
    d.w_dtype = _dtype("weight", weight)
    call = _Call(dout, ctx, stream, sum, rstd, weight, dsum)
    dres = None
    with call.alloc():
        dx = torch.empty(dout.shape, dtype=dout.dtype, device=dout.device)
        dweight = torch.empty(cols, dtype=torch.float32, device=dout.device)
        d.ld_dx = cols
        if keep_dres and sum.dtype != dout.dtype:
            dres = torch.empty(dout.shape, dtype=sum.dtype, device=dout.device)
            d.ld_dres = cols
        nbytes = call.ctx.lib.helix_rms_norm_grad_scratch_size(call.ctx.handle, C.byref(d))
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dout.device) if nbytes else None
    call.done(call.ctx.lib.helix_rms_norm_grad_encode(
        call.ctx.handle, call.handle, C.byref(d), _t(dout), _t(sum), _t(rstd), _t(weight), _t(dsum), _t(dx),
        _t(dres), _t(dweight), _t(scratch)))
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
    d = abi.Quant8Desc()
    d.n_row, d.n_col = x.shape
    d.x_dtype = _dtype("x", x)
    d.ld_x = _matrix("x", x)
    d.form = abi.HELIX_SCALE_BLOCKS if blocks else abi.HELIX_SCALE_ROWS
    d.transpose = transpose
    rows, cols = (x.shape[1], x.shape[0]) if transpose else x.shape
    call = _Call(x, ctx, stream)
    with call.alloc():
        q = _empty8((rows, cols), x.device)
        scale = torch.empty((_groups(rows) if blocks else rows, _groups(cols)), dtype=torch.float32, device=x.device)
    d.ld_q = -(-cols // 16) * 16
    d.ld_scale = _groups(cols)
    call.done(call.ctx.lib.helix_quant8_encode(call.ctx.handle, call.handle, C.byref(d), _t(x), _t(q), _t(scale)))
    return q, scale


def matmul8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, *,
            out_dtype: torch.dtype = torch.bfloat16, ctx: Optional[Context] = None, stream=None) -> torch.Tensor:
    """a b^T of 8-bit matrices a (..., k) and b (n, k): (..., n) in out_dtype.

    a_scale (..., ceil(k / 128)); b_scale (ceil(n / 128), ceil(k / 128)) by
    blocks or (n, ceil(k / 128)) by rows.  Rows of a and b must start at
    multiples of 16 bytes, as rms_norm and quantize8 leave them."""
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn:
        raise TypeError("a and b must be torch.float8_e4m3fn")
    if a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32:
        raise TypeError("scales must be torch.float32")
    if b.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError("b must be a matrix with as many columns as a")
    n, k = b.shape
    groups = _groups(k)
    d = abi.Matmul8Desc()
    d.m, d.n, d.k = (a.numel() // k if k else 0), n, k
    d.ld_a, d.ld_b = _matrix("a", a), _matrix("b", b)
    d.ld_a_scale = _matrix("a_scale", a_scale, (*a.shape[:-1], groups))
    d.b_form = abi.HELIX_SCALE_ROWS if tuple(b_scale.shape) == (n, groups) else abi.HELIX_SCALE_BLOCKS
    d.ld_b_scale = _matrix("b_scale", b_scale, (n if d.b_form == abi.HELIX_SCALE_ROWS else _groups(n), groups))
    try:
        d.out_dtype = _IO[out_dtype]
    except KeyError:
        raise TypeError(f"out_dtype {out_dtype} is not supported") from None
    d.ld_out = n
    call = _Call(a, ctx, stream, a_scale, b, b_scale)
    with call.alloc():
        out = torch.empty((*a.shape[:-1], n), dtype=out_dtype, device=a.device)
    call.done(call.ctx.lib.helix_matmul8_encode(call.ctx.handle, call.handle, C.byref(d), _t(a), _t(a_scale), _t(b),
                                                _t(b_scale), _t(out)))
    return out


def _tokens(name: str, t: torch.Tensor, shape, dtype) -> tuple[int, int]:
    """(token stride, sequence stride) of a (sequences, tokens, channels) tensor."""
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}")
    s, k, c = t.stride()
    if shape[2] > 1 and c != 1:
        raise ValueError(f"{name} needs unit stride along the channels")
    return k, s


def _state(name: str, t: torch.Tensor, shape) -> int:
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be torch.float32")
    return _matrix(name, t, shape)


def _lengths(t: Optional[torch.Tensor], seqs: int) -> None:
    if t is not None:
        _vector("lengths", t, seqs, torch.int32)


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
    d = abi.GatedScanDesc()
    d.n_seq, d.n_tok, d.n_chan = seqs, toks, chans = v.shape
    d.io_dtype = _dtype("v", v)
    d.s_v, d.seq_v = _tokens("v", v, v.shape, v.dtype)
    d.s_g, d.seq_g = _tokens("g", g, v.shape, v.dtype)
    _lengths(lengths, seqs)
    if h0 is not None:
        d.seq_h0 = _state("h0", h0, (seqs, chans))
    call = _Call(v, ctx, stream, g, h0, lengths, h1)
    with call.alloc():
        y = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        if h1 is None:
            h1 = torch.empty((seqs, chans), dtype=torch.float32, device=v.device)
        states = None
        if keep_states:
            states = torch.empty((seqs, -(-toks // abi.HELIX_GATED_CHUNK), chans), dtype=torch.float32, device=v.device)
    d.s_y, d.seq_y = chans, toks * chans
    d.seq_h1 = _state("h1", h1, (seqs, chans))
    call.done(call.ctx.lib.helix_gated_scan_encode(call.ctx.handle, call.handle, C.byref(d), _t(v), _t(g), _t(h0),
                                                   _t(lengths), _t(y), _t(h1), _t(states)))
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
    d = abi.GatedScanDesc()
    d.n_seq, d.n_tok, d.n_chan = seqs, toks, chans = v.shape
    d.io_dtype = _dtype("v", v)
    d.s_v, d.seq_v = _tokens("v", v, v.shape, v.dtype)
    d.s_g, d.seq_g = _tokens("g", g, v.shape, v.dtype)
    d.s_dy, d.seq_dy = _tokens("dy", dy, v.shape, v.dtype)
    if (states.dtype != torch.float32 or not states.is_contiguous()
            or tuple(states.shape) != (seqs, -(-toks // abi.HELIX_GATED_CHUNK), chans)):
        raise ValueError("states must be what gated_scan(keep_states=True) gave")
    _lengths(lengths, seqs)
    if dh1 is not None:
        d.seq_dh1 = _state("dh1", dh1, (seqs, chans))
    call = _Call(dy, ctx, stream, v, g, states, dh1, lengths, dv, dg)
    with call.alloc():
        dv = torch.empty(v.shape, dtype=v.dtype, device=v.device) if dv is None else dv
        dg = torch.empty(v.shape, dtype=v.dtype, device=v.device) if dg is None else dg
        dh0 = torch.empty((seqs, chans), dtype=torch.float32, device=v.device)
    d.s_dv, d.seq_dv = _tokens("dv", dv, v.shape, v.dtype)
    d.s_dg, d.seq_dg = _tokens("dg", dg, v.shape, v.dtype)
    d.seq_dh0 = chans
    call.done(call.ctx.lib.helix_gated_scan_grad_encode(
        call.ctx.handle, call.handle, C.byref(d), _t(dy), _t(v), _t(g), _t(states), _t(dh1), _t(lengths), _t(dv),
        _t(dg), _t(dh0)))
    return dv, dg, dh0
