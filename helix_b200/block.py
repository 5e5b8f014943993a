"""The operators of a recurrent block on torch tensors (include/helix/helix_block.h).

Each function makes one call of the C ABI on the tensors' device and on
`stream` (a torch.cuda.Stream, a raw handle, or None for torch's current
stream); the checks of its tensors and the allocation of its outputs and
scratch are in the extension module _block_torch (csrc/torch).  There is no
compute here and no fallback: what the library refuses raises HelixError, a
tensor of the wrong shape or device ValueError, one of the wrong type TypeError.
No autograd graph is recorded, whatever the tensors require: outputs are without
one, and the gradients are calls of their own.

8-bit tensors are torch.float8_e4m3fn with an fp32 scale per 128 columns of a
row (or per 128 x 128 block); their rows are padded to whole 16 bytes, which is
what the product needs of its operands.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import Context, _default_ctx, abi

abi.load()  # a missing library says how to build it
from . import _block_torch as _native  # noqa: E402


def _ctx(ctx: Optional[Context], t: torch.Tensor) -> int:
    """The helix_ctx of a call, as an integer; one per device without `ctx`."""
    index = t.get_device() if isinstance(t, torch.Tensor) else -1
    if index < 0:
        raise ValueError("tensors must be on a CUDA device")
    if ctx is None:
        ctx = _default_ctx.get(index)
        if ctx is None:
            ctx = _default_ctx.setdefault(index, Context(index))
    elif ctx.device is not None and ctx.device != index:
        raise ValueError(f"the context is of device {ctx.device}, the tensors are on device {index}")
    return ctx.handle.value


def _call(stream, fn, handle: int, *args):
    """fn on the current stream, or on `stream`.  There the outputs are
    allocated for that stream, and the tensors passed may be freed before it
    gets to the call."""
    if stream is None:
        return fn(handle, *args)
    tensors = [a for a in args if isinstance(a, torch.Tensor)]
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=tensors[0].device)
    if stream.cuda_stream != torch.cuda.current_stream(tensors[0].device).cuda_stream:
        for t in tensors:
            t.record_stream(stream)
    with torch.cuda.stream(stream):
        return fn(handle, *args)


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
    return Norm._make(_call(stream, _native.rms_norm, _ctx(ctx, x), x, weight, residual, eps, out_dtype, keep_rstd))


def rms_norm_grad(dout: torch.Tensor, sum: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor,
                  dsum: Optional[torch.Tensor] = None, *, keep_dres: bool = False, ctx: Optional[Context] = None,
                  stream=None):
    """Gradient of rms_norm: (dx, dweight), or (dx, dweight, dres) with
    keep_dres.

    dout is the gradient of the norm's output in x's type (rounding to 8 bits
    is passed through), dsum the one that reaches sum by another way; sum and
    rstd are what the forward pass gave.  dx has dout's type and dres, the
    same gradient for the residual, sum's (where that is dout's, it is dx
    itself); dweight is f32."""
    return _call(stream, _native.rms_norm_grad, _ctx(ctx, dout), dout, sum, rstd, weight, dsum, keep_dres)


def quantize8(x: torch.Tensor, *, blocks: bool = False, transpose: bool = False, ctx: Optional[Context] = None,
              stream=None):
    """The matrix x, or x transposed, in 8 bits: (q, scale).

    One scale per 128 columns of each of q's rows, or per 128 x 128 block.
    transpose lays an operand out for the products of a backward pass: blocks
    of a weight, or (by rows) 128 tokens of a column under one scale."""
    return _call(stream, _native.quantize8, _ctx(ctx, x), x, blocks, transpose)


def matmul8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, *,
            out_dtype: torch.dtype = torch.bfloat16, ctx: Optional[Context] = None, stream=None) -> torch.Tensor:
    """a b^T of 8-bit matrices a (..., k) and b (n, k): (..., n) in out_dtype.

    a_scale (..., ceil(k / 128)); b_scale (ceil(n / 128), ceil(k / 128)) by
    blocks or (n, ceil(k / 128)) by rows.  Rows of a and b must start at
    multiples of 16 bytes, as rms_norm and quantize8 leave them."""
    return _call(stream, _native.matmul8, _ctx(ctx, a), a, a_scale, b, b_scale, out_dtype)


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
    return _call(stream, _native.gated_scan, _ctx(ctx, v), v, g, h0, lengths, h1, keep_states)


def gated_scan_grad(dy: torch.Tensor, v: torch.Tensor, g: torch.Tensor, states: torch.Tensor,
                    dh1: Optional[torch.Tensor] = None, *, lengths: Optional[torch.Tensor] = None,
                    dv: Optional[torch.Tensor] = None, dg: Optional[torch.Tensor] = None,
                    ctx: Optional[Context] = None, stream=None):
    """Gradient of gated_scan: (dv, dg, dh0) from the gradients of y and of h1
    (zeros without), with the states the forward pass kept.  dv and dg are
    written into the tensors given (slices of one wider tensor, say) or new ones."""
    return _call(stream, _native.gated_scan_grad, _ctx(ctx, v), dy, v, g, states, dh1, lengths, dv, dg)
