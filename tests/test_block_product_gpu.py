"""GPU: the product of 8-bit matrices with a scale for each block of 128,
against its definition in 64 bits.

Bound.  Products of e4m3 values are exact in fp32.  The tensor core adds the
128 of a block in fp32, possibly truncating: at most 2^-23 of the running sum
of magnitudes per addition of 32 products, so 5 u of it with slack (u = 2^-24)
doubled for alignment of the products to the largest: 16 u.  Scaling costs 3 u,
and the sum over B blocks B u.  All of it is relative to
M = sum_b sa sb sum_k |a b|; the output's rounding is relative to out.
"""
import ctypes as C

import pytest
import torch

import block_ref as ref
import helix_b200
from helix_b200 import abi

pytestmark = pytest.mark.gpu
BF, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _padded(q, extra=0):
    """q with rows at multiples of 16 bytes, `extra` 16s further apart; NaN between."""
    rows, cols = q.shape
    held = torch.full((rows, -(-cols // 16) * 16 + 16 * extra), 0x7F, dtype=torch.uint8, device=q.device)
    held[:, :cols] = q.view(torch.uint8)
    return held.view(F8)[:, :cols]


def _operand(g, rows, cols, blocks):
    q = (ref.rand(g, rows, cols) * 100).clamp(-448, 448).to(F8)
    shape = (-(-rows // 128) if blocks else rows, -(-cols // 128))
    scale = torch.exp2(torch.rand(shape, generator=g, dtype=torch.float64) * 6 - 10).float()
    return q, scale


def _want(a, sa, b, sb, blocks):
    m, k = a.shape
    n = b.shape[0]
    av = a.double() * ref.spread(sa.double(), m, k, False)
    bv = b.double() * ref.spread(sb.double(), n, k, blocks)
    return av @ bv.T, av.abs() @ bv.abs().T


def _check(cuda, m, n, k, blocks, out, extra=0, seed=0):
    g = ref.generator(seed + m + 10 * n + 100 * k)
    a, sa = _operand(g, m, k, False)
    b, sb = _operand(g, n, k, blocks)
    want, mag = _want(a, sa, b, sb, blocks)
    got = helix_b200.matmul8(_padded(a.to(cuda), extra), sa.to(cuda), _padded(b.to(cuda), extra), sb.to(cuda),
                             out_dtype=out)
    assert got.dtype == out
    groups = -(-k // 128)
    ref.within(got, want, mag * (19 + groups) * ref.U32 + want.abs() * ref.HALF[out], f"{m}x{n}x{k}")


SHAPES = [(1, 1, 1), (1, 128, 128), (3, 130, 128), (16, 256, 512), (17, 129, 100), (5, 64, 1000), (32, 384, 640),
          (33, 1, 300), (64, 257, 4096), (16, 512, 4096), (65, 200, 128), (100, 100, 100), (128, 128, 2048),
          (129, 127, 129), (200, 1000, 384), (256, 256, 256), (300, 520, 1111), (513, 384, 640), (1000, 16, 256)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("blocks", [True, False])
@pytest.mark.parametrize("out", [BF, F32])
def test_product(cuda, ctx, m, n, k, blocks, out):
    _check(cuda, m, n, k, blocks, out)
    code = C.c_uint32(99)
    assert ctx.lib.helix_device_fault(ctx.handle, C.byref(code)) == abi.HELIX_OK and code.value == 0


@pytest.mark.parametrize("m,n,k", [(2000, 1500, 768), (1024, 2048, 1024), (2304, 2560, 512), (4100, 3001, 260)])
@pytest.mark.parametrize("blocks", [True, False])
@pytest.mark.parametrize("out", [BF, F32])
def test_product_many_tiles(cuda, m, n, k, blocks, out):
    _check(cuda, m, n, k, blocks, out)


@pytest.mark.parametrize("m", [1, 16, 40, 150, 700])
def test_strides_and_leading_dimensions(cuda, m):
    """Rows further apart than k (NaN between them), a with leading
    dimensions, scales and out with row strides of their own."""
    _check(cuda, m, 300, 333, True, BF, extra=3)
    g = ref.generator(8)
    a, sa = _operand(g, 6, 256, False)
    b, sb = _operand(g, 90, 256, True)
    got = helix_b200.matmul8(a.to(cuda).view(2, 3, 256), sa.to(cuda).view(2, 3, 2), b.to(cuda), sb.to(cuda),
                             out_dtype=F32)
    want, mag = _want(a, sa, b, sb, True)
    assert got.shape == (2, 3, 90)
    ref.within(got.view(6, 90), want, mag * 21 * ref.U32 + want.abs() * ref.U32, "leading")


@pytest.mark.parametrize("k,pitch", [(512, 4), (1536, 12), (700, 8), (700, 6), (700, 7), (1100, 12), (128, 4)])
@pytest.mark.parametrize("m,n,out", [(2048, 1280, F32), (1100, 1281, BF)])
def test_scale_strides(cuda, ctx, m, n, k, pitch, out):
    """Scales by rows whose rows are whole pieces of 16 bytes, or not, NaN
    between them: a piece's part past the last block counts for nothing."""
    g = ref.generator(k + pitch)
    a, sa = _operand(g, m, k, False)
    b, sb = _operand(g, n, k, False)
    want, mag = _want(a, sa, b, sb, False)
    groups = -(-k // 128)
    wide = []
    for s in (sa, sb):
        w = torch.full((s.shape[0], pitch), float("nan"), device=cuda)
        w[:, :groups] = s.to(cuda)
        wide.append(w)
    d = abi.Matmul8Desc()
    ctx.lib.helix_matmul8_desc_init(C.byref(d), m, n, k, abi.HELIX_SCALE_ROWS)
    d.out_dtype = abi.HELIX_F32 if out == F32 else abi.HELIX_BF16
    d.ld_a_scale = d.ld_b_scale = pitch
    T = helix_b200._t
    ag, bg = _padded(a.to(cuda)), _padded(b.to(cuda))
    got = torch.empty(m, n, dtype=out, device=cuda)
    st = ctx.lib.helix_matmul8_encode(ctx.handle, torch.cuda.current_stream().cuda_stream, C.byref(d), T(ag),
                                      T(wide[0]), T(bg), T(wide[1]), T(got))
    assert st == abi.HELIX_OK, ctx.last_error()
    ref.within(got, want, mag * (19 + groups) * ref.U32 + want.abs() * ref.HALF[out], f"{m}x{n}x{k}")


@pytest.mark.parametrize("m,swap_out", [(20, False), (300, False), (20, True), (300, True)])
def test_output_strides(cuda, ctx, m, swap_out):
    """out as rows of a wider buffer at an odd offset: nothing beside it is touched."""
    n, k = 203, 384
    g = ref.generator(m)
    a, sa = _operand(g, m, k, False)
    b, sb = _operand(g, n, k, not swap_out)
    want, mag = _want(a, sa, b, sb, not swap_out)
    held = torch.full((m, n + 37), 7.0, dtype=F32, device=cuda)
    out = held[:, 5:5 + n]
    d = abi.Matmul8Desc()
    ctx.lib.helix_matmul8_desc_init(C.byref(d), m, n, k, abi.HELIX_SCALE_ROWS if swap_out else abi.HELIX_SCALE_BLOCKS)
    d.out_dtype, d.ld_out = abi.HELIX_F32, n + 37
    wide = torch.zeros(m, 9, device=cuda)
    wide[:, :3] = sa.to(cuda)
    d.ld_a_scale = 9
    T = helix_b200._t
    ag, bg, sbg = a.to(cuda), b.to(cuda), sb.to(cuda)
    st = ctx.lib.helix_matmul8_encode(ctx.handle, torch.cuda.current_stream().cuda_stream, C.byref(d), T(ag), T(wide),
                                      T(bg), T(sbg), T(out))
    assert st == abi.HELIX_OK, ctx.last_error()
    ref.within(out, want, mag * 22 * ref.U32 + want.abs() * ref.U32, "out")
    held[:, 5:5 + n] = 7.0
    assert (held == 7.0).all()


@pytest.mark.parametrize("m", [4, 200])
def test_nan_stays_in_its_row_and_column(cuda, m):
    n, k = 140, 300
    g = ref.generator(77)
    a, sa = _operand(g, m, k, False)
    b, sb = _operand(g, n, k, True)
    a.view(torch.uint8)[2, 130] = 0x7F
    sa[3, 1] = float("inf")
    got = helix_b200.matmul8(_padded(a.to(cuda)), sa.to(cuda), _padded(b.to(cuda)), sb.to(cuda), out_dtype=F32)
    bad = ~got.cpu().isfinite()
    assert bad[2].all() and bad[3].all()
    bad[2:4] = False
    assert not bad.any()


def test_backward_products(cuda):
    """dX = dY W and dW = dY^T X from operands the quantiser lays out,
    against the products of the very 8-bit values."""
    m, n, k = 333, 260, 400
    g = ref.generator(5)
    x, w, dy = ref.rand(g, m, k).to(BF), ref.rand(g, n, k).float(), ref.rand(g, m, n).to(BF)
    qd, sd = helix_b200.quantize8(dy.to(cuda))
    qw, sw = helix_b200.quantize8(w.to(cuda), blocks=True, transpose=True)
    dx = helix_b200.matmul8(qd, sd, qw, sw, out_dtype=F32)
    want, mag = _want(qd.cpu(), sd.cpu(), qw.cpu(), sw.cpu(), True)
    ref.within(dx, want, mag * 24 * ref.U32 + want.abs() * ref.U32, "dx")
    qd, sd = helix_b200.quantize8(dy.to(cuda), transpose=True)
    qx, sx = helix_b200.quantize8(x.to(cuda), transpose=True)
    dw = helix_b200.matmul8(qd, sd, qx, sx, out_dtype=F32)
    assert dw.shape == (n, k)
    want, mag = _want(qd.cpu(), sd.cpu(), qx.cpu(), sx.cpu(), False)
    ref.within(dw, want, mag * 24 * ref.U32 + want.abs() * ref.U32, "dw")
    # 8 bits themselves: two roundings of 2^-4 a product, random over m
    exact = dy.double().T @ x.double()
    assert (dw.double().cpu() - exact).norm() <= 0.06 * exact.norm()


def test_the_same_twice(cuda):
    for m, n, k in ((16, 8192, 2048), (200, 300, 2048), (1500, 1500, 640)):
        g = ref.generator(m)
        a, sa = _operand(g, m, k, False)
        b, sb = _operand(g, n, k, True)
        args = [t.to(cuda) for t in (a, sa, b, sb)]
        assert torch.equal(helix_b200.matmul8(*args), helix_b200.matmul8(*args))


def test_captured_and_on_another_stream(cuda):
    g = ref.generator(2)
    a, sa = _operand(g, 24, 512, False)
    b, sb = _operand(g, 300, 512, True)
    want, mag = _want(a, sa, b, sb, True)
    args = [t.to(cuda) for t in (a, sa, b, sb)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = helix_b200.matmul8(*args, out_dtype=F32, stream=side)
    side.synchronize()
    ref.within(got, want, mag * 23 * ref.U32 + want.abs() * ref.U32, "side")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = helix_b200.matmul8(*args, out_dtype=F32)
    a2, sa2 = _operand(ref.generator(3), 24, 512, False)
    args[0].copy_(a2), args[1].copy_(sa2)
    graph.replay()
    torch.cuda.synchronize()
    want, mag = _want(a2, sa2, b, sb, True)
    ref.within(got, want, mag * 23 * ref.U32 + want.abs() * ref.U32, "graph")
    del graph


def test_refusals(cuda, ctx):
    a = torch.zeros(4, 256, dtype=torch.uint8, device=cuda).view(F8)
    s = torch.ones(4, 2, device=cuda)
    with pytest.raises(TypeError):
        helix_b200.matmul8(a.float(), s, a, s)
    with pytest.raises(TypeError):
        helix_b200.matmul8(a, s.double(), a, s)
    with pytest.raises(TypeError):
        helix_b200.matmul8(a, s, a, s, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        helix_b200.matmul8(a, s, a[:, :128], s)
    with pytest.raises(ValueError):
        helix_b200.matmul8(a, s[:3], a, s)
    with pytest.raises(ValueError):
        helix_b200.matmul8(a, s, a, s[:2])
    odd = torch.zeros(4, 250, dtype=torch.uint8, device=cuda).view(F8)
    with pytest.raises(helix_b200.HelixError, match="16-byte"):
        helix_b200.matmul8(odd, s, odd, s)
    with pytest.raises(helix_b200.HelixError, match="16-byte"):
        helix_b200.matmul8(a[:, 1:], s, a[:, 1:], s)
    T, st = helix_b200._t, torch.cuda.current_stream().cuda_stream
    out = torch.empty(4, 4, dtype=BF, device=cuda)

    def call(field=None, value=None, args=None):
        d = abi.Matmul8Desc()
        ctx.lib.helix_matmul8_desc_init(C.byref(d), 4, 4, 256, abi.HELIX_SCALE_ROWS)
        if field:
            setattr(d, field, value)
        return ctx.lib.helix_matmul8_encode(ctx.handle, st, C.byref(d), *(args or [T(a), T(s), T(a), T(s), T(out)]))

    assert call() == abi.HELIX_OK
    for field, value, status in (("m", -1, 1), ("k", 0, 1), ("b_form", 5, 1), ("out_dtype", abi.HELIX_F16, 1),
                                 ("out_dtype", abi.HELIX_E4M3, 1), ("ld_out", 3, 4), ("ld_a", 240, 4), ("ld_b", 8, 1),
                                 ("m", 2 ** 31 - 1, 1)):
        assert call(field, value) == status, field
    for i in range(5):
        args = [T(a), T(s), T(a), T(s), T(out)]
        args[i] = T(None)
        assert call(args=args) == abi.HELIX_ERR_INVALID_ARG and "null" in ctx.last_error()
    assert call(args=[T(a), T(s), T(a), T(s), T(a)]) == abi.HELIX_ERR_INVALID_ARG
    assert call(args=[T(a), T(s), T(a), T(s), T(s)]) == abi.HELIX_ERR_INVALID_ARG
    assert call("m", 0) == abi.HELIX_OK and call("n", 0) == abi.HELIX_OK
    assert helix_b200.matmul8(a[:0], s[:0], a, s).shape == (0, 4)
    torch.cuda.synchronize()
