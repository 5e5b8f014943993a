"""GPU: the RMS norm with the residual's addition, its 8-bit output, its
gradient, and the 8-bit quantiser, against their definitions in 64 bits.

Bounds.  A row's sum of squares is a chain of at most 32 additions in a lane,
5 in a warp and 16 across warps, so mean(s^2) is within 54 u of its value
(u = 2^-24) and rstd within 27 u + 3 u; with s (1 u), the products (2 u) a
value of n is within 40 u of the definition's, and one rounding to its type.
The gradient's mean is such a chain too; every term of ds carries at most 64 u
of its own magnitude.  dweight adds the rows of a slot in a chain (rows / 148
here at most) and the slots in two short ones.
"""
import ctypes as C

import pytest
import torch

import block_ref as ref
import helix_b200
from helix_b200 import abi

pytestmark = pytest.mark.gpu
BF, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
K = 40 * ref.U32

SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 127), (17, 128), (33, 129), (2, 255), (9, 256), (6, 257), (4, 1000),
          (70, 2501), (11, 8192), (3, 8200), (2, 16383), (1, 16384), (1000, 64), (300, 520)]
TYPES = [(BF, BF), (BF, F32), (F32, F32)]


def _pad(t, extra, dev, offset=0):
    """t on the GPU as a view with rows `extra` elements further apart, the
    first one `offset` elements into its memory; NaN around it."""
    rows, cols = t.shape
    held = torch.full((rows * (cols + extra) + offset,), float("nan"), dtype=t.dtype, device=dev)
    v = held[offset:].view(rows, cols + extra)[:, :cols]
    v.copy_(t)
    return v


def _inputs(seed, rows, cols, tx, tr):
    g = ref.generator(seed)
    x = ref.rand(g, rows, cols).to(tx)
    res = ref.rand(g, rows, cols, std=3.0).to(tr)
    w = ref.rand(g, cols, std=0.2, mean=1.0).float()
    return x, res, w


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("tx,tr", TYPES)
@pytest.mark.parametrize("out", ["e4m3", "x", "f32"])
def test_norm(cuda, rows, cols, tx, tr, out):
    to = {"e4m3": F8, "x": tx, "f32": F32}[out]
    x, res, w = _inputs(rows * 1000 + cols, rows, cols, tx, tr)
    for residual in (res, None):
        s, rstd, n = ref.norm(x.double(), None if residual is None else residual.double(), w.double(), 1e-5)
        got = helix_b200.rms_norm(x.to(cuda), w.to(cuda), None if residual is None else residual.to(cuda), eps=1e-5,
                                  out_dtype=to, keep_rstd=True)
        ref.within(got.rstd, rstd, rstd * K, "rstd")
        if residual is not None:
            assert got.sum.dtype == tr
            ref.within(got.sum, s, s.abs() * (ref.HALF[tr] + ref.U32), "sum")
        if to == F8:
            ref.check_8bit(got.out, got.scale, n, K, False, "out")
        else:
            ref.within(got.out, n, n.abs() * (K + ref.HALF[to]), "out")


@pytest.mark.parametrize("extra,offset", [(8, 0), (1, 0), (8, 8), (3, 1), (4, 4)])
@pytest.mark.parametrize("tx,tr", TYPES)
def test_norm_strides(cuda, extra, offset, tx, tr):
    """Row strides and bases of every alignment, a bf16 weight, leading
    dimensions; what lies between the rows is NaN and stays out."""
    rows, cols = 12, 392
    x, res, w = _inputs(7, rows, cols, tx, tr)
    w = w.to(BF)
    xs, rs = _pad(x, extra, cuda, offset), _pad(res, extra, cuda, offset)
    s, _, n = ref.norm(x.double(), res.double(), w.double(), 1e-6)
    for shape in ((rows, cols), (3, 4, cols)):
        v = xs if len(shape) == 2 else xs.unflatten(0, shape[:-1])
        r = rs if len(shape) == 2 else rs.unflatten(0, shape[:-1])
        got = helix_b200.rms_norm(v, w.to(cuda), r, out_dtype=F8)
        assert tuple(got.out.shape) == shape and tuple(got.sum.shape) == shape
        ref.check_8bit(got.out.flatten(0, -2), got.scale.flatten(0, -2), n, K, False, "out")
        ref.within(got.sum.flatten(0, -2), s, s.abs() * (ref.HALF[tr] + ref.U32), "sum")


def test_norm_special_rows(cuda):
    """Zeros, the largest and smallest magnitudes, NaN and infinity stay in
    their rows (and, in 8 bits, their effect in the row)."""
    cols = 300
    x = ref.rand(ref.generator(3), 7, cols).float()
    x[0] = 0.0
    x[1] = 1e-30
    x[2, 5] = float("nan")
    x[3, 290] = float("inf")
    x[4] = 1e18
    x[5] *= 0.0
    x[5, 0] = 1.0  # groups of zeros beside one that is not
    w = torch.ones(cols)
    s, rstd, n = ref.norm(x.double(), None, w.double(), 1e-6)
    got = helix_b200.rms_norm(x.to(cuda), w.to(cuda), eps=1e-6)
    ref.within(got.out, n, n.abs() * (K + ref.U32), "out")
    got = helix_b200.rms_norm(x.to(cuda), w.to(cuda), eps=1e-6, out_dtype=F8)
    q, sc = got.out.float().cpu(), got.scale.cpu()
    keep = [0, 1, 4, 5, 6]
    ref.check_8bit(got.out[keep], got.scale[keep], n[keep], K, False, "out")
    assert q[2].isnan().all() and sc[2].isnan().all()
    assert q[3, 290].isnan() and (q[3, :256] == 0).all()


def test_norm_in_place(cuda, ctx):
    """sum in place of the residual, and of x."""
    rows, cols = 40, 640
    for tx, tr, where in ((BF, F32, "res"), (BF, BF, "res"), (BF, BF, "x"), (F32, F32, "x")):
        x, res, w = _inputs(5, rows, cols, tx, tr)
        s, _, n = ref.norm(x.double(), res.double(), w.double(), 1e-6)
        xg, rg, wg = x.to(cuda), res.to(cuda), w.to(cuda)
        out = torch.empty_like(xg)
        d = abi.RmsNormDesc()
        ctx.lib.helix_rms_norm_desc_init(C.byref(d), rows, cols)
        d.x_dtype = d.out_dtype = abi.HELIX_BF16 if tx == BF else abi.HELIX_F32
        d.sum_dtype = abi.HELIX_BF16 if tr == BF else abi.HELIX_F32
        total = rg if where == "res" else xg
        T = helix_b200._t
        st = ctx.lib.helix_rms_norm_encode(ctx.handle, torch.cuda.current_stream().cuda_stream, C.byref(d), T(xg),
                                           T(rg), T(wg), T(out), T(None), T(total), T(None))
        assert st == abi.HELIX_OK, ctx.last_error()
        ref.within(total, s, s.abs() * (ref.HALF[tr] + ref.U32), "sum")
        ref.within(out, n, n.abs() * (K + ref.HALF[tx]), "out")


@pytest.mark.parametrize("rows,cols", SHAPES + [(0, 100), (3000, 200), (700, 4096)])
@pytest.mark.parametrize("tx,tr", TYPES)
@pytest.mark.parametrize("with_dsum", [False, True])
def test_norm_grad(cuda, rows, cols, tx, tr, with_dsum):
    g = ref.generator(rows * 77 + cols)
    s = ref.rand(g, rows, cols, std=2.0).to(tr)
    dout = ref.rand(g, rows, cols).to(tx)
    dsum = ref.rand(g, rows, cols).to(tr) if with_dsum else None
    w = ref.rand(g, cols, std=0.2, mean=1.0).float()
    rstd = (1.0 / torch.sqrt(s.double().square().mean(1) + 1e-6)).float()
    ds, dw, mag, dwmag = ref.norm_grad(dout.double(), s.double(), rstd.double(), w.double(),
                                       None if dsum is None else dsum.double())
    dx, dweight, dres = helix_b200.rms_norm_grad(dout.to(cuda), s.to(cuda), rstd.to(cuda), w.to(cuda),
                                                 None if dsum is None else dsum.to(cuda), keep_dres=True)
    assert dx.dtype == tx and dres.dtype == tr
    ref.within(dx, ds, mag * 64 * ref.U32 + ds.abs() * ref.HALF[tx], "dx")
    ref.within(dres, ds, mag * 64 * ref.U32 + ds.abs() * ref.HALF[tr], "dres")
    ref.within(dweight, dw, dwmag * (rows / 148 + 64) * ref.U32, "dweight")
    again = helix_b200.rms_norm_grad(dout.to(cuda), s.to(cuda), rstd.to(cuda), w.to(cuda),
                                     None if dsum is None else dsum.to(cuda))[1]
    assert torch.equal(dweight, again)


@pytest.mark.parametrize("extra,offset", [(8, 8), (1, 3), (4, 0)])
def test_norm_grad_strides(cuda, extra, offset):
    rows, cols = 21, 392
    g = ref.generator(4)
    s, dout, dsum = (ref.rand(g, rows, cols).to(t) for t in (F32, BF, F32))
    w = ref.rand(g, cols, std=0.2, mean=1.0).to(BF)
    rstd = (1.0 / torch.sqrt(s.double().square().mean(1) + 1e-6)).float()
    ds, dw, mag, dwmag = ref.norm_grad(dout.double(), s.double(), rstd.double(), w.double(), dsum.double())
    dx, dweight = helix_b200.rms_norm_grad(_pad(dout, extra, cuda, offset), _pad(s, extra, cuda, offset),
                                           rstd.to(cuda), w.to(cuda), _pad(dsum, extra, cuda, offset))
    ref.within(dx, ds, mag * 64 * ref.U32 + ds.abs() * ref.U16, "dx")
    ref.within(dweight, dw, dwmag * 65 * ref.U32, "dweight")


def test_norm_grad_against_differences(cuda):
    """The gradient along random directions against central differences of
    the definition in 64 bits: L = <out, dout> + <sum, dsum>.  The step 1e-5
    leaves 1e-9 of truncation and rounding; the kernel's own error is fp32."""
    rows, cols, eps = 6, 333, 1e-6
    g = ref.generator(12)
    x, res, dout, dsum = (ref.rand(g, rows, cols).float() for _ in range(4))
    w = ref.rand(g, cols, std=0.2, mean=1.0).float()
    n = helix_b200.rms_norm(x.to(cuda), w.to(cuda), res.to(cuda), eps=eps, keep_rstd=True)
    dx, dw = helix_b200.rms_norm_grad(dout.to(cuda), n.sum, n.rstd, w.to(cuda), dsum.to(cuda))

    def loss(xd, wd):
        s, _, out = ref.norm(xd, res.double(), wd, eps)
        return (out * dout.double()).sum() + (s * dsum.double()).sum()

    for k in range(4):
        px, pw = ref.rand(g, rows, cols), ref.rand(g, cols)
        h = 1e-5
        want = (loss(x.double() + h * px, w.double() + h * pw) - loss(x.double() - h * px, w.double() - h * pw)) / (2 * h)
        got = (dx.double().cpu() * px).sum() + (dw.double().cpu() * pw).sum()
        scale = dx.double().cpu().norm() * px.norm() + dw.double().cpu().norm() * pw.norm()
        assert abs(got - want) <= 1e-6 * scale


QSHAPES = [(1, 1), (1, 500), (5, 128), (128, 128), (129, 127), (300, 260), (16, 4096), (1000, 33), (257, 1111)]


@pytest.mark.parametrize("rows,cols", QSHAPES)
@pytest.mark.parametrize("tx", [BF, F32])
@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("extra,offset", [(0, 0), (3, 1)])
def test_quantize(cuda, rows, cols, tx, blocks, turn, extra, offset):
    g = ref.generator(rows + 3 * cols)
    x = ref.rand(g, rows, cols).to(tx)
    x[:, :: max(1, cols // 3)] *= 30
    x[rows // 2] = 0.0
    q, scale = helix_b200.quantize8(_pad(x, extra, cuda, offset), blocks=blocks, transpose=turn)
    v = x.double().T if turn else x.double()
    assert q.stride(0) % 16 == 0 or q.shape[0] == 1
    ref.check_8bit(q, scale, v, 2 * ref.U32, blocks, "x")


def test_quantize_nan_and_infinity(cuda):
    x = ref.rand(ref.generator(1), 256, 256).float()
    x[3, 5] = float("nan")
    x[200, 130] = float("-inf")
    for blocks in (False, True):
        for turn in (False, True):
            q, scale = helix_b200.quantize8(x.to(cuda), blocks=blocks, transpose=turn)
            q, scale = q.float().cpu(), scale.cpu()
            if turn:
                q, scale = q.T, scale.T
            # the group of the NaN is NaN, that of the infinity zeros and a NaN
            group = (slice(0, 128), slice(0, 128)) if blocks else ((slice(0, 128), 5) if turn else (3, slice(0, 128)))
            assert q[group].isnan().all()
            other = (slice(128, 256), slice(128, 256)) if blocks else (
                (slice(128, 256), 130) if turn else (200, slice(128, 256)))
            left = q[other].clone()
            assert int(left.isnan().sum()) == 1 and (left[~left.isnan()] == 0).all()
            clean = q.clone()
            clean[group] = 0.0
            clean[other] = 0.0
            assert clean.isfinite().all()
            assert int(scale.isnan().sum()) == 1 and int(scale.isinf().sum()) == 1


def test_another_stream(cuda):
    """Outputs written on a stream of the caller's, inputs freed at once."""
    x, res, w = _inputs(2, 512, 4096, BF, BF)
    s, _, n = ref.norm(x.double(), res.double(), w.double(), 1e-6)
    side = torch.cuda.Stream()
    xg, rg, wg = x.to(cuda), res.to(cuda), w.to(cuda)
    side.wait_stream(torch.cuda.current_stream())
    got = helix_b200.rms_norm(xg, wg, rg, out_dtype=F8, stream=side)
    q, sc = helix_b200.quantize8(rg, stream=side.cuda_stream)
    del xg, rg, wg
    torch.full((512, 4096), float("nan"), dtype=BF, device=cuda)
    side.synchronize()
    ref.check_8bit(got.out, got.scale, n, K, False, "out")
    ref.check_8bit(q, sc, res.double(), 2 * ref.U32, False, "q")


def test_captured_in_a_graph(cuda):
    x, res, w = _inputs(9, 64, 1024, BF, F32)
    xg, rg, wg = x.to(cuda), res.to(cuda), w.to(cuda)
    helix_b200.rms_norm(xg, wg, rg, out_dtype=F8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = helix_b200.rms_norm(xg, wg, rg, out_dtype=F8, keep_rstd=True)
        dx, dw = helix_b200.rms_norm_grad(xg, got.sum, got.rstd, wg)
        q, sc = helix_b200.quantize8(xg, transpose=True)
    x2 = ref.rand(ref.generator(10), 64, 1024).to(BF)
    xg.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    s, rstd, n = ref.norm(x2.double(), res.double(), w.double(), 1e-6)
    ref.check_8bit(got.out, got.scale, n, K, False, "out")
    ref.check_8bit(q, sc, x2.double().T, 2 * ref.U32, False, "q")
    ds, dwr, mag, dwmag = ref.norm_grad(x2.double(), got.sum.double().cpu(), got.rstd.double().cpu(), w.double(), None)
    ref.within(dx, ds, mag * 64 * ref.U32 + ds.abs() * ref.U16, "dx")
    ref.within(dw, dwr, dwmag * 65 * ref.U32, "dw")
    del graph


def test_refusals(cuda, ctx):
    x = torch.ones(4, 256, device=cuda)
    w = torch.ones(256, device=cuda)
    with pytest.raises(ValueError):
        helix_b200.rms_norm(x, w[:255])
    with pytest.raises(ValueError):
        helix_b200.rms_norm(x.T, torch.ones(4, device=cuda))
    with pytest.raises(ValueError):
        helix_b200.rms_norm(x, w, x[:3])
    with pytest.raises(TypeError):
        helix_b200.rms_norm(x.half(), w)
    with pytest.raises(TypeError):
        helix_b200.rms_norm(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        helix_b200.rms_norm(x, w.cpu())
    with pytest.raises(ValueError):
        helix_b200.rms_norm_grad(x, x, torch.ones(3, device=cuda), w)
    with pytest.raises(helix_b200.HelixError, match="sum_dtype"):  # an fp32 x cannot feed a bf16 residual stream
        helix_b200.rms_norm(x, w, x.bfloat16())
    with pytest.raises(helix_b200.HelixError, match="16384"):
        helix_b200.rms_norm(torch.ones(1, 16385, device=cuda), torch.ones(16385, device=cuda))
    with pytest.raises(helix_b200.HelixError, match="eps"):
        helix_b200.rms_norm(x, w, eps=-1.0)
    with pytest.raises(helix_b200.HelixError, match="eps"):
        helix_b200.rms_norm(x, w, eps=float("nan"))
    with pytest.raises(ValueError):
        helix_b200.quantize8(x[0])

    # through the C ABI: nulls, alignment, overlaps
    T, st = helix_b200._t, torch.cuda.current_stream().cuda_stream
    out, total = torch.empty_like(x), torch.empty_like(x)

    def call(d, **kw):
        a = dict(x=T(x), residual=T(None), weight=T(w), out=T(out), scale=T(None), sum=T(None), rstd=T(None))
        a.update(kw)
        return ctx.lib.helix_rms_norm_encode(ctx.handle, st, C.byref(d), *a.values())

    d = abi.RmsNormDesc()
    ctx.lib.helix_rms_norm_desc_init(C.byref(d), 4, 256)
    assert call(d) == abi.HELIX_OK
    for kw, word in ((dict(x=T(None)), "null"), (dict(out=T(None)), "null"), (dict(weight=T(None)), "null"),
                     (dict(x=abi.Tensor(x.data_ptr(), 2)), "aligned"), (dict(out=T(x)), "overlaps"),
                     (dict(sum=abi.Tensor(x.data_ptr(), 16)), "overlaps"), (dict(sum=T(total), rstd=T(total)), "overlaps"),
                     (dict(out=T(w)), "overlaps")):
        assert call(d, **kw) == abi.HELIX_ERR_INVALID_ARG, kw
        assert word in ctx.last_error(), ctx.last_error()
    d.out_dtype = abi.HELIX_E4M3
    assert call(d) == abi.HELIX_ERR_INVALID_ARG and "scale" in ctx.last_error()
    for field, value, status in (("n_row", -1, 1), ("n_col", 0, 1), ("x_dtype", abi.HELIX_F16, 1), ("out_dtype", 7, 1),
                                 ("w_dtype", abi.HELIX_E4M3, 1), ("ld_out", 255, 4), ("ld_x", -256, 4)):
        ctx.lib.helix_rms_norm_desc_init(C.byref(d), 4, 256)
        setattr(d, field, value)
        assert call(d) == status, field
    ctx.lib.helix_rms_norm_desc_init(C.byref(d), 4, 256)
    assert ctx.lib.helix_rms_norm_encode(None, st, C.byref(d), *[T(x)] * 7) == abi.HELIX_ERR_INVALID_ARG
    assert ctx.lib.helix_rms_norm_encode(ctx.handle, st, None, *[T(x)] * 7) == abi.HELIX_ERR_INVALID_ARG
    args = [T(x), T(x), T(w), T(w), T(None), T(out), T(None), T(w)]
    assert ctx.lib.helix_rms_norm_grad_encode(ctx.handle, st, C.byref(d), *args,
                                              T(None)) == abi.HELIX_ERR_SCRATCH_TOO_SMALL
    q = abi.Quant8Desc()
    ctx.lib.helix_quant8_desc_init(C.byref(q), 4, 256, 2, False)
    assert ctx.lib.helix_quant8_encode(ctx.handle, st, C.byref(q), T(x), T(out), T(total)) == 1
    ctx.lib.helix_quant8_desc_init(C.byref(q), 4, 256, 0, True)
    q.ld_q = 3
    assert ctx.lib.helix_quant8_encode(ctx.handle, st, C.byref(q), T(x), T(out), T(total)) == 4
    torch.cuda.synchronize()


def test_zero_rows(cuda):
    x = torch.empty(0, 300, device=cuda)
    got = helix_b200.rms_norm(x, torch.ones(300, device=cuda), x, out_dtype=F8)
    assert got.out.shape == (0, 300) and got.scale.shape == (0, 3) and got.sum.shape == (0, 300)
    q, sc = helix_b200.quantize8(x, blocks=True)
    assert q.shape == (0, 300) and sc.shape == (0, 3)
