"""GPU: the gated linear recurrence, its gradient and its single steps,
against the definition in 64 bits within running error bounds
(block_ref.gated: derived per step from the formula, fp32 arithmetic)."""
import ctypes as C

import pytest
import torch

import block_ref as ref
import helix_b200
from helix_b200 import abi

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _inputs(seed, S, T, Cn, t, mean=2.0, std=3.0):
    g = ref.generator(seed)
    v, gate, dy = ref.rand(g, S, T, Cn).to(t), ref.rand(g, S, T, Cn, mean=mean, std=std).to(t), ref.rand(g, S, T, Cn).to(t)
    return v, gate, dy, ref.rand(g, S, Cn).float(), ref.rand(g, S, Cn).float()


def _place(t, dev, form):
    """t on the GPU in one of the layouts a caller may have; NaN around it."""
    S, T, Cn = t.shape
    nan = float("nan")
    if form == "dense":
        return t.to(dev)
    if form == "slice":      # columns of a wider tensor, as a fused projection leaves them
        held = torch.full((S, T, 2 * Cn + 6), nan, dtype=t.dtype, device=dev)
        v = held[..., 4:4 + Cn]
    elif form == "odd":      # rows at odd addresses
        held = torch.full((S * T * (Cn + 3) + 1,), nan, dtype=t.dtype, device=dev)
        v = held[1:].view(S, T, Cn + 3)[..., :Cn]
    else:                    # "tok_first": tokens outermost
        held = torch.full((T, S, Cn + 2), nan, dtype=t.dtype, device=dev)
        v = held[..., :Cn].transpose(0, 1)
    v.copy_(t)
    return v


def _check(dev, S, T, Cn, t, form="dense", lengths=None, with_h0=True, seed=0, mean=2.0, std=3.0):
    v, g, dy, h0, dh1 = _inputs(seed + S + 7 * T + 13 * Cn, S, T, Cn, t, mean, std)
    h0_, dh1_ = (h0, dh1) if with_h0 else (None, None)
    dbl = lambda x: None if x is None else x.double()  # noqa: E731
    y, h1, hs, _, es, _, _ = ref.gated(v.double(), g.double(), dbl(h0_), lengths)
    vg, gg, dyg = (_place(x, dev, form) for x in (v, g, dy))
    if lengths is not None:
        for i, n in enumerate(lengths.tolist()):  # what lies past the end is never looked at
            for x in (vg, gg, dyg):
                x[i, max(n, 0):] = float("nan")
            vg[i, max(n, 0):] = float("inf")
    up = lambda x: None if x is None else x.to(dev)  # noqa: E731
    ln = up(lengths)
    gy, gh1, states = helix_b200.gated_scan(vg, gg, up(h0_), lengths=ln, keep_states=True)
    ref.within(gy, y, es[:, 1:] + y.abs() * ref.HALF[t] + 1e-37, "y")
    ref.within(gh1, h1, es[:, -1] + 1e-37, "h1")
    ref.within(states, hs[:, 0:T:128], es[:, 0:T:128] + 1e-37, "states")
    y2, h2 = helix_b200.gated_scan(vg, gg, up(h0_), lengths=ln)
    assert torch.equal(y2, gy) and torch.equal(h2, gh1)
    dv, dg, dh0, bv, bg, bh = ref.gated_grad(dy.double(), v.double(), g.double(), dbl(h0_), dbl(dh1_), lengths)
    gv, ggr, gh0 = helix_b200.gated_scan_grad(dyg, vg, gg, states, up(dh1_), lengths=ln)
    ref.within(gv, dv, bv + dv.abs() * ref.HALF[t] + 1e-37, "dv")
    ref.within(ggr, dg, bg + dg.abs() * ref.HALF[t] + 1e-37, "dg")
    ref.within(gh0, dh0, bh + 1e-37, "dh0")


SHAPES = [(1, 1, 1), (3, 1, 64), (64, 1, 300), (2, 2, 5), (1, 15, 64), (1, 16, 65), (2, 17, 130), (1, 127, 3),
          (3, 128, 64), (1, 129, 66), (2, 255, 33), (1, 300, 200), (2, 1000, 70), (1, 1025, 64), (1, 2100, 31)]


@pytest.mark.parametrize("S,T,Cn", SHAPES)
@pytest.mark.parametrize("t", [BF, F32])
def test_scan(cuda, S, T, Cn, t):
    _check(cuda, S, T, Cn, t)


@pytest.mark.parametrize("S,T,Cn", [(70, 300, 512), (5, 700, 4099), (300, 40, 130)])
@pytest.mark.parametrize("t", [BF, F32])
def test_scan_many_channels(cuda, S, T, Cn, t):
    """Enough channels that clusters are small, or single CTAs."""
    _check(cuda, S, T, Cn, t)


@pytest.mark.parametrize("form", ["slice", "odd", "tok_first"])
@pytest.mark.parametrize("Cn", [66, 129])
@pytest.mark.parametrize("t", [BF, F32])
def test_scan_layouts(cuda, form, Cn, t):
    _check(cuda, 3, 290, Cn, t, form)
    _check(cuda, 3, 1, Cn, t, form, with_h0=False)


@pytest.mark.parametrize("t", [BF, F32])
def test_scan_lengths(cuda, t):
    for T in (1, 130, 1100):
        n = torch.tensor([T, 0, 1, T // 2, T + 50, -3, max(T - 1, 0)], dtype=torch.int32)
        _check(cuda, 7, T, 67, t, lengths=n)


@pytest.mark.parametrize("form,Cn", [("dense", 64), ("odd", 67)])
def test_scan_ends_early(cuda, form, Cn):
    """Whole chunks, and whole turns of a cluster, past the ends."""
    n = torch.tensor([4000, 0, 130, 2049, 3999, 1024], dtype=torch.int32)
    _check(cuda, 6, 4000, Cn, BF, form, lengths=n)
    _check(cuda, 2, 4000, Cn, F32, form, lengths=torch.tensor([5, 0], dtype=torch.int32))


@pytest.mark.parametrize("mean,std", [(12.0, 1.0), (-12.0, 1.0), (0.0, 30.0), (60.0, 60.0)])
def test_scan_gates(cuda, mean, std):
    """Gates that keep for tens of thousands of tokens, that forget at once,
    and both beyond what exp can hold."""
    _check(cuda, 2, 1500, 40, F32, mean=mean, std=std)


def test_constant_gate_does_not_drift(cuda):
    """A gate of 1 - 2^-18 over 60000 tokens towards v = 1: 1 - (1 - z)^T.
    Rounding f itself would be off by 2^-25 / z in the exponent, 1e-2 here;
    the bound is the running one (4 roundings a step, doubled): 8 u T z-decayed,
    below 8 u / z (1 - e^-zT) = 2^-3 in the worst case but the folds of 128
    tokens leave 2 (T / 128 + 128) roundings of at most |h|: 1200 u."""
    T, z = 60000, 2.0 ** -18
    gate = torch.full((1, T, 64), float(torch.log(torch.tensor(1 / z - 1, dtype=torch.float64))))
    gg = gate.float().to(cuda)
    zz = 1.0 / (1.0 + torch.exp(gg[0, 0, 0].double().cpu()))
    y, h1 = helix_b200.gated_scan(torch.ones(1, T, 64, device=cuda), gg)
    want = -torch.expm1(T * torch.log1p(-zz))
    rel = (12 + 2 * 13 + 1200) * ref.U32
    assert (h1.double().cpu() - want).abs().max() <= rel * want


def test_grad_against_differences(cuda):
    """Along random directions, against central differences of the definition
    in 64 bits, L = <y, dy> + <h1, dh1>: truncation and rounding of the step
    1e-5 leave 1e-8, the kernel's fp32 1e-6 of the norms' product."""
    S, T, Cn = 2, 200, 11
    v, g, dy, h0, dh1 = _inputs(31, S, T, Cn, F32, mean=1.0, std=1.5)
    n = torch.tensor([200, 77], dtype=torch.int32)
    up = lambda x: x.to(cuda)  # noqa: E731
    _, _, states = helix_b200.gated_scan(up(v), up(g), up(h0), lengths=up(n), keep_states=True)
    got = helix_b200.gated_scan_grad(up(dy), up(v), up(g), states, up(dh1), lengths=up(n))

    def loss(v_, g_, h_):
        y, h1 = ref.gated(v_, g_, h_, n)[:2]
        return (y * dy.double()).sum() + (h1 * dh1.double()).sum()

    gen = ref.generator(5)
    for _ in range(4):
        p = [ref.rand(gen, *x.shape) for x in (v, g, h0)]
        at = [x.double() for x in (v, g, h0)]
        h = 1e-5
        want = (loss(*[a + h * b for a, b in zip(at, p)]) - loss(*[a - h * b for a, b in zip(at, p)])) / (2 * h)
        have = sum((x.double().cpu() * b).sum() for x, b in zip(got, p))
        scale = sum(x.double().cpu().norm() * b.norm() for x, b in zip(got, p))
        assert abs(have - want) <= 1e-6 * scale


def test_steps_continue_a_prefill(cuda):
    """A prefill and then single tokens in place give what one call gives."""
    S, T, Cn = 3, 140, 96
    v, g, _, h0, _ = _inputs(8, S, T, Cn, BF)
    vg, gg, state = v.to(cuda), g.to(cuda), h0.to(cuda)
    y, h1, hs, _, es, _, _ = ref.gated(v.double(), g.double(), h0.double(), None)
    y0, state = helix_b200.gated_scan(vg[:, :130], gg[:, :130], state)
    for t in range(130, T):
        yt, same = helix_b200.gated_scan(vg[:, t:t + 1], gg[:, t:t + 1], state, h1=state)
        assert same is state
        ref.within(yt, y[:, t:t + 1], 2 * es[:, t + 1:t + 2] + y[:, t:t + 1].abs() * ref.U16, "step")
    ref.within(state, h1, 2 * es[:, -1], "h1")


def test_in_place_long(cuda):
    """h1 in place of h0, dv of dy and dh0 of dh1 where many CTAs share a sequence."""
    S, T, Cn = 1, 3000, 64
    v, g, dy, h0, dh1 = _inputs(9, S, T, Cn, F32)
    vg, gg = v.to(cuda), g.to(cuda)
    a = helix_b200.gated_scan(vg, gg, h0.to(cuda), keep_states=True)
    state = h0.to(cuda)
    b = helix_b200.gated_scan(vg, gg, state, h1=state)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    want = helix_b200.gated_scan_grad(dy.to(cuda), vg, gg, a[2], dh1.to(cuda))
    dyg = dy.to(cuda)
    got = helix_b200.gated_scan_grad(dyg, vg, gg, a[2], dh1.to(cuda), dv=dyg)
    assert all(torch.equal(x, z) for x, z in zip(want, got))


def test_gradients_into_one_tensor(cuda):
    S, T, Cn = 2, 300, 64
    v, g, dy, h0, dh1 = _inputs(10, S, T, Cn, BF)
    vg, gg, dyg = v.to(cuda), g.to(cuda), dy.to(cuda)
    states = helix_b200.gated_scan(vg, gg, h0.to(cuda), keep_states=True)[2]
    want = helix_b200.gated_scan_grad(dyg, vg, gg, states, dh1.to(cuda))
    both = torch.full((S, T, 2 * Cn), float("nan"), dtype=BF, device=cuda)
    helix_b200.gated_scan_grad(dyg, vg, gg, states, dh1.to(cuda), dv=both[..., :Cn], dg=both[..., Cn:])
    assert torch.equal(both[..., :Cn], want[0]) and torch.equal(both[..., Cn:], want[1])


def test_offsets_past_32_bits(cuda):
    """Token strides that put the last tokens beyond 2^32 bytes and 2^31 elements."""
    T, Cn, stride = 40, 64, 1 << 26
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 20 GB of device memory")
    v, g, dy, h0, dh1 = _inputs(11, 1, T, Cn, BF)
    held = torch.empty(T * stride + 4 * Cn, dtype=BF, device=cuda)
    view = lambda k: torch.as_strided(held, (1, T, Cn), (T * stride, stride, 1), k * Cn)  # noqa: E731
    vv, gv = view(0), view(1)
    vv.copy_(v), gv.copy_(g)
    y, h1, _, _, es, _, _ = ref.gated(v.double(), g.double(), h0.double(), None)
    got, last, states = helix_b200.gated_scan(vv, gv, h0.to(cuda), keep_states=True)
    ref.within(got, y, es[:, 1:] + y.abs() * ref.U16, "y")
    ref.within(last, h1, es[:, -1], "h1")
    dv, dg, dh0, bv, bg, bh = ref.gated_grad(dy.double(), v.double(), g.double(), h0.double(), dh1.double(), None)
    out = helix_b200.gated_scan_grad(dy.to(cuda), vv, gv, states, dh1.to(cuda), dv=view(2), dg=view(3))
    ref.within(out[0], dv, bv + dv.abs() * ref.U16, "dv")
    ref.within(out[1], dg, bg + dg.abs() * ref.U16, "dg")
    ref.within(out[2], dh0, bh, "dh0")


def test_empty(cuda):
    h0 = torch.randn(3, 8, device=cuda)
    y, h1, states = helix_b200.gated_scan(torch.empty(3, 0, 8, device=cuda), torch.empty(3, 0, 8, device=cuda), h0,
                                          keep_states=True)
    assert y.shape == (3, 0, 8) and torch.equal(h1, h0) and states.shape == (3, 0, 8)
    e = torch.empty(3, 0, 8, device=cuda)
    dv, dg, dh0 = helix_b200.gated_scan_grad(e, e, e, states, h0)
    assert torch.equal(dh0, h0)
    e = torch.empty(0, 5, 8, device=cuda)
    y, h1 = helix_b200.gated_scan(e, e)
    assert y.shape == (0, 5, 8) and h1.shape == (0, 8)


def test_captured_and_on_another_stream(cuda):
    S, T, Cn = 2, 600, 64
    v, g, dy, h0, dh1 = _inputs(12, S, T, Cn, BF)
    vg, gg, dyg, hg = (x.to(cuda) for x in (v, g, dy, h0))
    want = helix_b200.gated_scan(vg, gg, hg, keep_states=True)
    wantg = helix_b200.gated_scan_grad(dyg, vg, gg, want[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = helix_b200.gated_scan(vg, gg, hg, keep_states=True, stream=side)
    b = helix_b200.gated_scan_grad(dyg, vg, gg, a[2], stream=side)
    side.synchronize()
    assert all(torch.equal(x, z) for x, z in zip(want, a)) and all(torch.equal(x, z) for x, z in zip(wantg, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = helix_b200.gated_scan(vg, gg, hg, keep_states=True)
        b = helix_b200.gated_scan_grad(dyg, vg, gg, a[2])
    hg.copy_(-h0)
    graph.replay()
    torch.cuda.synchronize()
    want = helix_b200.gated_scan(vg, gg, hg, keep_states=True)
    wantg = helix_b200.gated_scan_grad(dyg, vg, gg, want[2])
    assert all(torch.equal(x, z) for x, z in zip(want, a)) and all(torch.equal(x, z) for x, z in zip(wantg, b))
    del graph


def test_refusals(cuda, ctx):
    v = torch.randn(2, 4, 8, device=cuda)
    h = torch.zeros(2, 8, device=cuda)
    with pytest.raises(ValueError):
        helix_b200.gated_scan(v[0], v[0])
    with pytest.raises(ValueError):
        helix_b200.gated_scan(v, v[:, :3])
    with pytest.raises(TypeError):
        helix_b200.gated_scan(v, v.bfloat16())
    with pytest.raises(TypeError):
        helix_b200.gated_scan(v.half(), v.half())
    with pytest.raises(TypeError):
        helix_b200.gated_scan(v, v, h.bfloat16())
    with pytest.raises(ValueError):
        helix_b200.gated_scan(v, v, h[:1])
    with pytest.raises(ValueError):
        helix_b200.gated_scan(v.transpose(1, 2), v.transpose(1, 2))
    with pytest.raises(TypeError):
        helix_b200.gated_scan(v, v, lengths=torch.tensor([1, 2], device=cuda))
    with pytest.raises(ValueError):
        helix_b200.gated_scan(v, v, h.cpu())
    with pytest.raises(ValueError):
        helix_b200.gated_scan_grad(v, v, v, h)
    T, st = helix_b200._t, torch.cuda.current_stream().cuda_stream
    y, h1 = torch.empty_like(v), torch.empty_like(h)

    def call(edit=None, **kw):
        d = abi.GatedScanDesc()
        ctx.lib.helix_gated_scan_desc_init(C.byref(d), 4, 2, 8)
        for k, x in (edit or {}).items():
            setattr(d, k, x)
        a = dict(v=T(v), g=T(v), h0=T(h), lengths=T(None), y=T(y), h1=T(h1), states=T(None))
        a.update(kw)
        return ctx.lib.helix_gated_scan_encode(ctx.handle, st, C.byref(d), *a.values())

    assert call() == abi.HELIX_OK
    for edit, status in (({"n_tok": -1}, 1), ({"n_chan": -5}, 1), ({"io_dtype": 1}, 1), ({"io_dtype": 3}, 1),
                         ({"s_y": 7}, 4), ({"seq_y": 31}, 4), ({"s_v": -8}, 4), ({"seq_h1": 7}, 4),
                         ({"n_tok": 2 ** 31 - 1}, 1)):
        assert call(edit) == status, edit
    for kw in (dict(v=T(None)), dict(g=T(None)), dict(y=T(None)), dict(h1=T(None)), dict(y=T(v)),
               dict(h1=abi.Tensor(h.data_ptr(), 4)), dict(v=abi.Tensor(v.data_ptr(), 1)), dict(h1=T(v)),
               dict(states=T(y))):
        assert call(**kw) == abi.HELIX_ERR_INVALID_ARG, kw
    assert call({"n_tok": 0}) == abi.HELIX_OK and call({"n_seq": 0}) == abi.HELIX_OK
    assert ctx.lib.helix_gated_scan_states_size(None) == 0
    torch.cuda.synchronize()
