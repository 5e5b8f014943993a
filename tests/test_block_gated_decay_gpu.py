"""GPU: the gated recurrence where states and gradients decay by many orders
of magnitude, against the definition in 64 bits within bounds that are relative
to what is left (gated_ref)."""
import pytest
import torch

import block_ref as ref
import gated_ref
import helix_b200

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _inputs(kind, seed, S, T, Cn, t):
    """v, g, dy, h0, dh1 of a case where old values have to vanish."""
    gen = ref.generator(seed)
    r = lambda *shape, **kw: ref.rand(gen, *shape, **kw)  # noqa: E731
    v, g, dy = r(S, T, Cn), r(S, T, Cn), r(S, T, Cn)
    h0, dh1 = r(S, Cn), r(S, Cn)
    if kind.startswith("closed"):      # gates that keep next to nothing
        g += -float(kind[6:])
    elif kind == "large_start":        # a large first state and last gradient, then small values
        g = 0.5 * g - 0.7
        v, dy = v * 1e-3, dy * 1e-3
        h0, dh1 = h0 * 1e4, dh1 * 1e4
    elif kind == "ends_alone":         # nothing but the first state, and the last gradient
        g -= 2.0
        v, dy = torch.zeros_like(v), torch.zeros_like(dy)
    elif kind == "spikes":             # one value in 40 a million times the others
        g = 1.5 * g
        big = torch.rand(v.shape, generator=gen) < 1 / 40
        v, dy = torch.where(big, v * 1e3, v * 1e-3), torch.where(big.flip(1), dy * 1e3, dy * 1e-3)
    else:                              # "mixed": channels that keep for long beside those that forget at once
        assert kind == "mixed"
        g += torch.linspace(-12.0, 12.0, Cn, dtype=torch.float64)
    return v.to(t), g.to(t), dy.to(t), h0.float(), dh1.float()


def _odd(t):
    """A copy whose rows start at odd addresses, NaN around them."""
    S, T, Cn = t.shape
    held = torch.full((S * T * (Cn + 3) + 1,), float("nan"), dtype=t.dtype, device=t.device)
    rows = held[1:].view(S, T, Cn + 3)[..., :Cn]
    rows.copy_(t)
    return rows


def _check(dev, kind, S, T, Cn, t, odd=False, lengths=None):
    v, g, dy, h0, dh1 = _inputs(kind, S + 3 * T + 5 * Cn, S, T, Cn, t)
    dbl = [x.double() for x in (v, g, dy, h0, dh1)]
    hs, _, es = gated_ref.forward(dbl[0], dbl[1], dbl[3], lengths)
    live = gated_ref._live(v, lengths)
    place = _odd if odd else (lambda x: x)
    vg, gg, dyg = (place(x.to(dev)) for x in (v, g, dy))
    ln = None if lengths is None else lengths.to(dev)
    half, tiny = ref.HALF[t], gated_ref.TINY
    y, h1, states = helix_b200.gated_scan(vg, gg, h0.to(dev), lengths=ln, keep_states=True)
    want = hs[:, 1:] * live
    big = 1.0 + max(x.abs().max().item() for x in dbl if x is not dbl[1]) ** 2
    ref.within(y, want, es[:, 1:] + want.abs() * half + big * tiny, "y")
    ref.within(h1, hs[:, -1], es[:, -1] + big * tiny, "h1")
    ref.within(states, hs[:, 0:T:128], es[:, 0:T:128] + big * tiny, "states")
    dv, dg, dh0, bv, bg, bh = gated_ref.backward(dbl[2], dbl[0], dbl[1], dbl[3], dbl[4], lengths)
    gv, gr, gh = helix_b200.gated_scan_grad(dyg, vg, gg, states, dh1.to(dev), lengths=ln)
    ref.within(gv, dv * live, bv + dv.abs() * half + big * tiny, "dv")
    ref.within(gr, dg * live, bg + dg.abs() * half + big * tiny, "dg")
    ref.within(gh, dh0, bh + big * tiny, "dh0")


KINDS = ["closed8", "closed12", "closed18", "closed40", "closed75", "large_start", "ends_alone", "spikes", "mixed"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 3, 16])
@pytest.mark.parametrize("t", [BF, F32])
def test_few_tokens(cuda, kind, T, t):
    _check(cuda, kind, 3, T, 70, t)
    _check(cuda, kind, 2, T, 33, t, odd=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [17, 130, 1500])
@pytest.mark.parametrize("t", [BF, F32])
def test_long(cuda, kind, T, t):
    """Folds of runs, of a CTA's warps and of a cluster's CTAs."""
    _check(cuda, kind, 2, T, 70, t)
    _check(cuda, kind, 1, T, 33, t, odd=True)


@pytest.mark.parametrize("kind", ["closed8", "large_start", "ends_alone", "mixed"])
@pytest.mark.parametrize("S,T,Cn", [(70, 300, 512), (2, 700, 3001), (1, 1000, 2048), (1, 2500, 700)])
@pytest.mark.parametrize("t", [BF, F32])
def test_cuts(cuda, kind, S, T, Cn, t):
    """Wide and narrow rows, single CTAs and clusters of two to eight."""
    _check(cuda, kind, S, T, Cn, t)


@pytest.mark.parametrize("t", [BF, F32])
def test_long_with_lengths(cuda, t):
    n = torch.tensor([1100, 0, 1, 550, 130, 1099], dtype=torch.int32)
    for kind in ("large_start", "closed12"):
        _check(cuda, kind, 6, 1100, 67, t, lengths=n)
        _check(cuda, kind, 6, 1100, 67, t, odd=True, lengths=n)
