"""GPU: infinities and NaN among the tokens that count, in the states and in
the gradients: what 64-bit arithmetic makes of f h + (1 - f) v, with f and 1 - f
above zero.  A channel without them is not touched, bit for bit, and neither are
tokens that come before."""
import pytest
import torch

import block_ref as ref
import gated_ref
import helix_b200

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _run(dev, v, g, dy, h0, dh1, lengths, odd):
    def place(x):
        x = x.to(dev)
        if not odd:
            return x
        S, T, Cn = x.shape
        held = torch.zeros(S * T * (Cn + 3) + 1, dtype=x.dtype, device=dev)
        rows = held[1:].view(S, T, Cn + 3)[..., :Cn]
        rows.copy_(x)
        return rows
    vg, gg, dyg = place(v), place(g), place(dy)
    ln = None if lengths is None else lengths.to(dev)
    y, h1, st = helix_b200.gated_scan(vg, gg, h0.to(dev), lengths=ln, keep_states=True)
    dv, dg, dh0 = helix_b200.gated_scan_grad(dyg, vg, gg, st, dh1.to(dev), lengths=ln)
    return [x.cpu() for x in (y, h1, st, dv, dg, dh0)]


def _want(v, g, dy, h0, dh1, lengths):
    """The same six in 64 bits."""
    v, g, dy, h, c = (x.double() for x in (v, g, dy, h0, dh1))
    live = gated_ref._live(v, lengths)
    f, z = torch.sigmoid(g), torch.sigmoid(-g)
    T = v.shape[1]
    hs = [h]
    for t in range(T):
        h = torch.where(live[:, t], f[:, t] * h + z[:, t] * v[:, t], h)
        hs.append(h)
    hs = torch.stack(hs, 1)
    zero = torch.zeros(()).double()
    dv, dg = torch.zeros_like(v), torch.zeros_like(v)
    for t in range(T - 1, -1, -1):
        lam = c + dy[:, t]
        dv[:, t], dg[:, t] = z[:, t] * lam, lam * (hs[:, t] - v[:, t]) * (z[:, t] * f[:, t])
        c = torch.where(live[:, t], f[:, t] * lam, c)
    y, dv, dg = (torch.where(live, x, zero) for x in (hs[:, 1:], dv, dg))
    return [y, h, hs[:, 0:T:128], dv, dg, c]


def _kind(x):
    """0 finite, 1 and -1 the infinities, 2 NaN."""
    x = x.double()
    k = torch.where(x == INF, 1, torch.where(x == -INF, -1, 0))
    return torch.where(x.isnan(), 2, k)


@pytest.mark.parametrize("where", ["v", "v_both", "v_nan", "h0", "h0_v", "dy", "dy_both", "dh1"])
@pytest.mark.parametrize("S,T,Cn,odd", [(2, 1, 6, False), (2, 9, 6, False), (2, 16, 7, True), (2, 40, 66, False),
                                        (2, 300, 70, False), (2, 1500, 70, False), (2, 300, 67, True),
                                        (1, 2500, 700, False), (70, 300, 512, False)])
@pytest.mark.parametrize("t", [BF, F32])
def test_infinities(cuda, where, S, T, Cn, odd, t):
    gen = ref.generator(S + T + Cn)
    v, dy = ref.rand(gen, S, T, Cn).to(t), ref.rand(gen, S, T, Cn).to(t)
    g = ref.rand(gen, S, T, Cn, mean=1.0, std=2.0)
    g[..., 1] -= 20.0                       # in 16 tokens of these nothing is left
    g[..., 4] += 14.0
    g = g.to(t)
    h0, dh1 = ref.rand(gen, S, Cn).float(), ref.rand(gen, S, Cn).float()
    lengths = None
    if S == 2 and T > 1:
        lengths = torch.tensor([T, max(1, T - 5)], dtype=torch.int32)
    clean = _run(cuda, v, g, dy, h0, dh1, lengths, odd)
    at = [min(T - 1, T // 2 + k) for k in (0, 1)]
    hit = [1, 2, 4, Cn - 1]                 # channels; 3 is the neighbour of 2
    if where.startswith("v") or where == "h0_v":
        for c in hit:
            v[:, at[0], c] = {"v_nan": NAN}.get(where, INF if c != 2 else -INF)
        if where == "v_both" and T > 1:
            v[:, at[1], 2] = INF            # after -inf: NaN
    if where.startswith("h0"):
        for c in hit:
            h0[:, c] = -INF if c == 4 else INF
    if where.startswith("dy"):
        for c in hit:
            dy[:, at[1], c] = INF if c != 2 else -INF
        if where == "dy_both" and T > 1:
            dy[:, at[0], 2] = INF
    if where == "dh1":
        for c in hit:
            dh1[:, c] = -INF if c == 4 else INF
    got = _run(cuda, v, g, dy, h0, dh1, lengths, odd)
    want = _want(v, g, dy, h0, dh1, lengths)
    hs, ms, es = gated_ref.forward(v.double(), g.double(), h0.double(), lengths)
    same = (hs[:, :-1] - v.double()).abs() <= es[:, :-1] + ref.U32 * (ms[:, :-1] + v.double().abs())
    for name, a, b, w in zip(("y", "h1", "states", "dv", "dg", "dh0"), got, clean, want):
        bad = _kind(a) != _kind(w)
        if name == "dg":   # infinity times h - v, where fp32 cannot tell h from v
            bad &= ~(same & a.isnan())
        assert not bad.any(), (name, int(bad.sum()), bad.nonzero()[0].tolist(), a[bad][0].item(), w[bad][0].item())
        others = [c for c in range(Cn) if c not in hit]
        assert torch.equal(a[..., others], b[..., others]), f"{name}: other channels"
        untouched = {"y": where[0] == "d", "h1": where[0] == "d", "states": where[0] == "d",
                     "dv": where[0] != "d", "dg": False, "dh0": where[0] != "d"}[name]
        if untouched:
            assert torch.equal(a, b), f"{name}: it does not depend on what was changed"
    if where.startswith("v"):
        assert torch.equal(got[0][:, :at[0]], clean[0][:, :at[0]]), "y: earlier tokens"
    if where.startswith("dy"):
        assert torch.equal(got[3][:, at[1] + 1:], clean[3][:, at[1] + 1:]), "dv: later tokens"


@pytest.mark.parametrize("T", [1, 16, 300, 1500])
def test_magnitudes_at_the_end_of_the_range(cuda, T):
    """Values whose differences fp32 cannot hold."""
    gen = ref.generator(T)
    S, Cn = 2, 70
    v = torch.where(torch.rand(S, T, Cn, generator=gen) < 0.5, -3.3e38, 3.3e38).float()
    g, h0 = ref.rand(gen, S, T, Cn, std=3.0).float(), torch.full((S, Cn), -3.3e38)
    hs, _, es = gated_ref.forward(v.double(), g.double(), h0.double())
    y, h1 = helix_b200.gated_scan(v.to(cuda), g.to(cuda), h0.to(cuda))
    ref.within(y, hs[:, 1:], es[:, 1:] + hs[:, 1:].abs() * ref.U32, "y")
    ref.within(h1, hs[:, -1], es[:, -1], "h1")
