"""The block operators' definitions (include/helix/helix_block.h) in 64 bits,
and the error bounds their kernels are held to."""
from __future__ import annotations

import torch

GROUP, E4M3_MAX, AMAX_FLOOR = 128, 448.0, 2.0 ** -100
U32 = 2.0 ** -24      # half a unit in the last place of fp32, relative
U16 = 2.0 ** -8       # of bf16 (8 significant bits)
HALF = {torch.float32: U32, torch.bfloat16: U16}


def rand(gen, *shape, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=gen, dtype=torch.float64) * std + mean


def generator(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, bound, what):
    """|got - want| <= bound everywhere; NaN exactly where want has NaN."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN elsewhere"
    err = (got - want).abs()
    err[want.isnan()] = 0.0
    same = got == want                       # infinities
    bad = ~(err <= bound) & ~same & ~want.isnan()
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst "
                           f"{(err / bound)[bad].max().item():.3g} of the bound at {bad.nonzero()[0].tolist()}")


def group_amax(x, blocks):
    """Largest magnitude per (row, 128 columns), or per 128 x 128 block."""
    def along(t, dim):
        return torch.stack([c.abs().amax(dim) for c in t.split(GROUP, dim)], dim)
    a = along(x, 1)
    return along(a, 0) if blocks else a


def spread(scale, rows, cols, blocks):
    scale = scale.repeat_interleave(GROUP, 1)[:, :cols]
    return scale.repeat_interleave(GROUP, 0)[:rows] if blocks else scale


def check_8bit(q, scale, value, rel, blocks, what):
    """q and scale against the fp64 value, itself known to the kernel with a
    relative error `rel`.  The scale is one fp32 division off; q is value /
    scale times (1 + rel + 2^-22) rounded to 4 significant bits (2^-4 relative)
    or to the subnormal spacing 2^-9 (2^-10 absolute)."""
    rows, cols = value.shape
    want = group_amax(value, blocks).clamp_min(AMAX_FLOOR) / E4M3_MAX
    within(scale, want, want * (rel + 4 * U32), f"{what} scale")
    s = spread(scale.double().cpu(), rows, cols, blocks)
    unit = value / s
    bound = torch.maximum(unit.abs() * 2.0 ** -4, torch.full_like(unit, 2.0 ** -10)) + unit.abs() * (rel + 2.0 ** -22)
    within(q.double(), unit, bound, f"{what} q")


def norm(x, res, w, eps):
    """(sum, rstd, n) in fp64."""
    s = x if res is None else x + res
    rstd = 1.0 / torch.sqrt((s * s).mean(1) + eps)
    return s, rstd, s * rstd[:, None] * w


def norm_grad(dout, s, rstd, w, dsum):
    """(ds, dweight), and the magnitudes their errors scale with."""
    u = s * rstd[:, None]
    dw_ = dout * w
    along = (dw_ * u).mean(1, keepdim=True)
    ds = rstd[:, None] * (dw_ - u * along)
    mag = rstd[:, None] * (dw_.abs() + u.abs() * (dw_ * u).abs().mean(1, keepdim=True))
    if dsum is not None:
        ds, mag = ds + dsum, mag + dsum.abs()
    return ds, (dout * u).sum(0), mag, (dout * u).abs().sum(0)


def gated(v, g, h0, lengths):
    """The recurrence in fp64: (y, h1, hs with h_{-1} first, z, live, err).

    err bounds what fp32 makes of h.  1 - f is off by 12 u (exponential 4,
    sum, quotient 4, product, with slack) and 2 u |g| (the exponent's
    rounding); a step adds that times z |v - h| and 4 roundings of magnitudes
    up to M, M_t = f M_{t-1} + z |v| being the recurrence of the magnitudes;
    twice, because a run's fold rounds as a step does."""
    S, T, C = v.shape
    live = torch.ones(S, T, 1, dtype=torch.bool)
    if lengths is not None:
        live = (torch.arange(T)[None] < lengths[:, None].clamp(0, T))[:, :, None]
    z = torch.where(live, 1.0 / (1.0 + torch.exp(g)), torch.zeros(()).double())
    v = torch.where(live, v, torch.zeros(()).double())
    eg = torch.where(live, 12 + 2 * g.abs(), torch.zeros(()).double())
    h = h0 if h0 is not None else torch.zeros(S, C).double()
    m, e = h.abs(), torch.zeros(S, C).double()
    hs, ms, es = [h], [m], [e]
    for t in range(T):
        e = (1 - z[:, t]) * e + 2 * U32 * (4 * m + eg[:, t] * z[:, t] * (v[:, t].abs() + m))
        h = h + z[:, t] * (v[:, t] - h)
        m = (1 - z[:, t]) * m + z[:, t] * v[:, t].abs()
        hs.append(h), ms.append(m), es.append(e)
    hs, ms, es = (torch.stack(x, 1) for x in (hs, ms, es))
    return hs[:, 1:] * live, hs[:, -1], hs, ms, es, z, live


def gated_grad(dy, v, g, h0, dh1, lengths):
    """(dv, dg, dh0) in fp64 and bounds of their fp32 errors, as above."""
    S, T, C = v.shape
    _, _, hs, ms, es, z, live = gated(v, g, h0, lengths)
    zero = torch.zeros(()).double()
    dy, v = torch.where(live, dy, zero), torch.where(live, v, zero)
    f = torch.where(live, 1.0 / (1.0 + torch.exp(-g)), torch.ones(()).double())
    ga = torch.where(live, g.abs(), zero)
    c = dh1 if dh1 is not None else torch.zeros(S, C).double()
    mc, ec = c.abs(), torch.zeros(S, C).double()
    dv, dg, bv, bg = (torch.zeros(S, T, C).double() for _ in range(4))
    for t in range(T - 1, -1, -1):
        lam, ml = dy[:, t] + c, dy[:, t].abs() + mc
        el = ec + 2 * U32 * ml
        zt, s = z[:, t], z[:, t] * f[:, t]
        off, moff = hs[:, t] - v[:, t], ms[:, t] + v[:, t].abs()
        dv[:, t] = zt * lam
        bv[:, t] = zt * (el + ml * (14 + 2 * ga[:, t]) * U32)
        dg[:, t] = lam * off * s
        bg[:, t] = s * (el * moff + ml * es[:, t] + ml * moff * (24 + 2 * ga[:, t]) * U32)
        c = lam * (1 - zt)
        mc = ml * (1 - zt)
        ec = (1 - zt) * el + 2 * U32 * ml * (2 + (12 + 2 * ga[:, t]) * zt)
    return dv * live, dg * live, c, bv, bg, ec
