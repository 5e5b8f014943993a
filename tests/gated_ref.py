"""The gated recurrence and its gradient in 64 bits, and what fp32 may be off
by where a state or a gradient has to decay: the bounds here are relative to
what is left of it, not to what it was.

With u = 2^-24: the gate's smaller side, min(f, 1 - f) = t / (1 + t) with
t = e^-|g|, is off by (2 |g| + 14) u of itself (the exponent's rounding and its
constant's 2 |g| + 6, exponential 4, sum 1, reciprocal 2, product 1).  The
other is 1 minus it, or formed by a sum, a reciprocal and a product as well:
4 u of itself, and the smaller side's error.  A step h' = f h + z v, z = 1 - f,
adds two roundings of m' = f m + z |v|, the recurrence of the magnitudes, and so
does the gradient's.  Twice, because a run of tokens that is folded onto a
state rounds as its steps do."""
from __future__ import annotations

import torch

from block_ref import U32

TINY = 1e-35  # f or z below 2^-118 may count as 0 or as that; times magnitudes of order 1


def _gates(g, live):
    one, zero = torch.ones(()).double(), torch.zeros(()).double()
    f = torch.where(live, torch.sigmoid(g), one)
    z = torch.where(live, torch.sigmoid(-g), zero)
    a = torch.where(live, 2 * g.abs() + 14, zero)
    slack = torch.where(live, torch.full_like(g, 4.0), zero)
    return f, z, f * (z * a + slack) * U32, z * (f * a + slack) * U32


def _live(v, lengths):
    S, T, _ = v.shape
    if lengths is None:
        return torch.ones(S, T, 1, dtype=torch.bool)
    return (torch.arange(T)[None] < lengths[:, None].clamp(0, T))[:, :, None]


def forward(v, g, h0, lengths=None):
    """(states, h_{-1} first; their magnitudes; the bounds of their errors)."""
    live = _live(v, lengths)
    f, z, ef, ez = _gates(g, live)
    v = torch.where(live, v, torch.zeros(()).double())
    h, m, e = h0, h0.abs(), torch.zeros_like(h0)
    hs, ms, es = [h], [m], [e]
    for t in range(v.shape[1]):
        a = v[:, t].abs()
        after = f[:, t] * m + z[:, t] * a
        e = f[:, t] * e + 2 * (ef[:, t] * m + ez[:, t] * a + 2 * U32 * after * live[:, t])
        h, m = f[:, t] * h + z[:, t] * v[:, t], after
        hs.append(h), ms.append(m), es.append(e)
    return tuple(torch.stack(x, 1) for x in (hs, ms, es))


def backward(dy, v, g, h0, dh1, lengths=None):
    """(dv, dg, dh0) and the bounds of their errors."""
    hs, ms, es = forward(v, g, h0, lengths)
    live = _live(v, lengths)
    f, z, ef, ez = _gates(g, live)
    zero = torch.zeros(()).double()
    dy, v = torch.where(live, dy, zero), torch.where(live, v, zero)
    c, mc, ec = dh1, dh1.abs(), torch.zeros_like(dh1)
    dv, dg, bv, bg = (torch.zeros_like(v) for _ in range(4))
    for t in range(v.shape[1] - 1, -1, -1):
        ft, zt, eft, ezt = f[:, t], z[:, t], ef[:, t], ez[:, t]
        lam, ml = dy[:, t] + c, dy[:, t].abs() + mc
        el = ec + 2 * U32 * ml * live[:, t]
        off, moff = hs[:, t] - v[:, t], ms[:, t] + v[:, t].abs()
        eoff = es[:, t] + U32 * moff
        dv[:, t], dg[:, t] = zt * lam, lam * off * zt * ft
        bv[:, t] = zt * el + 2 * ml * (ezt + U32 * zt)
        bg[:, t] = zt * ft * (el * moff + ml * eoff) + 2 * ml * moff * (ezt * ft + zt * eft + 4 * U32 * zt * ft)
        c, mc = ft * lam, ft * ml
        ec = ft * el + 2 * (eft * ml + U32 * mc * live[:, t])
    return dv, dg, c, bv, bg, ec
