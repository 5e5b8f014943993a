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
