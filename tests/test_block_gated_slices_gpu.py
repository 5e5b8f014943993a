"""GPU: gradients written into slices of one wider tensor, whatever its layout:
padded sequences, tokens outermost.  Slices that do share elements are refused."""
import ctypes as C

import pytest
import torch

import block_ref as ref
import helix_b200
from helix_b200 import abi

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _case(dev, S, T, Cn, t):
    gen = ref.generator(S + T + Cn)
    v, g, dy = (ref.rand(gen, S, T, Cn, mean=m).to(t).to(dev) for m in (0.0, 2.0, 0.0))
    h0, dh1 = ref.rand(gen, S, Cn).float().to(dev), ref.rand(gen, S, Cn).float().to(dev)
    states = helix_b200.gated_scan(v, g, h0, keep_states=True)[2]
    return v, g, dy, dh1, states


def _wide(dev, S, T, Cn, t, form):
    """A tensor that holds two (S, T, Cn) side by side, seen as (S, T, 2 Cn)."""
    if form == "padded":               # sequences with room for more tokens
        return torch.full((S, T + 5, 2 * Cn), 7.0, dtype=t, device=dev)[:, :T]
    if form == "padded_odd":           # and a pitch between sequences that is no multiple of a token's
        held = torch.full((S * ((T + 1) * 2 * Cn + 3),), 7.0, dtype=t, device=dev)
        return torch.as_strided(held, (S, T, 2 * Cn), ((T + 1) * 2 * Cn + 3, 2 * Cn, 1))
    return torch.full((T, S, 2 * Cn), 7.0, dtype=t, device=dev).transpose(0, 1)


@pytest.mark.parametrize("form", ["padded", "padded_odd", "tok_first"])
@pytest.mark.parametrize("S,T,Cn", [(3, 9, 40), (3, 300, 64), (2, 300, 33)])
@pytest.mark.parametrize("t", [BF, F32])
def test_gradients_side_by_side(cuda, form, S, T, Cn, t):
    v, g, dy, dh1, states = _case(cuda, S, T, Cn, t)
    want = helix_b200.gated_scan_grad(dy, v, g, states, dh1)
    both = _wide(cuda, S, T, Cn, t, form)
    helix_b200.gated_scan_grad(dy, v, g, states, dh1, dv=both[..., :Cn], dg=both[..., Cn:])
    assert torch.equal(both[..., :Cn], want[0]) and torch.equal(both[..., Cn:], want[1])
    both.fill_(7.0)
    assert (both._base == 7.0).all()
    # dv in place of dy there
    both[..., :Cn] = dy
    helix_b200.gated_scan_grad(both[..., :Cn], v, g, states, dh1, dv=both[..., :Cn], dg=both[..., Cn:])
    assert torch.equal(both[..., :Cn], want[0]) and torch.equal(both[..., Cn:], want[1])


@pytest.mark.parametrize("form", ["padded", "padded_odd", "tok_first"])
def test_shared_elements_are_refused(cuda, form):
    S, T, Cn, t = 3, 20, 40, F32
    v, g, dy, dh1, states = _case(cuda, S, T, Cn, t)
    both = _wide(cuda, S, T, Cn, t, form)
    for dv, dg in ((both[..., :Cn], both[..., Cn - 1:-1]), (both[..., 1:Cn + 1], both[..., :Cn]),
                   (both[..., :Cn], both[..., :Cn]), (both[..., Cn:], both[..., Cn - 8:2 * Cn - 8])):
        with pytest.raises(helix_b200.HelixError, match="overlaps"):
            helix_b200.gated_scan_grad(dy, v, g, states, dh1, dv=dv, dg=dg)
    # one token, or one sequence, on: other rows of the same columns
    two = torch.zeros(S + 1, T + 1, 2 * Cn, device=cuda)
    for a, b in ((two[:S, :T], two[:S, 1:]), (two[:S, :T], two[1:, :T]), (two[:S, 1:], two[1:, :T])):
        with pytest.raises(helix_b200.HelixError, match="overlaps"):
            helix_b200.gated_scan_grad(dy, v, g, states, dh1, dv=a[..., :Cn], dg=b[..., :Cn])
        helix_b200.gated_scan_grad(dy, v, g, states, dh1, dv=a[..., :Cn], dg=b[..., Cn:])
    torch.cuda.synchronize()


def test_outputs_beside_inputs(cuda, ctx):
    """y between v and g, in sequences with room for more tokens (C ABI)."""
    S, T, Cn = 2, 50, 24
    v, g, _, _, _ = _case(cuda, S, T, Cn, F32)
    held = torch.zeros(S, T + 3, 3 * Cn, device=cuda)
    held[:, :T, :Cn], held[:, :T, 2 * Cn:] = v, g
    want, _ = helix_b200.gated_scan(v, g)
    d = abi.GatedScanDesc()
    ctx.lib.helix_gated_scan_desc_init(C.byref(d), T, S, Cn)
    d.s_v = d.s_g = d.s_y = 3 * Cn
    d.seq_v = d.seq_g = d.seq_y = (T + 3) * 3 * Cn
    h1 = torch.empty(S, Cn, device=cuda)
    part = [abi.Tensor(held.data_ptr(), 4 * Cn * k) for k in range(3)]
    none, st = helix_b200._t(None), torch.cuda.current_stream().cuda_stream
    call = lambda y: ctx.lib.helix_gated_scan_encode(  # noqa: E731
        ctx.handle, st, C.byref(d), part[0], part[2], none, none, y, helix_b200._t(h1), none)
    assert call(part[1]) == abi.HELIX_OK, ctx.last_error()
    assert torch.equal(held[:, :T, Cn:2 * Cn], want)
    for off in (4 * Cn - 4, 4 * Cn + 4, 0, 12 * Cn, 12 * Cn * (T + 3)):
        assert call(abi.Tensor(held.data_ptr(), off)) == abi.HELIX_ERR_INVALID_ARG, off
    torch.cuda.synchronize()


@pytest.mark.parametrize("S,T,Cn", [(2, 9, 33), (2, 300, 67), (1, 3000, 131), (40, 200, 321)])
@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("t", [BF, F32])
def test_in_place_of_copied_rows(cuda, S, T, Cn, shift, t):
    """dv in place of dy in rows that are copied in 16-byte pieces, which hold
    bytes of the rows and channels beside them; what lies between stays."""
    v, g, dy, dh1, states = _case(cuda, S, T, Cn, t)
    want = helix_b200.gated_scan_grad(dy, v, g, states, dh1)
    pitch = Cn + shift
    held = torch.full((S * T * pitch + shift,), 7.0, dtype=t, device=cuda)
    rows = held[shift:].view(S, T, pitch)[..., :Cn]
    rows.copy_(dy)
    got = helix_b200.gated_scan_grad(rows, v, g, states, dh1, dv=rows)
    assert got[0] is rows
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    rows.fill_(7.0)
    assert (held == 7.0).all()
    # h1 in place of h0, too
    state = dh1.clone()
    y, h1 = helix_b200.gated_scan(v, g, dh1)
    y2, same = helix_b200.gated_scan(v, g, state, h1=state)
    assert same is state and torch.equal(y, y2) and torch.equal(h1, state)
