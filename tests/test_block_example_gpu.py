"""GPU: the operators together, as examples/recurrent_block.py runs them.

Bounds.  e4m3 values are off by 2^-4 / sqrt(3) rms at most (2.6 % measured on
normal values), each product of two quantised operands by sqrt(2) of that,
3.7 %.  A value that has passed p products with independent errors is off by
about 3.7 sqrt(p) %; forward out: two products, 6 % with slack; a gradient has
the forward's two and one or two of its own: 10 %."""
import pytest
import torch

from examples.recurrent_block import RecurrentBlock

pytestmark = pytest.mark.gpu


def _plain(block, u, residual, weights, state):
    """The block in fp64 with autograd, unquantised."""
    total = u + residual
    n = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + 1e-6) * weights["w_norm"]
    vg = n @ weights["w_in"].T
    v, f = vg[..., :block.chans], torch.sigmoid(vg[..., block.chans:])
    h, ys = state, []
    for t in range(u.shape[1]):
        h = f[:, t] * h + (1 - f[:, t]) * v[:, t]
        ys.append(h)
    y = torch.stack(ys, 1)
    m = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weights["w_mid"]
    return m @ weights["w_out"].T, total, h


def _off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("S,T,width,chans", [(2, 260, 512, 640), (3, 37, 300, 200)])
def test_block_against_autograd(cuda, S, T, width, chans):
    block = RecurrentBlock(width, chans, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    u, residual, dout, dsum = (torch.randn(S, T, width, generator=gen, device="cuda").bfloat16() for _ in range(4))
    state = torch.randn(S, chans, generator=gen, device="cuda")
    out, total, h1, kept = block.forward(u, residual, state, keep=True)
    du, dstate, grads = block.backward(dout, dsum, kept)
    weights = {k: getattr(block, k).double().requires_grad_() for k in grads}
    ud, sd = u.double().requires_grad_(), state.double().requires_grad_()
    want, wtotal, wh1 = _plain(block, ud, residual.double(), weights, sd)
    ((want * dout.double()).sum() + (wtotal * dsum.double()).sum()).backward()
    assert _off(out, want.detach()) < 0.06 and _off(h1, wh1.detach()) < 0.06
    assert _off(total, wtotal.detach()) < 2 ** -8
    assert _off(du, ud.grad) < 0.10 and _off(dstate, sd.grad) < 0.10
    for k, g in grads.items():
        assert g.shape == weights[k].shape
        assert _off(g, weights[k].grad) < 0.10, k


def test_steps_follow_a_prefill(cuda):
    """Tokens one by one give what a prefill of all of them gives: the same
    8-bit values (a token's groups are its own), so only the order of the
    recurrence's and the products' sums differs: 2^-7 with bf16 outputs."""
    S, T, width, chans = 2, 40, 384, 256
    block = RecurrentBlock(width, chans, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    u, residual = (torch.randn(S, T, width, generator=gen, device="cuda").bfloat16() for _ in range(2))
    want, wstream, wstate = block.forward(u, residual)
    out, _, state = block.forward(u[:, :30].contiguous(), residual[:, :30].contiguous())
    assert _off(out, want[:, :30].double()) < 2 ** -7
    for t in range(30, T):
        out, stream = block.step(u[:, t:t + 1].contiguous(), residual[:, t:t + 1].contiguous(), state)
        assert _off(out, want[:, t:t + 1].double()) < 2 ** -7
        assert torch.equal(stream, wstream[:, t:t + 1])
    assert _off(state, wstate.double()) < 2 ** -7


def test_a_step_in_a_graph(cuda):
    """A decoder's step captured once and replayed on new inputs."""
    block = RecurrentBlock(512, 512, seed=5)
    gen = torch.Generator(device="cuda").manual_seed(6)
    u, residual = (torch.randn(4, 1, 512, generator=gen, device="cuda").bfloat16() for _ in range(2))
    state = torch.randn(4, 512, generator=gen, device="cuda")
    block.step(u, residual, state.clone())
    held = state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, stream = block.step(u, residual, held)
    held.copy_(state)
    for _ in range(3):
        u.normal_(generator=gen)
        before = held.clone()
        graph.replay()
        torch.cuda.synchronize()
        want, wstream = block.step(u, residual, before)
        assert torch.equal(out, want) and torch.equal(stream, wstream) and torch.equal(held, before)
    del graph


def test_training_lowers_the_loss(cuda):
    torch.manual_seed(7)
    block = RecurrentBlock(256, 256, seed=8)
    u, residual = (torch.randn(4, 64, 256, device="cuda").bfloat16() for _ in range(2))
    target = torch.randn(4, 64, 256, device="cuda")
    losses = []
    for _ in range(8):
        out, _, _, kept = block.forward(u, residual, keep=True)
        err = out.float() - target
        losses.append(err.square().mean().item())
        _, _, grads = block.backward((err * 2 / err[0, 0].numel()).bfloat16(), None, kept)
        for name, g in grads.items():
            getattr(block, name).sub_(g, alpha=2e-2)
        block.lay_out()
    assert losses[-1] < losses[0]
