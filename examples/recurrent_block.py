"""A recurrent block from the operators of helix_b200.block: prefill, decoding
by single tokens, and a training step.

    residual += u;  n = norm(residual)
    v, g      = n W_in^T            (8-bit product, one for both)
    y         = gated recurrence of v with gates g
    out       = norm(y) W_out^T     (8-bit product)

    python -m examples.recurrent_block
"""
from __future__ import annotations

import torch

import helix_b200 as hx

F8 = torch.float8_e4m3fn


class RecurrentBlock:
    """width: of the residual stream; chans: of the recurrence."""

    def __init__(self, width: int, chans: int, device="cuda", seed: int = 0):
        gen = torch.Generator(device=device).manual_seed(seed)

        def randn(*shape, std):
            return torch.randn(*shape, generator=gen, device=device) * std

        self.width, self.chans = width, chans
        self.w_norm = torch.ones(width, device=device)
        self.w_in = randn(2 * chans, width, std=width ** -0.5)
        self.w_in[chans:] *= 2.0  # gates
        self.w_mid = torch.ones(chans, device=device)
        self.w_out = randn(width, chans, std=chans ** -0.5)
        self.lay_out()

    def lay_out(self) -> None:
        """Puts the weights into 8 bits; again after every update."""
        self.in8, self.out8 = hx.quantize8(self.w_in, blocks=True), hx.quantize8(self.w_out, blocks=True)

    def forward(self, u, residual, state=None, lengths=None, keep=False):
        """u, residual (sequences, tokens, width) -> (out, residual + u, state
        after the last token[, what backward needs])."""
        n = hx.rms_norm(u, self.w_norm, residual, out_dtype=F8, keep_rstd=keep)
        vg = hx.matmul8(n.out, n.scale, *self.in8)
        v, g = vg[..., :self.chans], vg[..., self.chans:]
        y, state, *states = hx.gated_scan(v, g, state, lengths=lengths, keep_states=keep)
        m = hx.rms_norm(y, self.w_mid, out_dtype=F8, keep_rstd=keep)
        out = hx.matmul8(m.out, m.scale, *self.out8)
        if not keep:
            return out, n.sum, state
        return out, n.sum, state, (n.sum, n.rstd, vg, y, m.rstd, states[0], lengths)

    def step(self, u, residual, state):
        """One token of each sequence, the state updated in place."""
        n = hx.rms_norm(u, self.w_norm, residual, out_dtype=F8)
        vg = hx.matmul8(n.out, n.scale, *self.in8)
        y, _ = hx.gated_scan(vg[..., :self.chans], vg[..., self.chans:], state, h1=state)
        m = hx.rms_norm(y, self.w_mid, out_dtype=F8)
        return hx.matmul8(m.out, m.scale, *self.out8), n.sum

    def _linear_grad(self, dout, weight, x):
        """Gradients of x W^T: of x as an 8-bit product with W transposed, of
        W as one of both transposed, groups along the tokens."""
        dx = hx.matmul8(*hx.quantize8(dout), *hx.quantize8(weight, blocks=True, transpose=True))
        dw = hx.matmul8(*hx.quantize8(dout, transpose=True), *hx.quantize8(x, transpose=True), out_dtype=torch.float32)
        return dx, dw

    def backward(self, dout, dsum, kept):
        """Gradients of u (the residual's is the same), the first state and
        the four weights, from those of out and of the residual stream."""
        total, rstd, vg, y, rstd_mid, states, lengths = kept
        shape, c = dout.shape, self.chans
        m = hx.rms_norm(y, self.w_mid).out
        dm, dw_out = self._linear_grad(dout.flatten(0, 1), self.w_out, m.flatten(0, 1))
        dy, dw_mid = hx.rms_norm_grad(dm.view(y.shape), y, rstd_mid, self.w_mid)
        dvg = torch.empty_like(vg)
        _, _, dstate = hx.gated_scan_grad(dy, vg[..., :c], vg[..., c:], states, lengths=lengths, dv=dvg[..., :c],
                                          dg=dvg[..., c:])
        n = hx.rms_norm(total, self.w_norm).out
        dn, dw_in = self._linear_grad(dvg.flatten(0, 1), self.w_in, n.flatten(0, 1))
        du, dw_norm = hx.rms_norm_grad(dn.view(shape), total, rstd, self.w_norm, dsum)
        return du, dstate, {"w_norm": dw_norm, "w_in": dw_in, "w_mid": dw_mid, "w_out": dw_out}


def main() -> None:
    torch.manual_seed(0)
    S, T, width, chans = 4, 1024, 2048, 2048
    block = RecurrentBlock(width, chans)
    u = torch.randn(S, T, width, device="cuda").bfloat16()
    residual = torch.randn(S, T, width, device="cuda").bfloat16()

    out, stream, state = block.forward(u, residual)
    print(f"prefill: {S} x {T} tokens, out {tuple(out.shape)}, rms {out.float().square().mean().sqrt().item():.3f}")
    for _ in range(3):
        out, stream = block.step(out[:, -1:].contiguous(), stream[:, -1:].contiguous(), state)
    print(f"3 steps: state rms {state.square().mean().sqrt().item():.3f}")

    target = torch.randn(S, T, width, device="cuda")
    for i in range(5):
        out, _, _, kept = block.forward(u, residual, keep=True)
        err = out.float() - target
        _, _, grads = block.backward((err / err.numel() * 1e4).bfloat16(), None, kept)
        for name, g in grads.items():
            getattr(block, name).sub_(g, alpha=2e-2)
        block.lay_out()
        print(f"training step {i}: loss {err.square().mean().item():.4f}")


if __name__ == "__main__":
    main()
