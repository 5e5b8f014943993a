"""GPU: sizes whose indexes would not fit are refused before anything is read."""
import ctypes as C

import pytest
import torch

import helix_b200
from helix_b200 import abi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_tok", [0, 1, 1000])
@pytest.mark.parametrize("dtype", [abi.HELIX_F32, abi.HELIX_BF16])
@pytest.mark.parametrize("n_chan", [2 ** 31 - 1, 2 ** 31 - 33, 2 ** 31 - 64])
def test_channels(cuda, ctx, n_tok, dtype, n_chan):
    T, st = helix_b200._t, torch.cuda.current_stream().cuda_stream
    held = [torch.zeros(16, device=cuda) for _ in range(9)]
    d = abi.GatedScanDesc()
    ctx.lib.helix_gated_scan_desc_init(C.byref(d), n_tok, 1, n_chan)
    d.io_dtype = dtype
    v, g, y, h1, states, dy, dv, dg, dh0 = map(T, held)
    none = T(None)
    assert ctx.lib.helix_gated_scan_encode(ctx.handle, st, C.byref(d), v, g, none, none, y, h1,
                                           none) == abi.HELIX_ERR_UNSUPPORTED_SHAPE
    assert "n_chan" in ctx.last_error()
    assert ctx.lib.helix_gated_scan_grad_encode(ctx.handle, st, C.byref(d), dy, v, g, states, none, none, dv, dg,
                                                dh0) == abi.HELIX_ERR_UNSUPPORTED_SHAPE
    assert "n_chan" in ctx.last_error()
    torch.cuda.synchronize()
