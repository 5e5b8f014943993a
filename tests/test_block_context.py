"""CPU: the context a block operator is called with."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")


class OnDevice(torch.Tensor):
    """A tensor that says it is on a CUDA device."""
    index = 0

    def get_device(self):
        return self.index


def _tensor(index):
    t = torch.empty(1).as_subclass(OnDevice)
    t.index = index
    return t


def test_context_of_another_device_is_refused():
    """Its kernels would get the other device's pointers (and, on the default
    stream, run)."""
    from helix_b200 import block
    ctx = SimpleNamespace(device=0, handle=SimpleNamespace(value=17))
    assert block._ctx(ctx, _tensor(0)) == 17
    with pytest.raises(ValueError, match="device"):
        block._ctx(ctx, _tensor(1))
    with pytest.raises(ValueError, match="CUDA"):
        block._ctx(ctx, torch.empty(1))


def test_context_knows_its_device(monkeypatch):
    import helix_b200

    class Lib:
        asked = []

        def helix_ctx_create(self, out, device, path):
            self.asked.append(None if device is None else device._obj.value)
            return 0

        def helix_ctx_free(self, handle):
            pass

    lib = Lib()
    monkeypatch.setattr(helix_b200.abi, "load", lambda: lib)
    assert helix_b200.Context(3).device == 3
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)
    assert helix_b200.Context().device == 2
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: False)
    assert helix_b200.Context().device is None
    assert lib.asked == [3, 2, None]
