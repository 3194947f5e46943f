"""AttentionLayer.forward and TokenHead.forward refuse rows of another device than their buffers', and a call while another device
is current, before anything is queued. No GPU is needed: stand-ins for tensors have all that the checks look at."""
import types

import pytest

torch = pytest.importorskip("torch")

from libosmos_amd import block  # noqa: E402

N, DIM = 3, 64


def _tensor(device, shape=(N, DIM)):
    return types.SimpleNamespace(dtype=torch.float32, is_cuda=True, is_contiguous=lambda: True, shape=shape, device=torch.device("cuda", device),
                                 data_ptr=lambda: pytest.fail("an address was asked for"))


def _attention():
    layer = block.AttentionLayer.__new__(block.AttentionLayer)
    layer.dim, layer.norm, layer.eps = DIM, None, 1e-6
    calls = block._Calls((None, None))
    calls.owner, calls.n, calls.buffers = layer, N, dict(x16=_tensor(0), qkv=_tensor(0))
    return layer, calls


def _head():
    head = block.TokenHead.__new__(block.TokenHead)
    head.dim, head.norm, head.eps = DIM, None, 1e-6
    calls = block._Calls((None,))
    calls.owner, calls.n, calls.buffers = head, N, (_tensor(0), _tensor(0))
    return head, calls


@pytest.mark.parametrize("bad", ["x", "out", "add"])
def test_attention_rows_of_another_device(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    layer, calls = _attention()
    t = {name: _tensor(1 if name == bad else 0) for name in ("x", "out", "add")}
    with pytest.raises(ValueError, match="another device"):
        layer.forward(t["x"], calls, t["out"], add=t["add"])


@pytest.mark.parametrize("bad", ["x", "add"])
def test_head_rows_of_another_device(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    head, calls = _head()
    t = {name: _tensor(1 if name == bad else 0) for name in ("x", "add")}
    with pytest.raises(ValueError, match="another device"):
        head.forward(t["x"], calls, add=t["add"])


def test_another_device_is_current(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    layer, calls = _attention()
    with pytest.raises(RuntimeError, match="not current"):
        layer.forward(_tensor(0), calls, _tensor(0))
    head, calls = _head()
    with pytest.raises(RuntimeError, match="not current"):
        head.forward(_tensor(0), calls)
    with pytest.raises(ValueError, match="another device"):
        block._weight(types.SimpleNamespace(dtype=torch.float32, shape=(DIM,), is_contiguous=lambda: True, is_cuda=True,
                                            device=torch.device("cuda", 0)), DIM)
