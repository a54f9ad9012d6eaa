"""The group-decode operators' checks of their tensors (no GPU here: the tensors only say that
they are on one, and the launch is a recorder)."""

import pytest
import torch

from shellsmith_b200 import beam, paged, rotary


class OnDevice(torch.Tensor):
    """A CPU tensor that names a GPU as its device."""
    __torch_function__ = torch._C._disabled_torch_function_impl

    is_cuda = True
    index = 0

    def get_device(self):
        return self.index

    def new_empty(self, *args, **kw):
        return on(torch.Tensor.new_empty(self, *args, **kw), self.index)


def on(t, index=0):
    t = t.as_subclass(OnDevice)
    t.index = index
    return t


@pytest.fixture
def launched(monkeypatch):
    calls = []
    for module, name in ((rotary, "_append"), (beam, "_select"), (beam, "_reorder"),
                         (paged, "_shared_prefix")):
        monkeypatch.setattr(module, name, lambda *args, n=name: calls.append(n))
    for module in (rotary, beam, paged):
        monkeypatch.setattr(module, "fast", None)
        monkeypatch.setattr(module, "stream_of", lambda t: 0)
    return calls


def _bf(*shape):
    return on(torch.zeros(shape, dtype=torch.bfloat16))


def _plan(cls, *args, **kw):
    plan = cls(*args, device="cpu", **kw)
    plan.device_index = 0
    return plan


def test_rotary_takes_subclasses_of_tensor(launched):
    """A torch.nn.Parameter, say: the compiled caller takes it, and so does the wrapper."""
    plan = _plan(rotary.RotaryPlan, 64)
    pos = on(torch.zeros((1, 4), dtype=torch.int32))
    rotary.rotary(_bf(4, 2, 64), _bf(4, 1, 64), pos, plan)
    assert launched == ["_append"]
    for bad in (_bf(4, 2, 128)[..., ::2], _bf(4, 2, 32), _bf(4, 64)):
        with pytest.raises(ValueError):
            rotary.rotary(bad, _bf(4, 1, 64), pos, plan)
    with pytest.raises(TypeError):
        rotary.rotary(on(torch.zeros((4, 2, 64))), _bf(4, 1, 64), pos, plan)
    assert launched == ["_append"]
