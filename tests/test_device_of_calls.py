"""Sizes that depend on a device are asked for under the device that the call then runs on (no GPU needed: the
library and torch's device switch are stand-ins)."""

import contextlib

import pytest
import torch

from lava_dl_b200 import _native, _ops


class Device:
    """torch's current device, and a library that remembers which one it was called under."""

    def __init__(self, monkeypatch, current):
        self.current, self.calls = current, []
        monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: self.current)
        monkeypatch.setattr(torch.cuda, 'device', self.switch)
        monkeypatch.setattr(_native, '_lib', self)

    @contextlib.contextmanager
    def switch(self, index):
        before, self.current = self.current, torch.device('cuda', index).index if isinstance(index, int) else index.index
        yield
        self.current = before

    def __getattr__(self, name):
        if not name.startswith('sb_'):
            raise AttributeError(name)

        def entry(*args):
            self.calls.append((name, self.current))
            return 0
        return entry


@pytest.mark.parametrize('current', [0, 1])
@pytest.mark.parametrize('backward', [False, True])
def test_attention_scratch_is_sized_on_its_device(monkeypatch, current, backward):
    device = Device(monkeypatch, current)
    assert _ops._attention_scratch(4, 64, 64, 1000, backward, torch.device('cuda', 1)) is None    # (the stand-in says 0)
    assert device.calls == [('sb_linear_attention_scratch_bytes', 1)]
    assert device.current == current
