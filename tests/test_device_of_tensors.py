"""The calls for decoders launch with the device of their tensors current: the handle of a device's null stream is null,
and a launch on it goes to whichever device is current."""
import contextlib

import pytest
import torch

from torchsso import _hip, _ops


class Tensor(object):
    """What the wrappers look at of a tensor on the second device."""
    device, dtype = torch.device('cuda', 1), torch.float32

    def __init__(self, *shape, address=1 << 20):
        self.shape, self.address = torch.Size(shape), address

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def data_ptr(self):
        return self.address

    def reshape(self, *shape):
        return self

    def stride(self, i):
        return 1 if i == 1 else self.shape[-1]

    is_cuda = True


@pytest.fixture
def launches(monkeypatch):
    """(entry point, device that was current) of every call of the engine; device 0 is current outside of them"""
    current, seen = [0], []

    class Lib(object):

        def __getattr__(self, name):
            def call(*args):
                seen.append((name, current[-1]))
                return 64 if name.endswith('workspace_bytes') else 0
            return call

    @contextlib.contextmanager
    def use(device):
        current.append(device.index)
        yield
        current.pop()
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: current[-1])
    monkeypatch.setattr(torch.cuda, 'device', use)
    monkeypatch.setattr(_hip, 'load', lambda: Lib())
    monkeypatch.setattr(_hip, 'typed_ptr', lambda t, *args: t.data_ptr())
    monkeypatch.setattr(_hip, 'stream_ptr', lambda device=None, stream=None: 0)
    monkeypatch.setattr(_hip, 'workspace', lambda device, nbytes, stream=None: (None, nbytes))
    monkeypatch.setattr(torch, 'empty', lambda shape, dtype=None, device=None: Tensor(*shape))
    monkeypatch.setattr(torch, 'empty_like', lambda t: Tensor(*t.shape))
    return seen


def on_second(launches, name):
    assert [d for n, d in launches if n == name] == [1]


def test_orthogonalize(launches):
    _ops.orthogonalize_batched([Tensor(4, 5)], [Tensor(4, 5)], (1.5, -0.5, 0.), 1e-7)
    on_second(launches, 'kfac_orthogonalize_batched')


def test_muon(launches):
    _ops.muon_update_batched([Tensor(4, 5)], [Tensor(4, 5)], [Tensor(4, 5, address=1 << 21)], [0.1], [1.], 0.9, True,
                             (1.5, -0.5, 0.), 1e-7)
    on_second(launches, 'kfac_muon_update_batched')


def test_norm_backward(launches):
    _ops.rms_norm_backward(Tensor(4, 5), None, Tensor(4, 5), Tensor(5), 1e-6, 2)
    on_second(launches, 'kfac_rms_norm_backward')
