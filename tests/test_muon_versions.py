"""An update of Muon is a change in place that autograd sees, as those of torch's optimizers are."""
import pytest
import torch

import torchsso
from torchsso import _ops


def backward_over_a_step(device):
    p = torch.nn.Parameter(torch.randn(4, 6, device=device))
    opt = torchsso.optim.Muon([p], lr=0.1)
    x = torch.randn(3, 6, device=device, requires_grad=True)
    before = (x @ p.t()).square().sum()
    p.grad = torch.randn(4, 6, device=device)
    buffers = []
    for _ in range(2):
        version = p._version
        opt.step()
        assert p._version > version
        buffers.append(opt.state[p]['momentum_buffer']._version)
    assert buffers[1] > buffers[0]
    with pytest.raises(RuntimeError, match='inplace'):
        before.backward()
    (x @ p.t()).square().sum().backward()


def test_a_graph_from_before_a_step_is_refused(monkeypatch):
    monkeypatch.setattr(_ops, 'muon_update_batched', lambda *args: None)
    backward_over_a_step('cpu')


def test_the_function_alone(monkeypatch):
    monkeypatch.setattr(_ops, 'muon_update_batched', lambda *args: None)
    p, g, b = torch.zeros(4, 6), torch.zeros(4, 6), torch.zeros(4, 6)
    torchsso.optim.muon([p], [g], [b], lr=0.1)
    assert p._version > 0 and b._version > 0 and g._version == 0
    torchsso.optim.muon([], [], [], lr=0.1)


@pytest.mark.gpu
def test_a_graph_from_before_a_step_is_refused_on_the_device():
    backward_over_a_step('cuda')
