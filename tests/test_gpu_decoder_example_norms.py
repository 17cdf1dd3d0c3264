"""The decoder example with either norm: it runs, its gradients are those of the same model in torch's operations, and
its optimizers change every parameter."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

import torchsso

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location('decoder_example_norms', os.path.join(ROOT, 'examples', 'decoder.py'))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


@pytest.mark.parametrize('norm', ['rms', 'layer'])
def test_runs(norm):
    losses, follows = example.main(['--steps', '3', '--batch', '8', '--norm', norm])
    assert len(losses) == 3 and all(0. < x < 10. for x in losses) and 0. <= follows <= 1.


def plain_norm(module):
    def forward(x, residual):
        h = x + residual
        h32 = h.float()
        if isinstance(module, torchsso.nn.LayerNorm):
            y = F.layer_norm(h32, (module.dim,), module.weight, module.bias, module.eps)
        else:
            y = F.rms_norm(h32, (module.dim,), module.weight, module.eps)
        return y.to(h.dtype), h
    return forward


@pytest.mark.parametrize('norm', [torchsso.nn.RMSNorm, torchsso.nn.LayerNorm])
def test_gradients(norm):
    """Both models round to bfloat16 in the same places, the gradients of the norms aside: of a parameter's gradient some tens of
    roundings of 2^-9 on average are left, which is 2^-9 sqrt(50) = 1.4 %; three times that."""
    torch.manual_seed(0)
    model = example.Decoder(norm=norm)
    gen = torch.Generator().manual_seed(1)
    x = example.text(8, 33, gen, 'cuda')

    def gradients():
        model.zero_grad()
        F.cross_entropy(model(x[:, :-1]).reshape(-1, example.VOCAB), x[:, 1:].reshape(-1)).backward()
        return {name: p.grad.double() for name, p in model.named_parameters()}
    got = gradients()
    modules = [m for m in model.modules() if isinstance(m, norm)]
    for m in modules:
        m.forward = plain_norm(m)
    want = gradients()
    for name in want:
        error = ((got[name] - want[name]).norm() / want[name].norm()).item()
        assert error <= 0.042, (name, error)


def test_every_parameter_moves():
    torch.manual_seed(0)
    model = example.Decoder(norm=torchsso.nn.LayerNorm)
    norms = torch.nn.ModuleList(m for m in model.modules() if isinstance(m, torchsso.nn.LayerNorm))
    matrices = [m.weight for m in model.modules() if isinstance(m, torch.nn.Linear)]
    opts = [torchsso.optim.Muon(matrices, lr=0.02),
            torchsso.optim.SecondOrderOptimizer(norms, 'Cov', {'LayerNorm': 'Diag'}, {'damping': 1e-2}, lr=1e-2),
            torchsso.optim.AdamW(model.embedding.parameters(), lr=1e-2, state_bits=8)]
    before = [p.detach().clone() for p in model.parameters()]
    x = example.text(16, 33, torch.Generator().manual_seed(1), 'cuda')
    F.cross_entropy(model(x[:, :-1]).reshape(-1, example.VOCAB), x[:, 1:].reshape(-1)).backward()
    for opt in opts:
        opt.step()
    assert 'exp_avg_scale' in opts[2].state[model.embedding.weight]
    for p, b in zip(model.parameters(), before):
        assert torch.isfinite(p).all() and not torch.equal(p, b)
