"""The decoder example's answers: the last norm and layer in 8 bits against the same in bfloat16.

An element in 8 bits (three behind the leading one) is off by 2^-4 / sqrt(3) of its power of two at most on average, 2.6 %
of itself over an octave.  Of a logit, a sum over elements y of the norm and w of the weight, that is
    unit = sqrt(2) * 0.026 * sqrt(sum y^2 w^2) = 0.037 sqrt(sum y^2 w^2)
on average; bfloat16's own rounding is a tenth of it.
"""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def model():
    spec = importlib.util.spec_from_file_location('decoder_example', os.path.join(ROOT, 'examples', 'decoder.py'))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(0)
    model = example.Decoder()
    with torch.no_grad():
        # gains and rows of the last layer's weight of different sizes, so that every scale counts
        model.norm.weight.uniform_(0.5, 2.)
        model.head.weight.mul_(torch.linspace(0.2, 5., model.head.weight.shape[0], device='cuda').unsqueeze(1).bfloat16())
    return model


def logits_and_unit(model, x, stream):
    """In 64 bits from the norm on."""
    h = (x.float() + stream.float()).to(x.dtype).double()
    y = h / (h.square().mean(-1, keepdim=True) + model.norm.eps).sqrt() * model.norm.weight.double()
    w = model.head.weight.double().t().contiguous()
    return y @ w, 0.037 * (y.square() @ w.square()).sqrt()


@torch.no_grad()
def test_logits(model):
    tokens = torch.randint(0, 64, (48, 20), device='cuda')
    x, stream = model.body(tokens)
    # tokens whose largest elements differ, in the last place of the texts
    x, stream = x[:, -1].clone(), stream[:, -1].clone()
    x[::3, 5] += 20.
    want, unit = logits_and_unit(model, x, stream)
    got = model.logits_8(x, stream, *model.head_8()).double()
    off = (got - want) / unit
    assert off.square().mean().sqrt() <= 1.5 and off.abs().max() <= 8.


@torch.no_grad()
def test_what_is_generated_has_the_largest_logit(model):
    start = torch.randint(0, 64, (32, 9), device='cuda')
    out = model.generate(start, 5)
    assert torch.equal(out[:, :9], start) and out.shape == (32, 14)
    for t in range(9, 14):
        x, stream = model.body(out[:, :t])
        want, unit = logits_and_unit(model, x[:, -1], stream[:, -1])
        chosen = out[:, t:t + 1]
        most = want.max(-1, keepdim=True)
        # (both may be off, each by several units)
        short = (most.values - want.gather(1, chosen)) / torch.maximum(unit.gather(1, chosen), unit.gather(1, most.indices))
        assert short.max() <= 8.
