"""Orthogonalisation of numbers close to the ends of float32's range."""
import ctypes

import pytest
import torch

import torchsso
from torchsso import _hip

SCHEDULE = ((3.4445, -4.7750, 2.0315),) * 5
# (a matrix in one workgroup's LDS, one in 64-wide tiles, tall, and with sides that are not multiples of 8)
SHAPES = [(16, 20), (64, 200), (200, 96), (61, 131)]


def reference(g, eps):
    x = g.detach().cpu().double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.norm() + eps)
    for a, b, c in SCHEDULE:
        m = x @ x.t()
        x = a * x + (b * m + c * m @ m) @ x
    return x.t() if tall else x


def test_eps_has_to_be_a_positive_number_in_float32():
    for bad in (1e-50, 2. ** -150, 0., -1., float('nan'), float('inf'), 1e39):
        with pytest.raises(ValueError):
            torchsso.utils.orthogonalize(torch.zeros(4, 4), eps=bad)
        with pytest.raises(ValueError):
            torchsso.optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))], eps=bad)
    lib = _hip.load()
    one, fake, coeffs = _hip.int_array([4]), (ctypes.c_void_p * 1)(1 << 20), _hip.f32_array([1.5, -0.5, 0.])
    for bad, status in ((0., 1), (-1., 1), (float('nan'), 1), (float('inf'), 1), (1e-44, 2)):
        assert lib.kfac_orthogonalize_batched(1, one, one, 0, fake, fake, 1, coeffs, bad, 0, None, 0, None) == status
        assert lib.kfac_muon_update_batched(1, one, one, 0, fake, fake, fake, coeffs, coeffs, 0.9, 1, 1, coeffs, bad, 0,
                                            None, 0, None) == status


@pytest.mark.gpu
@pytest.mark.parametrize('eps', [1e-30, 1e-37, 2. ** -149])
@pytest.mark.parametrize('shape', SHAPES)
def test_zeros_stay_zeros(shape, eps):
    g = torch.zeros(shape, device='cuda')
    assert torch.equal(torchsso.utils.orthogonalize(g, eps=eps), g)
    p, buf = torch.ones(shape, device='cuda'), torch.zeros(shape, device='cuda')
    torchsso.optim.muon([p], [g], [buf], lr=0.1, eps=eps)
    assert torch.equal(p, torch.ones_like(p)) and torch.equal(buf, g)


# (tolerance: 15 products round operands to 2^-23 of an element each, which grows by the slope of the steps behind, about
# 1.5: 15 * 2^-22 * (1 + 1.5 + ... + 1.5^4) = 4.7e-5 if all errors of a step are of one sign)
@pytest.mark.gpu
@pytest.mark.parametrize('scale,eps', [(1e-40, 2. ** -149), (1e-42, 2. ** -149), (1e37, 1e-7), (3e37, 1e-7)])
@pytest.mark.parametrize('shape', SHAPES)
def test_the_smallest_and_the_largest_numbers(shape, scale, eps):
    g = (torch.randn(shape, generator=torch.Generator().manual_seed(0)) * scale).cuda()
    want = reference(g, eps)
    assert torch.isfinite(g).all()
    out = torchsso.utils.orthogonalize(g, eps=eps).cpu().double()
    assert (out - want).norm() <= 4.7e-5 * want.norm()
