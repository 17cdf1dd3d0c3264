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


def off(got, want):
    return ((got.detach().cpu().double() - want).norm() / want.norm()).item()


# (tolerances: 4.7e-5 as above; of a float16 result 2^-11, of a bfloat16 one 1.5 times 2^-8, the largest rounding of an element)
SMALL = {torch.float32: 4.7e-5, torch.float16: 2. ** -11 + 4.7e-5, torch.bfloat16: 1.5 * 2. ** -8}


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,scale,eps', [(torch.float32, s, e) for s, e in (
    (1e-8, 1e-7), (1e-10, 1e-7), (1e-13, 1e-7), (1e-16, 1e-7), (1e-20, 1e-7), (1e-30, 1e-7), (1e-36, 1e-2), (1., 1e12),
    (1e-3, 1e20))] + [(torch.bfloat16, 1e-20, 1e-7), (torch.bfloat16, 1e-12, 1e-7), (torch.float16, 1., 1e3), (torch.float16, 1e-1, 1e3)])
@pytest.mark.parametrize('shape', SHAPES)
def test_norms_that_are_small_beside_eps(shape, dtype, scale, eps):
    """The iterate is then small throughout, and as exact as any other."""
    g = (torch.randn(shape, generator=torch.Generator().manual_seed(0)) * scale).to(dtype).cuda()
    want = reference(g, eps)
    assert off(torchsso.utils.orthogonalize(g, eps=eps), want) <= SMALL[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize('scale', [1e-4, 1e-12, 1e-24])
@pytest.mark.parametrize('schedule', [((7.7, -14., 7.),), ((0.5, 0., 0.),) * 3, ((1.5, -0.5, 0.),) * 8,
                                      ((3.4, -4.7, 2.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375))])
def test_other_coefficients_on_small_norms(schedule, scale):
    for shape in SHAPES:
        g = (torch.randn(shape, generator=torch.Generator().manual_seed(1)) * scale).cuda()
        x = g.cpu().double()
        x = x / (x.norm() + 1e-7)
        for a, b, c in schedule:
            m = x @ x.t()
            x = a * x + (b * m + c * m @ m) @ x
        assert off(torchsso.utils.orthogonalize(g, len(schedule), schedule), x) <= 4.7e-5


@pytest.mark.gpu
def test_small_and_ordinary_matrices_in_one_list():
    """Every matrix has a scale of its own, in launches that reduce in pieces too."""
    shapes = [(300, 900), (900, 300), (64, 3000), (300, 900), (16, 20), (16, 20), (1100, 1300)]
    scales = [1., 1e-12, 1e-20, 1e-7, 1e-15, 1., 1e-18]
    mats = [(torch.randn(s, generator=torch.Generator().manual_seed(i)) * k).cuda()
            for i, (s, k) in enumerate(zip(shapes, scales))]
    for m, o in zip(mats, torchsso.utils.orthogonalize(mats)):
        assert off(o, reference(m, 1e-7)) <= 4.7e-5


@pytest.mark.gpu
def test_muon_of_small_gradients():
    shape = (70, 200)
    g = torch.randn(shape, generator=torch.Generator().manual_seed(0)) * 1e-18
    p, buf = torch.zeros(shape, device='cuda'), torch.zeros(shape, device='cuda')
    torchsso.optim.muon([p], [g.cuda()], [buf], lr=1., momentum=0.5, nesterov=False)
    assert off(p, -reference(g, 1e-7)) <= 4.7e-5
