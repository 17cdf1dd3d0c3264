"""Sums over rows of a norm's backward pass: what the launch that adds up the units' parts rounds away."""
import pytest
import torch

import torchsso
from torchsso import _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dim', [64, 71, 4096])
@pytest.mark.parametrize('samples,tokens', [(1024, 1), (1000, 1), (4, 128), (3, 300), (1, 1000), (200, 5)])
def test_sums_of_many_positive_terms(samples, tokens, dim):
    """Rows of 1 and -1 without eps have a norm of exactly 1, so that every row's term is a number of dy and a unit
    that holds one row knows it exactly (1024 rows or fewer).  What is left are the rounding of each group's
    sum, of 2^-24 of it, and that of the result; squares of a sample's sum take its rounding twice."""
    gen = torch.Generator().manual_seed(0)
    x = (torch.randint(0, 2, (samples, tokens, dim), generator=gen) * 2. - 1)
    dy = torch.rand((samples, tokens, dim), generator=gen) + 1
    terms = dy.double()
    curvature = torch.empty(dim, device='cuda')
    _, dgain = _ops.rms_norm_backward((dy * x).cuda(), None, x.cuda(), torch.ones(dim, device='cuda'), 0., samples,
                                      curvature=curvature)
    s = terms.sum(1)
    want, squares = s.sum(0), samples * s.square().sum(0)
    assert ((dgain.cpu().double() - want).abs() / want).max() <= 2 * 2 ** -24
    assert ((curvature.cpu().double() - squares).abs() / squares).max() <= 4 * 2 ** -24
