"""What steps in 11 bits at the end of an orthogonalisation of bfloat16 matrices add to its error."""
import pytest
import torch

import torchsso
from torchsso import _ops

pytestmark = pytest.mark.gpu

DEFAULT = (3.4445, -4.7750, 2.0315)
SCHEDULES = {'default': (DEFAULT,) * 5, 'one': (DEFAULT,), 'cubic': ((1.5, -0.5, 0.),) * 5,
             # (a direction of singular value 1 is taken to 0.9, 1.1 and close to zero in the end)
             'steep': ((2.6, -1.7, 0.),) * 5,
             'falling': ((3.4, -4.7, 2.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375))}


def matrices():
    gen = torch.Generator().manual_seed(0)
    rows, cols = 256, 512
    noise = torch.randn(rows, cols, generator=gen)
    one = torch.randn(rows, 1, generator=gen) @ torch.randn(1, cols, generator=gen)
    left, right = (torch.linalg.qr(torch.randn(n, n, generator=gen))[0] for n in (rows, cols))
    out = {'noise': noise}
    out.update(('one direction and %g of noise' % level, one + level * noise) for level in (1e-1, 1e-2, 1e-3, 1e-4))
    out.update(('spectrum k^-%d' % p, (left * torch.arange(1., rows + 1) ** -p) @ right[:rows]) for p in (1, 2, 4))
    return out


def reference(g, schedule):
    x = g.double()
    x = x / (x.norm() + 1e-7)
    for a, b, c in schedule:
        m = x @ x.t().contiguous()
        x = a * x + (b * m + c * m @ m) @ x
    return x


@pytest.mark.parametrize('name', sorted(SCHEDULES))
def test_one_and_a_half_times_the_rounding_of_the_result_at_most(name):
    schedule = SCHEDULES[name]
    for what, m in matrices().items():
        g = m.to(torch.bfloat16)
        want = reference(g, schedule)
        rounding = (want.to(torch.bfloat16).double() - want).norm()
        out = torchsso.utils.orthogonalize(g.cuda(), len(schedule), schedule)
        error = (out.cpu().double() - want).norm()
        # (beside that float32's own errors: the result's rounding is 2^-9, theirs 2^-20)
        assert error <= 1.5 * rounding + 2 ** -20 * want.norm(), (what, (error / rounding).item())


def test_more_late_steps_than_that_are_not_taken():
    flat = {name: tuple(v for t in s for v in t) for name, s in SCHEDULES.items()}
    late = {name: _ops.late_steps(torch.bfloat16, s) for name, s in flat.items()}
    assert late == {'default': 1, 'one': 1, 'cubic': 3, 'steep': 0, 'falling': 2}
    for dtype in (torch.float32, torch.float16):
        assert all(_ops.late_steps(dtype, s) == 0 for s in flat.values())


@pytest.mark.parametrize('shape', [(65, 300), (256, 512), (3, 4000), (1000, 40)])
@pytest.mark.parametrize('schedule', list(SCHEDULES.values()) + [
    ((1.5262, -1.7437, 0.8985), (2.7571, -1.7730, 1.9739), (0.9136, -0.6772, 0.2028))])
def test_single_elements_that_hold_the_norm(shape, schedule):
    """Their roundings do not average out: they may be 1.1 times the largest rounding of an element of the result, 2^-8, off."""
    gen = torch.Generator().manual_seed(0)
    for count, value in ((1, 1.), (1, 1.37), (1, 1.999), (2, 1.3)):
        m = 1e-3 * torch.randn(shape, generator=gen)
        for i in range(count):
            m[i, i + 5] = value
        g = m.to(torch.bfloat16)
        want = reference(g if shape[0] <= shape[1] else g.t(), schedule)
        want = want if shape[0] <= shape[1] else want.t()
        rounding = (want.to(torch.bfloat16).double() - want).norm()
        out = torchsso.utils.orthogonalize(g.cuda(), len(schedule), schedule)
        error = (out.cpu().double() - want).norm()
        assert error <= 1.5 * rounding + 8.9 / 8 * 2 ** -8 * want.norm(), (count, value, (error / want.norm()).item())
