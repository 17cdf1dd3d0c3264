"""The C entry points refuse coefficients under which an operand would leave the range of fp16, by the same rule as
torchsso.utils.orthogonalize."""
import ctypes
import random

import pytest

from torchsso import _hip
from torchsso.utils.linalg import newton_schulz_schedule


def status(coefficients, muon=False):
    """Of a call without scratch: 2 (KFAC_ERR_WORKSPACE) where the coefficients are taken, 1 where they are not."""
    lib = _hip.load()
    one, fake = _hip.int_array([4]), (ctypes.c_void_p * 1)(1 << 20)
    flat = [v for t in coefficients for v in t]
    steps, flat = len(coefficients), _hip.f32_array(flat)
    if muon:
        factor = _hip.f32_array([1.])
        return lib.kfac_muon_update_batched(1, one, one, 0, fake, fake, fake, factor, factor, 0.9, 1, steps, flat, 1e-7, 0,
                                            None, 0, None)
    return lib.kfac_orthogonalize_batched(1, one, one, 0, fake, fake, steps, flat, 1e-7, 0, None, 0, None)


@pytest.mark.parametrize('muon', [False, True])
def test_refused_coefficients(muon):
    good = (3.4445, -4.7750, 2.0315)
    assert status([good] * 5, muon) == 2 and status([good] * 64, muon) == 2 and status([good] * 65, muon) == 1
    # a norm of 5, whose square is beyond 8
    assert status([(5., 0., 0.), (1., 0., 0.)], muon) == 1
    assert status([(2.7, 0., 0.)], muon) == 2 and status([(2.8, 0., 0.)], muon) == 1
    assert status([(7.8, -7., 0.)], muon) == 1 and status([(7.7, -14., 7.)], muon) == 2
    for bad in (float('nan'), float('inf'), -float('inf')):
        for i in range(3):
            assert status([good, tuple(bad if j == i else v for j, v in enumerate(good))], muon) == 1


def test_the_same_rule_on_both_sides():
    rng = random.Random(0)
    seen = set()
    for _ in range(2000):
        size = rng.choice([1., 3., 8.])
        steps = [tuple(float(ctypes.c_float(rng.uniform(-size, size)).value) for _ in range(3))
                 for _ in range(rng.randint(1, 4))]
        if rng.random() < 0.3:
            steps = [t[:2] + (0.,) for t in steps]
        try:
            newton_schulz_schedule(len(steps), steps)
            want = 2
        except ValueError:
            want = 1
        assert status(steps) == want, steps
        seen.add(want)
    assert seen == {1, 2}
