"""The decoder example: a model whose matrices, gains and embedding are trained by the operators together."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_decoder_example_trains():
    spec = importlib.util.spec_from_file_location('decoder_example', os.path.join(ROOT, 'examples', 'decoder.py'))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, follows = example.main(['--steps', '120'])
    # (a uniform guess is log(64) = 4.16)
    assert losses[0] > 4. and losses[-1] < 0.8 * losses[0]
    assert 0. <= follows <= 1.
