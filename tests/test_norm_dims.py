"""Rows that are longer than the norm's kernels count are refused, whatever their length is in 32 bits."""
import pytest
import torch

import torchsso
from torchsso import _hip, _ops

LENGTHS = [(1 << 24) + 1, (1 << 32) + 8, (1 << 33) + 64]


def refused(length, device):
    x = torch.ones(1, 1, device=device, dtype=torch.bfloat16).expand(1, length)
    for call in (lambda: torchsso.nn.rms_norm(x), lambda: torchsso.nn.add_rms_norm(x, x),
                 lambda: torchsso.nn.rms_norm(x, out_dtype=torch.float8_e4m3fn),
                 lambda: _ops.rms_norm_backward(x, None, x, None, 1e-6, 1)):
        with pytest.raises(_hip.KfacHipError, match='1 to 16777216 elements'):
            call()


@pytest.mark.parametrize('length', LENGTHS)
def test_long_rows_are_refused(length):
    refused(length, 'cpu')


@pytest.mark.gpu
@pytest.mark.parametrize('length', LENGTHS)
def test_long_rows_are_refused_on_the_device(length):
    refused(length, 'cuda')


def test_the_limit_is_that_of_the_engine():
    lib = _hip.load()
    assert lib.kfac_rms_norm_backward_workspace_bytes(0, 4, _ops.NORM_MAX_DIM, 1, 0) > 0
    assert lib.kfac_rms_norm_backward_workspace_bytes(0, 4, _ops.NORM_MAX_DIM + 1, 1, 0) == 0
