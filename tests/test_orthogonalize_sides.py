"""Matrices with sides beyond what the orthogonalisation takes are named where they are refused."""
import pytest
import torch

import torchsso
from torchsso import _hip, _ops


def test_the_engine_takes_the_sides_that_the_wrappers_let_through():
    lib = _hip.load()
    for rows, cols in ((_ops.ORTH_MAX_SIDE, 3), (3, _ops.ORTH_MAX_SIDE)):
        assert lib.kfac_orthogonalize_workspace_bytes(1, _hip.int_array([rows]), _hip.int_array([cols])) > 0
        more = _hip.int_array([rows + (rows > cols)]), _hip.int_array([cols + (cols > rows)])
        assert lib.kfac_orthogonalize_workspace_bytes(1, *more) == 0


@pytest.mark.parametrize('shape', [(28672, 16), (16, 28672)])
def test_a_matrix_that_is_too_long_is_named(shape):
    small, large = torch.zeros(4, 4), torch.zeros(shape)
    with pytest.raises(_hip.KfacHipError, match='matrix 1 is %d x %d.*16384' % shape):
        torchsso.utils.orthogonalize([small, large])
    with pytest.raises(_hip.KfacHipError, match='parameter 1 is %d x %d.*16384' % shape):
        torchsso.optim.muon([small, large], [small, large], [small, large], lr=0.1)


@pytest.mark.parametrize('shape', [(28672, 16), (16, 28672), (4, 1024, 17)])
def test_the_optimizer_refuses_it_at_once(shape):
    params = [torch.nn.Parameter(torch.zeros(4, 4)), torch.nn.Parameter(torch.zeros(shape))]
    with pytest.raises(ValueError, match='16384.*%s' % shape[0]):
        torchsso.optim.Muon(params)
    torchsso.optim.Muon([torch.nn.Parameter(torch.zeros(4, 4096, 4))])
