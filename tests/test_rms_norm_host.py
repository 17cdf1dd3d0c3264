"""Argument checks of the root-mean-square norm that need no device."""
import pytest
import torch

import torchsso
from torchsso import _hip


def test_argument_errors_are_codes():
    lib = _hip.load()
    p = 1 << 20

    def call(kind=0, is_float=0, rows=4, dim=8, x=p, ldx=8, res=None, ldr=0, eps=1e-6, y=p, h=None):
        return lib.kfac_rms_norm(kind, is_float, rows, dim, x, ldx, res, ldr, None, eps, y, h, None, None)
    assert call(kind=3) == 1 and call(kind=-1) == 1 and call(is_float=2) == 1
    assert call(rows=-1) == 1 and call(rows=1 << 31) == 1 and call(dim=0) == 1 and call(dim=(1 << 24) + 1) == 1
    assert call(x=None) == 1 and call(y=None) == 1 and call(ldx=-1) == 1 and call(res=p, ldr=8) == 1
    assert call(eps=-1.) == 1 and call(eps=float('nan')) == 1
    assert call(rows=0) == 0

    def back(rows=4, dim=8, samples=2, dy=p, dh=None, h=p, dx=p, dgain=p, curvature=None, ws=p, size=1 << 20):
        return lib.kfac_rms_norm_backward(0, 0, rows, dim, samples, dy, 8, dh, 8, h, 8, None, 1e-6, dx, dgain,
                                          curvature, ws, size, None)
    assert back(rows=5) == 1 and back(samples=0) == 1 and back(rows=0) == 1 and back(dy=None) == 1 and back(h=None) == 1
    assert back(dh=p, dx=None) == 1
    assert back(ws=None) == 2 and back(size=4) == 2
    need = lib.kfac_rms_norm_backward_workspace_bytes
    assert need(0, 4, 8, 2, 0) > 0 and need(0, 4, 8, 3, 0) == 0 and need(0, 0, 8, 1, 0) == 0
    # a whole sample's sum and its square are kept by the units where samples are shorter than their rows
    assert need(0, 1 << 20, 8, 1 << 20, 1) == 3 * need(0, 1 << 20, 8, 1 << 20, 0)


def test_refusals():
    x = torch.zeros(2, 8)
    with pytest.raises(_hip.KfacHipError):
        torchsso.nn.rms_norm(x)                        # (on the host)
    with pytest.raises(ValueError):
        torchsso.nn.rms_norm(x, eps=float('nan'))
    with pytest.raises(TypeError):
        torchsso.DiagCovRMSNorm(torch.nn.Linear(2, 2))


def test_optimizer_finds_the_curvature():
    for kind in (torchsso.nn.RMSNorm, torch.nn.RMSNorm):
        model = torch.nn.Sequential(torch.nn.Linear(4, 6), kind(6))
        opt = torchsso.optim.SecondOrderOptimizer(model, 'Cov', {'Linear': 'Kron', 'RMSNorm': 'Diag'}, {})
        curv = opt.param_groups[1]['curv']
        assert type(curv) is torchsso.DiagCovRMSNorm and curv.shape == ((6,),)
