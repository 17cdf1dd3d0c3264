"""Argument checks of the layer norm that need no device."""
import contextlib

import pytest
import torch

import torchsso
from torchsso import _hip, _ops


def test_argument_errors_are_codes():
    lib = _hip.load()
    p = 1 << 20

    def call(kind=0, is_float=0, rows=4, dim=8, x=p, ldx=8, res=None, ldr=0, gain=None, bias=None, eps=1e-6, y=p, h=None,
             scale=None, stats=None):
        return lib.kfac_layer_norm(kind, is_float, rows, dim, x, ldx, res, ldr, gain, bias, eps, y, h, scale, stats, None)
    assert call(kind=3) == 1 and call(kind=-1) == 1 and call(is_float=2) == 1
    assert call(rows=-1) == 1 and call(rows=1 << 31) == 1 and call(dim=0) == 1 and call(dim=(1 << 24) + 1) == 1
    assert call(x=None) == 1 and call(y=None) == 1 and call(ldx=-1) == 1 and call(res=p, ldr=8) == 1
    assert call(eps=-1.) == 1 and call(eps=float('nan')) == 1 and call(bias=p) == 1
    assert call(y=None, stats=p, scale=p) == 1
    assert call(rows=0) == 0

    def back(rows=4, dim=8, samples=2, vectors=2, dy=p, dh=None, h=p, stats=p, dx=p, dgain=p, dbias=p, curvature=None, ws=p,
             size=1 << 20):
        return lib.kfac_layer_norm_backward(0, 0, rows, dim, samples, vectors, dy, 8, dh, 8, h, 8, stats, None, dx, dgain,
                                            dbias, curvature, ws, size, None)
    assert back(rows=5) == 1 and back(samples=0) == 1 and back(rows=0) == 1 and back(dy=None) == 1 and back(h=None) == 1
    assert back(dh=p, dx=None) == 1 and back(stats=None) == 1 and back(vectors=1) == 1 and back(vectors=3) == 1
    assert back(ws=None) == 2 and back(size=4) == 2
    need = lib.kfac_layer_norm_backward_workspace_bytes
    assert need(0, 4, 8, 2, 1, 0) > 0 and need(0, 4, 8, 3, 1, 0) == 0 and need(0, 0, 8, 1, 1, 0) == 0
    assert need(0, 4, 8, 2, 0, 0) == 0 and need(0, 4, 8, 2, 3, 0) == 0
    assert need(0, 999, 8, 3, 2, 0) == 2 * need(0, 999, 8, 3, 1, 0)
    # units of whole samples leave their samples' sums and squares
    assert need(0, 1 << 20, 8, 1 << 20, 2, 1) == 2 * need(0, 1 << 20, 8, 1 << 20, 2, 0)


def test_refusals():
    x, w = torch.zeros(2, 8), torch.zeros(8)
    with pytest.raises(_hip.KfacHipError):
        torchsso.nn.layer_norm(x)                        # (on the host)
    with pytest.raises(_hip.KfacHipError):
        torchsso.nn.add_layer_norm(x, x, w, w)
    for bad in (lambda: torchsso.nn.layer_norm(x, eps=float('nan')), lambda: torchsso.nn.layer_norm(x, eps=-1e-6),
                lambda: torchsso.nn.layer_norm(x, None, w), lambda: torchsso.nn.layer_norm(x, curvature=w),
                lambda: torchsso.nn.layer_norm(x, w, out_dtype=torch.float64),
                lambda: torchsso.nn.layer_norm(x, w, curvature=w, out_dtype=torch.float8_e4m3fn),
                lambda: torchsso.nn.layer_norm(x, w.clone().requires_grad_(), out_dtype=torch.float8_e4m3fn),
                lambda: torchsso.DiagCovLayerNorm(torch.nn.LayerNorm((5, 6))),
                lambda: torchsso.DiagCovLayerNorm(torch.nn.LayerNorm(5, elementwise_affine=False))):
        with pytest.raises(ValueError):
            bad()
    for module in (torch.nn.Linear(2, 2), torchsso.nn.RMSNorm(3)):
        with pytest.raises(TypeError):
            torchsso.DiagCovLayerNorm(module)
    with pytest.raises(TypeError):
        torchsso.DiagCovRMSNorm(torchsso.nn.LayerNorm(3))


@pytest.mark.parametrize('length', [(1 << 24) + 1, (1 << 32) + 8])
def test_long_rows_are_refused(length):
    x = torch.ones(1, 1, dtype=torch.bfloat16).expand(1, length)
    for call in (lambda: torchsso.nn.layer_norm(x), lambda: torchsso.nn.add_layer_norm(x, x),
                 lambda: _ops.layer_norm_stats(x, 1e-5),
                 lambda: _ops.layer_norm_backward(x, None, x, torch.zeros(1, 3), None, 1)):
        with pytest.raises(_hip.KfacHipError, match='1 to 16777216 elements'):
            call()


@pytest.mark.parametrize('bias', [True, False])
def test_optimizer_finds_the_curvature(bias):
    for kind in (torchsso.nn.LayerNorm, torch.nn.LayerNorm):
        model = torch.nn.Sequential(torch.nn.Linear(4, 6), kind(6, bias=bias))
        opt = torchsso.optim.SecondOrderOptimizer(model, 'Cov', {'Linear': 'Kron', 'LayerNorm': 'Diag'}, {})
        curv = opt.param_groups[1]['curv']
        assert type(curv) is torchsso.DiagCovLayerNorm and curv.shape == ((6,),) * (2 if bias else 1)
        assert len(opt.param_groups[1]['params']) == len(curv.shape)


def test_module():
    m = torchsso.nn.LayerNorm(6)
    assert sorted(m.state_dict()) == ['bias', 'weight'] and torch.equal(m.weight, torch.ones(6))
    assert sorted(torchsso.nn.LayerNorm(6, bias=False).state_dict()) == ['weight']
    other = torch.nn.LayerNorm(6)
    m.load_state_dict(other.state_dict())
    assert 'eps=1e-05' in repr(m)


def test_launches_go_to_the_device_of_the_tensors(monkeypatch):
    """Device 0 is current; the tensors are on device 1."""
    current, seen = [0], []

    class Tensor(object):
        device, dtype, is_cuda = torch.device('cuda', 1), torch.float32, True

        def __init__(self, *shape):
            self.shape = torch.Size(shape)

        def dim(self):
            return len(self.shape)

        def data_ptr(self):
            return 1 << 20

        def reshape(self, *shape):
            return self

        def stride(self, i):
            return 1 if i == 1 else self.shape[-1]

    class Lib(object):

        def __getattr__(self, name):
            def call(*args):
                seen.append((name, current[-1]))
                return 64 if name.endswith('workspace_bytes') else 0
            return call

    @contextlib.contextmanager
    def use(device):
        current.append(device.index)
        yield
        current.pop()
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: current[-1])
    monkeypatch.setattr(torch.cuda, 'device', use)
    monkeypatch.setattr(_hip, 'load', lambda: Lib())
    monkeypatch.setattr(_hip, 'typed_ptr', lambda t, *args: t.data_ptr())
    monkeypatch.setattr(_hip, 'stream_ptr', lambda device=None, stream=None: 0)
    monkeypatch.setattr(_hip, 'workspace', lambda device, nbytes, stream=None: (None, nbytes))
    monkeypatch.setattr(torch, 'empty', lambda shape, dtype=None, device=None: Tensor(*shape))
    monkeypatch.setattr(torch, 'empty_like', lambda t: Tensor(*t.shape))
    _ops.layer_norm_stats(Tensor(4, 5), 1e-5)
    _ops.layer_norm_backward(Tensor(4, 5), None, Tensor(4, 5), Tensor(4, 3), Tensor(5), 2)
    launches = [(n, d) for n, d in seen if not n.endswith('bytes')]
    assert launches == [('kfac_layer_norm', 1), ('kfac_layer_norm_backward', 1)]
