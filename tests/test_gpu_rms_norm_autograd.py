"""What autograd asks of torchsso.nn.rms_norm beside its gradients."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import torchsso
from torchsso import _hip

pytestmark = pytest.mark.gpu

EIGHT = torch.float8_e4m3fn


@pytest.mark.parametrize('requires_grad', [False, True])
@pytest.mark.parametrize('which', [0, 1, 2])
def test_forward_mode_is_refused(which, requires_grad):
    """(There is no such derivative; a result without a tangent would stand for one of zero.)"""
    x, residual, gain = torch.randn(4, 50, device='cuda'), torch.randn(4, 50, device='cuda'), torch.ones(50, device='cuda')
    with forward_ad.dual_level():
        args = [x, residual, gain]
        args[which] = forward_ad.make_dual(args[which].requires_grad_(requires_grad), torch.ones_like(args[which]))
        with pytest.raises(RuntimeError):
            torchsso.nn.add_rms_norm(*args)
        if which != 1:
            with pytest.raises(RuntimeError):
                torchsso.nn.rms_norm(args[0], args[2])
        if not requires_grad:
            with pytest.raises(RuntimeError):
                torchsso.nn.add_rms_norm(*args, out_dtype=EIGHT)
        # without a tangent, inside such a level, it works
        y = torchsso.nn.rms_norm(torch.ones(4, 50, device='cuda'))
        assert forward_ad.unpack_dual(y).tangent is None


@pytest.mark.parametrize('requires_grad', [False, True])
def test_running_out_of_memory_is_raised_as_torch_does(requires_grad):
    x = torch.ones(1, 1 << 17, device='cuda', dtype=torch.bfloat16, requires_grad=requires_grad)
    # (16 GiB asked of an allocator that may hand out 2 % of the memory: nothing is allocated)
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.02)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            torchsso.nn.rms_norm(x.expand(1 << 16, 1 << 17))
    finally:
        torch.cuda.set_per_process_memory_fraction(1.)
    assert torchsso.nn.rms_norm(x).shape == x.shape


@pytest.mark.parametrize('how', ['gradient', 'none', 'eight bits'])
def test_other_threads_run_during_a_norm(how):
    """The interpreter is released around the engine's entry point: in its place stands a function that returns
    whether this thread holds the interpreter, which the norm takes for a status (0: success)."""
    lib = _hip.load()
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value
    entries = [address(f) for f in (lib.kfac_rms_norm, lib.kfac_rms_norm_backward_workspace_bytes, lib.kfac_rms_norm_backward)]
    x = torch.ones(4, 50, device='cuda', requires_grad=how == 'gradient')
    more = dict(out_dtype=EIGHT) if how == 'eight bits' else {}
    torchsso.nn.rms_norm(x, **more)
    _hip._host.bind_norm(address(ctypes.pythonapi.PyGILState_Check), *entries[1:])
    try:
        torchsso.nn.rms_norm(x, **more)
    finally:
        _hip._host.bind_norm(*entries)
    assert torch.equal(torchsso.nn.rms_norm(torch.ones(4, 50, device='cuda')), torchsso.nn.rms_norm(x.detach()))
