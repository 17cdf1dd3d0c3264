"""Diagonal curvature of root-mean-square norm layers.

The reference has no such layer; as its other diagonal curvatures (curv/cov/linear.py:28-45) this is
the mean over the batch of the squared gradients of single samples, with the n^2 rescale of
curvature.py:154-158:
    curv = n * sum_n s_n^2,   s_n = sum over the positions of sample n of g * x / rms(x).
torchsso.nn.RMSNorm forms it in its backward pass; for torch.nn.RMSNorm a pass of its own does, over
the layer's input and output gradient.
"""
import torch
import torch.nn as nn

from torchsso import _ops
from torchsso.curv.curvature import DiagCurvature, _attach
from torchsso.nn.rms_norm import RMSNorm


class DiagCovRMSNorm(DiagCurvature):

    def __init__(self, module, *args, **kwargs):
        if not isinstance(module, (RMSNorm, nn.RMSNorm)):
            raise TypeError('expected an RMSNorm module, got %s' % type(module).__name__)
        if isinstance(module, nn.RMSNorm) and len(module.normalized_shape) != 1:
            raise ValueError('RMSNorm over one dimension expected, got %s' % (tuple(module.normalized_shape),))
        self._asked = []                # (tensor that a backward pass fills, its version before that)
        super(DiagCovRMSNorm, self).__init__(module, *args, **kwargs)
        if isinstance(module, RMSNorm):
            module._curvature = self

    _ASKED_MOST = 4

    def buffer(self, device):
        """A tensor that the backward pass of one forward pass fills."""
        t = torch.empty(self._module.dim, dtype=torch.float32, device=device)
        self._asked = self._asked[1 - self._ASKED_MOST:] + [(t, t._version)]
        return t

    @property
    def data(self):
        """Of the latest forward pass that has had its backward pass (which changes its tensor's version)."""
        for i in reversed(range(len(self._asked))):
            t, version = self._asked[i]
            if t._version != version:
                self._data = [t]
                self._asked = self._asked[i + 1:]
                break
        return self._data

    @data.setter
    def data(self, value):
        self._asked = []
        self._data = value

    def adjust_data_scale(self, scale):
        self.data                       # (takes what a backward pass has left)
        super(DiagCovRMSNorm, self).adjust_data_scale(scale)

    @property
    def shape(self):
        return self._get_shape()

    def forward_postprocess(self, module, input, output):
        assert self._module == module
        if isinstance(module, nn.RMSNorm):
            super(DiagCovRMSNorm, self).forward_postprocess(module, input, output)
            return
        _attach(module, 'data_input', input[0].detach())
        _attach(module, 'data_output', output[0] if isinstance(output, tuple) else output)

    def update_in_backward(self, grad_output):
        module, x = self._module, self._module.data_input
        eps = torch.finfo(x.dtype).eps if module.eps is None else module.eps
        curvature = torch.empty(x.shape[-1], dtype=torch.float32, device=x.device)
        _ops.rms_norm_backward(grad_output, None, x, None, eps, x.shape[0] if x.dim() > 1 else 1,
                               want_dx=False, want_dgain=False, curvature=curvature)
        self._data = [curvature]
