"""Diagonal curvature of layer norm layers:

    curv = n * sum_n s_n^2,   s_n = sum over the positions of sample n of g * (x - mean(x)) / std(x)   (gain)
                              s_n = sum over the positions of sample n of g                            (bias)

The reference has no such layer; scaled as its other diagonal curvatures are (curv/cov/linear.py:28-45,
curvature.py:154-158).
"""
import torch
import torch.nn as nn

from torchsso import _ops
from torchsso.curv.cov.row_norm import DiagCovRowNorm
from torchsso.nn.layer_norm import LayerNorm


class DiagCovLayerNorm(DiagCovRowNorm):

    own, torchs = LayerNorm, nn.LayerNorm

    def __init__(self, module, *args, **kwargs):
        if isinstance(module, self.torchs) and module.weight is None:
            raise ValueError('a LayerNorm without parameters has no curvature')
        super(DiagCovLayerNorm, self).__init__(module, *args, **kwargs)

    def _buffer_shape(self):
        dim = self._module.weight.shape[0]
        return (2, dim) if self.bias else (dim,)

    def _of_parameters(self, t):
        return [t] if t.dim() == 1 else list(t.unbind(0))

    def update_in_backward(self, grad_output):
        module, x = self._module, self._module.data_input
        curvature = torch.empty(self._buffer_shape(), dtype=torch.float32, device=x.device)
        _ops.layer_norm_backward(grad_output, None, x, _ops.layer_norm_stats(x, module.eps), None,
                                 x.shape[0] if x.dim() > 1 else 1, want_dx=False, curvature=curvature)
        self._data = self._of_parameters(curvature)
