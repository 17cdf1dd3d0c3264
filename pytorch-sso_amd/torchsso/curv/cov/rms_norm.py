"""Diagonal curvature of root-mean-square norm layers:

    curv = n * sum_n s_n^2,   s_n = sum over the positions of sample n of g * x / rms(x).

The reference has no such layer; scaled as its other diagonal curvatures are (curv/cov/linear.py:28-45,
curvature.py:154-158).
"""
import torch
import torch.nn as nn

from torchsso import _ops
from torchsso.curv.cov.row_norm import DiagCovRowNorm
from torchsso.nn.rms_norm import RMSNorm


class DiagCovRMSNorm(DiagCovRowNorm):

    own, torchs = RMSNorm, nn.RMSNorm

    def update_in_backward(self, grad_output):
        module, x = self._module, self._module.data_input
        eps = torch.finfo(x.dtype).eps if module.eps is None else module.eps
        curvature = torch.empty(x.shape[-1], dtype=torch.float32, device=x.device)
        _ops.rms_norm_backward(grad_output, None, x, None, eps, x.shape[0] if x.dim() > 1 else 1,
                               want_dx=False, want_dgain=False, curvature=curvature)
        self._data = [curvature]
