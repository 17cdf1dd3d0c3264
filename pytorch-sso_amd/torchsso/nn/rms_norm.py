"""Root-mean-square norm, with the residual's addition in front of it, on the HIP engine.

    h = x + residual                       (kept in the type of x)
    y = h / sqrt(mean(h^2) + eps) * gain

The reference's networks normalise with BatchNorm and its curvature (curv/cov/batchnorm.py:10-49);
this is the norm of a decoder's blocks.  Its backward pass forms the diagonal curvature of the gain
in the same pass over memory as the gradients (curv/cov/rms_norm.py hands it to an optimizer).
"""
import torch
import torch.nn as nn

from torchsso import _ops


def _apply(x, residual, gain, eps, curvature, out_dtype):
    if not eps >= 0:
        raise ValueError('Invalid eps: {}'.format(eps))
    if curvature is not None and gain is None:
        raise ValueError('a curvature belongs to a gain')
    if out_dtype is None or out_dtype == x.dtype:
        return _ops.rms_norm_autograd(x, residual, gain, eps, curvature)
    if out_dtype != torch.float8_e4m3fn:
        raise ValueError('Invalid out_dtype: {}'.format(out_dtype))
    if curvature is not None:
        raise ValueError('a result in 8 bits has no backward pass and no curvature')
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, gain)):
        raise ValueError('a result in 8 bits has no backward pass: call it under torch.no_grad()')
    return _ops.rms_norm_autograd(x, residual, gain, eps, None, True)


def rms_norm(x, gain=None, eps=1e-6, curvature=None, out_dtype=None):
    """y = x / sqrt(mean(x^2) + eps) * gain over the last dimension, in the type of x (float32,
    bfloat16, float16); gain: of that type, float32, or None.

    curvature: a float32 tensor of the gain's shape, which the backward pass fills with the diagonal
    curvature over the samples x[0], x[1], ... (batch * sum of the squared per-sample gradients).
    out_dtype=torch.float8_e4m3fn: returns (q, scale) with y = q * scale, a scale per row, of the
    shape that torch._scaled_mm takes; without a backward pass."""
    return _apply(x, None, gain, eps, curvature, out_dtype)


def add_rms_norm(x, residual, gain=None, eps=1e-6, curvature=None, out_dtype=None):
    """(y, h) with h = x + residual, of one type, and y = rms_norm(h): h is the residual stream that
    goes on beside the layer which reads y.  In 8 bits: (q, scale, h)."""
    return _apply(x, residual, gain, eps, curvature, out_dtype)


class RMSNorm(nn.Module):
    """rms_norm with a gain `weight`; module(x, residual) is add_rms_norm.  A DiagCovRMSNorm
    curvature of the module takes what the backward pass leaves."""

    def __init__(self, dim, eps=1e-6, device=None, dtype=None):
        super(RMSNorm, self).__init__()
        self.dim = int(dim)
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(self.dim, device=device, dtype=dtype))
        self._curvature = None             # a DiagCovRMSNorm: receives what the backward passes form

    def forward(self, x, residual=None):
        curvature = None
        if self._curvature is not None and torch.is_grad_enabled():
            curvature = self._curvature.buffer(x.device)
        return _apply(x, residual, self.weight, self.eps, curvature, None)

    def extra_repr(self):
        return '{}, eps={}'.format(self.dim, self.eps)
