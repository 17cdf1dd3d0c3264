"""Diagonal curvature of layers that normalise rows: what the curvatures of the single kinds have in common.

The reference has no such layers; as its other diagonal curvatures (curv/cov/linear.py:28-45) this is the mean over
the batch of the squared gradients of single samples, with the n^2 rescale of curvature.py:154-158.  Modules of
torchsso.nn form it in their backward pass; for those of torch.nn a pass of its own does, over the layer's input and
output gradient.
"""
import torch

from torchsso.curv.curvature import DiagCurvature, _attach


class DiagCovRowNorm(DiagCurvature):

    own, torchs = None, None        # the module classes of torchsso.nn and torch.nn

    def __init__(self, module, *args, **kwargs):
        name = self.own.__name__
        if not isinstance(module, (self.own, self.torchs)):
            raise TypeError('expected %s %s module, got %s' % ('an' if name[0] == 'R' else 'a', name, type(module).__name__))
        if isinstance(module, self.torchs) and len(module.normalized_shape) != 1:
            raise ValueError('%s over one dimension expected, got %s' % (name, tuple(module.normalized_shape),))
        self._asked = []                # (tensor that a backward pass fills, its version before that)
        super(DiagCovRowNorm, self).__init__(module, *args, **kwargs)
        if isinstance(module, self.own):
            module._curvature = self

    _ASKED_MOST = 4

    def buffer(self, device):
        """A tensor that the backward pass of one forward pass fills."""
        t = torch.empty(self._buffer_shape(), dtype=torch.float32, device=device)
        self._asked = self._asked[1 - self._ASKED_MOST:] + [(t, t._version)]
        return t

    def _buffer_shape(self):
        return (self._module.dim,)

    def _of_parameters(self, t):
        """The parts of such a tensor that belong to the module's parameters."""
        return [t]

    @property
    def data(self):
        """Of the latest forward pass that has had its backward pass (which changes its tensor's version)."""
        for i in reversed(range(len(self._asked))):
            t, version = self._asked[i]
            if t._version != version:
                self._data = self._of_parameters(t)
                self._asked = self._asked[i + 1:]
                break
        return self._data

    @data.setter
    def data(self, value):
        self._asked = []
        self._data = value

    def adjust_data_scale(self, scale):
        self.data                       # (takes what a backward pass has left)
        super(DiagCovRowNorm, self).adjust_data_scale(scale)

    @property
    def shape(self):
        return self._get_shape()

    def forward_postprocess(self, module, input, output):
        assert self._module == module
        if isinstance(module, self.torchs):
            super(DiagCovRowNorm, self).forward_postprocess(module, input, output)
            return
        _attach(module, 'data_input', input[0].detach())
        _attach(module, 'data_output', output[0] if isinstance(output, tuple) else output)
