"""Muon: momentum whose direction is orthogonalised before it is applied.

The reference has no such optimizer; it preconditions a layer's gradient with the inverses of the
layer's Kronecker factors (optim/secondorder.py:195-231).  Where those are too large to form and
invert, as for the projections of a decoder, an update with all singular values alike is what can
be had without them: no curvature state, one buffer per weight.

    buf = momentum * buf + g
    u   = g + momentum * buf     (nesterov)   or   buf
    p   = (1 - lr * weight_decay) * p - lr * sqrt(max(1, rows / columns)) * orthogonalize(u)
"""
import math

import torch
from torch.optim import Optimizer

from torchsso import _ops
from torchsso.utils.linalg import NEWTON_SCHULZ, check_orthogonalize_eps, newton_schulz_schedule


def _check(lr, momentum, weight_decay, eps):
    if not lr >= 0:
        raise ValueError('Invalid learning rate: {}'.format(lr))
    if not 0 <= momentum < 1:
        raise ValueError('Invalid momentum: {}'.format(momentum))
    if not weight_decay >= 0:
        raise ValueError('Invalid weight_decay value: {}'.format(weight_decay))
    check_orthogonalize_eps(eps)


def _matrix(t):
    """[rows, columns] view: the filters of a convolution are its rows."""
    return t if t.dim() == 2 else t.view(t.shape[0], -1)


@torch.no_grad()
def muon(params, grads, buffers, lr, momentum=0.95, nesterov=True, weight_decay=0., steps=5,
         coefficients=NEWTON_SCHULZ, eps=1e-7):
    """One update of a list of parameters, in place, with all matrices in the same launches.

    params, grads: tensors of two dimensions or more (of more, all but the first are columns), with
    at most 16384 rows and columns, of one type, float32, bfloat16 or float16, the parameters contiguous; buffers: contiguous float32
    tensors of the same shapes, zero before the first update."""
    _check(lr, momentum, weight_decay, eps)
    schedule = newton_schulz_schedule(steps, coefficients)
    if not len(params) == len(grads) == len(buffers):
        raise ValueError('%d parameters, %d gradients, %d buffers'
                         % (len(params), len(grads), len(buffers)))
    ps, gs, bs, sizes, keeps, written = [], [], [], [], [], []
    for p, g, b in zip(params, grads, buffers):
        if p.dim() < 2:
            raise ValueError('Muon updates matrices, got a parameter of shape {}'.format(tuple(p.shape)))
        if g.is_sparse:
            raise RuntimeError('Muon does not take sparse gradients')
        if p.numel() == 0:
            continue
        if not p.is_contiguous() or not b.is_contiguous():
            raise ValueError('parameters and momentum buffers have to be contiguous')
        written.extend((p, b))
        p = _matrix(p)
        ps.append(p)
        gs.append(_matrix(g.contiguous()))
        bs.append(_matrix(b))
        sizes.append(lr * math.sqrt(max(1., p.shape[0] / p.shape[1])))
        keeps.append(1. - lr * weight_decay)
    _ops.muon_update_batched(ps, gs, bs, sizes, keeps, momentum, nesterov, schedule, eps)
    # (a graph from before the update that goes through these weights is refused by its backward pass)
    torch.autograd.graph.increment_version(written)


class Muon(Optimizer):
    r"""Optimizer for the matrices of a model (see `muon`): the weights of Linear and Conv2d layers,
    in float32, bfloat16 or float16, with at most 16384 rows and columns.  Gains, biases and embeddings take another optimizer.

    Args:
        params: parameters of two dimensions or more, or param groups
        lr, momentum, nesterov, weight_decay
        steps, coefficients, eps: of the orthogonalisation (torchsso.utils.orthogonalize)
    """

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0., steps=5,
                 coefficients=NEWTON_SCHULZ, eps=1e-7):
        _check(lr, momentum, weight_decay, eps)
        newton_schulz_schedule(steps, coefficients)
        super(Muon, self).__init__(params, {
            'lr': lr, 'momentum': momentum, 'nesterov': nesterov, 'weight_decay': weight_decay,
            'steps': steps, 'coefficients': coefficients, 'eps': eps})
        for group in self.param_groups:
            for p in group['params']:
                if p.dim() < 2:
                    raise ValueError('Muon updates matrices, got a parameter of shape {}'
                                     .format(tuple(p.shape)))
                if max(p.shape[0], math.prod(p.shape[1:])) > _ops.ORTH_MAX_SIDE:
                    raise ValueError('Muon updates matrices with sides of up to {}, got a parameter of shape {}'
                                     .format(_ops.ORTH_MAX_SIDE, tuple(p.shape)))

    def load_state_dict(self, state_dict):
        super(Muon, self).load_state_dict(state_dict)
        # (the base class gives the buffers their parameter's type; they are float32)
        ids = [i for group in state_dict['param_groups'] for i in group['params']]
        params = [p for group in self.param_groups for p in group['params']]
        for i, p in zip(ids, params):
            saved = state_dict['state'].get(i, {}).get('momentum_buffer')
            if saved is not None:
                self.state[p]['momentum_buffer'] = saved.detach().to(device=p.device, dtype=torch.float32,
                                                                     copy=True)

    def step(self, closure=None):
        """One optimization step.  `closure` runs forward and backward and returns the loss or
        (loss, output); its return value is passed through."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_type = {}
            for p in group['params']:
                if p.grad is None:
                    continue
                state = self.state[p]
                if 'momentum_buffer' not in state:
                    state['momentum_buffer'] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                ps, gs, bs = by_type.setdefault((p.dtype, p.device), ([], [], []))
                ps.append(p)
                gs.append(p.grad)
                bs.append(state['momentum_buffer'])
            options = {k: group[k] for k in ('lr', 'momentum', 'nesterov', 'weight_decay', 'steps',
                                             'coefficients', 'eps')}
            for ps, gs, bs in by_type.values():
                muon(ps, gs, bs, **options)
        return loss
