"""AdamW over lists of tensors, with states in 32 or in 8 bits.

The reference has no such optimizer; it updates what it has preconditioned (optim/secondorder.py:225-312).
This one is for the parameters of a decoder that neither a curvature nor Muon takes: embeddings, gains and
biases, or all of a model.  Update number t of a parameter p with gradient g:

    m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
    p = (1 - lr weight_decay) p - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

States in 8 bits are kept by blocks of 128 elements with a float32 scale each: m / scale in float8_e4m3fn with
scale = max |m| / 448 of the block, v / scale in float8_e5m2 with scale = max v / 57344, both rounded at random
to one of the two neighbours, so that they keep on average what single updates add.  The random numbers
depend on the seed, the number of the update, the place in the list and that in the tensor: the same call
gives the same bits.
"""
import torch
from torch.optim import Optimizer

from torchsso import _ops

LEAST_EPS_8 = 1e-12          # of updates with states in 8 bits, where small enough a v is 0
_INF = float('inf')


def _check(lr, betas, eps, weight_decay, eight=False):
    if not isinstance(lr, torch.Tensor) and not 0 <= lr < _INF:
        raise ValueError('Invalid learning rate: {}'.format(lr))
    for i, beta in enumerate(betas):
        if not 0 <= beta < 1:
            raise ValueError('Invalid beta parameter at index {}: {}'.format(i, beta))
    if not (LEAST_EPS_8 if eight else 0) <= eps < _INF:
        raise ValueError('Invalid epsilon value: {}{}'.format(
            eps, ' (with states in 8 bits at least {})'.format(LEAST_EPS_8) if eight else ''))
    if not 0 <= weight_decay < _INF:
        raise ValueError('Invalid weight_decay value: {}'.format(weight_decay))


def adamw_states(param, bits=32):
    """(exp_avg, exp_avg_sq) of a parameter before its first update: zeros, in float32, or with bits=8 pairs (numbers
    in 8 bits, scales of the blocks).  They lie in memory as the parameter does."""
    if bits == 32:
        return tuple(torch.zeros_like(param, dtype=torch.float32, requires_grad=False) for _ in range(2))
    if bits != 8:
        raise ValueError('Invalid number of bits: {}'.format(bits))
    blocks = -(-param.numel() // _ops.STATE_BLOCK)
    return tuple((torch.zeros_like(param, dtype=dtype, requires_grad=False),
                  torch.zeros(blocks, dtype=torch.float32, device=param.device))
                 for dtype in (torch.float8_e4m3fn, torch.float8_e5m2))


def adamw(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, seed=0):
    """One update of a list of parameters and their states, in place, in few launches.

    params, grads: tensors of one type, float32, bfloat16 or float16, on one device, each once; a parameter's elements lie
    side by side in any order of the dimensions.  exp_avgs, exp_avg_sqs: their states as adamw_states makes them, all of
    one kind.
    step: the number of this update, from 1 on; or a list of one for each tensor; or a list of int32 tensors of one
    element, the updates so far, on the device, which the update raises by one: a recorded call then counts on
    at every replay.  lr: a number, or with such a list a float32 tensor of one element on the device.
    A parameter in bfloat16 or float16 is rounded to its nearest number: what an update adds has to reach half a
    step of that type, or it is lost (gains of size 1 in bfloat16 move by 2^-9 or not at all)."""
    beta1, beta2 = betas
    if not isinstance(step, (int, list, tuple)):
        step = int(step)
    if not ((isinstance(lr, torch.Tensor) or 0 <= lr < _INF) and 0 <= beta1 < 1 and 0 <= beta2 < 1 and 0 <= eps < _INF
            and 0 <= weight_decay < _INF and len(params) > 0
            and _ops.adamw(params, grads, exp_avgs, exp_avg_sqs, step, lr, beta1, beta2, eps, weight_decay, seed)):
        _refuse(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay)


def _refuse(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay):
    """Raises what is wrong with the arguments of an update (nothing, if there is nothing to update)."""
    lengths = tuple(len(t) for t in (params, grads, exp_avgs, exp_avg_sqs))
    if len(set(lengths)) != 1:
        raise ValueError('%d parameters, %d gradients, %d first and %d second moments' % lengths)
    pairs = [isinstance(t, (tuple, list)) for t in list(exp_avgs) + list(exp_avg_sqs)]
    eight = len(pairs) > 0 and all(pairs)
    if any(pairs) and not eight:
        raise ValueError('states in 32 bits and in 8 in one list')
    _check(lr, betas, eps, weight_decay, eight)
    if any(isinstance(g, torch.Tensor) and g.is_sparse for g in grads):
        raise RuntimeError('AdamW does not take sparse gradients')
    steps = step if isinstance(step, (tuple, list)) else [step] * len(params)
    if len(steps) != len(params):
        raise ValueError('%d parameters, %d steps' % (len(params), len(steps)))
    if len(set(isinstance(t, torch.Tensor) for t in steps)) > 1:
        raise ValueError('steps on the device and numbers in one list')
    if any(not isinstance(t, torch.Tensor) and t < 1 for t in steps):
        raise ValueError('Invalid step: {}'.format(step))
    if len(params) == 0:
        return
    scales = [None, None]
    if eight:
        if any(len(t) != 2 for t in list(exp_avgs) + list(exp_avg_sqs)):
            raise ValueError('a state in 8 bits is (numbers, scales)')
        (exp_avgs, scales[0]), (exp_avg_sqs, scales[1]) = (zip(*states) for states in (exp_avgs, exp_avg_sqs))
    _ops.check_adamw(params, grads, exp_avgs, exp_avg_sqs, *scales, step, lr)


class AdamW(Optimizer):
    r"""Optimizer for parameters of any shape in float32, bfloat16 or float16 (see `adamw`).

    Args:
        params: parameters, or param groups
        lr, betas, eps, weight_decay
        state_bits: 32, or 8 for parameters of `min_8bit_size` elements or more (gains and biases keep 32)
        capturable: count updates on the device, so that `step` can be recorded into a graph and replayed; lr may be
            a float32 tensor of one element on the device then
        seed: of the random numbers that 8-bit states are rounded by
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, min_8bit_size=4096,
                 capturable=False, seed=0):
        defaults = {'lr': lr, 'betas': betas, 'eps': eps, 'weight_decay': weight_decay, 'state_bits': state_bits,
                    'min_8bit_size': min_8bit_size, 'capturable': capturable, 'seed': seed}
        self._check_options(defaults)
        if state_bits == 8:
            _check(lr, betas, eps, weight_decay, True)
        super(AdamW, self).__init__(params, defaults)

    @staticmethod
    def _check_options(group):
        if isinstance(group['lr'], torch.Tensor) and not group['capturable']:
            raise ValueError('a learning rate on the device needs capturable=True')
        if group['state_bits'] not in (8, 32):
            raise ValueError('Invalid number of bits: {}'.format(group['state_bits']))
        # (eps for 8 bits: of a group whose tensors may all be too small for those an update says more)
        _check(group['lr'], group['betas'], group['eps'], group['weight_decay'])

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            self._check_options(dict(self.defaults, **param_group))
        super(AdamW, self).add_param_group(param_group)

    _KEPT = {'exp_avg': (torch.float32, torch.float8_e4m3fn), 'exp_avg_sq': (torch.float32, torch.float8_e5m2),
             'exp_avg_scale': (torch.float32,), 'exp_avg_sq_scale': (torch.float32,)}

    def load_state_dict(self, state_dict):
        """What state_dict of this class has saved, or of torch.optim.AdamW (states that are neither float32 nor 8 bits
        become float32).  States in 8 bits, whose blocks are those of a memory order, have to be in their parameter's."""
        for group in state_dict['param_groups']:
            for name in ('amsgrad', 'maximize'):
                if group.get(name):
                    raise ValueError('AdamW has no option {}'.format(name))
        # (what the base class numbers as it does here)
        own = [p for group in self.param_groups for p in group['params']]
        for p, i in zip(own, (i for group in state_dict['param_groups'] for i in group['params'])):
            saved = state_dict['state'].get(i) or {}
            for name in ('exp_avg', 'exp_avg_sq'):
                if name in saved and saved[name].numel() != p.numel():
                    raise ValueError('a state of shape {} is not that of a parameter of shape {}'.format(
                        tuple(saved[name].shape), tuple(p.shape)))
                if name + '_scale' in saved and _ops._strides(saved[name]) != _ops._strides(p):
                    raise ValueError('a state in 8 bits with strides {} does not lie in memory as its parameter, {}'.format(
                        saved[name].stride(), p.stride()))
        super(AdamW, self).load_state_dict(state_dict)
        for group in self.param_groups:
            for name, value in self.defaults.items():
                group.setdefault(name, value)
        # (the base class gives states their parameter's type; these keep their own, and a parameter's order in memory)
        ids = [i for group in state_dict['param_groups'] for i in group['params']]
        params = [(p, group) for group in self.param_groups for p in group['params']]
        for i, (p, group) in zip(ids, params):
            saved = state_dict['state'].get(i)
            if not saved:
                continue
            state = self.state[p]
            for name, types in self._KEPT.items():
                if name in saved:
                    t = saved[name].detach()
                    dtype = t.dtype if t.dtype in types else torch.float32
                    like = torch.empty(t.shape, dtype=dtype, device=p.device) if name.endswith('scale') \
                        else torch.empty_like(p, dtype=dtype, requires_grad=False)
                    state[name] = like.copy_(t)
            step = int(saved['step'])
            state['step'] = torch.full((), step, dtype=torch.int32, device=p.device) if group['capturable'] else step

    def _first_state(self, p, group, capturing):
        if capturing:
            raise RuntimeError('AdamW: a step has to be taken before one is recorded (it makes the states)')
        state = {'step': torch.zeros((), dtype=torch.int32, device=p.device) if group['capturable'] else 0}
        bits = 32 if group['state_bits'] == 8 and p.numel() < group['min_8bit_size'] else group['state_bits']
        m, v = adamw_states(p, bits)
        if bits == 8:
            (state['exp_avg'], state['exp_avg_scale']), (state['exp_avg_sq'], state['exp_avg_sq_scale']) = m, v
        else:
            state['exp_avg'], state['exp_avg_sq'] = m, v
        # (kept once it is whole: a step that runs out of memory here can be taken again)
        self.state[p] = state
        return state

    def step(self, closure=None):
        """One optimization step.  `closure` runs forward and backward and returns the loss or
        (loss, output); its return value is passed through."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        kept, lists = self.state, 0
        for group in self.param_groups:
            capturable = group['capturable']
            if capturing and not capturable:
                raise RuntimeError('AdamW: capturable=True is needed to record a step')
            alike, last = {}, None
            for p in group['params']:
                g = p.grad
                if g is None:
                    continue
                state = kept.get(p) or self._first_state(p, group, capturing)
                scale = state.get('exp_avg_scale')
                key = (p.dtype, p.get_device(), scale is None)
                if key != last:
                    last = key
                    ps, gs, ms, vs, states = alike.setdefault(key, ([], [], [], [], []))
                ps.append(p)
                gs.append(g)
                ms.append(state['exp_avg'] if scale is None else (state['exp_avg'], scale))
                vs.append(state['exp_avg_sq'] if scale is None else (state['exp_avg_sq'], state['exp_avg_sq_scale']))
                states.append(state)
            for ps, gs, ms, vs, states in alike.values():
                steps = [state['step'] for state in states]
                if not capturable:
                    steps = [step + 1 for step in steps]
                adamw(ps, gs, ms, vs, steps, lr=group['lr'], betas=group['betas'], eps=group['eps'],
                      weight_decay=group['weight_decay'], seed=group['seed'] + lists)
                lists += 1
                if not capturable:
                    for state, step in zip(states, steps):
                        state['step'] = step
        return loss
