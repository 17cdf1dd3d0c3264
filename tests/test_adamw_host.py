"""AdamW: what needs no device.  Refusals, the numbers that 8-bit states are rounded by, and what the class keeps."""
import ctypes

import pytest
import torch

import torchsso
from torchsso import _hip, _ops

from adamw_testlib import LARGEST, encode, mix, numbers, words


def test_argument_errors_are_codes():
    lib = _hip.load()
    p = 1 << 20

    def call(count=1, numel=100, kind=0, bits=32, params=p, grads=p, m=p, v=p, scales=None, steps=1, counters=None, lr=1e-3,
             on_device=None, b1=.9, b2=.999, eps=1e-8, decay=0., ws=None, size=0):
        def one(x):
            return None if x == 'none' else (ctypes.c_void_p * 1)(x)
        return lib.kfac_adamw_batched(
            count, (ctypes.c_int64 * 1)(numel), kind, bits, one(params), one(grads), one(m), one(v),
            None if scales is None else one(scales), None if scales is None else one(scales),
            None if steps is None else (ctypes.c_int64 * 1)(steps), None if counters is None else one(counters), lr, on_device,
            b1, b2, eps, decay, 0, ws, size, None)
    assert call(count=0) == 0 and call(numel=0) == 0 and call(numel=0, params=None) == 0
    assert call(count=-1) == 1 and call(numel=-1) == 1 and call(numel=1 << 50) == 1
    assert call(kind=3) == 1 and call(kind=-1) == 1 and call(bits=16) == 1 and call(bits=8) == 1
    for name in ('params', 'grads', 'm', 'v'):
        assert call(**{name: None}) == 1 and call(**{name: 'none'}) == 1
    assert call(bits=8, scales=None) == 1 and call(bits=8, scales=p, m=None) == 1
    assert call(steps=0) == 1 and call(steps=None) == 1 and call(steps=1, counters=p) == 1
    assert call(on_device=p) == 1
    assert call(steps=None, counters=p) == 2 and call(steps=None, counters=p, ws=p, size=4) == 2
    nan = float('nan')
    for bad in (dict(lr=-1.), dict(lr=nan), dict(b1=1.), dict(b1=-.1), dict(b2=nan), dict(eps=-1.), dict(eps=nan), dict(decay=-1.)):
        assert call(**bad) == 1
    assert call(bits=8, scales=p, eps=1e-13) == 1 and call(bits=8, scales=p, eps=0.) == 1
    assert lib.kfac_adamw_workspace_bytes(3, 0) == 0 and lib.kfac_adamw_workspace_bytes(3, 1) > 0


def test_refusals():
    p = torch.zeros(4, 5)
    adamw, states = torchsso.optim.adamw, torchsso.optim.adamw_states
    m, v = states(p)
    nan = float('nan')
    for more in (dict(lr=-1.), dict(lr=nan), dict(lr=float('inf')), dict(betas=(1., .9)), dict(betas=(.9, -.1)), dict(betas=(nan, .9)),
                 dict(eps=-1.), dict(eps=nan), dict(weight_decay=-1.), dict(weight_decay=nan), dict(step=0), dict(step=[0]),
                 dict(step=[1, 2]), dict(step=-3)):
        with pytest.raises(ValueError):
            adamw([p], [p], [m], [v], **dict(dict(step=1), **more))
    for lists in (([p], [], [m], [v]), ([p], [p], [m, m], [v]), ([p, p], [p, p], [m, states(p, 8)[0]], [v, states(p, 8)[1]]),
                  ([p], [p], [states(p, 8)[0]], [v]), ([p], [p], [states(p, 8)[0] * 2], [states(p, 8)[1] * 2])):
        with pytest.raises(ValueError):
            adamw(*lists, 1)
    m8, v8 = states(p, 8)
    with pytest.raises(ValueError, match='8 bits'):
        adamw([p], [p], [m8], [v8], 1, eps=0.)
    with pytest.raises(RuntimeError):
        adamw([p], [p.to_sparse()], [m], [v], 1)
    for bits in (8, 32):
        m, v = states(p, bits)
        with pytest.raises(_hip.KfacHipError, match='cpu'):
            adamw([p], [p], [m], [v], 1)
    adamw([], [], [], [], 1)
    with pytest.raises(ValueError):
        states(p, 16)


def test_class_refusals():
    p = torch.nn.Parameter(torch.zeros(4, 5))
    AdamW = torchsso.optim.AdamW
    for more in (dict(lr=-1.), dict(betas=(1., .9)), dict(eps=-1.), dict(weight_decay=-1.), dict(state_bits=16),
                 dict(lr=torch.tensor(1e-3)), dict(state_bits=8, eps=0.)):
        with pytest.raises(ValueError):
            AdamW([p], **more)
    AdamW([p], lr=torch.tensor(1e-3), capturable=True)


class Fake(object):
    """What the check of the arguments looks at of a tensor on a device"""

    def __init__(self, shape, dtype=torch.float32, device=0, address=0, strides=None):
        self.shape, self.dtype, self.device, self.address = torch.Size(shape), dtype, torch.device('cuda', device), address
        self.like = torch.empty(shape, device='meta') if strides is None else torch.empty_strided(shape, strides, device='meta')

    is_cuda = True

    def stride(self):
        return self.like.stride()

    def numel(self):
        return self.shape.numel()

    def data_ptr(self):
        return self.address

    def element_size(self):
        return torch.empty((), dtype=self.dtype).element_size()

    def is_contiguous(self):
        return self.like.is_contiguous()


@pytest.fixture
def reason(monkeypatch):
    """Why a list of the given tensors is refused"""
    monkeypatch.setattr(torch, 'Tensor', Fake)
    monkeypatch.setattr(torch._C, '_has_storage', lambda t: True)
    monkeypatch.setattr(torch.ops.aten, 'is_non_overlapping_and_dense',
                        lambda t: bool(torch._prims_common.is_non_overlapping_and_dense(t.like)), raising=False)

    def of(p=None, g=None, m=None, v=None, ms=None, vs=None, steps=1, lr=1e-3, bits=32, twice=False):
        kinds = (torch.float8_e4m3fn, torch.float8_e5m2) if bits == 8 else (torch.float32,) * 2
        p, g = p or Fake((10, 20), address=1 << 20), g or Fake((10, 20))
        m, v = m or Fake((10, 20), kinds[0], address=2 << 20), v or Fake((10, 20), kinds[1], address=3 << 20)
        ms, vs = ms or Fake((2,), address=4 << 20), vs or Fake((2,), address=5 << 20)
        n = 2 if twice else 1
        with pytest.raises(_hip.KfacHipError) as e:
            _ops.check_adamw([p] * n, [g] * n, [m] * n, [v] * n, [ms] * n if bits == 8 else None,
                              [vs] * n if bits == 8 else None, steps, lr)
        return str(e.value)
    return of


def test_what_is_refused_is_named(reason):
    assert 'cannot take' in reason() and 'cannot take' in reason(bits=8)            # (nothing is wrong with these)
    assert 'gradient 0 has dtype' in reason(g=Fake((10, 20), torch.bfloat16))
    assert 'gradient 0 has shape' in reason(g=Fake((20, 10)))
    assert 'gradient 0 is on' in reason(g=Fake((10, 20), device=1))
    assert 'parameter 0 has dtype' in reason(p=Fake((10, 20), torch.float64))
    assert 'side by side' in reason(p=Fake((10, 20), strides=(40, 2)))
    assert 'first moment 0 has dtype' in reason(m=Fake((10, 20), torch.bfloat16))
    assert 'lie in memory' in reason(v=Fake((10, 20), strides=(1, 10))) and 'lie in memory' in reason(m=Fake((20, 10)))
    assert 'has dtype' in reason(bits=8, v=Fake((10, 20), torch.float8_e4m3fn))
    assert 'scale 0 has shape' in reason(bits=8, ms=Fake((3,)))
    assert 'scale 0 has dtype' in reason(bits=8, vs=Fake((2,), torch.float64))
    assert 'step 0 has dtype' in reason(steps=[Fake((), torch.int64)])
    assert 'step 0 has shape' in reason(steps=[Fake((2,), torch.int32)])
    assert 'needs steps' in reason(lr=Fake(())) and 'learning rate' in reason(lr=Fake((2,)), steps=[Fake((), torch.int32, address=9)])
    assert 'share memory' in reason(twice=True)
    assert 'share memory' in reason(m=Fake((10, 20), address=(1 << 20) + 796))
    assert 'cannot take' in reason(m=Fake((10, 20), address=(1 << 20) + 800))


def test_gradients_in_memory_that_is_written_are_named(reason):
    for base in (1, 2, 3):
        for offset in (-796, 0, 796):
            assert 'gradient 0 shares memory' in reason(g=Fake((10, 20), address=(base << 20) + offset))
        for offset in (-800, 800):
            assert 'cannot take' in reason(g=Fake((10, 20), address=(base << 20) + offset))
    # (one that lies otherwise is copied first)
    assert 'cannot take' in reason(g=Fake((10, 20), strides=(1, 10), address=1 << 20))


def test_random_numbers():
    """16 bits for m and 16 for v of every element: uniform, and no two of them that a rounding meets go together.
    (Over n numbers a mean of uniform ones is off by 0.29 / sqrt(n) on average, a correlation by 1 / sqrt(n): 5 times that.)"""
    n = 1 << 20
    first = words(n, 7, 3, 0)
    others = [words(n, 7, 4, 0), words(n, 7, 3, 1), words(n, 8, 3, 0)]
    streams = [(first >> 16).double() / 65536, (first & 0xffff).double() / 65536]
    for w in others:
        streams += [(w >> 16).double() / 65536, (w & 0xffff).double() / 65536]
    for s in streams:
        assert abs(s.mean().item() - 0.5) <= 5 * 0.29 / n ** 0.5
        count = torch.histc(s, 64, 0, 1)
        # (of each of 64 intervals n / 64 on average, off by the root of that: 5.5 times for 512 of them)
        assert bool(((count - n / 64).abs() <= 5.5 * (n / 64) ** 0.5).all())
    z = torch.stack([(s - s.mean()) / s.std() for s in streams])
    c = z @ z.t() / n - torch.eye(len(z), dtype=torch.float64)
    assert c.abs().max().item() <= 5 / n ** 0.5
    for s in z[:2]:
        for lag in (1, 2, 7, 8, 9, 16, 128):
            assert abs((s[lag:] * s[:-lag]).mean().item()) <= 5 / n ** 0.5


def test_mix_is_one_to_one():
    x = torch.arange(1 << 20, dtype=torch.int64) * 4093
    assert torch.unique(mix(x)).numel() == x.numel()


@pytest.mark.parametrize('kind', ['m', 'v'])
def test_rounding_keeps_the_mean(kind):
    """(of the reference that the kernels are compared with)"""
    gen = torch.Generator().manual_seed(0)
    x = torch.rand(128, generator=gen, dtype=torch.float64) * 10 ** torch.randint(-6, 1, (128,), generator=gen).double()
    many = x.repeat(4000)
    random = torch.randint(0, 1 << 16, (many.numel(),), generator=gen)
    q, scale, step = encode(many, kind, random)
    mean = (q * scale[0]).view(4000, 128).mean(0)
    smallest = numbers(kind)[1] * scale[0]
    # (a rounding is off by at most half a step on average: 5 times that over the root of 4000; a v below the smallest
    # number becomes that, and 16 bits leave 2^-17 of a step)
    bound = step.view(4000, 128)[0] * scale[0] * (5 * 0.5 / 4000 ** 0.5 + 2. ** -17) + (smallest if kind == 'v' else 0)
    assert bool(((mean - x).abs() <= bound).all())
    assert scale[0] == x.max() / LARGEST[kind]


def test_state_lies_as_the_parameter_does():
    for p in (torch.zeros(6, 4), torch.zeros(6, 4).t(), torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last), torch.zeros(())):
        for t in torchsso.optim.adamw_states(p):
            assert t.dtype == torch.float32 and t.stride() == p.stride() and not t.any()
        (m, ms), (v, vs) = torchsso.optim.adamw_states(p, 8)
        assert m.dtype == torch.float8_e4m3fn and v.dtype == torch.float8_e5m2 and m.stride() == v.stride() == p.stride()
        assert ms.shape == vs.shape == (-(-p.numel() // 128),) and not ms.any() and not m.float().any() and not v.float().any()


def fake_update(calls):
    def update(params, grads, ms, vs, steps, lr, *rest):
        calls.append((len(params), isinstance(ms[0], tuple), list(steps) if isinstance(steps, list) else steps, lr, rest))
        with torch.no_grad():
            for p in params:
                p.sub_(1)
        return True
    return update


def test_class_keeps_steps_and_bits_of_each_parameter(monkeypatch):
    calls = []
    monkeypatch.setattr(_ops, 'adamw', fake_update(calls))
    big, small, late = (torch.nn.Parameter(torch.zeros(n)) for n in (5000, 100, 6000))
    half = torch.nn.Parameter(torch.zeros(5000, dtype=torch.bfloat16))
    opt = torchsso.optim.AdamW([{'params': [big, small, late], 'lr': 1e-2}, {'params': [half], 'betas': (.8, .9)}], state_bits=8, seed=5)
    for p in (big, small, half):
        p.grad = torch.ones_like(p)
    opt.step()
    assert [c[:4] for c in calls] == [(1, True, [1], 1e-2), (1, False, [1], 1e-2), (1, True, [1], 1e-3)]
    assert [c[4][-1] for c in calls] == [5, 6, 7] and calls[2][4][:2] == (.8, .9)
    late.grad = torch.ones_like(late)
    calls.clear()
    opt.step()
    assert [c[:3] for c in calls] == [(2, True, [2, 1]), (1, False, [2]), (1, True, [2])]
    assert 'exp_avg_scale' in opt.state[big] and 'exp_avg_scale' not in opt.state[small]
    # an update that is refused does not count
    monkeypatch.setattr(_ops, 'adamw', lambda *a: (_ for _ in ()).throw(_hip.KfacHipError('no')))
    with pytest.raises(_hip.KfacHipError):
        opt.step()
    assert opt.state[big]['step'] == 2
    loss = torchsso.optim.AdamW([torch.nn.Parameter(torch.zeros(2))]).step(lambda: (torch.tensor(3.), None))
    assert loss[0] == 3.


@pytest.mark.parametrize('capturable', [False, True])
def test_state_dict_keeps_types(monkeypatch, capturable, tmp_path):
    monkeypatch.setattr(_ops, 'adamw', lambda *a: True)
    made = []
    for _ in range(2):
        params = [torch.nn.Parameter(torch.zeros(5000, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(3, 4).t())]
        made.append((params, torchsso.optim.AdamW(params, state_bits=8, capturable=capturable)))
    (params, opt), (others, other) = made
    for p in params:
        p.grad = torch.ones_like(p)
    opt.step()
    gen = torch.Generator().manual_seed(0)
    for p in params:
        for name, t in opt.state[p].items():
            if name != 'step':
                t.copy_(torch.randn(t.shape, generator=gen))
        opt.state[p]['step'] = torch.tensor(7, dtype=torch.int32) if capturable else 7
    torch.save(opt.state_dict(), tmp_path / 'state')
    other.load_state_dict(torch.load(tmp_path / 'state', weights_only=True))
    for p, q in zip(params, others):
        assert sorted(opt.state[p]) == sorted(other.state[q])
        for name, t in opt.state[p].items():
            u = other.state[q][name]
            if name == 'step':
                assert u == 7 and (u.dtype == torch.int32 if capturable else type(u) is int)
            else:
                assert u.dtype == t.dtype and u.stride() == t.stride() and torch.equal(u.float(), t.float())
    # loading does not share memory with what was saved
    loaded = torchsso.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in params], state_bits=8, capturable=capturable)
    saved = opt.state_dict()
    loaded.load_state_dict(saved)
    a, b = saved['state'][0]['exp_avg'], loaded.state[loaded.param_groups[0]['params'][0]]['exp_avg']
    assert a.data_ptr() != b.data_ptr()


def test_states_in_8_bits_of_another_order_of_memory_are_refused(monkeypatch):
    """The blocks that have a scale each are runs of memory: numbers put into another order would lie under others' scales."""
    monkeypatch.setattr(_ops, 'adamw', lambda *a: True)
    p = torch.nn.Parameter(torch.zeros(8, 4, 16, 16).contiguous(memory_format=torch.channels_last))
    q = torch.nn.Parameter(p.detach().contiguous())
    for bits in (8, 32):
        opt, other = (torchsso.optim.AdamW([t], state_bits=bits) for t in (p, q))
        p.grad = torch.ones_like(p)
        opt.step()
        if bits == 32:
            other.load_state_dict(opt.state_dict())
            assert other.state[q]['exp_avg'].stride() == q.stride()
        else:
            with pytest.raises(ValueError, match='lie in memory'):
                other.load_state_dict(opt.state_dict())
            assert not other.state


def test_states_of_torchs_class_are_taken(monkeypatch):
    calls = []
    monkeypatch.setattr(_ops, 'adamw', fake_update(calls))
    params = [torch.nn.Parameter(torch.randn(4, 5, dtype=torch.bfloat16)), torch.nn.Parameter(torch.randn(3))]
    other = torch.optim.AdamW(params, lr=3e-3, betas=(.8, .95), eps=1e-7, weight_decay=.2, foreach=False)
    for p in params:
        p.grad = torch.randn_like(p)
    for _ in range(2):
        other.step()
    for capturable in (False, True):
        opt = torchsso.optim.AdamW(params, seed=3, capturable=capturable)
        saved = other.state_dict()
        for group in saved['param_groups']:
            group.pop('capturable')               # (torch's is False: a step is a number then)
        opt.load_state_dict(saved)
        for p in params:
            state = opt.state[p]
            assert sorted(state) == ['exp_avg', 'exp_avg_sq', 'step'] and state['step'] == 2
            assert state['exp_avg'].dtype == state['exp_avg_sq'].dtype == torch.float32
            assert torch.equal(state['exp_avg'], other.state[p]['exp_avg'].float())
        calls.clear()
        if not capturable:
            opt.step()
            assert [c[2:] for c in calls] == [([3], 3e-3, (.8, .95, 1e-7, .2, 3)), ([3], 3e-3, (.8, .95, 1e-7, .2, 4))]
    for name in ('amsgrad', 'maximize'):
        with pytest.raises(ValueError, match=name):
            torchsso.optim.AdamW(params).load_state_dict(torch.optim.AdamW(params, **{name: True}).state_dict())


def test_lr_scheduler(monkeypatch):
    calls = []
    monkeypatch.setattr(_ops, 'adamw', fake_update(calls))
    p = torch.nn.Parameter(torch.zeros(5))
    opt = torchsso.optim.AdamW([p], lr=1.)
    sched = torch.optim.lr_scheduler.ExponentialLR(opt, 0.5)
    for _ in range(3):
        p.grad = torch.ones_like(p)
        opt.step()
        sched.step()
    assert [c[3] for c in calls] == [1., .5, .25]


@pytest.mark.parametrize('capturable', [False, True])
def test_a_step_that_ran_out_of_memory_can_be_taken_again(monkeypatch, capturable):
    """(where the states are made: none of a parameter, or all)"""
    calls = []
    monkeypatch.setattr(_ops, 'adamw', fake_update(calls))
    p = torch.nn.Parameter(torch.zeros(5000))
    p.grad = torch.ones_like(p)
    opt = torchsso.optim.AdamW([p], state_bits=8, capturable=capturable)
    zeros_like, made = torch.zeros_like, []

    def full(*args, **more):
        if made:
            raise torch.OutOfMemoryError('no memory')
        made.append(1)
        return zeros_like(*args, **more)
    monkeypatch.setattr(torch, 'zeros_like', full)
    with pytest.raises(torch.OutOfMemoryError):
        opt.step()
    assert made and not calls and not opt.state_dict()['state']
    monkeypatch.setattr(torch, 'zeros_like', zeros_like)
    opt.step()
    assert len(calls) == 1 and int(calls[0][2][0]) == (0 if capturable else 1)
    assert sorted(opt.state[p]) == ['exp_avg', 'exp_avg_scale', 'exp_avg_sq', 'exp_avg_sq_scale', 'step']


def test_options_of_a_group_are_checked(monkeypatch):
    calls = []
    monkeypatch.setattr(_ops, 'adamw', fake_update(calls))
    p, q = (torch.nn.Parameter(torch.zeros(n)) for n in (5000, 10))
    AdamW = torchsso.optim.AdamW
    for more in (dict(lr=-1.), dict(lr=float('nan')), dict(betas=(1., .9)), dict(eps=-1.), dict(weight_decay=-1.), dict(state_bits=16),
                 dict(state_bits=4), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            AdamW([dict(params=[p], **more)])
        opt = AdamW([q])
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=[p], **more))
        assert len(opt.param_groups) == 1
    opt = AdamW([dict(params=[p], lr=torch.tensor(1e-3), capturable=True), dict(params=[q], state_bits=8, eps=0.)])
    opt.param_groups[0]['state_bits'] = 16            # (changed later: said where states are made)
    for t in (p, q):
        t.grad = torch.ones_like(t)
    with pytest.raises(ValueError, match='16'):
        opt.step()
    opt.param_groups[0]['state_bits'] = 8
    opt.step()
    # (tensors too small for states in 8 bits take any eps)
    assert [c[1] for c in calls] == [True, False]
    with pytest.raises(TypeError):
        AdamW([q]).add_param_group([p])


@pytest.mark.parametrize('bits', [8, 32])
def test_states_of_another_shape_are_refused(monkeypatch, bits):
    """(not spread over the parameter: a vector's state over the rows of a matrix)"""
    monkeypatch.setattr(_ops, 'adamw', lambda *a: True)
    make = lambda shape: torchsso.optim.AdamW([torch.nn.Parameter(torch.zeros(shape))], state_bits=bits, min_8bit_size=1)
    opt, other = make((20,)), make((3, 20))
    p, q = (o.param_groups[0]['params'][0] for o in (opt, other))
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(ValueError, match='shape'):
        other.load_state_dict(opt.state_dict())
    assert not other.state
    for shape in ((20,), (1, 20)):
        make(shape).load_state_dict(opt.state_dict())
