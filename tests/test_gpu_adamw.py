"""torchsso.optim.adamw / AdamW against the formulas in 64 bits (adamw_testlib.py, where the tolerances are derived)."""
import copy
import math
import threading

import pytest
import torch

import torchsso
from torchsso import _hip

from adamw_testlib import (BLOCK, Update, blocks_top, check_8, check_m, check_p, check_v, decode, encode, flat, numbers, spread,
                           words)

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
BITS = pytest.mark.parametrize('bits', [32, 8])
OPTIONS = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def random(shape, dtype=torch.float32, seed=0, scale=1.):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype).cuda()


def gradient(shape, dtype, seed):
    """Of rows whose sizes differ by orders of magnitude, with zeros among them"""
    g = random(shape, torch.float32, seed)
    size = 10. ** random(shape[:1] or (1,), torch.float32, seed + 1000)
    g = g * size.view(shape[:1] + (1,) * (len(shape) - 1)) if shape else g
    g[torch.rand(shape, generator=torch.Generator().manual_seed(seed + 2000)).cuda() < 0.05] = 0
    return g.to(dtype)


def values(state):
    """A state in 64 bits, flat in the order of memory"""
    if isinstance(state, tuple):
        return decode(flat(state[0]), state[1])
    return flat(state)


def update_and_check(params, grads, ms, vs, step, seed=0, **options):
    """One call, and each of its results against the formulas on what was there before it."""
    steps = step if isinstance(step, list) else [step] * len(params)
    before = [(flat(p), flat(g if g.stride() == p.stride() else torch.empty_like(p).copy_(g)), values(m), values(v))
              for p, g, m, v in zip(params, grads, ms, vs)]
    torchsso.optim.adamw(params, grads, ms, vs, step, seed=seed, **options)
    options = dict(OPTIONS, **options)
    for i, (p, m, v) in enumerate(zip(params, ms, vs)):
        u = Update(*before[i], steps[i], options['lr'], options['betas'], options['eps'], options['weight_decay'])
        check_p(flat(p), u, p.dtype)
        if isinstance(m, tuple):
            w = words(p.numel(), seed, steps[i], i)
            check_8(m[0], m[1], u.m, 'm', w >> 16)
            check_8(v[0], v[1], u.v, 'v', w & 0xffff)
        else:
            check_m(flat(m), u)
            check_v(flat(v), u)


SHAPES = [(1,), (2,), (7,), (8,), (9,), (127,), (128,), (129,), (), (1000,), (3, 5, 7), (2048,), (4095,), (4096,), (4097,), (61, 203),
          (16, 512), (1, 1), (300, 301)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@BITS
def test_updates_of_a_list(dtype, bits):
    params = [random(s, dtype, i) for i, s in enumerate(SHAPES)]
    states = [torchsso.optim.adamw_states(p, bits) for p in params]
    ms, vs = [s[0] for s in states], [s[1] for s in states]
    for t in range(1, 5):
        grads = [gradient(s, dtype, 10 * t + i) for i, s in enumerate(SHAPES)]
        update_and_check(params, grads, ms, vs, t, seed=17, **OPTIONS)


@BITS
@pytest.mark.parametrize('options', [dict(betas=(0., 0.)), dict(betas=(0.95, 0.5), weight_decay=0.), dict(lr=0.), dict(eps=1e-3),
                                     dict(betas=(0., 0.99), eps=1e-12), dict(step=1000003), dict(seed=2 ** 32 - 1), dict(seed=-1)], ids=str)
def test_options(bits, options):
    options = dict(dict(OPTIONS, step=3, seed=5), **options)
    step = options.pop('step')
    params, grads = [random((50, 37)), random((4100,), seed=1)], [gradient((50, 37), torch.float32, 2), gradient((4100,), torch.float32, 3)]
    states = [torchsso.optim.adamw_states(p, bits) for p in params]
    ms, vs = [s[0] for s in states], [s[1] for s in states]
    for k in range(2):
        update_and_check(params, grads, ms, vs, step + k, **options)


@BITS
def test_many_tensors_with_steps_of_their_own(bits):
    shapes = [(n % 40 + 1, n % 7 + 1) if n % 3 else (37 * n + 1,) for n in range(131)]
    params = [random(s, torch.bfloat16, i) for i, s in enumerate(shapes)]
    grads = [gradient(s, torch.bfloat16, i + 500) for i, s in enumerate(shapes)]
    states = [torchsso.optim.adamw_states(p, bits) for p in params]
    ms, vs = [s[0] for s in states], [s[1] for s in states]
    update_and_check(params, grads, ms, vs, [1 + i % 5 for i in range(len(shapes))], **OPTIONS)
    update_and_check(params, grads, ms, vs, [2 + i % 5 for i in range(len(shapes))], **OPTIONS)
    # (more different numbers than a launch holds)
    update_and_check(params, grads, ms, vs, [3 + i % 5 + 7 * (i % 23) for i in range(len(shapes))], **OPTIONS)


@BITS
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('offset', [0, 1, 3, 4, 8, 120])
def test_parts_of_a_buffer_and_nothing_around_them(bits, dtype, offset):
    """Tensors that begin anywhere: what lies beside them stays as it is, parameters and states alike."""
    n = 1000
    whole = dict(p=random((2000,), dtype), g=random((2000,), dtype, 1), m=random((2000,), seed=2), v=random((2000,), seed=3).abs())
    if bits == 8:
        whole['m'], whole['v'] = whole['m'].to(torch.float8_e4m3fn), whole['v'].to(torch.float8_e5m2)
        whole.update(ms=random((30,), seed=4).abs(), vs=random((30,), seed=5).abs())
    before = {k: t.clone() for k, t in whole.items()}
    part = {k: t[offset:offset + n] for k, t in whole.items()}
    if bits == 8:
        part['ms'], part['vs'] = whole['ms'][offset % 5:offset % 5 + 8], whole['vs'][offset % 5:offset % 5 + 8]
        part['m'], part['v'] = (part['m'], part['ms']), (part['v'], part['vs'])
    update_and_check([part['p']], [part['g']], [part['m']], [part['v']], 4, **OPTIONS)
    for k, t in whole.items():
        size, first = (8, offset % 5) if k in ('ms', 'vs') else (n, offset)
        raw = [x.view(torch.uint8) if x.element_size() == 1 else x for x in (t, before[k])]
        assert torch.equal(raw[0][:first], raw[1][:first]) and torch.equal(raw[0][first + size:], raw[1][first + size:])
    assert torch.equal(whole['g'], before['g'])


@BITS
def test_orders_of_memory(bits):
    base = [random((40, 30)).t(), random((4, 6, 5, 7)).to(memory_format=torch.channels_last), random((8, 3, 5)).permute(2, 0, 1),
            random((1, 50)).expand(1, 50)]
    for gradients in ('alike', 'other', 'spread', 'strided'):
        params = [p.clone(memory_format=torch.preserve_format) for p in base]
        assert [p.stride() for p in params[:3]] == [p.stride() for p in base[:3]]
        grads = [torch.empty_like(p).copy_(random(p.shape, seed=7)) for p in params]
        if gradients == 'other':
            grads = [g.contiguous() for g in grads]
        elif gradients == 'spread':
            grads = [random((), seed=8).expand(p.shape) for p in params]
        elif gradients == 'strided':
            grads = [random(p.shape + (2,), seed=9)[..., 1] for p in params]
        states = [torchsso.optim.adamw_states(p, bits) for p in params]
        update_and_check(params, grads, [s[0] for s in states], [s[1] for s in states], 2, **OPTIONS)


@BITS
def test_numbers_that_are_not_finite_stay_by_themselves(bits):
    n = 4 * BLOCK + 50
    grad, at = random((n,), seed=1), {3: math.nan, 130: math.inf, 131: -math.inf, 300: 1e30, 4 * BLOCK + 20: math.nan}
    clean = grad.clone()
    for i, x in at.items():
        grad[i], clean[i] = x, 0.
    results = []
    for g in (clean, grad):
        p = random((n,))
        m, v = torchsso.optim.adamw_states(p, bits)
        for t in (1, 2, 3):
            torchsso.optim.adamw([p], [g], [m], [v], t, **OPTIONS)
        results.append((flat(p), values(m), values(v)))
    others = torch.ones(n, dtype=torch.bool)
    others[list(at)] = False
    if bits == 8:
        # (1e30 is a number, and the largest m of its block: the others there are small beside it; its square is not finite)
        others[2 * BLOCK:3 * BLOCK] = False
    for a, b in zip(*results):
        assert torch.equal(a[others], b[others])
    p, m, v = results[1]
    for i in (3, 4 * BLOCK + 20):
        assert all(math.isnan(t[i]) for t in (p, m, v))
    for i in (130, 131):
        assert math.isnan(p[i]) and math.isinf(v[i]) and (math.isnan(m[i]) if bits == 8 else math.isinf(m[i]))
    assert math.isinf(v[300]) and math.isfinite(p[300]) and m[300] > 1e29
    if bits == 8:
        # the block's other elements have not been touched by that in p
        same = torch.arange(2 * BLOCK, 3 * BLOCK)
        assert torch.isfinite(p[same]).all()
        # ... and an infinite v alone in its block
        p, g = random((BLOCK,)), torch.zeros(BLOCK, device='cuda')
        g[5] = 1e30
        m, v = torchsso.optim.adamw_states(p, 8)
        first = flat(p)
        for t in (1, 2):
            torchsso.optim.adamw([p], [g], [m], [v], t, lr=1e-2, weight_decay=0.)
        assert torch.equal(flat(p), first) and math.isinf(values(v)[5]) and values(v)[[i for i in range(BLOCK) if i != 5]].eq(0).all()


@pytest.mark.parametrize('size', [0., 1e-45, 1e-30, 1e-18, 1e-12, 1e12])
def test_sizes_of_gradients_in_8_bits(size):
    p, g = random((1000,)), random((1000,), seed=1, scale=size)
    m, v = torchsso.optim.adamw_states(p, 8)
    for t in (1, 2, 3):
        update_and_check([p], [g], [m], [v], t, **OPTIONS)
    if size < 1e-20:
        assert not values(v).any()


def test_a_v_above_zero_stays_above_zero():
    """Beside an element whose gradient is 10^6 times as large: v's root is less than the smallest number then."""
    p, g = torch.zeros(BLOCK, device='cuda'), torch.full((BLOCK,), 1e-6, device='cuda')
    g[0] = 1.
    m, v = torchsso.optim.adamw_states(p, 8)
    for t in range(1, 30):
        torchsso.optim.adamw([p], [g], [m], [v], t, lr=1e-3, weight_decay=0.)
        assert bool((flat(v[0]) > 0).all())
    # each update is at most lr * m / sqrt(v), corrected: no larger than 32 bits would make it
    assert bool((flat(p).abs() <= 29 * 1e-3 * (1 + 1e-3)).all())


def test_states_in_8_bits_keep_what_single_updates_add():
    """A constant gradient: m and v go to g and g^2, by a tenth and a thousandth of the difference an update.

    Rounding at random keeps the mean of both.  Over n elements the mean of their ratios to what 64 bits give is off by
    their spread over the root of n: a single rounding is at most half a step off on average, an eighth of v (e5m2) and a
    sixteenth of m.  v keeps the last 1000 roundings of which each acts on the thousandth part of a step, so that
    its spread is at most sqrt(step / 2) = 0.36, m's at most 0.3: 5 times 0.36 / sqrt(n) = 0.006 for n = 10^5."""
    n = 100000
    g = random((n,)) + 3
    p = torch.zeros(n, device='cuda')
    m, v = torchsso.optim.adamw_states(p, 8)
    for t in range(1, 2001):
        torchsso.optim.adamw([p], [g], [m], [v], t, lr=0.)
    g = flat(g)
    some = g.abs() > 0.5
    for got, want in ((values(m), g), (values(v), g * g * -math.expm1(2000 * math.log(0.999)))):
        ratio = (got / want)[some]
        assert abs(ratio.mean().item() - 1) <= 0.006


def test_the_same_call_gives_the_same_bits_and_another_seed_others():
    def run(seed):
        p, g = random((5000,), torch.bfloat16), random((5000,), torch.bfloat16, 1)
        m, v = torchsso.optim.adamw_states(p, 8)
        for t in (1, 2):
            torchsso.optim.adamw([p], [g], [m], [v], t, seed=seed)
        return [p] + [t.view(torch.uint8) if t.element_size() == 1 else t for t in m + v]
    first, again, other = run(1), run(1), run(2)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert not torch.equal(first[1], other[1]) and not torch.equal(first[3], other[3])


@BITS
def test_recorded_updates_count_on(bits):
    """Counters on the device: every replay is the next update, as an eager call with numbers is, with other work and
    a changed learning rate between them."""
    shapes = [(50, 37), (4100,), (3,)] + [(5,)] * 300

    def make():
        params = [random(s, seed=i) for i, s in enumerate(shapes)]
        return params, [torchsso.optim.adamw_states(p, bits) for p in params]
    (params, states), (others, other_states) = make(), make()
    grads = [random(s, seed=500 + i) for i, s in enumerate(shapes)]
    steps = [torch.full((), i % 3, dtype=torch.int32, device='cuda') for i in range(len(shapes))]
    lr = torch.tensor(1e-2, device='cuda')
    args = (params, grads, [s[0] for s in states], [s[1] for s in states], steps)

    def number(k, rate):
        torchsso.optim.adamw(others, grads, [s[0] for s in other_states], [s[1] for s in other_states],
                             [i % 3 + k for i in range(len(shapes))], lr=rate, weight_decay=0.1, seed=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torchsso.optim.adamw(*args, lr=lr, weight_decay=0.1, seed=3)
    torch.cuda.current_stream().wait_stream(side)
    number(1, 1e-2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        torchsso.optim.adamw(*args, lr=lr, weight_decay=0.1, seed=3)
    for k in range(2, 6):
        rate = 1e-2 / k
        lr.fill_(rate)
        for g in grads:
            g.mul_(0.9)
        graph.replay()
        number(k, torch.tensor(rate).item())
        torch.cuda.synchronize()
        assert [int(s) for s in steps[:5]] == [i % 3 + k for i in range(5)]
        for p, q in zip(params, others):
            # (the device's logarithm and exponential are not the host's to the last of 64 bits, nor lr in 32 bits)
            assert bool(((p - q).abs() <= 1e-6 * (q.abs() + 1)).all())
        for s, o in zip(states, other_states):
            for a, b in zip(s, o):
                assert torch.equal(values(a), values(b))


@BITS
def test_two_graphs_and_another_stream(bits):
    """Graphs that share a pool of memory, replayed in turn"""
    def make(seed):
        p, g = random((3000,), seed=seed), random((3000,), seed=seed + 1)
        return p, g, torchsso.optim.adamw_states(p, bits), torch.zeros((), dtype=torch.int32, device='cuda')
    both, want = [make(0), make(10)], [make(0), make(10)]
    side, graphs, pool = torch.cuda.Stream(), [], None
    side.wait_stream(torch.cuda.current_stream())
    for p, g, s, t in both:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool, stream=side):
            torchsso.optim.adamw([p], [g], [s[0]], [s[1]], [t])
        graphs.append(graph)
        pool = graph.pool()
    for k in range(3):
        for graph in graphs:
            graph.replay()
        for p, g, s, t in want:
            torchsso.optim.adamw([p], [g], [s[0]], [s[1]], k + 1)
        torch.cuda.synchronize()
        for (p, _, s, _), (q, _, o, _) in zip(both, want):
            assert bool(((p - q).abs() <= 1e-6 * (q.abs() + 1)).all())
            assert all(torch.equal(values(a), values(b)) for a, b in zip(s, o))


@BITS
def test_two_threads_at_once(bits):
    def make(seed):
        p = random((100, 333), torch.bfloat16, seed)
        return p, random((100, 333), torch.bfloat16, seed + 1), torchsso.optim.adamw_states(p, bits)

    def work(p, g, s):
        for t in range(1, 30):
            torchsso.optim.adamw([p], [g], [s[0]], [s[1]], t)
    want, got = [make(k) for k in range(2)], [make(k) for k in range(2)]
    for w in want:
        work(*w)
    torch.cuda.synchronize()

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            work(*got[k])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for w, g in zip(want, got):
        assert torch.equal(w[0], g[0])
        assert all(torch.equal(values(a), values(b)) for a, b in zip(w[2], g[2]))


def test_refusals():
    p, g = random((40, 50)), random((40, 50), seed=1)
    m, v = torchsso.optim.adamw_states(p)
    m8, v8 = torchsso.optim.adamw_states(p, 8)
    before = [t.clone() for t in (p, m, v)]
    adamw = torchsso.optim.adamw
    count = torch.zeros((), dtype=torch.int32, device='cuda')
    for bad in (lambda: adamw([p], [g.bfloat16()], [m], [v], 1), lambda: adamw([p], [g[:39]], [m], [v], 1),
                lambda: adamw([p.double()], [g.double()], [m], [v], 1), lambda: adamw([p], [g.cpu()], [m], [v], 1),
                lambda: adamw([p], [g], [m.bfloat16()], [v], 1), lambda: adamw([p], [g], [m], [v.cpu()], 1),
                lambda: adamw([p, p], [g, g], [m, m.clone()], [v, v.clone()], 1), lambda: adamw([p], [g], [m], [m], 1),
                lambda: adamw([p], [g], [m.t().contiguous().t()], [v], 1), lambda: adamw([p[:, ::2]], [g[:, ::2]], [m[:, ::2]], [v[:, ::2]], 1),
                lambda: adamw([p[:, :20]], [g[:, :20]], [m[:, :20]], [v[:, :20]], 1),
                lambda: adamw([p], [g], [(m8[0], m8[1][:-1])], [v8], 1), lambda: adamw([p], [g], [v8], [m8], 1),
                lambda: adamw([p], [g], [(m8[0], v8[1])], [v8], 1),
                lambda: adamw([p[:30], p[20:]], [g[:30], g[20:]], [m[:30], m[20:].clone()], [v[:30], v[20:].clone()], 1),
                lambda: adamw([torch._neg_view(p)], [g], [m], [v], 1), lambda: adamw([p], [g], [torch._neg_view(m)], [v], 1),
                lambda: adamw([p], [g], [m], [v], [count.long()]), lambda: adamw([p], [g], [m], [v], [count.cpu()]),
                lambda: adamw([p, p.clone()], [g, g], [m, m.clone()], [v, v.clone()], [count, count]),
                lambda: adamw([p], [g], [m], [v], 1, lr=torch.tensor(1., device='cuda')),
                lambda: adamw([p], [g], [m], [v], [count], lr=torch.tensor(1.)),
                lambda: adamw([p, p.clone().bfloat16()], [g, g], [m, m.clone()], [v, v.clone()], 1)):
        with pytest.raises(_hip.KfacHipError):
            bad()
    assert all(torch.equal(a, b) for a, b in zip(before, (p, m, v))) and int(count) == 0
    adamw([], [], [], [], 1)
    empty = torch.zeros(0, 5, device='cuda')
    states = torchsso.optim.adamw_states(empty), torchsso.optim.adamw_states(empty, 8)
    for s in states:
        adamw([empty], [empty], [s[0]], [s[1]], 1)
    adamw([empty, p], [empty, g], [torch.zeros_like(empty), m], [torch.zeros_like(empty), v], [count, count.clone()])
    assert int(count) == 1 and not torch.equal(p, before[0])


@pytest.mark.parametrize('bits', [32, 8])
def test_gradients_in_memory_that_is_written(bits):
    """Refused where another thread may have written them already; a copy is made of those that lie otherwise."""
    buffer = random((3 * 4096,))
    p, q = buffer[:4096].view(64, 64), buffer[4096:8192].view(64, 64)
    states = [torchsso.optim.adamw_states(t, bits) for t in (p, q)]
    m, v = zip(*states)
    free = random((64, 64), seed=1)
    before = buffer.clone()
    for g in (q, p, buffer[100:4196].view(64, 64), buffer[8191:12287].view(64, 64)):
        with pytest.raises(_hip.KfacHipError):
            torchsso.optim.adamw([p, q], [g, free], m, v, 1)
    if bits == 32:
        with pytest.raises(_hip.KfacHipError):
            torchsso.optim.adamw([p, q], [free, v[0]], m, v, 1)
    assert torch.equal(buffer, before)
    want = [p.clone(), q.clone()]
    copies = [torchsso.optim.adamw_states(t, bits) for t in want]
    torchsso.optim.adamw(want, [q.t().contiguous(), buffer[8192:].view(64, 64)], *zip(*copies), 1)
    torchsso.optim.adamw([p, q], [q.t(), buffer[8192:].view(64, 64)], m, v, 1)
    assert torch.equal(p, want[0]) and torch.equal(q, want[1])


def test_an_update_is_a_change_in_place_that_autograd_sees():
    p = torch.nn.Parameter(random((4, 6)))
    x = random((3, 6)).requires_grad_()
    before = (x @ p.t()).square().sum()
    for bits in (32, 8):
        opt = torchsso.optim.AdamW([p], state_bits=bits, min_8bit_size=1)
        p.grad = random((4, 6), seed=1)
        version = p._version
        opt.step()
        assert p._version > version and opt.state[p]['exp_avg']._version > 0
    with pytest.raises(RuntimeError, match='inplace'):
        before.backward()


# ---------------------------------------------------------------------------------------
# the class
# ---------------------------------------------------------------------------------------

def model(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Embedding(50, 120), torchsso.nn.LayerNorm(120), torch.nn.Linear(120, 90), torch.nn.Tanh(),
                               torch.nn.Linear(90, 7)).cuda().to(dtype)


def backward(net, seed):
    gen = torch.Generator().manual_seed(seed)
    x, y = torch.randint(0, 50, (64,), generator=gen).cuda(), torch.randint(0, 7, (64,), generator=gen).cuda()
    net.zero_grad()
    loss = torch.nn.functional.cross_entropy(net(x).float(), y)
    loss.backward()
    return loss


@pytest.mark.parametrize('capturable', [False, True])
def test_class_against_torchs_in_64_bits(capturable):
    net = model()
    groups = lambda params: [{'params': params[:3], 'weight_decay': 0.}, {'params': params[3:], 'lr': 3e-3}]
    params = list(net.parameters())
    others = [p.detach().cpu().double().requires_grad_() for p in params]
    options = dict(lr=1e-3, betas=(0.9, 0.99), weight_decay=0.1)
    opt = torchsso.optim.AdamW(groups(params), capturable=capturable, **options)
    other = torch.optim.AdamW(groups(others), foreach=False, **options)
    for t in range(6):
        backward(net, t)
        for p, q in zip(params, others):
            q.grad = p.grad.cpu().double()
        if t == 2:
            params[4].grad = others[4].grad = None
        opt.step()
        other.step()
    for p, q in zip(params, others):
        # (six updates of at most 3e-3 (and twice that early on), each off by at most 2^-19 of it, and six roundings of p)
        assert bool(((p.detach().cpu().double() - q).abs() <= 6 * (6e-3 * 2. ** -19 + 2. ** -23 * q.abs())).all())
        assert int(opt.state[p]['step']) == int(other.state[q]['step'])


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('capturable', [False, True])
def test_saved_and_continued(bits, capturable, tmp_path):
    nets, opts = [], []
    for _ in range(2):
        nets.append(model(torch.bfloat16))
        opts.append(torchsso.optim.AdamW(nets[-1].parameters(), lr=1e-2, state_bits=bits, min_8bit_size=2000, capturable=capturable))
    for t in range(3):
        backward(nets[0], t)
        opts[0].step()
    kinds = set('exp_avg_scale' in s for s in opts[0].state.values())
    assert kinds == ({True, False} if bits == 8 else {False})
    torch.save([nets[0].state_dict(), opts[0].state_dict()], tmp_path / 'saved')
    saved = torch.load(tmp_path / 'saved', weights_only=True)
    nets[1].load_state_dict(saved[0])
    opts[1].load_state_dict(saved[1])
    for t in range(3, 6):
        for net, opt in zip(nets, opts):
            backward(net, t)
        for p, q in zip(nets[0].parameters(), nets[1].parameters()):
            q.grad.copy_(p.grad)              # (sums of the embedding's gradient are not in one order)
        for opt in opts:
            opt.step()
    for p, q in zip(nets[0].parameters(), nets[1].parameters()):
        assert torch.equal(p, q)
        for name, a in opts[0].state[p].items():
            b = opts[1].state[q][name]
            assert a == b if name == 'step' else a.dtype == b.dtype and torch.equal(a.float(), b.float())


@pytest.mark.parametrize('bits', [32, 8])
def test_a_recorded_step(bits):
    params = [torch.nn.Parameter(random((70, 80))), torch.nn.Parameter(random((9,)))]
    others = copy.deepcopy(params)
    make = lambda ps, **more: torchsso.optim.AdamW(ps, lr=1e-2, state_bits=bits, min_8bit_size=100, **more)
    opt, other = make(params, capturable=True), make(others)
    for p, q in zip(params, others):
        p.grad = random(p.shape, seed=3)
        q.grad = p.grad.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='before one is recorded'):
        with torch.cuda.graph(graph, stream=side):
            opt.step()
    with pytest.raises(RuntimeError, match='capturable'):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            other.step()
    opt.step()
    other.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step()
    for t in range(2, 5):
        graph.replay()
        other.step()
        torch.cuda.synchronize()
        for p, q in zip(params, others):
            assert bool(((p - q).abs() <= 1e-6 * (q.abs() + 1)).all()) and int(opt.state[p]['step']) == t
    # an eager step goes on from there
    opt.step()
    other.step()
    for p, q in zip(params, others):
        assert bool(((p - q).abs() <= 1e-6 * (q.abs() + 1)).all())


def test_beside_muon_and_a_curvature():
    """A layer norm by its curvature, a matrix by Muon, the rest by AdamW in 8 bits: a step of a model in parts"""
    net = model()
    before = [p.detach().clone() for p in net.parameters()]
    opts = [torchsso.optim.SecondOrderOptimizer(torch.nn.ModuleList([net[1]]), 'Cov', {'LayerNorm': 'Diag'}, {'damping': 1e-2}, lr=1e-2),
            torchsso.optim.Muon([net[2].weight]),
            torchsso.optim.AdamW([net[0].weight, net[2].bias, net[4].weight, net[4].bias], lr=1e-2, state_bits=8)]
    for t in range(3):
        loss = backward(net, t)
        for opt in opts:
            opt.step()
        assert torch.isfinite(loss)
    for p, b in zip(net.parameters(), before):
        assert torch.isfinite(p).all() and not torch.equal(p, b)


def test_numbers_on_the_device_whose_sign_is_still_to_be_applied():
    """A learning rate is read with it; a counter, which is written, is refused."""
    p, g = random((300,)), random((300,), seed=1)
    q = p.clone()
    step = lambda: torch.zeros((), dtype=torch.int32, device='cuda')
    rate = torch.tensor(1e-2, device='cuda')
    for t, lr in ((p, torch._neg_view(-rate)), (q, rate)):
        m, v = torchsso.optim.adamw_states(t)
        torchsso.optim.adamw([t], [g], [m], [v], [step()], **dict(OPTIONS, lr=lr))
    assert torch.equal(p, q)
    m, v = torchsso.optim.adamw_states(p)
    with pytest.raises(_hip.KfacHipError):
        torchsso.optim.adamw([p], [g], [m], [v], [torch._neg_view(step())], **OPTIONS)
    assert torch.equal(p, q)


@BITS
@pytest.mark.parametrize('on_device', [False, True])
@pytest.mark.parametrize('lr', [0., 1e-35])
def test_an_update_by_nothing_leaves_parameters_whose_v_overflows(bits, on_device, lr):
    """The first steps of a schedule from 0: m is a number, the root of v infinite, and the update 0."""
    p, g = random((300,)), random((300,), seed=1)
    g[::7] = 1e25
    before = p.clone()
    m, v = torchsso.optim.adamw_states(p, bits)
    step = [torch.zeros((), dtype=torch.int32, device='cuda')] if on_device else 1
    torchsso.optim.adamw([p], [g], [m], [v], step, **dict(OPTIONS, lr=torch.tensor(lr, device='cuda') if on_device else lr))
    assert bool(torch.isinf(flat(v[0] if bits == 8 else v)[::7]).all())
    # (1 - lr weight_decay is 1 in float32)
    assert torch.equal(p, before)


@BITS
@pytest.mark.parametrize('capturable', [False, True])
def test_states_made_in_inference_mode(bits, capturable):
    """Such tensors have no version to raise: what has been updated is not reported as an error."""
    p, g = random((70, 80)), random((70, 80), seed=1)
    q, plain = p.clone(), torchsso.optim.adamw_states(p, bits)
    with torch.inference_mode():
        m, v = torchsso.optim.adamw_states(p, bits)
        step = torch.zeros((), dtype=torch.int32, device='cuda')
    for t in (1, 2):
        torchsso.optim.adamw([p], [g], [m], [v], [step] if capturable else t, **OPTIONS)
        torchsso.optim.adamw([q], [g], [plain[0]], [plain[1]], t, **OPTIONS)
    assert p._version == 2 and (not capturable or int(step) == 2)
    if capturable:
        # (the device's logarithms may be off by some last bits of 64: no more than one of 32)
        assert bool(((p - q).abs() <= 1e-6 * (q.abs() + 1)).all())
    else:
        assert torch.equal(p, q) and torch.equal(values(m), values(plain[0])) and torch.equal(values(v), values(plain[1]))
    # a step of the class in that mode makes such states; it goes on outside
    w = torch.nn.Parameter(random((70, 80)))
    w.grad = g
    opt = torchsso.optim.AdamW([w], state_bits=bits, capturable=capturable)
    with torch.inference_mode():
        opt.step()
    opt.step()
    assert int(opt.state[w]['step']) == 2


# ---------------------------------------------------------------------------------------
# large
# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize('bits', [32, 8])
def test_more_elements_than_32_bits_count(bits):
    n = (1 << (32 if bits == 8 else 31)) + 5 * BLOCK + 77
    p = torch.zeros(n, device='cuda', dtype=torch.bfloat16)
    g = torch.zeros(n, device='cuda', dtype=torch.bfloat16)
    m, v = torchsso.optim.adamw_states(p, bits)
    parts = [slice(0, 300), slice(1 << 31, (1 << 31) + 70), slice((n - 205) // BLOCK * BLOCK, n)]
    few = []
    for i, s in enumerate(parts):
        k = len(range(*s.indices(n)))
        p[s], g[s] = random((k,), torch.bfloat16, 2 * i), random((k,), torch.bfloat16, 2 * i + 1)
        few.append((p[s].clone(), g[s].clone()))
    for t in (1, 2):
        torchsso.optim.adamw([p], [g], [m], [v], t, **OPTIONS)
    for s, (q, d) in zip(parts, few):
        if bits == 32:
            a, b = torchsso.optim.adamw_states(q)
            for t in (1, 2):
                torchsso.optim.adamw([q], [d], [a], [b], t, **OPTIONS)
            assert torch.equal(p[s], q) and torch.equal(m[s], a) and torch.equal(v[s], b)
            continue
        # (other random numbers than the same elements at the start of a tensor would have)
        x = torch.zeros(q.numel(), dtype=torch.float64)
        u = Update(flat(q), flat(d), x, x, 1, **OPTIONS)
        w = words(q.numel(), 0, 1, 0, s.start % (1 << 35))
        state = []
        for kind, want, r in (('m', u.m, w >> 16), ('v', u.v, w & 0xffff)):
            code, scale, _ = encode(want, kind, r)
            state.append(code * spread(scale, code.numel()))
        u = Update(u.p.bfloat16().double(), flat(d), *state, 2, **OPTIONS)
        # (of the first update a number in 2^14 may have been rounded otherwise, by up to a quarter: u's size twice)
        near = (flat(p[s]) - u.p).abs() <= 2. ** -8 * u.p.abs() + 2. ** -7 * (u.p_size + u.u_size)
        assert int((~near).sum()) <= 3
        blocks = slice(s.start // BLOCK, -(-(s.start + q.numel()) // BLOCK))
        assert bool((m[1][blocks] > 0).all())
    # what has no gradient has not moved
    assert not p[400:1 << 31].any()


def test_states_in_8_bits_behind_more_elements_than_32_bits_count():
    """Codes and scales there are those of their own places: of the blocks, and of the random numbers' units."""
    n = (1 << 32) + 5 * BLOCK + 77
    p = torch.zeros(n, device='cuda', dtype=torch.bfloat16)
    g = torch.zeros_like(p)
    m, v = torchsso.optim.adamw_states(p, 8)
    parts = [slice(0, 300), slice((1 << 31) - 40 * BLOCK, (1 << 31) + 70), slice((n - 205) // BLOCK * BLOCK, n)]
    for i, s in enumerate(parts):
        k = s.stop - s.start
        p[s], g[s] = random((k,), torch.bfloat16, 2 * i), random((k,), torch.bfloat16, 2 * i + 1)
    for t in (1, 2):
        blocks = [slice(s.start // BLOCK, -(-s.stop // BLOCK)) for s in parts]
        part = lambda state: [(state[0][s], state[1][b]) for s, b in zip(parts, blocks)]
        before = [(flat(p[s]), flat(g[s]), values(a), values(b)) for s, a, b in zip(parts, part(m), part(v))]
        torchsso.optim.adamw([p], [g], [m], [v], t, seed=3, **OPTIONS)
        for s, was, (mq, ms), (vq, vs) in zip(parts, before, part(m), part(v)):
            u = Update(*was, t, *(OPTIONS[k] for k in ('lr', 'betas', 'eps', 'weight_decay')))
            w = words(s.stop - s.start, 3, t, 0, s.start)
            check_p(flat(p[s]), u, p.dtype)
            check_8(mq, ms, u.m, 'm', w >> 16)
            check_8(vq, vs, u.v, 'v', w & 0xffff)
    # (and nothing beside them)
    assert not m[1][3:parts[1].start // BLOCK].any() and not v[1][parts[1].stop // BLOCK + 1:parts[2].start // BLOCK].any()
