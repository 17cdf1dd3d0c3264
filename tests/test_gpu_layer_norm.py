"""torchsso.nn.layer_norm / add_layer_norm / LayerNorm and DiagCovLayerNorm against the formulas in 64 bits.

Tolerances (2-norm of the difference over that of what is compared with).  Everything is computed in
float32 and rounded once, so a result may be as far from the exact one as the exact one's own rounding
to its type, 5 % more for elements that round the other way, and what float32 loses: of xh two
differences and a product, 2^-24 each, and of 1 / sqrt(var + eps), which all of a row share, half of a
mean of squares' 4 * 2^-24 and a root's 2^-23; a product and a sum behind that: 6e-7, taken as 1e-6 of the
terms of y (xh gain and bias), which is also what dx may be off in units of its terms.  The sums over
rows are random walks of such terms, 2e-6 (their squares 4e-6).
"""
import threading

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import torchsso
from torchsso import _hip, _ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5
EIGHT = torch.float8_e4m3fn


def random(shape, dtype=torch.float32, seed=0, scale=1., offset=0.):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale + offset).to(dtype).cuda()


def check(got, want, dtype, more, scale=None):
    """`got` (of `dtype`) is as near to `want` (float64) as float32 arithmetic and one rounding allow."""
    assert got.dtype == dtype and got.shape == want.shape
    got = got.detach().cpu().double()
    rounding = (want.to(dtype).double() - want).norm().item()
    size = want.norm().item() if scale is None else scale
    error = (got - want).norm().item()
    assert error <= 1.05 * rounding + more * size, (error / max(size, 1e-300), rounding / max(size, 1e-300))


class Want(object):
    """The formulas in 64 bits, from tensors anywhere"""

    def __init__(self, x, residual, gain, bias, dy=None, dh=None, samples=1, eps=EPS):
        dtype = x.dtype
        to = lambda t: None if t is None else t.detach().cpu().double()
        x, residual, gain, bias, dy, dh = map(to, (x, residual, gain, bias, dy, dh))
        self.h = h = x if residual is None else (x + residual).to(dtype).double()
        dim = h.shape[-1]
        w = torch.ones(dim, dtype=torch.float64) if gain is None else gain
        b = torch.zeros(dim, dtype=torch.float64) if bias is None else bias
        d = h - h.mean(-1, keepdim=True)
        r = 1 / (d.square().mean(-1, keepdim=True) + eps).sqrt()
        xh = d * r
        self.y = xh * w + b
        self.size = (xh * w).norm().item() + b.expand(h.shape).norm().item()
        if dy is None:
            return
        u = w * dy
        self.dx = r * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))
        self.dx_size = (r * u).norm().item()
        if dh is not None:
            self.dx, self.dx_size = self.dx + dh, self.dx_size + dh.norm().item()
        s = [t.reshape(samples, -1, dim).sum(1) for t in (dy * xh, dy)]
        self.dgain, self.dbias = (t.sum(0) for t in s)
        self.curvature = torch.stack([samples * t.square().sum(0) for t in s])


DIMS = [1, 2, 7, 64, 65, 256, 512, 1000, 1263, 2048, 2056, 4096, 5120, 8193, 16385, 33000]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', DIMS)
@pytest.mark.parametrize('residual', [False, True])
def test_forward(dtype, dim, residual):
    for rows in (1, 9):
        x, gain, bias = random((rows, dim), dtype, 0, 1., 0.5), random((dim,), dtype, 1), random((dim,), dtype, 2)
        res = random((rows, dim), dtype, 3, 3.) if residual else None
        for b in (bias, None):
            want = Want(x, res, gain, b)
            if residual:
                got, stream = torchsso.nn.add_layer_norm(x, res, gain, b, EPS)
                assert torch.equal(stream.cpu(), want.h.to(dtype))
            else:
                got = torchsso.nn.layer_norm(x, gain, b, EPS)
            check(got, want.y, dtype, 1e-6, want.size)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', DIMS)
def test_backward(dtype, dim):
    shape = (3, 5, dim)
    x, res = (random(shape, dtype, i, 1., 0.5).requires_grad_() for i in range(2))
    gain, bias = (random((dim,), dtype, 2 + i).requires_grad_() for i in range(2))
    dy, dh = random(shape, dtype, 4), random(shape, dtype, 5)
    curvature = torch.full((2, dim), float('nan'), device='cuda')
    y, h = torchsso.nn.add_layer_norm(x, res, gain, bias, EPS, curvature=curvature)
    dx, dres, dgain, dbias = torch.autograd.grad((y, h), (x, res, gain, bias), (dy, dh))
    want = Want(x, res, gain, bias, dy, dh, 3)
    check(y, want.y, dtype, 1e-6, want.size)
    check(dx, want.dx, dtype, 1e-6, want.dx_size)
    assert torch.equal(dx, dres)
    check(dgain, want.dgain, dtype, 2e-6)
    check(dbias, want.dbias, dtype, 2e-6)
    check(curvature, want.curvature, torch.float32, 4e-6)
    # without a bias
    curvature = torch.full((dim,), float('nan'), device='cuda')
    y, h = torchsso.nn.add_layer_norm(x, res, gain, None, EPS, curvature=curvature)
    other = torch.autograd.grad((y, h), (x, gain), (dy, dh))
    assert torch.equal(other[0], dx)
    check(other[1], want.dgain, dtype, 2e-6)
    check(curvature, want.curvature[0], torch.float32, 4e-6)


@pytest.mark.parametrize('samples,tokens', [(1, 1), (1, 300), (5, 37), (40, 1), (3, 3000), (2, 1025), (17, 129),
                                            (6000, 1), (2000, 3), (15, 7), (16, 64), (33, 100)])
@pytest.mark.parametrize('dim', [40, 71, 1024, 4104])
def test_curvature_of_samples(samples, tokens, dim):
    if samples * tokens * dim > 13000000:
        dim = 71
    x = random((samples, tokens, dim)).requires_grad_()
    gain, bias = (random((dim,), seed=1 + i).requires_grad_() for i in range(2))
    dy = random((samples, tokens, dim), seed=3)
    curvature = torch.empty(2, dim, device='cuda')
    y = torchsso.nn.layer_norm(x, gain, bias, EPS, curvature=curvature)
    dx, dgain, dbias = torch.autograd.grad(y, (x, gain, bias), dy)
    want = Want(x, None, gain, bias, dy, None, samples)
    check(dx, want.dx, torch.float32, 1e-6, want.dx_size)
    check(dgain, want.dgain, torch.float32, 2e-6)
    check(dbias, want.dbias, torch.float32, 2e-6)
    check(curvature[0], want.curvature[0], torch.float32, 4e-6)
    check(curvature[1], want.curvature[1], torch.float32, 4e-6)
    # without the curvature, and with it alone
    y = torchsso.nn.layer_norm(x, gain, bias, EPS)
    others = torch.autograd.grad(y, (x, gain, bias), dy)
    assert torch.equal(others[0], dx)
    check(others[1], want.dgain, torch.float32, 2e-6)
    check(others[2], want.dbias, torch.float32, 2e-6)
    stats = _ops.layer_norm_stats(x.detach(), EPS)
    for alone in (torch.empty(2, dim, device='cuda'), torch.empty(dim, device='cuda')):
        _ops.layer_norm_backward(dy, None, x.detach(), stats, gain.detach(), samples, False, False, False, alone)
        check(alone, want.curvature if alone.dim() == 2 else want.curvature[0], torch.float32, 4e-6)


@pytest.mark.parametrize('dim', [8, 100, 1263, 4096, 33000])
def test_rows_far_off_zero(dim):
    """A mean of a thousand standard deviations.  Each row's mean is a multiple of 2^-24 off where it is kept in one
    number (of 2000 that is 1.2e-4, where the deviation is 2); in two it is not, and neither y nor dx notice."""
    x, dy = random((4, 3, dim), seed=0, scale=2., offset=2000.), random((4, 3, dim), seed=1)
    x = x.requires_grad_()
    gain, bias = random((dim,), seed=2).requires_grad_(), random((dim,), seed=3).requires_grad_()
    y = torchsso.nn.layer_norm(x, gain, bias, EPS)
    dx, dgain, dbias = torch.autograd.grad(y, (x, gain, bias), dy)
    want = Want(x, None, gain, bias, dy, None, 4)
    check(y, want.y, torch.float32, 1e-6, want.size)
    check(dx, want.dx, torch.float32, 1e-6, want.dx_size)
    check(dgain, want.dgain, torch.float32, 2e-6)
    check(dbias, want.dbias, torch.float32, 2e-6)


def test_gradient_against_differences():
    """Directional derivatives of sum(dy * y) + sum(dh * h), by central differences in 64 bits."""
    x, res, gain, bias = (random(s, seed=i) for i, s in enumerate([(2, 3, 50), (2, 3, 50), (50,), (50,)]))
    dy, dh = random((2, 3, 50), seed=4), random((2, 3, 50), seed=5)

    def loss(x, gain, bias):
        h = x + res.cpu().double()
        d = h - h.mean(-1, keepdim=True)
        y = d / (d.square().mean(-1, keepdim=True) + EPS).sqrt() * gain + bias
        return (y * dy.cpu().double()).sum() + (h * dh.cpu().double()).sum()
    a, b, w, c = (t.clone().requires_grad_() for t in (x, res, gain, bias))
    y, h = torchsso.nn.add_layer_norm(a, b, w, c, EPS)
    grads = torch.autograd.grad((y, h), (a, w, c), (dy, dh))
    step = 1e-5
    at = [t.cpu().double() for t in (x, gain, bias)]
    for seed in range(5):
        for k, got in enumerate(grads):
            v = random(got.shape, seed=10 + 3 * seed + k).cpu().double()
            moved = [[t + s * step * v if i == k else t for i, t in enumerate(at)] for s in (1, -1)]
            want = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
            # (300 float32 terms of size one, and 1e-10 of the differences' own curvature)
            assert abs((got.cpu().double() * v).sum() - want) <= 1e-4


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gain_types(dtype):
    x = random((4, 6, 136), dtype).requires_grad_()
    dy = random((4, 6, 136), dtype, 1)
    check(torchsso.nn.layer_norm(x), Want(x, None, None, None).y, dtype, 1e-6)
    dx, = torch.autograd.grad(torchsso.nn.layer_norm(x), x, dy)
    want = Want(x, None, None, None, dy, None, 4)
    check(dx, want.dx, dtype, 1e-6, want.dx_size)
    for of in (dtype, torch.float32):
        gain, bias = (random((136,), of, 2 + i).requires_grad_() for i in range(2))
        y = torchsso.nn.layer_norm(x, gain, bias, EPS)
        want = Want(x, None, gain, bias, dy, None, 4)
        check(y, want.y, dtype, 1e-6, want.size)
        dx, dgain, dbias = torch.autograd.grad(y, (x, gain, bias), dy)
        check(dx, want.dx, dtype, 1e-6, want.dx_size)
        check(dgain, want.dgain, of, 2e-6)
        check(dbias, want.dbias, of, 2e-6)


@pytest.mark.parametrize('needs', ['x', 'gain', 'bias', 'residual', 'x bias', 'gain bias', 'x gain'])
def test_some_of_the_gradients(needs):
    names = ('x', 'residual', 'gain', 'bias')
    tensors = {n: random(s, seed=i) for i, (n, s) in enumerate(zip(names, [(3, 4, 50)] * 2 + [(50,)] * 2))}
    dy, dh = random((3, 4, 50), seed=5), random((3, 4, 50), seed=6)
    want = Want(*tensors.values(), dy, dh, 3)
    wanted = needs.split()
    for n in wanted:
        tensors[n].requires_grad_()
    for squares in (False, True):
        curvature = torch.empty(2, 50, device='cuda') if squares else None
        y, h = torchsso.nn.add_layer_norm(*tensors.values(), EPS, curvature=curvature)
        got = torch.autograd.grad((y, h) if h.requires_grad else y, [tensors[n] for n in wanted],
                                  (dy, dh) if h.requires_grad else dy)
        for n, g in zip(wanted, got):
            if n in ('x', 'residual'):
                check(g, want.dx, torch.float32, 1e-6, want.dx_size)
            else:
                check(g, want.dgain if n == 'gain' else want.dbias, torch.float32, 2e-6)
        if squares:
            check(curvature, want.curvature, torch.float32, 4e-6)


def test_strides():
    base = random((4, 10, 300))
    gain, bias = random((100,), seed=1), random((100,), seed=2)
    for x in (base[..., 100:200], base[..., 1:101], base[:, ::2, :100], base.transpose(0, 1)[..., :100],
              base[0].t()[:100, :10].t(), base[:, :1, :100].expand(4, 10, 100), base[0, 0, :100]):
        x = x.detach().requires_grad_()
        want = Want(x, None, gain, bias)
        check(torchsso.nn.layer_norm(x, gain, bias, EPS), want.y, torch.float32, 1e-6, want.size)
        y, h = torchsso.nn.add_layer_norm(x, x, gain, bias, EPS)
        want = Want(x, x, gain, bias)
        check(y, want.y, torch.float32, 1e-6, want.size)
        # a gradient that is one number spread out, and one with gaps
        for dy in (torch.ones((), device='cuda').expand(y.shape),
                   random(y.shape[:-1] + (200,), seed=3)[..., ::2] if y.dim() > 1 else random((200,), seed=3)[::2]):
            dx, = torch.autograd.grad(torchsso.nn.layer_norm(x, gain, bias, EPS), x, dy)
            want = Want(x, None, gain, bias, dy, None, x.shape[0] if x.dim() > 1 else 1)
            check(dx, want.dx, torch.float32, 1e-6, want.dx_size)


def test_gain_and_bias_off_16_bytes():
    x, base = random((5, 64)), random((200,), seed=1)
    for gain, bias in ((base[1:65], base[64:128]), (base[64:128], base[1:65]), (base[3:67], base[101:165])):
        want = Want(x, None, gain, bias)
        check(torchsso.nn.layer_norm(x, gain, bias, EPS), want.y, torch.float32, 1e-6, want.size)


def test_only_one_of_the_results_is_used():
    x, res = (random((3, 4, 50), seed=i).requires_grad_() for i in range(2))
    gain, bias, d = random((50,), seed=2).requires_grad_(), random((50,), seed=3).requires_grad_(), random((3, 4, 50), seed=4)
    curvature = torch.ones(2, 50, device='cuda')
    y, h = torchsso.nn.add_layer_norm(x, res, gain, bias, EPS, curvature=curvature)
    dx, dres, dgain, dbias = torch.autograd.grad(h, (x, res, gain, bias), d, allow_unused=True)
    assert torch.equal(dx, d) and torch.equal(dres, d) and dgain is None and dbias is None
    assert torch.equal(curvature, torch.zeros_like(curvature))
    y, h = torchsso.nn.add_layer_norm(x, res, gain, bias, EPS)
    dx, = torch.autograd.grad(y, x, d)
    want = Want(x, res, gain, bias, d, None, 3)
    check(dx, want.dx, torch.float32, 1e-6, want.dx_size)


def test_the_same_tensor_twice():
    x, gain = random((4, 3, 100)).requires_grad_(), random((100,), seed=1).requires_grad_()
    dy, dh = random((4, 3, 100), seed=2), random((4, 3, 100), seed=3)
    y, h = torchsso.nn.add_layer_norm(x, x, gain, gain, EPS)
    dx, dgain = torch.autograd.grad((y, h), (x, gain), (dy, dh))
    want = Want(x, x, gain, gain, dy, dh, 4)
    check(dx, 2 * want.dx, torch.float32, 1e-6, 2 * want.dx_size)
    check(dgain, want.dgain + want.dbias, torch.float32, 2e-6, want.dgain.norm().item() + want.dbias.norm().item())


@pytest.mark.parametrize('norm', ['layer_norm', 'rms_norm'])
def test_views_whose_sign_is_still_to_be_applied(norm):
    gen = torch.Generator().manual_seed(0)
    one, two, three = [torch.complex(*torch.randn(2, 6, 40, generator=gen)).cuda().conj().imag for _ in range(3)]
    assert one.is_neg() and two.is_neg()
    gain = torch.rand(40, generator=gen).cuda()
    results = []
    for x, r, dy in ((one, two, three), (one.resolve_neg(), two.resolve_neg(), three.resolve_neg())):
        x, r = x.detach().requires_grad_(), r.detach().requires_grad_()
        y, h = getattr(torchsso.nn, 'add_' + norm)(x, r, gain)
        results.append([y, h] + list(torch.autograd.grad([y, h], [x, r], [dy, dy])))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    with pytest.raises(_hip.KfacHipError):
        getattr(torchsso.nn, norm)(one, torch._neg_view(gain))
    backward = getattr(_ops, norm + '_backward')
    kept = (lambda x: _ops.layer_norm_stats(x, 1e-5)) if norm == 'layer_norm' else lambda x: None
    for a, b in zip(*[backward(dy, dy, x, *((kept(x), gain, 2) if norm == 'layer_norm' else (gain, 1e-5, 2)))
                      for x, dy in ((one, three), (one.resolve_neg(), three.resolve_neg()))]):
        assert torch.equal(a, b)


def test_empty():
    gain, bias = (random((50,), seed=i).requires_grad_() for i in range(2))
    x = torch.zeros(0, 4, 50, device='cuda', requires_grad=True)
    curvature = torch.ones(2, 50, device='cuda')
    y = torchsso.nn.layer_norm(x, gain, bias, EPS, curvature=curvature)
    assert y.shape == x.shape
    dx, dgain, dbias = torch.autograd.grad(y, (x, gain, bias), torch.zeros_like(y))
    assert dx.shape == x.shape
    for t in (dgain, dbias, curvature):
        assert torch.equal(t, torch.zeros_like(t))
    q, scale = torchsso.nn.layer_norm(x.detach(), out_dtype=EIGHT)
    assert q.shape == x.shape and scale.shape == (0, 4, 1)


def test_constant_rows_and_rows_that_are_not_finite_stay_by_themselves():
    x, gain, bias, dy = random((7, 500)), random((500,), seed=1), random((500,), seed=2), random((7, 500), seed=3)

    def passes(x):
        x = x.clone().requires_grad_()
        y = torchsso.nn.layer_norm(x, gain, bias, EPS)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]
    clean = passes(x)
    x[1] = 0
    x[2, 7] = float('nan')
    x[4, 9] = float('inf')
    x[6] = 3.7
    y, dx = passes(x)
    for i in (0, 3, 5):
        assert torch.equal(y[i], clean[0][i]) and torch.equal(dx[i], clean[1][i])
    # (a mean of equal numbers is at most 2^-24 of them off, and e takes that: y is the bias, but for rounding)
    assert torch.equal(y[1], bias) and bool(((y[6] - bias).abs() <= 1e-4).all())
    assert torch.isfinite(dx[[1, 6]]).all()
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all() and torch.isnan(dx[2]).all() and torch.isnan(dx[4]).all()
    q, scale = torchsso.nn.layer_norm(x, None, None, EPS, out_dtype=EIGHT)
    assert scale[1] == 1 and torch.equal(q[1].float(), torch.zeros_like(y[1]))
    assert torch.isnan(q[2].float()).all() and torch.isfinite(q[[0, 1, 3, 5]].float()).all()


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', [1, 7, 64, 1263, 4096, 5120, 16385, 33000])
def test_eight_bits(dtype, dim):
    for rows in (1, 7):
        x, res = random((rows, dim), dtype), random((rows, dim), dtype, 1)
        gain, bias = random((dim,), dtype, 2), random((dim,), dtype, 3)
        want = Want(x, res, gain, bias)
        q, scale, stream = torchsso.nn.add_layer_norm(x, res, gain, bias, EPS, out_dtype=EIGHT)
        assert q.dtype == EIGHT and q.shape == x.shape and scale.shape == (rows, 1)
        assert torch.equal(stream.cpu(), want.h.to(dtype))
        top = want.y.abs().amax(-1, keepdim=True)
        check(scale, torch.where(top > 0, top / 448, torch.ones_like(top)), torch.float32, 1e-6)
        got = q.cpu().float().double() * scale.cpu().double()
        # three bits behind the leading one: half a unit is 2^-4 of an element, or 2^-10 (of 448) where
        # that is less than the smallest normal number; and 1e-6 of the row's largest that y may be off
        bound = torch.maximum(want.y.abs() * 2 ** -4, scale.cpu().double() * 2 ** -10) * (1 + 1e-4) + 1e-5 * top
        assert bool(((got - want.y).abs() <= bound).all())


@pytest.mark.parametrize('dim', [1000, 33000])
@pytest.mark.parametrize('size', [1e-30, 1e-37, 1e-42, 1e30])
def test_eight_bits_of_small_and_large_results(dim, size):
    x, gain = random((3, dim)), torch.full((dim,), size, device='cuda')
    want = Want(x, None, gain, None)
    q, scale = torchsso.nn.layer_norm(x, gain, None, EPS, out_dtype=EIGHT)
    assert bool((scale >= 2. ** -120).all()) and torch.isfinite(q.float()).all()
    got = q.cpu().float().double() * scale.cpu().double()
    # (half a unit of an element, or of the smallest numbers, and of y the half of float32's smallest step)
    bound = torch.maximum(want.y.abs() * 2 ** -4, scale.cpu().double() * 2 ** -10) * (1 + 1e-4) + 2. ** -149
    assert bool(((got - want.y).abs() <= bound).all())


def test_in_a_recorded_graph_and_on_another_stream():
    x, res, gain, bias, dy = (random(s, seed=i) for i, s in enumerate([(6, 20, 300), (6, 20, 300), (300,), (300,), (6, 20, 300)]))

    def work():
        a, b, w, c = (t.detach().requires_grad_() for t in (x, res, gain, bias))
        curvature = torch.empty(2, 300, device='cuda')
        y, h = torchsso.nn.add_layer_norm(a, b, w, c, EPS, curvature=curvature)
        return (y.detach(), h.detach()) + torch.autograd.grad(y, (a, w, c), dy) + (curvature,)
    eager = [t.clone() for t in work()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.clone() for t in work()]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        recorded = work()
    for seed in range(3):
        x.copy_(random((6, 20, 300), seed=30 + seed))
        graph.replay()
        got = [t.clone() for t in recorded]
        for a, b in zip(got, work()):
            assert torch.equal(a, b)


@pytest.mark.parametrize('norm', ['layer_norm', 'rms_norm'])
def test_recording_while_an_eager_graph_of_the_leaves_lives_is_refused(norm):
    x, gain, dy = random((6, 20, 300)), random((300,), seed=1), random((6, 20, 300), seed=2)
    gain.requires_grad_()

    def work():
        y = getattr(torchsso.nn, norm)(x, gain)
        return torch.autograd.grad(y, gain, dy)[0]
    eager = getattr(torchsso.nn, norm)(x, gain)
    side = torch.cuda.Stream()
    with pytest.raises(RuntimeError, match='cannot be recorded'):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            work()
    assert torch.equal(eager, getattr(torchsso.nn, norm)(x, gain).detach())
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        recorded = work()
    for seed in range(3):
        x.copy_(random((6, 20, 300), seed=30 + seed))
        graph.replay()
        got = recorded.clone()
        assert torch.equal(got, work())


@pytest.mark.parametrize('norm', ['layer_norm', 'rms_norm'])
@pytest.mark.parametrize('ask', ['input', 'gain'])
def test_recording_while_an_eager_graph_of_leaves_that_get_nothing_lives(norm, ask):
    """... of the gain, where the gradient of the input alone is asked for, and the other way round"""
    x, gain, dy = random((6, 20, 300)), random((300,), seed=1), random((6, 20, 300), seed=2)
    other = (gain if ask == 'input' else x).requires_grad_()

    def work():
        leaf = (x if ask == 'input' else gain).detach().requires_grad_()
        y = getattr(torchsso.nn, norm)(*((leaf, gain) if ask == 'input' else (x, leaf)))
        return torch.autograd.grad(y, leaf, dy)[0]
    eager = getattr(torchsso.nn, norm)(x, gain)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        recorded = work()
    for seed in range(3):
        with torch.no_grad():
            dy.copy_(random((6, 20, 300), seed=30 + seed))
        graph.replay()
        got = recorded.clone()
        assert torch.equal(got, work())
    # (the graph from outside is whole)
    assert torch.autograd.grad(eager, other, dy)[0].shape == other.shape


def test_two_threads_at_once():
    inputs = [[random((7, 33, 1024), seed=2 * i + k) for k in range(2)] for i in range(2)]

    def work(x, dy):
        x, gain, bias = x.detach().requires_grad_(), torch.ones(1024, device='cuda', requires_grad=True), \
            torch.zeros(1024, device='cuda', requires_grad=True)
        curvature = torch.empty(2, 1024, device='cuda')
        y = torchsso.nn.layer_norm(x, gain, bias, EPS, curvature=curvature)
        return torch.autograd.grad(y, (x, gain, bias), dy) + (y.detach(), curvature)
    want = [work(*i) for i in inputs]
    torch.cuda.synchronize()
    got = [None, None]

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k] = work(*inputs[k])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for w, g in zip(want, got):
        for a, b in zip(w, g):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------
# modules and curvature
# ---------------------------------------------------------------------------------------

KINDS = pytest.mark.parametrize('kind', [torchsso.nn.LayerNorm, torch.nn.LayerNorm], ids=['torchsso', 'torch'])


@KINDS
@pytest.mark.parametrize('bias', [True, False])
def test_curvature_class(kind, bias):
    module = kind(60, eps=EPS, bias=bias).cuda()
    with torch.no_grad():
        module.weight.normal_()
        if bias:
            module.bias.normal_()
    curv = torchsso.DiagCovLayerNorm(module, ema_decay=1., damping=1e-3)
    x = random((5, 7, 60)).requires_grad_()
    dy = random((5, 7, 60), seed=1)
    module(x).backward(dy)
    want = Want(x, None, module.weight, module.bias, dy, None, 5)
    assert len(curv.data) == (2 if bias else 1)
    for k, t in enumerate(curv.data):
        check(t, want.curvature[k], torch.float32, 4e-6)
    # (torch's own gradient is a sum of 35 terms in float32 as well)
    check(module.weight.grad, want.dgain, torch.float32, 2e-6)
    curv.step()
    for k, t in enumerate(curv.inv):
        check(t, 1 / (want.curvature[k] + 1e-3), torch.float32, 1e-5)


def test_module_with_residual():
    module = torchsso.nn.LayerNorm(60, eps=EPS).cuda()
    curv = torchsso.DiagCovLayerNorm(module)
    x, res = random((5, 60)).requires_grad_(), random((5, 60), seed=1)
    y, h = module(x, res)
    dy, dh = random((5, 60), seed=2), random((5, 60), seed=3)
    torch.autograd.backward((y, h), (dy, dh))
    want = Want(x, res, module.weight, module.bias, dy, dh, 5)
    check(x.grad, want.dx, torch.float32, 1e-6, want.dx_size)
    for k in range(2):
        check(curv.data[k], want.curvature[k], torch.float32, 4e-6)
    with torch.no_grad():
        module(x, res)                        # (leaves the curvature alone)
    check(curv.data[0], want.curvature[0], torch.float32, 4e-6)


@KINDS
def test_second_order_optimizer(kind):
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(20, 30), kind(30), torch.nn.Tanh(), torch.nn.Linear(30, 4)).cuda()
    x, y = torch.randn(64, 20, device='cuda'), torch.randint(0, 4, (64,), device='cuda')
    opt = torchsso.optim.SecondOrderOptimizer(model, 'Cov', {'Linear': 'Kron', 'LayerNorm': 'Diag'},
                                              {'damping': 1e-2, 'ema_decay': 0.9}, lr=0.02, momentum=0.9)
    before = [p.detach().clone() for p in model[1].parameters()]

    def closure():
        opt.zero_grad()
        out = model(x)
        loss = torch.nn.functional.cross_entropy(out, y)
        loss.backward()
        return loss, out
    for _ in range(3):
        loss, _ = opt.step(closure=closure)
        assert torch.isfinite(loss)
    for p, b in zip(model[1].parameters(), before):
        assert torch.isfinite(p).all() and not torch.equal(p, b)
    # the last update of the norm's parameters: preconditioned by the inverse of the damped average
    group = opt.param_groups[1]
    for ema, inv in zip(group['curv'].ema, group['curv'].inv):
        check(inv, 1 / (ema.cpu().double() + 1e-2), torch.float32, 1e-6)


def test_refusals():
    x, w = random((4, 50)), random((50,))
    for bad in (lambda: torchsso.nn.layer_norm(x.double(), w, w), lambda: torchsso.nn.layer_norm(x, w[:49], w[:49]),
                lambda: torchsso.nn.layer_norm(x, w.bfloat16(), w.bfloat16()), lambda: torchsso.nn.layer_norm(x, w.cpu(), w.cpu()),
                lambda: torchsso.nn.layer_norm(x, w, w[:49]), lambda: torchsso.nn.layer_norm(x, w, w.cpu()),
                lambda: torchsso.nn.layer_norm(x.bfloat16(), w, w.bfloat16()), lambda: torchsso.nn.layer_norm(x, w, w.bfloat16()),
                lambda: torchsso.nn.layer_norm(x, w.expand(2, 50)[:, ::2].reshape(-1), w.repeat(2)[::2]),
                lambda: torchsso.nn.layer_norm(x.cpu(), w.cpu(), w.cpu()), lambda: torchsso.nn.add_layer_norm(x, x[:3], w, w),
                lambda: torchsso.nn.add_layer_norm(x, x.bfloat16(), w, w), lambda: torchsso.nn.layer_norm(x[:, :0], w[:0], w[:0]),
                lambda: torchsso.nn.layer_norm(x, w, w, curvature=torch.zeros(50, device='cuda')),
                lambda: torchsso.nn.layer_norm(x, w, curvature=torch.zeros(2, 50, device='cuda')),
                lambda: torchsso.nn.layer_norm(x, w, w, curvature=torch.zeros(50, 2, device='cuda').t()),
                lambda: _ops.layer_norm_backward(x, None, x, torch.zeros(4, 3, device='cuda'), w, 3),
                lambda: _ops.layer_norm_backward(x, None, x, torch.zeros(3, 3, device='cuda'), w, 2),
                lambda: _ops.layer_norm_backward(x, None, x, torch.zeros(4, 3, device='cuda'), w, 2,
                                                 curvature=torch.zeros(50, device='cuda'))):
        with pytest.raises(_hip.KfacHipError):
            bad()
    a = x.clone().requires_grad_()
    y = torchsso.nn.layer_norm(a, w, w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, a, torch.ones_like(y), create_graph=True)


@pytest.mark.parametrize('which', [0, 1, 2, 3])
def test_forward_mode_is_refused(which):
    args = [random((4, 50)), random((4, 50), seed=1), random((50,), seed=2), random((50,), seed=3)]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError):
            torchsso.nn.add_layer_norm(*args)
        with pytest.raises(RuntimeError):
            torchsso.nn.add_layer_norm(*args, out_dtype=EIGHT)


def test_saved_tensors_that_were_changed_are_refused():
    x, gain = random((4, 50)).requires_grad_(), random((50,), seed=1).requires_grad_()
    y, h = torchsso.nn.add_layer_norm(x, x.detach(), gain)
    with torch.no_grad():
        h.add_(1)
    with pytest.raises(RuntimeError, match='inplace'):
        torch.autograd.grad(y, x, torch.ones_like(y))


def test_more_elements_than_32_bits_count():
    rows, dim = (1 << 18) + 3, 8192
    x = torch.empty(rows, dim, device='cuda', dtype=torch.bfloat16).normal_().requires_grad_()
    gain, bias = torch.linspace(0.5, 2., dim, device='cuda'), torch.linspace(-1., 1., dim, device='cuda')
    y = torchsso.nn.layer_norm(x, gain, bias)
    dx, = torch.autograd.grad(y, x, x.detach())
    for part in (slice(0, 2), slice(rows // 2, rows // 2 + 2), slice(rows - 2, rows)):
        xs = x.detach()[part].clone().requires_grad_()
        ys = torchsso.nn.layer_norm(xs, gain, bias)
        assert torch.equal(y[part], ys)
        assert torch.equal(dx[part], torch.autograd.grad(ys, xs, xs.detach())[0])


def test_more_rows_than_a_launch_has_threads_for():
    rows, dim = (1 << 26) + 5, 8
    gen = torch.Generator(device='cuda').manual_seed(0)
    x, res = (torch.empty(rows, dim, device='cuda', dtype=torch.bfloat16).normal_(generator=gen) for _ in range(2))
    gain, bias = torch.linspace(0.5, 2., dim, device='cuda'), torch.linspace(-1., 1., dim, device='cuda')
    y, h = torchsso.nn.add_layer_norm(x, res, gain, bias)
    q, scale, stream = torchsso.nn.add_layer_norm(x, res, gain, bias, out_dtype=EIGHT)
    stats = _ops.layer_norm_stats(h, EPS)
    for part in (slice(0, 3), slice((1 << 25) - 2, (1 << 25) + 2), slice(rows - 3, rows)):
        few_y, few_h = torchsso.nn.add_layer_norm(x[part], res[part], gain, bias)
        few_q, few_scale, _ = torchsso.nn.add_layer_norm(x[part], res[part], gain, bias, out_dtype=EIGHT)
        assert torch.equal(y[part], few_y) and torch.equal(h[part], few_h) and torch.equal(stream[part], few_h)
        assert torch.equal(q[part].view(torch.uint8), few_q.view(torch.uint8)) and torch.equal(scale[part], few_scale)
        assert torch.equal(stats[part], _ops.layer_norm_stats(few_h, EPS))


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', [96, 1000, 5120])
def test_streams_beyond_the_caches_give_what_a_few_rows_give(dtype, dim):
    rows = (1 << 28) // (dim * 4) + 7           # (every tensor of them: 128 MiB or more)
    gen = torch.Generator(device='cuda').manual_seed(dim)
    x, res, dy, dh = (torch.empty(rows, dim, device='cuda', dtype=dtype).normal_(generator=gen) for _ in range(4))
    gain, bias = torch.linspace(0.5, 2., dim, device='cuda'), torch.linspace(-1., 1., dim, device='cuda')

    def passes(x, res, dy, dh):
        x, res = x.clone().requires_grad_(), res.clone().requires_grad_()
        y, h = torchsso.nn.add_layer_norm(x, res, gain, bias)
        with torch.no_grad():
            eight = torchsso.nn.add_layer_norm(x, res, gain, bias, out_dtype=EIGHT)
        return (y, h) + torch.autograd.grad((y, h), (x, res), (dy, dh)) + (eight[0].view(torch.uint8), eight[1], eight[2])

    whole = passes(x, res, dy, dh)
    for part in (slice(0, 3), slice(rows // 2, rows // 2 + 3), slice(rows - 3, rows)):
        few = passes(x[part], res[part], dy[part], dh[part])
        for a, b in zip(whole, few):
            assert torch.equal(a[part], b)
