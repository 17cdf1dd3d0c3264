"""torchsso.nn.rms_norm / add_rms_norm / RMSNorm and DiagCovRMSNorm against the formulas in 64 bits.

Tolerances (2-norm of the difference over that of what is compared with).  Everything is computed in
float32 and rounded once, so a result may be as far from the exact one as the exact one's own rounding
to its type, 5 % more for elements that round the other way, and what float32 loses: a root, a mean
of squares and at most six products of 2^-24 each, 1e-6.  The sums over rows are random walks of such
terms, 2e-6 (their squares 4e-6).  dx is a difference, and is compared in units of its terms.
"""
import pytest
import torch

import torchsso
from torchsso import _hip, _ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-6


def random(shape, dtype=torch.float32, seed=0, scale=1.):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype).cuda()


def check(got, want, dtype, more, scale=None):
    """`got` (of `dtype`) is as near to `want` (float64) as float32 arithmetic and one rounding allow."""
    assert got.dtype == dtype and got.shape == want.shape
    got = got.detach().cpu().double()
    rounding = (want.to(dtype).double() - want).norm().item()
    size = want.norm().item() if scale is None else scale
    error = (got - want).norm().item()
    assert error <= 1.05 * rounding + more * size, (error / max(size, 1e-300), rounding / max(size, 1e-300))


def reference(x, residual, gain, dy=None, dh=None, samples=1, eps=EPS):
    """(y, h, dx, dgain, curvature, scale of dx) in 64 bits, from tensors anywhere"""
    dtype = x.dtype
    to = lambda t: None if t is None else t.detach().cpu().double()
    x, residual, gain, dy, dh = map(to, (x, residual, gain, dy, dh))
    h = x if residual is None else (x + residual).to(dtype).double()
    dim = h.shape[-1]
    w = torch.ones(dim, dtype=torch.float64) if gain is None else gain
    r = 1 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    y = h * r * w
    if dy is None:
        return y, h
    dx = r * (w * dy - h * r * r * (w * dy * h).mean(-1, keepdim=True))
    scale = (r * w * dy).norm().item()
    if dh is not None:
        dx, scale = dx + dh, scale + dh.norm().item()
    s = (dy * h * r).reshape(samples, -1, dim).sum(1)
    return y, h, dx, s.sum(0), samples * s.square().sum(0), scale


DIMS = [1, 2, 7, 64, 65, 256, 512, 1000, 1263, 2048, 2056, 4096, 5120, 8193, 16385, 33000]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', DIMS)
@pytest.mark.parametrize('residual', [False, True])
def test_forward(dtype, dim, residual):
    for rows in (1, 9):
        x, gain = random((rows, dim), dtype), random((dim,), dtype, 1)
        res = random((rows, dim), dtype, 2, 3.) if residual else None
        y, h = reference(x, res, gain)
        if residual:
            got, stream = torchsso.nn.add_rms_norm(x, res, gain, EPS)
            assert torch.equal(stream.cpu(), h.to(dtype))
        else:
            got = torchsso.nn.rms_norm(x, gain, EPS)
        check(got, y, dtype, 1e-6)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', DIMS)
def test_backward(dtype, dim):
    shape = (3, 5, dim)
    x, res = (random(shape, dtype, i).requires_grad_() for i in range(2))
    gain = random((dim,), dtype, 2).requires_grad_()
    dy, dh = random(shape, dtype, 3), random(shape, dtype, 4)
    curvature = torch.full((dim,), float('nan'), device='cuda')
    y, h = torchsso.nn.add_rms_norm(x, res, gain, EPS, curvature=curvature)
    dx, dres, dgain = torch.autograd.grad((y, h), (x, res, gain), (dy, dh))
    _, _, wx, wg, wc, scale = reference(x, res, gain, dy, dh, 3)
    check(dx, wx, dtype, 1e-6, scale)
    assert torch.equal(dx, dres)
    check(dgain, wg, dtype, 2e-6)
    check(curvature, wc, torch.float32, 4e-6)


@pytest.mark.parametrize('samples,tokens', [(1, 1), (1, 300), (5, 37), (40, 1), (3, 3000), (2, 1025), (17, 129),
                                            (6000, 1), (2000, 3), (15, 7), (16, 64), (33, 100)])
@pytest.mark.parametrize('dim', [40, 71, 1024, 4104])
def test_curvature_of_samples(samples, tokens, dim):
    if samples * tokens * dim > 13000000:
        dim = 71
    x = random((samples, tokens, dim)).requires_grad_()
    gain, dy = random((dim,), seed=1).requires_grad_(), random((samples, tokens, dim), seed=2)
    curvature = torch.empty(dim, device='cuda')
    y = torchsso.nn.rms_norm(x, gain, EPS, curvature=curvature)
    dx, dgain = torch.autograd.grad(y, (x, gain), dy)
    _, _, wx, wg, wc, scale = reference(x, None, gain, dy, None, samples)
    check(dx, wx, torch.float32, 1e-6, scale)
    check(dgain, wg, torch.float32, 2e-6)
    check(curvature, wc, torch.float32, 4e-6)
    # without the curvature, and with it alone
    y = torchsso.nn.rms_norm(x, gain, EPS)
    other_dx, other = torch.autograd.grad(y, (x, gain), dy)
    assert torch.equal(other_dx, dx)
    check(other, wg, torch.float32, 2e-6)
    alone = torch.empty(dim, device='cuda')
    _ops.rms_norm_backward(dy, None, x.detach(), gain.detach(), EPS, samples, False, False, alone)
    check(alone, wc, torch.float32, 4e-6)


def test_gradient_against_differences():
    """Directional derivatives of sum(dy * y) + sum(dh * h), by central differences in 64 bits."""
    x, res, gain = random((2, 3, 50)), random((2, 3, 50), seed=1), random((50,), seed=2)
    dy, dh = random((2, 3, 50), seed=3), random((2, 3, 50), seed=4)

    def loss(x, gain):
        h = x + res.cpu().double()
        y = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * gain
        return (y * dy.cpu().double()).sum() + (h * dh.cpu().double()).sum()
    a, b, w = (t.clone().requires_grad_() for t in (x, res, gain))
    y, h = torchsso.nn.add_rms_norm(a, b, w, EPS)
    dx, dres, dgain = torch.autograd.grad((y, h), (a, b, w), (dy, dh))
    step = 1e-5
    for seed in range(5):
        v, u = random((2, 3, 50), seed=10 + seed).cpu().double(), random((50,), seed=20 + seed).cpu().double()
        x64, w64 = x.cpu().double(), gain.cpu().double()
        for got, want in (((dx.cpu().double() * v).sum(), (loss(x64 + step * v, w64) - loss(x64 - step * v, w64))),
                          ((dgain.cpu().double() * u).sum(), (loss(x64, w64 + step * u) - loss(x64, w64 - step * u)))):
            # (300 float32 terms of size one, and 1e-10 of the differences' own curvature)
            assert abs(got - want / (2 * step)) <= 1e-4


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gain_types(dtype):
    x = random((4, 6, 136), dtype).requires_grad_()
    dy = random((4, 6, 136), dtype, 1)
    for gain in (None, random((136,), dtype, 2).requires_grad_(), random((136,), torch.float32, 2).requires_grad_()):
        y = torchsso.nn.rms_norm(x, gain, EPS)
        want = reference(x, None, gain, dy, None, 4)
        check(y, want[0], dtype, 1e-6)
        grads = torch.autograd.grad(y, (x,) if gain is None else (x, gain), dy)
        check(grads[0], want[2], dtype, 1e-6, want[5])
        if gain is not None:
            check(grads[1], want[3], gain.dtype, 2e-6)


def test_strides():
    base = random((4, 10, 300))
    gain = random((100,), seed=1)
    for x in (base[..., 100:200], base[..., 1:101], base[:, ::2, :100], base.transpose(0, 1)[..., :100],
              base[0].t()[:100, :10].t(), base[:, :1, :100].expand(4, 10, 100), base[0, 0, :100]):
        x = x.detach().requires_grad_()
        check(torchsso.nn.rms_norm(x, gain, EPS), reference(x, None, gain)[0], torch.float32, 1e-6)
        y, h = torchsso.nn.add_rms_norm(x, x, gain, EPS)
        check(y, reference(x, x, gain)[0], torch.float32, 1e-6)
        # a gradient that is one number spread out, and one with gaps
        for dy in (torch.ones((), device='cuda').expand(y.shape),
                   random(y.shape[:-1] + (200,), seed=3)[..., ::2] if y.dim() > 1 else random((200,), seed=3)[::2]):
            dx, = torch.autograd.grad(torchsso.nn.rms_norm(x, gain, EPS), x, dy)
            want = reference(x, None, gain, dy, None, x.shape[0] if x.dim() > 1 else 1)
            check(dx, want[2], torch.float32, 1e-6, want[5])


def test_only_one_of_the_results_is_used():
    x, res = (random((3, 4, 50), seed=i).requires_grad_() for i in range(2))
    gain, d = random((50,), seed=2).requires_grad_(), random((3, 4, 50), seed=3)
    curvature = torch.ones(50, device='cuda')
    y, h = torchsso.nn.add_rms_norm(x, res, gain, EPS, curvature=curvature)
    dx, dres, dgain = torch.autograd.grad(h, (x, res, gain), d, allow_unused=True)
    assert torch.equal(dx, d) and torch.equal(dres, d) and dgain is None
    assert torch.equal(curvature, torch.zeros_like(curvature))
    y, h = torchsso.nn.add_rms_norm(x, res, gain, EPS)
    dx, = torch.autograd.grad(y, x, d)
    want = reference(x, res, gain, d, None, 3)
    check(dx, want[2], torch.float32, 1e-6, want[5])
    y, h = torchsso.nn.add_rms_norm(x.detach(), res.detach(), gain, EPS)
    dgain, = torch.autograd.grad(y, gain, d)
    check(dgain, want[3], torch.float32, 2e-6)


def test_empty():
    gain = random((50,)).requires_grad_()
    x = torch.zeros(0, 4, 50, device='cuda', requires_grad=True)
    y = torchsso.nn.rms_norm(x, gain, EPS)
    assert y.shape == x.shape
    dx, dgain = torch.autograd.grad(y, (x, gain), torch.zeros_like(y))
    assert dx.shape == x.shape and torch.equal(dgain, torch.zeros_like(gain))


def test_rows_that_are_zero_or_not_finite_stay_by_themselves():
    x, gain = random((6, 500)), random((500,), seed=1)
    clean = torchsso.nn.rms_norm(x, gain, EPS)
    x[1] = 0
    x[2, 7] = float('nan')
    x[4, 9] = float('inf')
    y = torchsso.nn.rms_norm(x, gain, EPS)
    for i in (0, 3, 5):
        assert torch.equal(y[i], clean[i])
    assert torch.equal(y[1], torch.zeros_like(y[1])) and torch.isnan(y[2]).all() and torch.isnan(y[4, 9])
    q, scale = torchsso.nn.rms_norm(x, gain, EPS, out_dtype=torch.float8_e4m3fn)
    assert scale[1] == 1 and torch.equal(q[1].float(), torch.zeros_like(y[1]))
    assert torch.isnan(q[2].float()).all() and torch.isfinite(q[[0, 1, 3, 5]].float()).all()


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', [1, 7, 64, 1263, 4096, 5120, 16385, 33000])
def test_eight_bits(dtype, dim):
    for rows in (1, 7):
        x, res, gain = random((rows, dim), dtype), random((rows, dim), dtype, 1), random((dim,), dtype, 2)
        y, h = reference(x, res, gain)
        q, scale, stream = torchsso.nn.add_rms_norm(x, res, gain, EPS, out_dtype=torch.float8_e4m3fn)
        assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (rows, 1)
        assert torch.equal(stream.cpu(), h.to(dtype))
        check(scale, y.abs().amax(-1, keepdim=True) / 448, torch.float32, 1e-6)
        got = q.cpu().float().double() * scale.cpu().double()
        # three bits behind the leading one: half a unit is 2^-4 of an element, or 2^-10 (of 448) where
        # that is less than the smallest normal number
        bound = torch.maximum(y.abs() * 2 ** -4, scale.cpu().double() * 2 ** -10) * (1 + 1e-4)
        assert bool(((got - y).abs() <= bound).all())


def test_in_a_recorded_graph_and_on_another_stream():
    x, res, gain, dy = (random(s, seed=i) for i, s in enumerate([(6, 20, 300), (6, 20, 300), (300,), (6, 20, 300)]))
    curvature = torch.empty(300, device='cuda')

    def work():
        y, h, _ = _ops.rms_norm(x, res, gain, EPS)
        dx, dgain = _ops.rms_norm_backward(dy, None, h, gain, EPS, 6, curvature=curvature)
        return y, h, dx, dgain, curvature
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


# ---------------------------------------------------------------------------------------
# modules and curvature
# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize('kind', [torchsso.nn.RMSNorm, torch.nn.RMSNorm], ids=['torchsso', 'torch'])
def test_curvature_class(kind):
    module = kind(60, eps=EPS).cuda()
    with torch.no_grad():
        module.weight.normal_()
    curv = torchsso.DiagCovRMSNorm(module, ema_decay=1., damping=1e-3)
    x = random((5, 7, 60)).requires_grad_()
    dy = random((5, 7, 60), seed=1)
    module(x).backward(dy)
    want = reference(x, None, module.weight, dy, None, 5)
    check(curv.data[0], want[4], torch.float32, 4e-6)
    check(module.weight.grad, want[3], torch.float32, 2e-6)
    curv.step()
    check(curv.inv[0], 1 / (want[4] + 1e-3), torch.float32, 1e-5)


def test_module_with_residual():
    module = torchsso.nn.RMSNorm(60, eps=EPS).cuda()
    curv = torchsso.DiagCovRMSNorm(module)
    x, res = random((5, 60)).requires_grad_(), random((5, 60), seed=1)
    y, h = module(x, res)
    dy, dh = random((5, 60), seed=2), random((5, 60), seed=3)
    torch.autograd.backward((y, h), (dy, dh))
    want = reference(x, res, module.weight, dy, dh, 5)
    check(x.grad, want[2], torch.float32, 1e-6, want[5])
    check(curv.data[0], want[4], torch.float32, 4e-6)
    with torch.no_grad():
        module(x, res)                        # (leaves the curvature alone)
    check(curv.data[0], want[4], torch.float32, 4e-6)


@pytest.mark.parametrize('kind', [torchsso.nn.RMSNorm, torch.nn.RMSNorm], ids=['torchsso', 'torch'])
def test_second_order_optimizer(kind):
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(20, 30), kind(30, eps=EPS), torch.nn.Tanh(), torch.nn.Linear(30, 4)).cuda()
    x, y = torch.randn(64, 20, device='cuda'), torch.randint(0, 4, (64,), device='cuda')
    opt = torchsso.optim.SecondOrderOptimizer(model, 'Cov', {'Linear': 'Kron', 'RMSNorm': 'Diag'},
                                              {'damping': 1e-2, 'ema_decay': 0.9}, lr=0.02, momentum=0.9)

    def closure():
        opt.zero_grad()
        out = model(x)
        loss = torch.nn.functional.cross_entropy(out, y)
        loss.backward()
        return loss, out
    losses = [opt.step(closure=closure)[0].item() for _ in range(20)]
    assert losses[-1] < 0.5 * losses[0]


def test_refusals():
    x, gain = random((4, 50)), random((50,))
    with pytest.raises(ValueError):
        torchsso.nn.rms_norm(x, gain, -1.)
    with pytest.raises(ValueError):
        torchsso.nn.rms_norm(x, None, EPS, curvature=torch.zeros(50, device='cuda'))
    with pytest.raises(ValueError):
        torchsso.nn.rms_norm(x, gain, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        torchsso.nn.rms_norm(x, gain.clone().requires_grad_(), out_dtype=torch.float8_e4m3fn)
    for bad in (lambda: torchsso.nn.rms_norm(x.double(), gain), lambda: torchsso.nn.rms_norm(x, gain[:49]),
                lambda: torchsso.nn.rms_norm(x, gain.bfloat16()), lambda: torchsso.nn.rms_norm(x, gain.cpu()),
                lambda: torchsso.nn.rms_norm(x.cpu(), gain.cpu()), lambda: torchsso.nn.add_rms_norm(x, x[:3], gain),
                lambda: torchsso.nn.add_rms_norm(x, x.bfloat16(), gain), lambda: torchsso.nn.rms_norm(x[:, :0], gain[:0]),
                lambda: _ops.rms_norm_backward(x, None, x, gain, EPS, 3)):
        with pytest.raises(_hip.KfacHipError):
            bad()
    with pytest.raises(_hip.KfacHipError):
        w = gain.clone().requires_grad_()
        torchsso.nn.rms_norm(x, w, curvature=torch.zeros(49, device='cuda')).sum().backward()
    with pytest.raises(TypeError):
        torchsso.DiagCovRMSNorm(torch.nn.LayerNorm(5))
    with pytest.raises(ValueError):
        torchsso.DiagCovRMSNorm(torch.nn.RMSNorm((5, 6)))


def test_more_elements_than_32_bits_count():
    rows, dim = (1 << 18) + 3, 8192
    x = torch.empty(rows, dim, device='cuda', dtype=torch.bfloat16).normal_().requires_grad_()
    gain = torch.linspace(0.5, 2., dim, device='cuda')
    y = torchsso.nn.rms_norm(x, gain)
    dx, = torch.autograd.grad(y, x, x.detach())
    for part in (slice(0, 2), slice(rows // 2, rows // 2 + 2), slice(rows - 2, rows)):
        xs = x.detach()[part].clone().requires_grad_()
        ys = torchsso.nn.rms_norm(xs, gain)
        assert torch.equal(y[part], ys)
        assert torch.equal(dx[part], torch.autograd.grad(ys, xs, xs.detach())[0])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('dim', [96, 1000, 5120])
def test_streams_beyond_the_caches_give_what_a_few_rows_give(dtype, dim):
    rows = (1 << 28) // (dim * 4) + 7           # (every tensor of them: 128 MiB or more)
    gen = torch.Generator(device='cuda').manual_seed(dim)
    x, res, dy, dh = (torch.empty(rows, dim, device='cuda', dtype=dtype).normal_(generator=gen) for _ in range(4))
    gain = torch.linspace(0.5, 2., dim, device='cuda')

    def passes(x, res, dy, dh):
        x, res = x.clone().requires_grad_(), res.clone().requires_grad_()
        y, h = torchsso.nn.add_rms_norm(x, res, gain)
        with torch.no_grad():
            eight = torchsso.nn.add_rms_norm(x, res, gain, out_dtype=torch.float8_e4m3fn)
        return (y, h) + torch.autograd.grad((y, h), (x, res), (dy, dh)) + (eight[0].view(torch.uint8), eight[1], eight[2])

    whole = passes(x, res, dy, dh)
    for part in (slice(0, 3), slice(rows // 2, rows // 2 + 3), slice(rows - 3, rows)):
        few = passes(x[part], res[part], dy[part], dh[part])
        for a, b in zip(whole, few):
            assert torch.equal(a[part], b)
