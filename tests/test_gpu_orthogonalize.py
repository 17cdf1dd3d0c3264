"""torchsso.utils.orthogonalize and torchsso.optim.muon / Muon against the iteration in 64 bits.

Tolerances (2-norm of the difference over that of the result).  A product rounds its operands to 22
bits (2^-23 of an element) and sums in float32; a step has three, and what a step rounds grows with
the steps behind it by the slope of the iteration, 3.4 at most and about 1.5 over the singular
values of the random matrices here: 15 * 2^-22 * (1 + 1.5 + ... + 1.5^4) = 4.7e-5 if all errors of a
step were of one sign, and 1 / sqrt(15) of that, 1.2e-5, as they are not.  A float16 result adds
2^-12 (2.5e-4), a bfloat16 one 2^-9 / sqrt(3) * 1.5 (1.7e-3, the mean over an octave) and two steps
of 11 bits, 3 roundings each of 2^-12 / sqrt(3) grown by 1.5 + 1: 6.2e-4.
"""
import pytest
import torch

import torchsso
from torchsso import _hip

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1.2e-5, torch.float16: 2.7e-4, torch.bfloat16: 2.4e-3}
TYPES = list(TOL)
COEFFS = (3.4445, -4.7750, 2.0315)


def reference(g, steps=5, coeffs=COEFFS, eps=1e-7):
    g = g.detach().cpu().double()
    if g.dim() > 2:
        return torch.stack([reference(m, steps, coeffs, eps) for m in g])
    triples = coeffs if isinstance(coeffs[0], tuple) else [coeffs] * steps
    x = g / (torch.linalg.matrix_norm(g) + eps)
    for a, b, c in triples:
        if x.shape[0] <= x.shape[1]:
            m = x @ x.T
            x = a * x + (b * m + c * m @ m) @ x
        else:
            m = x.T @ x
            x = a * x + x @ (b * m + c * m @ m)
    return x


def off(got, want):
    return (got.detach().cpu().double() - want).norm().item() / max(want.norm().item(), 1e-300)


def random(shape, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen).to(dtype).cuda()


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('shape', [(1, 1), (1, 7), (7, 1), (10, 16), (63, 65), (64, 64), (65, 64), (127, 129),
                                   (128, 128), (129, 128), (37, 1263), (1263, 37), (300, 1025), (517, 301),
                                   (3, 65, 130), (2, 1, 5, 9)])
def test_against_64_bits(shape, dtype):
    g = random(shape, dtype)
    flat = g.view((-1,) + g.shape[-2:]) if g.dim() > 2 else g
    out = torchsso.utils.orthogonalize(g)
    assert out.shape == g.shape and out.dtype == dtype
    assert off(out.view(flat.shape), reference(flat)) <= TOL[dtype]


@pytest.mark.parametrize('shape', [(8, 16384), (16384, 8), (513, 4609)])
def test_long_sides(shape):
    g = random(shape, torch.float32)
    assert off(torchsso.utils.orthogonalize(g), reference(g)) <= TOL[torch.float32]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_a_list_gives_what_each_gives_alone(dtype):
    shapes = [(10, 1000), (130, 70), (70, 130), (64, 64), (5, 33, 20), (200, 200), (130, 70), (0, 4), (2, 0, 3)]
    mats = [random(s, dtype, i) for i, s in enumerate(shapes)]
    outs = torchsso.utils.orthogonalize(mats)
    for m, o in zip(mats, outs):
        assert torch.equal(o, torchsso.utils.orthogonalize(m))


def test_more_shapes_than_a_launch_holds():
    mats = [random((3 + i, 70 + i), torch.float32, i) for i in range(60)]
    for m, o in zip(mats, torchsso.utils.orthogonalize(mats)):
        assert off(o, reference(m)) <= TOL[torch.float32]


def test_strided_input():
    g = random((300, 200), torch.float32)
    assert torch.equal(torchsso.utils.orthogonalize(g.t()), torchsso.utils.orthogonalize(g.t().contiguous()))
    odd = random((301 * 77 + 1,), torch.float32)[1:].view(301, 77)
    assert off(torchsso.utils.orthogonalize(odd), reference(odd)) <= TOL[torch.float32]


def test_zero_and_rank_deficient():
    assert torch.equal(torchsso.utils.orthogonalize(torch.zeros(70, 90, device='cuda')),
                       torch.zeros(70, 90, device='cuda'))
    g = random((200, 3), torch.float32) @ random((3, 150), torch.float32, 1)
    out = torchsso.utils.orthogonalize(g)
    # (singular values that are zero but for rounding grow by up to 3.4445^5 = 485)
    assert off(out, reference(g)) <= 485 * 2 ** -22


@pytest.mark.parametrize('scale', [1e-30, 1e-12, 1e30])
def test_scale_of_the_input(scale):
    g = random((100, 140), torch.float32) * scale
    out, want = torchsso.utils.orthogonalize(g, eps=1e-37), reference(g, eps=1e-37)
    assert off(out, want) <= TOL[torch.float32]


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_a_matrix_that_is_not_finite_stays_by_itself(bad):
    mats = [random((130, 70), torch.float32, i) for i in range(3)]
    clean = torchsso.utils.orthogonalize(mats)
    mats[1][3, 4] = bad
    outs = torchsso.utils.orthogonalize(mats)
    assert torch.equal(outs[0], clean[0]) and torch.equal(outs[2], clean[2])
    assert torch.isnan(outs[1]).all()


@pytest.mark.parametrize('steps,coeffs', [(1, COEFFS), (2, COEFFS), (3, (1.5, -0.5, 0.)),
                                          (3, ((3.4, -4.7, 2.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)))])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
def test_steps_and_coefficients(steps, coeffs, dtype):
    g = random((90, 200), dtype)
    assert off(torchsso.utils.orthogonalize(g, steps, coeffs), reference(g, steps, coeffs)) <= TOL[dtype]


def test_same_bits_every_time_and_on_another_stream():
    mats = [random((300, 500), torch.float32), random((64, 100), torch.float32, 1)]
    first = torchsso.utils.orthogonalize(mats)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = torchsso.utils.orthogonalize(mats)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_in_a_recorded_graph():
    g = random((200, 300), torch.float32)
    torchsso.utils.orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torchsso.utils.orthogonalize(g)          # (the scratch of that stream)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = torchsso.utils.orthogonalize(g)
    for seed in range(3):
        g.copy_(random((200, 300), torch.float32, seed))
        graph.replay()
        assert torch.equal(out, torchsso.utils.orthogonalize(g))


# ---------------------------------------------------------------------------------------
# Muon
# ---------------------------------------------------------------------------------------

def muon_reference(p, g, buf, lr, momentum, nesterov, weight_decay):
    p, g, buf = (t.detach().cpu().double() for t in (p, g, buf))
    shape = p.shape
    p, g, buf = (t.reshape(shape[0], -1) for t in (p, g, buf))
    buf = momentum * buf + g
    u = g + momentum * buf if nesterov else buf
    scale = max(1., p.shape[0] / p.shape[1]) ** 0.5
    p = p * (1 - lr * weight_decay) - lr * scale * reference(u)
    return p.reshape(shape), buf.reshape(shape)


# of the parameter, beyond what rounding the exact one to its type takes (of the few elements of some
# shapes here that is more than the mean over an octave): the update is of its size (lr 1), float32
# rounds it twice, and the two late steps of bfloat16 as above
MUON_TOL = {torch.float32: 1.2e-5 + 2 ** -23, torch.float16: 1.2e-5 + 2 ** -23, torch.bfloat16: 7e-4}


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('nesterov,weight_decay', [(True, 0.), (False, 0.1)])
def test_muon_against_64_bits(dtype, nesterov, weight_decay):
    shapes = [(30, 50), (200, 90), (1, 9), (16, 3, 5, 5), (129, 257)]
    ps = [random(s, dtype, i) for i, s in enumerate(shapes)]
    bufs = [torch.zeros(s, device='cuda') for s in shapes]
    for step in range(2):
        gs = [random(s, dtype, 10 + 10 * step + i) for i, s in enumerate(shapes)]
        want = [muon_reference(p, g, b, 1., 0.9, nesterov, weight_decay) for p, g, b in zip(ps, gs, bufs)]
        torchsso.optim.muon(ps, gs, bufs, lr=1., momentum=0.9, nesterov=nesterov, weight_decay=weight_decay)
        for p, b, (wp, wb) in zip(ps, bufs, want):
            assert off(b, wb) <= 2 ** -23
            assert off(p, wp) <= MUON_TOL[dtype] + off(wp.to(dtype), wp)


def test_muon_optimizer():
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 3, bias=False), torch.nn.Flatten(),
                                torch.nn.Linear(8 * 16, 5, bias=False)).cuda()
    x, y = torch.randn(32, 3, 6, 6, device='cuda'), torch.randint(0, 5, (32,), device='cuda')
    opt = torchsso.optim.Muon(model.parameters(), lr=0.05)

    def closure():
        opt.zero_grad()
        out = model(x)
        loss = torch.nn.functional.cross_entropy(out, y)
        loss.backward()
        return loss, out
    losses = [opt.step(closure)[0].item() for _ in range(15)]
    assert losses[-1] < 0.5 * losses[0]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
def test_muon_checkpoint(dtype):
    def make():
        p = torch.nn.Parameter(random((40, 30), dtype))
        return p, torchsso.optim.Muon([p], lr=0.1, weight_decay=0.1)
    (p, opt), (q, other) = make(), make()
    for i in range(3):
        p.grad = random((40, 30), dtype, i)
        opt.step()
    q.data.copy_(p.data)
    other.load_state_dict(opt.state_dict())
    assert other.state[q]['momentum_buffer'].dtype == torch.float32
    for w, o in ((p, opt), (q, other)):
        w.grad = random((40, 30), dtype, 9)
        o.step()
    assert torch.equal(p, q)


def test_muon_leaves_out_what_has_no_gradient():
    p, q = (torch.nn.Parameter(random((9, 12), torch.float32, i)) for i in range(2))
    opt = torchsso.optim.Muon([p, q])
    before = q.detach().clone()
    p.grad = random((9, 12), torch.float32, 5)
    opt.step()
    assert torch.equal(q, before) and q not in opt.state


def test_refusals_on_the_device():
    g = random((8, 8), torch.float32)
    with pytest.raises(_hip.KfacHipError):
        torchsso.utils.orthogonalize([g, g.to(torch.bfloat16)])
    with pytest.raises(_hip.KfacHipError):
        torchsso.utils.orthogonalize(g.double())
    with pytest.raises(_hip.KfacHipError):
        torchsso.utils.orthogonalize([g, g.cpu()])
    with pytest.raises(_hip.KfacHipError):
        torchsso.utils.orthogonalize(torch.zeros(1, 16385, device='cuda'))
    with pytest.raises(_hip.KfacHipError):
        torchsso.optim.muon([g, g], [g, g], [torch.zeros_like(g), torch.zeros_like(g)], lr=0.1)
    with pytest.raises(_hip.KfacHipError):
        torchsso.optim.muon([g], [g.to(torch.bfloat16)], [torch.zeros_like(g)], lr=0.1)
    with pytest.raises(_hip.KfacHipError):
        torchsso.optim.muon([g], [g], [torch.zeros(8, 8, device='cuda', dtype=torch.bfloat16)], lr=0.1)
    with pytest.raises(_hip.KfacHipError):
        torchsso.optim.muon([g], [torch.zeros(4, 16, device='cuda')], [torch.zeros_like(g)], lr=0.1)
    with pytest.raises(ValueError):
        torchsso.optim.muon([g.t()[:, :4]], [g[:, :4]], [torch.zeros(8, 4, device='cuda')], lr=0.1)


# ---------------------------------------------------------------------------------------
# large tiles, reductions in pieces, several batches
# ---------------------------------------------------------------------------------------

def reference_on_device(g):
    """`reference` of one matrix in 64 bits on the device (for sides that the host takes minutes for)."""
    a, b, c = COEFFS
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / (x.square().sum().sqrt() + 1e-7)
    for _ in range(5):
        m = x @ x.t().contiguous()
        y = m @ x
        x = a * x + b * y + c * (m @ y)
    return x.t() if tall else x


def off_on_device(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


LISTS = {
    # 256-wide tiles that fill the chip once and a little: the last round in pieces
    'square': [(4096, 4096)],
    'wide_and_tall': [(2048, 2310), (2310, 2048), (2047, 2304), (2100, 2050)],
    # long reductions of few tiles, small matrices beside large ones
    'long': [(512, 9000), (9001, 130), (64, 576), (20, 30)],
    'mixed': [(1300, 2900), (2048, 2048), (2048, 2048), (3000, 700), (600, 600), (100, 2000), (48, 50)],
    # many shapes of convolutions
    'convolutions': [(64, 147), (64, 576), (256, 64), (128, 1152), (512, 128), (256, 2304), (1024, 256), (512, 4608),
                     (2048, 512), (1000, 2048)],
}


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('name', sorted(LISTS))
def test_lists_of_all_sizes(name, dtype):
    mats = [random(s, dtype, i) for i, s in enumerate(LISTS[name])]
    for m, o in zip(mats, torchsso.utils.orthogonalize(mats)):
        assert off_on_device(o, reference_on_device(m)) <= TOL[dtype]


def test_more_than_a_batch():
    """A list whose operands do not fit the scratch at once is worked on in parts."""
    mats = [random((2048, 3500), torch.bfloat16, i) for i in range(16)]
    outs = torchsso.utils.orthogonalize(mats)
    for i in (0, 8, 15):
        assert off_on_device(outs[i], reference_on_device(mats[i])) <= TOL[torch.bfloat16]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_muon_of_large_matrices(dtype):
    shapes = [(2048, 2304), (2304, 2048), (2047, 2100), (2100, 2046), (300, 5000)]
    ps = [random(s, dtype, i) for i, s in enumerate(shapes)]
    gs = [random(s, dtype, 10 + i) for i, s in enumerate(shapes)]
    bufs = [random(s, torch.float32, 20 + i) for i, s in enumerate(shapes)]
    want = []
    for p, g, b in zip(ps, gs, bufs):
        m = 0.9 * b.double() + g.double()
        scale = max(1., p.shape[0] / p.shape[1]) ** 0.5
        want.append((p.double() * 0.9 - scale * reference_on_device(g.double() + 0.9 * m), m))
    torchsso.optim.muon(ps, gs, bufs, lr=1., momentum=0.9, weight_decay=0.1)
    for p, b, (wp, wb) in zip(ps, bufs, want):
        assert off_on_device(b, wb) <= 2 ** -23
        assert off_on_device(p, wp) <= MUON_TOL[dtype] + off_on_device(wp.to(dtype), wp)


def test_the_largest_side():
    g = random((16384, 1030), torch.float32)
    assert off_on_device(torchsso.utils.orthogonalize(g), reference_on_device(g)) <= TOL[torch.float32]
