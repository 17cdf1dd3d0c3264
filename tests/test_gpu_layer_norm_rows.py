"""Layer norm of rows of any length and alignment: accesses that end where the row does, sums of long rows by a pass of their
own, and nothing written beside the results."""
import pytest
import torch

import torchsso
from torchsso import _hip, _ops

from test_gpu_layer_norm import EPS, EIGHT, TYPES, Want, check, random

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', [3, 4, 5, 8, 9, 15, 17, 127, 129, 511, 513, 1023, 1025, 4095, 4100, 8190, 8200, 9001, 16383, 16392, 32769])
@pytest.mark.parametrize('samples,tokens', [(6, 1), (2, 3), (1, 7), (300, 1)])
def test_gradients(dtype, dim, samples, tokens):
    if samples * dim > 3000000:
        samples = 40
    shape = (samples, tokens, dim)
    x, res = (random(shape, dtype, i, 1., 0.5).requires_grad_() for i in range(2))
    gain, bias = (random((dim,), dtype, 2 + i).requires_grad_() for i in range(2))
    dy, dh = random(shape, dtype, 4), random(shape, dtype, 5)
    curvature = torch.full((2, dim), float('nan'), device='cuda')
    y, h = torchsso.nn.add_layer_norm(x, res, gain, bias, EPS, curvature=curvature)
    dx, dgain, dbias = torch.autograd.grad((y, h), (x, gain, bias), (dy, dh))
    want = Want(x, res, gain, bias, dy, dh, samples)
    check(y, want.y, dtype, 1e-6, want.size)
    check(dx, want.dx, dtype, 1e-6, want.dx_size)
    check(dgain, want.dgain, dtype, 2e-6)
    check(dbias, want.dbias, dtype, 2e-6)
    check(curvature, want.curvature, torch.float32, 4e-6)
    # the gradient of the stream alone, and the sums alone
    stats = _ops.layer_norm_stats(h.detach(), EPS)
    only, _, _ = _ops.layer_norm_backward(dy, dh, h.detach(), stats, gain.detach(), samples, True, False, False)
    check(only, want.dx, dtype, 1e-6, want.dx_size)
    alone = torch.empty_like(curvature)
    _, dgain, dbias = _ops.layer_norm_backward(dy, None, h.detach(), stats, gain.detach(), samples, False, True, True, alone)
    check(dgain, want.dgain, dtype, 2e-6)
    check(dbias, want.dbias, dtype, 2e-6)
    check(alone, want.curvature, torch.float32, 4e-6)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', [8, 64, 1000, 2048, 4096, 8192, 16384, 32768])
def test_rows_off_16_bytes_give_the_same_bits(dtype, dim):
    x, res = (random((5, dim + 1), dtype, i) for i in range(2))
    gain, bias = random((dim + 1,), dtype, 2), random((dim + 1,), dtype, 3)
    off = [t[..., 1:] for t in (x, res, gain, bias)]
    a = torchsso.nn.add_layer_norm(*[t.clone() for t in off], EPS)
    b = torchsso.nn.add_layer_norm(*off, EPS)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    a = torchsso.nn.add_layer_norm(*[t.clone() for t in off], EPS, out_dtype=EIGHT)
    b = torchsso.nn.add_layer_norm(*off, EPS, out_dtype=EIGHT)
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
    stats = _ops.layer_norm_stats(off[0], EPS)
    assert torch.equal(stats, _ops.layer_norm_stats(off[0].clone(), EPS))
    grads = [_ops.layer_norm_backward(g, None, h, stats, w, 5) for g, h, w in
             ((off[1], off[0], off[2].clone()), (off[1].clone(), off[0].clone(), off[2].clone()))]
    assert all(torch.equal(s, t) for s, t in zip(*grads))


class Guarded(object):
    """`n` elements, `offset` from a 16-byte boundary on, in a buffer that holds 7 around them"""

    def __init__(self, n, dtype, offset=0):
        self.n, self.first = n, 64 + offset
        self.whole = torch.full((n + 128 + offset,), 7, device='cuda', dtype=torch.float32).to(dtype)
        self.part = self.whole[self.first:self.first + n]

    def ptr(self):
        return self.part.data_ptr()

    def check(self):
        assert bool((self.whole[:self.first].float() == 7).all()) and bool((self.whole[self.first + self.n:].float() == 7).all())


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('dim', [1, 3, 7, 8, 9, 100, 1001, 2049, 5000, 8200, 9001, 33001])
@pytest.mark.parametrize('offset', [0, 1, 3])
def test_nothing_is_written_beside_the_results(dtype, dim, offset):
    lib, kind, rows, samples = _hip.load(), _hip.ELEMENT_TYPES[dtype], 6, 3
    x, dy = random((rows, dim), dtype), random((rows, dim), dtype, 1)
    gain, bias = random((dim,), dtype, 2), random((dim,), dtype, 3)
    stream = torch.cuda.current_stream().cuda_stream
    for eight in (False, True):
        y = Guarded(rows * dim, torch.float8_e4m3fn if eight else dtype, offset)
        h, scale, stats = Guarded(rows * dim, dtype, offset), Guarded(rows, torch.float32), Guarded(3 * rows, torch.float32)
        assert lib.kfac_layer_norm(kind, 0, rows, dim, x.data_ptr(), dim, dy.data_ptr(), dim, gain.data_ptr(), bias.data_ptr(), EPS,
                                   y.ptr(), h.ptr(), scale.ptr() if eight else None, stats.ptr(), stream) == 0
        for t in (y, h, scale, stats):
            t.check()
        want = Want(x, dy, gain, bias)
        assert torch.equal(h.part.view(rows, dim).cpu(), want.h.to(dtype))
        if not eight:
            check(y.part.view(rows, dim), want.y, dtype, 1e-6, want.size)
    for squares in (False, True):
        dx, dgain, dbias = (Guarded(n, dtype, offset) for n in (rows * dim, dim, dim))
        curvature = Guarded(2 * dim, torch.float32)
        size = lib.kfac_layer_norm_backward_workspace_bytes(kind, rows, dim, samples, 2, int(squares))
        scratch = Guarded(size // 4, torch.float32)
        assert lib.kfac_layer_norm_backward(
            kind, 0, rows, dim, samples, 2, dy.data_ptr(), dim, None, 0, h.ptr(), dim, stats.ptr(), gain.data_ptr(), dx.ptr(),
            dgain.ptr(), dbias.ptr(), curvature.ptr() if squares else None, scratch.ptr(), size, stream) == 0
        for t in (dx, dgain, dbias, curvature, scratch):
            t.check()
        want = Want(x, dy, gain, bias, dy, None, samples)
        check(dx.part.view(rows, dim), want.dx, dtype, 1e-6, want.dx_size)
        check(dgain.part, want.dgain, dtype, 2e-6)
        check(dbias.part, want.dbias, dtype, 2e-6)
        if squares:
            check(curvature.part.view(2, dim), want.curvature, torch.float32, 4e-6)
