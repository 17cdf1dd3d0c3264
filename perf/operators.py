"""The operators for training and running large language models, as cases that can be timed and
compared.

A case is a dict of plain values:

  kind = 'orth'   torchsso.utils.orthogonalize: Newton-Schulz orthogonalisation of a list of
                  matrices.  `shapes`: rows x columns, *k for a stack of k in one tensor; `dtype`
  kind = 'muon'   torchsso.optim.muon: one update of a list of matrices (momentum,
                  orthogonalisation, weight decay): `shapes`, `dtype`, `nesterov`, `weight_decay`
  kind = 'norm'   torchsso.nn.add_rms_norm / rms_norm without a backward pass: root-mean-square
                  norm of `batch` x `tokens` rows of `dim`, `residual` added first or not, in
                  `dtype`, and with `eight` the output in 8 bits with a scale per row
  kind = 'train'  the same with its backward pass, which also leaves the diagonal curvature of
                  the gain over the `batch` samples

The orthogonalisation of G (r x c, r <= c; a taller one is transposed) is
    X = G / (|G| + 1e-7);   5 times:  A = X X^T,  X = a X + (b A + c A A) X
with |G| the Frobenius norm.  The norm's stream h = x + residual is kept in its type, and
    y = h / sqrt(mean(h^2) + eps) * gain
is the norm of what is kept.  With s_n = sum over the tokens of sample n of dy * h / rms, the
gain's gradient is sum_n s_n and its curvature batch * sum_n s_n^2.
"""
import math

import torch

own = False
DEVICE = 'cuda:0'
A1, B1, C1 = 3.4445, -4.7750, 2.0315
STEPS = 5
NORM_EPS = 1e-7
RMS_EPS = 1e-6
LR, MOMENTUM = 0.02, 0.95
LARGEST_8 = 448.                       # of the 8-bit type float8_e4m3fn

RESNET50 = '64x147,64x64,64x576*3,256x64*4,64x256*2,128x256,128x1152*4,512x128*4,512x256,128x512*3,' \
           '256x512,256x2304*6,1024x256*6,1024x512,256x1024*5,512x1024,512x4608*3,2048x512*3,' \
           '2048x1024,512x2048*2,1000x2048'
DECODER = '2048x2048,512x2048,512x2048,2048x2048,5504x2048,5504x2048,2048x5504'


# ---------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------

def listed():
    return [
        # a toy classifier (20-16-10): nothing but launches
        dict(name='orth_toy', kind='orth', shapes='16x20,10x16', dtype='float32'),
        # the benchmark's multi-layer perceptron, 784-1000-1000-10: wide, square and ten rows
        dict(name='orth_mlp', kind='orth', shapes='1000x784,1000x1000,10x1000', dtype='float32'),
        # every convolution and the classifier of a ResNet-50, filters as matrices
        dict(name='orth_resnet50', kind='orth', shapes=RESNET50, dtype='float32'),
        # one projection of a layer of 16 experts, kept as a stack
        dict(name='orth_experts', kind='orth', shapes='1024x2752*16', dtype='bfloat16'),
        # the fully connected layers of AlexNet: the largest matrices
        dict(name='orth_alexnet_fc', kind='orth', shapes='4096x9216,4096x4096,1000x4096',
             dtype='float32'),
        # an update of a small perceptron with odd widths, weights in float32
        dict(name='muon_ragged', kind='muon', shapes='517x301,1263x517,37x1263', dtype='float32',
             nesterov=True, weight_decay=0.01),
        # an update of four decoder layers with shared key and value heads
        dict(name='muon_decoder', kind='muon', shapes=','.join([DECODER] * 4), dtype='bfloat16',
             nesterov=True, weight_decay=0.1),
        # a single new token of a decoder that answers
        dict(name='norm_token', kind='norm', batch=1, tokens=1, dim=4096, residual=True,
             eight=False, dtype='bfloat16'),
        # a long prompt, the norm handing 8 bits to the product behind it; odd number of rows
        dict(name='norm_prompt_8bit', kind='norm', batch=3, tokens=2731, dim=5120, residual=True,
             eight=True, dtype='bfloat16'),
        # a training pass with a ragged batch and an odd width
        dict(name='train_ragged', kind='train', batch=5, tokens=37, dim=1263, residual=True,
             dtype='float32'),
        # rows that are samples themselves
        dict(name='train_rows', kind='train', batch=1024, tokens=1, dim=4096, residual=False,
             dtype='float32'),
        # a decoder block's norm in a training pass
        dict(name='train_decoder', kind='train', batch=8, tokens=2048, dim=4096, residual=True,
             dtype='bfloat16'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['orth', 'orth', 'muon', 'norm', 'train'])
    dtype = rng.choice(['float32', 'float32', 'bfloat16', 'bfloat16', 'float16'])
    if kind in ('orth', 'muon'):
        shapes, spent = [], 0.
        for _ in range(rng.randint(1, 8)):
            r, c = _log_int(rng, 8, 4096), _log_int(rng, 8, 6000)
            stack = rng.choice([1, 1, 1, 2, 5]) if kind == 'orth' else 1
            spent += stack * _orth_flops(r, c)
            if spent > 2.5e12:
                break
            shapes.append('%dx%d' % (r, c) + ('*%d' % stack if stack > 1 else ''))
        shapes = ','.join(shapes) or '517x301'
        if kind == 'orth':
            return dict(kind=kind, shapes=shapes, dtype=dtype)
        return dict(kind=kind, shapes=shapes, dtype=dtype, nesterov=rng.random() < 0.7,
                    weight_decay=rng.choice([0., 0.1]))
    dim = rng.choice([_log_int(rng, 32, 8192), 8 * _log_int(rng, 4, 1024)])
    rows = _log_int(rng, 1, max(1, min(20000, 60000000 // dim)))
    batch = min(rows, rng.choice([1, 2, 8, 31, rows]))
    case = dict(kind=kind, batch=batch, tokens=max(1, rows // batch), dim=dim,
                residual=rng.random() < 0.7, dtype=dtype)
    if kind == 'norm':
        case['eight'] = rng.random() < 0.4
    return case


# ---------------------------------------------------------------------------------------
# states
# ---------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _shapes(case):
    """[(stack or None, rows, columns)]"""
    out = []
    for s in case['shapes'].split(','):
        s, _, stack = s.partition('*')
        r, c = s.split('x')
        out.append((int(stack) if stack else None, int(r), int(c)))
    return out


def _gradient(gen, stack, r, c, dtype):
    """What a backward pass leaves for a weight: output gradients times the layer's inputs, which
    sit behind a rectifier (so their mean is a strong direction), over some hundred tokens, and
    the many weaker directions of the other tokens."""
    n = 1 if stack is None else stack
    terms = 256
    out = torch.empty((n, r, c), device=DEVICE, dtype=dtype)
    for k in range(n):
        x = torch.randn(terms, c, device=DEVICE, generator=gen).clamp_(min=0)
        d = torch.randn(terms, r, device=DEVICE, generator=gen)
        d *= torch.rand(terms, 1, device=DEVICE, generator=gen)
        g = d.t().contiguous() @ x
        g /= terms
        g += torch.randn(r, c, device=DEVICE, generator=gen) * (0.3 / math.sqrt(terms))
        out[k] = g.mul_(1e-2)
    return out[0] if stack is None else out


def prepare(case, seed):
    gen = _generator(seed)
    dtype = getattr(torch, case['dtype'])
    state = dict(case)
    if case['kind'] in ('orth', 'muon'):
        state['grads'] = [_gradient(gen, *s, dtype) for s in _shapes(case)]
        if case['kind'] == 'muon':
            state['params'] = [(torch.randn(g.shape, device=DEVICE, generator=gen)
                                / math.sqrt(g.shape[-1])).to(dtype) for g in state['grads']]
            state['buffers'] = [g.float() * 8 + 0.02 * torch.randn(g.shape, device=DEVICE, generator=gen)
                                * g.float().norm() / math.sqrt(g.numel()) for g in state['grads']]
        return state
    shape = (case['batch'], case['tokens'], case['dim'])

    def rows(scale):
        t = torch.randn(shape, device=DEVICE, generator=gen)
        # tokens of different sizes, and a few channels that stand out
        t *= torch.rand(shape[:2] + (1,), device=DEVICE, generator=gen) * scale + 0.1
        t[..., ::97] *= 8
        return t.to(dtype)
    train = case['kind'] == 'train'
    state['x'] = rows(1.).requires_grad_(train)
    state['residual'] = rows(4.).requires_grad_(train) if case['residual'] else None
    state['gain'] = (1 + 0.2 * torch.randn(case['dim'], device=DEVICE, generator=gen)
                     ).to(dtype).requires_grad_(train)
    if train:
        state['dy'] = (torch.randn(shape, device=DEVICE, generator=gen) / shape[0]).to(dtype)
        state['dh'] = (torch.randn(shape, device=DEVICE, generator=gen) / shape[0]).to(dtype)
        state['curvature'] = torch.zeros(case['dim'], device=DEVICE)
    return state


# ---------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------

def _run_own(state):
    import os
    import sys
    path = os.path.join(os.getcwd(), 'pytorch-sso_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    import torchsso
    kind = state['kind']
    if kind == 'orth':
        return torchsso.utils.orthogonalize(state['grads'])
    if kind == 'muon':
        torchsso.optim.muon(state['params'], state['grads'], state['buffers'], lr=LR,
                            momentum=MOMENTUM, nesterov=state['nesterov'],
                            weight_decay=state['weight_decay'])
        return dict(params=state['params'], buffers=state['buffers'])
    x, residual, gain = state['x'], state['residual'], state['gain']
    if kind == 'norm':
        more = dict(out_dtype=torch.float8_e4m3fn) if state['eight'] else {}
        if residual is None:
            return torchsso.nn.rms_norm(x, gain, RMS_EPS, **more)
        return torchsso.nn.add_rms_norm(x, residual, gain, RMS_EPS, **more)
    curvature = state['curvature']
    if residual is None:
        y = torchsso.nn.rms_norm(x, gain, RMS_EPS, curvature=curvature)
        dx, dgain = torch.autograd.grad(y, (x, gain), state['dy'])
        return dict(y=y, dx=dx, dgain=dgain, curvature=curvature)
    y, h = torchsso.nn.add_rms_norm(x, residual, gain, RMS_EPS, curvature=curvature)
    dx, dres, dgain = torch.autograd.grad((y, h), (x, residual, gain), (state['dy'], state['dh']))
    return dict(y=y, h=h, dx=dx, dresidual=dres, dgain=dgain, curvature=curvature)


# ---------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------

def _newton_schulz(g):
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2).contiguous()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + NORM_EPS)
    for _ in range(STEPS):
        a = x @ x.transpose(-1, -2).contiguous()
        x = A1 * x + (B1 * a + C1 * (a @ a)) @ x
    return x.transpose(-1, -2) if tall else x


def _muon_scale(g):
    return math.sqrt(max(1., g.shape[0] / g.shape[1]))


@torch.no_grad()
def _run_plain(state):
    kind = state['kind']
    if kind == 'orth':
        return [_newton_schulz(g).to(g.dtype).contiguous() for g in state['grads']]
    if kind == 'muon':
        for p, g, buf in zip(state['params'], state['grads'], state['buffers']):
            g32 = g.float()
            buf.mul_(MOMENTUM).add_(g32)
            u = g32 + MOMENTUM * buf if state['nesterov'] else buf
            p.copy_(p.float() * (1 - LR * state['weight_decay'])
                    - LR * _muon_scale(g) * _newton_schulz(u))
        return dict(params=state['params'], buffers=state['buffers'])
    x, residual, gain = state['x'], state['residual'], state['gain'].float()
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    h32 = h.float()
    r = torch.rsqrt(h32.square().mean(-1, keepdim=True) + RMS_EPS)
    hat = h32 * r
    y32 = hat * gain
    if kind == 'norm':
        if state['eight']:
            top = y32.abs().amax(-1, keepdim=True)
            scale = torch.where(top > 0, top / LARGEST_8, torch.ones_like(top))
            out = ((y32 / scale).to(torch.float8_e4m3fn), scale)
        else:
            out = (y32.to(x.dtype),)
        return (out + (h,) if residual is not None else out if len(out) > 1 else out[0])
    y = y32.to(x.dtype)
    dy = state['dy'].float()
    wdy = gain * dy
    dx = r * (wdy - hat * (wdy * hat).mean(-1, keepdim=True))
    s = (dy * hat).sum(1)
    dgain = s.sum(0).to(state['gain'].dtype)
    state['curvature'].copy_(s.square().sum(0) * s.shape[0])
    if residual is None:
        return dict(y=y, dx=dx.to(x.dtype), dgain=dgain, curvature=state['curvature'])
    dx = (dx + state['dh'].float()).to(x.dtype)
    return dict(y=y, h=h, dx=dx, dresidual=dx, dgain=dgain, curvature=state['curvature'])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------

def _polar_64(g):
    """The iteration in 64 bits on the side of the rows, one product at a time."""
    x = g.detach().double()
    wide = x.shape[0] <= x.shape[1]
    x = x if wide else x.t().contiguous()
    x = x / (x.pow(2).sum().sqrt() + NORM_EPS)
    for _ in range(STEPS):
        gram = torch.mm(x, x.t().contiguous())
        once = torch.mm(gram, x)
        twice = torch.mm(gram, once)
        x = A1 * x + B1 * once + C1 * twice
    return x if wide else x.t().contiguous()


def _layers_64(g):
    return _polar_64(g) if g.dim() == 2 else torch.stack([_polar_64(m) for m in g])


def exact(case, seed):
    state = prepare(case, seed)
    kind = case['kind']
    with torch.no_grad():
        if kind == 'orth':
            return [_layers_64(g) for g in state['grads']]
        if kind == 'muon':
            params, buffers = [], []
            for p, g, buf in zip(state['params'], state['grads'], state['buffers']):
                m = buf.double() * MOMENTUM + g.double()
                direction = m * MOMENTUM + g.double() if case['nesterov'] else m
                step = LR * math.sqrt(max(1., g.shape[0] / g.shape[1])) * _polar_64(direction)
                params.append(p.double() - LR * case['weight_decay'] * p.double() - step)
                buffers.append(m)
            return dict(params=params, buffers=buffers)
        h = state['x'].double()
        if case['residual']:
            # (the stream is kept in its type, and what is kept is normalised)
            h = (h + state['residual'].double()).to(state['x'].dtype).double()
        gain = state['gain'].double()
        rms = (h.pow(2).sum(-1, keepdim=True) / case['dim'] + RMS_EPS).sqrt()
        hat = h / rms
        y = hat * gain
        if kind == 'norm':
            out = (y,)
            if case['eight']:
                top = y.abs().amax(-1, keepdim=True)
                scale = torch.where(top > 0, top / LARGEST_8, torch.ones_like(top))
                out = (y / scale, scale)
            return out + (h,) if case['residual'] else out if len(out) > 1 else y
        dy = state['dy'].double()
        # d y_i / d h_j = gain_i (delta_ij - hat_i hat_j / dim) / rms
        v = gain * dy
        dx = (v - hat * ((v * hat).sum(-1, keepdim=True) / case['dim'])) / rms
        per_sample = torch.stack([(dy[n] * hat[n]).sum(0) for n in range(case['batch'])])
        out = dict(y=y, dgain=per_sample.sum(0), curvature=case['batch'] * per_sample.pow(2).sum(0))
        if case['residual']:
            dx = dx + state['dh'].double()
            out.update(h=h, dresidual=dx)
        return dict(out, dx=dx)


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------

def _orth_flops(r, c):
    """Both symmetric products by one triangle."""
    r, c = float(min(r, c)), float(max(r, c))
    return STEPS * (r * r * c + r * r * r + 2 * r * r * c)


def work(case):
    size = 4. if case['dtype'] == 'float32' else 2.
    if case['kind'] in ('orth', 'muon'):
        flops = nbytes = 0.
        for stack, r, c in _shapes(case):
            n = float(stack or 1)
            flops += n * _orth_flops(r, c)
            # gradient in and result out; with the parameter and the float32 buffer, in and out
            nbytes += n * r * c * (2 * size if case['kind'] == 'orth' else 3 * size + 8.)
        return dict(flops=flops, bytes=nbytes)
    d = float(case['dim'])
    rows = float(case['batch'] * case['tokens'])
    streams = 1. + (2. if case['residual'] else 0.)          # x, residual and h
    nbytes = rows * d * size * streams + d * size
    if case['kind'] == 'norm':
        nbytes += rows * (d + 4.) if case['eight'] else rows * d * size
        return dict(flops=4. * rows * d, bytes=nbytes)
    # y out and dy in, the stream again, its gradient in (with a residual) and out
    nbytes += rows * d * size * (4. + (1. if case['residual'] else 0.)) + d * (2 * size + 4.)
    return dict(flops=14. * rows * d, bytes=nbytes)
