"""torchsso.utils.inv / torchsso.utils.cholesky / torchsso.utils.orthogonalize on the HIP engine.

Stand in for the reference's CuPy/cuSOLVER calls: inv = potrf + potrs against
the identity (torchsso/utils/inv_cupy.py:27-34,114-128), cholesky =
cupy.linalg.cholesky transposed (torchsso/utils/cholesky_cupy.py:9-14).
"""
import functools
import math

import torch

from torchsso import _ops


def inv(m):
    """Inverse of a symmetric positive definite matrix (new tensor)."""
    outs, _ = _ops.damped_inverse_batched([m.detach().contiguous()])
    return outs[0]


def cholesky(m, upper=True):
    """U (upper=True) with m = U^T U, or its transpose L with m = L L^T."""
    outs, _ = _ops.cholesky_upper_batched([m.detach().contiguous()])
    u = outs[0]
    return u if upper else u.t().contiguous()


# the quintic whose iterates take every singular value to within about 0.7 ... 1.2
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)
# what a kernel's operand may hold (they are fp16 numbers times 2^13)
_OPERAND_BOUND = 7.9
_MOST_STEPS = 64


def _largest(coeffs, x):
    """max over [0, x] of |a t + b t^3 + c t^5| and of |a + b t^2 + c t^4|."""
    a, b, c = coeffs

    def turns(p, q, r):
        # positive roots in s = t^2 of p + q s + r s^2
        if r == 0:
            roots = [] if q == 0 else [-p / q]
        else:
            d = q * q - 4 * p * r
            roots = [] if d < 0 else [(-q + math.sqrt(d)) / (2 * r), (-q - math.sqrt(d)) / (2 * r)]
        return [math.sqrt(s) for s in roots if 0 < s < x * x]
    value = max(abs(a * t + b * t ** 3 + c * t ** 5) for t in [x] + turns(a, 3 * b, 5 * c))
    factor = max(abs(a + b * t ** 2 + c * t ** 4) for t in [0., x] + ([] if c == 0 else turns(b, 2 * c, 0)))
    return value, factor


@functools.lru_cache(maxsize=64)
def _flat_schedule(steps, coefficients):
    if isinstance(steps, bool) or int(steps) != steps or not 1 <= steps <= _MOST_STEPS:
        raise ValueError('Invalid steps: {}'.format(steps))
    triples = coefficients if isinstance(coefficients[0], tuple) else (coefficients,) * int(steps)
    if len(triples) != steps or any(len(t) != 3 for t in triples):
        raise ValueError('coefficients have to be one triple, or one for each of the %d steps' % steps)
    bound = 1.
    for t in triples:
        if not all(math.isfinite(v) for v in t):
            raise ValueError('Invalid coefficients: {}'.format(t))
        bound, factor = _largest(t, bound)
        # (two per cent for what the products round)
        if 1.02 * max(bound, bound * bound, factor) > _OPERAND_BOUND:
            raise ValueError('coefficients {} make the iteration grow beyond its range'.format(t))
    return tuple(float(v) for t in triples for v in t)


def newton_schulz_schedule(steps, coefficients):
    """The coefficients of all steps as a flat tuple, from one triple or a triple for each step.
    ValueError where they are not that, or where an iterate could leave the range of the kernels'
    operands (a spectral norm above about 2.8)."""
    if len(coefficients) > 0 and isinstance(coefficients[0], (tuple, list)):
        key = tuple(tuple(float(v) for v in t) for t in coefficients)
    else:
        key = tuple(float(v) for v in coefficients)
    if len(key) == 0:
        raise ValueError('no coefficients')
    return _flat_schedule(steps, key)


def check_orthogonalize_eps(eps):
    # (the kernels take it in float32, where it must not become zero or infinite)
    if not 2. ** -149 <= eps < 2. ** 128:
        raise ValueError('Invalid eps: {}'.format(eps))


def orthogonalize(mats, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7):
    """Newton-Schulz iterates towards the orthogonal factor U V^T of each matrix G = U S V^T:
    X = G / (|G| + eps), then `steps` times X = a X + (b A + c A A) X with A = X X^T.

    `mats`: a tensor of two dimensions, or of more for a stack of matrices (its last two), or a
    list of such tensors, in float32, bfloat16 or float16 (one type a list), with sides of up to
    16384.  Returns new
    tensors of the same shapes and type.  `coefficients`: (a, b, c), or one triple per step.

    Products run on the fp16 matrix cores in two parts a number (as good as float32).  Of a bfloat16
    matrix the last steps run in one part, as many as add about as much error at most as rounding the
    result does (of the default steps one)."""
    schedule = newton_schulz_schedule(steps, coefficients)
    check_orthogonalize_eps(eps)
    single = isinstance(mats, torch.Tensor)
    sources = [m.detach().contiguous() for m in ([mats] if single else mats)]
    results = [torch.empty_like(m) for m in sources]
    ins, outs = [], []
    for m, r in zip(sources, results):
        if m.dim() < 2:
            raise ValueError('expected matrices, got a tensor of shape {}'.format(tuple(m.shape)))
        if m.dim() == 2:
            ins.append(m)
            outs.append(r)
        elif m.numel() > 0:
            ins.extend(m.view((-1,) + m.shape[-2:]).unbind())
            outs.extend(r.view((-1,) + r.shape[-2:]).unbind())
    _ops.orthogonalize_batched(ins, outs, schedule, eps)
    return results[0] if single else results
