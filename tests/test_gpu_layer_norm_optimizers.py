"""Layer norms in the optimizers that take curvatures: accumulation, checkpoints, the posterior of VIOptimizer."""
import pytest
import torch
import torch.nn.functional as F

import torchsso

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize('kind', [torchsso.nn.LayerNorm, torch.nn.LayerNorm], ids=['torchsso', 'torch'])
SHAPES = {'Linear': 'Kron', 'LayerNorm': 'Diag'}


def net(kind, bias=True):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(20, 31), kind(31, bias=bias), torch.nn.Tanh(), torch.nn.Linear(31, 4)).cuda()


def data(seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(32, 20, generator=gen).cuda(), torch.randint(0, 4, (32,), generator=gen).cuda()


def closure_of(opt, model, seed):
    x, y = data(seed)

    def closure():
        opt.zero_grad()
        out = model(x)
        loss = F.cross_entropy(out, y)
        loss.backward()
        return loss, out
    return closure


def per_sample(model, x, y, bias):
    """Gradients of the mean loss' parts by the norm's parameters in 64 bits, one sample after the other"""
    grads = []
    params = [p.detach().double().cpu() for p in model.parameters()]
    for i in range(x.shape[0]):
        ps = [p.clone().requires_grad_() for p in params]
        h = F.layer_norm(x[i:i + 1].double().cpu() @ ps[0].t() + ps[1], (31,), ps[2], ps[3] if bias else None, 1e-5)
        rest = ps[4 if bias else 3:]
        out = torch.tanh(h) @ rest[0].t() + rest[1]
        loss = F.cross_entropy(out, y[i:i + 1].cpu()) / x.shape[0]
        grads.append(torch.autograd.grad(loss, ps[2:4 if bias else 3]))
    return [torch.stack(g) for g in zip(*grads)]


@KINDS
@pytest.mark.parametrize('bias', [True, False])
def test_curvature_of_a_network(kind, bias):
    """batch * sum of the squared gradients of single samples.  (The factors in front are float32 products over 20 and 31
    terms: 10^-5.)"""
    model = net(kind, bias)
    opt = torchsso.optim.SecondOrderOptimizer(model, 'Cov', SHAPES, {'damping': 1e-2, 'ema_decay': 1.}, lr=0.)
    x, y = data(1)
    want = [x.shape[0] * g.square().sum(0) for g in per_sample(model, x, y, bias)]
    opt.step(closure=closure_of(opt, model, 1))
    got = opt.param_groups[1]['curv'].ema
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert ((a.cpu().double() - b).norm() / b.norm()).item() <= 1e-5


@KINDS
def test_accumulation_and_checkpoint(kind, tmp_path):
    options = dict(lr=1e-2, momentum=0.9)
    models = [net(kind) for _ in range(2)]
    opts = [torchsso.optim.SecondOrderOptimizer(m, 'Cov', SHAPES, {'damping': 1e-2, 'ema_decay': 0.5}, acc_steps=2, **options)
            for m in models]
    for t in range(4):
        opts[0].step(closure=closure_of(opts[0], models[0], t))
    torch.save([models[0].state_dict(), opts[0].state_dict()], tmp_path / 'saved')
    saved = torch.load(tmp_path / 'saved', weights_only=True)
    models[1].load_state_dict(saved[0])
    opts[1].load_state_dict(saved[1])
    for t in range(4, 8):
        for model, opt in zip(models, opts):
            opt.step(closure=closure_of(opt, model, t))
    for p, q in zip(*[m.parameters() for m in models]):
        assert torch.isfinite(p).all() and torch.equal(p, q)


@KINDS
def test_posterior(kind):
    model = net(kind)
    opt = torchsso.optim.VIOptimizer(model, dataset_size=1000, curv_type='Cov', curv_shapes=SHAPES,
                                     curv_kwargs={'damping': 1e-3, 'ema_decay': 0.1}, lr=1e-2, num_mc_samples=2)
    before = [p.detach().clone() for p in model[1].parameters()]
    for t in range(4):
        loss, _ = opt.step(closure=closure_of(opt, model, t))
        assert torch.isfinite(torch.as_tensor(loss)).all()
    for p, b in zip(model[1].parameters(), before):
        assert torch.isfinite(p).all() and not torch.equal(p, b)
    curv = opt.param_groups[1]['curv']
    assert len(curv.std) == 2 and all(bool((s > 0).all()) for s in curv.std)
