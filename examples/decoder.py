"""A small pre-norm decoder trained with second-order updates of all its parts, on synthetic text:

    python examples/decoder.py [--steps 400]

  matrices (bfloat16)   torchsso.optim.Muon: momentum, orthogonalised
  gains of the norms    torchsso.optim.SecondOrderOptimizer with DiagCovRMSNorm, whose curvature the
                        norms' backward passes form beside the gradients
  embedding             torch.optim.AdamW

Every block adds its input to the residual stream and normalises the sum in one pass
(torchsso.nn.RMSNorm with two arguments).  Afterwards the model continues a text; the product behind
the last norm then runs in 8 bits, on what the norm has left in 8 bits with a scale per token.

The text follows a rule (the next symbol is a fixed function of the last two, one time in ten any),
so that the loss can come down to about 0.1 log(64) + 0.33 = 0.74.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'pytorch-sso_amd'))

import torchsso  # noqa: E402

VOCAB = 64


def text(batch, tokens, gen, device):
    x = torch.randint(0, VOCAB, (batch, tokens), generator=gen)
    noise = torch.rand((batch, tokens), generator=gen)
    for t in range(2, tokens):
        rule = (3 * x[:, t - 1] + 5 * x[:, t - 2] + 1) % VOCAB
        x[:, t] = torch.where(noise[:, t] < 0.9, rule, x[:, t])
    return x.to(device)


class Block(nn.Module):

    def __init__(self, dim, heads, device):
        super().__init__()
        self.heads = heads
        linear = lambda i, o: nn.Linear(i, o, bias=False, device=device, dtype=torch.bfloat16)
        self.norm1 = torchsso.nn.RMSNorm(dim, device=device)
        self.q, self.k, self.v, self.o = (linear(dim, dim) for _ in range(4))
        self.norm2 = torchsso.nn.RMSNorm(dim, device=device)
        self.up, self.gate, self.down = linear(dim, 4 * dim), linear(dim, 4 * dim), linear(4 * dim, dim)

    def forward(self, x, stream):
        """x: what the layer before adds to the stream.  Returns what this one adds, and the stream."""
        y, stream = self.norm1(x, stream)
        n, t, d = y.shape
        q, k, v = (f(y).view(n, t, self.heads, d // self.heads).transpose(1, 2) for f in (self.q, self.k, self.v))
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2).reshape(n, t, d)
        y, stream = self.norm2(self.o(a), stream)
        return self.down(F.silu(self.gate(y)) * self.up(y)), stream


class Decoder(nn.Module):

    def __init__(self, dim=128, heads=4, layers=2, device='cuda'):
        super().__init__()
        self.embedding = nn.Embedding(VOCAB, dim, device=device)
        self.blocks = nn.ModuleList(Block(dim, heads, device) for _ in range(layers))
        self.norm = torchsso.nn.RMSNorm(dim, device=device)
        self.head = nn.Linear(dim, VOCAB, bias=False, device=device, dtype=torch.bfloat16)

    def body(self, tokens):
        x = self.embedding(tokens).to(torch.bfloat16)
        stream = torch.zeros_like(x)
        for block in self.blocks:
            x, stream = block(x, stream)
        return x, stream

    def forward(self, tokens):
        return self.head(self.norm(*self.body(tokens))[0]).float()

    def head_8(self):
        """The last layer's weight in 8 bits, with a scale for each symbol."""
        scale = (self.head.weight.float().abs().amax(1, keepdim=True) / 448.).clamp_(min=1e-12)
        return (self.head.weight.float() / scale).to(torch.float8_e4m3fn), scale

    @torch.no_grad()
    def logits_8(self, x, stream, weight, scale):
        """Of one token of each text, through the last norm and layer in 8 bits."""
        q, q_scale, _ = torchsso.nn.add_rms_norm(x, stream, self.norm.weight, self.norm.eps,
                                                 out_dtype=torch.float8_e4m3fn)
        return torch._scaled_mm(q, weight.t(), scale_a=q_scale, scale_b=scale.t().contiguous(),
                                out_dtype=torch.bfloat16).float()

    @torch.no_grad()
    def generate(self, tokens, count):
        weight, scale = self.head_8()
        for _ in range(count):
            x, stream = self.body(tokens)
            logits = self.logits_8(x[:, -1], stream[:, -1], weight, scale)
            tokens = torch.cat([tokens, logits.argmax(-1, keepdim=True)], 1)
        return tokens


def main(argv=None):
    parser = argparse.ArgumentParser()
    parser.add_argument('--steps', type=int, default=400)
    parser.add_argument('--batch', type=int, default=64)
    parser.add_argument('--tokens', type=int, default=64)
    args = parser.parse_args(argv)
    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(0)
    model = Decoder()
    norms = nn.ModuleList(m for m in model.modules() if isinstance(m, torchsso.nn.RMSNorm))
    matrices = [m.weight for m in model.modules() if isinstance(m, nn.Linear)]
    optimizers = [torchsso.optim.Muon(matrices, lr=0.02, weight_decay=0.01),
                  torchsso.optim.SecondOrderOptimizer(norms, 'Cov', {'RMSNorm': 'Diag'},
                                                      {'damping': 1e-2, 'ema_decay': 0.1}, lr=1e-2, momentum=0.9),
                  torch.optim.AdamW(model.embedding.parameters(), lr=1e-2)]
    losses = []
    for step in range(args.steps):
        x = text(args.batch, args.tokens + 1, gen, 'cuda')
        model.zero_grad()
        # (the first two symbols of a text follow no rule)
        loss = F.cross_entropy(model(x[:, :-1])[:, 1:].reshape(-1, VOCAB), x[:, 2:].reshape(-1))
        loss.backward()
        for optimizer in optimizers:
            optimizer.step()
        losses.append(loss.item())
        if step % 10 == 0 or step + 1 == args.steps:
            print('step %3d  loss %.3f' % (step, losses[-1]), flush=True)
    start = text(16, 16, gen, 'cuda')
    out = model.generate(start, 16)
    follows = (out[:, 2:] == (3 * out[:, 1:-1] + 5 * out[:, :-2] + 1) % VOCAB)[:, 14:].float().mean().item()
    print('of the symbols that the model adds %.0f %% follow the rule' % (100 * follows))
    return losses, follows


if __name__ == '__main__':
    main()
