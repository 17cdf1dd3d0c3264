"""How much scratch an orthogonalisation asks for, and how much of it is kept."""
import os
import random
import subprocess

import pytest
import torch

import torchsso
from torchsso import _hip

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'pytorch-sso_amd', 'csrc')

PROGRAM = r"""
#include <cstdio>
#include "orth_plan.h"
using namespace kfac;
int main() {
  int n;
  while (scanf("%d", &n) == 1) {
    std::vector<int> r(n), c(n);
    for (int i = 0; i < n; ++i) if (scanf("%d %d", &r[i], &c[i]) != 2) return 1;
    const OrthPlan p = orth_plan(n, r.data(), c.data(), true);
    for (const OrthBatch& b : p.batches)
      for (int product = 0; product < 3; ++product) {
        const OrthLaunch l = orth_launch(b, product);
        const long T = ORTH_KIND[l.kind].tile;
        if ((long)(l.blocks - l.pieces0) * T * T * 4 > orth_partial_bytes(b) || orth_partial_bytes(b) > ORTH_PARTIAL_BYTES) return 2;
      }
  }
}
"""


def need(shapes):
    rows, cols = _hip.int_array([r for r, _ in shapes]), _hip.int_array([c for _, c in shapes])
    return _hip.load().kfac_orthogonalize_workspace_bytes(len(shapes), rows, cols)


def test_the_pieces_fit(tmp_path):
    (tmp_path / 'main.cpp').write_text(PROGRAM)
    subprocess.run(['g++', '-std=c++17', '-I', CSRC, str(tmp_path / 'main.cpp'), '-o', str(tmp_path / 'plan')], check=True)
    rng = random.Random(0)
    side = lambda: int(round(2 ** rng.uniform(0, 14)))
    lists = [[(side(), side())] * rng.choice([1, 1, 3, 16]) + [(side(), side()) for _ in range(rng.randint(0, 8))]
             for _ in range(400)]
    lists += [[(517, 301), (1263, 517), (37, 1263)], [(1024, 2752)] * 16, [(4096, 9216), (4096, 4096), (1000, 4096)], [(10, 16384)],
              [(512, 4608)] * 3 + [(64, 576)] * 3, [(2048, 2048)] * 9 + [(600, 700)]]
    text = '\n'.join('%d %s' % (len(s), ' '.join('%d %d' % m for m in s)) for s in lists)
    assert subprocess.run([str(tmp_path / 'plan')], input=text, text=True).returncode == 0


def test_small_matrices_ask_for_little():
    # 2 X, A and B of a padded 100 x 100, in two parts: 4 * (128^2 + 128^2) halves, and tables
    assert need([(100, 100)]) < 4 * 2 * 128 * 128 * 2 + (1 << 17)
    assert need([(1000, 784), (1000, 1000), (10, 1000)]) < 64 << 20


def test_large_scratch_is_not_doubled(monkeypatch):
    empty = torch.empty
    monkeypatch.setattr(torch, 'empty', lambda size, dtype, device: empty(size, dtype=dtype, device='meta'))
    monkeypatch.setattr(_hip, 'stream_ptr', lambda device=None, stream=None: 1)
    workspace, device = _hip._Workspace(), torch.device('cuda', 0)
    last = 0
    for nbytes in (1, 1000, (1 << 20) + 1, 100 << 20, (256 << 20) + 1, (1 << 30) + 1, (1 << 30) + (70 << 20), (5 << 30) + 3):
        buf, size = workspace.get(device, nbytes)
        assert size == buf.numel() >= nbytes
        assert size <= max(2 * nbytes, 1 << 20) if nbytes <= 1 << 28 else size <= nbytes * 1.125
        # what grows slowly does not allocate each time
        assert workspace.get(device, size)[0] is buf


def test_the_pieces_of_narrow_matrices_beside_wider_ones_fit(tmp_path):
    """(64-wide tiles in a launch of 128-wide ones, whose reductions are cut into more pieces)"""
    (tmp_path / 'main.cpp').write_text(PROGRAM)
    subprocess.run(['g++', '-O2', '-std=c++17', '-I', CSRC, str(tmp_path / 'main.cpp'), '-o', str(tmp_path / 'plan')], check=True)
    rng = random.Random(1)
    side = lambda low, high: int(round(2 ** rng.uniform(low, high)))
    lists = [[(9, 5835), (65, 65), (16, 628)], [(51, 5863), (288, 343)], [(50, 5329), (329, 185)], [(64, 16384), (65, 70)]]
    lists += [[(side(0, 6), side(6, 14)) for _ in range(rng.randint(1, 4))] + [(side(6, 10), side(6, 12)) for _ in range(rng.randint(1, 5))]
              for _ in range(3000)]
    text = '\n'.join('%d %s' % (len(s), ' '.join('%d %d' % m for m in s)) for s in lists)
    assert subprocess.run([str(tmp_path / 'plan')], input=text, text=True).returncode == 0


@pytest.mark.gpu
@pytest.mark.parametrize('shapes', [[(9, 5835), (65, 65), (16, 628)], [(51, 5863), (288, 343)], [(64, 16384), (65, 70)]])
def test_narrow_matrices_beside_wider_ones(shapes):
    mats = [torch.randn(s, generator=torch.Generator().manual_seed(i)).cuda() for i, s in enumerate(shapes)]
    for m, o in zip(mats, torchsso.utils.orthogonalize(mats)):
        x = m.double() / (m.double().norm() + 1e-7)
        for _ in range(5):
            a = x @ x.t().contiguous()
            x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
        # (15 products round operands to 2^-23, which grows by 1.5 in each step behind, if all errors are of one sign)
        assert (o.double() - x).norm() <= 4.7e-5 * x.norm()
