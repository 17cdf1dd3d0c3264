"""Host side of the orthogonalisation: its checks of arguments, and its plan (csrc/orth_plan.h)."""
import ctypes
import os
import subprocess

import pytest
import torch

import torchsso
from torchsso import _hip
from torchsso.utils.linalg import newton_schulz_schedule

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), 'pytorch-sso_amd', 'csrc')


def test_schedule():
    assert newton_schulz_schedule(2, (1.5, -0.5, 0)) == (1.5, -0.5, 0.) * 2
    assert newton_schulz_schedule(2, [(1.5, -0.5, 0), (2., -1., 0.)]) == (1.5, -0.5, 0., 2., -1., 0.)
    for steps, coeffs in ((0, (1.5, -0.5, 0)), (2.5, (1.5, -0.5, 0)), (True, (1.5, -0.5, 0)), (2, ()), (2, (1., 2.)),
                          (2, [(1.5, -0.5, 0)]), (1, (float('nan'), 0, 0)), (1, (float('inf'), 0, 0)),
                          (1, (9., 0., 0.)), (4, (3., 0., 0.)), (8, (3.4, 1., 1.))):
        with pytest.raises(ValueError):
            newton_schulz_schedule(steps, coeffs)


def test_refusals():
    g = torch.zeros(4, 4)
    with pytest.raises(ValueError):
        torchsso.utils.orthogonalize(torch.zeros(4))
    with pytest.raises(ValueError):
        torchsso.utils.orthogonalize(g, eps=0.)
    with pytest.raises(_hip.KfacHipError):
        torchsso.utils.orthogonalize(g)                 # (on the host)
    assert torchsso.utils.orthogonalize([]) == []
    for bad in (dict(lr=-1.), dict(lr=float('nan')), dict(momentum=1.), dict(momentum=-0.1), dict(weight_decay=-1.),
                dict(eps=0.), dict(steps=0), dict(coefficients=(100., 0., 0.))):
        with pytest.raises(ValueError):
            torchsso.optim.Muon([torch.nn.Parameter(g)], **bad)
    with pytest.raises(ValueError):
        torchsso.optim.Muon([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError):
        torchsso.optim.muon([g], [g], [], lr=0.1)


def test_argument_errors_are_codes():
    lib = _hip.load()
    one, big, coeffs = _hip.int_array([4]), _hip.int_array([16385]), _hip.f32_array([3., -4., 2.])
    fake = (ctypes.c_void_p * 1)(1 << 20)
    null = (ctypes.c_void_p * 1)(None)
    need = lib.kfac_orthogonalize_workspace_bytes(1, one, one)
    assert need > 0 and lib.kfac_orthogonalize_workspace_bytes(0, None, None) == 0
    assert lib.kfac_orthogonalize_workspace_bytes(1, big, one) == 0

    def call(rows=one, cols=one, kind=0, src=fake, dst=fake, steps=1, c=coeffs, late=0, ws=1 << 20, size=need):
        return lib.kfac_orthogonalize_batched(1, rows, cols, kind, src, dst, steps, c, 1e-7, late, ws, size, None)
    assert call(rows=big) == 1 and call(rows=_hip.int_array([-1])) == 1
    assert call(kind=3) == 1 and call(kind=-1) == 1
    assert call(src=None) == 1 and call(dst=None) == 1 and call(src=null) == 1 and call(dst=null) == 1
    assert call(steps=0) == 1 and call(c=None) == 1 and call(late=-1) == 1
    assert call(size=need - 1) == 2 and call(ws=None) == 2
    assert call(rows=_hip.int_array([0])) == 0                    # nothing to do
    assert lib.kfac_orthogonalize_batched(0, None, None, 0, None, None, 1, None, 1e-7, 0, None, 0, None) == 0
    assert lib.kfac_muon_update_batched(1, one, one, 0, fake, fake, None, None, None, 0.9, 1, 1, coeffs, 1e-7, 0,
                                        1 << 20, need, None) == 1


PROGRAM = r'''
#include <cstdio>
#include "orth_plan.h"
using namespace kfac;
int main() {
  int n;
  while (scanf("%d", &n) == 1) {
    std::vector<int> r(n), c(n);
    for (int i = 0; i < n; ++i) if (scanf("%d %d", &r[i], &c[i]) != 2) return 1;
    OrthPlan p = orth_plan(n, r.data(), c.data());
    long seen = 0;
    for (auto& b : p.batches) {
      long end = 0;
      int count = 0, at = b.first;
      if ((int)b.groups.size() > ORTH_GROUPS) return 2;
      for (auto& g : b.groups) {
        if (g.first != at) return 3;
        at += g.count;
        count += g.count;
        if (g.R % g.pad || g.C % g.pad || b.pad % g.pad || g.R < g.r || g.C < g.c || g.r > g.c) return 4;
        const long x = 2L * g.R * g.C * g.count, a = 2L * g.R * g.R * g.count;
        // the four operands lie behind one another and behind the group before
        if (g.x[0] != end || g.x[1] != end + x || g.a != end + 2 * x || g.b != end + 2 * x + a) return 5;
        end += 2 * x + 2 * a;
        for (int k = g.first; k < g.first + g.count; ++k) {
          const int i = p.order[k];
          if (std::min(r[i], c[i]) != g.r || std::max(r[i], c[i]) != g.c) return 6;
        }
      }
      if (end > p.halves || count != b.count) return 7;
      for (int product = 0; product < 3; ++product)
        for (int kind = -1; kind < ORTH_KINDS; ++kind) {
          // the launch that is chosen, and those of all kinds that the padding allows
          OrthLaunch l;
          if (kind < 0) l = orth_launch(b, product);
          else if (ORTH_KIND[kind].tile > b.pad) continue;
          else orth_schedule(b, product, kind, l);
          const int T = ORTH_KIND[l.kind].tile;
          std::vector<int> owner(l.blocks, -1), fixed(l.fixes, -1);
          for (size_t i = 0; i < b.groups.size(); ++i) {
            const OrthGroup& g = b.groups[i];
            const OrthSlice& s = l.slices[i];
            if (s.tile > T || g.R % s.tile || g.C % s.tile) return 8;
            const long t = g.R / s.tile;
            if (s.tiles != g.count * (product == ORTH_APPLY ? t * (g.C / s.tile) : t * (t + 1) / 2)) return 9;
            if (s.whole < 0 || s.whole > s.tiles || (s.whole < s.tiles && s.cuts < 1)) return 10;
            if (s.tile0 % 8 || s.tile0 + (s.whole + 7) / 8 * 8 > l.pieces0) return 11;
            for (int k = 0; k < (s.whole + 7) / 8 * 8; ++k)
              if (owner[s.tile0 + k]++ != -1) return 12;
            if (s.cuts == 0) continue;
            // the pieces cover the reduction, none of them is empty
            const int all = (product == ORTH_GRAM ? g.C : g.R) / 64;
            if (s.len < 1 || s.len * s.cuts < all || s.len * (s.cuts - 1) >= all) return 13;
            if (s.piece0 < l.pieces0) return 14;
            for (int k = 0; k < (s.tiles - s.whole) * s.cuts; ++k)
              if (owner[s.piece0 + k]++ != -1) return 15;
            for (int k = 0; k < s.tiles - s.whole; ++k)
              if (s.fix0 + k >= l.fixes || fixed[s.fix0 + k]++ != -1) return 16;
          }
          for (int o : fixed) if (o != 0) return 17;
          for (int o : owner) if (o != 0) return 17;
          if ((long)(l.blocks - l.pieces0) * T * T * 4 > ORTH_PARTIAL_BYTES) return 18;
        }
      seen += count;
    }
    printf("%ld %ld %ld\n", seen, (long)p.batches.size(), p.halves);
  }
}
'''


@pytest.fixture(scope='module')
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp('orth')
    (d / 'main.cpp').write_text(PROGRAM)
    subprocess.run(['g++', '-std=c++17', '-I', CSRC, str(d / 'main.cpp'), '-o', str(d / 'plan')], check=True)

    def run(shapes):
        text = '%d %s' % (len(shapes), ' '.join('%d %d' % s for s in shapes))
        out = subprocess.run([str(d / 'plan')], input=text, capture_output=True, text=True)
        assert out.returncode == 0, 'plan check %d' % out.returncode
        return [int(v) for v in out.stdout.split()]
    return run


def test_plan_covers_every_matrix_once(plan):
    assert plan([(4, 4)])[:2] == [1, 1]
    assert plan([(4, 0), (0, 0), (5, 3)])[0] == 1
    many = [(3 + i, 70 + i) for i in range(100)]
    assert plan(many)[0] == 100 and plan(many)[1] > 1
    mixed = [(1000, 784), (10, 1000), (1000, 1000), (64, 147), (16384, 16384), (784, 1000)]
    assert plan(mixed)[0] == len(mixed)
    # tiles that fill the chip unevenly, and long reductions of few tiles
    for shapes in ([(4096, 9216), (4096, 4096), (1000, 4096)], [(10, 16384)], [(64, 16384), (300, 5000)],
                   [(512, 4608)] * 3 + [(64, 576)] * 3 + [(2048, 512)] * 3, [(2048, 2048)] * 9 + [(600, 700)],
                   [(16384, 16384)], [(1, 1)] * 40, [(513, 513)] * 31):
        assert plan(shapes)[0] == len(shapes)
    # matrices that do not fit a batch together share the scratch one after another
    one, five = plan([(16384, 16384)]), plan([(16384, 16384)] * 5)
    assert five[0] == five[1] == 5 and five[2] == one[2]
