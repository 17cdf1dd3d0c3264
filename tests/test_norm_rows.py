"""Norms of more rows than one launch can have threads for (csrc/norm_rows.h)."""
import os
import subprocess

import pytest
import torch

import torchsso

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'pytorch-sso_amd', 'csrc')

PROGRAM = r"""
#include <cstdio>
#include "norm_rows.h"
int main() {
  for (int threads : {256, 1024})
    for (int per : {1, 4})
      for (long rows : {1L, 3L, 4L, 5L, (1L << 21) - 1, 1L << 21, (1L << 21) + 1, (1L << 23) + 3, (1L << 24) + 1, (1L << 25) - 1,
                        1L << 25, (1L << 26) + 5, (1L << 31) - 1}) {
        long next = 0;
        bool ok = true;
        kfac::for_row_ranges(rows, threads, per, [&](long first, long n, unsigned blocks) {
          ok = ok && first == next && n > 0 && (long)blocks * threads < (1L << 32) && (long)blocks * per >= n &&
               (long)(blocks - 1) * per < n;
          next = first + n;
        });
        if (!ok || next != rows) { printf("%d %d %ld\n", threads, per, rows); return 1; }
      }
}
"""


def test_ranges_cover_the_rows_and_fit_a_launch(tmp_path):
    (tmp_path / 'main.cpp').write_text(PROGRAM)
    subprocess.run(['g++', '-std=c++17', '-I', CSRC, str(tmp_path / 'main.cpp'), '-o', str(tmp_path / 'ranges')], check=True)
    out = subprocess.run([str(tmp_path / 'ranges')], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim', [((1 << 26) + 5, 8), ((1 << 24) + 3, 1025)])
def test_many_rows(rows, dim):
    """A wave for each short row, and 256 threads for each long one: more than 2^32 threads in all."""
    few = torch.randn(1, dim, device='cuda').to(torch.bfloat16)
    gain = torch.linspace(0.5, 2., dim, device='cuda')
    want = torchsso.nn.rms_norm(few, gain)
    y = torchsso.nn.rms_norm(few.expand(rows, dim), gain)
    assert y.shape == (rows, dim)
    for first in range(0, rows, 1 << 22):
        assert bool((y[first:first + (1 << 22)] == want).all())


@pytest.mark.gpu
def test_all_streams_of_many_rows():
    rows, dim = (1 << 26) + 5, 8
    gen = torch.Generator(device='cuda').manual_seed(0)
    x, res = (torch.empty(rows, dim, device='cuda', dtype=torch.bfloat16).normal_(generator=gen) for _ in range(2))
    gain = torch.linspace(0.5, 2., dim, device='cuda')
    y, h = torchsso.nn.add_rms_norm(x, res, gain)
    q, scale, stream = torchsso.nn.add_rms_norm(x, res, gain, out_dtype=torch.float8_e4m3fn)
    for part in (slice(0, 3), slice((1 << 25) - 2, (1 << 25) + 2), slice(rows - 3, rows)):
        few_y, few_h = torchsso.nn.add_rms_norm(x[part], res[part], gain)
        few_q, few_scale, _ = torchsso.nn.add_rms_norm(x[part], res[part], gain, out_dtype=torch.float8_e4m3fn)
        assert torch.equal(y[part], few_y) and torch.equal(h[part], few_h) and torch.equal(stream[part], few_h)
        assert torch.equal(q[part].view(torch.uint8), few_q.view(torch.uint8)) and torch.equal(scale[part], few_scale)
