"""Clipping over ranks far from 1: gloo, two processes on the CPU."""
import pytest
import torch

from cinema_amd import parallel as par
from test_dp_gloo import WORLD, _run


def _worker(rank):
    g = torch.Generator().manual_seed(5)
    tables, shared = [torch.randn(40 + 7 * r, generator=g) for r in range(WORLD)], torch.randn(90, generator=g)
    for scale in (1e25, 1e30, 1e-25, 1e-30, 0.0):
        t, s = (tables[rank] * WORLD).double() * scale, shared.double() * scale
        want = float(torch.cat(tables + [shared]).double().norm() * scale)
        # the parts arrive as fp32 values, 2^-24 off each
        got = par.union_grad_norm(t.norm().float(), s.norm().float())
        assert abs(float(got) - want) <= want * 2.0 ** -23, scale
        assert abs(float(got.float()) - want) <= want * 2.0 ** -22, scale
    for bad in (float("inf"), float("nan")):
        got = float(par.union_grad_norm(torch.tensor(bad if rank == 1 else 1.0), torch.tensor(1.0)))
        assert str(got) == str(bad)


def test_union_grad_norm_of_large_and_small_gradients():
    _run(_worker)


def test_union_grad_norm_of_one_process_is_64_bit():
    for v in (3e25, 3e-25):
        assert float(par.union_grad_norm(torch.tensor(v), torch.tensor(v))) == pytest.approx(v * 2 ** 0.5, rel=2.0 ** -22)
