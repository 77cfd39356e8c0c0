"""Adapters of f32 rows, and factors between the two products, next to the largest finite number."""
from __future__ import annotations

import pytest
import torch

import nvjsel

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
MAX = torch.finfo(torch.float32).max


@pytest.mark.parametrize("table", ["bf16", "f16"])
@pytest.mark.parametrize("rows,rank", [(5, 16), (40, 16), (5, 64), (40, 64), (40, 160)])
def test_largest_activations(rows, rank, table):
    """The largest finite x, alone in its row: one product of each sum, so that y has its roundings to terms (2^-21 beside its
    f32 sum's and scale's 2^-23 each at most) and the second sum 3 R additions of magnitudes."""
    g = torch.Generator().manual_seed(rank + rows)
    x = torch.zeros(rows, 64)
    x[torch.arange(rows), torch.arange(rows) % 64] = MAX * torch.where(torch.arange(rows) % 2 == 0, 1.0, -1.0)
    x[0, 0] = 3.3961e38
    a = (0.5 + torch.rand(1, rank, 64, generator=g)) * 2.0 ** -12
    b = torch.randn(1, 90, rank, generator=g) * 2.0 ** -14
    a, b = a.to(DT[table]), b.to(DT[table])
    base = torch.zeros(rows, 90)
    got = nvjsel.apply_adapters(x.cuda(), base.cuda(), nvjsel.pack_adapters(a.cuda(), b.cuda()),
                                torch.zeros(rows, dtype=torch.int32, device="cuda")).cpu()
    y = x.double() @ a[0].double().T
    size = y.abs() @ b[0].double().abs().T
    tol = size * (2.0 ** -20 + (3 * rank + 4) * 2.0 ** -23) + y.abs().amax(1, keepdim=True) * 2.0 ** -38 * b[0].double().abs().sum(1)
    assert bool(torch.isfinite(got).all()) and bool(((got.double() - y @ b[0].double().T).abs() <= tol).all())


@pytest.mark.parametrize("table", ["bf16", "f16"])
@pytest.mark.parametrize("rows,rank", [(5, 16), (40, 64)])
def test_largest_factors(rows, rank, table):
    """y itself next to the largest finite number: one product, 2^127 (1 + 254/256) and more."""
    x = torch.zeros(rows, 32)
    x[:, 3] = torch.tensor(MAX)
    a = torch.zeros(1, rank, 32)
    a[0, :, 3] = 1.0
    b = torch.zeros(1, 70, rank)
    b[0, torch.arange(70), torch.arange(70) % rank] = 2.0 ** -14
    got = nvjsel.apply_adapters(x.cuda(), torch.zeros(rows, 70, device="cuda"),
                                nvjsel.pack_adapters(a.to(DT[table]).cuda(), b.to(DT[table]).cuda()),
                                torch.zeros(rows, dtype=torch.int32, device="cuda")).cpu()
    want = MAX * 2.0 ** -14
    assert bool(((got.double() - want).abs() <= want * 2.0 ** -20).all())
