"""Where a NaN or an infinity of an adapter's tables and scale shows in the results, and where not."""
from __future__ import annotations

import math

import pytest
import torch

import nvjsel

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("table", ["bf16", "f16"])
@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,rank", [(3, 16), (70, 16), (3, 64), (70, 64), (70, 160)])
def test_places(rows, rank, act, table, bad):
    g = torch.Generator().manual_seed(rank)
    x = torch.randn(rows, 96, generator=g).to(DT[act]).cuda()
    base = torch.randn(rows, 150, generator=g).to(DT[act]).cuda()
    a = (torch.randn(2, rank, 96, generator=g) / 10).to(DT[table])
    b = (torch.randn(2, 150, rank, generator=g) / 10).to(DT[table])
    ids = (torch.arange(rows) % 3 - 1).to(torch.int32).cuda()
    of = ids.cpu() == 1

    def run(a, b, scales):
        return nvjsel.apply_adapters(x, base, nvjsel.pack_adapters(a.cuda(), b.cuda(), scales), ids).cpu()

    clean = run(a, b, [1.0, 2.0])
    for which in ("a", "scale"):
        a_, scales = a.clone(), [1.0, 2.0]
        if which == "a":
            a_[1, rank - 3, 17] = bad
        else:
            scales[1] = bad
        got = run(a_, b, scales)
        assert bool(torch.isnan(got[of]).all()) and torch.equal(got[~of], clean[~of])
    b_ = b.clone()
    b_[1, 149, rank - 1] = bad
    got = run(a, b_, [1.0, 2.0])
    assert not bool(torch.isfinite(got[of][:, 149]).any())
    assert torch.equal(got[~of], clean[~of]) and torch.equal(got[:, :149], clean[:, :149])
