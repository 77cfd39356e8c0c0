"""Adapters of rows whose first element lies behind 2^31: x, base and out, in place and elsewhere."""
from __future__ import annotations

import pytest
import torch

import nvjsel
from tests.test_adapters_gpu import make, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [16, 40, 160])
@pytest.mark.parametrize("rows", [9, 40])  # more than 32 rows: kernels of their own
def test_rows_behind_2_31(rows, rank):
    stride = (1 << 28) if rows == 9 else (1 << 26) + 72  # element 2^31 lies in row 8, in row 31
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    x, y, a, b, s, ids = make(rows, 136, 500, [rank] * 3, seed=31)
    ids[:] = torch.arange(rows) % 4 - 1
    ids[-1] = 2  # behind 2^31, with an adapter
    want, tol = oracle(x, y, a, b, s, ids)
    table = nvjsel.pack_adapters([t.cuda() for t in a], [t.cuda() for t in b], s)
    buf = torch.zeros(rows, stride, dtype=torch.bfloat16, device="cuda")
    xv, base, out = buf[:, 3:139], buf[:, 207:707], buf[:, 1001:1501]
    xv.copy_(x)
    base.copy_(y)

    def check(got, rest):
        err = (got.double().cpu() - want).abs()
        assert bool((err <= tol).all()), (err / tol.clamp(min=1e-300)).max()
        head = buf[:, :2000].cpu()
        for first, last, value in rest:
            assert torch.equal(head[:, first:last], value.expand(rows, last - first))
        assert not bool((buf[:, 2000:].view(torch.int16) != 0).any())

    nothing = torch.zeros(1, 1, dtype=torch.bfloat16)
    around = [(0, 3, nothing), (3, 139, x), (139, 207, nothing), (707, 1001, nothing), (1501, 2000, nothing)]
    check(nvjsel.apply_adapters(xv, base, table, ids.cuda(), out=out), around + [(207, 707, y)])
    out.zero_()
    check(nvjsel.apply_adapters(xv, base, table, ids.cuda(), out=base), around + [(1001, 1501, nothing)])
