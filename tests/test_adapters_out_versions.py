"""apply_adapters(out=...) counts as a change of its output for autograd: logits that a gradient needs and that
it overwrites are not silently taken as they have become."""
from __future__ import annotations

import pytest
import torch

import nvjsel
from nvjsel import _lib, adapters as module
from nvjsel._tensors import _HERE

B16 = torch.bfloat16


@pytest.fixture
def launches(monkeypatch):
    """The entry point without a GPU; the launches' names."""
    names = []
    monkeypatch.setattr(module, "_require_cuda", lambda *ts: ts[0].device)
    monkeypatch.setattr(module, "_on_device", lambda device: _HERE)
    monkeypatch.setattr(module, "_stream_handle", lambda device: 0)
    monkeypatch.setattr(module, "_workspace", lambda *a: torch.zeros(1))
    monkeypatch.setattr(_lib, "call", lambda name, *a: names.append(name))
    return names


def _operands():
    table = nvjsel.AdapterTable(torch.zeros(2, 512, dtype=B16), torch.zeros(2, 1024, dtype=B16), torch.zeros(2), 8, 6, 16)
    return torch.zeros(3, 8), table, torch.zeros(3, dtype=torch.int32)


def test_the_version_moves(launches):
    x, table, ids = _operands()
    base, out = torch.zeros(3, 6), torch.zeros(3, 6)
    before = base._version, out._version, x._version
    nvjsel.apply_adapters(x, base, table, ids)
    assert (base._version, out._version, x._version) == before
    nvjsel.apply_adapters(x, base, table, ids, out=out)
    assert out._version > before[1] and (base._version, x._version) == (before[0], before[2])
    for view in (base, base.detach(), base[:], base.view(3, 6)):
        version = base._version
        nvjsel.apply_adapters(x, view, table, ids, out=view)
        assert base._version > version
    assert len(launches) == 6


def test_inference_tensors_have_no_version(launches):
    x, table, ids = _operands()
    with torch.inference_mode():
        out = torch.zeros(3, 6)
        assert nvjsel.apply_adapters(x, out, table, ids, out=out) is out
    assert nvjsel.apply_adapters(x, out, table, ids, out=out) is out


def test_saved_tensors_that_were_overwritten(launches):
    x, table, ids = _operands()
    leaf = torch.randn(3, 6, requires_grad=True)
    for change in ("no_grad", "detached"):
        logits = leaf * 1.0
        loss = torch.log_softmax(logits, 1).sum() + (logits * logits).sum()
        if change == "no_grad":
            with torch.no_grad():
                nvjsel.apply_adapters(x, logits, table, ids, out=logits)
        else:
            alias = logits.detach()
            nvjsel.apply_adapters(x, alias, table, ids, out=alias)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.gpu
def test_logits_that_a_gradient_needs():
    g = torch.Generator().manual_seed(1)
    table = nvjsel.pack_adapters(torch.randn(1, 4, 16, generator=g).to(B16).cuda(), torch.randn(1, 50, 4, generator=g).to(B16).cuda())
    x, ids = torch.randn(3, 16, generator=g).cuda(), torch.zeros(3, dtype=torch.int32, device="cuda")
    t = torch.tensor([1, 2, 3], device="cuda")
    leaf = torch.randn(3, 50, generator=g).cuda().requires_grad_()
    for change in ("no_grad", "detached"):
        logits = leaf * 1.0
        r = nvjsel.token_logprobs(logits, t)
        if change == "no_grad":
            with torch.no_grad():
                nvjsel.apply_adapters(x, logits, table, ids, out=logits)
        else:
            alias = logits.detach()
            nvjsel.apply_adapters(x, alias, table, ids, out=alias)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            r.logprobs.sum().backward()
    # elsewhere: the saved logits stay as they are
    logits = leaf * 1.0
    r = nvjsel.token_logprobs(logits, t)
    with torch.no_grad():
        nvjsel.apply_adapters(x, logits, table, ids, out=torch.empty_like(logits))
    r.logprobs.sum().backward()
